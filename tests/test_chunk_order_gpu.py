"""q_starts that descend or leave [0, total_q]: the sequence whose rows they bound and all behind it are
skipped and reported, so that no row has two owners; the sequences before it are computed as if the batch
ended there. A sequence of more rows than the host's bound is skipped alone."""
import pytest

import _chunk
from _chunk import NKV, call, make, reference
from test_chunk_attn_gpu import in_line_form

pytestmark = pytest.mark.gpu


def batch_of(form):
    """Sequences, and the index of the one whose rows are broken (its neighbours have rows)."""
    if form in ("cluster", "line"):
        return [(2, 700), (3, 300), (1, 90), (4, 1200), (2, 33)], 1
    if form == "line_large":  # more sequences than a warp's scan holds
        return [(1 + i % 4, 5 + 11 * i) for i in range(140)], 77
    if form == "pair":
        return [(2, 700), (70, 300), (5, 90), (130, 1200), (9, 33)], 1
    return [(1 + i % 9, 9 + 7 * (i % 61)) for i in range(300)], 200


def run(cuda, form, starts=None, qmax=None):
    """One call with weights; (the batch, its outputs, its weights)."""
    import torch
    seqs, at = batch_of(form)
    c = make(seqs, seed=30, rows_behind=2, gate=True)
    if form == "line":
        c = in_line_form(c)
    w = torch.ones((len(seqs), NKV, c["lmax"]), device="cuda")
    d = c if starts is None else dict(c, q_starts=torch.tensor(starts(list(c["starts"]), at), dtype=torch.int32, device="cuda"))
    out, lse = call(cuda, d, weights=w, qmax=qmax)
    torch.cuda.synchronize()
    return c, at, out, lse, w


def check(c, owners, out, lse, w):
    """The rows and weights of `owners` are right; no other is touched."""
    import torch
    rout, tol, rlse, ltol, rw = reference(c)
    own = torch.zeros(c["rows"], dtype=torch.bool, device="cuda")
    for b, (n, L) in enumerate(c["seqs"]):
        if b not in owners:
            assert (w[b] == 1).all()
            continue
        own[c["starts"][b]:c["starts"][b + 1]] = True
        assert ((w[b, :, :L].double() - 1 - rw[b][0]).abs() <= rw[b][1] + 2.0 ** -23 * (1 + rw[b][0])).all()
    assert ((out.double() - rout).abs()[own] <= tol[own]).all() and ((lse.double() - rlse).abs()[own] <= ltol[own]).all()
    assert (out[~own].float() == 7).all() and (lse[~own] == -7).all()


def descend(starts, at):
    # the next sequences have the rows of the one before again
    starts[at + 1] = starts[at] - 1
    return starts


def far_down(starts, at):
    starts[at + 1] = 0
    return starts


def negative(starts, at):
    starts[at + 1] = -3
    return starts


def leave(starts, at):
    starts[at + 1] = 1 << 30
    return starts


FORMS = ["cluster", "line", "line_large", "pair", "pair_large"]


@pytest.mark.parametrize("starts", [descend, far_down, negative, leave])
@pytest.mark.parametrize("form", FORMS)
def test_skipped_from_the_first_out_of_order(cuda, form, starts):
    c, at, out, lse, w = run(cuda, form, starts)
    assert cuda.device_error()[0] == 707
    check(c, range(at), out, lse, w)


@pytest.mark.parametrize("form", FORMS)
def test_nothing_before_the_first(cuda, form):
    c, at, out, lse, w = run(cuda, form, lambda s, at: [s[1] + 1] + s[1:])
    assert cuda.device_error() == (707, 0)
    check(c, (), out, lse, w)


@pytest.mark.parametrize("form", FORMS)
def test_too_many_rows_are_one_sequence(cuda, form):
    """One entry moved down: its sequence has fewer rows, the next more than the bound, and is skipped."""
    import torch
    seqs, at = batch_of(form)
    qmax = max(n for n, _ in seqs)
    at = max(b for b in range(1, len(seqs)) if seqs[b][0] == qmax)
    c, _, out, lse, w = run(cuda, form, lambda s, _: s[:at] + [s[at] - 1] + s[at + 1:], qmax=qmax)
    assert cuda.device_error() == (707, at)
    # the one before lost its last row: what it sees is another batch, so only the others are compared
    lost = slice(c["starts"][at - 1], c["starts"][at])
    assert (w[at] == 1).all() and (out[c["starts"][at]:c["starts"][at + 1]].float() == 7).all()
    out[lost], lse[lost], w[at - 1] = 7, -7, 1
    check(c, [b for b in range(len(seqs)) if b not in (at - 1, at)], out, lse, w)


@pytest.mark.parametrize("form", ["cluster", "line", "pair"])
def test_same_bits_beside_broken_rows(cuda, form):
    """Where two sequences owned the same rows, their results raced."""
    import torch
    runs = [run(cuda, form, descend)[2:] for _ in range(40)]
    assert cuda.device_error()[0] == 707
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))
