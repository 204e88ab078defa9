"""Attention whose scores all lie far from zero, against the float64 reference and the bounds of
_chunk.py. The softmax subtracts the row's own maximum: anything else that got into it, a stray value
near zero for instance, would let every probability underflow (scores near -256) and the row come out 0."""
import pytest

import _chunk

pytestmark = pytest.mark.gpu


def far(seqs, sign, seed):
    """q near 4, k near +-4: scores of +-256, spread by some 3."""
    import torch
    c = _chunk.make(seqs, seed=seed)
    c["q"] = (4 + 0.5 * c["q"].float()).to(torch.bfloat16)
    c["k"] = (4 * sign + 0.5 * c["k"].float()).to(torch.bfloat16)  # stale slots stay NaN
    return c


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("prefix,rows", [(0, 1), (0, 130), (100, 70), (777, 129), (3000, 37), (9000, 96)])
def test_prefill(cuda, prefix, rows, sign):
    import torch
    c = far([(rows, prefix + rows)], sign, prefix + rows)
    out = torch.full((rows, 16, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    n = cuda.prefill_workspace_bytes(prefix, rows)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda") if n else None
    cuda.prefill_attn(c["q"], c["k"], c["v"], c["tables"][0], prefix, rows, _chunk.SCALE, out, ws)
    ref, bound = _chunk.reference(c)[:2]
    assert ((out.double() - ref).abs() <= bound).all()
    assert cuda.device_error() == (0, 0)


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("seqs", [[(3, 900), (1, 40), (4, 4)], [(1, 17 + 50 * i) for i in range(50)], [(90, 900), (20, 4000), (1, 5)]])
def test_ragged(cuda, seqs, sign):
    import torch
    c = far(seqs, sign, len(seqs))
    before = torch.zeros((len(seqs), 4, c["lmax"]), device="cuda")
    w = before.clone()
    got = _chunk.call(cuda, c, weights=w)
    _chunk.check(c, got, _chunk.reference(c), w, before)
    assert cuda.device_error() == (0, 0)


@pytest.mark.parametrize("sign", [-1, 1])
def test_uniform_decode(cuda, sign):
    import torch
    c = far([(2, 4097), (2, 900), (2, 17)], sign, 3)
    out = torch.empty((c["rows"], 16, 256), dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(cuda.decode_workspace_bytes(3, 2, c["lmax"]), dtype=torch.uint8, device="cuda")
    cuda.decode_attn(c["q"], c["k"], c["v"], c["tables"], c["seq_lens"], c["lmax"], _chunk.SCALE, out, ws, num_queries=2)
    ref, bound = _chunk.reference(c)[:2]
    assert ((out.double() - ref).abs() <= bound).all()
    assert cuda.device_error() == (0, 0)
