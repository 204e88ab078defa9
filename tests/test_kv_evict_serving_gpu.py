"""Selection and compaction as a server calls them: in a captured graph that is replayed with other lengths,
behind one another without the host, and over pools and weight rows past 2^31 elements."""
import numpy as np
import pytest

import _chunk
from _chunk import D, NKV, PAGE
from test_chunk_attn_gpu import in_line_form
from test_kv_evict_gpu import ref_select

pytestmark = pytest.mark.gpu


def i32(x):
    import torch
    return torch.as_tensor(x, dtype=torch.int32).cuda()


def pools(pages, gen):
    """Random bit patterns."""
    import torch
    return [torch.randint(-32768, 32768, (pages, NKV, PAGE, D), generator=gen, device="cuda", dtype=torch.int16) for _ in range(2)]


def gathered(pool, table, ids, h):
    """Rows `ids` of kv head h in a paged pool."""
    import torch
    t = torch.from_numpy(np.asarray(ids)).cuda()
    return pool[table.long()[t // PAGE], h, t % PAGE]


def test_graph_replay_with_other_lengths(cuda):
    import torch
    lmax, budget, first, last, batch = 3000, 100, 3, 20, 4
    gen = torch.Generator(device="cuda").manual_seed(50)
    rng = np.random.default_rng(50)
    per, fresh = -(-lmax // PAGE), -(-budget // PAGE)
    k, v = pools(batch * per, gen)
    dk, dv = (torch.zeros((batch * fresh, NKV, PAGE, D), dtype=torch.int16, device="cuda") for _ in range(2))
    tables, dst = i32(rng.permutation(batch * per).reshape(batch, per)), i32(rng.permutation(batch * fresh).reshape(batch, fresh))
    w, out = (torch.zeros((batch, NKV, lmax), device="cuda") for _ in range(2))
    lens, kept, new = i32([lmax] * batch), torch.zeros((batch, NKV, budget), dtype=torch.int32, device="cuda"), i32([0] * batch)

    def both():
        cuda.kv_evict_select(w, lens, lmax, budget, first, last, kept, new, weights_out=out)
        cuda.kv_evict_compact(k, v, tables, kept, dk, dv, dst)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for now in ([3000, 2999, 101, 100], [0, 1, 99, 513], [0, 0, 0, 0], [4, 1500, 0, 3000]):
        host = rng.random((batch, NKV, lmax), dtype=np.float32)
        w.copy_(torch.from_numpy(host))
        lens.copy_(i32(now))
        for x in (out, dk, dv):
            x.fill_(-5)
        graph.replay()
        torch.cuda.synchronize()
        assert new.tolist() == [min(n, budget) for n in now]
        want_out, want_k, want_v = torch.full_like(out, -5), torch.full_like(dk, -5), torch.full_like(dv, -5)
        for b, n in enumerate(now):
            for h in range(NKV):
                ids = ref_select(host[b, h], n, budget, first, last)
                assert np.array_equal(kept[b, h].cpu().numpy(), np.concatenate([ids, np.full(budget - len(ids), -1)]))
                want_out[b, h, :n] = 0
                want_out[b, h, :len(ids)] = torch.from_numpy(host[b, h, ids]).cuda()
                i = torch.arange(len(ids), device="cuda")
                want_k[dst[b].long()[i // PAGE], h, i % PAGE] = gathered(k, tables[b], ids, h)
                want_v[dst[b].long()[i // PAGE], h, i % PAGE] = gathered(v, tables[b], ids, h)
        assert torch.equal(out, want_out) and torch.equal(dk, want_k) and torch.equal(dv, want_v)
    assert cuda.device_error() == (0, 0)


@pytest.mark.parametrize("seqs", [[(2, 700), (1, 300), (4, 90)], [(2, 700), (80, 300), (30, 1500)]])
def test_back_to_back(cuda, seqs):
    """Attention with weights, selection in place, compaction and attention over the compacted cache, over and
    over with nothing between the launches: each starts before the one ahead of it has ended. Every round is
    from the same start, so all must agree; two streams run the same on memory of their own at once."""
    import torch
    budget, rounds = 64, 60
    batch, fresh = len(seqs), 4

    class Run:
        def __init__(self):
            self.c = _chunk.make(seqs, seed=51, stale=0.0)
            self.stream = torch.cuda.Stream()
            self.start = torch.rand((batch, NKV, self.c["lmax"]), generator=torch.Generator(device="cuda").manual_seed(52), device="cuda")
            self.ws = torch.empty(cuda.chunk_workspace_bytes(batch, self.c["rows"], self.c["qmax"], self.c["lmax"], True),
                                  dtype=torch.uint8, device="cuda")
            self.dst = torch.arange(batch * fresh, device="cuda").to(torch.int32).reshape(batch, fresh)
            self.results = []

        def round(self):
            c = self.c
            w = self.start.clone()
            kept = torch.empty((batch, NKV, budget), dtype=torch.int32, device="cuda")
            new = torch.empty(batch, dtype=torch.int32, device="cuda")
            dk, dv = (torch.zeros((batch * fresh, NKV, PAGE, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
            out, lse = _chunk.call(cuda, c, weights=w, workspace=self.ws)
            cuda.kv_evict_select(w, c["seq_lens"], c["lmax"], budget, 2, 8, kept, new, weights_out=w)
            cuda.kv_evict_compact(c["k"], c["v"], c["tables"], kept, dk, dv, self.dst)
            short = dict(c, k=dk, v=dv, tables=self.dst, seq_lens=new)
            out2, lse2 = _chunk.call(cuda, short, weights=w, lmax=budget, workspace=self.ws)
            self.results.append((out, lse, w, kept, new, dk, dv, out2, lse2))

    runs = [Run(), Run()]
    torch.cuda.synchronize()
    for _ in range(rounds):
        for r in runs:
            with torch.cuda.stream(r.stream):
                r.round()
    torch.cuda.synchronize()
    assert cuda.device_error() == (0, 0)
    want = runs[0].results[0]
    for r in runs:
        for got in r.results:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    # and the first round is right: its selection, and the attention over what it kept
    c, (out, lse, w, kept, new, dk, dv, out2, lse2) = runs[0].c, want
    assert new.tolist() == [min(L, budget) for _, L in seqs]
    for b, (n, L) in enumerate(seqs):
        for h in range(NKV):
            ids = kept[b, h, :min(L, budget)].cpu().numpy()
            assert torch.equal(gathered(dk, runs[0].dst[b], np.arange(len(ids)), h), gathered(c["k"], c["tables"][b], ids, h))
            assert torch.equal(gathered(dv, runs[0].dst[b], np.arange(len(ids)), h), gathered(c["v"], c["tables"][b], ids, h))
    short = dict(c, seqs=[(n, min(L, budget)) for n, L in seqs], k=dk, v=dv, tables=runs[0].dst, seq_lens=new)
    _chunk.check(short, (out2, lse2), _chunk.reference(short))


def test_compact_past_2_31_elements(cuda):
    """Source pages at the end of a pool of more than 2^31 elements, destination pages at the end of another."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(53)
    pages = (1 << 31) // (NKV * PAGE * D) + 40
    k, v, dk, dv = (torch.zeros((pages, NKV, PAGE, D), dtype=torch.int16, device="cuda") for _ in range(4))
    k[-20:], v[-20:] = pools(20, gen)
    tables, dst = i32([list(range(pages - 20, pages))]), i32([[pages - 1, pages - 3]])
    kept = torch.randperm(320, generator=gen, device="cuda")[:32].sort().values.to(torch.int32).repeat(1, NKV, 1).contiguous()
    cuda.kv_evict_compact(k, v, tables, kept, dk, dv, dst)
    torch.cuda.synchronize()
    assert cuda.device_error() == (0, 0)
    ids = kept[0, 0].cpu().numpy()
    for pool, to in ((k, dk), (v, dv)):
        for h in range(NKV):
            assert torch.equal(gathered(to, dst[0], np.arange(32), h), gathered(pool, tables[0], ids, h))
        assert (to[:-3] == 0).all() and (to[-2] == 0).all()


def test_weights_past_2_31_elements(cuda):
    """Slots whose rows lie past 2^31 elements, for the selection and for both ways of adding weights."""
    import torch
    stride = 1 << 18
    slots = (1 << 31) // (NKV * stride) + 3
    w = torch.zeros((slots, NKV, stride), device="cuda")
    rng = np.random.default_rng(54)
    host = rng.random((2, NKV, 5000), dtype=np.float32)
    at, lens = [slots - 1, slots - 3], [5000, 3000]
    for i, s in enumerate(at):
        w[s, :, :5000] = torch.from_numpy(host[i]).cuda()
    kept = torch.zeros((2, NKV, 700), dtype=torch.int32, device="cuda")
    cuda.kv_evict_select(w, i32(lens), stride, 700, 4, 64, kept, weights_out=w, slots=i32(at))
    torch.cuda.synchronize()
    assert cuda.device_error() == (0, 0)
    for i, s in enumerate(at):
        for h in range(NKV):
            ids = ref_select(host[i, h], lens[i], 700, 4, 64)
            assert np.array_equal(kept[i, h].cpu().numpy(), ids)
            row = w[s, h, :5000].cpu().numpy()
            assert np.array_equal(row[:700], host[i, h, ids]) and (row[700:lens[i]] == 0).all()
            assert np.array_equal(row[lens[i]:], host[i, h, lens[i]:])
    for seqs in ([(2, 300), (1, 900)], [(2, 300), (70, 900)]):
        c = _chunk.make(seqs, seed=55)
        small = torch.ones((2, NKV, c["lmax"]), device="cuda")
        _chunk.call(cuda, c, weights=small)
        for i, s in enumerate(at):
            w[s].fill_(1)
        _chunk.call(cuda, c, weights=w, slots=i32(at))
        assert cuda.device_error() == (0, 0)
        for i, s in enumerate(at):
            assert torch.equal(w[s, :, :c["lmax"]], small[i]) and (w[s, :, c["lmax"]:] == 1).all()


def test_scores_past_2_31_elements(cuda):
    """A bound on the lengths that makes the score workspace of short rows larger than 2^31 floats."""
    import torch
    lmax = 1 << 21
    seqs = [(4, 50 + 90 * i) for i in range(17)]
    c = _chunk.make(seqs, seed=56)
    before = torch.rand((17, NKV, c["lmax"]), device="cuda")
    large = torch.nn.functional.pad(before, (0, lmax - c["lmax"]))
    got = _chunk.call(cuda, in_line_form(c, lmax), weights=large)
    assert cuda.device_error() == (0, 0)
    _chunk.check(c, got, _chunk.reference(c), large[:, :, :c["lmax"]], before)
    assert (large[:, :, c["lmax"]:] == 0).all()
