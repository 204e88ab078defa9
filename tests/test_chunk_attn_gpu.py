"""pgc_chunk_attn and pgc_chunk_attn_weights (ragged-batch attention over the paged cache) against a
float64 reference, through the C ABI, with the bounds derived in _chunk.py."""
import pytest

import _chunk
from _chunk import NKV, call, check, make, reference

pytestmark = pytest.mark.gpu

# (query rows, cached tokens) of the sequences of a batch; up to 4 rows each: the split kernel
SMALL = {
    "one_token": [(1, 1)],
    "config1": [(1, 4097)],
    "page_edges": [(1, 15), (1, 16), (1, 17), (1, 64), (1, 65), (2, 1024), (1, 1025)],
    "mixed_rows": [(4, 4), (1, 1), (0, 5), (2, 17), (3, 3000), (4, 1000)],
    "nothing_cached": [(1, 0), (2, 1), (4, 2), (1, 33)],
    "only_nothing": [(1, 0), (0, 0)],
    "long": [(1, 20000), (1, 100), (2, 7)],
    "many": [(1 + i % 4, 5 + 37 * i) for i in range(40)],
    "no_rows": [(0, 5), (0, 0)],
    "batch_129": [(i % 5, 3 + 5 * (i % 97)) for i in range(129)],
    "batch_4096": [(1 + i % 2, 1 + i % 40) if i % 8 == 0 else (0, 3) for i in range(4096)],
}
LARGE = {
    "five": [(5, 5)],
    "tile_edges": [(64, 64), (65, 65), (1, 300), (0, 7), (33, 1000), (63, 127), (8, 128), (9, 129)],
    "negative_positions": [(200, 190), (70, 3), (10, 0), (6, 6)],
    "chunk_over_prefix": [(130, 4000)],
    "one_of_all": [(600, 2111)],
    "long_prefix_few_rows": [(7, 20000), (512, 3000)],
    "tiny_chunks": [(5 + i % 60, 200 + 31 * i) for i in range(40)],
    "chunk_from_nothing": [(1000, 1000)],
    "decode_among_chunks": [(1, 700), (300, 900), (1, 1), (4, 5000), (0, 0), (129, 130)],
    "batch_300": [(i % 9, 9 + 7 * (i % 61)) for i in range(300)],
    "batch_4096_chunks": [(5, 5 + i % 30) if i % 8 == 0 else (0, 7) for i in range(4096)],
}


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("name", list(SMALL) + list(LARGE))
def test_against_reference(cuda, name, weights):
    import torch
    seqs = SMALL.get(name) or LARGE[name]
    c = make(seqs, seed=len(name), first_row=3, rows_behind=5, gate=len(name) % 2 == 0)
    w = before = None
    if weights:
        before = torch.rand((len(seqs), NKV, c["lmax"] + 3), device="cuda")
        w = before.clone()
    got = call(cuda, c, weights=w)
    torch.cuda.synchronize()
    assert cuda.device_error() == (0, 0)
    check(c, got, reference(c), w, before)


def test_no_rows_in_chunk_form(cuda):
    """Rows of nobody only: nothing is written."""
    import torch
    c = make([(0, 40), (0, 0)], seed=3, first_row=2, rows_behind=6)
    w = torch.ones((2, NKV, 40), device="cuda")
    out, lse = call(cuda, c, weights=w, qmax=64)
    torch.cuda.synchronize()
    assert (out.float() == 7.0).all() and (lse == -7.0).all() and (w == 1).all()
    assert cuda.device_error() == (0, 0)


@pytest.mark.parametrize("rows", [1, 3, 9])
def test_very_long_cache(cuda, rows):
    import torch
    c = make([(rows, 150001)], seed=rows, gate=True)
    before = torch.zeros((1, NKV, c["lmax"]), device="cuda")
    w = before.clone()
    got = call(cuda, c, weights=w)
    check(c, got, reference(c), w, before)


@pytest.mark.parametrize("seqs", [[(2, 900), (1, 40)], [(90, 900), (20, 40)]])
def test_peaked_scores(cuda, seqs):
    """Scores up to some hundreds: one or two keys take each row."""
    import torch
    c = make(seqs, seed=5, spread=12.0)
    before = torch.zeros((len(seqs), NKV, c["lmax"]), device="cuda")
    w = before.clone()
    got = call(cuda, c, weights=w)
    check(c, got, reference(c), w, before)


@pytest.mark.parametrize("seqs", [[(1, 900), (3, 2000), (1, 17)], [(90, 900), (700, 2000), (1, 17)]])
def test_same_bits_every_time(cuda, seqs):
    import torch
    c = make(seqs, seed=6, gate=True)
    runs = []
    for _ in range(3):
        w = torch.ones((len(seqs), NKV, c["lmax"]), device="cuda")
        runs.append((*call(cuda, c, weights=w), w))
    # without weights the attention is the same
    runs.append((*call(cuda, c), runs[0][2]))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_same_bits_over_many_launches(cuda):
    """A ring stage handed back before its last read is in shows as another bit pattern now and then."""
    import torch
    c = make(SMALL["many"], seed=1)
    want, lse = call(cuda, c)
    ws = torch.empty(cuda.chunk_workspace_bytes(len(c["seqs"]), c["rows"], c["qmax"], c["lmax"]), dtype=torch.uint8, device="cuda")
    outs = [want.clone() for _ in range(50)]
    for _ in range(300):
        for o in outs:
            call(cuda, c, out=o, lse=lse, workspace=ws)
        assert all(torch.equal(o, want) for o in outs)


def test_agrees_with_uniform_decode(cuda):
    """A batch of equal row counts is pgc_decode_attn's case: both within the reference's bound."""
    import torch
    for n in (1, 2, 4):
        seqs = [(n, 4097), (n, 900), (n, 17), (n, 3000)]
        c = make(seqs, seed=7 + n, gate=True)
        ref = reference(c)
        check(c, call(cuda, c), ref)
        out = torch.empty((c["rows"], 16, 256), dtype=torch.bfloat16, device="cuda")
        ws = torch.empty(cuda.decode_workspace_bytes(4, n, c["lmax"]), dtype=torch.uint8, device="cuda")
        cuda.decode_attn(c["q"], c["k"], c["v"], c["tables"], c["seq_lens"], c["lmax"], _chunk.SCALE, out, ws,
                         num_queries=n, gate=c["gate"])
        assert ((out.double() - ref[0]).abs() <= ref[1]).all()


@pytest.mark.parametrize("rows", [2, 70])
def test_slots(cuda, rows):
    """Weights in slots of the caller's choice; a slot named twice belongs to the first sequence, one
    out of range to nobody, and both are reported."""
    import torch
    seqs = [(rows, 300), (1, 77), (rows, 500)]
    c = make(seqs, seed=8)
    before = torch.rand((6, NKV, c["lmax"]), device="cuda")
    w = before.clone()
    slots = [4, 0, 5]
    got = call(cuda, c, weights=w, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
    assert cuda.device_error() == (0, 0)
    ref = reference(c)
    check(c, got, ref, w, before, slots)
    for bad in ([4, 4, 5], [4, -1, 5], [4, 6, 5]):
        w2 = before.clone()
        call(cuda, c, weights=w2, slots=torch.tensor(bad, dtype=torch.int32, device="cuda"))
        code, detail = cuda.device_error()
        assert code == (702 if rows <= 4 else 802) and detail == 1
        assert torch.equal(w2[4], w[4]) and torch.equal(w2[5], w[5]) and torch.equal(w2[0], before[0])


@pytest.mark.parametrize("rows", [3, 40])
def test_device_values_outside_host_bounds(cuda, rows):
    """Rows out of order or past the arrays skip the sequence, a length past the bound empties it, a
    page outside the pool reads page 0; all are reported and nothing else changes."""
    import torch
    seqs = [(rows, 300), (rows, 200), (1, 100)]
    c = make(seqs, seed=9, stale=0.0)
    ref = reference(c)
    check(c, call(cuda, c), ref)
    assert cuda.device_error() == (0, 0)
    r = c["starts"]

    def fine(got, *seqs):
        for b in seqs:
            rows = slice(r[b], r[b + 1])
            assert ((got[0].double() - ref[0]).abs()[rows] <= ref[1][rows]).all()
            assert ((got[1].double() - ref[2]).abs()[rows] <= ref[3][rows]).all()

    d = dict(c, seq_lens=torch.tensor([300, 201, 100], dtype=torch.int32, device="cuda"))
    call(cuda, d, lmax=300)
    assert cuda.device_error() == (0, 0)  # 201 <= 300: the bound is the host's
    d["seq_lens"] = torch.tensor([300, 301, 100], dtype=torch.int32, device="cuda")
    out, lse = call(cuda, d, lmax=300)
    code, detail = cuda.device_error()
    assert code == 708 and detail == 1
    fine((out, lse), 0, 2)
    assert (out[r[1]:r[2]] == 0).all() and (lse[r[1]:r[2]] == float("-inf")).all()

    for starts in ([0, rows, rows - 1, rows], [0, rows, 2 * rows + 2, 2 * rows + 3], [0, rows, 4 * rows, 4 * rows]):
        d = dict(c, q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
        got = call(cuda, d)
        assert cuda.device_error()[0] == 707
        # (in the first case the third sequence's row is the first's last one too)
        if starts[2] != rows - 1:
            fine(got, 0)

    d = dict(c, tables=c["tables"].clone())
    d["tables"][1, 0] = c["k"].shape[0]
    got = call(cuda, d)
    assert cuda.device_error() == (701, c["k"].shape[0])
    fine(got, 0, 2)


@pytest.mark.parametrize("seqs", [[(2, 900), (1, 400), (4, 30)], [(80, 900), (1, 400), (200, 230)]])
def test_graph_replay_with_other_lengths(cuda, seqs):
    """A captured call reads rows and lengths from the device: replayed with another batch of the same
    bounds it gives that batch's result."""
    import torch
    a, b = make(seqs, seed=10), make([(n, max(0, L - 13 * i)) for i, (n, L) in enumerate(reversed(seqs))], seed=11)
    lmax, qmax = a["lmax"], a["qmax"]
    live = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in a.items()}
    n = cuda.chunk_workspace_bytes(len(seqs), a["rows"], qmax, lmax, True)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    w = torch.zeros((len(seqs), NKV, lmax), device="cuda")
    out = torch.empty((a["rows"], 16, 256), dtype=torch.bfloat16, device="cuda")
    lse = torch.empty((a["rows"], 16), device="cuda")
    call(cuda, live, weights=w, out=out, lse=lse, lmax=lmax, qmax=qmax, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(cuda, live, weights=w, out=out, lse=lse, lmax=lmax, qmax=qmax, workspace=ws)
    width = live["tables"].shape[1]
    for c in (b, a):
        pages = min(live["k"].shape[0], c["k"].shape[0])
        live["q"].copy_(c["q"])
        live["q_starts"].copy_(c["q_starts"])
        live["seq_lens"].copy_(c["seq_lens"])
        assert c["tables"].shape[1] <= width and c["k"].shape[0] <= live["k"].shape[0]
        live["tables"][:, :c["tables"].shape[1]] = c["tables"]
        live["k"][:pages].copy_(c["k"])
        live["v"][:pages].copy_(c["v"])
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        w2 = torch.zeros_like(w)
        wide = torch.nn.functional.pad(c["tables"], (0, width - c["tables"].shape[1]))
        want = call(cuda, dict(c, tables=wide), weights=w2, lmax=lmax, qmax=qmax)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(w, w2)
    assert cuda.device_error() == (0, 0)


def test_two_streams(cuda):
    """Two calls at once on two streams, each with its own workspace."""
    import torch
    cs = [make([(70, 3000), (1, 500)], seed=12), make([(1, 3000), (2, 500)], seed=13)]
    want = [call(cuda, c) for c in cs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[torch.empty_like(x) for x in w] for w in want]
    ws = [torch.empty(cuda.chunk_workspace_bytes(2, c["rows"], c["qmax"], c["lmax"]), dtype=torch.uint8, device="cuda") for c in cs]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, s, o, x in zip(cs, streams, outs, ws):
            call(cuda, c, out=o[0], lse=o[1], stream=s, workspace=x)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])


def test_long_cache_offsets(cuda):
    """Pages beyond 2^31 elements of the pool."""
    import torch
    c = make([(1, 40), (6, 200)], seed=14)
    pages = (1 << 31) // (NKV * 16 * 256) + 64
    k = torch.zeros((pages, NKV, 16, 256), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    at = pages - c["k"].shape[0]
    k[at:], v[at:] = c["k"], c["v"]
    want = call(cuda, c)
    tables = torch.where(c["tables"] < (1 << 30), c["tables"] + at, c["tables"])
    got = call(cuda, dict(c, k=k, v=v, tables=tables))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert cuda.device_error() == (0, 0)


def in_line_form(c, lmax=40000):
    """The batch with a host bound that no cluster takes: units cut over the whole grid, joined by a second
    kernel. (Short batches within the bounds run as a cluster per sequence and kv head.)"""
    import torch
    width = -(-lmax // 16)
    return dict(c, lmax=lmax, tables=torch.nn.functional.pad(c["tables"], (0, width - c["tables"].shape[1]), value=1 << 30))


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("name", [n for n in SMALL if len(SMALL[n]) < 100])
def test_short_batches_in_line_form(cuda, name, weights):
    import torch
    c = in_line_form(make(SMALL[name], seed=20 + len(name), first_row=1, rows_behind=2, gate=len(name) % 2 == 1))
    w = before = None
    if weights:
        before = torch.rand((len(SMALL[name]), NKV, c["lmax"]), device="cuda")
        w = before.clone()
    got = call(cuda, c, weights=w)
    torch.cuda.synchronize()
    assert cuda.device_error() == (0, 0)
    check(c, got, reference(c), w, before)


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("batch", [1, 2, 3, 4, 7, 8, 9, 18, 19, 36, 37, 38])
def test_batch_sizes(cuda, batch, weights):
    """Every cluster size, its edges in the number of sequences, and lengths from none to the longest that
    it takes and one more; rows from none to 4."""
    import torch
    for longest in (40, 512, 513, 2048, 8192, 8193):
        if batch > 4 and longest > 2048:
            continue
        lens = [longest, 1, 0, 16, longest - 17, 17, 255, 33]
        seqs = [((4, 1, 2, 3, 0)[(i + longest) % 5], min(longest, lens[i % 8])) for i in range(batch)]
        if all(n == 0 for n, _ in seqs):
            seqs[0] = (1, seqs[0][1])
        c = make(seqs, seed=batch, first_row=2, rows_behind=1, gate=batch % 2 == 0)
        w = before = None
        if weights:
            before = torch.rand((batch, NKV, c["lmax"]), device="cuda")
            w = before.clone()
        got = call(cuda, c, weights=w)
        torch.cuda.synchronize()
        assert cuda.device_error() == (0, 0)
        check(c, got, reference(c), w, before)


def test_slots_in_line_form(cuda):
    import torch
    c = in_line_form(make([(2, 300), (1, 77), (2, 500)], seed=8))
    before = torch.rand((6, NKV, c["lmax"]), device="cuda")
    w, slots = before.clone(), [4, 0, 5]
    got = call(cuda, c, weights=w, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"))
    check(c, got, reference(c), w, before, slots)
    for bad in ([4, 4, 5], [4, -1, 5], [4, 6, 5]):
        w2 = before.clone()
        call(cuda, c, weights=w2, slots=torch.tensor(bad, dtype=torch.int32, device="cuda"))
        assert cuda.device_error() == (702, 1)
        assert torch.equal(w2[4], w[4]) and torch.equal(w2[5], w[5]) and torch.equal(w2[0], before[0])


@pytest.mark.parametrize("seqs", [[(1 + i % 4, 100 + 237 * i) for i in range(8)], [(4, 6000)], [(2, 300)] * 37])
def test_clusters_give_the_same_bits_over_many_launches(cuda, seqs):
    import torch
    c = make(seqs, seed=21, gate=True)
    runs = []
    ws = torch.empty(cuda.chunk_workspace_bytes(len(seqs), c["rows"], c["qmax"], c["lmax"], True), dtype=torch.uint8, device="cuda")
    for _ in range(200):
        w = torch.ones((len(seqs), NKV, c["lmax"]), device="cuda")
        runs.append((*call(cuda, c, weights=w, workspace=ws), w))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))
