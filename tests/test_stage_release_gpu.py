"""The kernels that stream pages through a TMA ring hand a stage back only when their last read of it
has arrived. A hand-back that comes too early shows as another bit pattern in a few launches of very
many: about 1 in 60 000 of the ragged decode's line form, at which rate the 240 000 launches here miss
it once in 55 runs of the test. Every launch's output is compared."""
import pytest

import _chunk

pytestmark = pytest.mark.gpu

LAUNCHES, PER_GRAPH = 240_000, 60


def soak(one, shape):
    """`one(out)` launched over and over in a graph; the launches whose output differs from the first's."""
    import torch
    want = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    one(want)
    torch.cuda.synchronize()
    outs = torch.empty((PER_GRAPH, *shape), dtype=torch.bfloat16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for o in outs:
            one(o)
    bad = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(LAUNCHES // PER_GRAPH):
        graph.replay()
        bad += (outs.view(torch.int16) != want.view(torch.int16)).flatten(1).any(1).sum()
    return int(bad)


# many stage rounds a launch: 40 sequences are more units than a wave of clusters (the line form); 8 of up
# to 1759 tokens run as clusters, whose ring is walked most often at 8 CTAs and fewer
@pytest.mark.parametrize("seqs", [[(1 + i % 4, 5 + 37 * i) for i in range(40)], [(1 + i % 4, 100 + 237 * i) for i in range(8)],
                                  [(2, 500)] * 37])
def test_ragged_decode(cuda, seqs):
    import torch
    c = _chunk.make(seqs, seed=1)
    lse = torch.empty((c["rows"], 16), device="cuda")
    ws = torch.empty(cuda.chunk_workspace_bytes(len(seqs), c["rows"], c["qmax"], c["lmax"]), dtype=torch.uint8, device="cuda")
    assert soak(lambda out: _chunk.call(cuda, c, out=out, lse=lse, workspace=ws), (c["rows"], 16, 256)) == 0
    assert cuda.device_error() == (0, 0)


@pytest.mark.parametrize("rows", [1, 2])
def test_uniform_decode(cuda, rows):
    import torch
    seqs = [(rows, 60 + 37 * i) for i in range(40)]
    c = _chunk.make(seqs, seed=2)
    ws = torch.empty(cuda.decode_workspace_bytes(40, rows, c["lmax"]), dtype=torch.uint8, device="cuda")
    assert soak(lambda out: cuda.decode_attn(c["q"], c["k"], c["v"], c["tables"], c["seq_lens"], c["lmax"], _chunk.SCALE, out,
                                             ws, num_queries=rows), (c["rows"], 16, 256)) == 0
    assert cuda.device_error() == (0, 0)
