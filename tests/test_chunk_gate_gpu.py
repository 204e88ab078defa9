"""Gates far from zero in every place where a row is finished. The kernels' v * sigmoid(gate) is off by
(4 + 2 |gate|) fp32 ulp down to gates of -87.3, and 0 below, where the sigmoid is less than 2^-126: 2^-126 |v|
in absolute terms. bf16 rounds the result, subnormal ones by half of 2^-133."""
import math

import pytest

from _chunk import NQ, call, make, reference
from test_chunk_attn_gpu import in_line_form

pytestmark = pytest.mark.gpu
GATES = [-math.inf, -1e4, -200.0, -100.0, -89.0, -88.5, -88.0, -87.5, -87.0, -86.0, -80.0, -20.0, 0.0, 20.0, 80.0, 88.0, 90.0, 200.0, 1e4,
         math.inf]


# a cluster a unit; units cut over the grid and whole ones, short rows and chunks
@pytest.mark.parametrize("seqs,line", [([(1, 300), (4, 900)], False), ([(1, 5000), (4, 900)], True),
                                       ([(1 + i % 4, 20 + 40 * i) for i in range(60)], False),
                                       ([(70, 300), (5, 9000), (1, 40)], False), ([(64, 64 + i) for i in range(80)], False)])
def test_gates(cuda, seqs, line):
    import torch
    c = make(seqs, seed=40)
    rout, tol = reference(c)[:2]
    gen = torch.Generator(device="cuda").manual_seed(41)
    gates = torch.tensor(GATES, device="cuda").to(torch.bfloat16)
    c["gate"] = gates[torch.randint(len(GATES), (c["rows"], NQ, 256), generator=gen, device="cuda")]
    out, _ = call(cuda, in_line_form(c) if line else c)
    g = c["gate"].double()
    sig = torch.sigmoid(g)
    bound = tol * sig + (4 + 2 * g.abs().clamp(max=200)) * 2.0 ** -23 * rout.abs() * sig + 2.0 ** -126 * rout.abs() + 2.0 ** -134
    assert ((out.double() - rout * sig).abs() <= bound).all()
    assert (out[g < -88.8] == 0).all()
    assert cuda.device_error() == (0, 0)
