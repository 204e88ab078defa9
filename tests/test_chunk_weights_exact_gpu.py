"""Received attention where each row's attention is one token: the last 256 tokens' keys are 512 times a
unit vector of their own and row i's query is a_i times that of its own token, so that its score is
s = 32 a_i >= 4096 and all others are 0, and exp(-4096) is 0 in fp32. All products and sums are exact.
The row's 4 heads then add 4 to its token's weight and nothing to any other.

Up to 4 rows a sequence the score x = fl(s c), c = scale log2(e), is also the row's maximum m; the sum of the
exponentials is 1, so the log-sum-exp in log2 units is m + 0 and each term exp2(x - m) = 1: exactly 4.
More rows: the attention's exponent is s c - m in one rounding, at most half an ulp of m away from 0, and so
is the second pass's s c - lse2 beside lse2 = fl(m + log2(sum)), which holds s c to half an ulp: with
|m| < 2^14, h = 2^-11, a term is 1 within ln2 h, the approximate exponentials of both passes (2 ulp
each) and the logarithm (2 ulp of a value within h of 0), 4 ulp in all. In natural units the
log-sum-exp would be rounded at its own size, and twice more on its way back."""
import math

import pytest

import _chunk
from _chunk import NKV, call, make
from test_chunk_attn_gpu import in_line_form

pytestmark = pytest.mark.gpu


def one_token_each(seqs, seed):
    import torch
    c = make(seqs, seed=seed, stale=0.0)
    c["k"].zero_()
    c["q"].zero_()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for b, (n, L) in enumerate(seqs):
        ids = c["tables"][b].long()
        t = torch.arange(max(0, L - 256), L, device="cuda")
        c["k"][ids[t // 16], :, t % 16, t % 256] = 512.0
        i = torch.arange(n, device="cuda")
        a = torch.randint(128, 256, (n,), generator=gen, device="cuda").to(torch.bfloat16)
        c["q"][c["starts"][b] + i, :, (L - n + i) % 256] = a[:, None].expand(n, 16)
    return c


def received(cuda, c):
    import torch
    w = torch.zeros((len(c["seqs"]), NKV, c["lmax"]), device="cuda")
    call(cuda, c, weights=w)
    torch.cuda.synchronize()
    assert cuda.device_error() == (0, 0)
    want = torch.zeros_like(w, dtype=torch.float64)
    for b, (n, L) in enumerate(c["seqs"]):
        want[b, :, L - n:L] = 4.0
    return w.double(), want


@pytest.mark.parametrize("line", [False, True])
@pytest.mark.parametrize("seqs", [[(1, 1)], [(4, 40), (1, 300), (2, 2000)], [(1 + i % 4, 4 + 211 * i) for i in range(40)]])
def test_short_rows(cuda, seqs, line):
    c = one_token_each(seqs, len(seqs))
    got, want = received(cuda, in_line_form(c, 12000) if line else c)
    assert (got == want).all()


@pytest.mark.parametrize("seqs", [[(200, 200)], [(64, 64), (5, 300), (250, 5000)], [(5 + 6 * i, 100 + 531 * i) for i in range(30)]])
def test_chunks(cuda, seqs):
    c = one_token_each(seqs, len(seqs))
    got, want = received(cuda, c)
    bound = 4 * (math.log(2) * 2.0 ** -11 + 4 * 2.0 ** -23)
    assert ((got - want).abs() <= bound * (want > 0)).all(), (got - want).abs().max().item()
