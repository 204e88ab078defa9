"""Ragged-batch inputs, the float64 reference of pgc_chunk_attn / pgc_chunk_attn_weights and the
error bounds that the tests of both use."""
import math

import torch

NQ, NKV, G, D, PAGE = 16, 4, 4, 256, 16
SCALE = 1.0 / 16
NAN = float("nan")


def make(seqs, seed, first_row=0, rows_behind=0, gate=False, spread=1.0, stale=NAN, spare_pages=3):
    """A batch of (rows, cached tokens) sequences. Slots past each sequence's end and the spare pages
    hold `stale`; `first_row` rows before the first sequence's and `rows_behind` behind the last."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)

    lens = [L for _, L in seqs]
    pages = [-(-L // PAGE) for L in lens]
    total = sum(pages) + spare_pages
    perm = torch.randperm(total, generator=g, device="cuda")
    width = max(1, max(pages))
    # entries behind a sequence's pages are never looked up: an id outside the pool
    tables = torch.full((len(seqs), width), 1 << 30, dtype=torch.int32, device="cuda")
    k = torch.full((total, NKV, PAGE, D), stale, dtype=torch.bfloat16, device="cuda")
    v = k.clone()
    at = 0
    for b, L in enumerate(lens):
        ids = perm[at:at + pages[b]]
        at += pages[b]
        tables[b, :pages[b]] = ids.to(torch.int32)
        t = torch.arange(L, device="cuda")
        k[ids[t // PAGE], :, t % PAGE] = (spread * torch.randn((L, NKV, D), generator=g, device="cuda")).to(torch.bfloat16)
        v[ids[t // PAGE], :, t % PAGE] = normal(L, NKV, D)
    ns = [n for n, _ in seqs]
    starts = [first_row]
    for n in ns:
        starts.append(starts[-1] + n)
    rows = starts[-1] + rows_behind
    return dict(seqs=seqs, starts=starts, rows=rows, k=k, v=v, tables=tables, q=normal(rows, NQ, D),
                gate=normal(rows, NQ, D) if gate else None,
                q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                qmax=max(ns), lmax=max(1, max(lens)))


def call(capi, c, weights=None, slots=None, out=None, lse=None, qmax=None, lmax=None, stream=None, workspace=None):
    """One call; returns (out, lse), whose untouched rows keep the marks 7 and -7."""
    qmax, lmax = qmax or max(1, c["qmax"]), lmax or c["lmax"]
    out = torch.full((c["rows"], NQ, D), 7.0, dtype=torch.bfloat16, device="cuda") if out is None else out
    lse = torch.full((c["rows"], NQ), -7.0, device="cuda") if lse is None else lse
    if workspace is None:
        n = capi.chunk_workspace_bytes(len(c["seqs"]), c["rows"], qmax, lmax, weights is not None)
        workspace = torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN patterns
    a = (c["q"], c["k"], c["v"], c["tables"], c["q_starts"], c["seq_lens"], qmax, lmax, SCALE, out)
    if weights is None:
        capi.chunk_attn(*a, workspace, gate=c["gate"], lse=lse, stream=stream)
    else:
        capi.chunk_attn_weights(*a, weights, workspace, gate=c["gate"], lse=lse, slots=slots, stream=stream)
    return out, lse


def rows_of(c, b, h):
    """K and V of one kv head of one sequence, float64 [L][256]."""
    L = c["seqs"][b][1]
    ids = c["tables"][b, :-(-L // PAGE)].long()
    return (x[ids, h].reshape(-1, D)[:L].double() for x in (c["k"], c["v"]))


def reference(c):
    """float64 (out, out bound, lse, lse bound, per-sequence received attention [4][L], its bound).

    Bounds, u = 2^-8 the half step of bf16 (probabilities and the output are rounded to it) and
    e = 2^-23 the whole step of fp32 (the tensor cores need not round a sum to nearest):
      a score of 256 products is off by at most ds = 256 e scale sum|q_d k_d| (every partial sum is
      at most that sum), so a probability by the factor exp(2 ds) and, with exp2 (2 ulp), the max
      subtraction (1 + |s| ulp) and the sums of at most L terms in fp32, dp = 2 ds + (L / 32 + 40) e
      (a thread sums at most L / 32 terms one after the other, the rest pairwise);
      lse: ds + (L / 32 + 40) e + e |lse|;
      out: the rounded P gives u sum p|v|, the statistics dp sum p|v|, the output rounding u |o| and
      the gate's sigmoid (4 + 2 |gate|) ulp: an approximate exponential (2), reciprocal (1) and a product,
      the exponent's rounding |gate| log2(e) half ulps;
      weights: dp + (rows of the sum) e, relative."""
    u, e = 2.0 ** -8, 2.0 ** -23
    dev = dict(dtype=torch.float64, device="cuda")
    out, tol = torch.zeros((c["rows"], NQ, D), **dev), torch.zeros((c["rows"], NQ, D), **dev)
    lse, ltol = torch.zeros((c["rows"], NQ), **dev), torch.zeros((c["rows"], NQ), **dev)
    weights = []
    for b, (n, L) in enumerate(c["seqs"]):
        w, wt = torch.zeros((NKV, L), **dev), torch.zeros((NKV, L), **dev)
        r0 = c["starts"][b]
        for h in range(NKV):
            if n == 0:
                continue
            k, v = rows_of(c, b, h)
            for a in range(0, n, 256):
                z = min(n, a + 256)
                pos = torch.arange(L - n + a, L - n + z, device="cuda")[:, None]
                hidden = torch.arange(L, device="cuda")[None] > pos
                for g in range(h * G, h * G + G):
                    q = c["q"][r0 + a:r0 + z, g].double()
                    s = (q @ k.T * SCALE).masked_fill(hidden, -math.inf)
                    ds = 256 * e * SCALE * (q.abs() @ k.abs().T).masked_fill(hidden, 0).amax(-1, keepdim=True) if L else torch.zeros((z - a, 1), **dev)
                    t = torch.logsumexp(s, -1, keepdim=True) if L else torch.full((z - a, 1), -math.inf, **dev)
                    p = (s - t).exp().masked_fill(hidden, 0)  # nothing visible: 0
                    dp = 2 * ds + (L / 32 + 40) * e
                    o, av = p @ v, p @ v.abs()
                    sig, gulp = 1.0, 4.0
                    if c["gate"] is not None:
                        sig = torch.sigmoid(c["gate"][r0 + a:r0 + z, g].double())
                        gulp = 4 + 2 * c["gate"][r0 + a:r0 + z, g].double().abs()
                    out[r0 + a:r0 + z, g] = o * sig
                    tol[r0 + a:r0 + z, g] = (u + dp) * av * sig + (u + gulp * e) * (o * sig).abs() + 1e-30
                    lse[r0 + a:r0 + z, g] = t[:, 0]
                    ltol[r0 + a:r0 + z, g] = (ds + (L / 32 + 40) * e + e * torch.where(t.isinf(), 0, t.abs()))[:, 0]
                    w[h] += p.sum(0)
                    wt[h] += (p * (dp + 4 * n * e)).sum(0)
        weights.append((w, wt))
    return out, tol, lse, ltol, weights


def check(c, got, ref, weights=None, before=None, slots=None):
    out, lse = got
    rout, tol, rlse, ltol, rw = ref
    own = torch.zeros(c["rows"], dtype=torch.bool, device="cuda")
    own[c["starts"][0]:c["starts"][-1]] = True
    assert (out[~own].float() == 7.0).all() and (lse[~own] == -7.0).all(), "a row of nobody was written"
    err = (out.double() - rout).abs()[own]
    assert torch.isfinite(out[own].float()).all()
    assert (err <= tol[own]).all(), (err - tol[own]).max().item()
    seen = own[:, None] & ~rlse.isinf()
    assert (lse[own[:, None] & rlse.isinf()] == -math.inf).all()
    lerr = (lse.double() - rlse).abs()
    assert (lerr[seen] <= ltol[seen]).all(), (lerr - ltol)[seen].max().item()
    if weights is None:
        return
    want = before.double().clone()
    bound = torch.zeros_like(want)
    for b, (w, wt) in enumerate(rw):
        s = b if slots is None else slots[b]
        L = w.shape[1]
        want[s, :, :L] += w
        bound[s, :, :L] = wt + 2.0 ** -23 * want[s, :, :L].abs()
    werr = (weights.double() - want).abs()
    assert (werr <= bound).all(), (werr - bound).max().item()
