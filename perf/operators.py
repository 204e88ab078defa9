"""Cases of the ragged-batch attention and cache-eviction operators, with their plain forms.

Four operators over the paged KV cache (16 query heads, 4 kv heads, head dim 256, 16-token
pages), as a batching server runs them:

  attn     causal attention of a ragged batch of chunks (one token to thousands a sequence)
  weights  the same, adding every token's received attention to running per-token weights
  select   per kv head, which cached tokens stay: the first, the last and the heaviest
  compact  the kept K/V rows gathered into fresh pages

A case gives sizes; the ragged lengths are drawn from its own `mix`, so that every seed of a case
does the same work on other values.
"""
import math

import numpy as np
import torch

own = False

NQ, NKV, G, D, PAGE = 16, 4, 4, 256, 16
SCALE = 1.0 / 16.0


def listed():
    return [
        # one request's decode step over a 4096-token cache: the smallest call, where latency counts
        dict(name="attn_decode_1x4097", op="attn", batch=1, qlo=1, qhi=1, llo=4097, lhi=4097, gate=True, mix=1),
        # a decode batch of a loaded server, lengths ragged
        dict(name="attn_decode_64_ragged", op="attn", batch=64, qlo=1, qhi=1, llo=1024, lhi=32768, gate=True, mix=2),
        # a continuous-batching step: chunks and single tokens of 16 requests together
        dict(name="attn_mixed_16", op="attn", batch=16, qlo=1, qhi=512, llo=300, lhi=8700, gate=False, mix=3),
        # one long chunk over a long cached prefix
        dict(name="attn_chunk_1600_over_24576", op="attn", batch=1, qlo=1600, qhi=1600, llo=26176, lhi=26176, gate=False, mix=4),
        # a decode batch whose caches are watched for eviction
        dict(name="weights_decode_16", op="weights", batch=16, qlo=1, qhi=1, llo=1000, lhi=16384, gate=True, mix=5),
        # the verification of a draft token: two queries over one long cache
        dict(name="weights_verify_2x32768", op="weights", batch=1, qlo=2, qhi=2, llo=32768, lhi=32768, gate=True, mix=6),
        # prompts of several requests arriving in chunks
        dict(name="weights_chunks_4", op="weights", batch=4, qlo=200, qhi=1600, llo=2000, lhi=12000, gate=False, mix=7),
        # one request cut back to a quarter
        dict(name="select_1x4097", op="select", batch=1, llo=4097, lhi=4097, budget=1024, first=4, last=256, mix=8),
        # a batch of long requests cut back to a fixed budget
        dict(name="select_64_to_4096", op="select", batch=64, llo=4000, lhi=65536, budget=4096, first=4, last=512, mix=9),
        # one request at the longest supported context
        dict(name="select_1x262144", op="select", batch=1, llo=262144, lhi=262144, budget=8192, first=4, last=1024, mix=10),
        # the rows of one small request
        dict(name="compact_1x4097", op="compact", batch=1, llo=4097, lhi=4097, budget=1024, first=4, last=256, mix=11),
        # the rows of a batch of long requests
        dict(name="compact_32_to_4096", op="compact", batch=32, llo=3000, lhi=16384, budget=4096, first=4, last=512, mix=12),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attn", "attn", "weights", "weights", "select", "compact"])
    mix = rng.randrange(1 << 20)
    if op in ("attn", "weights"):
        if rng.random() < 0.5:  # decode and verification: 1 to 4 tokens a sequence
            batch = log(1, 48)
            q, most = rng.randint(1, 4), min(32768, 600_000 // batch)
            qlo = rng.randint(1, q)
        else:  # chunks
            batch = log(1, 12)
            q, most = log(5, 1600), 24_000 // batch
            qlo = rng.randint(1, q)
        lhi = max(q + 1, log(100, max(200, most)))
        return dict(op=op, batch=batch, qlo=qlo, qhi=q, llo=max(q, lhi // rng.randint(1, 16)), lhi=lhi,
                    gate=rng.random() < 0.5, mix=mix)
    batch = log(1, 48) if op == "select" else log(1, 24)
    lhi = log(50, 65536) if op == "select" else log(50, 16384)
    budget = max(2, log(16, 4096))
    first = rng.randint(0, min(8, budget // 2))
    return dict(op=op, batch=batch, llo=max(1, lhi // rng.randint(1, 16)), lhi=lhi, budget=budget, first=first,
                last=rng.randint(0, budget - first), mix=mix)


def _lens(case):
    """The ragged lengths of a case: query tokens and cached tokens (queries included) a sequence."""
    r = np.random.RandomState(case["mix"])
    b = case["batch"]

    def spread(lo, hi):
        v = np.exp(r.uniform(math.log(lo), math.log(hi + 1), b)).astype(np.int64).clip(lo, hi)
        v[r.randint(b)] = hi  # the upper bounds are met
        return v

    L = spread(case["llo"], case["lhi"])
    n = spread(case["qlo"], case["qhi"]) if "qlo" in case else np.zeros(b, np.int64)
    return np.minimum(n, L), L


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)

    n, L = _lens(case)
    b, lmax = case["batch"], int(L.max())
    dev = dict(device="cuda")
    st = dict(case=case, n_host=n, L_host=L, lmax=lmax, seq_lens=torch.tensor(L, dtype=torch.int32, **dev))
    if case["op"] != "select":
        # pools whose pages the sequences hold in random order
        pages = -(-L // PAGE)
        total = int(pages.sum())
        perm = torch.randperm(total + 8, generator=gen, **dev).to(torch.int32)
        tables = torch.zeros((b, -(-lmax // PAGE)), dtype=torch.int32, **dev)
        at = 0
        for i, p in enumerate(pages.tolist()):
            tables[i, :p] = perm[at:at + p]
            at += p
        st.update(tables=tables, k=normal(total + 8, NKV, PAGE, D), v=normal(total + 8, NKV, PAGE, D))
    if case["op"] in ("attn", "weights"):
        # a share of the keys is what the queries look for: attention is far from uniform
        u = normal(NKV, 1, D)
        hot = torch.rand(st["k"].shape[:3] + (1,), generator=gen, **dev) < 0.02
        st["k"] = torch.where(hot, st["k"] + u, st["k"])
        rows = int(n.sum())
        st["q"] = (normal(rows, NKV, G, D) + 0.4 * u).reshape(rows, NQ, D).contiguous()
        st["gate"] = normal(rows, NQ, D) if case["gate"] else None
        st["q_starts"] = torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, **dev)
        st["qmax"] = int(n.max())
        st["out"] = torch.zeros((rows + 1, NQ, D), dtype=torch.bfloat16, **dev)  # a row over for the plain form
        st["lse"] = torch.zeros((rows + 1, NQ), dtype=torch.float32, **dev)
        if case["op"] == "weights":
            # what earlier steps have added
            st["weights"] = torch.rand((b, NKV, lmax), generator=gen, **dev)
    else:
        # received attention: a long tail, many equal values (tokens that nothing looked at)
        w = torch.exp(1.5 * torch.randn((b, NKV, lmax), generator=gen, **dev))
        w = w * (torch.rand(w.shape, generator=gen, **dev) > 0.1)
        B = case["budget"]
        if case["op"] == "select":
            st.update(weights=w, weights_out=torch.zeros_like(w), kept=torch.zeros((b, NKV, B), dtype=torch.int32, **dev),
                      new_lens=torch.zeros(b, dtype=torch.int32, **dev))
        else:
            # the tokens of a selection: ascending, -1 behind the last
            t = torch.arange(lmax, **dev)
            Lb = st["seq_lens"][:, None, None]
            w = torch.where((t < case["first"]) | (t >= Lb - case["last"]), math.inf, w)
            w = torch.where(t < Lb, w, -math.inf)
            top = torch.topk(w, min(B, lmax), dim=-1)
            kept = torch.where(top.values > -math.inf, top.indices, lmax).sort(dim=-1).values
            kept = torch.where(kept < lmax, kept, -1).to(torch.int32)
            st["kept"] = torch.nn.functional.pad(kept, (0, B - kept.shape[-1]), value=-1).contiguous()
            per = -(-B // PAGE)
            st["dst_tables"] = torch.randperm(b * per, generator=gen, **dev).to(torch.int32).reshape(b, per)
            st["dst_k"] = torch.zeros((b * per, NKV, PAGE, D), dtype=torch.bfloat16, **dev)
            st["dst_v"] = torch.zeros_like(st["dst_k"])
    return st


def _plain_attention(st, with_weights):
    q_starts, L, tables = st["q_starts"].long(), st["seq_lens"].long(), st["tables"].long()
    rows, T, lmax = st["q"].shape[0], st["qmax"], st["lmax"]
    n = q_starts[1:] - q_starts[:-1]
    i = torch.arange(T, device="cuda")
    t = torch.arange(lmax, device="cuda")
    live = i < n[:, None]
    row = torch.where(live, q_starts[:-1, None] + i, rows)  # rows: nobody's
    q = st["q"][row.clamp(max=rows - 1)].float().reshape(-1, T, NKV, G, D).permute(0, 2, 3, 1, 4)
    page = tables[:, t // PAGE]
    held = (t < L[:, None])[..., None, None]
    k = torch.where(held, st["k"][page, :, t % PAGE].float(), 0.0).permute(0, 2, 3, 1)
    s = torch.matmul(q.reshape(-1, NKV, G * T, D), k).mul_(SCALE).reshape(-1, NKV, G, T, lmax)
    del k
    seen = t <= (L - n)[:, None, None] + i[:, None]
    seen = (seen & live[..., None] & held[:, None, :, 0, 0])[:, None, None]
    s.masked_fill_(~seen, -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(s.sub_(m))
    l = p.sum(-1, keepdim=True)
    p = p / l.clamp(min=1e-38)
    lse = (m + torch.log(l)).squeeze(-1)
    v = torch.where(held, st["v"][page, :, t % PAGE].float(), 0.0).permute(0, 2, 1, 3)
    o = torch.matmul(p.reshape(-1, NKV, G * T, lmax), v).reshape(-1, NKV, G, T, D)
    o = o.permute(0, 3, 1, 2, 4).reshape(-1, T, NQ, D)
    if st["gate"] is not None:
        o = o * torch.sigmoid(st["gate"][row.clamp(max=rows - 1)].float())
    st["out"][row] = o.to(torch.bfloat16)
    st["lse"][row] = lse.permute(0, 3, 1, 2).reshape(-1, T, NQ)
    if with_weights:
        st["weights"] += p.sum((2, 3))
        return st["out"][:rows], st["lse"][:rows], st["weights"]
    return st["out"][:rows], st["lse"][:rows]


def _plain_select(st):
    case, w, L = st["case"], st["weights"], st["seq_lens"].long()[:, None, None]
    B, lmax = case["budget"], st["lmax"]
    t = torch.arange(lmax, device="cuda")
    rank = torch.where((t < case["first"]) | (t >= L - case["last"]), math.inf, w)
    rank = torch.where(t < L, rank, -math.inf)
    # heaviest first, of equal ones the lowest index
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :B]
    order = torch.where(order < L, order, lmax).sort(dim=-1).values
    live = order < lmax
    gathered = torch.where(live, torch.gather(w, 2, order.clamp(max=lmax - 1)), 0.0)
    m = order.shape[-1]
    st["kept"].fill_(-1)
    st["kept"][..., :m] = torch.where(live, order, -1)
    st["weights_out"][..., :m] = torch.where(t[:m] < L, gathered, st["weights_out"][..., :m])
    st["weights_out"][..., m:] = torch.where(t[m:] < L, 0.0, st["weights_out"][..., m:])
    st["new_lens"].copy_(L.clamp(max=B)[:, 0, 0])
    return st["kept"], st["new_lens"], st["weights_out"]


def _plain_compact(st):
    kept, tables, dst = st["kept"].long(), st["tables"].long(), st["dst_tables"].long()
    B = kept.shape[-1]
    i = torch.arange(B, device="cuda")
    h = torch.arange(NKV, device="cuda")[None, :, None]
    at = kept.clamp(min=0)
    page = torch.gather(tables[:, None].expand(-1, NKV, -1), 2, at // PAGE)
    to = dst[:, i // PAGE][:, None].expand(-1, NKV, -1)
    live = (kept >= 0)[..., None]
    slot = (i % PAGE).expand_as(to)
    hh = h.expand_as(to)
    st["dst_k"][to, hh, slot] = torch.where(live, st["k"][page, hh, at % PAGE], st["dst_k"][to, hh, slot])
    st["dst_v"][to, hh, slot] = torch.where(live, st["v"][page, hh, at % PAGE], st["dst_v"][to, hh, slot])
    return st["dst_k"], st["dst_v"]


def _own(st):
    from peregrine_b200 import capi

    case = st["case"]
    if case["op"] == "select":
        capi.kv_evict_select(st["weights"], st["seq_lens"], st["lmax"], case["budget"], case["first"], case["last"],
                             st["kept"], st["new_lens"], weights_out=st["weights_out"])
        return st["kept"], st["new_lens"], st["weights_out"]
    if case["op"] == "compact":
        capi.kv_evict_compact(st["k"], st["v"], st["tables"], st["kept"], st["dst_k"], st["dst_v"], st["dst_tables"])
        return st["dst_k"], st["dst_v"]
    rows = st["q"].shape[0]
    if "workspace" not in st:
        nbytes = capi.chunk_workspace_bytes(case["batch"], rows, st["qmax"], st["lmax"], case["op"] == "weights")
        st["workspace"] = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    a = (st["q"], st["k"], st["v"], st["tables"], st["q_starts"], st["seq_lens"], st["qmax"], st["lmax"], SCALE, st["out"])
    if case["op"] == "attn":
        capi.chunk_attn(*a, st["workspace"], gate=st["gate"], lse=st["lse"])
        return st["out"][:rows], st["lse"][:rows]
    capi.chunk_attn_weights(*a, st["weights"], st["workspace"], gate=st["gate"], lse=st["lse"])
    return st["out"][:rows], st["lse"][:rows], st["weights"]


def run(st):
    if own:
        return _own(st)
    if st["case"]["op"] == "select":
        return _plain_select(st)
    if st["case"]["op"] == "compact":
        return _plain_compact(st)
    return _plain_attention(st, st["case"]["op"] == "weights")


def work(case):
    n, L = _lens(case)
    row = D * 2  # a bf16 row
    if case["op"] in ("attn", "weights"):
        rows = int(n.sum())
        nbytes = int(L.sum()) * NKV * 2 * row + rows * NQ * (2 * row + 4 + (row if case["gate"] else 0))
        if case["op"] == "weights":
            nbytes += int(L.sum()) * NKV * 8
        pairs = int((n * (L - n) + n * (n + 1) // 2).sum())
        return dict(bytes=nbytes, flops=pairs * NQ * D * 4)
    kept = int(np.minimum(L, case["budget"]).sum()) * NKV
    if case["op"] == "select":
        return dict(bytes=int(L.sum()) * NKV * 8 + kept * 4, flops=int(L.sum()) * NKV)
    return dict(bytes=kept * (4 * row + 4), flops=kept)


def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence and head by head."""
    st = prepare(case, seed)
    if case["op"] in ("select", "compact"):
        return _exact_evict(case, st)
    rows = st["q"].shape[0]
    out = torch.zeros((rows, NQ, D), dtype=torch.float64, device="cuda")
    lse = torch.zeros((rows, NQ), dtype=torch.float64, device="cuda")
    weights = st["weights"].double() if case["op"] == "weights" else None
    row0 = 0
    for b, (n, L) in enumerate(zip(st["n_host"].tolist(), st["L_host"].tolist())):
        ids = st["tables"][b, :-(-L // PAGE)].long()
        for h in range(NKV):
            k = st["k"][ids, h].reshape(-1, D)[:L].double()
            v = st["v"][ids, h].reshape(-1, D)[:L].double()
            for a in range(0, n, 256):
                z = min(n, a + 256)
                end = torch.arange(L - n + a, L - n + z, device="cuda")[:, None]
                hidden = torch.arange(L, device="cuda")[None] > end
                for g in range(h * G, h * G + G):
                    score = st["q"][row0 + a:row0 + z, g].double() @ k.T / 16
                    score = score.masked_fill(hidden, -math.inf)
                    total = torch.logsumexp(score, -1, keepdim=True)
                    prob = (score - total).exp()
                    out[row0 + a:row0 + z, g] = prob @ v
                    lse[row0 + a:row0 + z, g] = total[:, 0]
                    if weights is not None:
                        weights[b, h, :L] += prob.sum(0)
        row0 += n
    if st["gate"] is not None:
        out = out / (1 + torch.exp(-st["gate"].double()))
    return (out, lse) if weights is None else (out, lse, weights)


def _exact_evict(case, st):
    if case["op"] == "compact":
        kept, src, dst = (st[x].cpu().numpy() for x in ("kept", "tables", "dst_tables"))
        outs = []
        for pool, to in ((st["k"], st["dst_k"]), (st["v"], st["dst_v"])):
            flat = torch.zeros(to.shape, dtype=torch.float64, device="cuda")
            for b in range(case["batch"]):
                for h in range(NKV):
                    t = kept[b, h][kept[b, h] >= 0]
                    i = np.arange(len(t))
                    rows = pool[torch.from_numpy(src[b, t // PAGE]).long().cuda(), h, torch.from_numpy(t % PAGE).long().cuda()]
                    flat[torch.from_numpy(dst[b, i // PAGE]).long().cuda(), h, torch.from_numpy(i % PAGE).long().cuda()] = rows.double()
            outs.append(flat)
        return tuple(outs)
    w = st["weights"].double().cpu().numpy()
    kept = np.full(st["kept"].shape, -1, np.int32)
    moved = np.zeros(w.shape)
    for b, L in enumerate(st["L_host"].tolist()):
        B = min(case["budget"], L)
        always = np.zeros(L, bool)
        always[:case["first"]] = True
        always[max(0, L - case["last"]):] = True
        for h in range(NKV):
            rest = np.flatnonzero(~always)
            take = rest[np.argsort(-w[b, h, rest], kind="stable")[:max(0, B - int(always.sum()))]]
            stay = np.sort(np.concatenate([np.flatnonzero(always), take]))[:B]
            kept[b, h, :len(stay)] = stay
            moved[b, h, :len(stay)] = w[b, h, stay]
    return torch.from_numpy(kept), None, torch.from_numpy(moved)
