"""pgc_kv_evict_select and pgc_kv_evict_compact against plain restatements (exact), and the whole run:
chunks and decode steps that gather weights, eviction, and decoding over the compacted cache."""
import math

import numpy as np
import pytest

import _chunk
from _chunk import D, NKV, NQ, PAGE

pytestmark = pytest.mark.gpu


def ref_select(w, L, budget, first, last):
    """Kept indices of one row of weights (numpy float32), by sorting."""
    if L <= budget:
        return np.arange(L)
    mid = np.arange(first, L - last)
    key = np.where(np.isnan(w[mid]), -np.inf, w[mid].astype(np.float64))
    # NaN below -inf: sort by (is NaN, -weight, index)
    order = np.lexsort((mid, -key, np.isnan(w[mid])))
    take = mid[order[:budget - first - last]]
    return np.sort(np.concatenate([np.arange(first), take, np.arange(L - last, L)])).astype(np.int64)


def run_select(cuda, w, lens, budget, first, last, slots=None, in_place=False, lmax=None, moved=True):
    import torch
    wd = torch.from_numpy(w).cuda()
    out = wd if in_place else torch.full_like(wd, -5.0) if moved else None
    b = len(lens)
    kept = torch.full((b, NKV, budget), -9, dtype=torch.int32, device="cuda")
    new = torch.full((b,), -9, dtype=torch.int32, device="cuda")
    cuda.kv_evict_select(wd, torch.tensor(lens, dtype=torch.int32, device="cuda"), lmax or max(1, max(lens)), budget, first,
                         last, kept, new, weights_out=out,
                         slots=None if slots is None else torch.tensor(slots, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    return kept.cpu().numpy(), new.cpu().numpy(), None if out is None else out.cpu().numpy()


def check_select(w, lens, budget, first, last, got, slots=None, in_place=False):
    kept, new, out = got
    want = w.copy() if in_place else np.full_like(w, -5.0)
    for b, L in enumerate(lens):
        s = b if slots is None else slots[b]
        assert new[b] == min(L, budget)
        for h in range(NKV):
            ids = ref_select(w[s, h], L, budget, first, last)
            assert np.array_equal(kept[b, h, :len(ids)], ids), (b, h)
            assert (kept[b, h, len(ids):] == -1).all()
            want[s, h, :L] = 0
            want[s, h, :len(ids)] = w[s, h, ids]
    if out is not None:
        assert np.array_equal(out, want, equal_nan=True)


def weights(rng, b, n, kind):
    if kind == "tail":
        w = np.exp(1.5 * rng.standard_normal((b, NKV, n)))
    elif kind == "ties":
        w = rng.integers(0, 4, (b, NKV, n)) * 0.25
    elif kind == "zero":
        w = np.zeros((b, NKV, n))
    elif kind == "close":  # values that differ in the last bits only
        w = 1.0 + rng.integers(0, 300, (b, NKV, n)) * 2.0 ** -23
    else:  # odd values: signed zeros, negative, infinite, NaN, subnormal
        w = rng.choice(np.array([0.0, -0.0, 1.0, -1.0, math.inf, -math.inf, math.nan, 1e-42, -1e-42, 3e38]), (b, NKV, n))
    return w.astype(np.float32)


@pytest.mark.parametrize("kind", ["tail", "ties", "zero", "close", "odd"])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,budget,first,last", [
    ([1], 1, 0, 0), ([0, 1, 2, 3], 1, 0, 1), ([5, 4, 6, 0], 4, 1, 2), ([700, 31, 32, 33, 512, 513], 32, 4, 28),
    ([4097], 1024, 4, 256), ([9000, 20000, 100], 300, 0, 0), ([8192, 8193, 16384, 16385], 4096, 7, 1000),
    ([65536, 1000], 65535, 1, 1), ([40000], 40000, 0, 5), ([33000], 1, 1, 0)])
def test_select(cuda, kind, in_place, lens, budget, first, last):
    rng = np.random.default_rng(len(lens) * 1000 + budget)
    w = weights(rng, len(lens), max(lens) + 5, kind)
    got = run_select(cuda, w, lens, budget, first, last, in_place=in_place)
    check_select(w, lens, budget, first, last, got, in_place=in_place)
    assert cuda.device_error() == (0, 0)


def test_select_longest(cuda):
    rng = np.random.default_rng(1)
    w = weights(rng, 2, cuda.EVICT_MAX_TOKENS, "tail")
    lens = [cuda.EVICT_MAX_TOKENS, 200001]
    check_select(w, lens, 8192, 4, 1024, run_select(cuda, w, lens, 8192, 4, 1024))
    check_select(w, lens, 8192, 4, 1024, run_select(cuda, w, lens, 8192, 4, 1024, moved=False))


@pytest.mark.parametrize("kind", ["tail", "close", "odd"])
@pytest.mark.parametrize("longest", [40000, 140000])
def test_select_large_batch(cuda, kind, longest):
    """More rows than the device holds at once: each row uses as many CTAs of its cluster as hold it."""
    rng = np.random.default_rng(longest)
    lens = [longest, 513] + [int(x) for x in np.exp(rng.uniform(np.log(100), np.log(longest), 40))]
    w = weights(rng, len(lens), longest, kind)
    for in_place in (False, True):
        got = run_select(cuda, w, lens, 512, 4, 100, in_place=in_place)
        check_select(w, lens, 512, 4, 100, got, in_place=in_place)
    assert cuda.device_error() == (0, 0)


@pytest.mark.parametrize("n", [255, 256, 257, 1000])
def test_select_crowded_value(cuda, n):
    """n distinct neighbouring values around the last one kept, beside others: the list of those that are
    left, at its size and past it, with need at either end."""
    rng = np.random.default_rng(n)
    L = 5000
    w = (2.0 + rng.random((4, NKV, L))).astype(np.float32)
    w[:, :, 1000:4000] = 2.0 ** rng.uniform(-30, 0, (4, NKV, 3000))
    crowd = np.float32(1.0) + np.arange(n, dtype=np.float32) * np.float32(2.0 ** -23)
    for s in range(4):
        for h in range(NKV):
            w[s, h, rng.choice(np.arange(1000, 4000), n, replace=False)] = rng.permutation(crowd)
    above = int((w[0, 0] >= 2).sum())
    for extra in (1, n // 2, n - 1, n, n + 1):
        lens = [L] * 4
        check_select(w, lens, above + extra, 0, 0, run_select(cuda, w, lens, above + extra, 0, 0))
    assert cuda.device_error() == (0, 0)


def test_select_slots_and_lengths(cuda):
    """Slots of the caller's choice; a slot named twice or out of range, or a length past the bound,
    keeps nothing and is reported."""
    rng = np.random.default_rng(2)
    w = weights(rng, 6, 3000, "tail")
    lens, slots = [3000, 1200, 40], [5, 0, 3]
    got = run_select(cuda, w, lens, 100, 2, 10, slots=slots)
    check_select(w, lens, 100, 2, 10, got, slots=slots)
    for bad in ([5, 5, 3], [5, 6, 3], [5, -1, 3]):
        kept, new, out = run_select(cuda, w, lens, 100, 2, 10, slots=bad)
        code, detail = cuda.device_error()
        assert code == 902 and detail == 1
        assert new.tolist() == [100, 0, 40] and (kept[1] == -1).all()
        assert np.array_equal(out[5], got[2][5]) and np.array_equal(out[3], got[2][3]) and (out[0] == -5).all()
    for bad in (1300, -1):
        kept, new, out = run_select(cuda, w, [1200, bad, 40], 100, 2, 10, slots=slots, lmax=1200)
        code, detail = cuda.device_error()
        assert code == 908 and detail == 1
        assert new.tolist() == [100, 0, 40] and (kept[1] == -1).all() and (out[0] == -5).all()


def test_compact(cuda):
    """Every bit pattern is copied; skipped entries leave their rows, bad ones are reported."""
    import torch
    rng = np.random.default_rng(3)
    for budget, lens in ((1, [1]), (16, [16, 300]), (100, [7, 1000, 100]), (33, [4000]), (1000, [5000, 2, 900])):
        b = len(lens)
        pages = [-(-n // PAGE) for n in lens]
        total = sum(pages) + 2
        perm = rng.permutation(total).astype(np.int32)
        tables = np.full((b, max(pages)), 1 << 30, np.int32)
        at = 0
        for i, n in enumerate(pages):
            tables[i, :n] = perm[at:at + n]
            at += n
        k = rng.integers(-32768, 32768, (total, NKV, PAGE, D)).astype(np.int16)
        v = rng.integers(-32768, 32768, (total, NKV, PAGE, D)).astype(np.int16)
        kept = np.full((b, NKV, budget), -1, np.int32)
        for i, n in enumerate(lens):
            for h in range(NKV):
                m = min(n, budget)
                kept[i, h, :m] = np.sort(rng.choice(n, m, replace=False))
        per = -(-budget // PAGE) + 1
        dtab = rng.permutation(b * per).astype(np.int32).reshape(b, per)
        dk = rng.integers(-32768, 32768, (b * per, NKV, PAGE, D)).astype(np.int16)
        dv = dk + 1
        dev = [torch.from_numpy(x).cuda() for x in (k, v, tables, kept, dk, dv, dtab)]
        cuda.kv_evict_compact(*dev)
        torch.cuda.synchronize()
        assert cuda.device_error() == (0, 0)
        for i in range(b):
            for h in range(NKV):
                for j in range(budget):
                    t = kept[i, h, j]
                    if t >= 0:
                        dk[dtab[i, j // PAGE], h, j % PAGE] = k[tables[i, t // PAGE], h, t % PAGE]
                        dv[dtab[i, j // PAGE], h, j % PAGE] = v[tables[i, t // PAGE], h, t % PAGE]
        assert np.array_equal(dev[4].cpu().numpy(), dk) and np.array_equal(dev[5].cpu().numpy(), dv)


def test_compact_bad_indices(cuda):
    import torch
    k = torch.ones((4, NKV, PAGE, D), dtype=torch.bfloat16, device="cuda")
    dk = torch.zeros((2, NKV, PAGE, D), dtype=torch.bfloat16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    tables, dtab = torch.tensor([[0, 1, 2]], **i32), torch.tensor([[0, 1]], **i32)
    kept = torch.arange(20, **i32).repeat(1, NKV, 1).contiguous()
    for what, code, detail in (("index", 905, 48), ("source page", 901, 4), ("destination page", 901, 2)):
        kp, tb, dt = kept.clone(), tables.clone(), dtab.clone()
        if what == "index":
            kp[0, 1, 3] = 48
        elif what == "source page":
            tb[0, 1] = 4
        else:
            dt[0, 1] = 2
        dk.zero_()
        cuda.kv_evict_compact(k, k, tb, kp, dk, dk.clone(), dt)
        assert cuda.device_error() == (code, detail)
        good = torch.ones((2, NKV, PAGE), device="cuda")
        good[1, :, 4:] = 0
        if what == "index":
            good[0, 1, 3] = 0
        else:
            good[1] = 0
        assert torch.equal(dk.float(), good[..., None].expand_as(dk))


def test_serving_run(cuda):
    """Two requests: prompts in chunks with weights, two decode steps, eviction to a budget, further
    decode steps over the compacted cache. Every step against float64 attention over what is kept."""
    import torch
    budget, first, last = 96, 4, 32
    gen = torch.Generator(device="cuda").manual_seed(4)
    prompt, steps = [200, 70], 3
    total = [n + 5 for n in prompt]
    pages = [-(-n // PAGE) for n in total]
    kx = [torch.randn((n, NKV, D), generator=gen, device="cuda").to(torch.bfloat16) for n in total]
    vx = [torch.randn((n, NKV, D), generator=gen, device="cuda").to(torch.bfloat16) for n in total]
    pool = sum(pages) + 2 * -(-(budget + 8) // PAGE)
    k = torch.full((pool, NKV, PAGE, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    v = k.clone()
    tables = torch.zeros((2, max(pages)), dtype=torch.int32, device="cuda")
    tables[0, :pages[0]] = torch.arange(pages[0])
    tables[1, :pages[1]] = torch.arange(pages[0], sum(pages))
    fresh = torch.arange(sum(pages), pool, device="cuda").to(torch.int32).reshape(2, -1)
    w = torch.zeros((2, NKV, 256), device="cuda")
    expect = torch.zeros((2, NKV, 256), dtype=torch.float64, device="cuda")
    lens = [0, 0]     # tokens in the cache
    seen = [0, 0]     # tokens of the request so far
    keep = [None, None]

    def step(ns):
        for b, n in enumerate(ns):
            for i in range(n):
                t = lens[b] + i
                page = int(tables[b, t // PAGE])
                k[page, :, t % PAGE], v[page, :, t % PAGE] = kx[b][seen[b] + i], vx[b][seen[b] + i]
            lens[b] += n
            seen[b] += n
        starts = [0, ns[0], ns[0] + ns[1]]
        c = dict(seqs=list(zip(ns, lens)), starts=starts, rows=starts[-1], k=k, v=v, tables=tables,
                 q=torch.randn((starts[-1], NQ, D), generator=gen, device="cuda").to(torch.bfloat16), gate=None,
                 q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                 seq_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), qmax=max(ns), lmax=max(lens))
        before = w.clone()
        got = _chunk.call(cuda, c, weights=w)
        _chunk.check(c, got, _chunk.reference(c), w, before)
        return c

    for a in ([128, 64], [72, 6], [1, 1], [1, 1]):
        step(a)
    # evict
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kept = torch.empty((2, NKV, budget), dtype=torch.int32, device="cuda")
    new = torch.empty(2, dtype=torch.int32, device="cuda")
    w_old, k_old, v_old = w.cpu().numpy(), k.clone(), v.clone()
    cuda.kv_evict_select(w, seq_lens, max(lens), budget, first, last, kept, new, weights_out=w)
    cuda.kv_evict_compact(k, v, tables, kept, k, v, fresh)
    assert new.tolist() == [budget, lens[1]]
    for b in range(2):
        for h in range(NKV):
            ids = ref_select(w_old[b, h], lens[b], budget, first, last)
            assert np.array_equal(kept[b, h, :len(ids)].cpu().numpy(), ids)
            i = torch.arange(len(ids), device="cuda")
            t = torch.from_numpy(ids).cuda()
            at = (fresh[b].long()[i // PAGE], h, i % PAGE)
            assert torch.equal(k[at], k_old[tables[b].long()[t // PAGE], h, t % PAGE])
            assert torch.equal(v[at], v_old[tables[b].long()[t // PAGE], h, t % PAGE])
    tables, lens = fresh, new.tolist()
    for a in ([1, 1], [1, 2]):
        step(a)
    assert cuda.device_error() == (0, 0)
