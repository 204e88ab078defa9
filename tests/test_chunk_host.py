"""Refusals of the ragged-batch and eviction entries: arguments are checked on the host before the
device is asked for, so none of this needs a GPU (no pointer here is ever read)."""
import pytest

INVALID, BOUNDS, WORKSPACE, ALIGN = -1, -2, -3, -5
A = 1 << 20  # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    from peregrine_b200 import build, capi
    build.build()
    return capi.lib()


CHUNK = dict(q=A, k=A, v=A, pages=100, tables=A, width=10, starts=A, lens=A, batch=2, rows=8, qmax=4, lmax=160,
             scale=0.0625, gate=None, out=A, lse=None, ws=A, ws_bytes=1 << 40, stream=None)
WEIGHTS = dict(weights=A, stride=160, num_slots=2, slots=None)


def chunk(lib, with_weights, **change):
    a = {**CHUNK, **WEIGHTS, **change}
    head = [a[x] for x in ("q", "k", "v", "pages", "tables", "width", "starts", "lens", "batch", "rows", "qmax", "lmax",
                           "scale", "gate", "out", "lse")]
    tail = [a["ws"], a["ws_bytes"], a["stream"]]
    if with_weights:
        return lib.pgc_chunk_attn_weights(*head, a["weights"], a["stride"], a["num_slots"], a["slots"], *tail)
    return lib.pgc_chunk_attn(*head, *tail)


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("change,status", [
    (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(tables=None), INVALID),
    (dict(starts=None), INVALID), (dict(lens=None), INVALID), (dict(out=None), INVALID), (dict(ws=None), WORKSPACE),
    (dict(pages=0), INVALID), (dict(batch=-1), INVALID), (dict(rows=-1), INVALID), (dict(qmax=-1), INVALID),
    (dict(lmax=-1), INVALID), (dict(lmax=0), INVALID), (dict(width=-1), INVALID), (dict(width=0), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(scale=0.0), INVALID), (dict(scale=-0.0625), INVALID), (dict(batch=4097, num_slots=5000), BOUNDS),
    (dict(width=9), BOUNDS), (dict(pages=1 << 25), BOUNDS), (dict(rows=(1 << 22) + 1), BOUNDS),
    (dict(lmax=(1 << 24) + 1, width=1 << 21, stride=1 << 25), BOUNDS), (dict(ws_bytes=0), WORKSPACE),
    (dict(q=A + 8), ALIGN), (dict(k=A + 2), ALIGN), (dict(v=A + 4), ALIGN), (dict(gate=A + 8), ALIGN),
    (dict(out=A + 2), ALIGN), (dict(ws=A + 4), ALIGN), (dict(lse=A + 2), ALIGN),
    (dict(batch=0), 0), (dict(rows=0), 0), (dict(qmax=0), 0)])
def test_chunk_refusals(lib, weights, change, status):
    assert chunk(lib, weights, **change) == status


@pytest.mark.parametrize("change,status", [
    (dict(weights=None), INVALID), (dict(weights=A + 2), ALIGN), (dict(stride=159), BOUNDS), (dict(num_slots=0), BOUNDS),
    (dict(num_slots=1), BOUNDS)])
def test_chunk_weights_refusals(lib, change, status):
    assert chunk(lib, True, **change) == status


@pytest.mark.parametrize("qmax", [4, 5])
@pytest.mark.parametrize("weights", [0, 1])
def test_workspace_is_required_in_full(lib, qmax, weights):
    need = lib.pgc_chunk_workspace_bytes(2, 8, qmax, 160, weights)
    assert need > 0
    assert chunk(lib, bool(weights), qmax=qmax, ws_bytes=need - 1) == WORKSPACE
    for bad in ((0, 8, 4, 160), (4097, 8, 4, 160), (2, 0, 4, 160), (2, (1 << 22) + 1, 4, 160), (2, 8, 0, 160),
                (2, 8, 4, 0), (2, 8, 4, (1 << 24) + 1)):
        assert lib.pgc_chunk_workspace_bytes(*bad, weights) == 0


def test_workspace_grows_with_the_shape(lib):
    f = lib.pgc_chunk_workspace_bytes
    assert f(2, 8, 4, 160, 1) > f(2, 8, 4, 160, 0)
    scores, lse = 8 * 4 * (1 << 15) * 4 * 4, 8 * 16 * 4
    assert f(2, 8, 4, 1 << 15, 1) - f(2, 8, 4, 1 << 15, 0) == scores + lse
    assert f(2, 8, 4, 1 << 20, 0) == f(2, 1 << 12, 4, 100, 0) <= 10 << 20
    assert f(4096, 1 << 20, 512, 1 << 20, 0) == f(1, 5, 5, 100, 0) <= 39 << 20


SELECT = dict(w=A, wo=None, stride=160, num_slots=2, slots=None, lens=A, batch=2, lmax=160, budget=32, first=4, last=8,
              kept=A, new=None, stream=None)


@pytest.mark.parametrize("change,status", [
    (dict(w=None), INVALID), (dict(lens=None), INVALID), (dict(kept=None), INVALID), (dict(new=A), INVALID),
    (dict(batch=-1), INVALID), (dict(lmax=-1), INVALID), (dict(budget=0), INVALID), (dict(first=-1), INVALID),
    (dict(last=-1), INVALID), (dict(first=25), INVALID), (dict(first=(1 << 31) - 1, last=(1 << 31) - 1), INVALID),
    (dict(num_slots=0), INVALID), (dict(num_slots=1), BOUNDS), (dict(stride=159), BOUNDS),
    (dict(lmax=262145, stride=1 << 20), BOUNDS), (dict(batch=65536, num_slots=70000), BOUNDS), (dict(w=A + 2), ALIGN),
    (dict(wo=A + 2), ALIGN), (dict(batch=0), 0)])
def test_select_refusals(lib, change, status):
    assert lib.pgc_kv_evict_select(*{**SELECT, **change}.values()) == status


COMPACT = dict(k=A, v=A, pages=100, tables=A, width=10, kept=A, batch=2, budget=32, dk=A, dv=A, dpages=10, dtables=A,
               dwidth=2, stream=None)


@pytest.mark.parametrize("change,status", [
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(tables=None), INVALID), (dict(kept=None), INVALID),
    (dict(dk=None), INVALID), (dict(dv=None), INVALID), (dict(dtables=None), INVALID), (dict(pages=0), INVALID),
    (dict(dpages=0), INVALID), (dict(width=-1), INVALID), (dict(batch=-1), INVALID), (dict(budget=-1), INVALID),
    (dict(dwidth=1), BOUNDS), (dict(batch=1 << 20, budget=1 << 10, dwidth=64), BOUNDS), (dict(k=A + 8), ALIGN),
    (dict(dv=A + 2), ALIGN), (dict(batch=0), 0), (dict(budget=0), 0)])
def test_compact_refusals(lib, change, status):
    assert lib.pgc_kv_evict_compact(*{**COMPACT, **change}.values()) == status


def test_index_arrays_must_be_aligned(lib):
    for name in ("tables", "starts", "lens"):
        for weights in (False, True):
            assert chunk(lib, weights, **{name: A + 2}) == ALIGN
    assert chunk(lib, True, slots=A + 1) == ALIGN
    for name in ("slots", "lens", "kept", "new"):
        assert lib.pgc_kv_evict_select(*{**SELECT, name: A + 2}.values()) == ALIGN
    for name in ("tables", "kept", "dtables"):
        assert lib.pgc_kv_evict_compact(*{**COMPACT, name: A + 1}.values()) == ALIGN


def test_select_budget_bound(lib):
    assert lib.pgc_kv_evict_select(*{**SELECT, "budget": (1 << 30) + 1}.values()) == BOUNDS
