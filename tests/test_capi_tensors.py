"""The tensor helpers of the ragged and eviction entries refuse tensors that do not agree, before a pointer
reaches the library: short or strided arrays, other types, another device. The library is a stand-in that
counts its calls, and CPU tensors play those of the current device (torch calls theirs device -1)."""
import pytest
import torch

INVALID, BOUNDS = -1, -2
B, ROWS, PAGES, WIDTH, LMAX, BUDGET = 3, 7, 9, 4, 60, 20


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


@pytest.fixture
def capi(monkeypatch):
    from peregrine_b200 import capi
    lib = Library()
    monkeypatch.setattr(capi, "lib", lambda: lib)
    monkeypatch.setattr(capi, "_torch_current", lambda: (lambda: -1, lambda d: 55))
    capi.seen = lib.calls
    return capi


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def b16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def chunk():
    return dict(q=b16(ROWS, 16, 256), k_pages=b16(PAGES, 4, 16, 256), v_pages=b16(PAGES, 4, 16, 256),
                block_tables=i32(B, WIDTH), q_starts=i32(B + 1), seq_lens=i32(B), max_q_len=4, max_seq_len=LMAX, scale=0.5,
                out=b16(ROWS, 16, 256), workspace=torch.zeros(640, dtype=torch.uint8), gate=b16(ROWS, 16, 256),
                lse=torch.zeros(ROWS, 16))


def chunk_weights():
    return dict(chunk(), weights=torch.zeros(5, 4, LMAX + 4), slots=i32(B))


def select():
    return dict(weights=torch.zeros(5, 4, LMAX), seq_lens=i32(B), max_seq_len=LMAX, budget=BUDGET, keep_first=1,
                keep_last=2, kept=i32(B, 4, BUDGET), new_lens=i32(B), weights_out=torch.zeros(5, 4, LMAX), slots=i32(B))


def compact():
    return dict(src_k=b16(PAGES, 4, 16, 256), src_v=b16(PAGES, 4, 16, 256), src_tables=i32(B, WIDTH), kept=i32(B, 4, BUDGET),
                dst_k=b16(6, 4, 16, 256), dst_v=b16(6, 4, 16, 256), dst_tables=i32(B, 2))


ENTRIES = dict(chunk_attn=chunk, chunk_attn_weights=chunk_weights, kv_evict_select=select, kv_evict_compact=compact)
SHAPED = [(f, n) for f, make in ENTRIES.items() for n, v in make().items() if torch.is_tensor(v)]


def strided(t):
    """The same numbers of t, every second element of an array twice as long."""
    return torch.zeros((*t.shape[:-1], 2 * t.shape[-1]), dtype=t.dtype)[..., ::2]


@pytest.mark.parametrize("entry", list(ENTRIES))
def test_agreeing_tensors_reach_the_library(capi, entry):
    a = ENTRIES[entry]()
    getattr(capi, entry)(**a)
    getattr(capi, entry)(**{n: v for n, v in a.items() if n not in ("gate", "lse", "slots", "new_lens", "weights_out")})
    getattr(capi, entry)(**a, stream=77)
    assert [n for n, _ in capi.seen] == ["pgc_" + entry] * 3
    assert [c[-1] for _, c in capi.seen] == [55, 55, 77]
    if entry.startswith("chunk"):
        assert capi.seen[0][1][3:6:2] == (PAGES, WIDTH) and capi.seen[0][1][8:12] == (B, ROWS, 4, LMAX)


def test_rows_behind_the_queries_are_allowed(capi):
    a = chunk()
    a.update(out=b16(ROWS + 1, 16, 256), gate=b16(ROWS + 2, 16, 256), lse=torch.zeros(ROWS + 1, 16), block_tables=i32(B + 1, WIDTH))
    capi.chunk_attn(**a)
    bits = {n: v.view(torch.int16) if torch.is_tensor(v) and v.dtype is torch.bfloat16 else v for n, v in a.items()}
    capi.chunk_attn(**bits)
    assert len(capi.seen) == 2


@pytest.mark.parametrize("entry,name", [x for x in SHAPED if x[1] != "workspace"])  # its bytes go to the library
def test_one_element_row_short(capi, entry, name):
    a = ENTRIES[entry]()
    others = [a[name][:-1], a[name].flatten()[:-1]]
    if name in ("q", "k_pages", "src_k", "dst_k"):  # these say how many there are: one more, and the others are short
        others[0] = torch.cat([a[name], a[name][:1]])
    elif entry.startswith("chunk") and name == "weights" or entry == "kv_evict_compact" and name == "kept":
        others = others[1:]  # these say the number of slots and the batch: there are fewer
    for other in others:
        with pytest.raises(capi.PgcError) as e:
            getattr(capi, entry)(**{**a, name: other})
        assert e.value.status == BOUNDS
    assert capi.seen == []


@pytest.mark.parametrize("entry,name", [x for x in SHAPED if x[1] != "workspace"])
def test_strided(capi, entry, name):
    a = ENTRIES[entry]()
    a[name] = strided(a[name])
    with pytest.raises(capi.PgcError) as e:
        getattr(capi, entry)(**a)
    assert e.value.status == INVALID and capi.seen == []


@pytest.mark.parametrize("entry,name,dtype", [
    ("chunk_attn", "q", torch.float16), ("chunk_attn", "out", torch.float32), ("chunk_attn", "k_pages", torch.float32),
    ("chunk_attn", "gate", torch.float32), ("chunk_attn", "lse", torch.float64), ("chunk_attn", "seq_lens", torch.int64),
    ("chunk_attn", "q_starts", torch.int64), ("chunk_attn", "block_tables", torch.int64),
    ("chunk_attn_weights", "weights", torch.float64), ("chunk_attn_weights", "slots", torch.int64),
    ("kv_evict_select", "weights", torch.int32), ("kv_evict_select", "kept", torch.int64),
    ("kv_evict_select", "seq_lens", torch.int64), ("kv_evict_select", "new_lens", torch.int64),
    ("kv_evict_select", "slots", torch.int64), ("kv_evict_select", "weights_out", torch.float64),
    ("kv_evict_compact", "kept", torch.int64), ("kv_evict_compact", "src_tables", torch.int64),
    ("kv_evict_compact", "dst_tables", torch.int64), ("kv_evict_compact", "src_k", torch.float16)])
def test_other_types(capi, entry, name, dtype):
    a = ENTRIES[entry]()
    a[name] = a[name].to(dtype)
    with pytest.raises(capi.PgcError):
        getattr(capi, entry)(**a)
    assert capi.seen == []


@pytest.mark.parametrize("entry", list(ENTRIES))
def test_other_heads_and_dims(capi, entry):
    a = ENTRIES[entry]()
    changes = dict(kv_evict_select=dict(weights=torch.zeros(5, 8, LMAX)), kv_evict_compact=dict(kept=i32(B, 8, BUDGET)),
                   chunk_attn=dict(q=b16(ROWS, 32, 256)), chunk_attn_weights=dict(weights=torch.zeros(5, 8, LMAX)))[entry]
    for change in [changes] + [dict(budget=n) for n in (BUDGET - 1, BUDGET + 1) if "budget" in a]:
        with pytest.raises(capi.PgcError):
            getattr(capi, entry)(**{**a, **change})
    assert capi.seen == []


@pytest.mark.parametrize("entry", list(ENTRIES))
def test_other_device(capi, monkeypatch, entry):
    monkeypatch.setattr(capi, "_torch_current", lambda: (lambda: 0, lambda d: 55))
    with pytest.raises(capi.PgcError) as e:
        getattr(capi, entry)(**ENTRIES[entry]())
    assert e.value.status == INVALID and capi.seen == []


@pytest.mark.gpu
@pytest.mark.parametrize("entry,name", [x for x in SHAPED])
def test_one_tensor_on_the_cpu(cuda, entry, name):
    a = {n: v.cuda() if torch.is_tensor(v) and n != name else v for n, v in ENTRIES[entry]().items()}
    with pytest.raises(cuda.PgcError) as e:
        getattr(cuda, entry)(**a)
    assert e.value.status == INVALID
