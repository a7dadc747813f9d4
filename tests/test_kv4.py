"""The paged 4-bit key / value cache without a GPU: sizes, and every refusal of a call's host arguments, through the C
ABI (nothing is launched: the refusals come before the first look at a device pointer) and through the torch view."""
import ctypes as C

import pytest
import torch

from jepa_b200 import kv4, lib as jlib

PTR = 1 << 20      # an aligned address that no refused call looks at


def _err():
    L = jlib.load()
    t = L.jepa_error_text().decode()
    L.jepa_error_reset()
    return t


def _cache(**kw):
    a = dict(q=PTR, d=PTR, n_pages=4, page_size=16, kv_heads=2, head_dim=64)
    a.update(kw)
    return kv4._Cache(*(a[n] for n, _ in kv4._Cache._fields_))


def _attn(**kw):
    a = dict(q=PTR, out=PTR, q_tok=256, q_head=64, o_tok=256, o_head=64, q_start=PTR, lens=PTR, table=PTR, n_req=2, n_rows=3,
             width=4, n_heads=4, type=1, frame=0, scale=0.125, max_len=0, max_new=0, workspace=None, workspace_bytes=0)
    a.update(kw)
    return kv4._Attn(*(a[n] for n, _ in kv4._Attn._fields_))


@pytest.mark.parametrize("pages,page,heads,dim", [(1, 16, 1, 32), (3, 64, 5, 96), (7, 256, 16, 128), ((1 << 31) - 1, 256, 1024, 128)])
def test_sizes(pages, page, heads, dim):
    L = kv4._load()
    q, d = C.c_size_t(), C.c_size_t()
    c = _cache(n_pages=pages, page_size=page, kv_heads=heads, head_dim=dim)
    assert L.jepa_b200_kv4_bytes(C.byref(c), C.byref(q), C.byref(d)) == 0
    assert q.value == pages * 2 * heads * page * dim // 2 and d.value == pages * 2 * heads * page * dim // 32 * 2


@pytest.mark.parametrize("bad,word", [(dict(head_dim=48), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(page_size=8), "page_size"),
                                      (dict(page_size=48), "page_size"), (dict(page_size=512), "page_size"), (dict(n_pages=0), "pages"),
                                      (dict(n_pages=1 << 31), "pages"), (dict(kv_heads=0), "heads"), (dict(kv_heads=1025), "heads")])
def test_refused_caches(bad, word):
    L = kv4._load()
    c = _cache(**bad)
    q, d = C.c_size_t(), C.c_size_t()
    a = _attn()
    calls = [lambda: L.jepa_b200_kv4_bytes(C.byref(c), C.byref(q), C.byref(d)),
             lambda: L.jepa_b200_kv4_store(C.byref(c), PTR, PTR, 1, 128, 64, 128, 64, PTR, 1, None),
             lambda: L.jepa_b200_kv4_load(C.byref(c), PTR, 1, PTR, PTR, 1, None),
             lambda: L.jepa_b200_kv4_attention(C.byref(c), C.byref(a), None),
             lambda: L.jepa_b200_kv4_attention_workspace(C.byref(c), C.byref(a))]
    for call in calls:
        assert call() == -1 and word in _err()


def test_refused_rows():
    L, c = kv4._load(), _cache()
    r = C.byref(c)
    assert L.jepa_b200_kv4_store(None, PTR, PTR, 1, 128, 64, 128, 64, PTR, 1, None) == -1 and "cache is null" in _err()
    assert L.jepa_b200_kv4_store(r, PTR, PTR, 2, 128, 64, 128, 64, PTR, 1, None) == -1 and "type 2" in _err()
    assert L.jepa_b200_kv4_store(r, PTR, PTR, 1, 128, 64, 128, 64, PTR, -1, None) == -1 and "tokens" in _err()
    assert L.jepa_b200_kv4_store(r, PTR, PTR, 1, 128, -64, 128, 64, PTR, 1, None) == -1 and "strides" in _err()
    assert L.jepa_b200_kv4_store(r, None, PTR, 1, 128, 64, 128, 64, PTR, 1, None) == -1 and "k is null" in _err()
    assert L.jepa_b200_kv4_store(r, PTR + 1, PTR, 1, 128, 64, 128, 64, PTR, 1, None) == -1 and "aligned" in _err()
    assert L.jepa_b200_kv4_store(r, PTR, PTR, 1, 128, 64, 128, 64, PTR + 4, 1, None) == -1 and "slots must be 8-byte" in _err()
    assert L.jepa_b200_kv4_load(r, PTR, 1, PTR + 8, PTR, 1, None) == -1 and "k must be 16-byte" in _err()
    assert L.jepa_b200_kv4_load(r, None, 1, PTR, PTR, 1, None) == -1 and "slots is null" in _err()
    assert L.jepa_b200_kv4_load(r, PTR, -1, PTR, PTR, 1, None) == -1
    assert L.jepa_b200_kv4_load(r, PTR, 1, PTR, PTR, 8, None) == -1 and "type 8" in _err()
    half = _cache(q=PTR + 8)
    assert L.jepa_b200_kv4_load(C.byref(half), PTR, 1, PTR, PTR, 1, None) == -1 and "cache.q must be 16-byte" in _err()
    # no rows: nothing to do, whatever the pointers
    assert L.jepa_b200_kv4_store(r, None, None, 1, 0, 0, 0, 0, None, 0, None) == 0
    assert L.jepa_b200_kv4_load(r, None, 0, None, None, 1, None) == 0


@pytest.mark.parametrize("bad,word", [
    (dict(type=0), "type 0"), (dict(n_heads=3), "query heads"), (dict(n_heads=0), "query heads"), (dict(n_heads=65536), "query heads"),
    (dict(n_req=-1), "requests"), (dict(n_req=65536), "requests"), (dict(n_rows=-1), "rows"), (dict(width=0), "columns"),
    (dict(width=1 << 27), "2^31"), (dict(n_rows=(1 << 28) + 1), "2^30"), (dict(frame=-1), "frame"), (dict(max_len=-1), "max_len"), (dict(max_new=-2), "max_new"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q_tok=-1), "strides"), (dict(o_tok=63), "overlap"),
    (dict(o_head=63), "overlap"), (dict(q=None), "q is null"), (dict(out=None), "out is null"), (dict(lens=PTR + 2), "lens must be 4-byte"),
    (dict(table=None), "table is null"), (dict(q_start=None), "q_start is null"), (dict(q=PTR + 1), "q must be 2-byte")])
def test_refused_attention(bad, word):
    L, c = kv4._load(), _cache()
    a = _attn(**bad)
    ws = L.jepa_b200_kv4_attention_workspace(C.byref(c), C.byref(_attn()))
    a.workspace, a.workspace_bytes = PTR, ws
    assert L.jepa_b200_kv4_attention(C.byref(c), C.byref(a), None) == -1
    assert word in _err()


def test_attention_over_nothing_is_no_call():
    L, c = kv4._load(), _cache()
    for bad in (dict(n_req=0), dict(n_rows=0)):
        a = _attn(q=None, out=None, lens=None, **bad)
        assert L.jepa_b200_kv4_attention(C.byref(c), C.byref(a), None) == 0
    assert L.jepa_b200_kv4_attention(C.byref(c), None, None) == -1 and "arguments are null" in _err()


@pytest.mark.parametrize("bad,word", [(dict(n_req=0), "n_req"), (dict(width=0), "width"), (dict(n_free=-1), "n_free"),
                                      (dict(n_slots=0), "n_slots"), (dict(n_slots=(1 << 30) + 1), "2^30"), (dict(n_req=(1 << 30) + 1), "2^30"),
                                      (dict(n_free=(1 << 30) + 1), "2^30"), (dict(page=24), "page_size"), (dict(page=8), "page_size"),
                                      (dict(cached=None), "cached is null"), (dict(slots=PTR + 4), "slots must be 8-byte"),
                                      (dict(free=None), "free_pages is null"), (dict(state=PTR + 2), "state must be 4-byte")])
def test_refused_tables(bad, word):
    L = kv4._load()
    a = dict(cached=PTR, n_req=2, page=16, width=4, free=PTR, n_free=8, slots=PTR, n_slots=8, state=PTR)
    a.update(bad)
    rc = L.jepa_b200_kv_tables(a["cached"], PTR, a["n_req"], a["page"], PTR, a["width"], a["free"], a["n_free"], PTR, PTR, a["slots"],
                               a["n_slots"], a["state"], None)
    assert rc == -1 and word in _err()


def test_torch_view_refuses_what_is_not_on_a_gpu():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    with pytest.raises(ValueError, match="cached must be on the CUDA device"):
        kv4.build_tables(i32(2), i32(2), i32(2, 4), i32(8), 16, 8)
    with pytest.raises(ValueError, match="q must be on the CUDA device"):
        kv4.KV4Cache.wrap(torch.zeros(4, 2, 2, 16, 32, dtype=torch.uint8), torch.zeros(4, 2, 2, 2, 16, dtype=torch.float16))
    with pytest.raises(ValueError, match="5-D"):
        kv4.KV4Cache.wrap(torch.zeros(4, 2, 2, 16, dtype=torch.uint8), torch.zeros(4, 2, 2, 2, 16, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="head_dim 80"):
        kv4.KV4Cache(4, 16, 2, 80, device="cpu")


def test_torch_view_refuses_rows_that_require_grad():
    """Codes have no gradient: a row that autograd follows would lose it without a word."""
    c = kv4.KV4Cache.__new__(kv4.KV4Cache)
    c.head_dim, c.kv_heads, c._dev = 64, 2, torch.device("cpu")
    x = torch.zeros(3, 2, 64, requires_grad=True)
    for t in (x, x * 2, (x * 2).half()):
        with pytest.raises(ValueError, match="k requires grad"):
            c._rows(t, "k", 3, 2)
        assert c._rows(t.detach(), "k", 3, 2) == (128, 64, 1)
        with torch.no_grad():
            assert c._rows(t, "k", 3, 2) == (128, 64, 1)


@pytest.mark.parametrize("heads", [1, 3, 8, 1024])
def test_more_tokens_than_a_grid_holds_are_refused(heads):
    L = kv4._load()
    r = C.byref(_cache(kv_heads=heads))
    most = (0x7fffffff // heads - 1) * 16
    assert -(-(-(-most // 4) * heads) // 4) <= 0x7fffffff         # blocks of four warps, four tokens of one head each
    for n in (most + 1, 1 << 40, 1 << 60, (1 << 61) + 8, (1 << 63) - 7, (1 << 63) - 1):
        assert L.jepa_b200_kv4_store(r, PTR, PTR, 1, 128, 64, 128, 64, PTR, n, None) == -1 and "out of range" in _err()
        assert L.jepa_b200_kv4_load(r, PTR, n, PTR, PTR, 0, None) == -1 and "out of range" in _err()
    # the largest count comes as far as the pointers
    assert L.jepa_b200_kv4_store(r, None, PTR, 1, 128, 64, 128, 64, PTR, most, None) == -1 and "k is null" in _err()
