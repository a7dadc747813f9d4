"""The paged 4-bit key / value cache on torch CUDA tensors: block tables and slot maps of a step, store, load, and the
attention that reads the cache (include/jepa_b200.h, the kv4 block). Every call runs on the current stream of the
tensors' device, without a synchronisation, and can be captured into a CUDA graph. There is no backward pass: rows that
require grad are refused while autograd is on.

    cache = KV4Cache(n_pages, page_size, kv_heads, head_dim)
    t = build_tables(cached, added, table, free_pages, page_size, n_slots)   # new pages, slots, row ranges
    cache.store(k, v, t.slots)                                              # this step's rows
    out = cache.attention(q, t.q_start, t.lens, table, frame=258, max_new=258)
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import lib as jlib

_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


class _Cache(C.Structure):
    _fields_ = [("q", C.c_void_p), ("d", C.c_void_p), ("n_pages", C.c_int64), ("page_size", C.c_int32),
                ("kv_heads", C.c_int32), ("head_dim", C.c_int32)]


class _Attn(C.Structure):
    _fields_ = [("q", C.c_void_p), ("out", C.c_void_p), ("q_tok", C.c_int64), ("q_head", C.c_int64), ("o_tok", C.c_int64),
                ("o_head", C.c_int64), ("q_start", C.c_void_p), ("lens", C.c_void_p), ("table", C.c_void_p),
                ("n_req", C.c_int32), ("n_rows", C.c_int32), ("width", C.c_int32), ("n_heads", C.c_int32),
                ("type", C.c_uint32), ("frame", C.c_int32), ("scale", C.c_float), ("max_len", C.c_int32),
                ("max_new", C.c_int32), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


_lib: Optional[C.CDLL] = None


def _load() -> C.CDLL:
    global _lib
    if _lib is None:
        L = jlib.load()
        vp, i32, i64, cp = C.c_void_p, C.c_int, C.c_int64, C.POINTER(_Cache)
        sig = {
            "jepa_b200_kv4_bytes": (i32, [cp, C.POINTER(C.c_size_t), C.POINTER(C.c_size_t)]),
            "jepa_b200_kv_tables": (i32, [vp, vp, i32, i32, vp, i32, vp, i32, vp, vp, vp, i32, vp, vp]),
            "jepa_b200_kv4_store": (i32, [cp, vp, vp, C.c_uint32, i64, i64, i64, i64, vp, i64, vp]),
            "jepa_b200_kv4_load": (i32, [cp, vp, i64, vp, vp, C.c_uint32, vp]),
            "jepa_b200_kv4_attention_workspace": (i64, [cp, C.POINTER(_Attn)]),
            "jepa_b200_kv4_attention_plan": (i32, [cp, C.POINTER(_Attn), C.POINTER(C.c_int)]),
            "jepa_b200_kv4_attention": (i32, [cp, C.POINTER(_Attn), vp]),
            "jepa_b200_kv4_attention_giving_up": (i32, [cp, C.POINTER(_Attn), i32, C.c_longlong, vp]),
            "jepa_b200_kv4_check": (i32, [vp]),
        }
        for name, (res, args) in sig.items():
            f = getattr(L, name)
            f.restype, f.argtypes = res, args
        _lib = L
    return _lib


def _stream(dev: torch.device) -> int:
    """The raw handle of the device's current stream (without a torch.cuda.Stream object, which takes 3 us to make)."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _call(name: str, dev: torch.device, *args) -> None:
    """One call on the device's current stream (the C entry works on the current device)."""
    fn = getattr(_lib or _load(), name)
    if dev.index == torch.cuda.current_device():
        rc = fn(*args, _stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream(dev))
    if rc != 0:
        _raise(_load(), name)


def _raise(L: C.CDLL, name: str) -> None:
    text = (L.jepa_error_text() or b"").decode(errors="replace").strip().splitlines()
    L.jepa_error_reset()
    raise RuntimeError(text[-1] if text else f"{name} failed")


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _index(t: torch.Tensor, name: str, dtype: torch.dtype, dev: Optional[torch.device], dim: int = 1) -> None:
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.dim() == dim and t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dim}-D tensor of {dtype}")
    if not (t.is_cuda and (dev is None or t.device == dev)):
        raise ValueError(f"{name} must be on the CUDA device of the others")


class Tables(NamedTuple):
    """What build_tables gives: the arrays that store and attention take, and state = [refusal code or 0, pages taken]."""
    lens: torch.Tensor
    q_start: torch.Tensor
    slots: torch.Tensor
    state: torch.Tensor


def build_tables(cached: torch.Tensor, added: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor, page_size: int,
                 n_slots: int) -> Tables:
    """The bookkeeping of one step from the requests' lengths (int32, on the GPU): fresh pages from the start of
    free_pages go into `table` [n_req, width] (changed in place), every new row gets its slot. n_slots is the size of
    the slot map, at least the number of new rows; the rest is -1. A refused step (state[0] != 0) changes nothing and
    gives empty row ranges: see jepa_b200_kv_tables."""
    _index(cached, "cached", torch.int32, None)
    dev, n = cached.device, cached.shape[0]
    _index(added, "added", torch.int32, dev)
    _index(table, "table", torch.int32, dev, 2)
    _index(free_pages, "free_pages", torch.int32, dev)
    rows, width = table.shape
    n_free = free_pages.shape[0]
    if added.shape[0] != n or rows != n:
        raise ValueError("cached, added and table must have one entry a request")
    if not (n >= 1 and width >= 1):
        raise ValueError("there must be a request and a table column")
    if not (1 <= n_slots <= 2 ** 30 and max(n, width, n_free, page_size) <= 2 ** 30):
        raise ValueError("n_slots must be 1 or more, and no count may pass 2^30")
    # lens, q_start and state share one allocation, each at a multiple of 4 bytes
    ints = cached.new_empty(2 * n + 3)
    lens, q_start, state = torch.split_with_sizes(ints, (n, n + 1, 2))
    slots = cached.new_empty(n_slots, dtype=torch.int64)
    base = ints.data_ptr()
    _call("jepa_b200_kv_tables", dev, cached.data_ptr(), added.data_ptr(), n, page_size, table.data_ptr(), width,
          free_pages.data_ptr(), n_free, base, base + 4 * n, slots.data_ptr(), n_slots, base + 4 * (2 * n + 1))
    return Tables(lens, q_start, slots, state)


class KV4Cache:
    """A pool of pages of token rows whose keys and values are held in 4 bits (layout: include/jepa_b200.h)."""

    def __init__(self, n_pages: int, page_size: int, kv_heads: int, head_dim: int, device="cuda"):
        c = _Cache(None, None, n_pages, page_size, kv_heads, head_dim)
        L, qb, db = _load(), C.c_size_t(), C.c_size_t()
        if L.jepa_b200_kv4_bytes(C.byref(c), C.byref(qb), C.byref(db)) != 0:
            _raise(L, "jepa_b200_kv4_bytes")
        self._bind(torch.zeros((n_pages, 2, kv_heads, page_size, head_dim // 2), dtype=torch.uint8, device=device),
                   torch.zeros((n_pages, 2, kv_heads, head_dim // 32, page_size), dtype=torch.float16, device=device))

    @classmethod
    def wrap(cls, q: torch.Tensor, d: torch.Tensor) -> "KV4Cache":
        """A cache over buffers that exist: q uint8 [pages, 2, heads, page, dim / 2], d f16 [pages, 2, heads, dim / 32, page]."""
        self = cls.__new__(cls)
        self._bind(q, d)
        return self

    def _bind(self, q: torch.Tensor, d: torch.Tensor) -> None:
        _index(q, "q", torch.uint8, None, 5)
        _index(d, "d", torch.float16, q.device, 5)
        n, two, heads, page, half = q.shape
        _need(two == 2 and d.shape == (n, 2, heads, half // 16, page) and half % 16 == 0, "q and d do not belong to one layout")
        self.q, self.d = q, d
        self.n_pages, self.page_size, self.kv_heads, self.head_dim = n, page, heads, 2 * half
        self._c = _Cache(q.data_ptr(), d.data_ptr(), n, page, heads, 2 * half)
        L, qb, db = _load(), C.c_size_t(), C.c_size_t()
        if L.jepa_b200_kv4_bytes(C.byref(self._c), C.byref(qb), C.byref(db)) != 0:
            _raise(L, "jepa_b200_kv4_bytes")
        _need(qb.value == q.numel() and db.value == 2 * d.numel(), "q and d do not belong to one layout")
        self._ref = C.byref(self._c)
        self._dev = q.device

    def _rows(self, t: torch.Tensor, name: str, n: int, heads: int) -> Tuple[int, ...]:
        """t is [n, heads, head_dim] on this device with contiguous channels; its strides."""
        if not (isinstance(t, torch.Tensor) and t.shape == (n, heads, self.head_dim)):
            raise ValueError(f"{name} must be [{n} rows, {heads}, {self.head_dim}]")
        if t.device != self._dev:
            raise ValueError(f"{name} must be on {self._dev}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires grad, and the 4-bit cache has no backward pass: detach it, or call under torch.no_grad()")
        stride = t.stride()
        if stride[2] != 1:
            raise ValueError(f"{name}'s channels must be contiguous")
        return stride

    def store(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantise rows k, v [n, kv_heads, head_dim] (f32, f16 or bf16, any strides of rows and heads) into slots [n]
        (int64; negative ones are skipped, the others must differ)."""
        _index(slots, "slots", torch.int64, self._dev)
        n = slots.shape[0]
        ks = self._rows(k, "k", n, self.kv_heads)
        vs = self._rows(v, "v", n, self.kv_heads)
        kind = _TYPE.get(k.dtype)
        if kind is None or v.dtype is not k.dtype:
            raise ValueError("k and v must be both f32, f16 or bf16")
        _call("jepa_b200_kv4_store", self._dev, self._ref, k.data_ptr(), v.data_ptr(), kind, ks[0], ks[1], vs[0], vs[1],
              slots.data_ptr(), n)

    def load(self, slots: torch.Tensor, dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
        """The values cached in slots [n] (int64): k, v [n, kv_heads, head_dim]; zeros for a slot outside the pool."""
        _index(slots, "slots", torch.int64, self._dev)
        if dtype not in _TYPE:
            raise ValueError(f"{dtype} is not f32, f16 or bf16")
        n = slots.shape[0]
        k = self.d.new_empty((n, self.kv_heads, self.head_dim), dtype=dtype)
        v = torch.empty_like(k)
        _call("jepa_b200_kv4_load", self._dev, self._ref, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), _TYPE[dtype])
        return k, v

    def attention(self, q: torch.Tensor, q_start: torch.Tensor, lens: torch.Tensor, table: torch.Tensor,
                  scale: Optional[float] = None, frame: int = 0, max_len: int = 0, max_new: int = 0,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of the rows q [rows, heads, head_dim] (f16 or bf16) over the cached rows of their requests:
        request r owns rows q_start[r] .. q_start[r + 1] - 1 and the first lens[r] positions of table[r]. frame: 0 =
        every cached key, 1 = causal, F = block-causal over frames of F tokens. max_len / max_new: bounds of lens and of
        a request's rows, which the launch is laid out for (they change no result beyond its rounding). out (zeros by
        default) keeps the rows of no request; it must not overlap q."""
        _need(isinstance(q, torch.Tensor) and q.dim() == 3, "q must be [rows, heads, head_dim]")
        rows, heads, _ = q.shape
        qs = self._rows(q, "q", rows, heads)
        if q.dtype is not torch.float16 and q.dtype is not torch.bfloat16:
            raise ValueError("q must be f16 or bf16")
        _index(lens, "lens", torch.int32, self._dev)
        _index(q_start, "q_start", torch.int32, self._dev)
        _index(table, "table", torch.int32, self._dev, 2)
        n, width = table.shape
        if q_start.shape[0] != n + 1 or lens.shape[0] != n:
            raise ValueError("lens, q_start and table must agree on the requests")
        if max(rows, n, width, frame, max_len, max_new) >= 2 ** 31:
            raise ValueError("no count may pass 2^31 - 1")
        if out is None:
            out = torch.zeros((rows, heads, self.head_dim), dtype=q.dtype, device=self._dev)
        elif out.dtype is not q.dtype:
            raise ValueError("out must be of q's type")
        os = self._rows(out, "out", rows, heads)
        a = _Attn(q.data_ptr(), out.data_ptr(), qs[0], qs[1], os[0], os[1], q_start.data_ptr(), lens.data_ptr(),
                  table.data_ptr(), n, rows, width, heads, _TYPE[q.dtype], frame,
                  1.0 / math.sqrt(self.head_dim) if scale is None else scale, max_len, max_new, None, 0)
        ref = C.byref(a)
        L = _lib or _load()
        need = L.jepa_b200_kv4_attention_workspace(self._ref, ref)
        if need < 0:
            _raise(L, "jepa_b200_kv4_attention")
        if need:
            # from the caching allocator, on the stream of the call: two calls, or two graphs, never share it
            ws = torch.empty(need, dtype=torch.uint8, device=self._dev)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        _call("jepa_b200_kv4_attention", self._dev, self._ref, ref)
        return out

    def check(self) -> None:
        """Waits for the current stream; raises if an attention kernel of this device, on any stream, has given up a wait
        that no check has told yet (the rows that it had not finished are NaN). Check in one place, behind all streams."""
        _call("jepa_b200_kv4_check", self._dev)
