"""How an attention call over the 4-bit cache is laid out (jepa_b200_kv4_attention_plan), without a GPU: over the whole range of
counts that a call may have, the key ranges cover the longest context, the grid exists and the workspace fits them."""
import ctypes as C
import random

import pytest

from jepa_b200 import kv4
from test_kv4 import _attn, _cache, _err

LAST = 2 ** 31 - 1 - 1024        # positions that a table row may have


def plan(page=16, kv_heads=2, head_dim=64, **kw):
    L = kv4._load()
    c = _cache(page_size=page, kv_heads=kv_heads, head_dim=head_dim)
    a = _attn(o_tok=kw["n_heads"] * head_dim, o_head=head_dim, **kw)
    out = (C.c_int * 4)()
    assert L.jepa_b200_kv4_attention_plan(C.byref(c), C.byref(a), out) == 0, _err()
    ws = L.jepa_b200_kv4_attention_workspace(C.byref(c), C.byref(a))
    cap = a.width * page
    longest = cap if a.max_len < 1 or a.max_len > cap else a.max_len
    tc, tiles, n_split, chunk = out
    assert n_split >= 1 and chunk >= 128 and chunk % 128 == 0
    assert (n_split - 1) * chunk < longest <= n_split * chunk
    assert tc in (0, 1) and 1 <= tiles and tiles * kv_heads <= 65535
    assert ws == (0 if n_split == 1 else n_split * a.n_rows * a.n_heads * (head_dim + 2) * 4)
    return tuple(out)


@pytest.mark.parametrize("n_req,n_rows,width", [(1024, 262144, 131072 // 16), (512, 131072, 262144 // 16), (65535, 1 << 24, LAST // 16),
                                                (65535, 1, LAST // 16), (1, 1 << 24, LAST // 16), (1, 1, LAST // 16), (2000, 4, LAST // 16)])
@pytest.mark.parametrize("max_new", [0, 1])
def test_counts_at_the_ends_of_their_ranges(n_req, n_rows, width, max_new):
    for heads, kv_heads in ((32, 8), (1, 1), (64, 1), (64, 64)):
        plan(kv_heads=kv_heads, n_heads=heads, n_req=n_req, n_rows=n_rows, width=width, max_new=max_new)


def test_any_counts():
    rng = random.Random(1)
    size = lambda top: int(2 ** rng.uniform(0, top))
    for _ in range(4000):
        kv_heads = min(1024, size(10.1))
        heads = kv_heads * min(65535 // kv_heads, size(7))
        page = 16 << rng.randrange(5)
        n_rows = min((1 << 30) // heads, size(30))
        plan(page=page, kv_heads=kv_heads, head_dim=32 * rng.randint(1, 4), n_heads=heads, n_req=min(65535, size(16)), n_rows=n_rows,
             width=min(LAST // page, size(31)), max_len=rng.choice([0, size(31) - 1]), max_new=rng.choice([0, size(30) - 1]))


def test_rules():
    many, few = 1, 0
    one = dict(kv_heads=8, head_dim=128, n_heads=32, page=64)
    # 64 sessions, one row each, up to 8190 keys: 4 columns a cache head, ranges of about four to a CTA's place
    assert plan(n_req=64, n_rows=64, width=128, max_len=8190, max_new=1, **one) == (few, 1, 5, 1792)
    # one session of 131,071 keys: ranges of 1024 at least (8 x 131,071 keys are 1771 for each of 592 CTAs)
    assert plan(n_req=1, n_rows=1, width=2048, max_len=131071, max_new=1, **one) == (few, 1, 128, 1024)
    # a short context is one range
    assert plan(n_req=1, n_rows=1, width=33, max_len=516, max_new=1, page=16, kv_heads=16, head_dim=64, n_heads=16) == (few, 1, 1, 640)
    # 33 columns are the first that take the tiles kernel
    assert plan(n_req=4, n_rows=132, width=64, max_len=1000, max_new=8, **one)[0] == few
    assert plan(n_req=4, n_rows=132, width=64, max_len=1000, max_new=9, **one)[0] == many
    # rows a request not known: all requests together have n_rows, so the ranges are those of a little more than that
    # (16 x 8 x 64,000 keys over 4 x 148 places are 13,838 a range; with 2 more CTAs' worth of columns 15,568)
    known = plan(n_req=16, n_rows=16 * 9, width=1024, max_len=64000, max_new=9, **one)
    unknown = plan(n_req=16, n_rows=16 * 9, width=1024, max_len=64000, **one)
    assert known == (many, 1, 5, 13952) and unknown == (many, 3, 5, 15616)


def test_refused_plans():
    L, c, out = kv4._load(), _cache(), (C.c_int * 4)()
    assert L.jepa_b200_kv4_attention_plan(C.byref(c), C.byref(_attn(n_req=0)), out) == -1 and "requests and rows" in _err()
    assert L.jepa_b200_kv4_attention_plan(C.byref(c), C.byref(_attn()), None) == -1 and "result's pointer" in _err()
    assert L.jepa_b200_kv4_attention_plan(C.byref(c), C.byref(_attn(frame=-1)), out) == -1 and "frame" in _err()
    assert L.jepa_b200_kv4_attention_plan(None, C.byref(_attn()), out) == -1 and "cache is null" in _err()


def test_out_overlaps():
    """Refused exactly where two (row, head) pieces of out share an element."""
    L, out = kv4._load(), (C.c_int * 4)()
    c = _cache(kv_heads=1, head_dim=32)
    rng = random.Random(5)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        rows, heads = rng.randint(1, 6), rng.randint(1, 6)
        tok, head = rng.randint(30, 300), rng.randint(30, 300)
        if rng.random() < 0.4:
            tok, head = rng.randint(1, 8) * 32, rng.randint(1, 8) * 32
        at = sorted(r * tok + h * head for r in range(rows) for h in range(heads))
        overlap = any(b - a < 32 for a, b in zip(at, at[1:]))
        rc = L.jepa_b200_kv4_attention_plan(C.byref(c), C.byref(_attn(n_rows=rows, n_heads=heads, o_tok=tok, o_head=head)), out)
        assert rc == (-1 if overlap else 0), (rows, heads, tok, head)
        assert not overlap or "overlap" in _err()
        seen[overlap] += 1
    assert min(seen.values()) > 500
    # the far ends: strides and counts whose products pass 63 bits
    big = 1 << 62
    for kw, rc in ((dict(n_rows=1 << 14, n_heads=65535, o_tok=big, o_head=big), -1), (dict(n_rows=1 << 14, n_heads=65535, o_tok=big, o_head=32), 0),
                   (dict(n_rows=1 << 14, n_heads=65535, o_tok=65535 * 32, o_head=32), 0), (dict(n_rows=1 << 14, n_heads=65535, o_tok=65535 * 32 - 1, o_head=32), -1),
                   (dict(n_rows=1 << 14, n_heads=65535, o_tok=32, o_head=32 << 14), 0), (dict(n_rows=1 << 14, n_heads=65535, o_tok=33, o_head=32 << 14), -1)):
        assert L.jepa_b200_kv4_attention_plan(C.byref(c), C.byref(_attn(**kw)), out) == rc, kw
        L.jepa_error_reset()
