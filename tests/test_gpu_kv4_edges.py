"""The 4-bit cache's attention where tiles, masks and what lies in the cache meet: long frames with pages that are not
there and scales that are not numbers, in every kernel and split."""
import math

import pytest
import torch

from jepa_b200 import kv4
from test_gpu_kv4 import attention_case, bound, check, i32, ref_attention

pytestmark = pytest.mark.gpu

NAN = float("nan")


def masked_case(lens, new, heads, kv_heads, dim, page, dtype, frame, seed, gone=(), broken=(), broken_keys=()):
    """Like attention_case, with the pages of the (request, page index) pairs `gone` taken out of the table, and the value
    scale of group 0 of the (request, key) pairs `broken`, the key scale of the last group of `broken_keys`, not a number. ref
    holds NaN where a row sees such a key: in the first 32 channels, or in all of them."""
    c, q, start, ln, table, _, _ = attention_case(lens, new, heads, kv_heads, dim, page, dtype, frame, seed)
    t = table.cpu().tolist()
    T = sum(new)
    ref, tol = torch.zeros(T, heads, dim, dtype=torch.float64), torch.zeros(T, heads, dim, dtype=torch.float64)
    at, group, scale = 0, heads // kv_heads, 1 / math.sqrt(dim)
    for r, (L, n) in enumerate(zip(lens, new)):
        slots = torch.tensor([t[r][j // page] * page + j % page for j in range(L)], dtype=torch.int64)
        k, v = (x.double().cpu() for x in c.load(slots.cuda(), torch.float32))
        held = torch.tensor([(r, j // page) not in gone for j in range(L)], dtype=torch.bool)
        bad, bad_key = (torch.tensor([(r, j) in where for j in range(L)], dtype=torch.bool) for where in (broken, broken_keys))
        pos = torch.arange(L - n, L)
        lim = torch.full_like(pos, L)
        if frame:
            lim = torch.where(pos < 0, 0, (torch.div(pos, frame, rounding_mode="floor") + 1) * frame).clamp(max=L)
        see = (torch.arange(L) < lim.unsqueeze(1)) & held
        for h in range(heads if n else 0):
            kk, vv, qq = k[:, h // group], v[:, h // group], q[at:at + n, h].double().cpu()
            s = (qq @ kk.T * scale).masked_fill(~see, -math.inf)
            m = s.amax(1, keepdim=True)
            p = torch.where(see, torch.exp(s - torch.where(m == -math.inf, 0.0, m)), 0.0)
            z = p.sum(1, keepdim=True)
            p = p / torch.where(z == 0, 1.0, z)
            size = (qq.abs() @ kk.abs().T * scale).masked_fill(~see, 0.0).amax(1, keepdim=True)
            mean = p @ vv.abs() + 2.0 ** -20 * (see.double() @ vv.abs())
            o = p @ vv
            tol[at:at + n, h] = bound(o, mean, size, dtype)
            o[(see & bad).any(1), :32] = NAN
            o[(see & bad_key).any(1)] = NAN
            ref[at:at + n, h] = o
        at += n
    for r, i in gone:
        table[r, i] = -3 if (r + i) % 2 else c.n_pages + i
    for r, j in broken:
        c.d[t[r][j // page], 1, :, 0, j % page] = NAN
    for r, j in broken_keys:
        c.d[t[r][j // page], 0, :, -1, j % page] = NAN
    return c, q, start, ln, table, ref, tol


def check_nan(out, ref, tol, what=""):
    got = out[:ref.shape[0]].double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), f"{what} NaN in {(got.isnan() != ref.isnan()).sum()} wrong places"
    ok = ~ref.isnan()
    err = (got - ref).abs()[ok]
    assert (err <= tol[ok]).all(), f"{what} {(err / tol[ok].clamp(min=1e-30)).max().item():.3g} of the bound"


@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16), (32, torch.bfloat16), (96, torch.float16)])
@pytest.mark.parametrize("frame,before", [(512, 1), (576, 1), (576, 2), (1024, 1), (1568, 1)])
def test_frames_longer_than_a_tile_with_missing_pages_and_broken_scales(frame, before, dim, dtype):
    """The second tile of 128 columns sees a whole frame more than the first, 8 to 25 blocks of 64 keys. Pages are missing
    at the end of the frame before and along the later one, and a value scale of the later frame is not a number: the
    masks of both tiles must stay apart."""
    n, page = frame + 128, 32
    L = frame * (before + 1)                       # rows 0 .. 127 lie in the frame before, the others in the last
    ends = frame * before // page
    gone = {(0, ends - 1), (0, ends - 3)} | {(0, i) for i in range(ends + 5, L // page, 3)}
    broken = {(0, frame * before + 6 * 64 + 40)}
    if any((0, j // page) in gone for _, j in broken):
        gone -= {(0, j // page) for _, j in broken}
    c, q, start, ln, table, ref, tol = masked_case([L], [n], 2, 2, dim, page, dtype, frame, frame + dim, gone, broken)
    assert ref[128:, :, :32].isnan().all() and not ref[:128].isnan().any()
    # (up to 768 keys are one range: told so of a longer context, a CTA walks all of its blocks)
    for max_len in (640, 640, 640, L):
        check_nan(c.attention(q, start, ln, table, frame=frame, max_len=max_len, max_new=n), ref, tol, f"max_len {max_len}")
    check_nan(c.attention(q, start, ln, table, frame=frame), ref, tol, "no bounds")
    c.check()


@pytest.mark.parametrize("n", [1, 40])
def test_row_ranges_outside_of_q_are_cut(n):
    """Whatever q_start holds, a request has rows of q or none: ranges that end before they start are empty, also where
    their difference passes 32 bits, and the others are cut to q."""
    c, q, start, ln, table, ref, tol = attention_case([300, 200], [n, n], 4, 2, 64, 32, torch.float16, 0, 5, tail=0)
    low, high = -2 ** 31, 2 ** 31 - 1
    for s in ([low, low, low], [n, low, n], [high, low, high], [high, high, high], [2 * n, low, high], [high, -1, low], [n, 0, low],
              [low, n, low], [n, n, high], [-5, n, high]):
        owner = torch.full((2 * n,), -1)
        for r in range(2):
            owner[min(max(0, s[r]), 2 * n):max(0, min(s[r + 1], 2 * n))] = r
        own = owner == torch.arange(2 * n) // n                 # the rows that ref gives to their request
        for bounds in (dict(max_len=300, max_new=n), {}):
            out = torch.full_like(q, 7.0)
            c.attention(q, i32(s), ln, table, out=out, **bounds)
            got = out.double().cpu()
            assert (got[owner < 0] == 7.0).all() and (got[owner >= 0] != 7.0).any(-1).all(), s
            assert ((got - ref).abs() <= tol)[own].all(), s


@pytest.mark.parametrize("n", [1, 5, 40, 300])
@pytest.mark.parametrize("frame", [0, 1, 48])
def test_lengths_past_the_table_are_cut_to_it(n, frame):
    """lens is taken as at most width * page_size, for what is cached and for where the rows stand; below 0 it is 0."""
    L, page = 208, 16                                   # 13 pages, each of them full: the table ends with the last key
    c, q, start, ln, table, ref, tol = attention_case([L], [n], 4, 2, 64, page, torch.bfloat16, frame, 23, tail=1)
    table = table[:, :L // page].contiguous()
    for bounds in (dict(max_len=L, max_new=n), {}):
        full = c.attention(q, start, ln, table, frame=frame, **bounds)
        err = (full[:n].double().cpu() - ref).abs()
        assert not full.isnan().any() and (err <= tol).all()
        for length in (L + 1, 5 * L, 2 ** 31 - 1):
            assert torch.equal(c.attention(q, start, i32([length]), table, frame=frame, **bounds), full), length
        for length in (0, -1, -2 ** 31):
            assert (c.attention(q, start, i32([length]), table, frame=frame, **bounds) == 0).all(), length


def test_many_requests_over_wide_tables_with_unknown_bounds():
    """1024 requests of 64 rows whose tables could hold 4 million positions each, and no bounds: the launch is laid out for
    what it is told, and the results are those of a call that knows better."""
    R, n, dim, page, width = 1024, 64, 32, 256, 16384
    g = torch.Generator("cuda").manual_seed(3)
    c = kv4.KV4Cache(4, page, 1, dim)
    x = torch.randn(2, 1024, 1, dim, generator=g, device="cuda")
    c.store(x[0], x[1], torch.arange(1024, device="cuda"))
    table = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    table[:, 0], table[:, 1] = torch.arange(R, device="cuda") % 4, torch.arange(R, device="cuda") // 4 % 4
    lens = (torch.arange(R, device="cuda", dtype=torch.int32) * 37) % 513
    start = torch.arange(R + 1, device="cuda", dtype=torch.int32) * n
    q = torch.randn(R * n, 1, dim, generator=g, device="cuda").half()
    a = c.attention(q, start, lens, table, frame=1)
    b = c.attention(q, start, lens, table, frame=1, max_len=512, max_new=n)
    k, v = (t[:, 0].double().cpu() for t in c.load(torch.arange(1024, device="cuda"), torch.float32))
    for r in (0, 1, 5, 500, 1023):
        L = int(lens[r])
        at = torch.tensor([int(table[r, j // page]) * page + j % page for j in range(L)], dtype=torch.int64)
        o, mean, size = ref_attention(q[r * n:(r + 1) * n, 0].double().cpu(), k[at], v[at], torch.arange(L - n, L), 1, dim ** -0.5)
        for out in (a, b):
            check(out[r * n:(r + 1) * n, 0], o, bound(o, mean, size, torch.float16), f"request {r}")
    half = torch.finfo(torch.float16).eps / 2
    assert ((a - b).abs().double() <= 2 * half * b.abs().double() + 2 * 2.0 ** -11 * float(v.abs().max())).all()


def test_rows_that_require_grad_are_refused():
    c = kv4.KV4Cache(4, 16, 2, 64)
    x = torch.randn(3, 2, 64, device="cuda").half().requires_grad_()
    slots, start, ln, table = torch.arange(3, device="cuda"), i32([0, 3]), i32([3]), i32([[0]])
    for call in (lambda a: c.store(a, a.detach(), slots), lambda a: c.store(a.detach(), a, slots), lambda a: c.attention(a, start, ln, table),
                 lambda a: c.attention(a.detach(), start, ln, table, out=a * 1)):
        with pytest.raises(ValueError, match="requires grad"):
            call(x)
        with torch.no_grad():
            call(x)


@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16), (32, torch.float16), (96, torch.bfloat16)])
@pytest.mark.parametrize("lens,new,heads,kv_heads", [
    ([70], [9], 1, 1), ([70, 90], [1, 16], 1, 1),                # one tile of 8 columns, two
    ([300], [30], 2, 2), ([300, 90], [4, 1], 14, 2),             # two passes over the columns; grouped heads
    ([400], [258], 1, 1), ([500, 80], [259, 3], 2, 2),           # whole tiles of 256 and 2 or 3 columns left over
    ([2600], [6], 2, 1), ([2600], [70], 2, 1),                   # several ranges of keys, joined at the end: few rows, many
    ([330], [40], 3, 1)])
def test_scales_that_are_not_numbers_reach_the_rows_that_see_them_and_no_other(lens, new, heads, kv_heads, dim, dtype):
    """A value scale, a key scale and a page that is not there, each among the keys that the rows of a causal chunk begin
    to see one after the other: NaN in the channels that they give, from the first row that sees them on, in both kernels."""
    page = 16
    broken = {(r, L - n + n // 2) for r, (L, n) in enumerate(zip(lens, new))}
    keys = {(r, L - 1 - n // 4) for r, (L, n) in enumerate(zip(lens, new)) if n > 4}
    gone = {(r, 1) for r in range(len(lens))}
    for frame in (1, 0):
        c, q, start, ln, table, ref, tol = masked_case(lens, new, heads, kv_heads, dim, page, dtype, frame, sum(lens) + dim, gone, broken, keys)
        assert ref.isnan().any() and (frame == 0 or max(new) < 5 or not ref.isnan().all(-1).all())
        for bounds in (dict(max_len=max(lens), max_new=max(new)), {}, dict(max_len=1, max_new=1)):
            check_nan(c.attention(q, start, ln, table, frame=frame, **bounds), ref, tol, str(bounds))
    # behind every row's mask: in the last page, past the last key
    c, q, start, ln, table, ref, tol = masked_case(lens, new, heads, kv_heads, dim, page, dtype, 1, sum(lens) + dim)
    assert not ref.isnan().any()
    check_nan(c.attention(q, start, ln, table, frame=1, max_new=max(new)), ref, tol)


@pytest.mark.parametrize("dtype,big", [(torch.bfloat16, 2.0 ** 40), (torch.bfloat16, 2.0 ** 90), (torch.bfloat16, 2.0 ** 118), (torch.float16, 2.0 ** 12),
                                       (torch.bfloat16, 2.0 ** 14)])
@pytest.mark.parametrize("n,lens", [(1, [700, 90]), (9, [2500, 64]), (40, [700, 90]), (300, [1500, 400])])
def test_a_huge_query_takes_the_value_of_its_key(n, lens, dtype, big):
    """Row i is the cached key t_i times 2^12 .. 2^118: the score of t_i is above every other by 2^8 and more, its weight is all
    there is, and the row is its value: off by the value's rounding to the type and, where weights go into the product
    rounded to f16 and into the sum as they are, by 2^-11 of it."""
    heads, kv_heads, dim, page = 2, 1, 64, 32
    c, _, start, ln, table, _, _ = attention_case(lens, [n, n], heads, kv_heads, dim, page, dtype, 1, 77)
    t = table.cpu().tolist()
    q, want = torch.zeros(2 * n, heads, dim, dtype=torch.float64), torch.zeros(2 * n, heads, dim, dtype=torch.float64)
    for r, L in enumerate(lens):
        slots = torch.tensor([t[r][j // page] * page + j % page for j in range(L)], device="cuda")
        k, v = (x[:, 0].double().cpu() for x in c.load(slots, torch.float32))
        dots = k @ k.T
        margin = dots.diag() - (dots - torch.diag(dots.diag() * 2)).amax(1)
        for i in range(n):
            seen = L - n + i + 1                                  # causal: keys that the row sees
            for h in range(heads):
                j = int(margin[:seen].sub(1e-3 * ((torch.arange(seen) * 37 + 11 * i + h) % 97)).argmax()) if i % 3 else seen - 1
                if margin[j] <= 4:
                    j = int(margin[:seen].argmax())
                assert margin[j] > 4                              # x 2^12 / sqrt(64): 2^11 apart
                q[r * n + i, h], want[r * n + i, h] = (k[j] * big).to(dtype).double(), v[j]
    assert torch.isfinite(q).all()
    half = torch.finfo(dtype).eps / 2
    for bounds in (dict(max_len=max(lens), max_new=n), {}):
        out = c.attention(q.to(dtype).cuda(), start, ln, table, frame=1, **bounds).double().cpu()
        assert ((out - want).abs() <= (half + 2.0 ** -11) * want.abs() + 1e-30).all()


_FIRST_CALLS = r"""
import sys
sys.path.insert(0, sys.argv[1])
import torch
from jepa_b200 import kv4
dev, page, dim, n = "cuda", 32, 64, [1, 3, 300]
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
c = kv4.KV4Cache(120, page, 2, dim)
cached, added, table, free = i32([0, 40, 1500]), i32(n), torch.arange(3 * 64, dtype=torch.int32, device=dev).view(3, 64) % 56, i32(list(range(56, 120)))
start_table = table.clone()
g = torch.Generator(dev).manual_seed(1)
k, v = (torch.randn(sum(n), 2, dim, generator=g, device=dev).half() for _ in range(2))
q = torch.randn(sum(n), 4, dim, generator=g, device=dev).half()

def step():
    t = kv4.build_tables(cached, added, table, free, page, sum(n))
    c.store(k, v, t.slots)
    return (c.attention(q, t.q_start, t.lens, table, frame=1, max_len=1800, max_new=300), *c.load(t.slots), t.slots, t.state)

side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    got = step()
graph.replay()
torch.cuda.synchronize()
got = [x.clone() for x in got]
table.copy_(start_table)
want = step()
c.check()
assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[4].tolist()[0] == 0 and bool((got[0] != 0).any())
print("SAME")
"""


def test_the_first_calls_of_a_process_can_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jepa.cpp_b200")
    r = subprocess.run([sys.executable, "-c", _FIRST_CALLS, root], capture_output=True, text=True, timeout=180)
    assert r.returncode == 0 and "SAME" in r.stdout, r.stderr[-2000:]
