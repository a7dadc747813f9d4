"""The paged 4-bit key / value cache on the GPU against plain 64-bit definitions: tables and slots exactly, stored and
loaded values exactly, attention within the roundings that its types and its sums make."""
import math
import random

import pytest
import torch

from jepa_b200 import kv4

pytestmark = pytest.mark.gpu

NAN = float("nan")


# ---------------------------------------------------------------------------------- definitions, float64 on the CPU

def ref_values(x):
    """x [..., hd] -> the cached values d (c - 8), group by group of 32 channels."""
    g = x.double().unflatten(-1, (x.shape[-1] // 32, 32))
    hi, lo = g.amax(-1, keepdim=True), g.amin(-1, keepdim=True)
    m = torch.where(hi >= -lo, hi, lo)
    d = (m / -8).float().to(torch.bfloat16).float().clamp(-8160, 8160).to(torch.float16).double()
    q = torch.floor(g / torch.where(d == 0, 1.0, d) + 0.5).clamp(-8, 7)
    v = torch.where(d == 0, 0.0, q * d)
    bad = ~torch.isfinite(g).all(-1, keepdim=True)
    return torch.where(bad, NAN, v).reshape(x.shape)


def ref_attention(q, k, v, pos, frame, scale):
    """One request and query head: q [n, hd], k, v [L, hd] float64, pos [n] -> out, and the bound's two parts: the mean
    of |v| under the weights, and the largest sum of |scale q_c k_c|."""
    L = k.shape[0]
    lim = torch.full_like(pos, L)
    if frame:
        lim = torch.where(pos < 0, 0, (torch.div(pos, frame, rounding_mode="floor") + 1) * frame).clamp(max=L)
    see = torch.arange(L) < lim.unsqueeze(1)
    s = (q @ k.T * scale).masked_fill(~see, -math.inf)
    m = s.amax(1, keepdim=True) if L else torch.full((q.shape[0], 1), -math.inf, dtype=torch.float64)
    p = torch.where(see, torch.exp(s - torch.where(m == -math.inf, 0.0, m)), 0.0)
    z = p.sum(1, keepdim=True)
    p = p / torch.where(z == 0, 1.0, z)
    size = (q.abs() @ k.abs().T * abs(scale)).masked_fill(~see, 0.0)
    # the mean of |v|, with the weights' step at the small end of f16 added (see bound): 2^-31 of |v| for every key seen
    mean = p @ v.abs() + 2.0 ** -20 * (see.double() @ v.abs())
    return p @ v, mean, size.amax(1, keepdim=True) if L else torch.zeros(q.shape[0], 1, dtype=torch.float64)


def bound(ref, mean_abs, size, dtype):
    # the output's rounding, half a step of its type; the weights' rounding to f16, half a step of each: 2^-11 of a
    # normal one, 2^-25 of a subnormal one, where the weights are scaled so that the largest is at least 2^6 (many rows;
    # 2^10 few rows) -- so at most 2^-11 w + 2^-31 w_max, and w_max / sum(w) <= 1: mean_abs carries the second part
    # as 2^-11 * 2^-20;
    # the scores' f32 sums of up to 128 products and the exponent's product: |error| <= 2^-18 of the sum of magnitudes,
    # which moves a weight by that much of itself, numerator and denominator both
    half = torch.finfo(dtype).eps / 2
    return half * ref.abs() + (2.0 ** -11 + 2 * 2.0 ** -18 * size) * mean_abs + torch.finfo(dtype).smallest_normal * half


# ---------------------------------------------------------------------------------- tables

def ref_tables(cached, added, table, free, page, n_slots):
    table = [row[:] for row in table]
    slots, start, taken = [], [0], 0
    for r, (c, n) in enumerate(zip(cached, added)):
        for i in range(-(-c // page), -(-(c + n) // page)):
            table[r][i] = free[taken]
            taken += 1
        slots += [table[r][p // page] * page + p % page for p in range(c, c + n)]
        start.append(start[-1] + n)
    return [c + n for c, n in zip(cached, added)], start, slots + [-1] * (n_slots - len(slots)), [0, taken], table


def make_tables(cached, added, page, spare, seed, width=None):
    rng = random.Random(seed)
    held = [-(-c // page) for c in cached]
    need = [-(-(c + n) // page) - h for c, n, h in zip(cached, added, held)]
    width = width or max(1, max(h + n for h, n in zip(held, need))) + 1
    pages = list(range(sum(held) + sum(need) + spare))
    rng.shuffle(pages)
    table = []
    for h in held:
        table.append([pages.pop() for _ in range(h)] + [-1 - rng.randrange(9) for _ in range(width - h)])
    return table, pages


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("n,page,cached,added,pad", [
    (1, 16, (0, 0), (1, 1), 0), (1, 16, (0, 0), (0, 0), 3), (1, 256, (516, 516), (258, 258), 0), (8, 16, (200, 800), (1, 1), 0),
    (127, 32, (0, 90), (0, 40), 5), (128, 64, (0, 0), (0, 300), 1), (129, 16, (15, 17), (0, 2), 0), (513, 16, (0, 70), (0, 9), 77),
    (1500, 64, (0, 4000), (0, 258), 1000), (5, 16, (0, 3), (0, 30000), 9)])
def test_tables(n, page, cached, added, pad):
    rng = random.Random(n + page)
    c, a = [rng.randint(*cached) for _ in range(n)], [rng.randint(*added) for _ in range(n)]
    table, free = make_tables(c, a, page, 3, n)
    n_slots = max(1, sum(a) + pad)
    lens, start, slots, state, want = ref_tables(c, a, table, free, page, n_slots)
    tab = i32(table)
    for _ in range(2):                       # a second pass over the filled table says the same
        t = kv4.build_tables(i32(c), i32(a), tab, i32(free), page, n_slots)
        assert t.lens.tolist() == lens and t.q_start.tolist() == start and t.state.tolist() == state
        assert t.slots.tolist() == slots and tab.tolist() == want


@pytest.mark.parametrize("n", [3, 600])
@pytest.mark.parametrize("code", [1, 2, 3, 4])
def test_tables_refuse_the_step_as_a_whole(n, code):
    c, a, page = [20] * n, [30] * n, 16
    table, free = make_tables(c, a, page, 0, 1, width=4)
    n_slots = 30 * n
    if code == 1:
        c[n - 1] = -1
        a[0] = 60                            # outgrows its row as well: the smaller code is told
    if code == 2:
        a[n // 2] = 45
    if code == 3:
        free = free[:-1]
    if code == 4:
        n_slots -= 1
    tab = i32(table)
    t = kv4.build_tables(i32(c), i32(a), tab, i32(free), page, n_slots)
    assert t.state.tolist() == [code, 0] and t.lens.tolist() == c and t.q_start.tolist() == [0] * (n + 1)
    assert tab.tolist() == table and (t.slots == -1).all()


def test_tables_count_past_32_bits():
    n = 4096                                 # 4096 x (2^20 - 64) new rows: the sum passes 2^31, no slot map holds it
    c, a = [0] * n, [2 ** 20 - 64] * n
    tab = torch.full((n, 4096), -1, dtype=torch.int32, device="cuda")
    t = kv4.build_tables(i32(c), i32(a), tab, i32(list(range(64))), 256, 1000)
    assert t.state.tolist() == [3, 0]
    t = kv4.build_tables(i32([2 ** 31 - 1] * 2), i32([1, 0]), tab[:2], i32([0]), 256, 8)
    assert t.state.tolist() == [2, 0]


def test_tables_without_a_free_page():
    tab = i32([[4, -7], [2, 3]])
    t = kv4.build_tables(i32([3, 17]), i32([13, 0]), tab, i32([]), 16, 13)
    assert t.state.tolist() == [0, 0] and t.slots.tolist() == list(range(67, 80)) and tab.tolist() == [[4, -7], [2, 3]]
    t = kv4.build_tables(i32([3, 17]), i32([14, 0]), tab, i32([]), 16, 14)
    assert t.state.tolist() == [3, 0]


def test_tables_with_a_negative_page_give_no_slot():
    t = kv4.build_tables(i32([20]), i32([14]), i32([[5, -3, 0]]), i32([9]), 16, 14)
    assert t.slots.tolist() == [-1] * 12 + [144, 145]


# ---------------------------------------------------------------------------------- store and load

def rows(seed, n, heads, dim, dtype, kind="normal"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, dim, generator=g)
    if kind == "hard":
        x = x * torch.exp2(torch.randint(-28, 24, (n, heads, dim // 32, 1), generator=g).float()).expand(-1, -1, -1, 32).reshape(n, heads, dim)
        pick = torch.randint(0, 8, (n, heads, dim // 32, 1), generator=g).expand(-1, -1, -1, 32).reshape(n, heads, dim)
        x = torch.where(pick == 1, 0.0, x)
        x = torch.where(pick == 2, torch.round(x.clamp(-60, 60)) / 2, x)          # quotients on the half steps
        x = torch.where(pick == 3, torch.sign(x) * 1.5, x)                        # two values of the largest magnitude
        x = torch.where(pick == 4, x * 1e-7, x)
    return x.to(dtype)


def same(a, b):
    """Equal values, NaN where the other is NaN (a group that went to infinity in f16 reads back as NaN)."""
    a, b = a.double().cpu(), b.double().cpu()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()], b[~b.isnan()])


def pool(pages, page, heads, dim, fill=True):
    c = kv4.KV4Cache(pages, page, heads, dim)
    if fill:
        c.q.random_(0, 256)
        c.d.copy_(torch.randn(c.d.shape, device="cuda"))
    return c


TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("kind", ["normal", "hard"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,heads,dim,page", [(1, 1, 32, 16), (7, 3, 64, 16), (8, 2, 96, 32), (9, 5, 128, 64), (130, 1, 128, 256), (500, 16, 64, 128)])
def test_store_then_load_is_the_definition(n, heads, dim, page, dtype, kind):
    k, v = rows(n, n, heads, dim, dtype, kind), rows(n + 1, n, heads, dim, dtype, kind)
    pages = -(-n // page) + 3
    c = pool(pages, page, heads, dim)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(n))[:n]
    if n > 1:
        slots[n // 2] = -1
    if n > 8:
        slots[3], slots[5] = pages * page, 2 ** 40            # behind the pool: skipped as well
    every = torch.arange(pages * page)
    before = [x.double().cpu() for x in c.load(every.cuda(), torch.float32)]
    c.store(k.cuda(), v.cuda(), slots.cuda())
    after = c.load(every.cuda(), torch.float32)
    half = c.load(every.cuda(), torch.float16)
    bf = c.load(every.cuda(), torch.bfloat16)
    ok = (slots >= 0) & (slots < pages * page)
    for old, new, h, b, x in zip(before, after, half, bf, (k, v)):
        old[slots[ok]] = ref_values(x[ok])
        assert same(new, old)
        assert same(h[slots[ok].cuda()], old[slots[ok]])     # f16 holds every stored value
        assert same(b, old.to(torch.bfloat16))


def test_store_of_values_that_are_not_finite():
    x = rows(3, 4, 2, 64, torch.float32)
    x[0, 0, 5], x[1, 1, 40], x[2, 0, 33], x[3, 1, 0] = NAN, math.inf, -math.inf, 3e38
    c = pool(1, 16, 2, 64)
    s = torch.arange(4, device="cuda")
    c.store(x.cuda(), x.cuda(), s)
    want = ref_values(x)
    assert want.isnan().sum() == 3 * 32
    for got in c.load(s, torch.float32):
        assert same(got, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_store_takes_any_strides(dtype):
    n, heads, dim = 37, 3, 64
    c = pool(4, 16, heads, dim)
    slots = torch.arange(n, device="cuda")
    base = rows(5, n + 2, heads * 2 * dim + 3, 1, dtype).cuda()[..., 0]
    odd = base[1:n + 1, 1:1 + heads * dim].unflatten(1, (heads, dim))                      # rows start off alignment
    turned = rows(6, heads, n, dim, dtype).cuda().transpose(0, 1)                       # heads outside, rows inside
    shared = rows(7, n, 1, dim, dtype).cuda().expand(n, heads, dim)                     # one row for every head
    for k, v in ((odd, turned), (turned, shared), (shared, odd)):
        c.store(k, v, slots)
        got = c.load(slots, torch.float32)
        assert torch.equal(got[0].double().cpu(), ref_values(k.cpu())) and torch.equal(got[1].double().cpu(), ref_values(v.cpu()))


def test_load_of_slots_outside_and_twice():
    c = pool(2, 16, 2, 96)
    s = torch.tensor([3, -1, 3, 32, 31, -(2 ** 40), 0], device="cuda")
    all_k, all_v = c.load(torch.arange(32, device="cuda"))
    k, v = c.load(s)
    for got, full in ((k, all_k), (v, all_v)):
        want = torch.stack([full[i] if 0 <= i < 32 else torch.zeros_like(full[0]) for i in s.tolist()])
        assert torch.equal(got, want)
    assert c.load(s[:0])[0].shape == (0, 2, 96)


# ---------------------------------------------------------------------------------- attention

def attention_case(lens, new, heads, kv_heads, dim, page, dtype, frame, seed, gain=1.0, poison=True, tail=2, q=None):
    """Inputs on the GPU, and the reference's rows with their bounds."""
    R = len(lens)
    table, free = make_tables([max(0, x) for x in lens], [0] * R, page, 2, seed)
    pages = sum(-(-max(0, x) // page) for x in lens) + 2
    c = kv4.KV4Cache(pages, page, kv_heads, dim)
    if poison:
        c.q.fill_(255)
        c.d.fill_(NAN)
    keys, vals = [], []
    for r in range(R):
        k = rows(seed + 10 * r, lens[r], kv_heads, dim, dtype) * gain
        v = rows(seed + 10 * r + 1, lens[r], kv_heads, dim, dtype)
        slots = torch.tensor([table[r][j // page] * page + j % page for j in range(lens[r])], dtype=torch.int64)
        c.store(k.cuda(), v.cuda(), slots.cuda())
        keys.append(ref_values(k))
        vals.append(ref_values(v))
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    if q is None:
        q = rows(seed + 5, start[-1] + tail, heads, dim, dtype)
    ref = torch.zeros(start[-1], heads, dim, dtype=torch.float64)
    tol = torch.zeros_like(ref)
    scale = 1 / math.sqrt(dim)
    for r in range(R):
        if not new[r]:
            continue
        pos = torch.arange(lens[r] - new[r], lens[r])
        for h in range(heads):
            kh = h // (heads // kv_heads)
            o, mean, size = ref_attention(q[start[r]:start[r + 1], h].double(), keys[r][:, kh], vals[r][:, kh], pos, frame, scale)
            ref[start[r]:start[r + 1], h] = o
            tol[start[r]:start[r + 1], h] = bound(o, mean, size, dtype)
    return c, q.cuda(), i32(start), i32(lens), i32(table), ref, tol


def check(out, ref, tol, what=""):
    err = (out[:ref.shape[0]].double().cpu() - ref).abs()
    worst = (err / tol.clamp(min=1e-30)).max().item() if ref.numel() else 0.0
    assert not err.isnan().any() and (err <= tol).all(), f"{what} {worst:.3g} of the bound"


CASES = [
    # lens, new, heads, kv_heads, dim, page, frame
    ([1], [1], 1, 1, 32, 16, 0),
    ([516], [1], 16, 16, 64, 16, 0),
    ([0, 5, 1], [1, 1, 1], 4, 2, 96, 16, 1),
    ([17, 64, 65, 300, 0, 1023], [1, 1, 1, 1, 1, 1], 8, 1, 128, 64, 1),
    ([130, 40, 77], [1, 1, 1], 14, 2, 64, 32, 0),
    ([700, 3], [1, 1], 48, 3, 128, 128, 1),
    ([2500], [1], 8, 2, 128, 16, 1),
    ([33, 200, 9], [4, 7, 9], 8, 2, 64, 16, 1),
    ([33, 200, 5], [4, 0, 9], 6, 6, 96, 32, 1),
    ([258 * 3, 258], [258, 258], 4, 4, 64, 32, 258),
    ([600, 130], [70, 129], 8, 2, 128, 64, 1),
    ([100, 333], [40, 333], 3, 1, 32, 256, 0),
    ([300], [20], 32, 2, 96, 16, 16),
    ([50, 60], [64, 61], 4, 2, 64, 16, 1),       # more rows than keys: the first rows see nothing
    ([20], [150], 7, 1, 128, 16, 16),
    ([1000, 0, 129, 128, 127], [130, 3, 129, 1, 0], 8, 4, 64, 128, 1),
    ([90, 300], [1, 1], 512, 1, 64, 16, 1),      # more columns of one row than a tile holds
    ([70, 20, 200], [3, 1, 6], 86, 1, 128, 32, 1),   # 258, 86 and 516 columns: whole tiles and 2, 86 and 4 left over
    ([640, 64, 900], [1, 64, 2], 4, 1, 96, 64, 0),   # single rows beside a chunk
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,new,heads,kv_heads,dim,page,frame", CASES)
def test_attention(lens, new, heads, kv_heads, dim, page, frame, dtype):
    c, q, start, ln, table, ref, tol = attention_case(lens, new, heads, kv_heads, dim, page, dtype, frame, sum(lens) + dim)
    out = torch.full_like(q, 7.0)
    got = c.attention(q, start, ln, table, frame=frame, max_len=max(1, max(lens)), max_new=max(new), out=out)
    assert got is out
    check(out, ref, tol)
    assert (out[ref.shape[0]:] == 7.0).all()              # rows behind the last request's
    # the bounds shape the launch only: unknown, or too small, they change no row beyond its rounding
    check(c.attention(q, start, ln, table, frame=frame), ref, tol, "no bounds")
    check(c.attention(q, start, ln, table, frame=frame, max_len=1, max_new=1), ref, tol, "small bounds")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_attention_of_sharp_scores_and_of_extreme_queries(dtype, n):
    """Scores of +-1000 (one key takes all) and queries whose type's range f16 does not have."""
    lens, heads, dim = [700, 90], 4, 64
    c, q, start, ln, table, ref, tol = attention_case(lens, [n, n], heads, 2, dim, 32, dtype, 1, 11, gain=30.0)
    check(c.attention(q, start, ln, table, frame=1, max_new=n), ref, tol)
    big = 2.0 ** 40 if dtype is torch.bfloat16 else 2.0 ** 12
    for f in (1.0 / big, big, 0.0):
        qs = (q * f).to(dtype).cpu()
        c, q2, start, ln, table, ref, tol = attention_case(lens, [n, n], heads, 2, dim, 32, dtype, 1, 11, gain=1 / 64, q=qs)
        ok = tol < 0.5 * ref.abs().amax()
        out = c.attention(q2, start, ln, table, frame=1, max_new=n)
        err = (out[:ref.shape[0]].double().cpu() - ref).abs()
        assert not err.isnan().any() and ((err <= tol) | ~ok).all()


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_attention_scales(scale, n):
    """0: the mean of what a row sees; below 0: the smallest product counts most."""
    lens, heads, dim = [300, 41], 6, 96
    c, q, start, ln, table, _, _ = attention_case(lens, [n, n], heads, 2, dim, 16, torch.float16, 1, 31)
    out = c.attention(q, start, ln, table, scale=scale, frame=1, max_new=n)
    t = table.cpu().tolist()
    for r in range(2):
        slots = torch.tensor([t[r][j // 16] * 16 + j % 16 for j in range(lens[r])], device="cuda")
        k, v = (x.double().cpu() for x in c.load(slots, torch.float32))
        for h in range(heads):
            rows_ = slice(r * n, r * n + n)
            o, mean, size = ref_attention(q[rows_, h].double().cpu(), k[:, h // 3], v[:, h // 3], torch.arange(lens[r] - n, lens[r]), 1, scale)
            check(out[rows_, h], o, bound(o, mean, size, torch.float16))
    c.check()                                             # no bounded wait ran out


@pytest.mark.parametrize("size", [1e-6, 1.0, 3e4])
def test_attention_of_small_and_large_values(size):
    """Values near the ends of f16, f32 rows: the weights' range must not limit them."""
    lens, n, heads, dim = [900], 2, 8, 128
    g = torch.Generator().manual_seed(1)
    k = torch.randn(900, 2, dim, generator=g)
    v = torch.randn(900, 2, dim, generator=g).clamp(-2, 2) * size
    for n in (2, 64):
        q = rows(2, n, heads, dim, torch.bfloat16)
        c = kv4.KV4Cache(60, 16, 2, dim)
        c.store(k.cuda(), v.cuda(), torch.arange(900, device="cuda"))
        out = c.attention(q.cuda(), i32([0, n]), i32(lens), i32([list(range(57))]), max_new=n)
        kk, vv = ref_values(k), ref_values(v)
        for h in range(heads):
            o, mean, s = ref_attention(q[:, h].double(), kk[:, h // 4], vv[:, h // 4], torch.arange(900 - n, 900), 0, 1 / math.sqrt(dim))
            check(out[:, h], o, bound(o, mean, s, torch.bfloat16))


@pytest.mark.parametrize("n", [1, 5, 100])
def test_attention_strides(n):
    c, q, start, ln, table, ref, tol = attention_case([400, 70], [n, n], 6, 3, 64, 32, torch.float16, 1, 4)
    T = q.shape[0]
    wide = torch.full((T, 6 * 64 + 5), NAN, dtype=q.dtype, device="cuda")
    odd = wide[:, 3:3 + 6 * 64].unflatten(1, (6, 64))
    odd.copy_(q)
    turned = torch.empty(6, T, 64, dtype=q.dtype, device="cuda").transpose(0, 1)
    turned.copy_(q)
    for src in (odd, turned):
        for make in (lambda: torch.zeros_like(wide)[:, 1:1 + 6 * 64].unflatten(1, (6, 64)),
                     lambda: torch.zeros(6, T, 64, dtype=q.dtype, device="cuda").transpose(0, 1)):
            check(c.attention(src, start, ln, table, frame=1, max_new=n, out=make()), ref, tol)


@pytest.mark.parametrize("n", [1, 40])
def test_attention_leaves_out_pages_that_are_not_there(n):
    lens, page = [200], 16
    c, q, start, ln, table, _, _ = attention_case(lens, [n], 4, 2, 64, page, torch.float16, 0, 21)
    t = table.cpu()[0].tolist()
    held = [j for j in range(200) if j // page not in (2, 7)]
    slots = torch.tensor([t[j // page] * page + j % page for j in held], device="cuda")
    k, v = (x.double().cpu() for x in c.load(slots, torch.float32))
    bad = table.clone()
    bad[0, 2], bad[0, 7] = -5, c.n_pages
    out = c.attention(q, start, ln, bad, max_new=n)
    for h in range(4):
        o, mean, size = ref_attention(q[:n, h].double().cpu(), k[:, h // 2], v[:, h // 2], torch.arange(n), 0, 1 / 8)
        check(out[:n, h], o, bound(o, mean, size, torch.float16))
    # no page at all: nothing is seen; lengths past the table, and below zero, are cut to what there is
    gone = c.attention(q, start, ln, torch.full_like(table, 2 ** 31 - 1), max_new=n)
    assert (gone == 0).all()
    full = c.attention(q, start, i32([table.shape[1] * page]), bad, max_new=n)
    past = c.attention(q, start, i32([2 ** 31 - 1]), bad, max_new=n)
    assert torch.equal(full, past) or n > 1 or full.isnan().any()
    assert (c.attention(q, start, i32([-4]), table, max_new=n) == 0).all()


def test_nan_reaches_only_the_rows_that_see_it():
    lens, n = [64], 20
    c, q, start, ln, table, ref, tol = attention_case(lens, [n], 2, 1, 64, 16, torch.float16, 1, 3)
    page = table[0, 50 // 16].item()
    c.d[page, 1, 0, 0, 50 % 16] = NAN                     # the value of key 50, first 32 channels
    out = c.attention(q, start, ln, table, frame=1, max_new=n)[:n].double().cpu()
    first = 50 - (64 - n)                                # the row at position 50
    assert out[first:, :, :32].isnan().all() and not out[:first].isnan().any() and not out[:, :, 32:].isnan().any()
    assert ((out[:first] - ref[:first]).abs() <= tol[:first]).all()


def test_pages_shared_by_requests_and_offsets_past_32_bits():
    """Two requests read one prefix; the pool is larger than 4 GiB and its last pages are in use."""
    page, heads, dim, n = 256, 16, 128, 3
    pages = (5 << 30) // (2 * heads * page * dim // 2)
    c = kv4.KV4Cache.wrap(torch.empty(pages, 2, heads, page, dim // 2, dtype=torch.uint8, device="cuda"),
                          torch.empty(pages, 2, heads, dim // 32, page, dtype=torch.float16, device="cuda"))
    L = [300, 600]
    table = [[pages - 1, pages - 2, -1], [pages - 1, pages - 3, pages - 4]]
    k, v = rows(1, 600, heads, dim, torch.float16), rows(2, 600, heads, dim, torch.float16)
    k2, v2 = rows(3, 44, heads, dim, torch.float16), rows(4, 44, heads, dim, torch.float16)
    at = lambda r, j: table[r][j // page] * page + j % page
    c.store(k.cuda(), v.cuda(), torch.tensor([at(1, j) for j in range(600)], device="cuda"))
    c.store(k2.cuda(), v2.cuda(), torch.tensor([at(0, j) for j in range(256, 300)], device="cuda"))
    got = c.load(torch.tensor([at(1, 599)], device="cuda"), torch.float32)
    assert torch.equal(got[0].double().cpu()[0], ref_values(k)[599])
    for n in (1, 40):
        q = rows(9, 2 * n, heads, dim, torch.float16)
        out = c.attention(q.cuda(), i32([0, n, 2 * n]), i32(L), i32(table), frame=1, max_new=n)
        for r in range(2):
            kk = ref_values(torch.cat((k[:256], k2)) if r == 0 else k)
            vv = ref_values(torch.cat((v[:256], v2)) if r == 0 else v)
            for h in (0, 7, 15):
                o, m, s = ref_attention(q[r * n:(r + 1) * n, h].double(), kk[:, h], vv[:, h], torch.arange(L[r] - n, L[r]), 1, dim ** -0.5)
                check(out[r * n:(r + 1) * n, h], o, bound(o, m, s, torch.float16))


def test_attention_twice_gives_the_same_bits():
    for lens, new in (([3000, 800], [1, 1]), ([900, 500], [200, 7])):
        c, q, start, ln, table, ref, tol = attention_case(lens, new, 8, 2, 128, 64, torch.float16, 1, 8)
        a = c.attention(q, start, ln, table, frame=1, max_len=3000, max_new=max(new))
        b = c.attention(q, start, ln, table, frame=1, max_len=3000, max_new=max(new))
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------- together

class Session:
    """The cache's state as a plain program keeps it: the rows of every request, in float64."""

    def __init__(self, n, heads, dim):
        self.k = [torch.zeros(0, heads, dim, dtype=torch.float64) for _ in range(n)]
        self.v = [torch.zeros(0, heads, dim, dtype=torch.float64) for _ in range(n)]

    def step(self, k, v, q, added, group, frame, dtype):
        ref, tol, at = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), 0
        for r, n in enumerate(added):
            self.k[r] = torch.cat((self.k[r], ref_values(k[at:at + n])))
            self.v[r] = torch.cat((self.v[r], ref_values(v[at:at + n])))
            L = self.k[r].shape[0]
            for h in range(q.shape[1] if n else 0):
                o, m, s = ref_attention(q[at:at + n, h].double(), self.k[r][:, h // group], self.v[r][:, h // group],
                                        torch.arange(L - n, L), frame, q.shape[2] ** -0.5)
                ref[at:at + n, h], tol[at:at + n, h] = o, bound(o, m, s, dtype)
            at += n
        return ref[:at], tol[:at]


@pytest.mark.parametrize("captured", [False, True])
def test_steps_of_growing_sessions(captured):
    """Tables, store and attention as a serving loop runs them, step after step, with idle requests and whole frames;
    captured, the same three launches are one replayed graph and only the device inputs change."""
    R, heads, kv_heads, dim, page, frame, cap, dtype = 5, 8, 2, 64, 16, 10, 40, torch.float16
    c = kv4.KV4Cache(64, page, kv_heads, dim)
    c.d.fill_(NAN)
    table = torch.full((R, 12), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(64, generator=torch.Generator().manual_seed(2)).to(torch.int32).cuda()
    cached, added = i32([0] * R), i32([0] * R)
    k, v = (torch.zeros(cap, kv_heads, dim, dtype=dtype, device="cuda") for _ in range(2))
    q, out = torch.zeros(cap, heads, dim, dtype=dtype, device="cuda"), torch.zeros(cap, heads, dim, dtype=dtype, device="cuda")

    def step():
        t = kv4.build_tables(cached, added, table, free, page, cap)
        c.store(k, v, t.slots)
        c.attention(q, t.q_start, t.lens, table, frame=frame, max_len=160, max_new=10, out=out)
        return t

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = None
    if captured:
        with torch.cuda.stream(side):
            step()                                             # no new rows yet: changes nothing
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            t = step()
    s, used = Session(R, kv_heads, dim), 0
    rng = random.Random(4)
    for i in range(12):
        add = [rng.choice([0, 1, 1, 3, 10]) for _ in range(R)] if i != 5 else [0] * R
        n = sum(add)
        kk, vv, qq = rows(i, cap, kv_heads, dim, dtype), rows(i + 50, cap, kv_heads, dim, dtype), rows(i + 90, cap, heads, dim, dtype)
        added.copy_(i32(add))
        k.copy_(kk.cuda()); v.copy_(vv.cuda()); q.copy_(qq.cuda()); out.fill_(3.0)
        torch.cuda.synchronize()
        if captured:
            graph.replay()
        else:
            with torch.cuda.stream(side):
                t = step()
        torch.cuda.synchronize()
        ref, tol = s.step(kk, vv, qq[:n], add, heads // kv_heads, frame, dtype)
        check(out, ref, tol, f"step {i}")
        assert (out[n:] == 3.0).all() and (t.slots[n:] == -1).all() and t.state[0].item() == 0
        taken = t.state[1].item()
        cached.copy_(t.lens)
        free[:64 - taken].copy_(free[taken:].clone())
        used += taken
    assert used == sum(-(-x.shape[0] // page) for x in s.k)


def test_a_captured_chunk_follows_its_inputs():
    """Tiles, left-over columns, key ranges and their merge in one graph, replayed for other lengths and row counts than
    it was captured with; the check of the waits refuses to be captured and leaves the capture as it was."""
    new, lens = [100, 3, 258], [1500, 900, 2500]
    c, q, start, ln, table, ref, tol = attention_case(lens, new, 2, 2, 64, 32, torch.float16, 258, 17)
    out = torch.zeros_like(q)
    some_start, some_len = i32([0, 1, 2, 3]), i32([5, 6, 7])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.attention(q, some_start, some_len, table, frame=258, max_len=2500, max_new=258, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.attention(q, some_start, some_len, table, frame=258, max_len=2500, max_new=258, out=out)
        with pytest.raises(RuntimeError, match="capturing"):
            c.check()
    some_start.copy_(start)
    some_len.copy_(ln)
    for _ in range(3):
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        check(out, ref, tol)
        assert (out[ref.shape[0]:] == 5.0).all()
    c.check()


def test_two_graphs_and_a_third_stream_at_once():
    """Graphs captured one after the other do not share what a call leaves behind: replayed side by side they agree
    with the eager calls."""
    cases = [attention_case([2000, 900], [1, 1], 8, 2, 128, 64, torch.float16, 1, 8),
             attention_case([700, 1500], [1, 1], 8, 2, 128, 64, torch.float16, 1, 9)]
    outs, graphs, want = [], [], []
    for c, q, start, ln, table, ref, tol in cases:
        out = torch.zeros_like(q)
        want.append(c.attention(q, start, ln, table, frame=1, max_len=2000, max_new=1))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.attention(q, start, ln, table, frame=1, max_len=2000, max_new=1, out=out)
        outs.append(out)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            c, q, start, ln, table, ref, tol = cases[0]
            eager = c.attention(q, start, ln, table, frame=1, max_len=2000, max_new=1)
    torch.cuda.synchronize()
    for out, w in zip(outs + [eager], want + want[:1]):
        assert torch.equal(out, w)


def test_refusals_on_the_device():
    c = pool(4, 16, 2, 64)
    q = rows(1, 3, 4, 64, torch.float16).cuda()
    start, ln, table = i32([0, 3]), i32([10]), i32([[0, 1]])
    with pytest.raises(ValueError, match="f16 or bf16"):
        c.attention(q.float(), start, ln, table)
    with pytest.raises(ValueError, match="lens must be"):
        c.attention(q, start, ln.long(), table)
    with pytest.raises(ValueError, match="agree on the requests"):
        c.attention(q, i32([0, 1, 3]), ln, table)
    with pytest.raises(ValueError, match="channels must be contiguous"):
        c.attention(rows(1, 64, 4, 3, torch.float16).cuda().permute(2, 1, 0), start, ln, table)
    with pytest.raises(ValueError, match="must be on cuda"):
        c.attention(q.cpu(), start, ln, table)
    with pytest.raises(RuntimeError, match="query heads"):
        c.attention(q[:, :3], start, ln, table)
    with pytest.raises(RuntimeError, match="frame -1"):
        c.attention(q, start, ln, table, frame=-1)
    with pytest.raises(RuntimeError, match="overlap"):
        c.attention(q, start, ln, table, out=torch.zeros(3, 1, 64, dtype=q.dtype, device="cuda").expand(3, 4, 64))
    with pytest.raises(ValueError, match="k must be"):
        c.store(q[:, :2], q[:, :2], torch.arange(2, device="cuda"))
    with pytest.raises(ValueError, match="both f32"):
        c.store(q[:, :2], q[:, :2].float(), torch.arange(3, device="cuda"))
    with pytest.raises(ValueError, match="not f32, f16 or bf16"):
        c.load(torch.arange(3, device="cuda"), torch.float64)
    with pytest.raises(ValueError, match="do not belong"):
        kv4.KV4Cache.wrap(c.q, c.d[:, :, :, :1].contiguous())
    # a host pointer is refused before any kernel sees it
    host = torch.zeros(8, dtype=torch.int64)
    L = kv4._load()
    assert L.jepa_b200_kv4_load(c._ref, host.data_ptr(), 8, q.data_ptr(), q.data_ptr(), 1, None) == -1
    assert b"slots is not memory of the current device" in L.jepa_error_text()
    L.jepa_error_reset()
    assert c.attention(q[:0], i32([0, 0]), ln, table).shape == (0, 4, 64)
    # a workspace that is too small
    a = kv4._Attn(q.data_ptr(), q.data_ptr(), 256, 64, 256, 64, start.data_ptr(), ln.data_ptr(), table.data_ptr(), 1, 3, 4000, 4, 1, 1,
                  0.125, 0, 3, None, 0)
    need = L.jepa_b200_kv4_attention_workspace(c._ref, kv4.C.byref(a))
    a.workspace, a.workspace_bytes = q.data_ptr(), need - 1
    assert need > 0 and L.jepa_b200_kv4_attention(c._ref, kv4.C.byref(a), None) == -1
    assert b"the workspace holds" in L.jepa_error_text()
    L.jepa_error_reset()
    with pytest.raises(ValueError, match="2\\^30"):
        kv4.build_tables(ln, ln, table, ln, 16, 2 ** 30 + 1)
    with pytest.raises(ValueError, match="2\\^31"):
        c.attention(q, start, ln, table, frame=2 ** 31)
