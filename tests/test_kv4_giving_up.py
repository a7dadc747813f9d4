"""What follows when the attention kernel for many rows gives up one of its bounded waits: the rows that it has not finished
are NaN, jepa_b200_kv4_check says so once, and the next call is right. The wait that gives up is chosen by the host
(jepa_b200_kv4_attention_giving_up); nothing faults and nothing hangs, and the other waits run out after about a millisecond."""
import ctypes as C

import pytest
import torch

from jepa_b200 import kv4
from test_kv4 import PTR, _attn, _cache, _err

LIMIT = 2_000_000       # clock cycles


def test_refused():
    L, c = kv4._load(), _cache()
    call = lambda a, wait, limit: L.jepa_b200_kv4_attention_giving_up(C.byref(c), C.byref(a), wait, limit, None)
    for wait, limit in ((39, 1), (52, 1), (40, 0), (40, 4_000_000_001)):
        assert call(_attn(), wait, limit) == -1 and "40 <= wait <= 51" in _err()
    assert call(_attn(q=None, workspace=PTR, workspace_bytes=1 << 40), 40, 1) == -1 and "giving_up: q is null" in _err()
    assert call(_attn(frame=-1), 40, 1) == -1 and "frame" in _err()
    assert call(_attn(n_rows=0), 40, 1) == 0


def giving_up(c, q, start, ln, table, out, wait, frame, max_len, max_new):
    L = kv4._load()
    a = kv4._Attn(q.data_ptr(), out.data_ptr(), *q.stride()[:2], *out.stride()[:2], start.data_ptr(), ln.data_ptr(), table.data_ptr(),
                  table.shape[0], q.shape[0], table.shape[1], q.shape[1], kv4._TYPE[q.dtype], frame, c.head_dim ** -0.5, max_len, max_new,
                  None, 0)
    need = L.jepa_b200_kv4_attention_workspace(c._ref, C.byref(a))
    ws = torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda")      # finite partial sums, were they taken for results
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    assert L.jepa_b200_kv4_attention_giving_up(c._ref, C.byref(a), wait, LIMIT, kv4._stream(q.device)) == 0, L.jepa_error_text()
    torch.cuda.synchronize()


# all rows fail at 43, 44, 45, 47, at 41 and 46 where there are blocks enough; a wait that is not met changes nothing
@pytest.mark.gpu
@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("shape", ["one_range", "column_groups", "key_ranges", "long_frame"])
@pytest.mark.parametrize("wait", range(40, 52))
def test_a_wait_that_gives_up(wait, shape, dim, dtype):
    from test_gpu_kv4 import attention_case, check
    lens, new, heads, kv_heads, frame, max_len, max_new = {
        "one_range": ([700, 512], [300, 256], 2, 1, 1, 700, 300),
        "column_groups": ([700, 512], [300, 256], 4, 1, 0, 700, 20),     # a CTA takes group after group of 256 columns
        "key_ranges": ([3000], [300], 2, 1, 1, 3000, 300),               # partial sums, joined by a second kernel
        "long_frame": ([1152], [704], 1, 1, 576, 700, 704)}[shape]
    c, q, start, ln, table, ref, tol = attention_case(lens, new, heads, kv_heads, dim, 32, dtype, frame, 7)
    T = sum(new)
    for old in (7.0, float("inf")):
        out = torch.full_like(q, old)
        giving_up(c, q, start, ln, table, out, wait, frame, max_len, max_new)
        got = out[:T].double().cpu()
        nan = got.isnan().all(-1)
        assert torch.equal(nan, got.isnan().any(-1))                      # a row's head is given up as a whole
        good = ((got - ref).abs() <= tol).all(-1)
        assert (nan | good).all()
        assert (out[T:] == old).all()
        short = shape == "key_ranges"                                     # ranges of 256 keys: four blocks
        if wait in (43, 44, 45, 47, 49) or (wait in (41, 46) and not short):
            assert nan.all()
        if wait in (50, 51) and shape == "column_groups":                 # what is done is right, what was to come is not there
            assert nan.any() and good.any()
        if nan.any():
            with pytest.raises(RuntimeError, match="gave up"):
                c.check()
    try:
        c.check()                             # (waits 50 and 51 may give up behind finished rows alone)
    except RuntimeError:
        c.check()
    check(c.attention(q, start, ln, table, frame=frame, max_len=max_len, max_new=max_new), ref, tol)
    c.check()


@pytest.mark.gpu
def test_a_failure_is_told_once_whoever_asks():
    from test_gpu_kv4 import attention_case
    c, q, start, ln, table, _, _ = attention_case([300], [100], 1, 1, 64, 32, torch.float16, 1, 3)
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()

    def told(stream):
        with torch.cuda.stream(stream):
            try:
                c.check()
            except RuntimeError as e:
                assert "gave up" in str(e)
                return 1
        return 0

    here = torch.cuda.current_stream()
    assert told(here) == 0
    with torch.cuda.stream(side):
        giving_up(c, q, start, ln, table, out, 43, 1, 300, 100)
    assert (told(here), told(side), told(here)) == (1, 0, 0)
    giving_up(c, q, start, ln, table, out, 47, 1, 300, 100)
    giving_up(c, q, start, ln, table, out, 44, 1, 300, 100)
    assert (told(side), told(here)) == (1, 0)


@pytest.mark.gpu
def test_a_failure_during_a_check_is_not_lost():
    """Checks on one stream while kernels of another give up: one of those that follow a failure tells it."""
    from test_gpu_kv4 import attention_case
    c, q, start, ln, table, _, _ = attention_case([300], [100], 1, 1, 64, 32, torch.float16, 1, 3)
    out, L, side = torch.zeros_like(q), kv4._load(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = kv4._Attn(q.data_ptr(), out.data_ptr(), *q.stride()[:2], *out.stride()[:2], start.data_ptr(), ln.data_ptr(), table.data_ptr(),
                  1, q.shape[0], table.shape[1], 1, 1, 1, 0.125, 300, 100, None, 0)
    for _ in range(50):
        assert L.jepa_b200_kv4_attention_giving_up(c._ref, C.byref(a), 43, LIMIT, side.cuda_stream) == 0
        told = 0
        for k in range(20):
            if k == 19:
                side.synchronize()
            try:
                c.check()
            except RuntimeError:
                told += 1
        assert told == 1
