"""GPU parity of the paged 8-bit cache (plan, write, attention) against the 64-bit restatement.

Plan and write are compared bit for bit.  Attention: with u = 2^-24, n keys, head dim D, a score (base 2) is off by at
most (D + 4) u reach, a probability by the relative ln 2 times that, one exp2 (2 u) and n u for the sums, twice for
numerator and denominator; the weights and the output are rounded to 11 or 8 bits at half a step each.  A V scale of code
e enters as score + (e - 121), one more rounding of a sum of magnitude reach + |e - 121|, and leaves the same way in the
log-sum-exp (codes here are within 54 of 121)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import paged as orc
from triton_tenstorrent_amd import kernels as K, runtime as rt

pytestmark = pytest.mark.gpu
U = 2.0**-24
I32 = dict(dtype=torch.int32, device="cuda")


def i32(v):
    return torch.tensor(np.asarray(v), **I32)


# ---- plan -------------------------------------------------------------------
def run_plan(ctx, new, table, free, P, T, start=None):
    t = i32(table)
    p = K.paged_plan(i32(ctx), i32(new), t, i32(free), P, T, None if start is None else i32([start]))
    want = orc.plan(ctx, new, np.asarray(table), np.asarray(free), P, T, start or 0)
    got = (t, p.lens, p.cu_new, p.slot_map, p.free_end)
    for g, w, name in zip(got, (*want[:4], [want[4]]), ("table", "lens", "cu_new", "slot_map", "free_end")):
        assert np.array_equal(g.cpu().numpy(), np.asarray(w)), name


@pytest.mark.parametrize("B,P,hi", [(1, 1, 5), (3, 16, 100), (17, 64, 300), (1023, 7, 3), (1024, 16, 40), (1025, 32, 20), (5000, 16, 30)])
@pytest.mark.parametrize("slack", [0, 77])
def test_plan_against_the_plain_form(B, P, hi, slack):
    rng = np.random.default_rng(B + P)
    ctx, new = rng.integers(0, hi, B), rng.integers(0, hi, B)
    new[rng.random(B) < 0.3] = 0
    width = int(max(-(-(ctx + new) // P))) + 1
    ids = rng.permutation(int(sum(-(-(ctx + new) // P))) + 5)
    table, used = np.full((B, width), -1), 0
    for b in range(B):
        n = -(-ctx[b] // P)
        table[b, :n] = ids[used:used + n]
        used += n
    run_plan(ctx, new, table, ids[used:], P, int(new.sum()) + slack)


def test_plan_where_pages_tokens_or_the_table_run_out():
    table = np.full((4, 3), -1)
    table[1, :2] = [11, 12]
    run_plan([0, 7, 0, 0], [9, 3, 6, 2], table, [1, 2, 3, 4], 4, 20)              # four pages for seven
    run_plan([0, 7, 0, 0], [9, 3, 6, 2], table, np.arange(20, 40), 4, 13)         # tokens cut at 13
    run_plan([0, 7, 0, 0], [50, 30, 6, 2], table, np.arange(20, 40), 4, 40)       # twelve positions a row
    run_plan([0, 7, 0, 0], [9, 3, 6, 2], table, np.arange(20, 40), 4, 20, start=5)
    run_plan([0, 7, 0, 0], [9, 3, 6, 2], table, np.arange(20, 40), 4, 20, start=18)
    run_plan([-3, 7, 0, 100], [9, -3, 6, 2], table, np.arange(20, 40), 4, 20)     # negative, and past the table
    run_plan([0, 0], [0, 0], np.full((2, 3), -1), [3], 4, 6)                      # nothing new
    run_plan([1], [2**31 - 1], np.array([[3, -1, -1]]), [7, 8], 4, 9)
    run_plan([5, 0], [2**31 - 1, 2**31 - 1], np.array([[3, 4, -1], [-1] * 3]), [7, 8], 4, 9)


def test_plan_without_new_tokens_or_free_pages():
    p = K.paged_plan(i32([3, 0]), i32([0, 0]), i32([[4], [-1]]), torch.empty(0, **I32), 4, 0)
    assert p.lens.tolist() == [3, 0] and p.cu_new.tolist() == [0, 0, 0] and p.slot_map.numel() == 0 and p.free_end.tolist() == [0]


def test_plan_of_a_table_with_row_stride():
    big = torch.full((6, 9), -7, **I32)
    t = big[1:5, 2:7]
    p = K.paged_plan(i32([0] * 4), i32([3, 9, 0, 5]), t, i32(range(10, 20)), 4, 17)
    want = orc.plan([0] * 4, [3, 9, 0, 5], np.full((4, 5), -7), np.arange(10, 20), 4, 17)
    assert np.array_equal(t.cpu().numpy(), want[0]) and np.array_equal(p.slot_map.cpu().numpy(), want[3])
    big[1:5, 2:7] = -7
    assert (big == -7).all()


# ---- write ------------------------------------------------------------------
def filled(pages, H, P, D, seed):
    """A cache of random codes and scales, some codes NaN."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 256, (2, pages, H, P, D)).astype(np.uint8)
    codes[(codes & 127) == 127] -= 1
    codes[:, :, :, P - 1] = 0x7F if P > 1 else 0
    return codes, rng.integers(110, 125, (2, pages, H)).astype(np.int64)


def device_cache(codes, scales, layout="phtd"):
    k, v = (torch.from_numpy(c.copy()).cuda() for c in codes)
    if layout == "pthd":        # pages of whole tokens: the same shape, other strides
        k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    return K.PagedCache(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn),
                        *(torch.from_numpy(s.astype(np.uint8)).cuda() for s in scales))


def plain(codes):
    """Codes with one pattern for NaN, whose sign bit means nothing."""
    return np.where((codes & 127) == 127, 127, codes)


def check_write(x, slots, codes, scales, layout="phtd"):
    cache = device_cache(codes, scales, layout)
    K.paged_write(x[0], x[1], i32(slots), cache)
    for j, (c, s) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
        wc, ws = codes[j].copy(), scales[j].copy()
        orc.write(x[j].cpu().double().numpy(), np.asarray(slots), wc, ws)
        assert np.array_equal(s.cpu().numpy(), ws), "scale"
        bad = np.argwhere(plain(c.view(torch.uint8).cpu().numpy()) != plain(wc))
        assert len(bad) == 0, f"codes at {bad[:5].tolist()}"


def runs(spec, P):
    """[(page, first row, tokens)] -> slots."""
    return np.concatenate([np.arange(p * P + r, p * P + r + n) for p, r, n in spec])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,P,D", [(1, 16, 128), (8, 64, 128), (3, 32, 64), (2, 128, 256), (2, 16, 40), (1, 5, 33), (4, 64, 16), (1, 1, 64),
                                   (2, 256, 128), (2, 1000, 64)])
def test_write_against_the_plain_form(dtype, H, P, D):
    codes, scales = filled(9, H, P, D, seed=P + D)
    spec = [(4, 0, P), (0, P // 2, P - P // 2), (7, 0, 1), (3, P - 1, 1), (8, 0, max(1, P // 3))]
    slots = runs(spec, P)
    g = torch.Generator().manual_seed(D)
    x = torch.randn(2, len(slots), H, D, generator=g) * torch.tensor([1.0, 30.0, 1e-3])[torch.randint(0, 3, (len(slots), 1, 1), generator=g)]
    check_write(x.to(dtype).cuda(), slots, codes, scales)


@pytest.mark.parametrize("layout", ["phtd", "pthd"])
def test_write_of_many_single_tokens(layout):
    H, P, D = 4, 16, 64
    codes, scales = filled(300, H, P, D, seed=1)
    slots = np.random.default_rng(2).permutation(300)[:257] * P + np.arange(257) % P
    x = (torch.randn(2, 257, H, D) * 4).to(torch.bfloat16).cuda()
    check_write(x, slots, codes, scales, layout)


def test_write_skips_slots_outside_and_runs_meet():
    H, P, D = 2, 16, 64
    codes, scales = filled(4, H, P, D, seed=3)
    slots = [-1, 5, 6, 7, -1, -1, 64, 1000000, 14 + 16, 15 + 16, 32, 33, -5, 48]   # 31 ends page 1, 32 begins page 2
    x = torch.randn(2, len(slots), H, D).to(torch.float16).cuda()
    check_write(x, slots, codes, scales)


def test_write_of_special_values():
    H, P, D = 2, 16, 64
    codes, scales = filled(6, H, P, D, seed=4)
    x = torch.randn(2, 20, H, D)
    x[0, 0, 0, 3], x[0, 1, 1, 5], x[1, 2, 0, 7] = float("inf"), -float("inf"), float("nan")
    x[:, 3] = 0.0
    x[:, 4:8] = 0.0                     # a page of zeros
    x[0, 8], x[1, 8] = 3e38, -1e-38     # the ends of bf16's range
    x[0, 9], x[1, 9] = float("nan"), float("inf")   # nothing finite in the run
    x[:, 10:] *= torch.exp2(torch.randint(-20, 20, (2, 10, 1, 1)).float())
    slots = runs([(0, 0, 4), (1, 0, 4), (2, 3, 1), (3, 0, 1), (4, 2, 10)], P)
    check_write(x.to(torch.bfloat16).cuda(), slots, codes, scales)


@pytest.mark.parametrize("D,pad", [(128, 0), (128, 8), (128, 1), (64, 3)])
def test_write_of_strided_inputs(D, pad):
    # k and v as columns of one projection's output, rows padded so that they begin off a 16-byte boundary
    H, P, T = 3, 32, 70
    codes, scales = filled(5, H, P, D, seed=5)
    qkv = torch.randn(T, 3 * H * D + pad).to(torch.bfloat16).cuda()
    k, v = (qkv[:, i * H * D + pad:(i + 1) * H * D + pad].view(T, H, D) for i in (1, 2))
    slots = runs([(0, 0, 32), (2, 10, 22), (4, 0, 16)], P)
    check_write((k, v), slots, codes, scales)


def test_write_keeps_nan_codes_of_earlier_rows():
    H, P, D = 2, 64, 128
    codes, scales = filled(3, H, P, D, seed=8)
    codes[:, :, :, 2, 5], codes[:, :, :, 33, 7] = 0x7F, 0xFF
    x = (torch.randn(2, 11, H, D) * 3e6).to(torch.bfloat16).cuda()      # every scale grows
    check_write(x, runs([(0, 40, 10), (2, 63, 1)], P), codes, scales)


@pytest.mark.parametrize("D", [64, 128, 256, 48])
def test_write_grows_scales_token_by_token(D):
    H, P = 2, 16
    codes, scales = filled(2, H, P, D, seed=6)
    cache = device_cache(codes, scales)
    want = [(codes[j].copy(), scales[j].copy()) for j in range(2)]
    x = (torch.randn(2, P, H, D) * torch.exp2(torch.arange(P) * 0.7)[None, :, None, None]).to(torch.bfloat16).cuda()
    for t in range(P):
        K.paged_write(x[0, t:t + 1], x[1, t:t + 1], i32([P + t]), cache)
        for j in range(2):
            orc.write(x[j, t:t + 1].cpu().double().numpy(), [P + t], *want[j])
    for (wc, ws), c, s in zip(want, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        assert np.array_equal(s.cpu().numpy(), ws) and np.array_equal(c.view(torch.uint8).cpu().numpy(), wc)


# ---- attention --------------------------------------------------------------
def make(lens, n_q, Hq, H, P, D, dtype, seed=0, spare=3, q_scale=2.0, layout="phtd"):
    """Queries, cache and tables; rows behind a sequence's end and pages of no sequence hold NaN codes."""
    rng = np.random.default_rng(seed)
    need = [-(-n // P) for n in lens]
    pages = sum(need) + spare
    width = max(max(need), 1) + 1
    ids = rng.permutation(pages)
    table, at = np.full((len(lens), width), -1), 0
    codes = np.full((2, pages, H, P, D), 0x7F, np.uint8)
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
        pos = np.arange(lens[b])
        codes[:, table[b, pos // P], :, pos % P] = orc.encode(np.clip(rng.standard_normal((lens[b], 2, H, D)) * 100, -448, 448))
    scales = rng.integers(118, 123, (2, pages, H)).astype(np.int64)
    cu = np.concatenate([[0], np.cumsum(n_q)])
    q = torch.from_numpy(rng.standard_normal((cu[-1], Hq, D)) * q_scale).to(dtype)
    return q, codes, scales, table, np.asarray(lens), cu


def compare(o, lse, want, n, D, dtype):
    wo, wl, spread, reach = want
    o, lse = o.cpu().double().numpy(), lse.cpu().double().numpy()
    rows = ~np.isnan(wl)
    assert np.array_equal(np.isneginf(lse[rows]), np.isneginf(wl[rows]))
    fine = rows & np.isfinite(wl)
    ds = (D + 5) * U * reach + 54 * U
    rel = 2 * (np.log(2.0) * ds + 2 * U + n * U)
    tol = spread * (2.0**-11 + rel[..., None]) + torch.finfo(dtype).eps / 2 * (np.abs(wo) + spread * 2.0**-10) + 2.0**-24
    assert (np.abs(o - wo)[fine] <= tol[fine]).all(), np.nanmax((np.abs(o - wo) / tol)[fine])
    ltol = ds + (n + 4) * U / np.log(2.0) + 2 * U * np.abs(np.where(fine, wl, 0.0)) + 64 * U
    assert (np.abs(lse - np.where(fine, wl, 0.0))[fine] <= ltol[fine]).all()
    none = rows & np.isneginf(wl)
    assert (o[none] == 0).all()


def check_attention(lens, n_q, Hq, H, P, D, dtype=torch.bfloat16, causal=True, max_q=None, sm_scale=None, layout="phtd", **kw):
    q, codes, scales, table, lens, cu = make(lens, n_q, Hq, H, P, D, dtype, **kw)
    sm_scale = D ** -0.5 if sm_scale is None else sm_scale
    cache = device_cache(codes, scales, layout)
    o, lse = K.paged_attention(q.cuda(), cache, i32(table), i32(lens), i32(cu), sm_scale, max_q=max_q, causal=causal, return_lse=True)
    want = orc.attention(q.double().numpy(), codes[0], codes[1], scales[0], scales[1], table, lens, cu, sm_scale, causal)
    compare(o, lse, want, max(max(lens), 1), D, dtype)
    return rt.last_kernel_name()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,H", [(1, 1), (4, 4), (8, 2), (6, 2), (8, 1), (16, 1), (24, 2), (33, 1), (48, 1)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_head_layouts(dtype, Hq, H, D):
    check_attention([1, 63, 200, 0, 129], [1, 1, 1, 1, 1], Hq, H, 32, D, dtype, max_q=1, seed=Hq + D)


@pytest.mark.parametrize("P", [16, 32, 64, 128, 256, 1, 8, 24, 48])
@pytest.mark.parametrize("D", [64, 128])
def test_decode_page_sizes(P, D):
    check_attention([1, 15, 16, 17, 64, 65, 255, 256, 257, 700], [1] * 10, 8, 2, P, D, max_q=1, seed=P)


@pytest.mark.parametrize("D", [1, 8, 16, 32, 40, 80, 96, 112, 160, 192, 255])
@pytest.mark.parametrize("n", [1, 9])
def test_other_head_dims(D, n):
    check_attention([70, 33], [n, n], 4, 2, 16, D, torch.float16, max_q=n, seed=D)


@pytest.mark.parametrize("lens,n_q", [
    ([5000], [1]), ([20001], [1]), ([3, 9000, 1, 0, 2500], [1, 1, 1, 1, 1]), ([300] * 40, [1] * 40),
    ([100, 200, 300], [1, 0, 1]), ([0, 0], [1, 1]), ([0, 0], [0, 0]), ([2000, 1999, 2001], [0, 1, 0])])
def test_decode_lengths(lens, n_q):
    check_attention(lens, n_q, 4, 2, 64, 128, max_q=1, seed=len(lens))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Hq,H,D", [(2, 2, 128), (8, 2, 128), (6, 2, 64), (4, 1, 256), (40, 1, 64)])
def test_rows_of_many_queries(dtype, causal, Hq, H, D):
    check_attention([130, 64, 1, 300, 0, 77], [130, 10, 1, 33, 0, 70], Hq, H, 32, D, dtype, causal, seed=D)


@pytest.mark.parametrize("P", [16, 64, 128, 256, 8, 24])
def test_rows_page_sizes(P):
    check_attention([200, 129, 500], [200, 5, 100], 4, 2, P, 128, seed=P)
    check_attention([200, 129, 500], [2, 5, 10], 2, 2, P, 64, torch.float16, seed=P)


@pytest.mark.parametrize("lens,n_q", [
    ([3, 0, 10], [5, 4, 10]),                   # more queries than keys: the first see none
    ([4000], [3]), ([6000, 20], [17, 20]),      # few rows over many keys
    ([1] * 50, [1] * 50), ([257], [257]), ([1000, 1, 999], [1000, 1, 1])])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_lengths(lens, n_q, causal):
    check_attention(lens, n_q, 4, 2, 64, 128, causal=causal, seed=len(lens))


@pytest.mark.parametrize("sm_scale", [0.0, -0.1, 1.0, 3.0])
@pytest.mark.parametrize("n", [1, 40])
def test_scales_of_the_scores(sm_scale, n):
    check_attention([333, 90], [n, n], 4, 2, 32, 128, max_q=n, sm_scale=sm_scale)


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("layout", ["phtd", "pthd"])
def test_cache_layouts(n, layout):
    check_attention([333, 90], [n, n], 8, 4, 32, 128, max_q=n, layout=layout)


@pytest.mark.parametrize("n", [1, 30])
def test_pages_of_very_different_scales(n):
    # scales 2^-60 .. 2^40 side by side: sums must not overflow, and the small pages must not disturb the large ones
    q, codes, scales, table, lens, cu = make([300, 150], [n, n], 4, 2, 16, 128, torch.bfloat16, seed=9)
    rng = np.random.default_rng(1)
    scales[1] = rng.integers(67, 168, scales[1].shape)
    cache = device_cache(codes, scales)
    o, lse = K.paged_attention(q.cuda(), cache, i32(table), i32(lens), i32(cu), 0.09, max_q=n, return_lse=True)
    want = orc.attention(q.double().numpy(), codes[0], codes[1], scales[0], scales[1], table, lens, cu, 0.09, True)
    compare(o, lse, want, 300, 128, torch.bfloat16)


@pytest.mark.parametrize("n", [1, 20])
def test_pages_outside_the_cache_count_as_absent(n):
    q, codes, scales, table, lens, cu = make([300, 150, 64], [n, n, n], 4, 2, 32, 64, torch.bfloat16, seed=10)
    table[0, 3], table[0, 5], table[1, 0], table[2, :] = -1, 10**6, codes.shape[1], -1
    cache = device_cache(codes, scales)
    o, lse = K.paged_attention(q.cuda(), cache, i32(table), i32(lens), i32(cu), 0.1, max_q=n, return_lse=True)
    want = orc.attention(q.double().numpy(), codes[0], codes[1], scales[0], scales[1], table, lens, cu, 0.1, True)
    compare(o, lse, want, 300, 64, torch.bfloat16)


@pytest.mark.parametrize("n", [1, 20])
def test_lengths_past_the_table_end_there(n):
    q, codes, scales, table, lens, cu = make([96, 96], [n, n], 2, 2, 32, 64, torch.bfloat16, seed=11)
    table = np.ascontiguousarray(table[:, :3])
    cache = device_cache(codes, scales)
    args = (i32(table), i32([96, 2**31 - 1]), i32(cu), 0.1)
    o, lse = K.paged_attention(q.cuda(), cache, *args, max_q=n, return_lse=True)
    want = orc.attention(q.double().numpy(), codes[0], codes[1], scales[0], scales[1], table, [96, 96], cu, 0.1, True)
    compare(o, lse, want, 96, 64, torch.bfloat16)
    o, lse = K.paged_attention(q.cuda(), cache, i32(table), i32([96, -5]), i32(cu), 0.1, max_q=n, return_lse=True)
    assert (o[n:] == 0).all() and torch.isneginf(lse[n:]).all()


@pytest.mark.parametrize("n", [1, 20])
def test_rows_behind_the_last_sequence_stay(n):
    q, codes, scales, table, lens, cu = make([90, 40], [n, n], 4, 2, 32, 128, torch.float16, seed=12)
    cache = device_cache(codes, scales)
    rows = 2 * n + 13
    big = torch.full((rows, 4, 128), float("nan"), dtype=torch.float16, device="cuda")
    big[:2 * n] = q.cuda()
    out = torch.full_like(big, 7.0)
    o, lse = K.paged_attention(big, cache, i32(table), i32(lens), i32(cu), 0.1, max_q=n, return_lse=True, out=out)
    want = orc.attention(q.double().numpy(), codes[0], codes[1], scales[0], scales[1], table, lens, cu, 0.1, True)
    compare(o[:2 * n], lse[:2 * n], want, 90, 128, torch.float16)
    assert o.data_ptr() == out.data_ptr() and (out[2 * n:] == 7.0).all()


@pytest.mark.parametrize("n", [1, 20])
def test_strided_queries_and_results(n):
    q, codes, scales, table, lens, cu = make([90, 300], [n, n], 4, 2, 32, 128, torch.bfloat16, seed=13)
    cache = device_cache(codes, scales)
    wide = torch.zeros(2 * n, 4 * 128 + 2 * 2 * 128 + 8, dtype=torch.bfloat16, device="cuda")
    qv = wide[:, :512].view(2 * n, 4, 128)
    qv.copy_(q)
    want = orc.attention(q.double().numpy(), codes[0], codes[1], scales[0], scales[1], table, lens, cu, 0.1, True)
    for off in (0, 8, 3):
        hold = torch.zeros(4, 2 * n, 128 + off, dtype=torch.bfloat16, device="cuda")
        out = hold[:, :, off:].transpose(0, 1)
        o, lse = K.paged_attention(qv, cache, i32(table), i32(lens), i32(cu), 0.1, max_q=n, return_lse=True, out=out)
        compare(o, lse, want, 300, 128, torch.bfloat16)
        assert (hold[:, :, :off] == 0).all()


@pytest.mark.parametrize("n", [1, 20])
def test_nan_keys_reach_the_queries_that_attend_them_only(n):
    P, D = 16, 64
    q, codes, scales, table, lens, cu = make([100, 70], [n, n], 2, 1, P, D, torch.bfloat16, seed=14)
    bad = [(0, 30, 0), (0, 95, 1), (0, 97, 0), (1, 69, 1)]          # (sequence, position, of K or of V)
    for b, pos, j in bad:
        codes[j, table[b, pos // P], 0, pos % P, 5] = 0x7F
    cache = device_cache(codes, scales)
    o, lse = K.paged_attention(q.cuda(), cache, i32(table), i32(lens), i32(cu), 0.1, max_q=n, return_lse=True)
    o = o.float().cpu().numpy()
    for b, L in ((0, 100), (1, 70)):
        for i in range(n):
            last = L - n + i
            row = np.isnan(o[cu[b] + i])
            k_bad = any(j == 0 and bb == b and pos <= last for bb, pos, j in bad)
            v_bad = any(j == 1 and bb == b and pos <= last for bb, pos, j in bad)
            assert row.all() if k_bad else (row[:, 5].all() == v_bad and not np.delete(row, 5, 1).any()), (b, i)


@pytest.mark.parametrize("n", [1, 20])
def test_infinite_queries_give_nan_in_their_row_only(n):
    q, codes, scales, table, lens, cu = make([100, 70], [n, n], 2, 1, 16, 64, torch.bfloat16, seed=15)
    q[0, 0, 0] = float("inf")
    cache = device_cache(codes, scales)
    o, _ = K.paged_attention(q.cuda(), cache, i32(table), i32(lens), i32(cu), 0.1, max_q=n, return_lse=True)
    assert torch.isnan(o[0, 0]).all() and torch.isfinite(o[0, 1]).all() and torch.isfinite(o[1:]).all()


def test_results_do_not_change_from_call_to_call():
    for n in (1, 30):
        q, codes, scales, table, lens, cu = make([3000, 70, 900], [n] * 3, 8, 2, 64, 128, torch.bfloat16, seed=16)
        cache = device_cache(codes, scales)
        args = (q.cuda(), cache, i32(table), i32(lens), i32(cu), 0.09)
        o, lse = K.paged_attention(*args, max_q=n, return_lse=True)
        for _ in range(5):
            o2, lse2 = K.paged_attention(*args, max_q=n, return_lse=True)
            assert torch.equal(o, o2) and torch.equal(lse, lse2)
        assert torch.equal(o, K.paged_attention(*args, max_q=n))


def test_offsets_past_32_bits():
    # a cache of over 4 GiB of codes a side, the sequences at its far end
    P, H, D, pages = 128, 8, 128, 33000
    cache = K.paged_cache(pages, H, D, P)
    assert cache.k.numel() > 2**32
    ids = np.arange(pages - 8, pages)[::-1].copy()
    lens, g = [500, 300], torch.Generator().manual_seed(3)
    table = i32([ids[:4], ids[4:]])
    x = torch.randn(2, 800, H, D, generator=g).to(torch.bfloat16).cuda()
    pos = np.concatenate([np.arange(n) for n in lens])
    seq = np.repeat([0, 1], lens)
    slots = ids.reshape(2, 4)[seq, pos // P] * P + pos % P
    K.paged_write(x[0], x[1], i32(slots), cache)
    codes = np.full((2, 8, H, P, D), 0x7F, np.uint8)
    scales = np.zeros((2, 8, H), np.int64)
    local = (slots - (pages - 8) * P)
    for j in range(2):
        orc.write(x[j].cpu().double().numpy(), local, codes[j], scales[j])
    for n in (1, 20):
        q = torch.randn(2 * n, 16, D, generator=g).to(torch.bfloat16)
        cu = [0, n, 2 * n]
        o, lse = K.paged_attention(q.cuda(), cache, table, i32(lens), i32(cu), 0.09, max_q=n, return_lse=True)
        want = orc.attention(q.double().numpy(), codes[0], codes[1], scales[0], scales[1], ids.reshape(2, 4) - (pages - 8), lens, cu, 0.09, True)
        compare(o, lse, want, 500, D, torch.bfloat16)


# ---- refusals, which the library makes before anything is launched ----------
def test_attention_refusals():
    q, codes, scales, table, lens, cu = make([300, 150], [1, 1], 4, 2, 16, 64, torch.bfloat16)
    c, tb, ln, cq, q = device_cache(codes, scales), i32(table), i32(lens), i32(cu), q.cuda()
    out = torch.empty_like(q)
    run = lambda grid=(2, 4), qq=q, cc=c, t=tb, ws=None, sm=0.1, mq=1, o=out: K.paged_attn_kernel[grid](
        qq, *cc, t, ln, cq, o, None, ws, sm, mq, CAUSAL=True)
    for bad in (dict(grid=(2, 3)), dict(grid=(3, 4)), dict(grid=(2, 4, 2)), dict(sm=float("inf")), dict(sm=float("nan")), dict(mq=0),
                dict(mq=-1), dict(o=out[:1].expand(2, 4, 64))):
        with pytest.raises(ValueError):
            run(**bad)
    wide = K.paged_cache(4, 1, 320, 16)
    with pytest.raises(NotImplementedError):
        K.paged_attention(torch.zeros(2, 1, 320, dtype=torch.bfloat16, device="cuda"), wide, tb, ln, cq, 0.1)
    # a table that allows long sequences: parts need room
    t2 = torch.cat([tb, torch.full((2, 400), -1, **I32)], 1)
    for ws in (None, torch.empty(16, dtype=torch.uint8, device="cuda")):
        with pytest.raises(ValueError, match="workspace"):
            run(t=t2, ws=ws)
    assert rt.load() is not None and torch.isfinite(K.paged_attention(q, c, t2, ln, cq, 0.1, max_q=1).float()).all()


def test_plan_and_write_refusals():
    t, one = i32(np.full((2, 3), -1)), i32([1, 1])
    with pytest.raises(ValueError):
        K.paged_plan(one, one, t, i32([0, 1]), 0, 4)
    with pytest.raises(NotImplementedError):
        K.paged_plan(one, one, t, i32([0, 1]), 2**30, 4)
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16, device="cuda")
    cache = K.paged_cache(2, 1, 64, 16)
    with pytest.raises(ValueError):
        K.paged_write_kernel[(3, )](x, x, one, *cache)
    with pytest.raises(ValueError):     # pages on top of one another
        K.paged_write(x, x, one, K.PagedCache(cache.k[:1].expand(2, 1, 16, 64), *cache[1:]))


def test_which_kernel_runs():
    for lens, n, Hq, H, D, max_q, want in (
            ([90], [1], 4, 2, 128, 1, "paged_attn_one_bf16_d128_r1"), ([5000], [1], 4, 2, 128, 1, "paged_attn_join_bf16_d128_r1"),
            ([90], [1], 20, 1, 64, 1, "paged_attn_one_bf16_d64_r2"), ([90, 40], [5, 2], 8, 2, 128, 5, "paged_attn_few_bf16_d128_r2"),
            ([90, 40], [5, 2], 6, 2, 256, 5, "paged_attn_few_bf16_d256_r1"), ([90, 40], [60, 1], 4, 2, 128, 60, "paged_attn_rows_join_bf16_d128_r1"),
            ([60, 40], [60, 1], 4, 2, 64, 60, "paged_attn_rows_bf16_d64_r2"), ([90], [1], 4, 2, 80, 1, "paged_attn_any_bf16")):
        q, codes, scales, table, ln, cu = make(lens, n, Hq, H, 16, D, torch.bfloat16)
        table = np.ascontiguousarray(table[:, :-1])
        K.paged_attention(q.cuda(), device_cache(codes, scales), i32(table), i32(ln), i32(cu), 0.1, max_q=max_q)
        assert rt.last_kernel_name() == want


# ---- together ---------------------------------------------------------------
def serve(steps, H, Hq, D, P, pages, B, seed, capture=False):
    """Plan, write and attend step by step (each step: new tokens of each sequence); every step against the 64-bit form."""
    rng = np.random.default_rng(seed)
    width = 20
    free = rng.permutation(pages)
    cache = K.paged_cache(pages, H, D, P)
    codes = np.full((2, pages, H, P, D), 0x7F, np.uint8)
    for c in cache[:2]:
        c.view(torch.uint8).fill_(0x7F)
    scales = np.zeros((2, pages, H), np.int64)
    table, lens, start = i32(np.full((B, width), -1)), i32([0] * B), i32([0])
    wt, wl, ws = np.full((B, width), -1), np.zeros(B, int), 0
    for new in steps:
        T = int(sum(new))
        x = torch.from_numpy(rng.standard_normal((2, T, H, D)) * rng.choice([1, 9], (1, T, 1, 1))).to(torch.bfloat16)
        q = torch.from_numpy(rng.standard_normal((T, Hq, D))).to(torch.bfloat16)
        plan = K.paged_plan(lens, i32(new), table, i32(free), P, T, start)
        K.paged_write(x[0].cuda(), x[1].cuda(), plan.slot_map, cache)
        o, lse = K.paged_attention(q.cuda(), cache, table, plan.lens, plan.cu_new, D ** -0.5, max_q=max(new), return_lse=True)
        lens, start = plan.lens, plan.free_end
        wt, wl, cu, slots, ws = orc.plan(wl, new, wt, free, P, T, ws)
        for j in range(2):
            orc.write(x[j].double().numpy(), slots, codes[j], scales[j])
        want = orc.attention(q.double().numpy(), codes[0], codes[1], scales[0], scales[1], wt, wl, cu, D ** -0.5, True)
        compare(o, lse, want, max(wl), D, torch.bfloat16)
    for j in range(2):
        assert np.array_equal(cache[j].view(torch.uint8).cpu().numpy(), codes[j])
        assert np.array_equal(cache[2 + j].cpu().numpy(), scales[j])


def test_prompts_then_decode_steps_then_a_late_prompt():
    serve([[37, 64, 0, 1]] + [[1, 1, 0, 1]] * 5 + [[0, 1, 90, 3]] + [[1, 1, 1, 1]] * 4, 2, 8, 64, 16, 80, 4, seed=0)
    serve([[100, 20]] + [[1, 1]] * 3 + [[4, 4]] * 3, 2, 4, 128, 64, 12, 2, seed=1)


def test_a_decode_step_captured_into_a_graph():
    H, Hq, D, P, B, pages = 2, 8, 128, 16, 3, 60
    g = torch.Generator().manual_seed(0)
    eager, graphed = (dict(cache=K.paged_cache(pages, H, D, P), table=i32(np.full((B, 20), -1)), lens=i32([0] * B), start=i32([0]))
                      for _ in range(2))
    free = i32(np.random.default_rng(0).permutation(pages))
    x, q = torch.empty(2, B, H, D, dtype=torch.bfloat16, device="cuda"), torch.empty(B, Hq, D, dtype=torch.bfloat16, device="cuda")
    ones = i32([1] * B)

    def step(s):
        p = K.paged_plan(s["lens"], ones, s["table"], free, P, B, s["start"])
        K.paged_write(x[0], x[1], p.slot_map, s["cache"])
        o, lse = K.paged_attention(q, s["cache"], s["table"], p.lens, p.cu_new, D ** -0.5, max_q=1, return_lse=True)
        s["lens"].copy_(p.lens)
        s["start"].copy_(p.free_end)
        return o, lse

    prompt = [30, 7, 150]
    xs = torch.randn(2, sum(prompt), H, D, generator=g).to(torch.bfloat16).cuda()
    for s in (eager, graphed):
        for c in s["cache"][:2]:
            c.view(torch.uint8).fill_(0x7F)
        p = K.paged_plan(s["lens"], i32(prompt), s["table"], free, P, sum(prompt), s["start"])
        K.paged_write(xs[0], xs[1], p.slot_map, s["cache"])
        s["lens"].copy_(p.lens)
        s["start"].copy_(p.free_end)
    x.copy_(torch.randn(x.shape, generator=g))
    q.copy_(torch.randn(q.shape, generator=g))
    step(eager), step(graphed)                  # outside the graph: code objects are loaded here
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(graphed)
    for i in range(6):
        x.copy_(torch.randn(x.shape, generator=g) * (1 + i))
        q.copy_(torch.randn(q.shape, generator=g))
        graph.replay()
        o, lse = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(out[0], o) and torch.equal(out[1], lse), i
        assert torch.equal(eager["table"], graphed["table"]) and torch.equal(eager["lens"], graphed["lens"])
        for a, b in zip(eager["cache"], graphed["cache"]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_two_streams_at_once():
    made = [make([900, 2000], [n, n], 8, 2, 64, 128, torch.bfloat16, seed=20 + n) for n in (1, 24)]
    args, alone = [], []
    for n, (q, codes, scales, table, lens, cu) in zip((1, 24), made):
        args.append(((q.cuda(), device_cache(codes, scales), i32(table), i32(lens), i32(cu), 0.09), n))
        alone.append(K.paged_attention(*args[-1][0], max_q=n, return_lse=True))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s, (a, n) in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(K.paged_attention(*a, max_q=n, return_lse=True))
        torch.cuda.synchronize()
        for (o, lse), (wo, wl) in zip(got, alone):
            assert torch.equal(o, wo) and torch.equal(lse, wl)


def test_two_captured_graphs_replayed_side_by_side():
    # a prompt's piece and a decode step over long sequences, both with parts to join, each with its own workspace
    made = [make([2500, 4000], [n, n], 8, 2, 64, 128, torch.bfloat16, seed=30 + n) for n in (1, 24)]
    graphs, eager, out = [], [], []
    for n, (q, codes, scales, table, lens, cu) in zip((1, 24), made):
        args = (q.cuda(), device_cache(codes, scales), i32(table), i32(lens), i32(cu), 0.09)
        eager.append(K.paged_attention(*args, max_q=n, return_lse=True))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out.append(K.paged_attention(*args, max_q=n, return_lse=True))
        graphs.append((g, args))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(6):
        for o in out:
            o[0].zero_()
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (o, lse), (wo, wl) in zip(out, eager):
            assert torch.equal(o, wo) and torch.equal(lse, wl)


def test_many_sequences_and_a_long_prompt_together():
    # over 64 sequences (each lane scans several), prompts beside single tokens and empty ones
    rng = np.random.default_rng(5)
    lens = rng.integers(0, 200, 150)
    n = np.minimum(rng.integers(0, 2, 150), lens)
    n[[3, 70, 149]] = np.minimum([150, 37, 20], lens[[3, 70, 149]])
    for Hq, H, D in ((4, 2, 64), (2, 1, 128)):
        check_attention(list(lens), list(n), Hq, H, 32, D, max_q=int(max(n)), seed=1)
        check_attention(list(lens), list(np.minimum(n, 1)), Hq, H, 32, D, max_q=1, seed=2)
        check_attention(list(lens), list(np.minimum(n, 4)), Hq, H, 32, D, max_q=4, seed=3)


def dense_on_gpu(q, codes, scales, table, lens, cu, sm_scale, causal):
    """The 64-bit form with a whole (sequence, head) at a time, for sizes that the row-by-row one is too slow for."""
    T, Hq, D = q.shape
    H, P = codes.shape[2], codes.shape[3]
    values = torch.from_numpy(orc.E4M3).cuda()
    two = torch.from_numpy(np.ldexp(1.0, np.arange(-127, 129))).cuda()
    c, s, qd = torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), q.cuda().double()
    o, lse = torch.zeros(T, Hq, D, dtype=torch.float64, device="cuda"), torch.zeros(T, Hq, dtype=torch.float64, device="cuda")
    spread, reach = torch.zeros_like(o), torch.zeros_like(lse)
    for b in range(len(lens)):
        n, L = int(cu[b + 1] - cu[b]), int(lens[b])
        at = torch.from_numpy(table[b, :-(-L // P)]).cuda()
        hide = torch.arange(L, device="cuda") > torch.arange(L - n, L, device="cuda")[:, None] if causal else torch.zeros(n, L, dtype=torch.bool, device="cuda")
        for h in range(Hq):
            k, v = ((values[c[j][at, h * H // Hq].long()] * two[s[j][at, h * H // Hq]][:, None, None]).reshape(-1, D)[:L] for j in range(2))
            rows = slice(int(cu[b]), int(cu[b + 1]))
            x = (qd[rows, h] @ k.T * sm_scale).masked_fill(hide, -torch.inf)
            z = torch.logsumexp(x, 1)
            p = torch.exp(x - z[:, None])
            o[rows, h], spread[rows, h], lse[rows, h] = p @ v, p @ v.abs(), z / np.log(2.0)
            reach[rows, h] = (qd[rows, h].abs() @ k.abs().T).amax(1) * abs(sm_scale) / np.log(2.0)
    return tuple(x.cpu().numpy() for x in (o, lse, spread, reach))


@pytest.mark.parametrize("n,lens,Hq,H,D,causal", [
    ([1400, 700], [1400, 1500], 64, 64, 64, True), ([1100, 1], [1111, 300], 32, 16, 256, True),     # a workgroup for each row tile
    ([1900, 150], [1900, 4000], 32, 4, 128, True), ([900, 20], [2000, 3000], 8, 8, 128, False)])    # an even share of the steps
def test_prompts_of_many_row_tiles(n, lens, Hq, H, D, causal):
    q, codes, scales, table, lens, cu = make(lens, n, Hq, H, 64, D, torch.bfloat16, seed=D)
    o, lse = K.paged_attention(q.cuda(), device_cache(codes, scales), i32(table), i32(lens), i32(cu), D ** -0.5, max_q=max(n),
                               causal=causal, return_lse=True)
    compare(o, lse, dense_on_gpu(q, codes, scales, table, lens, cu, D ** -0.5, causal), max(lens), D, torch.bfloat16)


@pytest.mark.parametrize("a,b", [("ctx_lens", "lens"), ("new_lens", "lens"), ("free_start", "free_end"), ("block_table", "lens"),
                                 ("free_pages", "slot_map"), ("cu_new", "slot_map"), ("lens", "cu_new")])
def test_plan_refuses_outputs_over_other_arguments(a, b):
    make = lambda: dict(ctx_lens=i32([3, 0]), new_lens=i32([1, 1]), block_table=i32([[4, -1], [-1, -1]]), free_pages=i32([1, 2, 3]),
                        free_start=i32([0]), lens=i32([0, 0]), cu_new=i32([0, 0, 0]), slot_map=i32([0, 0, 0]), free_end=i32([0]))
    v = make()
    n = v[b].numel()
    whole = i32([0] * 8)
    v[a] = whole[:v[a].numel()].view(v[a].shape)
    v[b] = whole[v[a].numel() - 1:][:n]        # the last element of the one is the first of the other
    with pytest.raises(ValueError, match="overlap"):
        K.paged_plan_kernel[(2, )](*v.values(), PAGE_SIZE=4)
    v[b] = whole[v[a].numel():][:n].view(v[b].shape) if v[a].numel() + n <= 8 else i32([0] * n)
    K.paged_plan_kernel[(2, )](*v.values(), PAGE_SIZE=4)       # side by side


def test_plan_of_no_sequence_is_refused():
    with pytest.raises(ValueError):
        K.paged_plan(i32([]), i32([]), torch.empty(0, 3, **I32), i32([1]), 4, 2)


@pytest.mark.parametrize("P,width,B,n,kernel", [
    (16, 2**27 - 1, 1, 1, "any"),            # positions up to 2^31 - 16
    (16, 2**27 - 1, 1, 9, "any"),
    (8192, 2**18 - 1, 130, 1, "one"),        # 130 sequences of up to 2^24 units of 128 keys: each is one workgroup's
    (8192, 2**18 - 1, 66, 10, "rows"),       # the same for row tiles
])
def test_tables_of_nearly_31_bits(P, width, B, n, kernel):
    q, codes, scales, narrow, lens, cu = make([7 * b % 40 + n for b in range(B)], [n] * B, 4, 1, P, 128, torch.bfloat16)
    table = torch.full((B, width), -1, **I32)
    table[:, :narrow.shape[1]] = i32(narrow)
    cache = device_cache(codes, scales)
    o, lse = K.paged_attention(q.cuda(), cache, table, i32(lens), i32(cu), 0.09, max_q=n, return_lse=True)
    assert f"_{kernel}_" in rt.last_kernel_name()
    want = orc.attention(q.double().numpy(), codes[0], codes[1], scales[0], scales[1], narrow, lens, cu, 0.09, True)
    compare(o, lse, want, max(lens), 128, torch.bfloat16)


def test_a_page_of_more_elements_than_31_bits_is_refused():
    n = ctypes.c_size_t()
    c = rt.pack_paged_cache(1, 1, 1, 1, *([0] * 10), 1, 1, 2**25, 64)
    assert rt.load().tt_paged_attn_workspace(1, 1, 1, 1, 1, c, ctypes.byref(n)) == rt.RT_ERR_UNSUPPORTED
    c = rt.pack_paged_cache(1, 1, 1, 1, *([0] * 10), 1, 1, 2**25 - 1, 64)
    assert rt.load().tt_paged_attn_workspace(1, 1, 1, 1, 1, c, ctypes.byref(n)) == rt.RT_OK


@pytest.mark.parametrize("P,D", [(34087042, 63), (2**31 // 33, 33), (2**31 // 7, 7), (2**31 - 63, 1)])
def test_a_page_whose_last_step_of_64_elements_would_pass_31_bits_is_refused(P, D):
    # P * D is one of the last 63 values below 2^31; the largest page size below those is taken
    n = ctypes.c_size_t()
    ask = lambda P: rt.init(0).tt_paged_attn_workspace(1, 1, 1, 1, 1, rt.pack_paged_cache(1, 1, 1, 1, *([0] * 10), 1, 1, P, D), ctypes.byref(n))
    assert 2**31 - 64 < P * D < 2**31 and ask(P) == rt.RT_ERR_UNSUPPORTED
    assert ask((2**31 - 64) // D) == rt.RT_OK


def compare_far(o, lse, want, n, D, dtype, apart):
    """As `compare` (a weight is off by at most 2^-11 of itself, so a channel by 2^-11 of its own sum), without that one's absolute
    term: only fp16 results, which can be subnormal, have half a step of 2^-24.  V's exponents enter scores as offsets of magnitude up to `apart`."""
    wo, wl, spread, reach = want
    o, lse = o.cpu().double().numpy(), lse.cpu().double().numpy()
    ds = (D + 5) * U * reach + (apart + 54) * U
    rel = 2 * (np.log(2.0) * ds + 2 * U + n * U)
    tol = spread * (2.0**-11 + rel[..., None]) + torch.finfo(dtype).eps / 2 * (np.abs(wo) + spread * 2.0**-10)
    tol += 2.0**-25 if dtype is torch.float16 else 0.0
    assert np.isfinite(wl).all() and (np.abs(o - wo) <= tol).all(), (np.abs(o - wo) / tol).max()
    ltol = ds + (n + 4) * U / np.log(2.0) + 2 * U * np.abs(wl) + 64 * U
    assert (np.abs(lse - wl) <= ltol).all(), (np.abs(lse - wl) / ltol).max()


@pytest.mark.parametrize("n,Hq,H,D,kernel", [(1, 4, 2, 64, "one"), (1, 4, 2, 128, "one"), (1, 32, 1, 64, "one"), (1, 32, 1, 128, "one"),
                                             (1, 2, 2, 256, "one"), (5, 4, 2, 64, "few"), (16, 4, 2, 128, "few"), (8, 4, 2, 256, "few"),
                                             (30, 4, 2, 64, "rows"), (30, 8, 2, 128, "rows"), (30, 4, 2, 256, "rows"), (3, 4, 2, 40, "any")])
@pytest.mark.parametrize("apart", [7, 12, 13, 20, 30, 60, 100])
def test_channels_that_only_pages_of_a_small_scale_fill(n, Hq, H, D, kernel, apart):
    # half of the channels are zeros in every page of the large scale: what the small pages hold there is the result
    fp16 = apart <= 20
    dtype, top = (torch.float16, 133) if fp16 else (torch.bfloat16, 160)
    q, codes, scales, table, lens, cu = make([1100, 90], [n, n], Hq, H, 16, D, dtype, seed=apart + n, q_scale=0.5)
    rng = np.random.default_rng(apart)
    small = rng.random(scales[1].shape) < 0.5
    small[table[1, 0]], small[table[1, 1]] = False, True
    scales[1] = np.where(small, top - apart, top)
    codes[1, :, :, :, :D // 2] = np.where(~small[..., None, None] & (codes[1, :, :, :, :D // 2] != 0x7F), 0, codes[1, :, :, :, :D // 2])
    o, lse = K.paged_attention(q.cuda(), device_cache(codes, scales), i32(table), i32(lens), i32(cu), 0.09, max_q=n, return_lse=True)
    assert f"_{kernel}_" in rt.last_kernel_name() or "_join_" in rt.last_kernel_name()
    want = orc.attention(q.double().numpy(), codes[0], codes[1], scales[0], scales[1], table, lens, cu, 0.09, True)
    compare_far(o, lse, want, 1100, D, dtype, apart)
    assert (want[2][:, :, :D // 2] > 0).all()


@pytest.mark.parametrize("n,Hq,H,D", [(1, 4, 2, 64), (1, 4, 2, 128), (1, 2, 2, 256), (5, 4, 2, 128), (30, 8, 2, 128), (30, 4, 2, 64), (3, 4, 2, 40)])
@pytest.mark.parametrize("top", [127, 135, 160, 200])
def test_pages_of_zeros_beside_any_others(n, Hq, H, D, top):
    # a page of zeros has the smallest scale there is; its keys count in the sum of probabilities like any others
    q, codes, scales, table, lens, cu = make([1100, 90, 40], [n, n, n], Hq, H, 16, D, torch.bfloat16, seed=top + n)
    rng = np.random.default_rng(top)
    zero = rng.random(scales[1].shape) < 0.5
    zero[table[1, :3]] = True
    zero[table[0, 20:60]] = True            # whole shares of a long sequence
    zero[table[2, :3]] = True               # nothing but zeros
    scales[1] = np.where(zero, orc.MIN_SCALE, top)
    codes[1] = np.where(zero[..., None, None] & (codes[1] != 0x7F), 0, codes[1])
    o, lse = K.paged_attention(q.cuda(), device_cache(codes, scales), i32(table), i32(lens), i32(cu), 0.09, max_q=n, return_lse=True)
    want = orc.attention(q.double().numpy(), codes[0], codes[1], scales[0], scales[1], table, lens, cu, 0.09, True)
    compare_far(o, lse, want, 1100, D, torch.bfloat16, top - orc.MIN_SCALE)


@pytest.mark.parametrize("n,Hq,H,D", [(1, 4, 2, 64), (1, 4, 2, 128), (1, 2, 2, 256), (5, 4, 2, 128), (8, 4, 2, 256), (30, 8, 2, 128), (30, 4, 2, 64),
                                      (3, 4, 2, 40)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sm_scale", [0.1, -0.1])
def test_a_query_whose_scores_all_are_minus_infinity_gives_what_one_without_a_key_does(n, Hq, H, D, dtype, sm_scale):
    q, codes, scales, table, lens, cu = make([100, 0, 700], [n, n, n], Hq, H, 16, D, dtype, seed=D)
    at = codes[0, ..., 0] != 0x7F
    codes[0, ..., 0][at] = 0x38             # component 0 of every key is 1 times its scale
    sign = -np.sign(sm_scale)
    for row, x in ((0, sign), (2 * n, sign), (3 * n - 1, -sign)):
        q[row, 1, 0] = x * float("inf")
    o, lse = K.paged_attention(q.cuda(), device_cache(codes, scales), i32(table), i32(lens), i32(cu), sm_scale, max_q=n, return_lse=True)
    nan, none = torch.zeros(3 * n, Hq, dtype=torch.bool), torch.zeros(3 * n, Hq, dtype=torch.bool)
    none[n:2 * n], none[0, 1], none[2 * n, 1] = True, True, True
    nan[3 * n - 1, 1], none[3 * n - 1, 1] = True, False     # every score is +inf
    o, lse = o.cpu(), lse.cpu()
    assert torch.equal(torch.isnan(o).all(-1), nan) and torch.equal(torch.isnan(o).any(-1), nan) and torch.equal(torch.isnan(lse), nan)
    assert torch.equal(torch.isneginf(lse), none) and (o[none] == 0).all()


def test_more_workgroups_than_a_launch_takes_are_refused():
    # (all of it in memory that exists: no token has a slot, no row a sequence)
    H, T = 64, 2**19
    cache = K.paged_cache(1, H, 1, 16)
    x = torch.zeros(T + 1, H, 1, dtype=torch.bfloat16, device="cuda")
    none = torch.full((T + 1, ), -1, **I32)
    with pytest.raises(NotImplementedError, match="grid"):
        K.paged_write(x, x, none, cache)                    # 2^24 + 16 workgroups
    K.paged_write(x[:-2], x[:-2], none[:-2], cache)
    T = 2**26
    q = torch.zeros(T, 1, 1, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(NotImplementedError, match="grid"):
        K.paged_attention(q, K.paged_cache(1, 1, 1, 16), i32([[0]]), i32([0]), i32([0, 0]), 1.0)


def test_more_pairs_of_sequence_and_head_than_a_launch_takes():
    H, B = 17, 2**20                                        # 2^24 + 2^20 pairs: the kernel for any shape, a workgroup for each row
    q, codes, scales, table, lens, cu = make([13, 9], [1, 1], H, H, 16, 64, torch.bfloat16)
    wide = torch.full((B, 1), -1, **I32)
    many, ends = torch.zeros(B, **I32), torch.zeros(B + 1, **I32)
    for i, b in ((0, 5), (1, B - 1)):
        wide[b, 0], many[b] = int(table[i, 0]), int(lens[i])
        ends[b + 1:] += 1
    o, lse = K.paged_attention(q.cuda(), device_cache(codes, scales), wide, many, ends, 0.1, max_q=1, return_lse=True)
    want = orc.attention(q.double().numpy(), codes[0], codes[1], scales[0], scales[1], table, lens, cu, 0.1, True)
    compare(o, lse, want, 13, 64, torch.bfloat16)


def test_rt_launch_refuses_a_dimension_of_more_threads_than_32_bits_count():
    lib, m, k = rt.init(0), ctypes.c_void_p(), ctypes.c_void_p()
    rt.check(lib.rt_builtin_module(b"paged", ctypes.byref(m)))
    rt.check(lib.rt_get_kernel(m, b"paged_plan", ctypes.byref(k)))
    three = lambda *v: (ctypes.c_uint32 * 3)(*v)
    for grid, block in (((2**24, 1, 1), (256, 1, 1)), ((2**32 - 1, 1, 1), (2, 1, 1)), ((1, 2**31, 1), (1, 2, 1)), ((1, 1, 2**26), (1, 1, 64))):
        assert lib.rt_launch(k, three(*grid), three(*block), 0, None, None, 0) == rt.RT_ERR_UNSUPPORTED


# ---- the kernel for a few queries of a sequence, and it beside the one for many, where masks and codes are special ----
FEW = [(5, 4, 2, 64), (16, 4, 2, 64), (5, 4, 2, 128), (16, 4, 2, 128), (8, 4, 2, 256), (3, 33, 3, 64), (3, 30, 3, 64)]   # n, Hq, H, D


def few_or_rows(n, Hq, H, D):
    """Queries times group up to 32 rows (16 at head dim 256) are the few-queries kernel's."""
    return "_few_" if n * Hq // H <= (16 if D == 256 else 32) else "_rows_"


def attend(q, codes, scales, table, lens, cu, sm_scale=0.1, **kw):
    return K.paged_attention(q.cuda(), device_cache(codes, scales), i32(table), i32(lens), i32(cu), sm_scale, return_lse=True, **kw)


def oracle_of(q, codes, scales, table, lens, cu, sm_scale=0.1, causal=True):
    return orc.attention(q.double().numpy(), codes[0], codes[1], scales[0], scales[1], table, lens, cu, sm_scale, causal)


@pytest.mark.parametrize("n,Hq,H,D", FEW)
@pytest.mark.parametrize("causal", [True, False])
def test_few_pages_outside_the_cache_count_as_absent(n, Hq, H, D, causal):
    q, codes, scales, table, lens, cu = make([300, 150, 64, 4000], [n] * 4, Hq, H, 32, D, torch.bfloat16, seed=40)
    table[0, 3], table[0, 5], table[1, 0], table[2, :], table[3, 60] = -1, 10**6, codes.shape[1], -1, -5
    o, lse = attend(q, codes, scales, table, lens, cu, max_q=n, causal=causal)
    compare(o, lse, oracle_of(q, codes, scales, table, lens, cu, causal=causal), 4000, D, torch.bfloat16)
    short = (q[:3 * n], codes, scales, table[:3, :12].copy(), lens[:3], cu[:4])
    o, lse = attend(*short, max_q=n, causal=causal)
    assert few_or_rows(n, Hq, H, D) in rt.last_kernel_name()
    compare(o, lse, oracle_of(*short, causal=causal), 300, D, torch.bfloat16)


@pytest.mark.parametrize("n,Hq,H,D", FEW)
def test_few_lengths_past_the_table_and_below_zero(n, Hq, H, D):
    q, codes, scales, table, lens, cu = make([96, 96], [n, n], Hq, H, 32, D, torch.float16, seed=41)
    table = np.ascontiguousarray(table[:, :3])
    o, lse = attend(q, codes, scales, table, [96, 2**31 - 1], cu, max_q=n)
    assert few_or_rows(n, Hq, H, D) in rt.last_kernel_name()
    compare(o, lse, oracle_of(q, codes, scales, table, [96, 96], cu), 96, D, torch.float16)
    o, lse = attend(q, codes, scales, table, [96, -5], cu, max_q=n)
    assert (o[n:] == 0).all() and torch.isneginf(lse[n:]).all()
    compare(o[:n], lse[:n], tuple(x[:n] for x in oracle_of(q, codes, scales, table, [96, 96], cu)), 96, D, torch.float16)


@pytest.mark.parametrize("n,Hq,H,D", FEW)
def test_few_strided_queries_and_results_and_rows_of_no_sequence(n, Hq, H, D):
    q, codes, scales, table, lens, cu = make([90, 300], [n, n], Hq, H, 32, D, torch.bfloat16, seed=42)
    rows = 2 * n + 7
    wide = torch.full((rows, Hq * D + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    qv = wide[:, :Hq * D].view(rows, Hq, D)
    qv[:2 * n] = q.cuda()
    want = oracle_of(q, codes, scales, table, lens, cu)
    for off in (0, 8, 3):       # 3: rows off the alignment the fast kernels need
        hold = torch.full((Hq, rows, D + off), 7.0, dtype=torch.bfloat16, device="cuda")
        out = hold[:, :, off:].transpose(0, 1)
        o, lse = K.paged_attention(qv, device_cache(codes, scales), i32(table), i32(lens), i32(cu), 0.1, max_q=n, return_lse=True, out=out)
        assert (few_or_rows(n, Hq, H, D) if off != 3 else "_any_") in rt.last_kernel_name()
        compare(o[:2 * n], lse[:2 * n], want, 300, D, torch.bfloat16)
        assert (hold[:, :, :off] == 7).all() and (out[2 * n:] == 7).all()


def check_nan(lens, n_q, Hq, H, P, D, bad, causal, apart=0, kernel=None, dtype=torch.bfloat16):
    """bad: (sequence, position, 0 for K or 1 for V): one NaN code, in channel 5 of head 0."""
    q, codes, scales, table, lens, cu = make(lens, n_q, Hq, H, P, D, dtype, seed=43)
    if apart:
        scales[1] = np.where(np.random.default_rng(3).random(scales[1].shape) < 0.5, 130 - apart, 130)
        scales[1][table[0, 0]], scales[1][table[0, 1]] = 130, 130 - apart
    for b, pos, j in bad:
        codes[j, table[b, pos // P], 0, pos % P, 5] = 0x7F if pos % 2 else 0xFF
    o, lse = attend(q, codes, scales, table, lens, cu, max_q=int(max(n_q)), causal=causal)
    if kernel:
        assert kernel in rt.last_kernel_name()
    clean = codes.copy()
    clean[:, table[table >= 0]] = np.where((clean[:, table[table >= 0]] & 127) == 127, 0, clean[:, table[table >= 0]])
    wo = oracle_of(q, clean, scales, table, lens, cu, causal=causal)[0]
    o = o.double().cpu().numpy()
    for b, L in enumerate(lens):
        for i in range(n_q[b]):
            last = L - n_q[b] + i if causal else L - 1
            hits = {j for bb, pos, j in bad if bb == b and pos <= last}
            for h in range(Hq):
                row = np.isnan(o[cu[b] + i, h])
                if h * H // Hq or not hits:
                    assert not row.any(), (b, i, h)
                elif 0 in hits:
                    assert row.all(), (b, i, h)
                else:
                    assert row[5] and not np.delete(row, 5).any(), (b, i, h)
                if not hits:        # (the oracle's rows that see no bad key: compared roughly, a NaN that was counted as a key would show)
                    assert np.allclose(o[cu[b] + i, h], wo[cu[b] + i, h], rtol=0.05, atol=0.02 * np.abs(wo[cu[b] + i, h]).max())


@pytest.mark.parametrize("n,Hq,H,D", FEW)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("apart", [0, 40])
def test_few_nan_codes_reach_the_queries_that_attend_them_only(n, Hq, H, D, causal, apart):
    # (sequence 1: NaN in V at the last keys, which only the last queries attend; sequence 2: in K too; 3: none)
    bad = [(0, 30, 1), (1, 69, 1), (1, 68, 1), (1, 66, 1), (2, 97, 1), (2, 99, 0)]
    check_nan([60, 70, 100, 33], [n] * 4, Hq, H, 16, D, bad, causal, apart, few_or_rows(n, Hq, H, D))


@pytest.mark.parametrize("Hq,H,D", [(4, 2, 64), (8, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("apart", [0, 40])
def test_nan_codes_where_few_and_many_queries_share_a_launch(Hq, H, D, causal, apart):
    bad = [(0, 97, 1), (0, 30, 1), (1, 69, 1), (2, 130, 1), (2, 199, 1), (3, 0, 0)]
    check_nan([100, 70, 200, 40, 90], [4, 1, 150, 3, 60], Hq, H, 16, D, bad, causal, apart, "_rows_")


@pytest.mark.parametrize("n_q", [[1, 1, 1], [5, 3, 4], [60, 40, 90], [60, 1, 4]])
@pytest.mark.parametrize("apart", [0, 40])
def test_results_over_the_queries(n_q, apart):
    # out may be q itself: a row is read before it is written, also where a second pass follows
    q, codes, scales, table, lens, cu = make([100, 2000, 90], n_q, 8, 2, 16, 128, torch.bfloat16, seed=44)
    if apart:
        scales[1] = np.where(np.random.default_rng(4).random(scales[1].shape) < 0.5, 130 - apart, 130)
    args = (device_cache(codes, scales), i32(table), i32(lens), i32(cu), 0.1)
    o, lse = K.paged_attention(q.cuda(), *args, max_q=max(n_q), return_lse=True)
    x = q.cuda()
    o2, lse2 = K.paged_attention(x, *args, max_q=max(n_q), return_lse=True, out=x)
    assert o2 is x and torch.equal(o, o2) and torch.equal(lse, lse2)


# ---- the write's infinities and NaN, in runs of every kind ----
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,P", [(64, 64), (128, 64), (256, 64), (64, 256), (128, 256), (256, 256), (40, 64)])
def test_write_of_special_values_in_runs_that_wavefronts_share(dtype, D, P):
    H = 2
    codes, scales = filled(9, H, P, D, seed=D + P)
    spec = [(0, 0, P), (1, 0, P), (2, 0, P), (3, 7, P - 7), (4, 0, P), (5, P // 2, P // 2), (6, 0, P - 1), (7, 3, 1)]
    slots, g = runs(spec, P), torch.Generator().manual_seed(D * P)
    at = np.cumsum([0] + [n for _, _, n in spec])
    x = torch.randn(2, len(slots), H, D, generator=g)
    x[:, at[3]:at[4]] *= 3e4 if dtype is torch.bfloat16 else 1e3       # the scale grows behind earlier rows
    x[:, at[5]:at[6]] *= 1e-3                                          # and here it does not
    x = x.to(dtype)
    inf, nan = float("inf"), float("nan")
    x[0, at[0] + P // 2 + 3, 0, 5], x[1, at[0] + P - 1, 1, D - 1] = inf, -inf      # one wavefront's rows only; runs 1 and 6 have none
    x[:, at[2]:at[3], 0, ::3], x[0, at[2]:at[3], 1] = nan, inf                     # nothing finite in K's head 1
    x[0, at[3] + 1, 0, 0], x[1, at[3], 0, 1] = nan, inf
    x[:, at[4]:at[5]] = torch.finfo(dtype).max
    x[1, at[4] + P // 4, 1, 2] = -inf
    x[:, at[5]] = -inf
    x[0, at[7], 1, 3], x[1, at[7]] = inf, nan
    check_write(x.cuda(), slots, codes, scales)


def test_plan_of_sequences_taken_back():
    # (drafts that were rejected: the entries behind the shorter length are replaced, the page that it ends in stays)
    table = np.array([[5, 6, 7, -1], [8, 9, -1, -1], [3, 2, 1, -1]])
    run_plan([5, 4, 0], [4, 3, 5], table, np.arange(20, 30), 4, 12)


@pytest.mark.parametrize("Hq,H,D", [(4, 2, 64), (2, 1, 128)])
@pytest.mark.parametrize("most", [1, 4, 150])
def test_many_sequences_of_scales_far_apart(Hq, H, D, most):
    # over 64 sequences, each lane of a scan several; some workgroups meet near and far ones
    rng = np.random.default_rng(6)
    lens = rng.integers(0, 200, 150)
    n = np.minimum(rng.integers(0, 2, 150), lens)
    n[[3, 70, 149]] = np.minimum([150, 37, 20], lens[[3, 70, 149]])
    n = np.minimum(n, most)
    q, codes, scales, table, lens, cu = make(list(lens), list(n), Hq, H, 32, D, torch.bfloat16, seed=7)
    far = rng.random(scales[1].shape) < 0.2
    scales[1] = np.where(far, 60, 130)
    o, lse = attend(q, codes, scales, table, lens, cu, max_q=most)
    compare(o, lse, oracle_of(q, codes, scales, table, lens, cu), 200, D, torch.bfloat16)
