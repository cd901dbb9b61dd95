"""Plain 64-bit restatement of the paged 8-bit cache: plan, write and attention, sequence by sequence (test infrastructure).

Codes are e4m3 bytes (uint8 arrays), scales exponents (code s stands for 2^(s - 127)); everything else is float64."""
import numpy as np

MIN_SCALE = 27


def _e4m3_values() -> np.ndarray:
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0**-9, (8 + m) * 2.0**(e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >> 7, -v, v)


E4M3 = _e4m3_values()
_POS = E4M3[:127]                                   # ascending magnitudes of codes 0 .. 126
_MID = (_POS[1:] + _POS[:-1]) / 2


def encode(x: np.ndarray) -> np.ndarray:
    """Round to nearest, ties to the even code; beyond 448 saturates, NaN stays NaN."""
    a = np.abs(x)
    lo = np.searchsorted(_MID, a, side="left")      # a tie goes to the lower neighbour here
    tie = (lo < 126) & (a == _MID[np.minimum(lo, 125)])
    code = np.where(tie & (lo % 2 == 1), lo + 1, lo)
    code = np.where(np.isnan(x), 127, code)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def scale_of(amax: float) -> int:
    """Code of the smallest power of two 2^e with amax <= 448 * 2^e."""
    s = MIN_SCALE
    while amax > 448.0 * 2.0**(s - 127):
        s += 1
    return s


def plan(ctx, new, table, free, P, T, start=0):
    """-> (table, lens, cu, slots, free_end)."""
    table = table.copy()
    width = table.shape[1] * P
    slots, lens, cu, used = np.full(T, -1, np.int64), [], [0], start
    for b, (a, n) in enumerate(zip(ctx, new)):
        a = min(max(int(a), 0), width)
        n = min(max(int(n), 0), width - a, T - cu[-1])
        for i in range(n):
            blk, row = divmod(a + i, P)
            if blk >= -(-a // P) and row == 0:
                table[b, blk] = free[used] if 0 <= used < len(free) else -1
                used += 1
            if table[b, blk] >= 0:
                slots[cu[-1] + i] = int(table[b, blk]) * P + row
        lens.append(a + n)
        cu.append(cu[-1] + n)
    return table, np.array(lens), np.array(cu), slots, used


def write(x, slots, codes, scales):
    """x [T, H, D] into codes [pages, H, P, D], scales [pages, H], in place."""
    pages, H, P, _ = codes.shape
    t = 0
    while t < len(slots):
        slot, n = int(slots[t]), 1
        if not 0 <= slot < pages * P:
            t += 1
            continue
        page, row = divmod(slot, P)
        while t + n < len(slots) and row + n < P and slots[t + n] == slot + n:
            n += 1
        for h in range(H):
            run = x[t:t + n, h]
            fine = np.abs(run[np.isfinite(run)])
            s = scale_of(fine.max() if fine.size else 0.0)
            if row:
                old = int(scales[page, h])
                if s > old:
                    codes[page, h, :row] = encode(E4M3[codes[page, h, :row]] * 2.0**(old - s))
                s = max(s, old)
            codes[page, h, row:row + n] = encode(run * 2.0**(127 - s))
            scales[page, h] = s
        t += n


def attention(q, kc, vc, ks, vs, table, lens, cu, sm_scale, causal):
    """q [T, Hq, D] -> (o, lse in base 2, spread, reach): spread = sum p |v| / l bounds what a rounding of p or v costs o;
    reach = the largest sum |q| |k| |sm_scale| log2(e) of a row bounds what a rounding of the products costs a score.
    Rows outside every sequence are NaN."""
    pages, H, P, D = kc.shape
    T, Hq, _ = q.shape
    o, spread = np.full((T, Hq, D), np.nan), np.full((T, Hq, D), np.nan)
    lse, reach = np.full((T, Hq), np.nan), np.zeros((T, Hq))
    for b in range(len(lens)):
        n, L = int(cu[b + 1] - cu[b]), int(lens[b])
        key = np.arange(L)
        at, row = table[b, key // P], key % P
        here = (at >= 0) & (at < pages)
        key, at, row = key[here], at[here], row[here]
        for h in range(Hq):
            hk = h * H // Hq
            k = E4M3[kc[at, hk, row]] * 2.0**(ks[at, hk].astype(np.float64) - 127)[:, None]
            v = E4M3[vc[at, hk, row]] * 2.0**(vs[at, hk].astype(np.float64) - 127)[:, None]
            for i in range(n):
                t = cu[b] + i
                sees = key <= (L - n + i if causal else L - 1)
                s = k[sees] @ q[t, h] * sm_scale
                if (s == -np.inf).all():            # also where it sees no key
                    o[t, h], lse[t, h], spread[t, h] = 0.0, -np.inf, 0.0
                    continue
                m = s.max()
                p = np.exp(s - m)
                l = p.sum()
                o[t, h], spread[t, h] = p @ v[sees] / l, p @ np.abs(v[sees]) / l
                lse[t, h] = (m + np.log(l)) / np.log(2.0)
                reach[t, h] = (np.abs(k[sees]) @ np.abs(q[t, h])).max() * abs(sm_scale) / np.log(2.0)
    return o, lse, spread, reach
