"""The 64-bit restatement of the paged cache against closed forms (CPU)."""
import numpy as np
import torch

from oracle import paged as orc


def test_e4m3_matches_torchs_type():
    x = torch.cat([torch.randn(20000, dtype=torch.float64) * s for s in (1e-3, 0.05, 1.0, 100.0)]).clamp(-448, 448)
    x = torch.cat([x, torch.from_numpy(orc.E4M3[:127].copy()), torch.from_numpy(orc._MID.copy()), torch.zeros(1, dtype=torch.float64)])
    # fp32 inputs: torch rounds from fp32, which holds every midpoint exactly
    x = x.float()
    assert np.array_equal(orc.encode(x.double().numpy()), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert orc.encode(np.array([np.nan, np.inf, -np.inf, 500.0])).tolist() == [127, 126, 254, 126]


def test_scale_is_the_smallest_that_holds():
    for amax, s in ((448.0, 127), (448.1, 128), (224.0, 126), (1.75, 119), (1.0, 119), (0.0, orc.MIN_SCALE)):
        assert orc.scale_of(amax) == s


def test_plan_closed_form():
    table = np.array([[5, 6, -1, -1], [-1] * 4, [7, -1, -1, -1]])
    t, lens, cu, slots, end = orc.plan([6, 0, 3], [3, 5, 0], table, np.array([9, 8, 3, 2]), 4, 10)
    assert t.tolist() == [[5, 6, 9, -1], [8, 3, -1, -1], [7, -1, -1, -1]]
    assert lens.tolist() == [9, 5, 3] and cu.tolist() == [0, 3, 8, 8] and end == 3
    assert slots.tolist() == [26, 27, 36, 32, 33, 34, 35, 12, -1, -1]


def test_write_appends_equal_one_write_of_all():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((8, 2, 16)) * np.array([1, 1, 30, 1, 200, 1, 1, 1])[:, None, None]
    a = np.full((1, 2, 8, 16), 0x7F, np.uint8)
    b, sa, sb = a.copy(), np.zeros((1, 2), np.int64), np.zeros((1, 2), np.int64)
    orc.write(x, np.arange(8), a, sa)
    for t in range(8):
        orc.write(x[t:t + 1], np.array([t]), b, sb)
    assert np.array_equal(sa, sb)
    # rounding twice moves a code by at most one step where it has become subnormal, and not at all elsewhere
    va, vb = orc.E4M3[a], orc.E4M3[b]
    assert np.abs(va - vb).max() <= 2.0**-9 and np.array_equal(va[np.abs(va) >= 2.0**-5], vb[np.abs(va) >= 2.0**-5])


def test_attention_of_equal_keys_is_the_mean():
    vc = orc.encode(np.random.default_rng(1).standard_normal((3, 1, 4, 8)) * 50)
    kc = np.zeros_like(vc)
    s = np.full((3, 1), 127)
    o, lse, _, _ = orc.attention(np.ones((2, 2, 8)), kc, vc, s, s, np.array([[2, 0, -1]]), [7], [0, 2], 1.0, True)
    v = orc.E4M3[np.concatenate([vc[2, 0], vc[0, 0]])]
    assert np.allclose(o[0, 0], v[:6].mean(0)) and np.allclose(o[1, 1], v[:7].mean(0)) and np.allclose(lse[:, 0], np.log2([6, 7]))
