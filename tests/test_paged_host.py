"""Host side of the paged 8-bit cache, no GPU: what the launch functions hand to the C ABI, and what they refuse."""
import json
import struct

import pytest
import torch

from triton_tenstorrent_amd import kernels as K, runtime as rt
from triton_tenstorrent_amd.backend import compiler, driver as drv

E4M3, BF16, I32, U8 = torch.float8_e4m3fn, torch.bfloat16, torch.int32, torch.uint8


class Fake:
    """Looks like a tensor on GPU ``device``; never dereferenced."""

    def __init__(self, shape, dtype, ptr=0x7f0000000000, device=0, strides=None):
        self.shape, self.dtype, self._ptr, self._device = torch.Size(shape), dtype, ptr, device
        st, acc = [], 1
        for d in reversed(self.shape):
            st.insert(0, acc)
            acc *= d
        self._st = tuple(strides or st)
        self.is_cuda = device >= 0

    def data_ptr(self):
        return self._ptr

    def stride(self):
        return self._st

    def get_device(self):
        return self._device


class Recording:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def fn(*args):
            self.calls.append((name, args))
            return 0
        return fn


@pytest.fixture
def lib(monkeypatch):
    rec = Recording()
    monkeypatch.setattr(rt, "init", lambda device=0: rec)
    monkeypatch.setattr(drv.TTDriver, "get_current_device", lambda self: 0)
    monkeypatch.setattr(drv.TTDriver, "get_current_stream", lambda self, d=None: 0x1234)
    for k in (K.paged_plan_kernel, K.paged_write_kernel, K.paged_attn_kernel):
        k._cache.clear()
        k._plan = None
    return rec


def plan_args(**kw):
    a = dict(ctx_lens=Fake((4, ), I32), new_lens=Fake((4, ), I32), block_table=Fake((4, 9), I32, strides=(12, 1)),
             free_pages=Fake((30, ), I32), free_start=None, lens=Fake((4, ), I32), cu_new=Fake((5, ), I32),
             slot_map=Fake((100, ), I32), free_end=Fake((1, ), I32))
    a.update(kw)
    return list(a.values())


def cache(pages=20, H=2, P=16, D=64, dtype=E4M3):
    return [Fake((pages, H, P, D), dtype, ptr=0x1000), Fake((pages, H, P, D), dtype, ptr=0x2000), Fake((pages, H), U8, ptr=0x3000),
            Fake((pages, H), U8, ptr=0x4000)]


def attn_args(c=None, **kw):
    c = c or cache()
    a = dict(q=Fake((6, 8, 64), BF16), k=c[0], v=c[1], ks=c[2], vs=c[3], table=Fake((3, 5), I32), lens=Fake((3, ), I32),
             cu_q=Fake((4, ), I32), out=Fake((6, 8, 64), BF16), lse=None, workspace=None, sm_scale=0.5, max_q=4)
    a.update(kw)
    return list(a.values())


def test_plan_hands_over_sizes_and_strides(lib):
    K.paged_plan_kernel[(4, )](*plan_args(), PAGE_SIZE=16)
    name, a = lib.calls[-1]
    assert name == "tt_paged_plan" and a[3:6] == (12, 4, 9) and a[7:11] == (30, None, 16, 100) and list(a[15]) == [4, 1, 1]
    K.paged_plan_kernel[(4, )](*plan_args(free_start=Fake((1, ), I32, ptr=0x77)), PAGE_SIZE=16)
    assert lib.calls[-1][1][8] == 0x77


def test_write_hands_over_the_cache(lib):
    k = Fake((7, 2, 64), BF16, strides=(500, 64, 1))
    K.paged_write_kernel[(7, )](k, Fake((7, 2, 64), BF16), Fake((7, ), I32), *cache())
    name, a = lib.calls[-1]
    assert name == "tt_paged_write" and struct.unpack("=2q", a[2]) == (500, 64) and a[5] == 7 and a[7] == rt.TT_BF16
    c = struct.unpack("=4Q10q4i", a[6])
    assert c[:4] == (0x1000, 0x2000, 0x3000, 0x4000) and c[4:10] == (2048, 1024, 64) * 2 and c[10:14] == (2, 1, 2, 1)
    assert c[14:] == (20, 2, 16, 64)


@pytest.mark.parametrize("max_q", [1, 4])      # 1 is folded into the specialisation
def test_attention_hands_over_its_arguments(lib, max_q):
    K.paged_attn_kernel[(6, 8)](*attn_args(max_q=max_q), CAUSAL=True)
    name, a = lib.calls[-1]
    assert name == "tt_paged_attn" and a[4:7] == (5, 3, 5) and a[9:15] == (6, 8, max_q, 0.5, True, rt.TT_BF16)
    assert a[17:20] == (None, None, 0) and list(a[20]) == [6, 8, 1]


REFUSED = [
    ("plan", dict(ctx_lens=Fake((3, ), I32))), ("plan", dict(cu_new=Fake((4, ), I32))), ("plan", dict(lens=Fake((4, ), torch.int64))),
    ("plan", dict(block_table=Fake((4, 9), I32, strides=(1, 4)))), ("plan", dict(block_table=Fake((4, ), I32))),
    ("plan", dict(free_pages=Fake((30, ), I32, device=1))), ("plan", dict(slot_map=Fake((100, ), I32, device=-1))),
    ("plan", dict(free_end=Fake((2, ), I32))), ("plan", dict(new_lens=3)),
    ("attn", dict(q=Fake((6, 8, 64), torch.float32))), ("attn", dict(q=Fake((6, 7, 64), BF16), out=Fake((6, 7, 64), BF16))),
    ("attn", dict(q=Fake((6, 8, 32), BF16), out=Fake((6, 8, 32), BF16))), ("attn", dict(out=Fake((6, 8, 64), torch.float16))),
    ("attn", dict(out=Fake((5, 8, 64), BF16))), ("attn", dict(q=Fake((6, 8, 64), BF16, strides=(512, 1, 8)))),
    ("attn", dict(cu_q=Fake((3, ), I32))), ("attn", dict(lens=Fake((3, ), torch.int64))), ("attn", dict(table=Fake((3, 5), torch.int64))),
    ("attn", dict(lse=Fake((6, 8), BF16))), ("attn", dict(lse=Fake((8, 6), torch.float32))),
    ("attn", dict(lse=Fake((6, 8), torch.float32, strides=(9, 1)))), ("attn", dict(workspace=Fake((64, ), torch.float32))),
    ("attn", dict(q=Fake((6, 8, 64), BF16, device=1))), ("attn", dict(c=cache(dtype=torch.int8))),
    ("attn", dict(v=Fake((20, 2, 16, 32), E4M3))), ("attn", dict(ks=Fake((20, 3), U8))), ("attn", dict(vs=Fake((20, 2), torch.float32))),
]


@pytest.mark.parametrize("which,change", REFUSED)
def test_refusals(lib, which, change):
    with pytest.raises(rt.InvalidLaunch):
        if which == "plan":
            K.paged_plan_kernel[(4, )](*plan_args(**change), PAGE_SIZE=16)
        else:
            K.paged_attn_kernel[(6, 8)](*attn_args(**change), CAUSAL=True)
    assert not lib.calls


def test_write_refusals(lib):
    ok = dict(k=Fake((7, 2, 64), BF16), v=Fake((7, 2, 64), BF16), slots=Fake((7, ), I32))
    for change in (dict(k=Fake((7, 2, 64), torch.float32)), dict(v=Fake((7, 2, 64), torch.float16)), dict(v=Fake((6, 2, 64), BF16)),
                   dict(k=Fake((7, 3, 64), BF16), v=Fake((7, 3, 64), BF16)), dict(slots=Fake((8, ), I32)),
                   dict(slots=Fake((7, ), torch.int64)), dict(k=torch.zeros(7, 2, 64, dtype=BF16)), dict(v=Fake((7, 2, 64), BF16, device=2))):
        with pytest.raises(rt.InvalidLaunch):
            K.paged_write_kernel[(7, )](*{**ok, **change}.values(), *cache())
    assert not lib.calls


def test_another_current_device_is_refused(lib, monkeypatch):
    monkeypatch.setattr(drv.TTDriver, "get_current_device", lambda self: 1)
    with pytest.raises(rt.InvalidLaunch, match="current device"):
        K.paged_attn_kernel[(6, 8)](*attn_args(), CAUSAL=True)


def test_another_current_device_is_refused_in_a_repeated_launch(lib, monkeypatch):
    for _ in range(3):
        K.paged_attn_kernel[(6, 8)](*attn_args(), CAUSAL=True)
    monkeypatch.setattr(drv.TTDriver, "get_current_device", lambda self: 1)
    with pytest.raises(rt.InvalidLaunch, match="current device"):
        K.paged_attn_kernel[(6, 8)](*attn_args(), CAUSAL=True)
    assert len(lib.calls) == 3


def test_tensors_on_the_cpu_are_refused_by_the_wrappers():
    q = torch.zeros(2, 4, 64, dtype=BF16)
    c = K.paged_cache(4, 2, 64, 16, device="cpu")
    i = lambda *v: torch.tensor(v, dtype=I32)
    if not torch.cuda.is_available():
        with pytest.raises((rt.RuntimeError_, AssertionError, RuntimeError)):
            K.paged_attention(q, c, i(0, 1).view(2, 1), i(1, 1), i(0, 1, 2), 1.0, max_q=1)


def test_nothing_is_launched_for_no_rows():
    c = K.paged_cache(4, 2, 64, 16, device="cpu")
    q = torch.zeros(0, 4, 64, dtype=BF16)
    i = lambda *v: torch.tensor(v, dtype=I32)
    o, lse = K.paged_attention(q, c, i(0, 1).view(2, 1), i(1, 1), i(0, 0, 0), 1.0, return_lse=True)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    assert K.paged_write(q[:, :2], q[:, :2], i(), c) is c


def test_a_users_kernel_of_the_same_name_is_not_bound_to_it():
    assert not set(drv.OWN_KERNELS) & set(drv.KERNEL_TABLE)
    text = 'module { tt.func public @paged_attn_kernel(%a: !tt.ptr<f32>) attributes {noinline = false} { tt.return } }'
    try:
        record = compiler.TTBackend.make_binary(text, {}, type("O", (), {"arch": "gfx950"}))
        assert b"paged" not in record       # the empty kernel, by its body
    except RuntimeError:
        pass


@pytest.mark.parametrize("n", [2**31, 2**32 + 1, 2**32 + 16, -2**31 - 1])
def test_numbers_of_more_than_31_bits_are_refused_not_cut(lib, n):
    with pytest.raises(rt.InvalidLaunch, match="31 bits"):
        K.paged_attn_kernel[(6, 8)](*attn_args(max_q=n), CAUSAL=True)
    with pytest.raises(rt.InvalidLaunch, match="31 bits"):
        K.paged_plan_kernel[(4, )](*plan_args(), PAGE_SIZE=n)
    assert not lib.calls


def test_tensors_of_more_than_31_bits_are_refused_not_cut(lib):
    n = 2**32 + 4
    for args in (plan_args(free_pages=Fake((n, ), I32)), plan_args(slot_map=Fake((n, ), I32)), plan_args(block_table=Fake((4, n), I32))):
        with pytest.raises(rt.InvalidLaunch, match="31 bits"):
            K.paged_plan_kernel[(4, )](*args, PAGE_SIZE=16)
    long = Fake((n, 2, 64), BF16)
    with pytest.raises(rt.InvalidLaunch, match="31 bits"):
        K.paged_write_kernel[(4, )](long, long, Fake((n, ), I32), *cache())
    with pytest.raises(rt.InvalidLaunch, match="31 bits"):
        K.paged_write_kernel[(7, )](Fake((7, 2, 64), BF16), Fake((7, 2, 64), BF16), Fake((7, ), I32), *cache(pages=n))
    long = Fake((n, 8, 64), BF16)
    with pytest.raises(rt.InvalidLaunch, match="31 bits"):
        K.paged_attn_kernel[(4, 8)](*attn_args(q=long, out=long), CAUSAL=True)
    with pytest.raises(rt.InvalidLaunch, match="31 bits"):
        K.paged_attn_kernel[(6, 8)](*attn_args(table=Fake((3, n), I32)), CAUSAL=True)
    assert not lib.calls


@pytest.mark.parametrize("name", sorted(drv.OWN_KERNELS))
def test_a_users_kernel_of_an_own_name_is_bound_by_its_body(name):
    text = "module {\n  tt.func public @%s(%%arg0: !tt.ptr<f32>) attributes {noinline = false} {\n%s    tt.return\n  }\n}\n"
    options = type("O", (), {"arch": "gfx950"})
    assert json.loads(compiler.TTBackend.make_binary(text % (name, ""), {}, options))["kernel"] == "empty_kernel"
    with pytest.raises(RuntimeError, match=f"'{name}' has no prebuilt"):
        compiler.TTBackend.make_binary(text % (name, "    %0 = tt.get_program_id x : i32\n"), {}, options)


def test_the_wrappers_refuse_tensors_on_the_cpu(lib):
    q = torch.zeros(2, 4, 64, dtype=BF16)
    c = K.paged_cache(4, 2, 64, 16, device="cpu")
    i = lambda *v: torch.tensor(v, dtype=I32)
    for call in (lambda: K.paged_attention(q, c, i(0, 1).view(2, 1), i(1, 1), i(0, 1, 2), 1.0, max_q=1),
                 lambda: K.paged_write(q[:, :2], q[:, :2], i(0, 1), c),
                 lambda: K.paged_plan(i(0, 0), i(1, 1), i(-1, -1).view(2, 1), i(0, 1), 16, 2)):
        with pytest.raises(rt.InvalidLaunch, match="on the GPU"):
            call()
    assert not lib.calls
