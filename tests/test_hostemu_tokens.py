"""The token operators (csrc/rmsnorm.hip, tokens.hip, expert.hip; include/ymk_tokens.h) on the CPU lane emulator, through the product's own wrappers:
every check of tests/token_cases.py, the refusals of the wrappers and of the C entry points, and the header against its ctypes table."""
import ctypes as C
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from tests import token_cases as tc
from tests.hostemu import build as hostemu_build

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def libs():
    from yolo_master_amd import _lib

    out = {}
    for f16 in (False, True):
        path = hostemu_build.build(f16=f16)
        if path is None:
            pytest.skip("no host clang++ to build the kernel emulation")
        h = C.CDLL(str(path))
        for name, (res, args) in _lib.SYMBOLS_TOKENS.items():
            fn = getattr(h, name)
            fn.restype, fn.argtypes = res, args
        out[f16] = h
    return out


@pytest.fixture
def ops(libs, monkeypatch):
    from yolo_master_amd import ops

    class Router:
        def __getattr__(self, name):
            return getattr(libs[getattr(ops._TLS, "fmt", None) is torch.float16], name)

    monkeypatch.setattr(ops, "lib", Router())
    monkeypatch.setattr(ops, "_stream", lambda: None)
    monkeypatch.setattr(ops, "require_gpu", lambda t, what="": None)
    return ops


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", tc.NORMS)
def test_norm(ops, dtype, case):
    tc.check_norm(ops, dtype, case)


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_in_place_and_special_rows(ops, dtype):
    tc.check_norm_in_place(ops, dtype)
    tc.check_norm_special(ops, dtype)


def test_norm_gradient_against_differences(ops):
    tc.check_norm_differences(ops)


@pytest.mark.parametrize("case", tc.SORTS)
def test_sort(ops, case):
    tc.check_sort(ops, case)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", tc.MOVES)
def test_moves(ops, dtype, case):
    tc.check_moves(ops, dtype, case)


def test_plans_of_ones_own(ops):
    tc.check_plans_of_ones_own(ops)


@pytest.mark.parametrize("dtype", DTYPES)
def test_views(ops, dtype):
    tc.check_views(ops, dtype)


def test_dispatch_8bit(ops):
    tc.check_dispatch_8bit(ops)


@pytest.mark.parametrize("dtype", DTYPES + [torch.float8_e4m3fn])
@pytest.mark.parametrize("case", tc.PRODUCTS)
def test_product(ops, dtype, case):
    tc.check_product(ops, dtype, case)


@pytest.mark.parametrize("case", tc.PRODUCTS)
def test_product_exact_sums(ops, case):
    tc.check_product_exact(ops, case)


def test_product_forms(ops):
    tc.check_product(ops, torch.bfloat16, ([3, 9], 1, 24, 40, None, 8), bias=False, start=2)
    tc.check_product(ops, torch.float32, ([3, 9], 1, 20, 36, "silu", 4), bias=True)
    tc.check_product(ops, torch.float8_e4m3fn, ([3, 9], 1, 48, 24, "gelu", 0), bias=False, out_dtype=torch.float32)
    tc.check_product(ops, torch.float8_e4m3fn, ([2, 1], 0, 16, 8, None, 0), out_dtype=torch.float16)
    tc.check_product(ops, torch.bfloat16, ([0] * 70 + [2] + [0] * 100 + [3], 0, 16, 8, None, 0))   # more experts than a wave has lanes


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", tc.PRODUCTS)
def test_product_gradient(ops, dtype, case):
    tc.check_product_gradient(ops, dtype, case)


def test_product_gradient_in_32_bits(ops):
    tc.check_product_gradient(ops, torch.bfloat16, ([40, 3], 0, 24, 40, None, 8), dw_dtype=torch.float32)


@pytest.mark.parametrize("tile", ["64", "128", "256"])
def test_product_at_every_tile(tile, libs):
    """Each tile on sizes that the rule would give to another (the switch is read once a process)."""
    code = (
        "import torch, ctypes as C\n"
        "from tests import token_cases as tc\n"
        "from tests.hostemu import build\n"
        "from yolo_master_amd import _lib, ops\n"
        "h = C.CDLL(str(build.build()))\n"
        "for name, (res, args) in _lib.SYMBOLS_TOKENS.items(): fn = getattr(h, name); fn.restype, fn.argtypes = res, args\n"
        "ops.lib, ops._stream, ops.require_gpu = h, lambda: None, lambda t, what='': None\n"
        "for c in (([130, 0, 1, 37], 3, 80, 144, 'gelu', 0), ([5, 129], 0, 208, 16, 'sigmoid', 0), ([3, 0, 200, 1, 2, 7, 0, 1, 5, 9, 1, 1, 4, 260], 2, 48, 40, None, 0)):\n"
        "    for d in (torch.float32, torch.bfloat16): tc.check_product(ops, d, c); tc.check_product_gradient(ops, d, c)\n"
        "    tc.check_product_exact(ops, c)\n"
        "    tc.check_product(ops, torch.float8_e4m3fn, c, out_dtype=torch.float32)\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=str(Path(__file__).resolve().parent.parent), env={**os.environ, "YMK_EXPERT_TILE": tile}, timeout=600)


@pytest.mark.parametrize("dtype", DTYPES)
def test_block(ops, dtype):
    tc.check_block(ops, dtype)


def test_block_gradient(ops):
    tc.check_block_gradient(ops)


def test_offsets_outside_the_rows_are_clamped(ops):
    """Device-side offsets are not trusted: nothing outside x and y is touched, whatever they say."""
    x, w = torch.ones(6, 16), torch.ones(3, 8, 16)
    for off in ([0, 2, 4, 99], [-5, 2, 1, 6], [6, 0, 2**31 - 1, -1], [3, 3, 3, 3]):
        o = torch.tensor(off, dtype=torch.int32)
        y = ops.expert_linear(x, w, o)
        assert y.shape == (6, 8)
        dx, dw, db = ops.expert_linear_backward(torch.ones(6, 8), x, w, o)
        assert bool(torch.isfinite(dw).all()) and bool(torch.isfinite(db).all())


def test_refusals(ops):
    x, w = torch.zeros(4, 16), torch.zeros(16)
    for bad in (lambda: ops.rms_norm(x.double(), w), lambda: ops.rms_norm(x, w.half()), lambda: ops.rms_norm(x, torch.zeros(15)), lambda: ops.rms_norm(x.t(), torch.zeros(4)),
                lambda: ops.rms_norm(torch.zeros(2, 16385), torch.zeros(16385)), lambda: ops.rms_norm(x, w, residual=torch.zeros(4, 15)), lambda: ops.rms_norm(x[:1].expand(4, 16), w),
                lambda: ops.rms_norm(x, w, residual=x.bfloat16()), lambda: ops.rms_norm(x, w, residual_out=x), lambda: ops.rms_norm(torch.zeros(16), w),
                lambda: ops.rms_norm(x[:3], w, residual=torch.zeros(3, 16), residual_out=x[1:]), lambda: ops.rms_norm(torch.zeros(2, 0), torch.zeros(0)),
                lambda: ops.rms_norm(torch.zeros(4, 3, 32)[:, :2, :16], w),
                lambda: ops.rms_norm_backward(x, x, w, torch.zeros(3)), lambda: ops.rms_norm_backward(x[:2], x, w, torch.zeros(4))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        ops.rms_norm(x, w, eps=-1.0)
    idx = torch.zeros(3, 2, dtype=torch.int32)
    for bad in (lambda: ops.token_sort(idx.float(), 4), lambda: ops.token_sort(idx.t(), 4), lambda: ops.token_sort(idx, 0), lambda: ops.token_sort(idx, 257),
                lambda: ops.token_sort(torch.zeros(3, 17, dtype=torch.int32), 4), lambda: ops.token_sort(idx[0], 4), lambda: ops.token_sort(torch.zeros(3, 0, dtype=torch.int32), 4)):
        with pytest.raises(ValueError):
            bad()
    plan = ops.token_sort(idx, 4)
    g = torch.zeros(3, 2)
    for bad in (lambda: ops.token_dispatch(x, plan), lambda: ops.token_dispatch(x[:3], plan, scale=torch.zeros(2)), lambda: ops.token_combine(x, plan, g),
                lambda: ops.token_combine(torch.zeros(6, 8), plan, g.half()), lambda: ops.token_combine(torch.zeros(6, 8), plan, None),
                lambda: ops.token_combine(torch.zeros(6, 8), plan, g[:2]), lambda: ops.token_combine(torch.zeros(6, 8).to(torch.float8_e4m3fn), plan, g),
                lambda: ops.token_dispatch_backward(torch.zeros(5, 8), plan), lambda: ops.token_combine_backward(torch.zeros(3, 7), torch.zeros(6, 8), plan, g),
                lambda: ops.token_combine_backward(torch.zeros(3, 8).half(), torch.zeros(6, 8), plan, g)):
        with pytest.raises(ValueError):
            bad()
    off = torch.zeros(3, dtype=torch.int32)
    wt = torch.zeros(2, 8, 16)
    q, qw = x.to(torch.float8_e4m3fn), wt.to(torch.float8_e4m3fn)
    for bad in (lambda: ops.expert_linear(x, wt.half(), off), lambda: ops.expert_linear(x, wt[0], off), lambda: ops.expert_linear(x, wt, off.long()), lambda: ops.expert_linear(x, wt, off[:2]),
                lambda: ops.expert_linear(x, wt.transpose(1, 2), off), lambda: ops.expert_linear(x[:, :8], wt, off), lambda: ops.expert_linear(torch.zeros(4, 18)[:, :16], wt, off),
                lambda: ops.expert_linear(torch.zeros(4, 6), torch.zeros(2, 8, 6), off), lambda: ops.expert_linear(x, torch.zeros(2, 6, 16), off),
                lambda: ops.expert_linear(torch.zeros(65)[1:].view(4, 16), wt, off), lambda: ops.expert_linear(x, wt, off, act="relu"), lambda: ops.expert_linear(x, wt, off, torch.zeros(2, 7)),
                lambda: ops.expert_linear(q, qw, off), lambda: ops.expert_linear(x, wt, off, x_scale=torch.zeros(4)), lambda: ops.expert_linear(x, wt, off, out_dtype=torch.bfloat16),
                lambda: ops.expert_linear(q, qw, off, x_scale=torch.zeros(4), w_scale=torch.zeros(2)), lambda: ops.expert_linear(x, torch.zeros(257, 8, 16), torch.zeros(258, dtype=torch.int32)),
                lambda: ops.expert_linear_backward(torch.zeros(3, 8), x, wt, off), lambda: ops.expert_linear_backward(torch.zeros(4, 8).half(), x, wt, off),
                lambda: ops.expert_linear_backward(torch.zeros(4, 8), x, wt, off, dw_dtype=torch.bfloat16), lambda: ops.expert_linear_backward(torch.zeros(4, 8), x, wt, off, need_dw=False),
                lambda: ops.expert_linear_backward(q, q, qw, off)):
        with pytest.raises(ValueError):
            bad()


def test_the_c_entry_points_refuse(libs):
    """What the wrappers never pass: null pointers, unknown types, short workspaces — an error code, nothing launched, nothing written."""
    h = libs[False]
    t = torch.full((64,), 5.0)
    p = C.c_void_p(t.data_ptr())
    odd = C.c_void_p(t.data_ptr() + 2)
    assert h.ymk_rms_norm(2, p, 8, None, 0, None, 0, p, 8, None, 2, 8, p, 1e-6, None) == -1
    assert h.ymk_rms_norm(0, None, 8, None, 0, None, 0, p, 8, None, 2, 8, p, 1e-6, None) == -1
    assert h.ymk_rms_norm(0, odd, 8, None, 0, None, 0, p, 8, None, 2, 8, p, 1e-6, None) == -1
    assert h.ymk_rms_norm(0, p, 7, None, 0, None, 0, p, 8, None, 2, 8, p, 1e-6, None) == -1
    assert h.ymk_rms_norm(0, p, 8, p, 8, None, 0, p, 8, None, 2, 8, p, 1e-6, None) == -1
    assert h.ymk_rms_norm(0, p, 8, None, 0, None, 0, p, 8, None, -1, 8, p, 1e-6, None) == -1
    assert h.ymk_rms_norm_quant(0, p, 8, None, 0, None, 0, p, 8, None, 2, 8, p, 1e-6, None) == -1
    assert h.ymk_rms_norm_backward(0, p, 8, p, 8, p, p, None, 0, p, 8, p, 2, 8, p, 63, None) == -3
    assert h.ymk_rms_norm_backward(0, p, 8, p, 8, p, p, None, 0, p, 8, p, 2, 8, None, 0, None) == -3
    assert h.ymk_token_sort(p, 2, 2, 2, 4, p, p, p, None, 0, None) == -1
    assert h.ymk_token_sort(p, 4, 2, 2, 4, None, p, p, None, 0, None) == -1
    assert h.ymk_token_sort(p, 4, 1 << 40, 2, 4, p, p, p, None, 0, None) == -1
    assert h.ymk_token_sort(p, 4, 1 << 20, 2, 4, p, p, p, p, 16, None) == -3
    assert h.ymk_token_dispatch(p, 16, 32, None, p, 32, None, p, 2, 2, None) == -1
    assert h.ymk_token_dispatch(p, 32, 32, p, p, 32, None, p, 2, 2, None) == -1
    assert h.ymk_token_combine(2, p, 8, p, p, p, 8, 2, 2, 8, None) == -1
    assert h.ymk_token_combine_backward(0, p, 8, p, 8, p, None, p, 8, p, 2, 2, 8, None) == -1
    assert h.ymk_expert_linear(0, 1, p, 16, None, p, None, None, p, p, 8, 4, 1, 16, 8, 0, None) == -1
    assert h.ymk_expert_linear(2, 1, p, 16, None, p, None, None, p, p, 8, 4, 1, 16, 8, 0, None) == -1
    assert h.ymk_expert_linear(0, 0, p, 16, None, p, None, None, p, p, 8, 4, 1, 16, 8, 9, None) == -1
    assert h.ymk_expert_linear(0, 0, p, 1 << 21, None, p, None, None, p, p, 8, 4, 1, 16, 8, 0, None) == -1
    assert h.ymk_expert_linear_dx(2, p, 16, p, p, p, 16, 4, 1, 16, 16, None) == -1
    assert h.ymk_expert_linear_dw(0, 1, p, 8, p, 16, p, p, None, 4, 1, 16, 8, None) == -1
    assert bool((t == 5).all())


def test_header_and_ctypes_table():
    from tests.test_capi import header_functions, header_prototypes
    from yolo_master_amd import _lib

    assert sorted(_lib.SYMBOLS_TOKENS) == header_functions("ymk_tokens.h")
    protos = header_prototypes("ymk_tokens.h")
    for name, (_, argtypes) in _lib.SYMBOLS_TOKENS.items():
        assert len(protos[name]) == len(argtypes), name
        for d, t in zip(protos[name], argtypes):
            assert ("*" in d) == (t is C.c_void_p), (name, d)
