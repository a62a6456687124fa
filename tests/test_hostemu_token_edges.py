"""Calls at the edges of what the token operators' wrappers accept, on the CPU lane emulator: operands that look right by their shape alone, empty
batches of any rank, strides that do not fit the C interface, values that are not finite."""
import os
import subprocess
import sys
import warnings
from pathlib import Path

import pytest
import torch

from tests import token_cases as tc
from tests.test_hostemu_tokens import libs, ops  # noqa: F401  (fixtures)


def test_a_plan_is_dense_int32(ops):
    """The moves read plan.row as dense int32 [tokens][top_k]: anything else of that shape is refused, by all who take a plan."""
    T, K, E, n = 6, 2, 4, 16
    plan = ops.token_sort(torch.arange(T * (K + 1), dtype=torch.int32).view(T, K + 1) % E, E)
    w = torch.ones(T, K)
    x, ys = torch.zeros(T, n), torch.zeros(T * K, n)
    good = plan.row[:, :K].contiguous()
    bad = {"a slice": plan.row[:, :K], "int64": good.long(), "int16": good.short(), "int8": good.to(torch.int8), "float": good.float(), "transposed": good.t().contiguous().t(),
           "expanded": good[:1].expand(T, K), "one value": good[:1, :1].expand(T, K), "flat": good.view(-1), "three dims": good.view(T, K, 1)}
    ops.token_dispatch(x, plan._replace(row=good))
    for what, row in bad.items():
        p = plan._replace(row=row)
        for call in (lambda: ops.token_dispatch(x, p), lambda: ops.token_dispatch(x, p, scale=torch.ones(T)), lambda: ops.token_combine(ys, p, w), lambda: ops.token_dispatch_backward(ys, p),
                     lambda: ops.token_combine_backward(x, ys, p, w)):
            with pytest.raises(ValueError, match="plan"):
                call()
                pytest.fail(f"{what} row was taken")


@pytest.mark.parametrize("case", tc.DEEP_FEW + tc.DEEP_MANY)
def test_sums_of_8bit_products(ops, case):
    tc.check_product_deep_sums(ops, case, torch.float32)
    if case in tc.DEEP_FEW:
        for dtype in (torch.bfloat16, torch.float16):
            tc.check_product_deep_sums(ops, case, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_empty_batches(ops, dtype):
    tc.check_empty_batches(ops, dtype)


def test_strides_that_do_not_fit_are_refused(ops):
    """Row strides and widths go to the kernels as 32-bit numbers of elements (dispatch: 64-bit bytes): one of 2^32 + 16 must not arrive as 16."""
    far = torch.empty(2**32 + 64, dtype=torch.bfloat16)   # never touched but for its ends
    n, gate = 16, torch.ones(2, 1)
    x = far.as_strided((2, n), (2**32 + 16, 1))
    x[0], x[1] = 1, 2
    near, w = torch.ones(2, n, dtype=torch.bfloat16), torch.ones(n)
    plan = ops.token_sort(torch.tensor([[1], [0]], dtype=torch.int32), 2)
    off = torch.tensor([0, 2], dtype=torch.int32)
    wt = torch.ones(1, n, n, dtype=torch.bfloat16)
    for bad in (lambda: ops.rms_norm(x, w), lambda: ops.rms_norm(near, w, residual=x), lambda: ops.rms_norm(near, w, residual=near, residual_out=x), lambda: ops.rms_norm_quant(x, w),
                lambda: ops.rms_norm_backward(x, near, w, torch.ones(2)), lambda: ops.rms_norm_backward(near, x, w, torch.ones(2)),
                lambda: ops.rms_norm_backward(near, near, w, torch.ones(2), dres=x), lambda: ops.token_combine(x, plan, gate), lambda: ops.token_dispatch_backward(x, plan),
                lambda: ops.token_combine_backward(x, near, plan, gate), lambda: ops.token_combine_backward(near, x, plan, gate), lambda: ops.expert_linear(x, wt, off),
                lambda: ops.expert_linear_backward(x, near, wt, off), lambda: ops.expert_linear_backward(near, x, wt, off)):
        with pytest.raises(ValueError, match="2\\^31"):
            bad()
    wide = far[:2**32 + 16].view(1, -1)
    one = ops.token_sort(torch.zeros(1, 1, dtype=torch.int32), 1)
    for bad in (lambda: ops.token_combine(wide, one, gate[:1]), lambda: ops.token_combine_backward(wide, wide, one, gate[:1]), lambda: ops.token_dispatch_backward(wide, one)):
        with pytest.raises(ValueError, match="2\\^31"):
            bad()
    assert torch.equal(ops.token_dispatch(x, plan), torch.tensor([[2.0], [1.0]]).expand(2, n).bfloat16())
    m = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="meta")   # noqa: E731
    for bad in (lambda: ops.expert_linear(m(2, 8), m(1, 2**32 + 8, 8), off), lambda: ops.expert_linear_backward(m(2, 2**32 + 8), m(2, 8), m(1, 2**32 + 8, 8), off)):
        with pytest.raises(ValueError, match="2\\^23"):
            bad()


def test_residual_out_beside_an_input(ops):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        tc.check_residual_out_beside(ops, dtype)
    buf, r, w = torch.zeros(6, 96), torch.zeros(4, 40), torch.ones(40)
    for out in (buf[:4, 1:41], buf[:4, 39:79], buf[1:5, :40], buf.view(-1)[160:544].view(4, 96)[:, :40], buf.view(-1)[41:341].view(4, 75)[:, :40]):   # shifted, a row on, the end of the row before, other strides
        with pytest.raises(ValueError, match="overlaps"):
            ops.rms_norm(buf[:4, :40], w, residual=r, residual_out=out)
        with pytest.raises(ValueError, match="overlaps"):
            ops.rms_norm(r, w, residual=buf[:4, :40], residual_out=out)
    for out in (buf[2:6, 56:], buf[1:5, 40:80]):   # other rows' columns 56 .. 95 and 40 .. 79: none of x's 0 .. 39
        assert ops.rms_norm(buf[:4, :40], w, residual=r, residual_out=out)[1] is out


@pytest.mark.parametrize("act", [None, "silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("rows", [3, 40])
def test_activations_of_sums_that_are_not_finite(ops, act, rows):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        tc.check_activations(ops, dtype, act, rows)
        tc.check_activations(ops, torch.float8_e4m3fn, act, rows, dtype)


def test_residual_out_right_behind_an_input(ops):
    """Tensors apart from each other, with rows of different strides, at neighbouring addresses (as an allocator hands them out)."""
    pool, w = torch.randn(2000), torch.ones(40)
    dense, far = pool[:200].view(5, 40), pool[200:600].view(5, 80)[:, :40]
    behind = pool[600:800].view(5, 40)   # from the end of the strided rows' last padding on
    for x, out in ((dense, far), (far, behind), (behind, far), (far, dense)):
        want = ops.rms_norm(x.clone(), w, residual=torch.ones(5, 40))
        got = ops.rms_norm(x, w, residual=torch.ones(5, 40), residual_out=out)
        assert torch.equal(got[0], want[0]) and torch.equal(out, want[1])


def test_rows_too_wide_for_the_kernels_counters(libs):
    """Column numbers of the moves are 32-bit: a width whose round-up to whole vectors passes 2^31 is refused, not walked from a negative column."""
    h = libs[False]
    t = torch.full((64,), 5.0)
    row = torch.zeros(1, dtype=torch.int32)
    p, r = t.data_ptr(), row.data_ptr()
    for dtype in (0, 1):
        for wide in (2**31 - 15, 2**31 - 7, 2**31 - 1):
            assert h.ymk_token_combine(dtype, p, wide, r, p, p, wide, 1, 1, wide, None) == -1
            assert h.ymk_token_combine_backward(dtype, p, wide, p, wide, r, p, p, wide, p, 1, 1, wide, None) == -1
    assert h.ymk_token_dispatch(p, 2**24 + 1, 2**24 + 1, None, p, 2**24 + 1, None, r, 1, 1, None) == -1
    assert bool((t == 5).all())


@pytest.mark.parametrize("counts", [[2], [30, 9]])
def test_scales_whose_product_is_subnormal(ops, counts):
    tc.check_product_small_scales(ops, counts)


def test_operands_that_require_gradients(ops):
    """Outputs carry no gradient: the forward calls say so where an operand asks for one, and are silent everywhere else."""
    x, w, wt, off = torch.ones(4, 16), torch.ones(16), torch.ones(2, 8, 16), torch.tensor([0, 2, 4], dtype=torch.int32)
    idx, gate = torch.tensor([[0], [1], [0], [1]], dtype=torch.int32), torch.ones(4, 1)
    plan = ops.token_sort(idx, 2)
    g = lambda t: t.clone().requires_grad_(True)   # noqa: E731
    calls = [lambda f: ops.rms_norm(f(x), w), lambda f: ops.rms_norm(x, f(w), residual=x), lambda f: ops.rms_norm(x, w, residual=f(x)), lambda f: ops.rms_norm_quant(x, f(w)),
             lambda f: ops.token_dispatch(f(x), plan), lambda f: ops.token_combine(x, plan, f(gate)), lambda f: ops.expert_linear(f(x), wt, off), lambda f: ops.expert_linear(x, f(wt), off),
             lambda f: ops.expert_linear(x, wt, off, f(torch.ones(2, 8)))]
    for call in calls:
        with pytest.warns(UserWarning, match="requires gradients"):
            out = call(g)
        assert not (out[0] if isinstance(out, tuple) else out).requires_grad   # (rms_norm's h without a residual is x itself)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for call in calls:
            call(lambda t: t)
            with torch.no_grad():
                call(g)
        ops.rms_norm_backward(x, x, g(w), torch.ones(4))
        ops.expert_linear_backward(torch.ones(4, 8), x, g(wt), off)
        ops.token_combine_backward(x, x, plan, g(gate))
        ops.token_dispatch_backward(x, plan)


@pytest.mark.parametrize("tile", ["64", "128", "256"])
def test_8bit_products_with_16bit_outputs_at_every_tile(tile, libs):
    """The switch is read once a process."""
    code = (
        "import torch, ctypes as C\n"
        "from tests import token_cases as tc\n"
        "from tests.hostemu import build\n"
        "from yolo_master_amd import _lib, ops\n"
        "h = C.CDLL(str(build.build()))\n"
        "for name, (res, args) in _lib.SYMBOLS_TOKENS.items(): fn = getattr(h, name); fn.restype, fn.argtypes = res, args\n"
        "ops.lib, ops._stream, ops.require_gpu = h, lambda: None, lambda t, what='': None\n"
        "for c in (([130, 0, 1, 37], 80, 144), ([5, 129], 208, 16)): tc.check_product_exact_16(ops, *c, torch.bfloat16)\n"
        "tc.check_product(ops, torch.float8_e4m3fn, ([70, 0, 3], 1, 144, 40, 'gelu', 16))\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=str(Path(__file__).resolve().parent.parent), env={**os.environ, "YMK_EXPERT_TILE": tile}, timeout=600)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_norm_over_its_own_inputs(ops, dtype):
    tc.check_norm_aliases(ops, dtype)


def test_bias_sums(ops):
    tc.check_long_bias_sums(ops, torch.float32, [12000, 0, 31], 1.0001)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        tc.check_long_bias_sums(ops, dtype, [100, 1, 64], 1.0)
        tc.check_bias_sums_that_are_not_finite(ops, dtype)


def test_weight_gradients_of_many_rows(ops):
    tc.check_long_weight_sums(ops, torch.float32, [12000, 0, 511, 513], 1.0001)


def test_products_of_many_channels(ops):
    tc.check_long_products(ops, 30, 20000)
    tc.check_long_products(ops, 2, 60000)
