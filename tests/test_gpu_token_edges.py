"""What tests/test_hostemu_token_edges.py checks of the token operators' kernels, on the GPU, where the matrix instructions' own sums show."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from tests import token_cases as tc
from tests.test_gpu_tokens import DEV, DTYPES, ops  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", tc.DEEP_FEW + tc.DEEP_MANY)
def test_sums_of_8bit_products(ops, case):
    tc.check_product_deep_sums(ops, case, torch.float32, DEV)
    if case in tc.DEEP_FEW:
        for dtype in (torch.bfloat16, torch.float16):
            tc.check_product_deep_sums(ops, case, dtype, DEV)


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_batches(ops, dtype):
    tc.check_empty_batches(ops, dtype, DEV)


@pytest.mark.parametrize("dtype", DTYPES)
def test_residual_out_beside_an_input(ops, dtype):
    tc.check_residual_out_beside(ops, dtype, DEV)


@pytest.mark.parametrize("act", [None, "silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("rows", [3, 40])
def test_activations_of_sums_that_are_not_finite(ops, act, rows):
    for dtype in DTYPES:
        tc.check_activations(ops, dtype, act, rows, dev=DEV)
        tc.check_activations(ops, torch.float8_e4m3fn, act, rows, dtype, DEV)


@pytest.mark.parametrize("counts", [[2], [30, 9], [90, 70]])
def test_scales_whose_product_is_subnormal(ops, counts):
    tc.check_product_small_scales(ops, counts, DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,Cin,Cout", [([3000, 0, 2100, 4097, 700, 6000], 208, 2576), ([300, 0, 517, 1], 336, 520), ([130] * 40, 1040, 1544), ([3, 0, 1], 2048, 136)])
def test_8bit_products_with_16bit_outputs(ops, counts, Cin, Cout, dtype):
    """By the rule: tiles of 256 (12 row tiles of 11 channel tiles and more), of 64, of 128 and few rows."""
    tc.check_product_exact_16(ops, counts, Cin, Cout, dtype, DEV)
    torch.cuda.synchronize()


@pytest.mark.parametrize("tile", ["16", "64", "128", "256"])
def test_8bit_products_with_16bit_outputs_at_every_tile(tile):
    code = (
        "import torch\n"
        "from tests import token_cases as tc, test_gpu_tokens as t\n"
        "from yolo_master_amd import ops\n"
        "for c in (([130, 0, 1, 37], 80, 144), ([5, 129], 208, 16), ([300, 0, 517, 1], 336, 520)):\n"
        "    for d in (torch.bfloat16, torch.float16): tc.check_product_exact_16(ops, *c, d, t.DEV)\n"
        "for c in t.BIG:\n"
        "    if c[2] % 16 == 0 and c[5] % 16 == 0:\n"
        "        for d in (torch.bfloat16, torch.float16): tc.check_product(ops, t.E4M3, c, t.DEV, out_dtype=d)\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=str(Path(__file__).resolve().parent.parent), env={**os.environ, "YMK_EXPERT_TILE": tile}, timeout=110)


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_over_its_own_inputs(ops, dtype):
    tc.check_norm_aliases(ops, dtype, DEV)


def test_bias_sums(ops):
    tc.check_long_bias_sums(ops, torch.float32, [12000, 0, 31], 1.0001, DEV)
    tc.check_long_bias_sums(ops, torch.float32, [100003, 40000], 1.0001, DEV)
    for dtype, value in ((torch.bfloat16, 1 + 2.0**-7), (torch.float16, 1 + 2.0**-10)):
        tc.check_long_bias_sums(ops, dtype, [700001, 33], value, DEV)
    for dtype in DTYPES:
        tc.check_bias_sums_that_are_not_finite(ops, dtype, DEV)


def test_weight_gradients_of_many_rows(ops):
    tc.check_long_weight_sums(ops, torch.float32, [12000, 0, 511, 513], 1.0001, DEV)
    tc.check_long_weight_sums(ops, torch.float32, [100003, 512], 1.0001, DEV)


@pytest.mark.parametrize("rows,K", [(30, 20000), (200, 100000), (2, 100000)])
def test_products_of_many_channels(ops, rows, K):
    tc.check_long_products(ops, rows, K, DEV)
