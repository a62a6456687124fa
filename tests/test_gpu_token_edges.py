"""What tests/test_hostemu_token_edges.py checks of the token operators' kernels, on the GPU, where the matrix instructions' own sums show."""
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
