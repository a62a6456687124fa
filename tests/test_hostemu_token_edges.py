"""Calls at the edges of what the token operators' wrappers accept, on the CPU lane emulator: operands that look right by their shape alone, empty
batches of any rank, strides that do not fit the C interface, values that are not finite."""
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
