"""The token operators (include/ymk_tokens.h) on the GPU: the checks of tests/token_cases.py that the lane emulator runs too, the sizes it is too slow
for, and what only the hardware shows — captured graphs, side streams, the same bits on every run."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from tests import token_cases as tc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
E4M3 = torch.float8_e4m3fn


@pytest.fixture
def ops():
    from yolo_master_amd import ops

    return ops


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", tc.NORMS + [(5, 4096, 0, True), (700, 4096, 0, True), (3, 16384, 0, True), (2, 16383, 1, True), (1300, 2048, 8, True), (4000, 256, 0, True),
                                             (1000, 1021, 0, True), (520, 6144, 0, True), (530, 8200, 0, False), (20011, 72, 0, True)])
def test_norm(ops, dtype, case):
    tc.check_norm(ops, dtype, case, DEV)


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_in_place_and_special_rows(ops, dtype):
    tc.check_norm_in_place(ops, dtype, DEV)
    tc.check_norm_special(ops, dtype, DEV)


def test_norm_gradient_against_differences(ops):
    tc.check_norm_differences(ops, DEV)


@pytest.mark.parametrize("case", tc.SORTS + [(65536, 8, 64, 0.0, True), (400000, 2, 200, 0.1, False), (100003, 1, 2, 0.0, False)])
def test_sort(ops, case):
    tc.check_sort(ops, case, DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", tc.MOVES + [(5000, 2, 8, 512, 0, 0.1), (1000, 6, 16, 2056, 8, 0.0), (300, 3, 8, 4099, 0, 0.2)])
def test_moves(ops, dtype, case):
    tc.check_moves(ops, dtype, case, DEV)


def test_plans_of_ones_own(ops):
    tc.check_plans_of_ones_own(ops, DEV)


@pytest.mark.parametrize("dtype", DTYPES)
def test_views(ops, dtype):
    tc.check_views(ops, dtype, DEV)


def test_dispatch_8bit(ops):
    tc.check_dispatch_8bit(ops, DEV)


BIG = [([300, 0, 517, 1], 9, 328, 520, "silu", 8), ([1000, 24], 0, 1024, 256, "gelu", 0), ([3, 1, 0, 2, 1, 1, 0, 0], 0, 2048, 1024, None, 0), ([17, 33, 16, 15], 1, 512, 272, "gelu", 0),
       ([700, 900, 20], 5, 512, 768, None, 0), ([1], 0, 4096, 4096, "silu", 0)]


@pytest.mark.parametrize("dtype", DTYPES + [E4M3])
@pytest.mark.parametrize("case", tc.PRODUCTS + BIG)
def test_product(ops, dtype, case):
    if dtype == E4M3:
        case = (case[0], case[1], -(-case[2] // 16) * 16) + case[3:5] + (-(-case[5] // 16) * 16,)
    tc.check_product(ops, dtype, case, DEV)


@pytest.mark.parametrize("case", tc.PRODUCTS + [c for c in BIG if c[2] % 16 == 0])
def test_product_exact_sums(ops, case):
    tc.check_product_exact(ops, case, DEV)


def test_product_forms(ops):
    tc.check_product(ops, torch.bfloat16, ([3, 9], 1, 24, 40, None, 8), DEV, bias=False, start=2)
    tc.check_product(ops, torch.float32, ([3, 9], 1, 20, 36, "silu", 4), DEV, bias=True)
    tc.check_product(ops, E4M3, ([3, 9], 1, 48, 24, "gelu", 0), DEV, bias=False, out_dtype=torch.float32)
    tc.check_product(ops, E4M3, ([2, 1], 0, 16, 8, None, 0), DEV, out_dtype=torch.float16)
    tc.check_product(ops, E4M3, ([400, 301], 0, 336, 264, None, 0), DEV, out_dtype=torch.float32)
    tc.check_product(ops, torch.bfloat16, ([0] * 70 + [2] + [0] * 100 + [3], 0, 16, 8, None, 0), DEV)   # more experts than a wave has lanes
    tc.check_product(ops, torch.float16, ([0] * 255 + [140], 3, 64, 64, None, 0), DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", tc.PRODUCTS + BIG)
def test_product_gradient(ops, dtype, case):
    tc.check_product_gradient(ops, dtype, case, DEV)


def test_product_gradient_in_32_bits(ops):
    tc.check_product_gradient(ops, torch.bfloat16, ([40, 3], 0, 24, 40, None, 8), DEV, dw_dtype=torch.float32)
    tc.check_product_gradient(ops, torch.bfloat16, ([1400, 0, 300], 0, 256, 320, None, 0), DEV, dw_dtype=torch.float32)


@pytest.mark.parametrize("tile", ["16", "64", "128", "256"])
def test_product_at_every_tile(tile):
    """Each tile of the product on sizes that the rule would give to another (the switch is read once a process)."""
    code = (
        "import torch\n"
        "from tests import token_cases as tc, test_gpu_tokens as t\n"
        "from yolo_master_amd import ops\n"
        "for c in tc.PRODUCTS + t.BIG:\n"
        "    for d in t.DTYPES: tc.check_product(ops, d, c, t.DEV); tc.check_product_gradient(ops, d, c, t.DEV)\n"
        "    if c[2] % 16 == 0: tc.check_product_exact(ops, c, t.DEV)\n"
        "tc.check_product_gradient(ops, torch.bfloat16, t.BIG[0], t.DEV, dw_dtype=torch.float32)\n"
        "tc.check_product(ops, t.E4M3, t.BIG[1], t.DEV, out_dtype=torch.float32)\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=str(Path(__file__).resolve().parent.parent), env={**os.environ, "YMK_EXPERT_TILE": tile}, timeout=110)


@pytest.mark.parametrize("dtype", DTYPES)
def test_block(ops, dtype):
    tc.check_block(ops, dtype, DEV)
    tc.check_block(ops, dtype, DEV, T=1, C=256, H=512, E=8, K=2)
    tc.check_block(ops, dtype, DEV, T=150, C=128, H=256, E=4, K=3)


def test_block_gradient(ops):
    tc.check_block_gradient(ops, DEV)


def test_offsets_outside_the_rows_are_clamped(ops):
    x, w = torch.ones(6, 16, device=DEV), torch.ones(3, 8, 16, device=DEV)
    for off in ([0, 2, 4, 99], [-5, 2, 1, 6], [6, 0, 2**31 - 1, -1], [3, 3, 3, 3]):
        o = torch.tensor(off, dtype=torch.int32, device=DEV)
        assert ops.expert_linear(x, w, o).shape == (6, 8)
        _, dw, db = ops.expert_linear_backward(torch.ones(6, 8, device=DEV), x, w, o)
        assert bool(torch.isfinite(dw).all()) and bool(torch.isfinite(db).all())


def _step(ops, s, K):
    """Forward and backward of one expert layer, every output."""
    y, h, rstd = ops.rms_norm(s["x"], s["norm"], residual=s["res"])
    q, qs, _ = ops.rms_norm_quant(s["x"], s["norm"], residual=s["res"])
    plan = ops.token_sort(s["idx"], s["w"].shape[0])
    xs, (xq, xqs) = ops.token_dispatch(y, plan), ops.token_dispatch(q, plan, scale=qs)
    z = ops.expert_linear(xs, s["w"], plan.offsets, s["b"], act="gelu")
    zq = ops.expert_linear(xq, s["wq"], plan.offsets, s["b"], x_scale=xqs, w_scale=s["ws"], act="silu")
    out = ops.token_combine(z, plan, s["gate"])
    dz, dgate = ops.token_combine_backward(s["dout"], z, plan, s["gate"])
    dxs, dw, db = ops.expert_linear_backward(dz, xs, s["w"], plan.offsets)
    dx, dnorm = ops.rms_norm_backward(ops.token_dispatch_backward(dxs, plan), h, s["norm"], rstd)
    return [y, h, q.view(torch.uint8), qs, plan.offsets, plan.src, plan.row, z, zq, out, dz, dgate, dxs, dw, db, dx, dnorm]


def _state(seed, T, C, H, E, K, dtype=torch.bfloat16):
    g = tc.gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    wq = r(E, H, C)
    ws = wq.abs().amax(-1) / 448
    s = {"x": r(T, C).to(dtype), "res": r(T, C).to(dtype), "norm": 1 + 0.1 * r(C), "idx": r(T, E).topk(K, dim=1).indices, "gate": r(T, K).softmax(1), "w": (r(E, H, C) * C**-0.5).to(dtype),
         "b": r(E, H), "wq": (wq / ws[..., None]).to(E4M3), "ws": ws, "dout": r(T, H).to(dtype)}
    return {k: v.to(DEV) for k, v in s.items()}


@pytest.mark.parametrize("T,C,H,E,K", [(5, 256, 512, 8, 2), (777, 128, 256, 6, 2), (5000, 64, 128, 4, 2)])
def test_captured_replayed_and_again(ops, T, C, H, E, K):
    """A graph of the whole layer, forward and backward, replayed with new inputs between eager work: every replay equals the eager run, which
    itself gives the same bits twice."""
    s = _state(1, T, C, H, E, K)
    fill = lambda o: {k: v.copy_(o[k]) for k, v in s.items()}   # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(ops, s, K)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _step(ops, s, K)
    for seed in (2, 3, 4, 2):
        fill(_state(seed, T, C, H, E, K))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want, again = _step(ops, s, K), _step(ops, s, K)
        torch.cuda.synchronize()
        for i, (a, b, c) in enumerate(zip(got, want, again)):
            assert torch.equal(b.view(torch.uint8), c.view(torch.uint8)), f"output {i} differs from run to run"
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), f"output {i} of the replay differs from the eager run"


def test_side_streams(ops):
    """Two streams at once, each with its own state: the calls go to the current stream and share nothing."""
    a, b = _state(5, 3000, 128, 256, 8, 2), _state(6, 2500, 128, 256, 8, 2)
    want = [[t.clone() for t in _step(ops, s, 2)] for s in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i] = _step(ops, s, 2)
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(g, w))


def test_refusals_on_the_gpu(ops):
    x, w = torch.zeros(4, 16, device=DEV), torch.zeros(16, device=DEV)
    with pytest.raises(RuntimeError):
        ops.rms_norm(x.cpu(), w.cpu())
    with pytest.raises(ValueError):
        ops.rms_norm(x, w.cpu())
    with pytest.raises(ValueError):
        ops.expert_linear(x, torch.zeros(2, 8, 16, device=DEV), torch.zeros(3, dtype=torch.int32))


def test_large_offsets(ops):
    """Rows whose byte offsets pass 2^31 and 2^32: 300000 rows of 8192 16-bit elements (4.9 GB)."""
    T, C, K, E = 150000, 8192, 2, 4
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randint(-100, 100, (T, C), generator=g, device=DEV, dtype=torch.int16).view(torch.bfloat16)
    idx = torch.randint(0, E, (T, K), generator=g, device=DEV)
    plan = ops.token_sort(idx, E)
    xs = ops.token_dispatch(x, plan)
    tok = (plan.src // K).long()
    for rows in (slice(0, 1000), slice(T, T + 1000), slice(T * K - 1000, T * K)):
        assert torch.equal(xs[rows].view(torch.int16), x[tok[rows]].view(torch.int16))
    xs.normal_(generator=g)
    w = torch.rand(T, K, generator=g, device=DEV)
    y = ops.token_combine(xs, plan, w)
    for t in (0, T // 2, T - 1):
        want = (xs[plan.row[t].long()].double() * w[t].double()[:, None]).sum(0)
        tc.close(y[t], want, want.abs() * 2.0**-8 + 1e-6, "combine")
    del x, y
    w = (torch.randn(E, 64, C, generator=g, device=DEV) * C**-0.5).bfloat16()
    z = ops.expert_linear(xs, w, plan.offsets)
    off = plan.offsets.tolist()
    dz = torch.randn(T * K, 64, generator=g, device=DEV).bfloat16()
    dx, dw, _ = ops.expert_linear_backward(dz, xs, w, plan.offsets)
    for e in range(E):
        for r in (off[e], off[e + 1] - 1):
            want = w[e].double() @ xs[r].double()
            tc.close(z[r], want, want.abs() * 2.0**-8 + 1e-3, "product")
            want = dz[r].double() @ w[e].double()
            tc.close(dx[r], want, want.abs() * 2.0**-8 + 1e-4, "dx")
        want = dz[off[e]:off[e + 1]].double().t() @ xs[off[e]:off[e + 1], :8].double()
        tc.close(dw[e][:, :8], want, want.abs() * 2.0**-8 + (off[e + 1] - off[e]) * 8 * 2.0**-24, "dw")


def test_product_wide_tiles_by_the_rule(ops):
    """More tiles of 256 than CUs, by the rule: ragged experts, an empty one, more experts than a wave has lanes."""
    for counts, Cin, Cout in (([3000, 0, 2100, 4097, 700, 6000], 200, 2576), ([250] * 70, 64, 1032)):
        tc.check_product(ops, torch.bfloat16, (counts, 3, Cin, Cout, "silu", 8), DEV)
        g = torch.Generator(device=DEV).manual_seed(3)
        off = tc.make_offsets(counts)
        R, E = int(off[-1]), len(counts)
        x, w, dy = (torch.randn(*s, generator=g, device=DEV) for s in ((R, Cin), (E, Cout, Cin), (R, Cout)))
        for dt in (torch.bfloat16, torch.float32):
            xt, wt, dt_ = x.to(dt), (w * Cin**-0.5).to(dt), dy.to(dt)
            y = ops.expert_linear(xt, wt, off.to(DEV))
            dx, dw, db = ops.expert_linear_backward(dt_, xt, wt, off.to(DEV))
            for e in range(E):
                s = slice(int(off[e]), int(off[e + 1]))
                a, b, d = xt[s].double(), wt[e].double(), dt_[s].double()
                for got, want, mag, n in ((y[s], a @ b.t(), a.abs() @ b.abs().t(), Cin), (dx[s], d @ b, d.abs() @ b.abs(), Cout), (dw[e], d.t() @ a, d.abs().t() @ a.abs(), len(a)),
                                          (db[e], d.sum(0), d.abs().sum(0), len(a))):
                    tc.close(got, want, mag * ((n + 8) * tc.U) + want.abs() * tc.half(got.dtype), f"{dt} expert {e}")
