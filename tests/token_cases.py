"""Cases and 64-bit checks of the token operators (include/ymk_tokens.h), shared by tests/test_hostemu_tokens.py (CPU lane emulator) and
tests/test_gpu_tokens.py.  Tolerances: u = 2^-24 is half a step of fp32, `half(t)` half a step of the stored type (relative), and a sum of n fp32
terms is off by at most (its longest chain of additions) * u * (the sum of the terms' magnitudes)."""
import torch

U = 2.0**-24
TINY = {torch.float32: 2.0**-150, torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25}   # half a step of the subnormals


def half(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rows_of(g, M, C, dtype, pad=0, dev="cpu", scale=1.0):
    """[M, C] view with `pad` extra columns of NaN behind every row."""
    buf = torch.full((max(M, 1), C + pad), float("nan"), dtype=dtype)
    buf[:, :C] = (torch.randn((max(M, 1), C), generator=g) * scale).to(dtype)
    return buf.to(dev)[:M, :C]


def close(got, want, tol, what):
    got, want, tol = got.double().cpu(), want.double().cpu(), tol.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol.clamp_min(1e-300))[bad].max()):.3g} x the tolerance"


# ------------------------------------------------------------------------------------------------------------------ norm
# rows, channels, padding of the rows, residual
NORMS = [(1, 1, 0, True), (3, 8, 0, True), (5, 33, 0, False), (70, 64, 8, True), (17, 100, 3, True), (2, 513, 0, True), (9, 1021, 0, True), (3, 2048, 8, True),
         (2, 2056, 0, False), (600, 40, 0, True), (513, 24, 1, True), (0, 16, 0, True)]


def check_norm(ops, dtype, case, dev="cpu", eps=1e-5):
    M, C, pad, res = case
    g = gen(M * 31 + C)
    x, r = rows_of(g, M, C, dtype, pad, dev), rows_of(g, M, C, dtype, 0, dev) if res else None
    w = (1 + 0.3 * torch.randn(C, generator=g)).to(dev)
    y, h, rstd = ops.rms_norm(x, w, eps, residual=r)
    want_h = (x.float() + r.float()).to(dtype) if res else x
    assert torch.equal(h, want_h) and h.dtype == y.dtype == dtype
    h64 = want_h.double().cpu()
    r64 = 1 / (h64.square().mean(-1) + eps).sqrt()
    # longest chain: 32 terms a lane, 10 levels of the tree; half of it reaches the root, and a handful of single roundings follow
    rel = 40 * U
    close(rstd, r64, r64 * rel, "rstd")
    y64 = h64 * r64[:, None] * w.double().cpu()
    close(y, y64, y64.abs() * (half(dtype) * (1 + rel) + rel) + TINY[dtype], "y")
    q, scale, h2 = ops.rms_norm_quant(x, w, eps, residual=r)
    assert torch.equal(h2, want_h) and q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32
    top = y64.abs().amax(-1) if M else y64.new_zeros(0)
    close(scale, top / 448, top / 448 * rel, "scale")
    s = scale.double().cpu()[:, None]
    q64 = q.cpu().double()
    close(q64 * s, y64, torch.maximum(2.0**-4 * y64.abs(), 2.0**-10 * s) * (1 + 2.0**-12) + 2 * rel * y64.abs(), "q")
    assert not M or bool((q64.abs().amax(-1) == 448).all())
    # gradient
    dy, dres = rows_of(g, M, C, dtype, pad, dev), rows_of(g, M, C, dtype, 0, dev)
    dx, dw = ops.rms_norm_backward(dy, h, w, rstd, dres=dres)
    d64, n64, w64 = dy.double().cpu(), h64 * r64[:, None], w.double().cpu()
    g64 = d64 * w64
    gn, gn_abs = ((g64 * n64).mean(-1, keepdim=True), (g64 * n64).abs().mean(-1, keepdim=True)) if M else (g64, g64)
    rr = r64[:, None]
    want = rr * (g64 - n64 * gn) + dres.double().cpu()
    parts = rr * (g64.abs() + n64.abs() * gn_abs) + dres.double().cpu().abs()
    close(dx, want, parts * (120 * U) + want.abs() * half(dtype) + TINY[dtype], "dx")
    # a lane's rows, the groups of a workgroup, the partial rows of the workgroups: fewer than 256 additions in a chain for these sizes and for
    # the largest (200000 rows, four groups a workgroup: 40 a lane, 4 groups, 20 partial rows a strand, 18 levels of the strands' sum); rstd's own error comes on top
    close(dw, (d64 * n64).sum(0), (d64 * n64).abs().sum(0) * ((256 + 40) * U) + 1e-30, "dweight")
    dx2, none = ops.rms_norm_backward(dy, h, w, rstd, need_dweight=False)
    assert none is None
    close(dx2, want - dres.double().cpu(), (parts - dres.double().cpu().abs()) * (120 * U) + want.abs() * half(dtype) + dres.double().cpu().abs() * half(dtype) + TINY[dtype], "dx alone")


def check_norm_in_place(ops, dtype, dev="cpu"):
    """The residual stream updated where it lies: h over residual, and over x."""
    g = gen(5)
    for C in (40, 37, 2100):
        x, r = rows_of(g, 7, C, dtype, 0, dev), rows_of(g, 7, C, dtype, 0, dev)
        w = torch.ones(C, device=dev)
        y, h, _ = ops.rms_norm(x, w, residual=r)
        x1, r1 = x.clone(), r.clone()
        y1, h1, _ = ops.rms_norm(x1, w, residual=r1, residual_out=r1)
        assert h1 is r1 and torch.equal(r1, h) and torch.equal(y1, y) and torch.equal(x1, x)
        q2, s2, h2 = ops.rms_norm_quant(x1, w, residual=r, residual_out=x1)
        assert h2 is x1 and torch.equal(x1, h)


def check_norm_special(ops, dtype, dev="cpu"):
    """All-zero rows, rows with NaN or infinity, rows of the type's smallest values; their neighbours are untouched by them."""
    C = 72
    x = torch.ones(6, C, dtype=dtype, device=dev)
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    x[4] = torch.finfo(dtype).tiny
    w = torch.ones(C, device=dev)
    q, s, _ = ops.rms_norm_quant(x, w, 0.0 if dtype == torch.float32 else 1e-6)
    q, s = q.float().cpu(), s.cpu()
    one = 1.0 if dtype == torch.float32 else float((1 / torch.tensor(1.0 + 1e-6)).sqrt())
    for r in (0, 5):
        assert bool((q[r] == 448).all()) and abs(float(s[r]) - one / 448) < 1e-6
    if dtype != torch.float32:
        assert float(s[1]) == 1.0 and bool((q[1] == 0).all())
    assert bool(torch.isnan(s[2:4]).all()) and bool(torch.isnan(q[2:4]).all())
    y, _, _ = ops.rms_norm(x, w, 1e-6)
    y = y.float().cpu()
    assert bool((y[1] == 0).all()) and bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[3, 7])) and bool(torch.isfinite(y[[0, 4, 5]]).all())


def check_norm_differences(ops, dev="cpu"):
    """<dx, u> and <dweight, v> against central differences of the forward."""
    g = gen(9)
    M, C, eps, d = 4, 48, 1e-5, 2.0**-6
    x, dy = rows_of(g, M, C, torch.float32, 0, dev), rows_of(g, M, C, torch.float32, 0, dev)
    w = (1 + 0.3 * torch.randn(C, generator=g)).to(dev)
    u, v = torch.randn(M, C, generator=g).to(dev), torch.randn(C, generator=g).to(dev)
    loss = lambda x_, w_: float((ops.rms_norm(x_, w_, eps)[0].double() * dy.double()).sum())   # noqa: E731
    _, h, rstd = ops.rms_norm(x, w, eps)
    dx, dw = ops.rms_norm_backward(dy, h, w, rstd)
    # truncation d^2 / 6 times a third derivative of order one a row and unit direction (|u| ~ 7 a row), plus rounding u |L| / d
    assert abs((loss(x + d * u, w) - loss(x - d * u, w)) / (2 * d) - float((dx.double() * u.double()).sum())) < 0.05
    assert abs((loss(x, w + d * v) - loss(x, w - d * v)) / (2 * d) - float((dw.double() * v.double()).sum())) < 0.01


# ---------------------------------------------------------------------------------------------------------------- tokens
# tokens, top_k, experts, share without an expert, int64 indexes
SORTS = [(0, 2, 4, 0.0, False), (1, 1, 1, 0.0, False), (1, 2, 8, 0.0, True), (5, 3, 7, 0.4, False), (300, 2, 16, 0.0, False), (257, 16, 255, 0.1, True), (64, 1, 256, 1.0, False),
         (2048, 2, 5, 0.2, True), (1366, 3, 7, 0.0, False), (4096, 2, 3, 0.0, False), (4097, 2, 5, 0.3, True), (9001, 1, 64, 0.05, False), (5000, 3, 256, 0.5, False), (8200, 1, 1, 0.5, False)]


def make_idx(g, T, K, E, dropped, wide):
    idx = torch.randint(0, E, (T, K), generator=g)
    gone = torch.rand(T, K, generator=g) < dropped
    bad = torch.tensor([-1, E, -2**31, E + 7] + ([2**40, -2**40 + 1] if wide else []))
    idx = torch.where(gone, bad[torch.randint(0, len(bad), (T, K), generator=g)], idx)
    return idx if wide else idx.to(torch.int32)


def sort_oracle(idx, E):
    flat = idx.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.argsort(key, stable=True)
    n = int((key < E).sum())
    src = torch.full((flat.numel(),), -1, dtype=torch.int32)
    src[:n] = order[:n].to(torch.int32)
    row = torch.full((flat.numel(),), -1, dtype=torch.int32)
    row[order[:n]] = torch.arange(n, dtype=torch.int32)
    offsets = torch.zeros(E + 1, dtype=torch.int32)
    offsets[1:] = torch.bincount(key, minlength=E + 1)[:E].cumsum(0).to(torch.int32)
    return offsets, src, row.reshape(idx.shape), n


def check_sort(ops, case, dev="cpu"):
    T, K, E, dropped, wide = case
    idx = make_idx(gen(T + K + E), T, K, E, dropped, wide)
    p = ops.token_sort(idx.to(dev), E)
    offsets, src, row, _ = sort_oracle(idx, E)
    assert torch.equal(p.offsets.cpu(), offsets) and torch.equal(p.src.cpu(), src) and torch.equal(p.row.cpu(), row) and p.experts == E


# tokens, top_k, experts, channels, row padding, share without an expert
MOVES = [(0, 2, 4, 8, 0, 0.0), (1, 1, 2, 8, 0, 0.0), (7, 2, 3, 40, 8, 0.3), (33, 3, 5, 37, 0, 0.2), (16, 16, 20, 24, 4, 0.1), (5, 2, 4, 1, 0, 0.0), (130, 2, 4, 264, 0, 0.5), (4, 4, 4, 16, 0, 1.0), (3, 2, 4, 520, 0, 0.0)]


def check_moves(ops, dtype, case, dev="cpu"):
    import ctypes as C_

    T, K, E, C, pad, dropped = case
    g = gen(T * 7 + C)
    idx = make_idx(g, T, K, E, dropped, False)
    plan = ops.token_sort(idx.to(dev), E)
    _, src, row, n = sort_oracle(idx, E)
    tok = (src[:n] // K).long()
    x = rows_of(g, T, C, dtype, pad, dev)
    xs = ops.token_dispatch(x, plan)
    assert xs.shape == (T * K, C) and torch.equal(xs[:n].cpu(), x.cpu()[tok])
    # rows behind the last expert's, and the padding, stay as they were
    buf = torch.full((T * K, C + 3), 7.0, dtype=dtype, device=dev)
    es = buf.element_size()
    if T == 0:
        assert ops.token_combine(rows_of(g, 0, C, dtype, 0, dev), plan, torch.zeros(0, K, device=dev)).shape == (0, C)
        assert ops.token_combine_backward(x, xs, plan, torch.zeros(0, K, device=dev))[1].shape == (0, K)
        return
    rc = ops.lib.ymk_token_dispatch(C_.c_void_p(x.data_ptr()), (C + pad) * es if T > 1 else C * es, C * es, None, C_.c_void_p(buf.data_ptr()), (C + 3) * es, None,
                                    C_.c_void_p(plan.row.data_ptr()), T, K, ops._stream())
    assert rc == 0 and torch.equal(buf[:n, :C].cpu(), x.cpu()[tok]) and bool((buf[n:] == 7).all()) and bool((buf[:, C:] == 7).all())
    ys = rows_of(g, T * K, C, dtype, pad, dev)
    if n < T * K:
        ys[n:] = float("nan")   # never read
    w = torch.randn(T, K, generator=g)
    w_ = torch.where(row >= 0, w, float("nan")).to(dev)   # nor is the weight of a pair without a row
    kept = (row >= 0)[..., None]
    part = torch.where(kept, ys.double().cpu()[row.clamp_min(0).long()], 0.0)
    y64, mag = (part * w.double()[..., None]).sum(1), (part * w.double()[..., None]).abs().sum(1)
    close(ops.token_combine(ys, plan, w_), y64, mag * (2 * K * U) + y64.abs() * half(dtype) + TINY[dtype], "combine")
    close(ops.token_dispatch_backward(ys, plan), part.sum(1), part.abs().sum(1) * (2 * K * U) + part.sum(1).abs() * half(dtype) + TINY[dtype], "dispatch backward")
    dy = rows_of(g, T, C, dtype, pad, dev)
    dys, dw = ops.token_combine_backward(dy, ys, plan, w_)
    d64 = w.reshape(-1)[src[:n].long()].double()[:, None] * dy.double().cpu()[tok]
    close(dys[:n], d64, d64.abs() * (half(dtype) + U) + TINY[dtype], "dys")
    t = part * dy.double().cpu()[:, None]
    close(dw, t.sum(-1), t.abs().sum(-1) * ((C // 8 + 40) * U) + 1e-30, "dw")


def check_dispatch_8bit(ops, dev="cpu"):
    g = gen(3)
    for C in (16, 40, 33):
        x = torch.randint(0, 255, (9, C), generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn)
        scale = torch.rand(9, generator=g)
        idx = make_idx(g, 9, 2, 4, 0.2, False)
        xs, ss = ops.token_dispatch(x.to(dev), plan := ops.token_sort(idx.to(dev), 4), scale=scale.to(dev))
        _, src, _, n = sort_oracle(idx, 4)
        tok = (src[:n] // 2).long()
        assert torch.equal(xs.view(torch.uint8)[:n].cpu(), x.view(torch.uint8)[tok]) and torch.equal(ss[:n].cpu(), scale[tok]) and plan.experts == 4


# --------------------------------------------------------------------------------------------------------------- product
# rows per expert, rows behind them, Cin, Cout, activation, row padding of x
PRODUCTS = [([0, 0], 0, 16, 24, "silu", 0), ([1], 0, 16, 16, None, 0), ([0, 3, 0, 5], 2, 64, 48, "silu", 16), ([130, 0, 1, 37], 3, 80, 144, "gelu", 0), ([5, 129], 0, 208, 16, "sigmoid", 0),
            ([0, 0], 4, 32, 32, None, 0), ([64, 20], 0, 144, 272, None, 16)]


def act64(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.5**0.5))
    return torch.sigmoid(v) if act == "sigmoid" else v


def make_offsets(counts, start=0):
    return torch.tensor([start] + (start + torch.tensor(counts).cumsum(0)).tolist(), dtype=torch.int32)


def check_product(ops, dtype, case, dev="cpu", bias=True, start=0, out_dtype=None):
    counts, behind, Cin, Cout, act, pad = case
    g = gen(sum(counts) + Cin * 3 + Cout)
    E, used = len(counts), sum(counts)
    off = make_offsets(counts, start)
    rows = start + used + behind
    f8 = dtype == torch.float8_e4m3fn
    b = 0.2 * torch.randn(E, Cout, generator=g)
    live = torch.zeros(rows, dtype=torch.bool)
    live[start:start + used] = True
    if f8:
        x32, w32 = torch.randn(rows, Cin, generator=g), torch.randn(E, Cout, Cin, generator=g)
        xs, ws = x32.abs().amax(-1) / 448, w32.abs().amax(-1) / 448
        x, w = (x32 / xs[:, None]).to(dtype), (w32 / ws[..., None]).to(dtype)
        x.view(torch.uint8)[~live] = 0x7f   # NaN
        x64, w64 = x.double() * xs.double()[:, None], w.double() * ws.double()[..., None]
        buf = torch.full((rows, Cin + pad), 0x7f, dtype=torch.uint8)
        buf[:, :Cin] = x.view(torch.uint8)
        xd, wd = buf.view(dtype).to(dev)[:, :Cin], w.to(dev)
        y = ops.expert_linear(xd, wd, off.to(dev), b.to(dev) if bias else None, act=act, x_scale=xs.to(dev), w_scale=ws.to(dev), out_dtype=out_dtype)
        odt = out_dtype or torch.bfloat16
    else:
        xd = rows_of(g, rows, Cin, dtype, pad, dev)
        xd[~live.to(dev)] = float("nan")
        w = (torch.randn(E, Cout, Cin, generator=g) * Cin**-0.5).to(dtype)
        x64, w64, wd, odt = xd.double().cpu(), w.double(), w.to(dev), dtype
        y = ops.expert_linear(xd, wd, off.to(dev), b.to(dev) if bias else None, act=act)
    assert y.dtype == odt and y.shape == (rows, Cout)
    for e, n in enumerate(counts):
        s = slice(int(off[e]), int(off[e]) + n)
        v = x64[s] @ w64[e].t()
        mag = x64[s].abs() @ w64[e].abs().t() + 1
        if bias:
            v = v + b[e].double()
        want = act64(v, act)
        if f8 and len(v):
            # The 8-bit matrix instruction adds 16 products at the largest one's exponent and drops what lies below 2^-13 of it (1 - 1 + 2^-12 gives
            # 2^-12, 1 - 1 + 2^-14 gives 0, in 16 places of K; in different 16 both survive).  So a product loses less than 2^-12 of the group's
            # largest, and a 64-deep instruction less than 4 * 15 * 2^-12 of the largest of its 64.
            p = (x64[s][:, None] * w64[e][None]).abs()
            p = torch.nn.functional.pad(p, (0, -Cin % 64)).unflatten(-1, (-1, 64)).amax(-1).sum(-1)
            mag = mag + p * (60 * 2.0**-12) / (U * (Cin + 8))
        # (Cin + 8) additions and scalings before the activation, whose slope is at most 1.13 and which adds a few roundings of its own
        close(y[s], want, mag * (1.13 * (Cin + 8) + 8) * U + want.abs() * half(odt) + TINY[odt], f"expert {e}")


def check_product_exact(ops, case, dev="cpu"):
    """8-bit codes whose products span fewer bits than the instruction keeps, and scales that are powers of two: every sum is exact, so is the output."""
    counts, behind, Cin, Cout, _, _ = case
    g = gen(Cin + Cout)
    E, rows = len(counts), sum(counts) + behind
    pick = lambda *s: (torch.randint(8, 16, s, generator=g) * torch.tensor([0.125, 0.25, -0.25])[torch.randint(0, 3, s, generator=g)]).to(torch.float8_e4m3fn)   # noqa: E731
    x, w = pick(rows, Cin), pick(E, Cout, Cin)
    xs, ws = 2.0 ** torch.randint(-3, 3, (rows,), generator=g).float(), 2.0 ** torch.randint(-3, 3, (E, Cout), generator=g).float()
    off = make_offsets(counts)
    y = ops.expert_linear(x.to(dev), w.to(dev), off.to(dev), x_scale=xs.to(dev), w_scale=ws.to(dev), out_dtype=torch.float32).cpu()
    for e, n in enumerate(counts):
        s = slice(int(off[e]), int(off[e]) + n)
        assert torch.equal(y[s].double(), (x[s].double() @ w[e].double().t()) * xs[s].double()[:, None] * ws[e].double()), e


def check_product_gradient(ops, dtype, case, dev="cpu", dw_dtype=None):
    counts, behind, Cin, Cout, _, pad = case
    g = gen(sum(counts) + Cin + Cout * 5)
    E, used = len(counts), sum(counts)
    off = make_offsets(counts)
    rows = used + behind
    x, dy = rows_of(g, rows, Cin, dtype, pad, dev), rows_of(g, rows, Cout, dtype, pad, dev)
    if behind:
        x[used:], dy[used:] = float("nan"), float("nan")
    w = (torch.randn(E, Cout, Cin, generator=g) * Cin**-0.5).to(dtype).to(dev)
    dx, dw, db = ops.expert_linear_backward(dy, x, w, off.to(dev), dw_dtype=dw_dtype)
    odt = dw_dtype or dtype
    assert dx.dtype == dtype and dw.dtype == odt and db.dtype == torch.float32
    x64, d64, w64 = x.double().cpu(), dy.double().cpu(), w.double().cpu()
    for e, n in enumerate(counts):
        s = slice(int(off[e]), int(off[e]) + n)
        want = d64[s] @ w64[e]
        close(dx[s], want, (d64[s].abs() @ w64[e].abs()) * ((Cout + 8) * U) + want.abs() * half(dtype) + TINY[dtype], f"dx {e}")
        want = d64[s].t() @ x64[s]
        close(dw[e], want, (d64[s].abs().t() @ x64[s].abs()) * ((n + 8) * U) + want.abs() * half(odt) + TINY[odt], f"dw {e}")
        close(db[e], d64[s].sum(0), d64[s].abs().sum(0) * ((n + 8) * U) + 1e-30, f"db {e}")
    only = ops.expert_linear_backward(dy, x, w, off.to(dev), need_dx=False, need_db=False, dw_dtype=dw_dtype)
    assert only[0] is None and only[2] is None and torch.equal(only[1], dw)


# -------------------------------------------------------------------------------------------- as they are used together
def expert_block(ops, x, res, p, K, dtype):
    """A pre-norm expert layer of a serving program: residual sum, norm, routing, two products with an activation, and back."""
    y, h, _ = ops.rms_norm(x, p["norm"], residual=res)
    score = (y.float() @ p["router"]).softmax(-1)
    gate, idx = score.topk(K, dim=-1)
    plan = ops.token_sort(idx, p["w1"].shape[0])
    a = ops.expert_linear(ops.token_dispatch(y, plan), p["w1"], plan.offsets, p["b1"], act="gelu")
    return ops.token_combine(ops.expert_linear(a, p["w2"], plan.offsets, p["b2"]), plan, gate.contiguous()), h, plan, gate, y, a


def block_params(g, C, H, E, dtype, dev):
    r = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    return {"norm": (1 + 0.1 * r(C)).to(dev), "router": (r(C, E) * C**-0.5).to(dev), "w1": (r(E, H, C) * C**-0.5).to(dtype).to(dev), "b1": (0.1 * r(E, H)).to(dev),
            "w2": (r(E, C, H) * H**-0.5).to(dtype).to(dev), "b2": (0.1 * r(E, C)).to(dev)}


def check_block(ops, dtype, dev="cpu", T=23, C=64, H=128, E=5, K=2):
    g = gen(T + C)
    x, res, p = rows_of(g, T, C, dtype, 0, dev), rows_of(g, T, C, dtype, 0, dev), block_params(g, C, H, E, dtype, dev)
    out, h, plan, gate, y, a = expert_block(ops, x, res, p, K, dtype)
    d = {k: v.double().cpu() for k, v in p.items()}
    y64 = y.double().cpu()   # the router's choice is taken as made: it depends on the norm's rounding
    row, src = plan.row.cpu().long(), plan.src.cpu().long()
    off = plan.offsets.cpu()
    e = torch.bucketize(row.reshape(-1), off[1:].long(), right=True).reshape(row.shape)
    want = torch.zeros(T, C, dtype=torch.float64)
    mag = torch.zeros(T, C, dtype=torch.float64)
    for k in range(K):
        for t in range(T):
            a64 = act64(d["w1"][e[t, k]] @ y64[t] + d["b1"][e[t, k]], "gelu")
            z = d["w2"][e[t, k]] @ a64 + d["b2"][e[t, k]]
            want[t] += gate[t, k].double().cpu() * z
            # the hidden row is rounded once, its products add up; the expert's answer is rounded once
            mag[t] += gate[t, k].double().cpu() * (d["w2"][e[t, k]].abs() @ a64.abs() + z.abs())
    close(out, want, mag * (half(dtype) * 1.2 + (C + H + 32) * U) + want.abs() * half(dtype) + TINY[dtype], "block")
    assert torch.equal(h, (x.float() + res.float()).to(dtype)) and int(off[-1]) == T * K and torch.equal(src.sort().values, torch.arange(T * K))


def check_block_gradient(ops, dev="cpu", T=11, C=32, H=48, E=3, K=2):
    """The gradients chained by hand, in fp32, against autograd of the same block in 64 bits."""
    g = gen(77)
    x, res, p = rows_of(g, T, C, torch.float32, 0, dev), rows_of(g, T, C, torch.float32, 0, dev), block_params(g, C, H, E, torch.float32, dev)
    y, h, rstd = ops.rms_norm(x, p["norm"], residual=res)
    gate = torch.rand(T, K, generator=g).to(dev)
    idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).to(dev)
    plan = ops.token_sort(idx, E)
    xs = ops.token_dispatch(y, plan)
    a1 = ops.expert_linear(xs, p["w1"], plan.offsets, p["b1"])
    a = a1 * torch.sigmoid(a1)
    z = ops.expert_linear(a, p["w2"], plan.offsets, p["b2"])
    out = ops.token_combine(z, plan, gate)
    dout = torch.randn(T, C, generator=g).to(dev)
    dz, dgate = ops.token_combine_backward(dout, z, plan, gate)
    da, dw2, db2 = ops.expert_linear_backward(dz, a, p["w2"], plan.offsets)
    s = torch.sigmoid(a1)
    da1 = da * (s * (1 + a1 * (1 - s)))
    dxs, dw1, db1 = ops.expert_linear_backward(da1, xs, p["w1"], plan.offsets)
    dx, dnorm = ops.rms_norm_backward(ops.token_dispatch_backward(dxs, plan), h, p["norm"], rstd, dres=dout)   # out + h leave the block
    q = {k: v.double().cpu().requires_grad_(True) for k, v in p.items() if k != "router"}
    x64, gate64 = x.double().cpu().requires_grad_(True), gate.double().cpu().requires_grad_(True)
    h64 = x64 + res.double().cpu()
    y64 = h64 * (h64.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * q["norm"]
    ref = torch.zeros(T, C, dtype=torch.float64)
    for k in range(K):
        e = idx[:, k].cpu()
        v = torch.nn.functional.silu((q["w1"][e] @ y64[..., None])[..., 0] + q["b1"][e])
        ref = ref + gate64[:, k, None] * ((q["w2"][e] @ v[..., None])[..., 0] + q["b2"][e])
    ((ref + h64) * dout.double().cpu()).sum().backward()
    # a chain of five fp32 operators, each within (its length + 40) u of its terms' magnitudes, whose sums exceed the results by some tens here
    for got, want, what in ((out, ref.detach(), "out"), (dx, x64.grad, "dx"), (dnorm, q["norm"].grad, "dnorm"), (dgate, gate64.grad, "dgate"), (dw1, q["w1"].grad, "dw1"),
                            (db1, q["b1"].grad, "db1"), (dw2, q["w2"].grad, "dw2"), (db2, q["b2"].grad, "db2")):
        close(got, want, torch.full_like(want, 5 * 128 * 40 * U * float(want.abs().max())), what)


def check_plans_of_ones_own(ops, dev="cpu"):
    """A plan with rows outside the pairs (it did not come from token_sort): nothing is read or written there, those pairs have no row."""
    T, K, C = 6, 2, 40
    row = torch.tensor([[0, 12], [1, -1], [-7, 2**31 - 1], [3, 4], [-2**31, 5], [11, 2]], dtype=torch.int32)
    good = (row >= 0) & (row < T * K)
    plan = ops.TokenPlan(torch.zeros(3, dtype=torch.int32, device=dev), torch.zeros(T * K, dtype=torch.int32, device=dev), row.to(dev), 2)
    g = gen(8)
    x, ys, w = rows_of(g, T, C, torch.float32, 0, dev), rows_of(g, T * K, C, torch.float32, 0, dev), torch.rand(T, K, generator=g).to(dev)
    xs = ops.token_dispatch(x, plan)
    at = row[good].long()
    assert torch.equal(xs.cpu()[at], x.cpu()[:, None].expand(T, K, C)[good])
    part = torch.where(good[..., None], ys.cpu().double()[row.clamp(0, T * K - 1).long()], 0.0)
    close(ops.token_combine(ys, plan, w), (part * w.cpu().double()[..., None]).sum(1), torch.full((T, C), 1e-5), "combine")
    dys, dw = ops.token_combine_backward(x, ys, plan, w)
    close(dw, (part * x.cpu().double()[:, None]).sum(-1), torch.full((T, K), 1e-4), "dw")
    close(dys.cpu()[at], (w.cpu()[..., None] * x.cpu()[:, None])[good].double(), torch.full((len(at), C), 1e-6), "dys")


def check_views(ops, dtype, dev="cpu"):
    """Views that begin at any element, of one row, of three dims, and with rows far apart: the same bits as their dense copies."""
    g = gen(21)
    buf = torch.randn(9, 3, 70, generator=g).to(dtype).to(dev)
    w = torch.rand(41, generator=g).to(dev)
    for v in (buf[:, 1, 1:42], buf[:, :, 3:44], buf[2:3, 2, 5:46], buf[::2, 0, 7:48], buf[0, :, 29:]):
        c = v.contiguous()
        y, h, rstd = ops.rms_norm(v, w, residual=v)
        y2, h2, rstd2 = ops.rms_norm(c, w, residual=c)
        assert y.shape == v.shape and rstd.shape == v.shape[:-1] and torch.equal(y, y2) and torch.equal(h, h2) and torch.equal(rstd, rstd2)
        q, s, _ = ops.rms_norm_quant(v, w)
        q2, s2, _ = ops.rms_norm_quant(c, w)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
        dx, dw = ops.rms_norm_backward(v, h, w, rstd, dres=v)
        dx2, dw2 = ops.rms_norm_backward(c, h2, w, rstd2, dres=c)
        assert torch.equal(dx, dx2) and torch.equal(dw, dw2)
        M = c.numel() // 41
        plan = ops.token_sort((torch.arange(M)[:, None] % 3).to(torch.int32).to(dev), 3)
        xs = ops.token_dispatch(v, plan)
        assert torch.equal(xs, c.reshape(M, 41)[plan.src.long()])
        assert torch.equal(ops.token_dispatch_backward(v, plan), c.reshape(M, 41)[plan.row[:, 0].long()])
        gate = torch.ones(M, 1, device=dev)
        a, b = ops.token_combine_backward(v, v, plan, gate), ops.token_combine_backward(c, c, plan, gate)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# rows per expert, rows behind them, Cin, Cout: few rows (under 32 an expert, where 16-bit outputs come from 32-bit sums too), and many
DEEP_FEW = [([1], 0, 16, 8), ([3, 0, 5, 1], 2, 1024, 48), ([2, 2, 0, 7], 0, 336, 136), ([16], 1, 1008, 40), ([9, 0, 70, 20], 0, 272, 72)]
DEEP_MANY = [([130, 0, 1, 37], 3, 80, 144), ([64, 20], 0, 1024, 264), ([400, 301], 1, 496, 520)]


def check_product_deep_sums(ops, case, out_dtype, dev="cpu"):
    """8-bit products of -2^14 .. 2^14, whole numbers whose sums stay below 2^24: a sum held in 32 bits is exact in any order, and the output is that sum
    rounded once (scales are powers of two).  Products that cancel leave the small ones, which an addition at fewer bits loses."""
    counts, behind, Cin, Cout = case
    g = gen(Cin * 5 + Cout)
    E, rows = len(counts), sum(counts) + behind
    whole = torch.arange(1, 129).float()
    whole = whole[whole.to(torch.float8_e4m3fn).float() == whole]
    pick = lambda *s: (whole[torch.randint(0, len(whole), s, generator=g)] * (2.0 * torch.randint(0, 2, s, generator=g) - 1))   # noqa: E731
    x, w = pick(rows, Cin), pick(E, Cout, Cin)
    x[:, 1:8:2], w[..., 1:8:2] = x[:, :8:2], -w[..., :8:2]   # neighbours cancel
    x, w = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    assert float((x.double().abs().max() * w.double().abs().max()) * Cin) <= 2.0**24
    xs, ws = 2.0 ** torch.randint(-12, -9, (rows,), generator=g).float(), 2.0 ** torch.randint(-6, 0, (E, Cout), generator=g).float()
    off = make_offsets(counts)
    y = ops.expert_linear(x.to(dev), w.to(dev), off.to(dev), x_scale=xs.to(dev), w_scale=ws.to(dev), out_dtype=out_dtype).cpu()
    for e, n in enumerate(counts):
        s = slice(int(off[e]), int(off[e]) + n)
        want = (x[s].double() @ w[e].double().t()) * xs[s].double()[:, None] * ws[e].double()
        assert torch.equal(y[s], want.to(out_dtype)), (e, float((y[s].double() - want).abs().max()))


def check_empty_batches(ops, dtype, dev="cpu"):
    """No rows, in batches of any rank: outputs of the same rank without rows, zero sums over none of them."""
    C, E, K = 16, 3, 2
    w = torch.ones(C, device=dev)
    wt = torch.ones(E, 8, C, dtype=dtype, device=dev)
    plan = ops.token_sort(torch.zeros(0, K, dtype=torch.int32, device=dev), E)
    gate = torch.zeros(0, K, device=dev)
    for shape in ((0, C), (2, 0, C), (0, 2, C), (3, 0, 5, C), (2, 3, 0, C), (1, 0, 1, C)):
        for x in (torch.zeros(shape, dtype=dtype, device=dev), torch.zeros(*shape[:-1], 2 * C, dtype=dtype, device=dev)[..., :C]):
            y, h, rstd = ops.rms_norm(x, w, residual=x)
            assert y.shape == h.shape == shape and rstd.shape == shape[:-1]
            q, scale, _ = ops.rms_norm_quant(x, w, residual=x, residual_out=h)
            assert q.shape == shape and scale.shape == shape[:-1]
            dx, dw = ops.rms_norm_backward(x, h, w, rstd, dres=x)
            assert dx.shape == shape and torch.equal(dw, torch.zeros_like(w))
            assert ops.token_dispatch(x, plan).shape == (0, C) and ops.token_dispatch_backward(x, plan).shape == (0, C)
            assert ops.token_combine(x, plan, gate).shape == (0, C) and ops.token_combine_backward(x, x, plan, gate)[0].shape == (0, C)
            off = torch.zeros(E + 1, dtype=torch.int32, device=dev)
            assert ops.expert_linear(x, wt, off).shape == (0, 8)
            dx, dw, db = ops.expert_linear_backward(torch.zeros(0, 8, dtype=dtype, device=dev), x, wt, off)
            assert dx.shape == (0, C) and torch.equal(dw, torch.zeros_like(wt)) and torch.equal(db, torch.zeros(E, 8, device=dev))


def check_residual_out_beside(ops, dtype, dev="cpu"):
    """h written to the other part of the rows that x or the residual lies in: no element is shared, and nothing else of the buffer changes."""
    g = gen(31)
    w = torch.rand(40, generator=g).to(dev)
    for T, width, at, to in ((5, 80, 0, 40), (5, 80, 40, 0), (7, 123, 3, 83), (1, 80, 0, 40), (6, 200, 100, 17)):
        buf = torch.randn(T, width, generator=g).to(dtype).to(dev)
        other = rows_of(g, T, 40, dtype, 0, dev)
        for swap in (False, True):
            b = buf.clone()
            x, r = (other, b[:, at:at + 40]) if swap else (b[:, at:at + 40], other)
            y, h, rstd = ops.rms_norm(x.clone(), w, residual=r.clone())
            y2, h2, rstd2 = ops.rms_norm(x, w, residual=r, residual_out=b[:, to:to + 40])
            want = buf.clone()
            want[:, to:to + 40] = h
            assert torch.equal(y, y2) and torch.equal(h, h2) and torch.equal(rstd, rstd2) and torch.equal(b, want)


def check_activations(ops, dtype, act, rows, out_dtype=None, dev="cpu"):
    """act of sums that are not finite, huge, tiny, and in the tails: the bias alone makes them (x is zero).  Not-a-number and infinities come out where the
    definition has them.  Finite values: short forms (16-bit outputs) round the exponent's argument, at most 89 here, to half of 2^-17, and their
    reciprocal gives zero for results below 2^-118; exact ones (fp32) add 1 + erf to half of 2^-23 and multiply by v / 2."""
    inf, nan = float("inf"), float("nan")
    b = torch.cat([torch.tensor([inf, -inf, nan, 0.0, -0.0, 1e30, -1e30, 3e38, -3e38, 6e4, -6e4, 1e-30, -1e-30]), torch.linspace(-100, 100, 203)])
    E, Cin, Cout = 1, 16, b.numel()
    f8 = dtype == torch.float8_e4m3fn
    x, w = torch.zeros(rows, Cin, dtype=dtype, device=dev), torch.ones(E, Cout, Cin).to(dtype).to(dev)
    scales = {"x_scale": torch.ones(rows, device=dev), "w_scale": torch.ones(E, Cout, device=dev), "out_dtype": out_dtype} if f8 else {}
    y = ops.expert_linear(x, w, make_offsets([rows]).to(dev), b[None].to(dev), act=act, **scales).cpu()
    odt = out_dtype or dtype
    v = b.double()
    want = 0.5 * v * torch.special.erfc(-v * 0.5**0.5) if act == "gelu" else act64(v, act)   # 1 + erf would leave 2^-53 of the tail
    stored = want.to(odt)
    for r in range(rows):
        assert torch.equal(torch.isnan(y[r]), torch.isnan(stored)), (r, b[torch.isnan(y[r]) != torch.isnan(stored)])
        assert torch.equal(torch.isinf(y[r]), torch.isinf(stored)) and torch.equal(y[r][torch.isinf(stored)], stored[torch.isinf(stored)])
        f = torch.isfinite(stored)
        tol = want.abs() * (half(odt) + (2.0**-17 if half(odt) > U else 8 * U)) + TINY[odt] + (2.0**-118 if half(odt) > U else 0.0)
        if half(odt) == U:
            tol = tol + v.abs().clamp_max(1e30) * (2 * U) * (v < 0) + 2.0**-126
        close(y[r][f], want[f], tol[f], f"{act} row {r}")


def check_product_small_scales(ops, counts, dev="cpu"):
    """Scales whose product is no normal number while the sum's is one: each is multiplied in for itself."""
    Cin, Cout, E = 4096, 16, len(counts)
    rows = sum(counts)
    x, w = torch.full((rows, Cin), 448.0).to(torch.float8_e4m3fn), torch.full((E, Cout, Cin), 448.0).to(torch.float8_e4m3fn)
    xs, ws = torch.full((rows,), 3e-23), torch.full((E, Cout), 3.1e-23)
    want = 448.0**2 * Cin * float(xs[0]) * float(ws[0, 0])
    for dtype in (torch.float32, torch.bfloat16):
        y = ops.expert_linear(x.to(dev), w.to(dev), make_offsets(counts).to(dev), x_scale=xs.to(dev), w_scale=ws.to(dev), out_dtype=dtype)
        close(y, torch.full((rows, Cout), want, dtype=torch.float64), torch.full((rows, Cout), want * (half(dtype) + (Cin + 8) * U)), "small scales")


def check_product_exact_16(ops, counts, Cin, Cout, out_dtype, dev="cpu"):
    """check_product_exact with a 16-bit output: products span 10 bits, fewer than the 8-bit instruction keeps, so the output is the exact sum rounded once."""
    g = gen(Cin * 3 + Cout)
    E, rows = len(counts), sum(counts) + 2
    pick = lambda *s: (torch.randint(8, 16, s, generator=g) * torch.tensor([0.125, 0.25, -0.25])[torch.randint(0, 3, s, generator=g)]).to(torch.float8_e4m3fn)   # noqa: E731
    x, w = pick(rows, Cin), pick(E, Cout, Cin)
    xs, ws = 2.0 ** torch.randint(-3, 3, (rows,), generator=g).float(), 2.0 ** torch.randint(-3, 3, (E, Cout), generator=g).float()
    off = make_offsets(counts)
    y = ops.expert_linear(x.to(dev), w.to(dev), off.to(dev), x_scale=xs.to(dev), w_scale=ws.to(dev), out_dtype=out_dtype).cpu()
    for e, n in enumerate(counts):
        s = slice(int(off[e]), int(off[e]) + n)
        want = (x[s].to(dev).double() @ w[e].to(dev).double().t()).cpu() * xs[s].double()[:, None] * ws[e].double()
        assert torch.equal(y[s], want.to(out_dtype)), e


def check_norm_aliases(ops, dtype, dev="cpu"):
    """The C functions' outputs over their inputs, same stride: y over x or residual beside h over the other one, codes apart; dx over dy, h and dres."""
    g = gen(41)
    dt, s, lib = ops.DT[dtype], ops._stream(), ops._lib_for(dtype)
    for M, C, pad in ((5, 3, 0), (7, 37, 5), (9, 40, 0), (70, 64, 8), (3, 1021, 2), (6, 2100, 0)):
        ld = C + pad
        new = lambda: rows_of(g, M, C, dtype, pad, dev)   # noqa: E731
        x, r, w = new(), new(), (1 + 0.1 * torch.randn(C, generator=g)).to(dev)
        y, h, rstd = ops.rms_norm(x, w, residual=r)
        copy = lambda t: torch.empty(M, ld, dtype=dtype, device=dev)[:, :C].copy_(t)   # noqa: E731
        for swap in (False, True):
            a, b = copy(x), copy(r)
            ho, yo = (b, a) if swap else (a, b)
            assert lib.ymk_rms_norm(dt, a.data_ptr(), ld, b.data_ptr(), ld, ho.data_ptr(), ld, yo.data_ptr(), ld, None, M, C, w.data_ptr(), 1e-6, s) == 0
            assert torch.equal(ho, h) and torch.equal(yo, y), (C, swap)
        a = copy(x)
        assert lib.ymk_rms_norm(dt, a.data_ptr(), ld, None, 0, None, 0, a.data_ptr(), ld, None, M, C, w.data_ptr(), 1e-6, s) == 0
        assert torch.equal(a, ops.rms_norm(x, w)[0])
        dy, dres = new(), new()
        dx, _ = ops.rms_norm_backward(dy, h, w, rstd, dres=dres, need_dweight=False)
        for i in range(3):
            t = [copy(v) for v in (dy, h, dres)]
            assert lib.ymk_rms_norm_backward(dt, t[0].data_ptr(), ld, t[1].data_ptr(), ld, rstd.data_ptr(), w.data_ptr(), t[2].data_ptr(), ld, t[i].data_ptr(), ld, None, M, C, None, 0, s) == 0
            assert torch.equal(t[i], dx), (C, i)


def check_long_bias_sums(ops, dtype, counts, value, dev="cpu"):
    """db of many rows of one value, where a running fp32 sum grows until each addition loses the value's last bits.  Four steps of a lane are a chain of 64
    additions (of two 16-bit values at a time, one rounding each), each off by at most u of the sum of magnitudes so far; these sums are added with their rounding
    errors kept, which leaves a few u: 64 + 8."""
    E, Cin, Cout = len(counts), 16 // torch.empty(0, dtype=dtype).element_size(), 8
    rows = sum(counts)
    x, dy = torch.ones(rows, Cin, dtype=dtype, device=dev), torch.full((rows, Cout), value, device=dev).to(dtype)
    dy[:, 1::2] *= -1
    _, _, db = ops.expert_linear_backward(dy, x, torch.ones(E, Cout, Cin, dtype=dtype, device=dev), make_offsets(counts).to(dev), need_dx=False)
    want = torch.tensor(counts, dtype=torch.float64)[:, None] * dy[:1].double().cpu()
    close(db, want, want.abs() * (72 * U), "db")


def check_bias_sums_that_are_not_finite(ops, dtype, dev="cpu"):
    inf, nan = float("inf"), float("nan")
    n, Cin, Cout = 300, 8, 8
    dy = torch.ones(n, Cout, dtype=dtype)
    dy[70, 0], dy[3, 1], dy[5, 2], dy[250, 3], dy[40, 3], dy[:, 4] = inf, -inf, nan, inf, -inf, torch.finfo(dtype).max
    x = torch.ones(n, Cin, dtype=dtype)
    _, _, db = ops.expert_linear_backward(dy.to(dev), x.to(dev), torch.ones(1, Cout, Cin, dtype=dtype, device=dev), make_offsets([n]).to(dev), need_dx=False)
    want = dy.double().sum(0).float()
    db = db[0].cpu()
    assert torch.equal(torch.isnan(db), torch.isnan(want)) and torch.equal(db[torch.isinf(want)], want[torch.isinf(want)]), (db, want)
    f = torch.isfinite(want)
    close(db[f], want[f], want[f].double().abs() * (72 * U), "db")


def check_long_weight_sums(ops, dtype, counts, value, dev="cpu", dw_dtype=None):
    """dW of many rows of one value: blocks of 512 rows are chains of 256 additions (of two products each) or fewer, the blocks a chain of their own; each addition is
    off by half a step of the running sum.  One chain over all the rows would lose the value's last bits at every step."""
    E, Cin, Cout = len(counts), 24, 40
    rows = sum(counts)
    x, dy = torch.ones(rows, Cin, dtype=dtype, device=dev), torch.full((rows, Cout), value, device=dev).to(dtype)
    dy[:, 1::2] *= -1
    _, dw, _ = ops.expert_linear_backward(dy, x, torch.ones(E, Cout, Cin, dtype=dtype, device=dev), make_offsets(counts).to(dev), need_dx=False, dw_dtype=dw_dtype)
    for e, n in enumerate(counts):
        want = (n * dy[0].double().cpu())[:, None].expand(Cout, Cin)
        close(dw[e], want, want.abs() * ((256 + n // 512 + 8) * U + (half(dw.dtype) if dw.dtype != torch.float32 else 0.0)), f"dw {e}")


def check_long_products(ops, rows, K, dev="cpu"):
    """y and dx in fp32 over K channels of one value, as check_long_weight_sums does with rows."""
    off = make_offsets([rows, 0, 1]).to(dev)
    one, many = torch.ones(rows + 1, K, device=dev), torch.full((3, 8, K), 1.0001, device=dev)
    y = ops.expert_linear(one, many, off)
    dx, _, _ = ops.expert_linear_backward(one, torch.ones(rows + 1, 8, device=dev), many.transpose(1, 2).contiguous(), off, need_dw=False, need_db=False)
    want = torch.full((rows + 1, 8), K, dtype=torch.float64) * float(many[0, 0, 0])
    for got, what in ((y, "y"), (dx, "dx")):
        close(got, want, want * ((256 + K // 512 + 8) * U), what)
