"""Measured cases of the token operators: the normalisation that precedes a layer of routed experts, the tokens' way to their experts and back, and the
experts' product, each with its gradient and with its form for 8-bit data.

    rms_norm, rms_norm_quant, rms_norm_backward      residual sum + root-mean-square norm, output in the input's type or in e4m3 with a scale per row
    token_sort, token_dispatch, token_combine        rows sorted by expert (stable), moved there and back, weights applied; *_backward their gradients
    expert_linear, expert_linear_backward            y[r] = act(x[r] W[e]^T + b[e]) for the rows r of expert e, with dx, dW and db

`run` computes one pass, in the plain form below or (own = True) through yolo_master_amd.ops."""
import math

import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}
TOP = 448.0  # the largest finite e4m3 value
MOST_FLOPS, MOST_BYTES = 1.2e12, 2.0e9


def listed():
    return [
        # the residual sum, norm and 8-bit output in front of an expert layer, for a handful of tokens: all latency
        {"name": "norm_quant_decode", "op": "norm_quant", "dtype": "bf16", "rows": 4, "cols": 4096},
        # the same for a batch of images' tokens (64 maps of 20 x 20 and more) at a language model's width
        {"name": "norm_quant_batch", "op": "norm_quant", "dtype": "bf16", "rows": 25600, "cols": 2048},
        # forward and backward over the tokens of 64 maps of 40 x 40 at the detector's width
        {"name": "norm_grad_maps", "op": "norm_grad", "dtype": "bf16", "rows": 102400, "cols": 256},
        # an odd width that no vector load divides, in full precision
        {"name": "norm_grad_odd_f32", "op": "norm_grad", "dtype": "f32", "rows": 2041, "cols": 1021},
        # two of eight experts for a few tokens: latency of the sort and of both moves
        {"name": "tokens_decode", "op": "tokens", "dtype": "bf16", "tokens": 8, "cols": 2048, "experts": 8, "top_k": 2, "dropped": 0.0},
        # training: 16 maps of 40 x 40, two of sixteen experts, some pairs dropped by a threshold
        {"name": "tokens_grad_maps", "op": "tokens_grad", "dtype": "bf16", "tokens": 25600, "cols": 512, "experts": 16, "top_k": 2, "dropped": 0.1},
        # a long prompt in 8 bits, many experts
        {"name": "tokens_e4m3_prompt", "op": "tokens", "dtype": "e4m3", "tokens": 16383, "cols": 2048, "experts": 64, "top_k": 6, "dropped": 0.0},
        # a few tokens through eight experts' first layer: the weights' bytes count
        {"name": "product_decode", "op": "product", "dtype": "bf16", "tokens": 8, "cin": 2048, "cout": 4096, "experts": 8, "top_k": 2, "act": "gelu"},
        # the same for one token, in 8 bits, of many experts
        {"name": "product_e4m3_decode", "op": "product", "dtype": "e4m3", "tokens": 1, "cin": 4096, "cout": 2048, "experts": 64, "top_k": 6, "act": "silu"},
        # full precision, the experts of one image's map, a training step
        {"name": "product_grad_f32", "op": "product_grad", "dtype": "f32", "tokens": 1601, "cin": 256, "cout": 520, "experts": 16, "top_k": 2, "act": ""},
        # a training step of a wide expert layer
        {"name": "product_grad_train", "op": "product_grad", "dtype": "bf16", "tokens": 16384, "cin": 1024, "cout": 4096, "experts": 8, "top_k": 2, "act": ""},
        # a long prompt in 8 bits
        {"name": "product_e4m3_prompt", "op": "product", "dtype": "e4m3", "tokens": 16383, "cin": 2048, "cout": 4096, "experts": 32, "top_k": 4, "act": "silu"},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_quant", "norm_grad", "tokens", "tokens_grad", "product", "product_grad"])
    if op.startswith("norm"):
        c = {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "rows": _spread(rng, 1, 200000), "cols": _spread(rng, 24, 8192)}
        if rng.random() < 0.5:
            c["cols"] = -(-c["cols"] // 8) * 8
        c["rows"] = max(1, min(c["rows"], int(MOST_BYTES / 10 / (c["cols"] * SIZE[c["dtype"]]))))
        return c
    experts = _spread(rng, 2, 128)
    c = {"op": op, "tokens": _spread(rng, 1, 65536), "experts": experts, "top_k": rng.randint(1, min(8, experts))}
    c["dtype"] = rng.choice(["bf16", "f16", "f32"] if op.endswith("grad") else ["bf16", "f16", "f32", "e4m3"])
    if op.startswith("tokens"):
        c["cols"] = _spread(rng, 24, 6144)
        if rng.random() < 0.7:
            c["cols"] = -(-c["cols"] // 16) * 16
        c["dropped"] = rng.choice([0.0, 0.05, 0.5])
        c["tokens"] = max(1, min(c["tokens"], int(MOST_BYTES / 2 / (c["cols"] * SIZE[c["dtype"]] * (3 + 6 * c["top_k"])))))
        return c
    c["cin"], c["cout"] = (16 * max(1, _spread(rng, 4, 256)) for _ in range(2))
    if c["dtype"] != "e4m3" and rng.random() < 0.5:  # rows of an odd number of 16-byte pieces
        c["cin"] += 8
    c["act"] = "" if op.endswith("grad") else rng.choice(["", "silu", "gelu"])
    one = 2.0 * c["cin"] * c["cout"] * c["top_k"] * (3 if op.endswith("grad") else 1) * (6 if c["dtype"] == "f32" else 1)
    c["experts"] = max(c["top_k"], min(c["experts"], int(MOST_BYTES / 4 / (c["cin"] * c["cout"] * SIZE[c["dtype"]]))))
    c["tokens"] = max(1, min(c["tokens"], int(MOST_FLOPS / one)))
    return c


# ---------------------------------------------------------------------------------------------------------------- inputs
def _routing(g, tokens, experts, top_k, dropped):
    """top_k experts a token, from scores with some experts liked better; int32 [tokens, top_k], -1 where a pair is dropped."""
    score = torch.randn((tokens, experts), generator=g, device="cuda") + 0.3 * torch.randn((1, experts), generator=g, device="cuda")
    val, idx = score.topk(top_k, dim=1)
    idx = idx.to(torch.int32)
    gone = int(dropped * tokens * top_k)  # as many in every state, so that outputs keep their shapes
    if gone:
        idx.view(-1)[torch.rand((tokens * top_k,), generator=g, device="cuda").topk(gone).indices] = -1
    return idx.contiguous(), val.softmax(1).contiguous()


def _values(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _in_8_bits(g, shape, spread):
    """What a quantiser leaves: e4m3 values whose rows reach 448, and a scale a row."""
    v = torch.randn(shape, generator=g, device="cuda") * spread
    s = v.abs().amax(-1, keepdim=True).clamp_min(1e-12) / TOP
    return (v / s).clamp(-TOP, TOP).to(torch.float8_e4m3fn), s.squeeze(-1).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    c, dt = case, TYPES[case["dtype"]]
    s = {"case": dict(c)}
    if c["op"].startswith("norm"):
        shape = (c["rows"], c["cols"])
        s["x"], s["residual"] = _values(g, shape, dt), _values(g, shape, dt)
        s["weight"] = 1.0 + 0.1 * torch.randn((c["cols"],), generator=g, device="cuda")
        if c["op"] == "norm_grad":
            s["dy"], s["dres"] = _values(g, shape, dt), _values(g, shape, dt)
        return s
    idx, gate = _routing(g, c["tokens"], c["experts"], c["top_k"], c.get("dropped", 0.0))
    pairs = c["tokens"] * c["top_k"]
    if c["op"].startswith("tokens"):
        s["idx"], s["gate"], s["rows"] = idx, gate, pairs - int(c["dropped"] * pairs)
        s["scale"] = None
        if c["dtype"] == "e4m3":
            s["x"], s["scale"] = _in_8_bits(g, (c["tokens"], c["cols"]), 1.0)
        else:
            s["x"] = _values(g, (c["tokens"], c["cols"]), dt)
        s["ys"] = _values(g, (pairs, c["cols"]), torch.bfloat16 if c["dtype"] == "e4m3" else dt)  # the experts' answers: 16 bits after 8-bit products
        if c["op"] == "tokens_grad":
            s["dy"], s["dxs"] = _values(g, (c["tokens"], c["cols"]), dt), _values(g, (pairs, c["cols"]), dt)
        return s
    count = torch.bincount(idx.reshape(-1).long(), minlength=c["experts"])
    s["offsets"] = torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32)
    s["most"] = int(count.max())  # rows of the fullest expert
    shape = (c["experts"], c["cout"], c["cin"])
    s["x_scale"] = s["w_scale"] = None
    if c["dtype"] == "e4m3":
        s["x"], s["x_scale"] = _in_8_bits(g, (pairs, c["cin"]), 1.0)
        s["w"], s["w_scale"] = _in_8_bits(g, shape, c["cin"] ** -0.5)
    else:
        s["x"], s["w"] = _values(g, (pairs, c["cin"]), dt), (torch.randn(shape, generator=g, device="cuda") * c["cin"] ** -0.5).to(dt)
    s["bias"] = 0.1 * torch.randn((c["experts"], c["cout"]), generator=g, device="cuda")
    if c["op"] == "product_grad":
        s["dy"] = _values(g, (pairs, c["cout"]), dt)
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms
def _norm(s):
    h = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)  # the sum as it is kept is what gets normalised
    f = h.float()
    return h, f, torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)


def _norm_quant(s):
    h, f, rstd = _norm(s)
    y = f * rstd * s["weight"]
    scale = y.abs().amax(-1, keepdim=True) / TOP
    scale = torch.where(scale > 0, scale, 1.0)
    return {"q": (y / scale).clamp(-TOP, TOP).to(torch.float8_e4m3fn), "scale": scale.squeeze(-1), "h": h}


def _norm_grad(s):
    h, f, rstd = _norm(s)
    n, dy = f * rstd, s["dy"].float()
    g = dy * s["weight"]
    dx = rstd * (g - n * (g * n).mean(-1, keepdim=True)) + s["dres"].float()
    return {"y": (n * s["weight"]).to(h.dtype), "h": h, "dx": dx.to(h.dtype), "dweight": (dy * n).sum(0)}


def _plan(s):
    c = s["case"]
    flat = s["idx"].reshape(-1)
    key = torch.where(flat >= 0, flat, c["experts"])
    order = torch.argsort(key, stable=True)[: s["rows"]]
    row = torch.full_like(flat, -1)
    row[order] = torch.arange(s["rows"], device=flat.device, dtype=torch.int32)
    count = (flat[:, None] == torch.arange(c["experts"], device=flat.device)).sum(0)
    return torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32), order, row.reshape(s["idx"].shape)


def _tokens(s):
    c = s["case"]
    offsets, order, row = _plan(s)
    token = order // c["top_k"]
    kept = (row >= 0).unsqueeze(-1)
    at = row.clamp_min(0).long()
    out = {"offsets": offsets, "src": order.to(torch.int32), "row": row, "xs": s["x"].view(torch.uint8)[token].view(s["x"].dtype) if s["scale"] is not None else s["x"][token]}
    if s["scale"] is not None:
        out["xs_scale"] = s["scale"][token]
    part = torch.where(kept, s["ys"].float()[at], 0.0)
    out["y"] = (part * s["gate"].unsqueeze(-1)).sum(1).to(s["ys"].dtype)
    if c["op"] == "tokens_grad":
        dy = s["dy"].float()
        out["dx"] = torch.where(kept, s["dxs"].float()[at], 0.0).sum(1).to(s["x"].dtype)
        out["dys"] = (s["gate"].reshape(-1)[order].unsqueeze(-1) * dy[token]).to(s["x"].dtype)
        out["dgate"] = (part * dy.unsqueeze(1)).sum(-1)
    return out


def _by_expert(rows, at, experts, most):
    """[rows, C] -> [experts, most, C], zeros behind each expert's last row."""
    out = rows.new_zeros((experts * most, rows.shape[1]))
    out[at] = rows
    return out.view(experts, most, rows.shape[1])


def _product(s):
    c = s["case"]
    rows, E, most = s["x"].shape[0], c["experts"], s["most"]
    off = s["offsets"].long()
    e = torch.searchsorted(off[1:], torch.arange(rows, device=off.device), right=True)
    at = e * most + torch.arange(rows, device=off.device) - off[e]  # a row's place among its expert's
    x, w = s["x"].float(), s["w"].float()
    out_type = s["x"].dtype
    if s["x_scale"] is not None:
        x, w, out_type = x * s["x_scale"].unsqueeze(-1), w * s["w_scale"].unsqueeze(-1), torch.bfloat16
    x = _by_expert(x, at, E, most)
    y = torch.bmm(x, w.transpose(1, 2)) + s["bias"].unsqueeze(1)
    if c["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif c["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * 0.5**0.5))
    out = {"y": y.view(E * most, -1)[at].to(out_type)}
    if c["op"] == "product_grad":
        dy = _by_expert(s["dy"].float(), at, E, most)
        out["dx"] = torch.bmm(dy, w).view(E * most, -1)[at].to(out_type)
        out["dw"] = torch.bmm(dy.transpose(1, 2), x).to(out_type)
        out["dbias"] = dy.sum(1)
    return out


# ------------------------------------------------------------------------------------------------------- the framework's
def _own(s):
    from yolo_master_amd import ops

    c = s["case"]
    if c["op"] == "norm_quant":
        q, scale, h = ops.rms_norm_quant(s["x"], s["weight"], EPS, residual=s["residual"])
        return {"q": q, "scale": scale, "h": h}
    if c["op"] == "norm_grad":
        y, h, rstd = ops.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"])
        dx, dweight = ops.rms_norm_backward(s["dy"], h, s["weight"], rstd, dres=s["dres"])
        return {"y": y, "h": h, "dx": dx, "dweight": dweight}
    if c["op"].startswith("tokens"):
        n = s["rows"]  # what lies behind the last expert's rows is not written
        plan = ops.token_sort(s["idx"], c["experts"])
        out = {"offsets": plan.offsets, "src": plan.src[:n], "row": plan.row}
        if s["scale"] is not None:
            xs, xs_scale = ops.token_dispatch(s["x"], plan, scale=s["scale"])
            out["xs_scale"] = xs_scale[:n]
        else:
            xs = ops.token_dispatch(s["x"], plan)
        out["xs"], out["y"] = xs[:n], ops.token_combine(s["ys"], plan, s["gate"])
        if c["op"] == "tokens_grad":
            dys, out["dgate"] = ops.token_combine_backward(s["dy"], s["ys"], plan, s["gate"])
            out["dx"], out["dys"] = ops.token_dispatch_backward(s["dxs"], plan), dys[:n]
        return out
    out = {"y": ops.expert_linear(s["x"], s["w"], s["offsets"], s["bias"], act=c["act"] or None, x_scale=s["x_scale"], w_scale=s["w_scale"])}
    if c["op"] == "product_grad":
        out["dx"], out["dw"], out["dbias"] = ops.expert_linear_backward(s["dy"], s["x"], s["w"], s["offsets"])
    return out


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "norm_quant":
        return _norm_quant(state)
    if op == "norm_grad":
        return _norm_grad(state)
    return _tokens(state) if op.startswith("tokens") else _product(state)


# -------------------------------------------------------------------------------------------------------------- the work
def work(case):
    c, b = case, SIZE[case["dtype"]]
    if c["op"] == "norm_quant":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (3 * b + 1) + 4 * (c["rows"] + c["cols"]), "flops": 8 * n}
    if c["op"] == "norm_grad":  # x, residual, dy, dres in; y, h, dx out
        n = c["rows"] * c["cols"]
        return {"bytes": 7 * n * b + 8 * c["cols"], "flops": 16 * n}
    pairs = c["tokens"] * c["top_k"]
    if c["op"].startswith("tokens"):
        kept = pairs - int(c["dropped"] * pairs)
        row, yb = c["cols"] * b, c["cols"] * (2 if c["dtype"] == "e4m3" else b)
        plan = 4 * (4 * pairs + c["experts"])
        bytes_ = plan + c["tokens"] * (row + yb) + kept * (row + yb)
        if c["op"] == "tokens_grad":  # dy, dxs in; dx, dys, dgate out (ys is counted above)
            bytes_ += 2 * c["tokens"] * row + 2 * kept * row + 4 * pairs
        return {"bytes": bytes_, "flops": (2 if c["op"] == "tokens" else 6) * kept * c["cols"]}
    used = min(c["experts"], pairs)
    yb = 2 if c["dtype"] == "e4m3" else b
    bytes_ = pairs * (c["cin"] * b + c["cout"] * yb) + used * c["cout"] * (c["cin"] * b + 4)
    flops = 2 * pairs * c["cin"] * c["cout"]
    if c["op"] == "product_grad":  # dy in; dx, dw, dbias out
        bytes_ += pairs * (c["cin"] + c["cout"]) * b + c["experts"] * c["cout"] * (c["cin"] * b + 4)
        flops *= 3
    return {"bytes": bytes_, "flops": flops}


# ----------------------------------------------------------------------------------------------- the definitions, 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = case
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if c["op"].startswith("norm"):
        whole = d["x"] + d["residual"]
        h = whole.to(s["x"].dtype).double()
        norm = (h.pow(2).sum(1) / c["cols"] + EPS).sqrt()[:, None]
        y = h / norm * d["weight"][None]
        if c["op"] == "norm_quant":
            scale = torch.linalg.vector_norm(y, ord=math.inf, dim=1) / TOP
            return {"q": y / scale[:, None], "scale": scale, "h": whole}
        # L = sum(dy y) + sum(dres h), by the chain rule through norm(h)
        dh = d["dy"] * d["weight"] / norm - h * (d["dy"] * d["weight"] * h).sum(1, keepdim=True) / (c["cols"] * norm.pow(3)) + d["dres"]
        return {"y": y, "h": whole, "dx": dh, "dweight": torch.mv((d["dy"] * h / norm).t().contiguous(), torch.ones(c["rows"], dtype=torch.float64, device="cuda"))}
    if c["op"].startswith("tokens"):
        flat = s["idx"].reshape(-1).cpu().tolist()
        lists = [[] for _ in range(c["experts"])]
        for pair, e in enumerate(flat):
            if e >= 0:
                lists[e].append(pair)
        src = [p for part in lists for p in part]
        offsets, row = [0], [-1] * len(flat)
        for part in lists:
            offsets.append(offsets[-1] + len(part))
        for r, p in enumerate(src):
            row[p] = r
        at = torch.tensor(src, dtype=torch.long, device="cuda")
        tok = torch.div(at, c["top_k"], rounding_mode="floor")
        whole = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        out = {"offsets": whole(offsets), "src": whole(src), "row": whole(row).reshape(s["idx"].shape), "xs": d["x"].index_select(0, tok)}
        if s["scale"] is not None:
            out["xs_scale"] = d["scale"].index_select(0, tok)
        ys, gate = d["ys"][: len(src)], d["gate"].reshape(-1)[at][:, None]
        zero = torch.zeros((c["tokens"], c["cols"]), dtype=torch.float64, device="cuda")
        out["y"] = zero.index_add(0, tok, ys * gate)
        if c["op"] == "tokens_grad":
            out["dx"] = zero.index_add(0, tok, d["dxs"][: len(src)])
            out["dys"] = gate * d["dy"][tok]
            dgate = torch.zeros(len(flat), dtype=torch.float64, device="cuda")
            dgate[at] = (d["dy"][tok] * ys).sum(1)
            out["dgate"] = dgate.reshape(s["idx"].shape)
        return out
    if c["experts"] * c["cin"] * c["cout"] > 6e8:
        return None
    off = s["offsets"].cpu().tolist()
    y, dx = torch.empty((s["x"].shape[0], c["cout"]), dtype=torch.float64, device="cuda"), torch.empty_like(d["x"])
    dw, db = torch.zeros(s["w"].shape, dtype=torch.float64, device="cuda"), torch.zeros_like(d["bias"])
    for e in range(c["experts"]):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        x, w = d["x"][a:b], d["w"][e]
        if s["x_scale"] is not None:
            x, w = x * d["x_scale"][a:b, None], w * d["w_scale"][e][:, None]
        v = x @ w.t() + d["bias"][e]
        if c["act"] == "silu":
            v = v / (1.0 + torch.exp(-v))
        elif c["act"] == "gelu":
            v = v * torch.special.ndtr(v)
        y[a:b] = v
        if c["op"] == "product_grad":
            dx[a:b], dw[e], db[e] = d["dy"][a:b] @ w, d["dy"][a:b].t() @ x, d["dy"][a:b].sum(0)
    return {"y": y, "dx": dx, "dw": dw, "dbias": db} if c["op"] == "product_grad" else {"y": y}
