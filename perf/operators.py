"""Operators of transformer blocks on irreps features: measured cases, their plain forms and their definitions in 64 bits.

* ``rms``    ``nn.RMSNorm``: the norm before a block
* ``norm``   ``nn.NormGateResidual``: norm after a block, Gate, residual with learned scale, norm before the next block
* ``bias``   ``nn.RelativeBias``: distance buckets of the edges, learned bias per bucket and head
* ``attn``   ``nn.NeighborAttention``: multi-head softmax attention over the incoming edges of every node, with the
             bias by buckets and a cutoff weight per edge

``run`` computes a pass from elementary torch operations (``own`` false) or through the package's modules (``own`` true).
A case with ``train`` is the pass with the gradients of everything that learns or is differentiated.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-5
# <f(z)^2>^(-1/2), z ~ N(0,1), of silu and sigmoid as Gate estimates it (a million samples)
_SILU, _SIGMOID = 1.6791767923989418, 1.8467055342154763


def listed():
    return [
        # norm before the first block of a hidden layer, small molecules in training
        {"name": "rms_train_4k", "op": "rms", "rows": 4001, "mul0": 32, "gated": "32x1o+32x2e", "type": "fp32", "train": True},
        # block boundary of a small molecule in inference: latency
        {"name": "norm_64", "op": "norm", "rows": 64, "mul0": 32, "gated": "32x1o+32x2e", "type": "fp32", "train": False},
        # odd multiplicities (rows that no vector width divides), 16-bit training of a minibatch
        {"name": "norm_odd_20k", "op": "norm", "rows": 20011, "mul0": 17, "gated": "9x1o+5x2e", "type": "fp16", "train": True},
        # training on periodic cells
        {"name": "norm_train_16k", "op": "norm", "rows": 16384, "mul0": 64, "gated": "64x1o+64x2e+64x3o", "type": "fp32", "train": True},
        # inference on a large cell, 16-bit features
        {"name": "norm_262k", "op": "norm", "rows": 262144, "mul0": 64, "gated": "64x1o+64x2e+64x3o", "type": "bf16", "train": False},
        # edges of a solvated molecule in inference
        {"name": "bias_100k", "op": "bias", "nodes": 4001, "edges": 104026, "buckets": 32, "heads": 8, "r_max": 5.0, "r_linear": 5.0,
         "type": "fp32", "train": False},
        # edges of a large graph in training, buckets linear near and logarithmic far
        {"name": "bias_train_2m", "op": "bias", "nodes": 65536, "edges": 2097152, "buckets": 64, "heads": 16, "r_max": 12.0, "r_linear": 3.0,
         "type": "fp32", "train": True},
        # a small molecule in inference: latency
        {"name": "attn_64", "op": "attn", "dst": 64, "src": 64, "edges": 1009, "ragged": False, "mul0": 32, "gated": "32x1o+32x2e", "heads": 4,
         "buckets": 32, "weight": False, "per_edge": False, "type": "fp32", "train": False},
        # one probe atom that attends to every atom of a cell: a single query over a long list
        {"name": "attn_probe_50k", "op": "attn", "dst": 1, "src": 50021, "edges": 50021, "ragged": False, "mul0": 64, "gated": "64x1o+64x2e",
         "heads": 8, "buckets": 32, "weight": False, "per_edge": True, "type": "bf16", "train": False},
        # inference on a large random graph
        {"name": "attn_2m", "op": "attn", "dst": 65536, "src": 65536, "edges": 2097152, "ragged": False, "mul0": 64, "gated": "64x1o+64x2e",
         "heads": 8, "buckets": 32, "weight": False, "per_edge": False, "type": "fp32", "train": False},
        # training on periodic cells, 16-bit features, smooth cutoff, uneven numbers of neighbours and isolated atoms
        {"name": "attn_train_16k", "op": "attn", "dst": 16384, "src": 16384, "edges": 425984, "ragged": True, "mul0": 64,
         "gated": "64x1o+64x2e+64x3o", "heads": 8, "buckets": 32, "weight": True, "per_edge": False, "type": "bf16", "train": True},
        # training with keys and values made per edge by a tensor product, three heads
        {"name": "attn_edge_150k", "op": "attn", "dst": 10007, "src": 10007, "edges": 150001, "ragged": True, "mul0": 48, "gated": "24x1o+12x2e",
         "heads": 3, "buckets": 0, "weight": True, "per_edge": True, "type": "fp32", "train": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rms", "norm", "norm", "bias", "attn", "attn", "attn"])
    case = {"op": op, "type": rng.choice(["fp32", "fp32", "bf16", "fp16"]), "train": rng.random() < 0.5}
    if op == "bias":
        r_max = rng.choice([4.0, 5.0, 8.0, 12.0])
        case.update(nodes=_log_int(rng, 16, 65536), edges=_log_int(rng, 64, 2097152), buckets=_log_int(rng, 2, 256), heads=rng.randint(1, 16),
                    r_max=r_max, r_linear=rng.choice([r_max, 0.25 * r_max, 0.5 * r_max]))
        return case
    heads = rng.choice([1, 2, 3, 4, 5, 8, 16]) if op == "attn" else 1
    per_head = rng.choice([1, 2, 3, 4, 8, 16]) if op == "attn" else rng.randint(3, 64)
    while heads * per_head > 64:
        per_head //= 2
    lmax = rng.randint(1, 3)
    muls = [heads * max(1, per_head // rng.choice([1, 1, 2])) for _ in range(lmax + 1)]
    case.update(mul0=muls[0], gated="+".join(f"{muls[l]}x{l}{'o' if l % 2 else 'e'}" for l in range(1, lmax + 1)))
    if op != "attn":
        case["rows"] = _log_int(rng, 1, 262144 if not case["train"] else 131072)
        return case
    dst = _log_int(rng, 1, 32768)
    edges = min(_log_int(rng, 1, 64) * dst, 800000 if not case["train"] else 400000) if dst > 16 else _log_int(rng, 1, 60000)
    case.update(dst=dst, src=_log_int(rng, 1, 65536), edges=edges, ragged=rng.random() < 0.5, heads=heads, buckets=rng.choice([0, 8, 32, 128]),
                weight=rng.random() < 0.5, per_edge=rng.random() < 0.4)
    return case


# ---------------------------------------------------------------------------------------------------------- layouts and inputs
def _gated(text):
    """``"64x1o+64x2e"`` -> ``[(64, 3), (64, 5)]``: channels and components."""
    return [(int(t.split("x")[0]), 2 * int(t.split("x")[1][:-1]) + 1) for t in text.split("+")]


def _blocks(case):
    """Blocks (channels, components) of the features and of the Gate's input rows (scalars and gates are one block)."""
    gated = _gated(case["gated"])
    return [(case["mul0"], 1)] + gated, [(case["mul0"] + sum(m for m, _ in gated), 1)] + gated


def _dim(blocks):
    return sum(m * d for m, d in blocks)


def _muls(blocks):
    return sum(m for m, _ in blocks)


def _inputs(case, seed):
    """What a user's program has in hand, as plain tensors: the same for the plain form, the modules and the definition."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["type"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device="cuda") * std + mean

    x = {}
    if case["op"] in ("rms", "norm"):
        out, inner = _blocks(case)
        rows = case["rows"]
        x["residual"] = normal(rows, _dim(out)).to(dtype)
        x["weight_pre"] = normal(_muls(out), std=0.1, mean=1.0)
        if case["op"] == "norm":
            x["y"] = normal(rows, _dim(inner), std=3.0).to(dtype)
            x["weight_post"] = normal(_muls(inner), std=0.1, mean=1.0)
            x["scale"] = normal(_muls(out), std=0.1, mean=0.3)
        if case["train"]:
            x["grad_h"] = normal(rows, _dim(out)).to(dtype)
            if case["op"] == "norm":
                x["grad_z"] = normal(rows, _dim(out)).to(dtype)
        return x
    if case["op"] == "bias":
        n, e, r_max = case["nodes"], case["edges"], case["r_max"]
        box = (n / 0.05) ** (1 / 3)
        x["pos"] = torch.rand(n, 3, generator=gen, device="cuda") * box
        x["dst"] = torch.randint(n, (e,), generator=gen, device="cuda").sort().values
        x["src"] = torch.randint(n, (e,), generator=gen, device="cuda")
        # periodic images that put the neighbours evenly into the ball of the cutoff
        vec = normal(e, 3)
        vec = vec / vec.norm(dim=1, keepdim=True) * (r_max * torch.rand(e, 1, generator=gen, device="cuda") ** (1 / 3))
        x["shift"] = vec - (x["pos"][x["src"]] - x["pos"][x["dst"]])
        x["table"] = normal(case["buckets"], case["heads"], std=0.5).to(dtype)
        if case["train"]:
            x["grad"] = normal(e, case["heads"]).to(dtype)
        return x
    blocks, _ = _blocks(case)
    n, e, d = case["dst"], case["edges"], _dim(blocks)
    if case["ragged"]:      # uneven numbers of neighbours, about one node in ten without any
        share = torch.rand(n, generator=gen, device="cuda") ** 2 * (torch.rand(n, generator=gen, device="cuda") > 0.1)
        if n == 1:
            share = torch.ones_like(share)
        ends = torch.cumsum(share.double(), 0)
        ends = (ends / ends[-1].clamp(min=1e-30) * e).round().long().clamp(max=e)
    else:
        ends = torch.arange(1, n + 1, device="cuda") * e // n
    ends[-1] = e
    x["rowptr"] = torch.cat([ends.new_zeros(1), ends])
    x["src"] = None if case["per_edge"] else torch.randint(case["src"], (e,), generator=gen, device="cuda")
    keys = e if case["per_edge"] else case["src"]
    x["q"] = normal(n, d).to(dtype)
    x["k"] = normal(keys, d).to(dtype)
    x["v"] = normal(keys, d).to(dtype)
    if case["buckets"]:
        x["table"] = normal(case["buckets"], case["heads"], std=0.5)
        x["bucket"] = torch.randint(case["buckets"], (e,), generator=gen, device="cuda", dtype=torch.int32)
    if case["weight"]:      # a smooth cutoff of distances even in the ball; a few edges lie outside
        r = 1.02 * torch.rand(e, generator=gen, device="cuda") ** (1 / 3)
        x["weight"] = torch.where(r < 1, 0.5 * (torch.cos(math.pi * r) + 1), 0.0)
    if case["train"]:
        x["grad"] = normal(n, d).to(dtype)
    return x


def _thresholds(case):
    """Lower ends of the buckets 1, 2, ...: linear up to r_linear, logarithmic from there to r_max."""
    b, lin, far = case["buckets"], case["r_linear"], case["r_max"]
    n = b if lin >= far else (b + 1) // 2
    return torch.tensor([lin * i / n if i <= n else lin * (far / lin) ** ((i - n) / (b - n)) for i in range(1, b)], dtype=torch.float64)


def prepare(case, seed):
    s = {"case": case, "x": _inputs(case, seed)}
    x = s["x"]
    if case["op"] != "bias":
        s["layout"] = {"columns": [_column_channels(b) for b in _blocks(case)], "heads": _head_columns(case) if case["op"] == "attn" else None}
    if case["op"] == "attn":
        counts = x["rowptr"][1:] - x["rowptr"][:-1]
        s["dst"] = torch.repeat_interleave(torch.arange(case["dst"], device="cuda"), counts)
    if case["op"] == "bias":
        s["thresholds"] = _thresholds(case).cuda()
    if not own:
        return s
    import e3nn_b200
    from e3nn_b200 import nn

    irreps = f"{case.get('mul0')}x0e+{case.get('gated')}"
    with torch.no_grad():
        if case["op"] == "rms":
            s["module"] = nn.RMSNorm(irreps, eps=_EPS).cuda()
            s["module"].weight.copy_(x["weight_pre"])
        elif case["op"] == "norm":
            gates = sum(m for m, _ in _gated(case["gated"]))
            gate = nn.Gate(f"{case['mul0']}x0e", [torch.nn.functional.silu], f"{gates}x0e", [torch.sigmoid], case["gated"])
            s["module"] = nn.NormGateResidual(gate, eps=_EPS).cuda()
            for name in ("weight_post", "scale", "weight_pre"):
                getattr(s["module"], name).copy_(x[name])
        elif case["op"] == "bias":
            s["module"] = nn.RelativeBias(case["buckets"], case["heads"], case["r_max"], r_linear=case["r_linear"]).cuda()
            s["module"].to(x["table"].dtype).weight.copy_(x["table"])
        else:
            s["module"] = nn.NeighborAttention(irreps, irreps, case["heads"]).cuda()
            if case["train"] and not case["per_edge"]:
                s["transpose"] = e3nn_b200.csr_from_dst(x["src"], case["src"])
    return s


# ---------------------------------------------------------------------------------------------------------- the package's modules
def _leaf(t):
    return None if t is None else t.detach().requires_grad_()


def _run_own(s):
    case, x, module = s["case"], s["x"], s["module"]
    train = case["train"]
    with torch.set_grad_enabled(train):
        if case["op"] == "rms":
            if not train:
                return {"h": module(x["residual"])}
            residual = _leaf(x["residual"])
            h = module(residual)
            gx, gw = torch.autograd.grad(h, (residual, module.weight), x["grad_h"])
            return {"h": h.detach(), "grad_residual": gx, "grad_weight_pre": gw}
        if case["op"] == "norm":
            if not train:
                z, h = module(x["residual"], x["y"])
                return {"z": z, "h": h}
            residual, y = _leaf(x["residual"]), _leaf(x["y"])
            z, h = module(residual, y)
            grads = torch.autograd.grad((z, h), (residual, y, module.weight_post, module.scale, module.weight_pre), (x["grad_z"], x["grad_h"]))
            return {"z": z.detach(), "h": h.detach(), "grad_residual": grads[0], "grad_y": grads[1], "grad_weight_post": grads[2],
                    "grad_scale": grads[3], "grad_weight_pre": grads[4]}
        if case["op"] == "bias":
            buckets = module.buckets(x["pos"], x["src"], x["dst"], x["shift"])
            bias = module(buckets)
            if not train:
                return {"buckets": buckets, "bias": bias}
            (grad,) = torch.autograd.grad(bias, (module.weight,), x["grad"])
            return {"buckets": buckets, "bias": bias.detach(), "grad_table": grad}
        args = [x["q"], x["k"], x["v"], x.get("table"), x.get("weight")]
        if train:
            args = [_leaf(t) for t in args]
        q, k, v, table, weight = args
        out = module(q, k, v, x["rowptr"], x["src"], bias=table, buckets=x.get("bucket"), edge_weight=weight, transpose=s.get("transpose"))
        if not train:
            return {"out": out}
        wanted = {n: t for n, t in (("q", q), ("k", k), ("v", v), ("table", table), ("weight", weight)) if t is not None}
        grads = torch.autograd.grad(out, tuple(wanted.values()), x["grad"])
        return {"out": out.detach(), **{"grad_" + n: g for n, g in zip(wanted, grads)}}


# ---------------------------------------------------------------------------------------------------------- plain forms, 32 bits
def _column_channels(blocks):
    """Channel of every column."""
    counts = torch.tensor([d for m, d in blocks for _ in range(m)])
    return torch.repeat_interleave(torch.arange(_muls(blocks)), counts).cuda()


def _channel_sums(columns, blocks):
    """Columns [D] -> sums over the components of every channel."""
    parts, at = [], 0
    for m, d in blocks:
        parts.append(columns[at:at + m * d].reshape(m, d).sum(1))
        at += m * d
    return torch.cat(parts)


def _per_block(x, blocks, f):
    parts, at = [], 0
    for m, d in blocks:
        part = x[:, at:at + m * d]
        parts.append(f(part).expand(-1, m * d))
        at += m * d
    return torch.cat(parts, 1)


def _rstd(x, blocks):
    return _per_block(x, blocks, lambda p: torch.rsqrt(p.square().mean(1, keepdim=True) + _EPS))


def _norm_backward(g, x, rstd, w, blocks):
    """Gradients of w * x * rstd(x) w.r.t. x (rows) and w (columns)."""
    n = x * rstd
    gn = g * w
    mean = _per_block(gn * n, blocks, lambda p: p.mean(1, keepdim=True))
    return rstd * (gn - n * mean), (g * n).sum(0)


def _plain_rms(case, x, columns):
    blocks, _ = _blocks(case)
    r, w = x["residual"].float(), x["weight_pre"][columns[0]]
    rstd = _rstd(r, blocks)
    out = {"h": (r * rstd * w).to(x["residual"].dtype)}
    if case["train"]:
        gx, gw = _norm_backward(x["grad_h"].float(), r, rstd, w, blocks)
        out.update(grad_residual=gx.to(x["residual"].dtype), grad_weight_pre=_channel_sums(gw, blocks))
    return out


def _plain_norm(case, x, columns):
    blocks, inner = _blocks(case)
    dtype, m0, gated = x["y"].dtype, case["mul0"], _gated(case["gated"])
    ng = _muls(gated)
    y, res = x["y"].float(), x["residual"].float()
    wp, sc, wn = x["weight_post"][columns[1]], x["scale"][columns[0]], x["weight_pre"][columns[0]]
    rstd_y = _rstd(y, inner)
    n = y * rstd_y * wp
    scal, gates, feats = n[:, :m0], n[:, m0:m0 + ng], n[:, m0 + ng:]
    sig_s, sig_g = torch.sigmoid(scal), torch.sigmoid(gates)
    gate_cols = (_SIGMOID * sig_g)[:, columns[0][m0:] - m0]
    val = torch.cat([_SILU * scal * sig_s, feats * gate_cols], 1)
    z = res + sc * val
    rstd_z = _rstd(z, blocks)
    out = {"z": z.to(dtype), "h": (z * rstd_z * wn).to(dtype)}
    if not case["train"]:
        return out
    gz, gw_pre = _norm_backward(x["grad_h"].float(), z, rstd_z, wn, blocks)
    gz = gz + x["grad_z"].float()
    g_scale = _channel_sums((gz * val).sum(0), blocks)
    gv = gz * sc
    g_scal = gv[:, :m0] * _SILU * sig_s * (1 + scal * (1 - sig_s))
    prod, parts, at = gv[:, m0:] * feats, [], 0
    for m, d in gated:
        parts.append(prod[:, at:at + m * d].reshape(-1, m, d).sum(2))
        at += m * d
    g_gates = torch.cat(parts, 1) * _SIGMOID * sig_g * (1 - sig_g)
    gy, gw_post = _norm_backward(torch.cat([g_scal, g_gates, gv[:, m0:] * gate_cols], 1), y, rstd_y, wp, inner)
    out.update(grad_residual=gz.to(dtype), grad_y=gy.to(dtype), grad_weight_post=_channel_sums(gw_post, inner), grad_scale=g_scale,
               grad_weight_pre=_channel_sums(gw_pre, blocks))
    return out


def _plain_bias(case, x, thresholds):
    # distances in 64 bits: a distance next to a border must not change its bucket
    vec = x["pos"].double()[x["src"]] - x["pos"].double()[x["dst"]] + x["shift"].double()
    buckets = torch.bucketize(vec.square().sum(1), thresholds.square(), right=True).int()
    out = {"buckets": buckets, "bias": x["table"][buckets]}
    if case["train"]:
        grad = torch.zeros(x["table"].shape, device="cuda", dtype=torch.float64)
        out["grad_table"] = grad.index_add_(0, buckets, x["grad"].double()).to(x["table"].dtype)
    return out


def _head_columns(case):
    """Columns of every head [heads, D / heads]: mul / heads channels of each block."""
    cols, at = [[] for _ in range(case["heads"])], 0
    for m, d in _blocks(case)[0]:
        n = m // case["heads"] * d
        for h in range(case["heads"]):
            cols[h] += range(at + h * n, at + (h + 1) * n)
        at += m * d
    return torch.tensor(cols, device="cuda")


def _plain_attn(case, x, dst, cols):
    dtype, heads, n = x["q"].dtype, case["heads"], case["dst"]
    scale = cols.shape[1] ** -0.5
    q, k, v = (x[name].float()[:, cols] for name in "qkv")
    src = x["src"]
    kd, vd = (k, v) if src is None else (k[src], v[src])
    a = (q[dst] * kd).sum(2) * scale
    if "table" in x:
        a = a + x["table"][x["bucket"]]
    if "weight" in x:
        # the weight's logarithm joins the logit: the shares of a node whose edges all have tiny weights keep their digits
        a = a + torch.log(x["weight"].clamp(min=0))[:, None]
    top = torch.full((n, heads), -math.inf, device="cuda").scatter_reduce_(0, dst[:, None].expand(-1, heads), a, "amax")
    p = torch.exp(a - torch.where(torch.isfinite(top), top, 0.0)[dst])
    total = torch.zeros(n, heads, device="cuda").index_add_(0, dst, p)
    p = p * torch.where(total > 0, 1 / total, 0.0)[dst]
    out = torch.zeros(n, *cols.shape, device="cuda").index_add_(0, dst, p[:, :, None] * vd)

    def columns(t, rows):
        return torch.empty(rows, cols.numel(), device="cuda").index_copy_(1, cols.flatten(), t.reshape(rows, -1)).to(dtype)

    result = {"out": columns(out, n)}
    if not case["train"]:
        return result
    g = x["grad"].float()[:, cols][dst]
    dp = (g * vd).sum(2)
    delta = torch.zeros(n, heads, device="cuda").index_add_(0, dst, p * dp)[dst]
    da = p * (dp - delta)
    gv = p[:, :, None] * g
    gk = (scale * da)[:, :, None] * q[dst]
    gq = torch.zeros_like(q).index_add_(0, dst, (scale * da)[:, :, None] * kd)
    if src is not None:
        gk = torch.zeros_like(k).index_add_(0, src, gk)
        gv = torch.zeros_like(v).index_add_(0, src, gv)
    result.update(grad_q=columns(gq, n), grad_k=columns(gk, k.shape[0]), grad_v=columns(gv, v.shape[0]))
    if "table" in x:
        result["grad_table"] = torch.zeros(x["table"].shape, device="cuda", dtype=torch.float64).index_add_(0, x["bucket"], da.double()).float()
    if "weight" in x:
        result["grad_weight"] = torch.where(x["weight"] > 0, da.sum(1) / x["weight"], 0.0)
    return result


def run(state):
    if own:
        return _run_own(state)
    case, x = state["case"], state["x"]
    with torch.no_grad():
        if case["op"] == "rms":
            return _plain_rms(case, x, state["layout"]["columns"])
        if case["op"] == "norm":
            return _plain_norm(case, x, state["layout"]["columns"])
        if case["op"] == "bias":
            return _plain_bias(case, x, state["thresholds"])
        return _plain_attn(case, x, state["dst"], state["layout"]["heads"])


# ---------------------------------------------------------------------------------------------------------- definitions, 64 bits
def _exact_norm(x, w, blocks):
    """Every block divided by the root of its mean square, times the weight of the channel."""
    parts, col, chan = [], 0, 0
    for m, d in blocks:
        b = x[:, col:col + m * d].reshape(-1, m, d)
        rms = ((b ** 2).sum((1, 2)) / (m * d) + _EPS).sqrt()
        parts.append((b / rms[:, None, None] * w[None, chan:chan + m, None]).reshape(-1, m * d))
        col, chan = col + m * d, chan + m
    return torch.cat(parts, 1)


def _exact_block(case, t):
    blocks, inner = _blocks(case)
    if case["op"] == "rms":
        return {"h": _exact_norm(t["residual"], t["weight_pre"], blocks)}
    n = _exact_norm(t["y"], t["weight_post"], inner)
    m0, col, chan = case["mul0"], 0, 0
    scalars = n[:, :m0]
    gates = _SIGMOID / (1 + torch.exp(-n[:, m0:inner[0][0]]))
    parts = [_SILU * scalars / (1 + torch.exp(-scalars)) * t["scale"][:m0]]
    col = inner[0][0]
    for m, d in blocks[1:]:
        b = n[:, col:col + m * d].reshape(-1, m, d) * gates[:, chan:chan + m, None] * t["scale"][m0 + chan:m0 + chan + m, None]
        parts.append(b.reshape(-1, m * d))
        col, chan = col + m * d, chan + m
    z = t["residual"] + torch.cat(parts, 1)
    return {"z": z, "h": _exact_norm(z, t["weight_pre"], blocks)}


def _exact_rows(case, x):
    """Row by row in turns, so that a large batch fits; gradients of the parameters are added over the turns."""
    params = [p for p in ("weight_post", "scale", "weight_pre") if p in x]
    rows = [r for r in ("residual", "y") if r in x]
    total, pieces = {}, []
    for r0 in range(0, case["rows"], 16384):
        t = {p: x[p].double() for p in params}
        t.update({r: x[r][r0:r0 + 16384].double() for r in rows})
        if not case["train"]:
            pieces.append(_exact_block(case, t))
            continue
        t = {name: v.requires_grad_() for name, v in t.items()}
        piece = _exact_block(case, t)
        wanted = rows + params
        grads = dict(zip(wanted, torch.autograd.grad(list(piece.values()), [t[w] for w in wanted],
                                                     [x["grad_" + o][r0:r0 + 16384].double() for o in piece])))
        for p in params:
            total["grad_" + p] = total.get("grad_" + p, 0) + grads[p]
        pieces.append({**{o: v.detach() for o, v in piece.items()}, **{"grad_" + r: grads[r] for r in rows}})
    return {**{name: torch.cat([p[name] for p in pieces]) for name in pieces[0]}, **total}


def _exact_bias(case, x):
    # the inputs' 32-bit coordinates are exact in 64 bits; buckets are whole numbers: the number of borders not above the distance
    d = x["pos"][x["src"]].double() - x["pos"][x["dst"]].double() + x["shift"].double()
    r2 = d[:, 0] * d[:, 0] + d[:, 1] * d[:, 1] + d[:, 2] * d[:, 2]
    buckets = torch.zeros_like(r2, dtype=torch.int32)
    for t in _thresholds(case).tolist():
        buckets += (r2 >= t * t).int()
    out = {"buckets": buckets, "bias": x["table"].double()[buckets.long()]}
    if case["train"]:
        order = torch.argsort(buckets, stable=True)
        sums = torch.cat([x["grad"].new_zeros(1, case["heads"], dtype=torch.float64), x["grad"].double()[order].cumsum(0)])
        ends = torch.searchsorted(buckets[order].contiguous(), torch.arange(case["buckets"] + 1, device="cuda", dtype=torch.int32))
        out["grad_table"] = sums[ends[1:]] - sums[ends[:-1]]
    return out


def _exact_attn(case, x):
    n, e, heads = case["dst"], case["edges"], case["heads"]
    index = torch.searchsorted(x["rowptr"][1:].contiguous(), torch.arange(e, device="cuda"), right=True)
    src = torch.arange(e, device="cuda") if x["src"] is None else x["src"]
    names = [name for name in ("q", "k", "v") if name in x]
    outs = {name: torch.zeros(x[name].shape, dtype=torch.float64, device="cuda") for name in names} if case["train"] else {}
    out = torch.zeros(n, x["q"].shape[1], dtype=torch.float64, device="cuda")
    table_grad, weight_grad = [], 0
    for h in range(heads):
        cols, at = [], 0
        for m, d in _blocks(case)[0]:
            cols += [at + c for c in range(h * (m // heads) * d, (h + 1) * (m // heads) * d)]
            at += m * d
        cols = torch.tensor(cols, device="cuda")
        t = {name: x[name][:, cols].double() for name in names}
        if "table" in x:
            t["table"] = x["table"][:, h].double()
        if "weight" in x:
            t["weight"] = x["weight"].double()
        if case["train"]:
            t = {name: v.requires_grad_() for name, v in t.items()}
        with torch.set_grad_enabled(case["train"]):
            logit = torch.einsum("ed,ed->e", t["q"][index], t["k"][src]) / math.sqrt(len(cols))
            if "table" in x:
                logit = logit + t["table"][x["bucket"].long()]
            # logits of a few tens at most: their exponentials need no shift in 64 bits
            num = torch.exp(logit)
            if "weight" in x:
                num = num * torch.where(t["weight"] > 0, t["weight"], torch.zeros_like(t["weight"]))
            den = torch.zeros(n, dtype=torch.float64, device="cuda").index_add(0, index, num)
            share = num / torch.where(den > 0, den, torch.ones_like(den))[index]
            o = torch.zeros(n, len(cols), dtype=torch.float64, device="cuda").index_add(0, index, share[:, None] * t["v"][src])
        out[:, cols] = o.detach()
        if case["train"]:
            grads = dict(zip(t, torch.autograd.grad(o, list(t.values()), x["grad"][:, cols].double())))
            for name in names:
                outs[name][:, cols] = grads[name]
            if "table" in x:
                table_grad.append(grads["table"])
            if "weight" in x:
                weight_grad = weight_grad + grads["weight"]
    result = {"out": out, **{"grad_" + name: g for name, g in outs.items()}}
    if case["train"] and "table" in x:
        result["grad_table"] = torch.stack(table_grad, 1)
    if case["train"] and "weight" in x:
        result["grad_weight"] = weight_grad
    return result


def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] in ("rms", "norm"):
        return _exact_rows(case, x)
    if case["op"] == "bias":
        return _exact_bias(case, x)
    return _exact_attn(case, x)


# ---------------------------------------------------------------------------------------------------------- work of a pass
def work(case):
    size = 4 if case["type"] == "fp32" else 2
    train = case["train"]
    if case["op"] in ("rms", "norm"):
        out, inner = _blocks(case)
        d, di, rows = _dim(out), _dim(inner), case["rows"]
        if case["op"] == "rms":
            columns, params, flops = (2 * d, _muls(out), 5 * d) if not train else (4 * d, 2 * _muls(out), 17 * d)
        else:
            n_params = _muls(inner) + 2 * _muls(out)
            columns, params, flops = (di + 3 * d, n_params, 8 * di + 10 * d)
            if train:
                columns, params, flops = 2 * di + 6 * d, 2 * n_params, 24 * di + 30 * d
        return {"bytes": rows * columns * size + 4 * params, "flops": rows * flops}
    e = case["edges"]
    if case["op"] == "bias":
        h, table = case["heads"], case["buckets"] * case["heads"] * size
        moved = 12 * case["nodes"] + e * (16 + 12 + 4 + h * size) + table
        if train:
            moved += e * h * size + table
        return {"bytes": moved, "flops": e * (20 + (h if train else 0))}
    d, h, n = _dim(_blocks(case)[0]), case["heads"], case["dst"]
    keys = e if case["per_edge"] else case["src"]
    nodes, edges = (2 * n + 2 * keys) * d * size, 0 if case["per_edge"] else 8 * e
    table = 4 * case["buckets"] * h
    if case["buckets"]:
        edges += 4 * e
    if case["weight"]:
        edges += 4 * e
    flops = e * (4 * d + 8 * h)
    if train:       # further: the output's gradient in, the gradients of q, k and v out
        nodes += (2 * n + 2 * keys) * d * size
        edges += 4 * e if case["weight"] else 0
        table *= 2
        flops += e * (8 * d + 12 * h)
    return {"bytes": nodes + edges + table + 8 * (n + 1), "flops": flops}
