"""Neighbour attention in 64 bits with its gradients written out, and how far a kernel that computes in fp32 may be from each number.

    a = scale <q, k> + bias + log w      p = softmax(a)      out = sum p v
    dp = <g, v>      delta = <g, out>      da = p (dp - delta)
    grad q = scale sum da k      grad k = scale sum da q      grad v = sum p g      grad bias = da      grad w = sum_h da / w

Bounds, with u = 2^-24, d = min(columns a head, 38) (a lane adds at most 32 of them, five shuffles the lanes), n edges a row, L the largest sum of magnitudes behind a logit of the row (scale <|q|, |k|> +
|bias| + |log w|).  A logit is off by (d + 3) u L; an exponential by 2 (2 + 1.18 * 2L) u of itself (its documented error) and by the
logit's error, its own and the one in the row's sum; the sum adds n u, every rise of the running maximum (at most n) 4 u and, all
together, 5 L u.  So a share is within  eps = (16 + 5n + (4d + 32) L) u  of itself.  The rest are sums of products, one rounding each,
of terms whose magnitudes are added up here one by one: sum p |v| for the output, P = p (<|g|, |v|> + <|g|, sum p |v|>) for da.  A result is
rounded once to its type, by half a step at most (below the normal numbers, half the step there); shares below 2^-126 may be zero.
"""
import math

import torch

from e3nn_b200 import o3

U32 = 2.0 ** -24


def head_columns(irreps, heads):
    cols, at = [[] for _ in range(heads)], 0
    for mul, ir in o3.Irreps(irreps):
        run = mul // heads * ir.dim
        for h in range(heads):
            cols[h] += range(at + h * run, at + (h + 1) * run)
        at += mul * ir.dim
    return torch.tensor(cols)


def formula(irreps_qk, irreps_v, heads, t, dtype, steps=None):
    """``{name: (value, bound)}`` of out and the gradients of q, k, v, bias and weight (where `t` has them), on the device of `t`.
    `t`: q, k, v, g, rowptr and, or None, src, perm, bias, buckets, weight.  `steps`: additions that follow one another in any sum, at most
    (default: as many as it has terms); long sums are split."""
    dev = t["q"].device
    cq, cv = head_columns(irreps_qk, heads).to(dev), head_columns(irreps_v, heads).to(dev)
    (H, d), dv, scale = cq.shape, cv.shape[1], cq.shape[1] ** -0.5
    N, S, rowptr = t["q"].shape[0], t["k"].shape[0], t["rowptr"]
    E = S if t["src"] is None else t["src"].shape[0]
    dst = torch.repeat_interleave(torch.arange(N, device=dev), rowptr[1:] - rowptr[:-1])
    slots = torch.arange(int(rowptr[0]), int(rowptr[-1]), device=dev)
    e = slots if t["perm"] is None else t["perm"][slots]
    r = e if t["src"] is None else t["src"][e]
    q, k, v, g = (t[n].double() for n in ("q", "k", "v", "g"))
    b = torch.zeros(len(e), H, dtype=torch.float64, device=dev)
    use = torch.ones(len(e), H, dtype=torch.bool, device=dev)
    if t["buckets"] is not None:
        b = t["bias"].double()[t["buckets"][e].long()]
    elif t["bias"] is not None:
        b = t["bias"].double()[e]
        use = b > -math.inf
    w = torch.ones(len(e), dtype=torch.float64, device=dev) if t["weight"] is None else t["weight"].double()[e]
    use = use & (w > 0)[:, None]

    def where(x):                                   # what is masked is not looked at
        return torch.where(use[:, :, None], x, torch.zeros_like(x))
    def rows(x, index, size):                       # sums over the edges of a row
        return torch.zeros(size, *x.shape[1:], dtype=torch.float64, device=dev).index_add(0, index, x)
    def columns(x, cols, width):
        return torch.zeros(x.shape[0], width, dtype=torch.float64, device=dev).index_copy(1, cols.flatten(), x.flatten(1))

    Q, K, V, G = where(q[:, cq][dst]), where(k[:, cq][r]), where(v[:, cv][r]), g[:, cv]
    b, lw = torch.where(use, b, 0.0), torch.where(use, w[:, None], 1.0).log()
    a = scale * (Q * K).sum(2) + b + lw
    high = torch.full((N, H), -math.inf, dtype=torch.float64, device=dev)
    amax = lambda x: high.scatter_reduce(0, dst[:, None].expand(-1, H), torch.where(use, x, -math.inf), "amax")
    ex = torch.where(use, torch.exp(a - torch.where(use, amax(a)[dst], 0.0)), 0.0)
    total = rows(ex, dst, N)
    p = ex / torch.where(total > 0, total, 1.0)[dst]
    out = rows(p[:, :, None] * V, dst, N)
    out_abs = rows(p[:, :, None] * V.abs(), dst, N)
    Gd = where(G[dst])
    da = p * ((Gd * V).sum(2) - (Gd * out[dst]).sum(2))
    at_most = lambda x: x if steps is None else x.clamp(max=steps)
    n = at_most((rowptr[1:] - rowptr[:-1]).double()[:, None])
    L = amax(scale * (Q.abs() * K.abs()).sum(2) + b.abs() + lw.abs()).clamp(min=0.0)
    d_steps, v_steps = min(d, 38), min(dv, 38)
    eps = U32 * (16 + 5 * n + (4 * d_steps + 32) * L)
    P = p * ((Gd.abs() * V.abs()).sum(2) + (Gd.abs() * out_abs[dst]).sum(2))
    e_da = 2 * eps[dst] + (v_steps + 2 * n[dst] + 6) * U32       # relative to P; with the roundings of a sum over the row

    per = dst if t["src"] is None else r
    n_out = 1.0 if t["src"] is None else at_most(torch.bincount(r, minlength=S).double()[r][:, None]) if len(r) else 1.0
    e_out = U32 * n_out
    value, bound = {}, {}
    value["out"], bound["out"] = columns(out, cv, v.shape[1]), columns(out_abs * (eps + (n + 2) * U32)[:, :, None], cv, v.shape[1])
    value["q"] = columns(scale * rows(da[:, :, None] * K, dst, N), cq, q.shape[1])
    bound["q"] = columns(scale * rows((P * e_da)[:, :, None] * K.abs(), dst, N), cq, q.shape[1])
    value["k"] = columns(scale * rows(da[:, :, None] * Q, r, S), cq, k.shape[1])
    bound["k"] = columns(scale * rows((P * (e_da + e_out))[:, :, None] * Q.abs(), r, S), cq, k.shape[1])
    value["v"] = columns(rows(p[:, :, None] * Gd, r, S), cv, v.shape[1])
    bound["v"] = columns(rows((p * (eps[dst] + e_out + 2 * U32))[:, :, None] * Gd.abs(), r, S), cv, v.shape[1])
    if t["bias"] is not None:
        if t["buckets"] is None:
            value["bias"], bound["bias"] = rows(da, e, E), rows(P * e_da, e, E)
        else:
            bucket, num = t["buckets"][e].long(), t["bias"].shape[0]
            count = at_most(torch.bincount(bucket, minlength=num).double()[bucket][:, None]) if len(e) else 1.0
            value["bias"], bound["bias"] = rows(da, bucket, num), rows(P * (e_da + count * U32), bucket, num)
    if t["weight"] is not None:
        inv = torch.where(w > 0, 1 / torch.where(w > 0, w, 1.0), 0.0)
        value["weight"], bound["weight"] = rows(da.sum(1) * inv, e, E), rows((P * (e_da + (H + 2) * U32)).sum(1) * inv, e, E)
    result = {}
    for name, x in value.items():
        to = torch.float32 if name in ("bias", "weight") else dtype
        result[name] = (x, bound[name] + torch.finfo(to).eps / 2 * (x.abs() + torch.finfo(to).tiny) + 2.0 ** -120, to)
    return result


def compare(got, want, sharp=0.25):
    """Every number within its bound; and the bounds say something: on average they are below `sharp` of the values' size."""
    for name, x in got.items():
        value, bound, dtype = want[name]
        assert x.dtype == dtype and x.shape == value.shape, name
        if value.numel() == 0:
            continue
        excess = ((x.to(value.device).double() - value).abs() / bound).max().item()
        assert excess <= 1.0, f"{name}: {excess:.2f} x the bound"
        size = value.abs().mean().item()
        if sharp is not None and size > 0:
            assert bound.mean().item() < sharp * size, f"{name}: a bound of {bound.mean().item():.2e} tells nothing about values of {size:.2e}"
