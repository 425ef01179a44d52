"""NeighborAttention against its formula in 64 bits, row by row, gradients by automatic differentiation of that formula.

Bounds.  Outputs and gradients are rounded once to their type (`finfo.eps / 2` of the value).  Before that they are fp32.  A logit is a
sum of up to d products, off by (d / lanes + 12) 2^-24 of sum |q k| scale and by 2^-24 of itself per further step; with d <= 64 a
head and logits of a few units here that is below 64 2^-24 =: r relative in a share, and the sum over n edges adds n 2^-24, so an output is
within (64 + n) 2^-24 of sum share |v|.  Gradients multiply a share (r), dp - delta (sums of d products) and k or q, and add n such terms:
(256 + n) 2^-24 of the sum of the magnitudes, which is bounded by the largest |g| |v| d |k| n (scale) there is.
"""
import math

import pytest
import torch

import e3nn_b200
from e3nn_b200 import nn as bnn
from e3nn_b200 import o3
from oracle import e3nn_oracle as orc
from test_gpu_norm import gate64, norm64

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def head_columns(irreps, heads):
    cols, at = [[] for _ in range(heads)], 0
    for mul, ir in o3.Irreps(irreps):
        run = mul // heads * ir.dim
        for h in range(heads):
            cols[h] += range(at + h * run, at + (h + 1) * run)
        at += mul * ir.dim
    return cols


def attention64(irreps_qk, irreps_v, heads, q, k, v, rowptr, src=None, perm=None, bias=None, buckets=None, weight=None):
    rows = []
    cqk, cv = head_columns(irreps_qk, heads), head_columns(irreps_v, heads)
    for n in range(len(rowptr) - 1):
        slots = torch.arange(rowptr[n], rowptr[n + 1])
        e = slots if perm is None else perm[slots]
        if weight is not None:
            e = e[weight[e] > 0]
        r = e if src is None else src[e]
        out = torch.zeros(v.shape[1], dtype=torch.float64)
        pieces = []
        for h in range(heads):
            a = (q[n, cqk[h]] * k[r][:, cqk[h]]).sum(1) / math.sqrt(len(cqk[h]))
            keep = torch.ones(len(e), dtype=torch.bool)
            if buckets is not None:
                a = a + bias[buckets[e].long(), h]
            elif bias is not None:
                keep = bias[e, h].detach() > -math.inf
                a = a[keep] + bias[e, h][keep]
            if weight is not None:
                a = a + torch.log(weight[e][keep])
            if a.numel() == 0:
                pieces.append(torch.zeros(len(cv[h]), dtype=torch.float64))
                continue
            pieces.append(torch.softmax(a, 0) @ v[r][keep][:, cv[h]])
        out = torch.zeros(v.shape[1], dtype=torch.float64).index_add(0, torch.tensor(sum(cv, [])), torch.cat(pieces))
        rows.append(out)
    return torch.stack(rows) if rows else torch.zeros(0, v.shape[1], dtype=torch.float64)


def close(got, ref, dtype, terms, size):
    assert got.dtype == dtype and got.shape == ref.shape
    if ref.numel() == 0:
        return
    half = torch.finfo(dtype).eps / 2
    bound = half * ref.abs() + terms * U32 * size + torch.finfo(dtype).tiny
    excess = ((got.cpu().double() - ref).abs() / bound).max().item()
    assert excess <= 1.0, f"{excess:.2f} x the bound"


DEGREES = {
    "one edge": [1],
    "ragged": [0, 3, 1, 0, 0, 37, 2, 5, 33, 0],
    "many empty": [0] * 300 + [4] + [0] * 100,
    "long row": [700],
    "hub": [2, 1, 600, 0, 3],
    "no edges": [0, 0, 0],
}
SHAPES = [("1x0e", "1x0e", 1), ("4x0e+4x1o", "4x0e+4x1o", 2), ("6x0e+3x1o", "3x0e+3x2e", 3), ("8x0e+8x1o+8x2e", "16x0e+8x1o", 8),
          ("40x0e+20x1o", "20x0e+20x1o", 20), ("34x0e", "34x1o", 34)]


def make(irreps_qk, irreps_v, heads, degrees, dtype, per_edge, bias, weight, perm, seed=0, sources=23):
    gen = torch.Generator().manual_seed(seed + heads + len(degrees))
    N, E = len(degrees), sum(degrees)
    dqk, dv = o3.Irreps(irreps_qk).dim, o3.Irreps(irreps_v).dim
    S = E if per_edge else sources
    t = {"rowptr": torch.tensor([0] + degrees).cumsum(0), "src": None if per_edge else torch.randint(S, (E,), generator=gen),
         "perm": torch.randperm(E, generator=gen) if perm else None, "buckets": None, "bias": None, "weight": None,
         "q": torch.randn(N, dqk, generator=gen).to(dtype), "k": torch.randn(S, dqk, generator=gen).to(dtype),
         "v": torch.randn(S, dv, generator=gen).to(dtype), "g": torch.randn(N, dv, generator=gen).to(dtype)}
    if bias == "table":
        t["buckets"] = torch.randint(9, (E,), generator=gen, dtype=torch.int32)
        t["bias"] = torch.randn(9, heads, generator=gen)
    elif bias == "edges":
        t["bias"] = torch.randn(E, heads, generator=gen)
        t["bias"][torch.rand(E, heads, generator=gen) < 0.2] = -math.inf
    if weight:
        t["weight"] = 0.05 + 0.95 * torch.rand(E, generator=gen)
        t["weight"][torch.rand(E, generator=gen) < 0.2] = 0.0
    return t


NAMES = ("q", "k", "v", "bias", "weight")


def check(irreps_qk, irreps_v, heads, t, dtype, transposed=True):
    mod = bnn.NeighborAttention(irreps_qk, irreps_v, heads).cuda()
    dev = {n: None if x is None else x.cuda() for n, x in t.items()}
    leaves = {n: dev[n].requires_grad_() for n in NAMES if dev[n] is not None}
    transpose = None
    if t["src"] is not None and transposed:
        transpose = e3nn_b200.csr_from_dst(dev["src"], t["k"].shape[0])
    out = mod(dev["q"], dev["k"], dev["v"], dev["rowptr"], dev["src"], perm=dev["perm"], bias=dev["bias"], buckets=dev["buckets"],
              edge_weight=dev["weight"], transpose=transpose)
    got = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), dev["g"], retain_graph=True)))
    again = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), dev["g"])))
    assert all(torch.equal(got[n], again[n]) for n in got)
    with torch.no_grad():
        assert torch.equal(out, mod(dev["q"], dev["k"], dev["v"], dev["rowptr"], dev["src"], perm=dev["perm"], bias=dev["bias"],
                                    buckets=dev["buckets"], edge_weight=dev["weight"]))
    ref_leaves = {n: t[n].double().requires_grad_() for n in leaves}
    x = {n: ref_leaves.get(n) for n in NAMES}
    ref = attention64(irreps_qk, irreps_v, heads, x["q"], x["k"], x["v"], t["rowptr"], t["src"], t["perm"], x["bias"], t["buckets"], x["weight"])
    n = int((t["rowptr"][1:] - t["rowptr"][:-1]).max()) if len(t["rowptr"]) > 1 else 0
    close(out.detach(), ref.detach(), dtype, 64 + n, t["v"].double().abs().max() if t["v"].numel() else 1.0)
    if ref.requires_grad:
        refs = torch.autograd.grad(ref, list(ref_leaves.values()), t["g"].double(), allow_unused=True)
    else:
        refs = [None] * len(ref_leaves)
    e3nn_b200.check_status()
    d, dvh = o3.Irreps(irreps_qk).dim // heads, o3.Irreps(irreps_v).dim // heads
    big = {m: t[m].double().abs().max().item() if t[m] is not None and t[m].numel() else 1.0 for m in ("q", "k", "v", "g")}
    da = 2 * big["g"] * big["v"] * dvh                     # |p (dp - delta)| per edge
    out_deg = int(torch.bincount(t["src"], minlength=1).max()) if t["src"] is not None and t["src"].numel() else 1
    sizes = {"q": da * big["k"] * d ** -0.5, "k": da * big["q"] * d ** -0.5 * out_deg, "v": big["g"] * out_deg,
             "bias": da * (max(1, t["buckets"].numel()) if t["buckets"] is not None else 1), "weight": da * heads / 0.05}
    for m, r in zip(ref_leaves, refs):
        r = torch.zeros_like(ref_leaves[m]) if r is None else r
        close(got[m], torch.nan_to_num(r), torch.float32 if m in ("bias", "weight") else dtype, 256 + max(n, out_deg), sizes[m])
    return out, got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}-{s[2]}")
@pytest.mark.parametrize("per_edge", [False, True])
def test_heads_types_and_layouts(shape, per_edge, dtype):
    check(*shape, make(*shape, DEGREES["ragged"], dtype, per_edge, "table", True, False), dtype)


@pytest.mark.parametrize("degrees", list(DEGREES))
@pytest.mark.parametrize("per_edge", [False, True])
@pytest.mark.parametrize("bias,weight,perm", [(None, False, False), ("table", False, True), ("edges", True, True), ("edges", False, False)])
def test_lengths_biases_weights_and_permuted_edges(degrees, per_edge, bias, weight, perm):
    shape = ("4x0e+4x1o", "4x0e+4x1o", 2)
    check(*shape, make(*shape, DEGREES[degrees], torch.float32, per_edge, bias, weight, perm), torch.float32)


def test_transposed_edges_are_built_when_they_are_not_given():
    shape = ("4x0e+4x1o", "4x0e+4x1o", 2)
    t = make(*shape, DEGREES["ragged"], torch.float32, False, "table", True, True)
    _, a = check(*shape, t, torch.float32)
    _, b = check(*shape, t, torch.float32, transposed=False)
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("irreps,heads", [("256x0e+256x1o", 1), ("1023x0e", 1), ("64x0e+64x1o+64x2e+64x3o", 8), ("64x0e+64x1o+64x2e+64x3o", 16),
                                          ("20x0e+20x1o+20x2e", 2), ("4096x0e", 8)])
def test_wide_heads(irreps, heads):
    t = make(irreps, irreps, heads, [3, 0, 40], torch.float32, False, "table", False, False)
    t["q"] *= 0.3                                       # logits of a few units, as the bound assumes
    mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
    ref = attention64(irreps, irreps, heads, *(t[n].double() for n in "qkv"), t["rowptr"], t["src"], None, t["bias"].double(), t["buckets"])
    out = mod(*(t[n].cuda() for n in "qkv"), t["rowptr"].cuda(), t["src"].cuda(), bias=t["bias"].cuda(), buckets=t["buckets"].cuda())
    close(out, ref, torch.float32, 64 + 40 + o3.Irreps(irreps).dim // heads, t["v"].double().abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("irreps,heads", [("8x0e+8x1o", 4), ("6x0e+3x1o", 3), ("64x0e+64x1o+64x2e+64x3o", 8)])
@pytest.mark.parametrize("per_edge", [False, True])
def test_large_graph(irreps, heads, per_edge, dtype):
    """Enough edges for whole blocks of warps, uneven rows and one hub: the formula in 64 bits over all edges at once."""
    gen = torch.Generator().manual_seed(heads)
    N, D = 900, o3.Irreps(irreps).dim
    degrees = (torch.rand(N, generator=gen) ** 3 * 40).long()
    degrees[17], degrees[400:420] = 900, 0
    rowptr = torch.cat([torch.zeros(1, dtype=torch.int64), degrees.cumsum(0)])
    E = int(rowptr[-1])
    S = E if per_edge else 700
    src = None if per_edge else torch.randint(S, (E,), generator=gen)
    q, k, v, g = (torch.randn(n, D, generator=gen).to(dtype).cuda() for n in (N, S, S, N))
    weight = (0.1 + 0.9 * torch.rand(E, generator=gen)).cuda()
    table, buckets = torch.randn(7, heads, generator=gen).cuda(), torch.randint(7, (E,), generator=gen, dtype=torch.int32).cuda()
    dst = torch.repeat_interleave(torch.arange(N), degrees).cuda()
    mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
    leaves = [t.clone().requires_grad_() for t in (q, k, v, table, weight)]
    src_d = None if src is None else src.cuda()
    out = mod(*leaves[:3], rowptr.cuda(), src_d, bias=leaves[3], buckets=buckets, edge_weight=leaves[4],
              transpose=None if src is None else e3nn_b200.csr_from_dst(src_d, S))
    got = torch.autograd.grad(out, leaves, g)
    e3nn_b200.check_status()
    cols = torch.tensor(head_columns(irreps, heads)).cuda()
    x = [t.double().requires_grad_() for t in (q, k, v, table, weight)]
    r = torch.arange(S, device="cuda") if src is None else src_d
    a = (x[0][:, cols][dst] * x[1][:, cols][r]).sum(2) * cols.shape[1] ** -0.5 + x[3][buckets.long()] + torch.log(x[4])[:, None]
    top = torch.full((N, heads), -math.inf, dtype=torch.float64, device="cuda").scatter_reduce(0, dst[:, None].expand(-1, heads), a.detach(), "amax")
    p = torch.exp(a - top[dst])
    p = p / torch.zeros(N, heads, dtype=torch.float64, device="cuda").index_add(0, dst, p)[dst]
    o = torch.zeros(N, *cols.shape, dtype=torch.float64, device="cuda").index_add(0, dst, p[:, :, None] * x[2][:, cols][r])
    ref = torch.zeros(N, D, dtype=torch.float64, device="cuda").index_copy(1, cols.flatten(), o.reshape(N, D))
    refs = torch.autograd.grad(ref, x, g.double())
    n, d = 900, D // heads
    out_deg = 1 if src is None else int(torch.bincount(src).max())
    close(out.detach(), ref.detach().cpu(), dtype, 64 + n, v.abs().max().item())
    da = 2 * g.abs().max().item() * v.abs().max().item() * d
    sizes = (da * k.abs().max().item() * d ** -0.5, da * q.abs().max().item() * d ** -0.5 * out_deg, g.abs().max().item() * out_deg, da * E, da * heads / 0.1)
    for a, b, size, t in zip(got, refs, sizes, (dtype, dtype, dtype, torch.float32, torch.float32)):
        close(a, b.cpu(), t, 256 + max(n, out_deg), size)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_single_query_over_a_long_list(dtype):
    """Parts inside one row are added up in blocks first; the join reads the blocks' sums."""
    irreps, heads, E = "8x0e+8x1o", 4, 30011
    t = make(irreps, irreps, heads, [E], dtype, True, "table", False, False)
    mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
    q, k, v = (t[n].cuda().requires_grad_() for n in "qkv")
    out = mod(q, k, v, t["rowptr"].cuda(), bias=t["bias"].cuda(), buckets=t["buckets"].cuda())
    q64, k64, v64 = (t[n].double().requires_grad_() for n in "qkv")
    ref = attention64(irreps, irreps, heads, q64, k64, v64, t["rowptr"], None, None, t["bias"].double(), t["buckets"])
    # sums of parts of at most 256 edges, then of at most E / 32 parts
    terms = 64 + 256 + E // 32
    close(out.detach(), ref.detach(), dtype, terms, 1.0)
    for got, r, size in zip(torch.autograd.grad(out, (q, k, v), t["g"].cuda()), torch.autograd.grad(ref, (q64, k64, v64), t["g"].double()), (20.0, 1.0, 1.0)):
        close(got, r, dtype, terms, size)


def test_many_sources_of_one_node_and_one_source_of_many():
    """One source that every edge leaves from: its gradient row is joined from many parts."""
    irreps, heads = "4x0e+4x1o", 2
    t = make(irreps, irreps, heads, [3] * 400, torch.float32, False, None, False, False)
    t["src"][:] = 5
    check(irreps, irreps, heads, t, torch.float32)


def test_one_edge_has_share_one_and_no_gradient_through_it():
    irreps, heads, N = "4x0e+4x1o", 2, 50
    t = make(irreps, irreps, heads, [1] * N, torch.float32, True, None, False, False)
    mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
    weight = torch.logspace(-30, 0, N).cuda().requires_grad_()          # down to a weight that is nearly nothing
    q, k, v = (t[n].cuda().requires_grad_() for n in "qkv")
    out = mod(q, k, v, t["rowptr"].cuda(), edge_weight=weight)
    assert torch.equal(out, v)
    gq, gk, gv, gw = torch.autograd.grad(out, (q, k, v, weight), t["g"].cuda())
    for zero in (gq, gk, gw):
        assert torch.equal(zero, torch.zeros_like(zero))
    assert torch.equal(gv, t["g"].cuda())


def test_masked_places_may_hold_anything():
    irreps, heads, E = "4x0e+4x1o", 2, 40
    t = make(irreps, irreps, heads, [10, 30], torch.float32, True, None, False, False)
    mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
    rowptr = t["rowptr"].cuda()
    bad = torch.zeros(E, dtype=torch.bool)
    bad[[0, 3, 11, 25, 39]] = True
    for value in (float("nan"), float("inf"), -float("inf")):
        def run(fill, **kw):
            k, v = t["k"].clone(), t["v"].clone()
            if fill:
                k[bad], v[bad] = value, value
            leaves = [x.cuda().requires_grad_() for x in (t["q"], k, v)]
            out = mod(*leaves, rowptr, **kw)
            return [out.detach(), *torch.autograd.grad(out, leaves, t["g"].cuda())]
        weight = torch.where(bad, 0.0, 1.0).cuda()
        mask = torch.where(bad, -float("inf"), 0.0)[:, None].repeat(1, heads).cuda()
        for kw in ({"edge_weight": weight}, {"bias": mask}):
            for a, b in zip(run(True, **kw), run(False, **kw)):
                assert torch.equal(a, b)
    # a row whose mask leaves nothing, by either way: zeros, and no gradient
    for kw in ({"edge_weight": torch.zeros(E).cuda()}, {"bias": torch.full((E, heads), -float("inf")).cuda()}):
        leaves = [t[n].cuda().requires_grad_() for n in "qkv"]
        out = mod(*leaves, rowptr, **kw)
        assert torch.equal(out, torch.zeros_like(out))
        assert all(torch.equal(g, torch.zeros_like(g)) for g in torch.autograd.grad(out, leaves, t["g"].cuda()))
    # the type's lowest value everywhere in a row: all alike, so the plain mean of the values
    low = torch.full((E, heads), torch.finfo(torch.float32).min).cuda()
    out = mod(*(t[n].cuda() for n in "qkv"), rowptr, bias=low)
    ref = torch.stack([t["v"][:10].double().mean(0), t["v"][10:].double().mean(0)])
    close(out, ref, torch.float32, 64 + 30, t["v"].double().abs().max())


def test_slots_behind_the_last_row_are_left_alone():
    irreps, heads = "4x0e+4x1o", 2
    for per_edge in (True, False):
        t = make(irreps, irreps, heads, [5, 0, 9], torch.float32, per_edge, "edges", True, False, sources=14)
        t["bias"].clamp_(min=-3.0)
        pad = 300
        mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
        def run(padded):
            x = {n: None if y is None else y.clone() for n, y in t.items()}
            if padded:
                x["bias"] = torch.cat([x["bias"], torch.full((pad, heads), float("nan"))])
                x["weight"] = torch.cat([x["weight"], torch.full((pad,), float("nan"))])
                if per_edge:
                    x["k"], x["v"] = (torch.cat([x[n], torch.full((pad, 16), float("nan"))]) for n in "kv")
                else:
                    x["src"] = torch.cat([x["src"], torch.zeros(pad, dtype=torch.int64)])
            x = {n: None if y is None else y.cuda() for n, y in x.items()}
            leaves = [x[n].requires_grad_() for n in NAMES]
            out = mod(x["q"], x["k"], x["v"], x["rowptr"], x["src"], bias=x["bias"], edge_weight=x["weight"])
            return [out.detach(), *torch.autograd.grad(out, leaves, x["g"])]
        for a, b in zip(run(True), run(False)):
            n = b.shape[0]
            assert torch.equal(a[:n], b) and torch.equal(a[n:], torch.zeros_like(a[n:]))


def test_strides_slices_and_broadcast_rows():
    irreps, heads = "4x0e+4x1o", 2
    t = make(irreps, irreps, heads, DEGREES["ragged"], torch.float32, False, None, False, False, sources=10)
    mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
    rowptr, src = t["rowptr"].cuda(), t["src"].cuda()
    packed = torch.cat([t["q"], t["k"], t["v"]], 1).cuda()
    q, k, v = (t[n].cuda() for n in "qkv")
    ref = mod(q, k, v, rowptr, src)
    p = packed.requires_grad_()
    out = mod(*p.split([16, 16, 16], 1), rowptr, src)
    assert torch.equal(out, ref)                           # rows 48 elements apart: the same vectors
    (gp,) = torch.autograd.grad(out, p, t["g"].cuda())
    leaves = [x.requires_grad_() for x in (q, k, v)]
    assert torch.equal(gp, torch.cat(torch.autograd.grad(mod(*leaves, rowptr, src), leaves, t["g"].cuda()), 1))
    tol = dict(rtol=0, atol=100 * U32 * 5)
    odd = torch.zeros(10, 51, device="cuda")               # rows 51 elements apart: single elements
    odd[:, 1:49] = packed.detach()
    assert torch.allclose(mod(*odd[:, 1:49].split([16, 16, 16], 1), rowptr, src), ref, **tol)
    turned = q.detach().T.contiguous().T                   # columns apart: copied
    assert torch.equal(mod(turned, k, v, rowptr, src), ref)
    one = q.detach()[:1].expand(10, 16).requires_grad_()
    (g1,) = torch.autograd.grad(mod(one, k.detach(), v.detach(), rowptr, src), one, t["g"].cuda())
    dense = one.detach().clone().requires_grad_()
    (g2,) = torch.autograd.grad(mod(dense, k.detach(), v.detach(), rowptr, src), dense, t["g"].cuda())
    assert torch.equal(g1, g2)
    wrong = torch.zeros(17 * 10, device="cuda")[1:161].view(10, 16).copy_(t["g"])      # a cotangent that is not aligned
    out = mod(*leaves, rowptr, src)
    for a, b in zip(torch.autograd.grad(out, leaves, wrong, retain_graph=True), torch.autograd.grad(out, leaves, t["g"].cuda())):
        assert torch.equal(a, b)


def test_rows_beyond_32_bit_offsets():
    """Keys and values whose last rows start past 2^31 elements."""
    irreps, heads, d = "256x0e", 8, 256
    S = 2 ** 31 // d + 1000
    k = torch.zeros(S, d, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(0)
    E = 40
    rows = torch.randn(E, d, generator=gen).bfloat16()
    src = torch.cat([torch.arange(20), torch.arange(S - 20, S)])
    k[src.cuda()] = rows.cuda()
    q = torch.randn(2, d, generator=gen).bfloat16()
    rowptr = torch.tensor([0, 17, 40])
    mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
    out = mod(q.cuda(), k, k, rowptr.cuda(), src.cuda())
    ref = attention64(irreps, irreps, heads, q.double(), rows.double(), rows.double(), rowptr)
    close(out, ref, torch.bfloat16, 64 + 40, rows.double().abs().max())


def test_difference_quotient():
    irreps, heads = "2x0e+2x1o", 2
    t = make(irreps, irreps, heads, [3, 6], torch.float32, False, "table", True, False, sources=5)
    t["weight"][:] = 0.2 + 0.5 * torch.rand(9, generator=torch.Generator().manual_seed(1))
    mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
    x = {n: None if y is None else y.cuda() for n, y in t.items()}
    gen = torch.Generator().manual_seed(2)
    step = {n: (0.3 * torch.randn(t[n].shape, generator=gen)).cuda() for n in NAMES}
    def value(s):
        y = {n: x[n] + s * step[n] for n in NAMES}
        return (mod(y["q"], y["k"], y["v"], x["rowptr"], x["src"], bias=y["bias"], buckets=x["buckets"], edge_weight=y["weight"]).double() * x["g"]).sum()
    leaves = {n: x[n].clone().requires_grad_() for n in NAMES}
    out = mod(leaves["q"], leaves["k"], leaves["v"], x["rowptr"], x["src"], bias=leaves["bias"], buckets=x["buckets"], edge_weight=leaves["weight"])
    slope = sum((g.double() * step[n]).sum() for n, g in zip(NAMES, torch.autograd.grad(out, list(leaves.values()), x["g"])))
    s = 2.0 ** -7
    quotient = (value(s) - value(-s)) / (2 * s)
    # truncation s^2 / 6 of a third derivative of about a hundred, roundings of the values 2^-24 * 50 / s
    assert abs(slope - quotient) < 200 * s * s / 6 + 50 * U32 / s


def test_bad_indices_are_reported_and_left_out():
    irreps, heads = "4x0e+4x1o", 2
    t = make(irreps, irreps, heads, [4, 6], torch.float32, False, "table", False, False)
    mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
    x = {n: None if y is None else y.cuda() for n, y in t.items()}
    good = torch.tensor([i for i in range(10) if i not in (1, 7)])
    rowptr = torch.tensor([0, 3, 8]).cuda()
    want = mod(x["q"], x["k"], x["v"], rowptr, x["src"][good.cuda()], bias=x["bias"], buckets=x["buckets"][good.cuda()])
    e3nn_b200.check_status()
    def run(**kw):
        a = dict(rowptr=x["rowptr"], edge_src=x["src"], bias=x["bias"], buckets=x["buckets"])
        a.update(kw)
        out = mod(x["q"], x["k"], x["v"], **a)
        with pytest.raises(IndexError):
            e3nn_b200.check_status()
        assert torch.allclose(out, want, rtol=0, atol=100 * U32 * 5)
    src, buckets, perm = x["src"].clone(), x["buckets"].clone(), torch.arange(10, device="cuda")
    src[1], src[7] = 23, -1
    run(edge_src=src)
    buckets[1], buckets[7] = 9, -5
    run(buckets=buckets)
    perm[1], perm[7] = 10, -1
    run(perm=perm)
    with pytest.raises(IndexError):
        mod(x["q"], x["k"], x["v"], x["rowptr"], src, check_indices=True)
    # a row pointer that runs past the edges, or backwards, reads nothing outside them
    mod(x["q"], x["k"], x["v"], torch.tensor([0, 8, 40], device="cuda"), x["src"])
    mod(x["q"], x["k"], x["v"], torch.tensor([5, 8, 2], device="cuda"), x["src"])
    e3nn_b200.check_status()


def test_captured_and_replayed_and_on_another_stream():
    irreps, heads = "4x0e+4x1o", 2
    t = make(irreps, irreps, heads, DEGREES["hub"], torch.float32, False, "table", True, False)
    mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
    x = {n: None if y is None else y.cuda() for n, y in t.items()}
    transpose = e3nn_b200.csr_from_dst(x["src"], 23)
    def step(q, k, v, bias, weight):
        leaves = [y.detach().requires_grad_() for y in (q, k, v, bias, weight)]
        out = mod(*leaves[:3], x["rowptr"], x["src"], bias=leaves[3], buckets=x["buckets"], edge_weight=leaves[4], transpose=transpose)
        return (out.detach(), *torch.autograd.grad(out, leaves, x["g"]))
    static = [x[n].clone() for n in NAMES]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        aside = step(*static)
    torch.cuda.current_stream().wait_stream(stream)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for graph in graphs:                                     # two graphs: neither uses the other's scratch memory
        with torch.cuda.graph(graph):
            outs.append(step(*static))
    for a, b in zip(aside, step(*static)):
        assert torch.equal(a, b)
    for s, n in zip(static, NAMES):
        if n != "weight":
            s.add_(0.1 * torch.randn_like(s))
    want = step(*static)
    graphs[0].replay()
    graphs[1].replay()
    for out in outs:
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_refusals():
    mod = bnn.NeighborAttention("4x0e+4x1o", "4x0e+4x1o", 2).cuda()
    q, rowptr, src = torch.randn(3, 16, device="cuda"), torch.tensor([0, 1, 2, 3], device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    ok = mod(q, q, q, rowptr, src)
    assert ok.shape == (3, 16)
    for args, kw in (((q, q.half(), q, rowptr, src), {}), ((q.double(), q.double(), q.double(), rowptr, src), {}), ((q, q, q, rowptr.int(), src), {}),
                     ((q, q, q, rowptr, src.int()), {}), ((q, q, q, rowptr, src), {"bias": torch.zeros(4, 2).cuda(), "buckets": src})):
        with pytest.raises(TypeError):
            mod(*args, **kw)
    for args, kw in (((q, q, q, rowptr[:3], src), {}), ((q, q, q[:, :15], rowptr, src), {}), ((q[0], q, q, rowptr, src), {}),
                     ((q, q, q[:2], rowptr, src), {}), ((q, q, q, rowptr, src), {"bias": torch.zeros(3, 3).cuda()}),
                     ((q, q, q, rowptr, src), {"edge_weight": torch.ones(2).cuda()}), ((q, q, q, rowptr, src), {"perm": src[:2]}),
                     ((q, q, q, rowptr, src), {"transpose": (src, rowptr[:3])})):
        with pytest.raises((AssertionError, RuntimeError)):
            mod(*args, **kw)
    with pytest.raises(ValueError):
        mod(q, q, q, rowptr, src, buckets=src.int())
    with pytest.raises((RuntimeError, NotImplementedError)):
        mod(q, q, q, rowptr.cpu(), src)
    with pytest.raises(RuntimeError, match="same device"):
        bnn.NeighborAttention("4x0e", "4x0e", 2)(q[:, :4], q[:, :4], q[:, :4], rowptr, src)
    x = q.clone().requires_grad_()
    for out in (mod(x, q, q, rowptr, src), mod(x, q, q, rowptr, src).pow(2)):      # the cotangent a constant, or a function of the leaf
        (g,) = torch.autograd.grad(out.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def graph_of_atoms(N, gen):
    pos = (N / 0.05) ** (1 / 3) * torch.rand(N, 3, generator=gen)
    box = max(15.0, (N / 0.05) ** (1 / 3))
    src, dst, shift, rowptr = bnn.neighbor_list_pbc(pos.cuda(), box, 5.0)
    return pos.cuda(), src, dst, shift, rowptr


def test_attention_block_as_it_is_used():
    """Norm, attention with distance bias and cutoff, norm-gate-residual, and the convolution block after it: against the same
    steps in 64 bits, and its gradients against differences."""
    torch.manual_seed(0)
    gen = torch.Generator().manual_seed(0)
    irreps, heads = "8x0e+8x1o+4x2e", 4
    pos, src, dst, shift, rowptr = graph_of_atoms(60, gen)
    N = pos.shape[0]
    pre = bnn.RMSNorm(irreps).cuda()
    bias = bnn.RelativeBias(16, heads, 5.0, r_linear=2.5).cuda()
    with torch.no_grad():
        bias.weight.normal_(0, 0.5)
    block = bnn.AttentionBlock(irreps, heads, linear_math_mode="fp32", scale_init=0.5).cuda()
    x = torch.randn(N, o3.Irreps(irreps).dim, generator=gen).cuda()
    r = (pos[src] - pos[dst] + shift).norm(dim=1)
    cutoff = 0.5 * (torch.cos(math.pi * r / 5.0) + 1)
    buckets = bias.buckets(pos, src, dst, shift)
    def run(x):
        return block(x, pre(x), rowptr, src, bias=bias.weight, buckets=buckets, edge_weight=cutoff)
    z, h = run(x)

    # the same in 64 bits
    c = lambda t: t.detach().cpu().double()
    ones = torch.ones(20, dtype=torch.float64)
    h0 = norm64(c(x), ones, irreps, 1e-5)
    key = str(o3.Irreps(irreps))
    qkv = orc.linear(key, str(o3.Irreps(irreps) + o3.Irreps(irreps) + o3.Irreps(irreps)), h0, c(block.lin_qkv.weight))
    D = o3.Irreps(irreps).dim
    att = attention64(irreps, irreps, heads, *qkv.split([D, D, D], 1), rowptr.cpu(), src.cpu(), None, c(bias.weight), buckets.cpu(), c(cutoff))
    y = orc.linear(key, str(block.lin_out.irreps_out), att, c(block.lin_out.weight))
    val = gate64(bnn.Gate("8x0e", [torch.nn.functional.silu], "12x0e", [torch.sigmoid], "8x1o+4x2e"),
                 norm64(y, torch.ones(block.post.weight_post.numel()).double(), str(block.post.irreps_in), 1e-5))
    z64 = c(x) + 0.5 * val
    h64 = norm64(z64, ones, irreps, 1e-5)
    # five steps of at most 512 terms each
    for got, ref in ((z, z64), (h, h64)):
        assert (got.detach().cpu().double() - ref).abs().max() < 1e-5 * ref.pow(2).mean().sqrt() * 5

    # a training step through all of it, followed by a convolution block; the slope along a direction against a difference
    conv = bnn.InteractionBlock(irreps, lmax=1, num_basis=4, hidden=32, r_max=5.0, num_neighbors=5.0, linear_math_mode="fp32", radial_math_mode="fp32").cuda()
    post = bnn.NormGateResidual(irreps=irreps).cuda()
    def loss(x):
        z, h = run(x)
        z, h = post(z, conv(pos, h, src, dst, rowptr, shift))
        return (z.double().pow(2).mean() + h.double().mean())
    params = [p for m in (pre, bias, block, conv, post) for p in m.parameters()]
    xr = x.clone().requires_grad_()
    grads = torch.autograd.grad(loss(xr), [xr] + params)
    assert all(torch.isfinite(g).all() for g in grads) and all(g.abs().max() > 0 for g in grads)
    direction = torch.randn(x.shape, generator=gen).cuda()
    s = 2.0 ** -6
    with torch.no_grad():
        quotient = (loss(x + s * direction) - loss(x - s * direction)) / (2 * s)
    slope = (grads[0].double() * direction).sum()
    assert abs(quotient - slope) < 2e-3 * max(1.0, abs(slope.item()))


def test_attention_block_commutes_with_rotations():
    torch.manual_seed(1)
    gen = torch.Generator().manual_seed(1)
    irreps = o3.Irreps("8x0e+8x1o+4x2e")
    pos, src, dst, shift, rowptr = graph_of_atoms(50, gen)
    block, pre = bnn.AttentionBlock(irreps, 2, linear_math_mode="fp32").cuda(), bnn.RMSNorm(irreps).cuda()
    x = torch.randn(pos.shape[0], irreps.dim, generator=gen).cuda()
    D = irreps.D_from_matrix(o3.rand_matrix()).float().cuda()
    a = block(x @ D.T, pre(x @ D.T), rowptr, src)
    for got, ref in zip(a, block(x, pre(x), rowptr, src)):
        assert (got - ref @ D.T).abs().max() < 1e-4
