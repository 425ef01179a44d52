"""RMSNorm and NormGateResidual against their formulas in 64 bits.

Bounds.  An output is rounded once (half a step of its type, `finfo.eps / 2` of the value).  Before that it is fp32: a value passes
a few dozen roundings (a sum of squares in a tree of at most a few hundred terms, its root, products, an activation of 2 ulp), each
2^-24 of a number not above the row's largest; 64 of them are allowed.  A parameter gradient is a sum over rows in which each
term has those roundings and the sum adds one per addition: (64 + rows) 2^-24 of the sum of the terms' magnitudes.
"""
import pytest
import torch

import e3nn_b200
from e3nn_b200 import nn as bnn
from e3nn_b200 import o3

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U32 = 2.0 ** -24


def norm64(x, w, irreps, eps):
    out, col, chan = [], 0, 0
    for mul, ir in o3.Irreps(irreps):
        b = x[:, col:col + mul * ir.dim].reshape(-1, mul, ir.dim)
        s = (b.pow(2).mean((1, 2), keepdim=True) + eps).rsqrt()
        out.append((b * s * w[None, chan:chan + mul, None]).reshape(-1, mul * ir.dim))
        col, chan = col + mul * ir.dim, chan + mul
    return torch.cat(out, 1)


ACT64 = {0: torch.nn.functional.silu, 1: torch.tanh, 2: torch.relu, 3: lambda t: t, 4: torch.sigmoid, 5: torch.abs}


def gate64(gate, n):
    """The gate from its own column table (input column, gate column, activation) and constants."""
    cols = []
    for (src, g, act), cst in zip(gate._out_tbl.tolist(), gate._out_cst.tolist()):
        cols.append(cst * ACT64[act](n[:, src]) if g < 0 else n[:, src] * cst * ACT64[act](n[:, g]))
    return torch.stack(cols, 1)


def close(got, ref, dtype, terms=64, size=None):
    """`size`: magnitude that the fp32 roundings are relative to (default: the largest of the row)."""
    assert got.dtype == dtype and got.shape == ref.shape
    if ref.numel() == 0:
        return
    size = ref.abs().amax(-1, keepdim=True) if size is None else size
    bound = torch.finfo(dtype).eps / 2 * ref.abs() + terms * U32 * size + torch.finfo(dtype).tiny
    excess = ((got.cpu().double() - ref).abs() / bound).max().item()
    assert excess <= 1.0, f"{excess:.2f} x the bound"


def rows_of(rows, dim, dtype, gen, std=1.0):
    return (std * torch.randn(rows, dim, generator=gen)).to(dtype)


LAYOUTS = ["1x0e", "3x1o", "4x0e+4x1o", "17x0e+9x1o+5x2e", "64x0e+64x1o+64x2e+64x3o", "2x5e+1x0o+3x0e", "16x0e+16x0e+8x1e",
           "700x0e+300x1o+200x2e", "1000x0e+501x1o"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("irreps", LAYOUTS)
@pytest.mark.parametrize("rows", [1, 2, 150])
def test_rms_norm(irreps, rows, dtype):
    gen = torch.Generator().manual_seed(rows)
    irreps = o3.Irreps(irreps)
    mod = bnn.RMSNorm(irreps, eps=1e-5).cuda()
    x, g = rows_of(rows, irreps.dim, dtype, gen, 3.0), rows_of(rows, irreps.dim, dtype, gen)
    w = 1 + 0.3 * torch.randn(irreps.num_irreps, generator=gen)
    with torch.no_grad():
        mod.weight.copy_(w)
    xd, wd = x.cuda().requires_grad_(), mod.weight
    h = mod(xd)
    gx, gw = torch.autograd.grad(h, (xd, wd), g.cuda())
    x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
    ref = norm64(x64, w64, irreps, 1e-5)
    rx, rw = torch.autograd.grad(ref, (x64, w64), g.double())
    close(h, ref.detach(), dtype)
    # the gradient subtracts two terms of the size of rstd * (g w): roundings are relative to those
    size = (norm64(x64, w64, irreps, 1e-5) / x64).abs().nan_to_num(0).amax(1, keepdim=True) * (g.double().abs() * w.abs().max()).amax(1, keepdim=True)
    close(gx, rx, dtype, size=size.detach())
    ones = torch.ones(irreps.num_irreps, dtype=torch.float64)
    terms = (g.double() * norm64(x.double(), ones, irreps, 1e-5)).abs()
    per_channel, col = [], 0
    for mul, ir in irreps:
        per_channel.append(terms[:, col:col + mul * ir.dim].reshape(rows, mul, ir.dim).sum((0, 2)))
        col += mul * ir.dim
    close(gw, rw, torch.float32, terms=64 + rows, size=torch.cat(per_channel))


def gates():
    silu, sig = torch.nn.functional.silu, torch.sigmoid
    return {
        "l2": bnn.Gate("32x0e", [silu], "64x0e", [sig], "32x1o+32x2e"),
        "odd": bnn.Gate("5x0e+3x0o", [silu, torch.tanh], "7x0e", [sig], "4x1o+2x1e+1x3o"),
        "odd gates": bnn.Gate("4x0e", [torch.relu], "4x0o", [torch.tanh], "4x1o"),
        "no scalars": bnn.Gate("", [], "4x0e", [sig], "4x1o"),
        "activation": bnn.Activation("8x0e+4x0o+4x1o", [silu, torch.abs, None]),
        "wide": bnn.Gate("600x0e", [silu], "500x0e", [sig], "300x1o+200x2e"),
        "wide odd": bnn.Gate("601x0e", [silu], "500x0e", [sig], "299x1o+201x2e"),
        "none": None,
        "l3": bnn.Gate("64x0e", [silu], "192x0e", [sig], "64x1o+64x2e+64x3o"),
    }


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", [n for n in gates() if n != "l3"])
@pytest.mark.parametrize("rows", [1, 77])
@pytest.mark.parametrize("pre", [True, False])
def test_norm_gate_residual(name, rows, dtype, pre):
    if pre is False and (dtype != torch.float32 or rows == 1):
        pytest.skip("one form of it is enough")
    check_norm_gate(name, rows, dtype, pre)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", [n for n in gates() if not n.startswith("wide")] + ["l3"])
@pytest.mark.parametrize("pre", [True, False])
def test_many_rows(name, dtype, pre):
    """From 1,184 rows on the forward pass takes a row per warp."""
    check_norm_gate(name, 1301, dtype, pre)


def check_norm_gate(name, rows, dtype, pre):
    gen = torch.Generator().manual_seed(len(name) + rows)
    gate = gates()[name]
    mod = bnn.NormGateResidual(gate, irreps="6x0e+3x1o" if gate is None else None, eps=1e-5, pre_norm=pre, scale_init=0.7)
    din, dout = mod.irreps_in.dim, mod.irreps_out.dim
    r, y = rows_of(rows, dout, dtype, gen), rows_of(rows, din, dtype, gen, 3.0)
    gz, gh = rows_of(rows, dout, dtype, gen), rows_of(rows, dout, dtype, gen)
    params = [mod.weight_post, mod.scale] + ([mod.weight_pre] if pre else [])
    with torch.no_grad():
        for p in params:
            p.copy_(1 + 0.3 * torch.randn(p.shape, generator=gen))
    p64 = [p.detach().clone().double().requires_grad_() for p in params]
    r64, y64 = r.double().requires_grad_(), y.double().requires_grad_()
    n = norm64(y64, p64[0], mod.irreps_in, 1e-5)
    val = n if gate is None else gate64(gate, n)
    per_col = torch.repeat_interleave(torch.arange(mod.scale.numel()), torch.tensor([ir.dim for mul, ir in mod.irreps_out for _ in range(mul)]))
    z64 = r64 + p64[1][per_col] * val
    outs64 = [z64] + ([norm64(z64, p64[2], mod.irreps_out, 1e-5)] if pre else [])
    cot = [gz, gh][:len(outs64)]
    refs = torch.autograd.grad(outs64, [r64, y64] + p64, [c.double() for c in cot])
    mod = mod.cuda()
    params = [mod.weight_post, mod.scale] + ([mod.weight_pre] if pre else [])
    rd, yd = r.cuda().requires_grad_(), y.cuda().requires_grad_()
    outs = mod(rd, yd)
    outs = outs if pre else (outs,)
    got = torch.autograd.grad(outs, [rd, yd] + params, [c.cuda() for c in cot])
    again = torch.autograd.grad(mod(rd, yd), [rd, yd] + params, [c.cuda() for c in cot])
    for a, b in zip(got, again):
        assert torch.equal(a, b)                                   # fixed order
    close(outs[0], z64.detach(), dtype)
    if pre:
        # h = z * rstd(z) * w: where z cancels, its rounding is relative to the terms of z
        amp = (outs64[1].abs().amax(1, keepdim=True) / z64.abs().amax(1, keepdim=True).clamp(min=1e-3)).detach()
        close(outs[1], outs64[1].detach(), dtype, size=outs64[1].detach().abs().amax(1, keepdim=True) + amp * z64.detach().abs().amax(1, keepdim=True))
    # both gradients pass the chain twice, through sums of up to din terms of either sign: relative to the largest of the
    # batch times the largest rstd of a row (a gradient is multiplied by it)
    amp_z = (1 / z64.detach().pow(2).mean(1, keepdim=True).sqrt().clamp(min=1e-2)).clamp(min=1.0)
    close(got[0], refs[0], dtype, terms=256, size=amp_z * (gz.abs().max() + gh.abs().max()).double())
    amp_y = (1 / y64.detach().pow(2).mean(1, keepdim=True).sqrt().clamp(min=1e-2)).clamp(min=1.0)
    close(got[1], refs[1], dtype, terms=256, size=amp_z * amp_y * (gz.abs().max() + gh.abs().max()).double() * 10)
    for a, b in zip(got[2:], refs[2:]):
        # terms: at most the largest cotangent times the largest normalised value (below sqrt(columns)), per row and component
        size = rows * 7 * (gz.abs().max() + gh.abs().max()).double() * val.detach().abs().max().clamp(min=1.0) * amp_z.max()
        close(a, b, torch.float32, terms=64 + rows, size=size)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gate", ["4096x0e", "4095x0e", "4093x0e activated", "4096x0e activated"])
def test_widest_rows(gate, dtype):
    """What the constructor takes has to fit both directions."""
    irreps = gate.split()[0]
    act = bnn.Activation(irreps, [torch.nn.functional.silu]) if "activated" in gate else None
    mod = bnn.NormGateResidual(act, irreps=None if act else irreps).cuda()
    gen = torch.Generator().manual_seed(0)
    r, y, gz, gh = (rows_of(3, mod.irreps_out.dim, dtype, gen) for _ in range(4))
    rd, yd = r.cuda().requires_grad_(), y.cuda().requires_grad_()
    z, h = mod(rd, yd)
    grads = torch.autograd.grad((z, h), (rd, yd, mod.scale), (gz.cuda(), gh.cuda()))
    n = norm64(y.double(), torch.ones(mod.scale.numel(), dtype=torch.float64), irreps, 1e-5)
    z64 = r.double() + (n if act is None else gate64(act, n))
    close(z, z64, dtype, terms=64)
    h64 = norm64(z64, torch.ones(mod.scale.numel(), dtype=torch.float64), irreps, 1e-5)
    close(h, h64, dtype, terms=64, size=2 * h64.abs().amax(1, keepdim=True))
    assert all(torch.isfinite(g).all() for g in grads)


def test_gradients_of_one_output_alone_and_of_some_inputs():
    gen = torch.Generator().manual_seed(3)
    gate = gates()["l2"]
    mod = bnn.NormGateResidual(gate).cuda()
    r, y = rows_of(40, 288, torch.float32, gen).cuda().requires_grad_(), rows_of(40, 352, torch.float32, gen).cuda().requires_grad_()
    g = rows_of(40, 288, torch.float32, gen).cuda()
    z, h = mod(r, y)
    zero = torch.zeros_like(g)
    for both, one in ((torch.autograd.grad((z, h), (r, y), (g, zero), retain_graph=True), torch.autograd.grad(z, (r, y), g, retain_graph=True)),
                      (torch.autograd.grad((z, h), (r, y), (zero, g), retain_graph=True), torch.autograd.grad(h, (r, y), g, retain_graph=True))):
        for a, b in zip(both, one):
            assert torch.allclose(a, b, rtol=0, atol=64 * U32 * a.abs().max().item())
    (gs,) = torch.autograd.grad(mod(r.detach(), y.detach())[0], (mod.scale,), g)
    (gs2,) = torch.autograd.grad(mod(r, y)[0], (mod.scale,), g)
    assert torch.equal(gs, gs2)


def test_difference_quotient():
    gen = torch.Generator().manual_seed(5)
    mod = bnn.NormGateResidual(bnn.Gate("4x0e", [torch.tanh], "2x0e", [torch.sigmoid], "2x1o")).cuda()
    r, y = rows_of(3, 10, torch.float32, gen).cuda(), rows_of(3, 12, torch.float32, gen).cuda()
    c1, c2, dr, dy = (rows_of(3, d, torch.float32, gen).cuda() for d in (10, 10, 10, 12))
    def value(t):
        z, h = mod(r + t * dr, y + t * dy)
        return (z.double() * c1).sum() + (h.double() * c2).sum()
    rd, yd = r.clone().requires_grad_(), y.clone().requires_grad_()
    z, h = mod(rd, yd)
    gr, gy = torch.autograd.grad((z, h), (rd, yd), (c1, c2))
    slope = (gr * dr).double().sum() + (gy * dy).double().sum()
    t = 2.0 ** -7
    quotient = (value(t) - value(-t)) / (2 * t)
    # truncation t^2 / 6 of a third derivative of a few hundred, roundings 2^-24 * 100 / t
    assert abs(slope - quotient) < 200 * t * t / 6 + 100 * U32 / t


def test_shapes_strides_and_empty_rows():
    gen = torch.Generator().manual_seed(0)
    mod = bnn.RMSNorm("4x0e+4x1o").cuda()
    wide = rows_of(6, 33, torch.float32, gen).cuda()
    for x in (wide[:, 3:19], wide[::2, :16], wide[:, :16].reshape(2, 3, 16), wide[:1, :16].expand(5, 16), wide.flatten()[1:17].reshape(1, 16)):
        close(mod(x).reshape(-1, 16).detach(), norm64(x.reshape(-1, 16).cpu().double(), torch.ones(8).double(), "4x0e+4x1o", 1e-5), torch.float32)
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    h = mod(x)
    gx, gw = torch.autograd.grad(h, (x, mod.weight), h)
    assert h.shape == gx.shape == (0, 16) and torch.equal(gw, torch.zeros_like(gw))
    assert torch.equal(mod(torch.zeros(2, 16, device="cuda")), torch.zeros(2, 16, device="cuda"))
    plain = bnn.RMSNorm("4x0e+4x1o", affine=False).cuda()
    assert torch.equal(plain(wide[:, :16]), mod(wide[:, :16]))
    post = bnn.NormGateResidual(irreps="4x0e").cuda()
    z, h = post(torch.zeros(0, 4, device="cuda"), torch.zeros(0, 4, device="cuda"))
    assert z.shape == h.shape == (0, 4)


def test_nan_and_infinity_stay_in_their_row():
    mod = bnn.NormGateResidual(gates()["l2"]).cuda()
    gen = torch.Generator().manual_seed(1)
    r, y = rows_of(9, 288, torch.float32, gen).cuda(), rows_of(9, 352, torch.float32, gen).cuda()
    clean = mod(r, y)
    r2, y2 = r.clone(), y.clone()
    r2[4, 7], y2[6, 100] = float("nan"), float("inf")
    for a, b in zip(mod(r2, y2), clean):
        keep = [i for i in range(9) if i not in (4, 6)]
        assert torch.equal(a[keep], b[keep])
        assert torch.isnan(a[4]).any() and not torch.isfinite(a[6]).all()


def test_rotation_commutes():
    irreps = o3.Irreps("8x0e+8x1o+4x2e")
    gen = torch.Generator().manual_seed(2)
    D = irreps.D_from_matrix(o3.rand_matrix()).float().cuda()
    mod = bnn.RMSNorm(irreps).cuda()
    x = rows_of(20, irreps.dim, torch.float32, gen).cuda()
    # two products with D (52 terms) and two norms
    assert (mod(x @ D.T) - mod(x) @ D.T).abs().max() < 4 * 64 * U32 * 10


def test_captured_and_replayed_on_another_stream():
    gen = torch.Generator().manual_seed(4)
    mod = bnn.NormGateResidual(gates()["l2"]).cuda()
    ins = [rows_of(50, d, torch.float32, gen).cuda() for d in (288, 352, 288, 288)]
    def step(r, y, gz, gh):
        r, y = r.detach().requires_grad_(), y.detach().requires_grad_()
        z, h = mod(r, y)
        return (z.detach(), h.detach(), *torch.autograd.grad((z, h), (r, y, mod.scale), (gz, gh)))
    static = [t.clone() for t in ins]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*static)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    new = [rows_of(50, t.shape[1], torch.float32, gen).cuda() for t in ins]
    for s, t in zip(static, new):
        s.copy_(t)
    graph.replay()
    for a, b in zip(outs, step(*new)):
        assert torch.equal(a, b)


def test_refusals():
    x = torch.randn(4, 16, device="cuda")
    with pytest.raises(TypeError):
        bnn.RMSNorm("4x0e+4x1o").cuda()(x.double())
    with pytest.raises(RuntimeError, match="same device"):
        bnn.RMSNorm("4x0e+4x1o")(x)
    with pytest.raises((AssertionError, RuntimeError)):
        bnn.RMSNorm("4x0e+4x1o").cuda()(x[:, :15])
    post = bnn.NormGateResidual(irreps="4x0e+4x1o").cuda()
    with pytest.raises(TypeError):
        post(x, x.half())
    with pytest.raises((AssertionError, RuntimeError)):
        post(x, x[:3])
    with pytest.raises((NotImplementedError, RuntimeError)):
        post(x, x.cpu())
    with pytest.raises(e3nn_b200.E3BError):
        bnn.RMSNorm("9000x0e").cuda()(torch.randn(1, 9000, device="cuda"))       # more columns than a thread block takes
    y = x.clone().requires_grad_()
    for out in (bnn.RMSNorm("4x0e+4x1o").cuda()(y), bnn.RMSNorm("4x0e+4x1o").cuda()(y).pow(2)):      # the cotangent a constant, or a function of the leaf
        (g,) = torch.autograd.grad(out.sum(), y, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()
