"""RMSNorm and NormGateResidual at the sizes and places where a row can go wrong, gradients with a bound on every number."""
import pytest
import torch

from e3nn_b200 import nn as bnn
from e3nn_b200 import o3
from test_gpu_norm import ACT64, U32, close, gate64, gates, norm64, rows_of

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("irreps", ["4100x0e", "8192x0e", "1000x0e+1000x1o+400x2e"])
def test_wide_rows_that_start_anywhere(irreps, dtype):
    """Rows of more than 4,096 columns in a view that no vector of four starts, with such a cotangent."""
    gen = torch.Generator().manual_seed(0)
    mod = bnn.RMSNorm(irreps).cuda()
    dim, rows = o3.Irreps(irreps).dim, 3
    x, g = rows_of(rows, dim, dtype, gen, 3.0), rows_of(rows, dim, dtype, gen)
    def shifted(t):
        wide = torch.empty(rows * dim + 1, dtype=dtype, device="cuda")
        wide[1:] = t.flatten().cuda()
        return wide[1:].view(rows, dim)
    plain, moved = x.cuda().requires_grad_(), shifted(x).requires_grad_()
    assert moved.data_ptr() % (4 * moved.element_size()) != 0
    h = mod(moved)
    want = mod(plain)
    close(h.detach(), norm64(x.double(), torch.ones(o3.Irreps(irreps).num_irreps).double(), irreps, 1e-5), dtype)
    assert torch.equal(h, want)
    for a, b in zip(torch.autograd.grad(h, (moved, mod.weight), shifted(g)), torch.autograd.grad(want, (plain, mod.weight), g.cuda())):
        assert torch.equal(a, b)


@pytest.mark.parametrize("irreps", ["+".join(["1x0e"] * 1001), "+".join(["1x0e", "1x1o"] * 904), "+".join(["4x0e"] * 1808)], ids=["1001 of one", "904 of two", "1808 of four"])
def test_rows_of_many_blocks(irreps):
    """As many as the forward pass takes: the gradient's two sums a block have to fit as well."""
    gen = torch.Generator().manual_seed(0)
    irreps, rows = o3.Irreps(irreps), 700
    mod = bnn.RMSNorm(irreps, eps=0.1).cuda()
    x, g = rows_of(rows, irreps.dim, torch.float32, gen), rows_of(rows, irreps.dim, torch.float32, gen)
    xd = x.cuda().requires_grad_()
    h = mod(xd)
    gx, gw = torch.autograd.grad(h, (xd, mod.weight), g.cuda())
    at, col = torch.tensor([b for b, (mul, ir) in enumerate(irreps) for _ in range(mul * ir.dim)]), torch.tensor([1.0 / (mul * ir.dim) for mul, ir in irreps]).double()
    mean = lambda t: torch.zeros(rows, len(irreps), dtype=torch.float64).index_add_(1, at, t) * col
    rstd = (mean(x.double() ** 2) + 0.1).rsqrt()[:, at]
    n = x.double() * rstd
    close(h.detach(), n, torch.float32)
    close(gx, rstd * (g.double() - n * mean(g.double() * n)[:, at]), torch.float32, size=(rstd * (g.double().abs() + n.abs() * mean((g.double() * n).abs())[:, at])))
    chan = torch.tensor([c for c, d in enumerate([ir.dim for mul, ir in irreps for _ in range(mul)]) for _ in range(d)])
    add = lambda t: torch.zeros(irreps.num_irreps, dtype=torch.float64).index_add_(0, chan, t.sum(0))
    close(gw, add(g.double() * n), torch.float32, terms=64 + rows, size=add((g.double() * n).abs()))


@pytest.mark.parametrize("rows,columns", [(3, 2048), (1200, 256)])       # a row by thread blocks, by warps
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
def test_activations_far_from_zero(act, rows, columns):
    """Columns of ones, so that the activation's argument is the weight: relative error below (6 + 1.2 |x|) 2^-23 above -87, one more rounding for
    the scale and one for the sum with a residual of zero; below that an absolute error of 2^-125 |x|."""
    f = {"silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid}[act]
    gate = bnn.Activation(f"{columns}x0e", [f])
    cst = gate._in_cst.double()
    mod = bnn.NormGateResidual(gate, eps=0.0, pre_norm=False).cuda()
    w = torch.linspace(-130.0, 130.0, columns)
    with torch.no_grad():
        mod.weight_post.copy_(w)
        z = mod(torch.zeros(rows, columns, device="cuda"), torch.ones(rows, columns, device="cuda")).cpu().double()
    ref, x = cst * f(w.double()), w.double().abs()
    bound = torch.where(w > -87, (6 + 1.2 * x + 2) * 2.0 ** -23 * ref.abs(), 2.0 ** -125 * x * cst) + 2.0 ** -149
    assert ((z - ref).abs() <= bound).all()


def parameter_terms(mod, r, y, gz, gh, gate):
    """Gradients of the norm-gate-residual in 64 bits, written out, and per parameter the sum of the magnitudes of what is added."""
    ins, outs = mod.irreps_in, mod.irreps_out
    def channels(irreps):
        return torch.tensor([c for c, d in enumerate([ir.dim for mul, ir in irreps for _ in range(mul)]) for _ in range(d)])
    def blocks(irreps):
        return torch.tensor([b for b, (mul, ir) in enumerate(irreps) for _ in range(mul * ir.dim)])
    ci, co, bi, bo = channels(ins), channels(outs), blocks(ins), blocks(outs)
    def mean(x, b):
        n = torch.bincount(b).double()
        return (torch.zeros(x.shape[0], len(n), dtype=torch.float64).index_add(1, b, x) / n)[:, b]
    wp, sc, wn = mod.weight_post.detach().cpu().double()[ci], mod.scale.detach().cpu().double()[co], mod.weight_pre.detach().cpu().double()[co]
    y, r, gz, gh = (t.double() for t in (y, r, gz, gh))
    n = y * (mean(y * y, bi) + mod.eps).rsqrt()
    pre = (n * wp).requires_grad_()
    val = gate64(gate, pre) if gate is not None else pre * 1.0
    x, val_abs = pre.detach(), pre.detach().abs()
    if gate is not None:
        parts = []
        for (src, gcol, act), cst in zip(gate._out_tbl.tolist(), gate._out_cst.tolist()):
            arg = x[:, src] if gcol < 0 else x[:, gcol]
            parts.append(cst * (ACT64[act](arg).abs() + arg.abs()) * (1.0 if gcol < 0 else x[:, src].abs()))
        val_abs = torch.stack(parts, 1)
    z, z_abs = r + sc * val.detach(), r.abs() + sc.abs() * val_abs
    rz = (mean(z * z, bo) + mod.eps).rsqrt()
    t = gh * wn
    gz2 = gz + rz * (t - z * rz * rz * mean(t * z, bo))
    gz_abs = gz.abs() + rz * (t.abs() + z_abs * rz * rz * mean(t.abs() * z_abs, bo))
    (g_pre,) = torch.autograd.grad(val, pre, gz2 * sc, retain_graph=True)
    # the same chain with magnitudes: a gate's cotangent adds the products of its components; a slope is at most `steep` and what it is the
    # difference of; an argument that is off by a part of itself moves function and slope (whose own slopes are at most one) by as much of it
    steep = {0: lambda x: torch.sigmoid(x) * (1 + x.abs()), 1: torch.ones_like, 2: torch.ones_like, 3: torch.ones_like, 4: torch.sigmoid, 5: torch.ones_like}
    def jacobian_abs(g):
        if gate is None:
            return g
        out = torch.zeros_like(pre)
        rows = gate._out_tbl.tolist()
        for j, (src, gcol, act) in enumerate(rows):
            cst = float(gate._out_cst[j])
            arg = x[:, src] if gcol < 0 else x[:, gcol]
            f, d = ACT64[act](arg).abs() + arg.abs(), steep[act](arg) + arg.abs()
            if gcol < 0:
                out[:, src] += cst * d * g[:, j]
            else:
                out[:, src] += cst * f * g[:, j]
                out[:, gcol] += cst * d * x[:, src].abs() * g[:, j]
        return out.detach()
    pre_abs = jacobian_abs(gz_abs * sc.abs())
    add = lambda x, c, num: torch.zeros(num, dtype=torch.float64).index_add(0, c, x.sum(0))
    num_in, num_out = ins.num_irreps, outs.num_irreps
    values = add(g_pre * n, ci, num_in), add(gz2 * val.detach(), co, num_out), add(gh * z * rz, co, num_out)
    sizes = add(pre_abs * n.abs(), ci, num_in), add(gz_abs * val_abs, co, num_out), add(gh.abs() * z_abs * rz, co, num_out)
    s = (mean(y * y, bi) + mod.eps).rsqrt()
    gx = s * (g_pre * wp - n * mean(g_pre * wp * n, bi))
    gx_abs = s * (pre_abs * wp.abs() + n.abs() * mean(pre_abs * wp.abs() * n.abs(), bi))
    return (gz2, gx, *values), (gz_abs, gx_abs, *sizes)


# Of what is added, each part is off by: a root mean square (a tree of sums of at most 32 + 5 + 16 additions, its root) 60 roundings, used twice for z,
# twice for y; the two means of products 60 each; activations 30 (an exponential with an argument that the norm keeps below the root of the
# columns, a division); the products on the way 40.  Where a cotangent is a difference its parts count with their magnitudes, and z with those
# of the residual and of what is added to it.
ROUNDINGS = 450


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["l2", "odd", "odd gates", "no scalars", "activation", "wide", "wide odd", "none", "l3"])
@pytest.mark.parametrize("rows", [3, 1301])
def test_gradients_with_a_bound_on_every_number(name, rows, dtype):
    if name.startswith("wide") and rows > 3:
        rows = 400                                         # several rows a thread block all the same
    gen = torch.Generator().manual_seed(len(name) + rows)
    gate = gates()[name]
    mod = bnn.NormGateResidual(gate, irreps="6x0e+3x1o" if gate is None else None, eps=1e-3, scale_init=0.7).cuda()
    din, dout = mod.irreps_in.dim, mod.irreps_out.dim
    r, y, gz, gh = (rows_of(rows, d, dtype, gen) for d in (dout, din, dout, dout))
    params = [mod.weight_post, mod.scale, mod.weight_pre]
    with torch.no_grad():
        for p in params:
            p.copy_(1 + 0.3 * torch.randn(p.shape, generator=gen))
    rd, yd = r.cuda().requires_grad_(), y.cuda().requires_grad_()
    got = torch.autograd.grad(mod(rd, yd), [rd, yd] + params, (gz.cuda(), gh.cuda()))
    refs, sizes = parameter_terms(mod, r, y, gz, gh, gate)
    # a thread block adds its rows one by one, at most 148 blocks' sums by 32 threads, a channel up to 7 components
    adds = rows // 148 + 2 + 148 * 4 // 32 + 32 + 7
    for a, ref, size, what in zip(got, refs, sizes, ("residual", "y", "weight_post", "scale", "weight_pre")):
        to = dtype if what in ("residual", "y") else torch.float32
        assert a.dtype == to and a.shape == ref.shape
        bound = torch.finfo(to).eps / 2 * ref.abs() + (ROUNDINGS + (0 if what in ("residual", "y") else adds)) * U32 * size + torch.finfo(to).tiny
        excess = ((a.cpu().double() - ref).abs() / bound).max().item()
        assert excess <= 1.0, f"{what}: {excess:.2f} x the bound"
        assert bound.mean() < 0.05 * ref.abs().mean(), what


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("irreps", ["4096x0e", "4095x0e", "4093x0e activated", "4096x0e activated"])
def test_gradients_of_the_widest_rows(irreps, dtype):
    act = bnn.Activation(irreps.split()[0], [torch.nn.functional.silu]) if "activated" in irreps else None
    mod = bnn.NormGateResidual(act, irreps=None if act else irreps, eps=1e-3).cuda()
    gen = torch.Generator().manual_seed(0)
    r, y, gz, gh = (rows_of(3, mod.irreps_out.dim, dtype, gen) for _ in range(4))
    rd, yd = r.cuda().requires_grad_(), y.cuda().requires_grad_()
    got = torch.autograd.grad(mod(rd, yd), (rd, yd, mod.weight_post, mod.scale, mod.weight_pre), (gz.cuda(), gh.cuda()))
    refs, sizes = parameter_terms(mod, r, y, gz, gh, act)
    for a, ref, size, to in zip(got, refs, sizes, (dtype, dtype) + (torch.float32,) * 3):
        bound = torch.finfo(to).eps / 2 * ref.abs() + (ROUNDINGS + 3) * U32 * size + torch.finfo(to).tiny
        assert ((a.cpu().double() - ref).abs() <= bound).all() and bound.mean() < 0.05 * ref.abs().mean()
