"""RMSNorm and NormGateResidual at the sizes and places where a row can go wrong, gradients with a bound on every number."""
import pytest
import torch

from e3nn_b200 import nn as bnn
from e3nn_b200 import o3
from test_gpu_norm import close, norm64, rows_of

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
