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
