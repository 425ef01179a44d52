"""RelativeBias: buckets are whole numbers and have to be equal; the bias is a copy; the gradient of the table is a sum of n terms in fp32
(one rounding each) that is rounded once to the table's type."""
import pytest
import torch

import e3nn_b200
from e3nn_b200 import nn as bnn

pytestmark = pytest.mark.gpu


def buckets64(mod, vec):
    r2 = (vec.double() ** 2).sum(1)
    out = torch.zeros(vec.shape[0], dtype=torch.int32)
    for t in mod.lower_ends[1:]:
        out += (r2 >= t * t).int()
    return out


@pytest.mark.parametrize("num,r_linear", [(1, 5.0), (2, 5.0), (2, 1.0), (7, 2.0), (32, 5.0), (32, 1.25), (1024, 3.0)])
@pytest.mark.parametrize("edges", [1, 31, 5000])
def test_buckets(num, r_linear, edges):
    gen = torch.Generator().manual_seed(num + edges)
    mod = bnn.RelativeBias(num, 4, 5.0, r_linear=r_linear).cuda()
    pos = 10 * torch.rand(20, 3, generator=gen)
    src, dst = torch.randint(20, (edges,), generator=gen), torch.randint(20, (edges,), generator=gen)
    shift = 3 * torch.randn(edges, 3, generator=gen)
    got = mod.buckets(pos.cuda(), src.cuda(), dst.cuda(), shift.cuda())
    assert got.dtype == torch.int32
    assert torch.equal(got.cpu(), buckets64(mod, pos.double()[src] - pos.double()[dst] + shift.double()))
    assert torch.equal(mod.buckets(pos.cuda(), src.cuda(), dst.cuda()).cpu(), buckets64(mod, pos.double()[src] - pos.double()[dst]))


def test_distances_on_and_next_to_a_border():
    mod = bnn.RelativeBias(8, 1, 8.0).cuda()              # borders 1, 2, .. 7
    up, down = torch.nextafter(torch.tensor(3.0), torch.tensor(9.0)), torch.nextafter(torch.tensor(3.0), torch.tensor(0.0))
    x = torch.stack([torch.tensor(v) for v in (0.0, 1.0, 3.0, float(up), float(down), 7.0, 100.0)])
    pos = torch.zeros(8, 3)
    pos[1:, 0] = x
    pos[7, 0] = -100.0
    src, dst = torch.arange(1, 8), torch.zeros(7, dtype=torch.int64)
    got = mod.buckets(pos.cuda(), src.cuda(), dst.cuda()).cpu().tolist()
    assert got == [0, 1, 3, 3, 2, 7, 7]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("num,heads", [(1, 1), (5, 3), (32, 8), (64, 16), (130, 5), (1024, 33), (1000, 70)])
@pytest.mark.parametrize("edges", [1, 63, 20001])
def test_bias_and_table_gradient(num, heads, edges, dtype):
    gen = torch.Generator().manual_seed(num * heads + edges)
    mod = bnn.RelativeBias(num, heads, 5.0).cuda().to(dtype)
    b = torch.randint(num, (edges,), generator=gen, dtype=torch.int32)
    if num > 2:
        b[b == 1] = 2                                       # a bucket without edges
    g = torch.randn(edges, heads, generator=gen).to(dtype)
    out = mod(b.cuda())
    assert out.dtype == dtype and torch.equal(out, mod.weight[b.cuda().long()])
    (got,) = torch.autograd.grad(out, (mod.weight,), g.cuda(), retain_graph=True)
    assert got.dtype == dtype and torch.equal(got, torch.autograd.grad(out, (mod.weight,), g.cuda())[0])
    ref = torch.zeros(num, heads, dtype=torch.float64).index_add_(0, b.long(), g.double())
    mag = torch.zeros(num, heads, dtype=torch.float64).index_add_(0, b.long(), g.double().abs())
    n = torch.bincount(b.long(), minlength=num)[:, None]
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    bound = half * ref.abs() + n * 2.0 ** -24 * mag + torch.finfo(dtype).tiny
    assert ((got.cpu().double() - ref).abs() <= bound).all()
    if num > 2:
        assert torch.equal(got[1], torch.zeros_like(got[1]))


def test_no_edges_and_bad_indices():
    mod = bnn.RelativeBias(4, 2, 5.0).cuda()
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    out = mod(none)
    assert out.shape == (0, 2) and torch.equal(torch.autograd.grad(out, (mod.weight,), out)[0], torch.zeros_like(mod.weight))
    pos = torch.rand(3, 3, device="cuda")
    idx = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert mod.buckets(pos, idx, idx).shape == (0,)
    e3nn_b200.check_status()
    bad = mod(torch.tensor([0, 4, -1, 3], dtype=torch.int32, device="cuda"))
    with pytest.raises(IndexError):
        e3nn_b200.check_status()
    assert torch.equal(bad[1:3], torch.zeros(2, 2, device="cuda")) and torch.equal(bad[3], mod.weight[3])
    got = mod.buckets(pos, torch.tensor([0, 3], device="cuda"), torch.tensor([1, 0], device="cuda"))
    with pytest.raises(IndexError):
        e3nn_b200.check_status()
    assert got[1] == 0


def test_half_precision_module_keeps_its_borders():
    pos = 4 * torch.rand(200, 3, device="cuda")
    src, dst = torch.randint(200, (3000,), device="cuda"), torch.randint(200, (3000,), device="cuda")
    a = bnn.RelativeBias(50, 2, 6.0, r_linear=2.0).cuda()
    b = bnn.RelativeBias(50, 2, 6.0, r_linear=2.0).cuda().half()
    assert torch.equal(a.buckets(pos, src, dst), b.buckets(pos, src, dst))


def test_refusals():
    mod = bnn.RelativeBias(4, 2, 5.0).cuda()
    pos, idx = torch.rand(3, 3, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(TypeError):
        mod.buckets(pos.double(), idx, idx)
    with pytest.raises(TypeError):
        mod.buckets(pos, idx.int(), idx)
    with pytest.raises((AssertionError, RuntimeError)):
        mod.buckets(pos, idx, idx[:1])
    with pytest.raises((AssertionError, RuntimeError)):
        mod.buckets(pos, idx, idx, torch.zeros(1, 3, device="cuda"))
    with pytest.raises((RuntimeError, NotImplementedError)):
        mod.buckets(pos, idx.cpu(), idx)
    with pytest.raises(TypeError):
        mod(idx)
    with pytest.raises(RuntimeError, match="same device"):
        bnn.RelativeBias(4, 2, 5.0)(idx.int())
