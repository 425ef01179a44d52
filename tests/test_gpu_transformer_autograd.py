"""Calls of the transformer modules that someone else follows although no backward pass is asked for: forward-mode levels,
transforms of `torch.func` and the tracer of `torch.jit`.  A module may refuse them; it may not answer without their knowledge."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import e3nn_b200
from e3nn_b200 import nn as bnn

pytestmark = pytest.mark.gpu


NAMES = ["rms", "norm", "norm alone", "attention"]


def modules():
    """{name: (module, inputs, another set of inputs of another size)}"""
    gen = torch.Generator().manual_seed(0)
    def rows(n, d):
        return torch.randn(n, d, generator=gen).cuda()
    def edges(N, E, S):
        dst = torch.randint(N, (E,), generator=gen).sort().values
        rowptr = torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(dst, minlength=N).cumsum(0)])
        return rowptr.cuda(), torch.randint(S, (E,), generator=gen).cuda()
    def attention(N, E, S):
        return (rows(N, 16), rows(S, 16), rows(S, 16), *edges(N, E, S))
    gate = bnn.Gate("4x0e", [torch.tanh], "4x0e", [torch.sigmoid], "4x1o")
    return {
        "rms": (bnn.RMSNorm("4x0e+4x1o"), (rows(5, 16),), (rows(9, 16),)),
        "norm": (bnn.NormGateResidual(gate), (rows(5, 16), rows(5, 20)), (rows(9, 16), rows(9, 20))),
        "norm alone": (bnn.NormGateResidual(gate, pre_norm=False), (rows(5, 16), rows(5, 20)), (rows(9, 16), rows(9, 20))),
        "attention": (bnn.NeighborAttention("4x0e+4x1o", "4x0e+4x1o", 2), attention(6, 20, 7), attention(11, 33, 5)),
    }


def flat(out):
    return out if isinstance(out, tuple) else (out,)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("recorded", [False, True])
def test_a_tangent_is_not_lost(name, recorded):
    mod, inputs, _ = modules()[name]
    mod = mod.cuda()
    for p in mod.parameters():
        p.requires_grad_(recorded)
    with torch.set_grad_enabled(recorded), fw.dual_level():
        x = fw.make_dual(inputs[0], torch.ones_like(inputs[0]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            mod(x, *inputs[1:])
        mod(*inputs)                              # nothing to lose
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda x: mod(x, *inputs[1:]), (inputs[0],), (torch.ones_like(inputs[0]),))


def test_a_tangent_of_a_table_is_not_lost():
    mod = bnn.RelativeBias(4, 2, 5.0).cuda()
    buckets = torch.tensor([0, 3, 1], dtype=torch.int32, device="cuda")
    weight = mod.weight.detach()
    del mod.weight
    with torch.no_grad(), fw.dual_level():
        mod.register_parameter("weight", None)
        mod._parameters["weight"] = fw.make_dual(weight, torch.ones_like(weight))
        with pytest.raises((RuntimeError, NotImplementedError)):
            mod(buckets)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("recorded", [False, True])
def test_a_traced_module_computes(name, recorded):
    mod, inputs, others = modules()[name]
    mod = mod.cuda()
    for p in mod.parameters():
        p.requires_grad_(recorded)
    with torch.set_grad_enabled(recorded):
        traced = torch.jit.trace(mod, inputs)
        wide = tuple(torch.randn(x.shape[0], 2 * x.shape[1], device="cuda")[:, ::2].copy_(x) if x.is_floating_point() else x for x in others)
        for args in (inputs, others, wide):       # (the last one: columns apart)
            junk = torch.full((4096,), float("nan"), device="cuda")
            del junk                              # what an output that is never written would show
            for a, b in zip(flat(traced(*args)), flat(mod(*args))):
                assert torch.equal(a, b)


def test_traced_buckets_and_bias():
    class Both(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.bias = bnn.RelativeBias(8, 2, 5.0)
        def forward(self, pos, src, dst):
            buckets = self.bias.buckets(pos, src, dst)
            return buckets, self.bias(buckets)
    mod = Both().cuda()
    gen = torch.Generator().manual_seed(1)
    def graph(N, E):
        return (5 * torch.rand(N, 3, generator=gen).cuda(), torch.randint(N, (E,), generator=gen).cuda(), torch.randint(N, (E,), generator=gen).cuda())
    with torch.no_grad():
        traced = torch.jit.trace(mod, graph(10, 30))
        args = graph(20, 77)
        for a, b in zip(traced(*args), mod(*args)):
            assert torch.equal(a, b)
    e3nn_b200.check_status()


@pytest.mark.parametrize("changed", ["rowptr", "src", "perm", "buckets", "transpose", "q", "bias"])
def test_what_the_backward_pass_reads_again_may_not_change(changed):
    gen = torch.Generator().manual_seed(2)
    N, E, S = 4, 12, 5
    mod = bnn.NeighborAttention("4x0e+4x1o", "4x0e+4x1o", 2).cuda()
    q, k, v = (torch.randn(n, 16, generator=gen).cuda().requires_grad_() for n in (N, S, S))
    bias = torch.randn(6, 2, generator=gen).cuda().requires_grad_()
    src, perm, buckets = torch.randint(S, (E,), generator=gen).cuda(), torch.randperm(E, generator=gen).cuda(), torch.randint(6, (E,), generator=gen).int().cuda()
    rowptr = torch.tensor([0, 3, 3, 8, E]).cuda()
    transpose = e3nn_b200.csr_from_dst(src, S)
    out = mod(q, k, v, rowptr, src, perm=perm, bias=bias, buckets=buckets, transpose=transpose)
    out.sum().backward(retain_graph=True)
    with torch.no_grad():
        {"rowptr": rowptr, "src": src, "perm": perm, "buckets": buckets, "transpose": transpose[0], "q": q, "bias": bias}[changed].zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_gradients_come_in_the_types_of_the_inputs():
    gen = torch.Generator().manual_seed(3)
    mod = bnn.NeighborAttention("4x0e+4x1o", "4x0e+4x1o", 2).cuda()
    q, k, v = (torch.randn(3, 16, generator=gen).cuda().requires_grad_() for _ in range(3))
    bias, weight = torch.randn(3, 2, generator=gen).cuda().bfloat16().requires_grad_(), torch.rand(3, generator=gen).cuda().half().requires_grad_()
    rowptr = torch.tensor([0, 0, 1, 3]).cuda()
    grads = torch.autograd.grad(mod(q, k, v, rowptr, bias=bias, edge_weight=weight).pow(2).sum(), (bias, weight))
    exact = [t.detach().float().requires_grad_() for t in (bias, weight)]
    full = torch.autograd.grad(mod(q, k, v, rowptr, bias=exact[0], edge_weight=exact[1]).pow(2).sum(), exact)
    for a, b, t in zip(grads, full, (bias, weight)):
        assert a.dtype == t.dtype and torch.equal(a, b.to(t.dtype))


def test_edges_by_source_are_not_built_in_a_capture():
    mod, (q, k, v, rowptr, src), _ = modules()["attention"]
    mod = mod.cuda()
    transpose = e3nn_b200.csr_from_dst(src, k.shape[0])
    k = k.requires_grad_()
    def step(**kw):
        return torch.autograd.grad(mod(q, k, v, rowptr, src, **kw).sum(), k)[0]
    want = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(transpose=transpose)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="transpose=csr_from_dst"):
            step()
        got = step(transpose=transpose)           # the capture goes on
    graph.replay()
    assert torch.equal(got, want)


def test_every_parameter_of_a_block_against_differences():
    """Norm, bias, attention with a cutoff, norm-gate-residual and a convolution block: the slope along a direction in each parameter
    and input against a difference quotient."""
    import math

    from e3nn_b200 import o3

    torch.manual_seed(0)
    gen = torch.Generator().manual_seed(0)
    irreps, heads, N = o3.Irreps("8x0e+8x1o+4x2e"), 4, 40
    pos = (12.0 * torch.rand(N, 3, generator=gen)).cuda()
    src, dst, shift, rowptr = bnn.neighbor_list_pbc(pos, 15.0, 5.0)
    pre, bias = bnn.RMSNorm(irreps).cuda(), bnn.RelativeBias(8, heads, 5.0, r_linear=2.5).cuda()
    block = bnn.AttentionBlock(irreps, heads, linear_math_mode="fp32", scale_init=0.5).cuda()
    conv = bnn.InteractionBlock(irreps, lmax=1, num_basis=4, hidden=32, r_max=5.0, num_neighbors=5.0, linear_math_mode="fp32", radial_math_mode="fp32").cuda()
    post = bnn.NormGateResidual(irreps=irreps).cuda()
    with torch.no_grad():
        bias.weight.normal_(0, 0.5)
    buckets = bias.buckets(pos, src, dst, shift)
    cutoff = 0.5 * (torch.cos(math.pi * (pos[src] - pos[dst] + shift).norm(dim=1) / 5.0) + 1)
    x, c1, c2 = (torch.randn(N, irreps.dim, generator=gen).cuda() for _ in range(3))
    transpose = e3nn_b200.csr_from_dst(src, N)
    def loss(x):
        z, h = block(x, pre(x), rowptr, src, bias=bias.weight, buckets=buckets, edge_weight=cutoff, transpose=transpose)
        z, h = post(z, conv(pos, h, src, dst, rowptr, shift))
        return (z.double() * c1).sum() + (h.double() * c2).sum()
    leaves = {"x": x, **{f"{i}.{n}": p for i, m in enumerate((pre, bias, block, conv, post)) for n, p in m.named_parameters()}}
    x.requires_grad_()
    grads = dict(zip(leaves, torch.autograd.grad(loss(x), list(leaves.values()))))
    for name, leaf in leaves.items():
        direction = torch.randn(leaf.shape, generator=gen).cuda()
        direction *= leaf.detach().pow(2).mean().sqrt() / direction.pow(2).mean().sqrt()
        slope = (grads[name].double() * direction).sum().item()
        size = grads[name].double().norm().item() * direction.double().norm().item() / leaf.numel() ** 0.5      # of a slope along a random direction
        def at(s):
            with torch.no_grad():
                start = leaf.clone()
                leaf.add_(direction, alpha=s)
                value = loss(x).item()
                leaf.copy_(start)
            return value
        # central differences at three steps: truncation falls with the square, the rounding of z and h (2^-24 of a few units, some thousand numbers of
        # either sign) grows with the inverse; the two larger ones give the truncation (Richardson)
        d = [(at(s) - at(-s)) / (2 * s) for s in (2.0 ** -5, 2.0 ** -6)]
        best, doubt = (4 * d[1] - d[0]) / 3, abs(d[1] - d[0])
        noise = 2.0 ** -24 * 4 * (x.numel() * 2) ** 0.5 * 32 / 2.0 ** -6
        assert abs(best - slope) <= doubt + noise, (name, best, slope, doubt, noise)
        assert doubt + noise < 0.5 * max(size, abs(slope)), (name, slope, doubt, noise, size)


@pytest.mark.parametrize("name", NAMES)
def test_a_pickled_module_computes(name):
    import copy
    import pickle

    mod, inputs, _ = modules()[name]
    mod = mod.cuda()
    want = flat(mod(*inputs))
    for other in (pickle.loads(pickle.dumps(mod)), copy.deepcopy(mod)):
        assert all(torch.equal(a, b) for a, b in zip(flat(other(*inputs)), want))


@pytest.mark.parametrize("how", ["parametrized", "pruned", "plain attributes"])
def test_parameters_that_something_else_provides(how):
    """Parametrisations, pruning and wrappers that put views of one flat tensor in the place of parameters take them out of the module's table."""
    import copy

    from torch.nn.utils import parametrize, prune

    class Double(torch.nn.Module):
        def forward(self, w):
            return 2 * w

    buckets = torch.tensor([0, 3, 1], dtype=torch.int32, device="cuda")
    cases = [(*modules()[n][:2], names) for n, names in (("rms", ["weight"]), ("norm", ["weight_post", "scale", "weight_pre"]))]
    cases.append((bnn.RelativeBias(4, 2, 5.0), (buckets,), ["weight"]))
    for mod, inputs, names in cases:
        mod = mod.cuda()
        changed = copy.deepcopy(mod)
        for name in names:
            value = getattr(mod, name)
            if how == "parametrized":
                parametrize.register_parametrization(changed, name, Double())
            elif how == "pruned":
                prune.custom_from_mask(changed, name, (torch.arange(value.numel(), device="cuda") % 2).reshape(value.shape))
            else:
                delattr(changed, name)
                setattr(changed, name, (3 * value.detach()).requires_grad_())
            with torch.no_grad():
                value.mul_({"parametrized": 2, "plain attributes": 3}.get(how, 1))
                if how == "pruned":
                    value.mul_((torch.arange(value.numel(), device="cuda") % 2).reshape(value.shape))
        got, want = flat(changed(*inputs)), flat(mod(*inputs))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(a.requires_grad for a in got)
