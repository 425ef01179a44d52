"""NeighborAttention on layouts of every kind of kernel, against the formula in 64 bits with bounds on every number (attention_formula)."""
import math

import pytest
import torch

import e3nn_b200
from attention_formula import compare, formula
from e3nn_b200 import nn as bnn
from e3nn_b200 import o3

pytestmark = pytest.mark.gpu

# layout, heads -> vector widths in fp32 and in 16 bits; 16-byte vectors (4, 8) travel in bulk copies, the others are loaded one by one
LAYOUTS = {"bulk": ("16x0e+16x1o", 2, 4, 8), "bulk in fp32": ("8x0e+8x1o+8x2e", 2, 4, 4), "loads": ("6x0e+3x1o", 3, 1, 1)}
DEGREES = {"ragged": [0, 3, 1, 0, 0, 37, 2, 5, 33, 0], "hub": [2, 1, 600, 0, 3] + [4] * 40, "one edge": [1] * 7}
NAMES = ("q", "k", "v", "bias", "weight")


def make(irreps, heads, degrees, dtype, per_edge, bias=None, weight=False, perm=False, sources=23, front=0, behind=0, seed=0):
    """Edges of the rows, and `front` and `behind` edges that belong to no row."""
    gen = torch.Generator().manual_seed(seed + heads + len(degrees))
    N, E, D = len(degrees), front + sum(degrees) + behind, o3.Irreps(irreps).dim
    S = E if per_edge else sources
    t = {"rowptr": front + torch.tensor([0] + degrees).cumsum(0), "src": None if per_edge else torch.randint(S, (E,), generator=gen),
         "perm": torch.randperm(E, generator=gen) if perm else None, "buckets": None, "bias": None, "weight": None}
    for name, rows in (("q", N), ("k", S), ("v", S), ("g", N)):
        t[name] = torch.randn(rows, D, generator=gen).to(dtype)
    if bias == "table":
        t["buckets"], t["bias"] = torch.randint(9, (E,), generator=gen, dtype=torch.int32), torch.randn(9, heads, generator=gen)
    elif bias == "edges":
        t["bias"] = torch.randn(E, heads, generator=gen)
        t["bias"][torch.rand(E, heads, generator=gen) < 0.2] = -math.inf
    if weight:
        t["weight"] = 0.05 + 0.95 * torch.rand(E, generator=gen)
        t["weight"][torch.rand(E, generator=gen) < 0.2] = 0.0
    return {n: None if x is None else x.cuda() for n, x in t.items()}


def module(layout, dtype, t):
    irreps, heads, wide, narrow = LAYOUTS[layout]
    mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
    call = mod._checked(*(t[n] for n in ("q", "k", "v", "bias", "weight", "rowptr", "src", "perm", "buckets")), None, None)
    assert call.vec == (wide if dtype == torch.float32 else narrow)
    return mod


def run(mod, t, transposed=True):
    leaves = {n: t[n].detach().requires_grad_() for n in NAMES if t[n] is not None}
    x = {**t, **leaves}
    transpose = e3nn_b200.csr_from_dst(t["src"], t["k"].shape[0]) if t["src"] is not None and transposed else None
    out = mod(x["q"], x["k"], x["v"], t["rowptr"], t["src"], perm=t["perm"], bias=x["bias"], buckets=t["buckets"], edge_weight=x["weight"], transpose=transpose)
    grads = torch.autograd.grad(out, list(leaves.values()), t["g"])
    return {"out": out.detach(), **dict(zip(leaves, grads))}


def check(layout, t, dtype, sharp=0.25):
    mod = module(layout, dtype, t)
    got = run(mod, t)
    compare(got, formula(*LAYOUTS[layout][:1], *LAYOUTS[layout][:2], t, dtype), sharp)
    e3nn_b200.check_status()
    return mod, got


TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("per_edge", [False, True])
@pytest.mark.parametrize("perm", [False, True])
def test_rows_in_a_window_of_the_edges(layout, per_edge, perm, dtype):
    """A row pointer that starts above zero: slots before it belong to no row, whatever they hold."""
    for front, behind in ((1, 0), (300, 0), (77, 250)):
        t = make(*LAYOUTS[layout][:2], DEGREES["ragged"], dtype, per_edge, "table", True, perm, front=front, behind=behind)
        _, got = check(layout, t, dtype)
        if not per_edge or perm:
            continue
        outside = torch.ones(t["k"].shape[0], dtype=torch.bool, device="cuda")
        outside[front:front + sum(DEGREES["ragged"])] = False
        x = {n: None if y is None else y.clone() for n, y in t.items()}
        for n in ("k", "v", "weight"):
            x[n][outside] = float("nan")
        again = run(module(layout, dtype, x), x)
        assert all(torch.equal(again[n], got[n]) for n in got)
        assert all(not got[n][outside].any() for n in ("k", "v", "weight"))


@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_nodes_of_a_graph_alone(layout):
    """rowptr[a:b+1] gives the nodes a .. b-1 as the whole graph does."""
    t = make(*LAYOUTS[layout][:2], DEGREES["hub"], torch.float32, False, "table", True)
    whole = module(layout, torch.float32, t)(t["q"], t["k"], t["v"], t["rowptr"], t["src"], bias=t["bias"], buckets=t["buckets"], edge_weight=t["weight"])
    for a, b in ((1, 4), (3, 20), (44, 45), (4, 4)):
        x = {**t, "q": t["q"][a:b], "g": t["g"][a:b], "rowptr": t["rowptr"][a:b + 1]}
        _, got = check(layout, x, torch.float32, None if a == b else 0.25)
        want = formula(*LAYOUTS[layout][:1], *LAYOUTS[layout][:2], t, torch.float32)["out"]
        assert ((got["out"].double() - whole[a:b].double()).abs() <= 2 * want[1][a:b]).all()


def fill_free_memory():
    """NaN in what the allocator hands out next: an element that no kernel writes shows."""
    junk = [torch.full((n,), float("nan"), device="cuda") for n in [64, 256, 1024, 4096, 16384, 65536] * 40]
    del junk


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("per_edge", [False, True])
def test_edges_that_a_permutation_leaves_out(layout, per_edge, dtype):
    """Bad entries, and a padded permutation whose last slots name any edge: an edge of no row has zeros for gradients, the others are
    what they are without it."""
    degrees = DEGREES["ragged"]
    E = sum(degrees)
    t = make(*LAYOUTS[layout][:2], degrees, dtype, per_edge, "edges", True, True, behind=40)
    t["bias"].clamp_(min=-2.0)
    t["weight"].fill_(1.0)
    mod = module(layout, dtype, t)
    zeros = {**t, "perm": t["perm"].clone()}
    zeros["perm"][E:] = t["perm"][0]                       # padding that names an edge of the rows
    fill_free_memory()
    got = run(mod, zeros)
    compare(got, formula(*LAYOUTS[layout][:1], *LAYOUTS[layout][:2], zeros, dtype))
    want = run(mod, t)
    assert all(torch.equal(got[n], want[n]) for n in got)
    e3nn_b200.check_status()

    bad = torch.tensor([4, 30, 31, E - 1], device="cuda")
    without = {**t, "weight": t["weight"].clone()}
    without["weight"][t["perm"][bad]] = 0.0
    want = run(mod, without)
    out_of_range = {**t, "perm": t["perm"].clone()}
    out_of_range["perm"][bad] = torch.tensor([-1, E + 40, 2 ** 40, -2 ** 40], device="cuda")
    for _ in range(3):
        fill_free_memory()
        got = run(mod, out_of_range)
        with pytest.raises(IndexError):
            e3nn_b200.check_status()
        for n in got:
            assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("per_edge", [False, True])
def test_an_edge_named_twice_is_reported_by_the_backward_pass(layout, per_edge):
    t = make(*LAYOUTS[layout][:2], DEGREES["hub"], torch.float32, per_edge, "table", False, True)
    mod = module(layout, torch.float32, t)
    run(mod, t)
    e3nn_b200.check_status()
    t["perm"][3] = t["perm"][650]
    run(mod, t)
    with pytest.raises(IndexError, match="twice"):
        e3nn_b200.check_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("per_edge", [False, True])
@pytest.mark.parametrize("mask", ["weight", "bias", "share"])
def test_what_a_masked_edge_may_lie_next_to(layout, per_edge, mask, dtype):
    """Row 5 holds infinities or NaN in q and in its cotangent, and masked edges: these, and sources that only they lead to, have zeros
    for gradients.  Masked: by weight, by bias, or by a bias so low that the share is zero in fp32."""
    degrees = DEGREES["ragged"]
    t = make(*LAYOUTS[layout][:2], degrees, dtype, per_edge, "edges" if mask != "weight" else None, mask == "weight", sources=60)
    row = torch.arange(int(t["rowptr"][5]), int(t["rowptr"][6]), device="cuda")
    masked = row[::2]
    if t["src"] is not None:                               # sources of their own
        t["src"] %= 30
        t["src"][masked] = 30 + torch.arange(len(masked), device="cuda")
    if mask == "weight":
        t["weight"][row] = 0.5
        t["weight"][masked] = 0.0
    else:
        t["bias"].clamp_(min=-2.0)
        t["bias"][masked] = -math.inf if mask == "bias" else -1000.0
    mod = module(layout, dtype, t)
    clean = run(mod, t)
    reached = masked if per_edge else t["src"][masked]
    for value in (float("inf"), float("nan")):
        for name in ("g",) if mask == "share" else ("g", "q"):      # (of a NaN in q nothing is masked by a low bias)
            x = {**t, name: t[name].clone()}
            x[name][5] = value
            got = run(mod, x)
            for n in ("k", "v"):
                assert not got[n][reached].any(), (name, n)
            if mask != "weight":
                assert not got["bias"][masked].any()
            else:
                assert not got["weight"][masked].any()
            others = [n for n in range(len(degrees)) if n != 5]
            assert torch.equal(got["out"][others], clean["out"][others]) and torch.equal(got["q"][others], clean["q"][others])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("per_edge", [False, True])
def test_a_share_of_zero_adds_nothing(layout, per_edge, dtype):
    """Infinities and NaN in v (and, for the gradients of others, in k) behind a share that is zero in fp32: as without the edge."""
    degrees = DEGREES["ragged"]
    t = make(*LAYOUTS[layout][:2], degrees, dtype, per_edge, "edges", sources=60)
    edges = torch.tensor([0, 5, 20, 60], device="cuda")
    rows = edges
    if t["src"] is not None:
        t["src"] %= 30
        rows = t["src"][edges] = 30 + torch.arange(4, device="cuda")
    t["bias"].clamp_(min=-2.0)
    mod = module(layout, dtype, t)
    gone = {**t, "bias": t["bias"].clone()}
    gone["bias"][edges] = -math.inf
    want = run(mod, gone)
    t["bias"][edges] = torch.finfo(torch.float32).min
    for value in (float("inf"), -float("inf"), float("nan")):
        x = {**t, "v": t["v"].clone()}
        x["v"][rows] = value
        got = run(mod, x)
        for n in got:
            assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("layout", ["bulk", "loads"])
@pytest.mark.parametrize("num", [1025, 3000, 60000])
def test_tables_of_many_buckets(layout, num):
    """More than the 1,024 that RelativeBias makes: the gradient takes them in windows."""
    gen = torch.Generator().manual_seed(num)
    t = make(*LAYOUTS[layout][:2], DEGREES["hub"], torch.float32, False, "table", True)
    t["bias"] = torch.randn(num, LAYOUTS[layout][1], generator=gen).cuda()
    t["buckets"] = torch.randint(num, t["buckets"].shape, generator=gen, dtype=torch.int32).cuda()
    t["buckets"][:50], t["buckets"][50:60] = num - 1, 0
    check(layout, t, torch.float32)
    t["buckets"][7], t["buckets"][300] = num, -1
    run(module(layout, torch.float32, t), t)
    with pytest.raises(IndexError):
        e3nn_b200.check_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("num,heads,edges", [(1665, 32, 5000), (6000, 8, 20011), (1700, 70, 301), (54000, 1, 4000)])
def test_gradient_of_a_large_table(num, heads, edges, dtype):
    """Sums of n terms in fp32, one rounding each, and one to the table's type."""
    from e3nn_b200.nn._relative_bias import bias_table_grad

    gen = torch.Generator().manual_seed(num)
    b = torch.randint(num, (edges,), generator=gen, dtype=torch.int32)
    b[: edges // 2] %= 3
    g = torch.randn(edges, heads, generator=gen).to(dtype)
    got = bias_table_grad(g.cuda(), b.cuda(), num, dtype).cpu()
    add = lambda x: torch.zeros(num, heads, dtype=torch.float64).index_add_(0, b.long(), x)
    ref, n = add(g.double()), torch.bincount(b.long(), minlength=num)[:, None]
    bound = (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2) * ref.abs() + n * 2.0 ** -24 * add(g.double().abs()) + torch.finfo(dtype).tiny
    assert ((got.double() - ref).abs() <= bound).all()


def test_tables_that_32_bits_do_not_index_are_refused():
    t = make("6x0e+3x1o", 3, DEGREES["one edge"], torch.float32, False, "table")
    mod = bnn.NeighborAttention("6x0e+3x1o", "6x0e+3x1o", 3).cuda()
    with pytest.raises(NotImplementedError):
        mod(t["q"], t["k"], t["v"], t["rowptr"], t["src"], bias=torch.zeros(1, 3, device="cuda").expand(2 ** 30, 3), buckets=t["buckets"])


ALL_DEGREES = {**DEGREES, "many empty": [0] * 300 + [4] + [0] * 100, "long row": [700], "no edges": [0, 0, 0]}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("degrees", list(ALL_DEGREES))
@pytest.mark.parametrize("per_edge", [False, True])
def test_lengths_biases_weights_and_permuted_edges(degrees, per_edge, layout, dtype):
    for i, (bias, weight, perm) in enumerate(((None, False, False), ("table", False, True), ("edges", True, True), ("edges", False, False))):
        t = make(*LAYOUTS[layout][:2], ALL_DEGREES[degrees], dtype, per_edge, bias, weight, perm, seed=i)
        check(layout, t, dtype, 0.25 if sum(ALL_DEGREES[degrees]) > 20 else None)      # (of a handful of edges most gradients cancel)


WIDE = [("256x0e+256x1o", 1), ("1023x0e", 1), ("64x0e+64x1o+64x2e+64x3o", 8), ("64x0e+64x1o+64x2e+64x3o", 16), ("20x0e+20x1o+20x2e", 2), ("4096x0e", 8),
        ("40x0e+20x1o", 20), ("34x0e", 34), ("64x0e+64x1o", 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("irreps,heads", WIDE)
@pytest.mark.parametrize("per_edge", [False, True])
def test_gradients_of_wide_and_of_many_heads(irreps, heads, per_edge, dtype):
    """Up to the 1,024 columns a head that there may be (32 single columns a lane), and more heads than a warp has lanes."""
    t = make(irreps, heads, [3, 0, 40, 1], dtype, per_edge, "table", True, True)
    t["q"] *= 0.3                                          # logits of a few units
    got = run(bnn.NeighborAttention(irreps, irreps, heads).cuda(), t)
    compare(got, formula(irreps, irreps, heads, t, dtype))
    e3nn_b200.check_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("irreps,heads", [("16x0e+16x1o", 2), ("8x0e+8x1o+8x2e", 2), ("6x0e+3x1o", 3), ("64x0e+64x1o+64x2e+64x3o", 8)])
@pytest.mark.parametrize("per_edge", [False, True])
def test_large_graph(irreps, heads, per_edge, dtype):
    """Enough edges for whole blocks of warps, uneven rows and a hub."""
    gen = torch.Generator().manual_seed(heads)
    degrees = (torch.rand(900, generator=gen) ** 3 * 40).long()
    degrees[17], degrees[400:420] = 900, 0
    t = make(irreps, heads, degrees.tolist(), dtype, per_edge, "table", True, sources=700)
    compare(run(bnn.NeighborAttention(irreps, irreps, heads).cuda(), t), formula(irreps, irreps, heads, t, dtype))
    e3nn_b200.check_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("shape", ["one query", "one query, nodes", "a popular source", "two hubs"])
def test_rows_over_many_blocks(layout, shape, dtype):
    """Parts inside one row are added up in blocks first, in all three passes: one destination, one source."""
    E = 30011
    degrees = {"one query": [E], "one query, nodes": [E], "a popular source": [101] * 297, "two hubs": [14000, 0, 16000] + [1] * 5}[shape]
    t = make(*LAYOUTS[layout][:2], degrees, dtype, shape == "one query", "table", False, sources=900)
    if shape == "a popular source":                        # 95 of 100 edges leave from it
        t["k"], t["v"], t["src"] = t["k"][:2], t["v"][:2], (torch.arange(len(t["src"]), device="cuda") % 20 == 0).long()
    t["q"] *= 0.5
    mod = module(layout, dtype, t)
    got = run(mod, t)
    # a part has at most 30,308 items / 592 warps = 52 edges; up to 16 of them are added in a block, the blocks' sums by 16 warps, at most
    # 1,895 parts / 16 after one another, then the 16: below 52 + 16 + 119 + 16
    compare(got, formula(*LAYOUTS[layout][:1], *LAYOUTS[layout][:2], t, dtype, steps=203), sharp=1.0)
    again = run(mod, t)
    assert all(torch.equal(got[n], again[n]) for n in got)
    e3nn_b200.check_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_one_edge_has_share_one_and_no_gradient_through_it(layout, dtype):
    irreps, heads = LAYOUTS[layout][:2]
    N = 50
    for per_edge in (True, False):
        t = make(irreps, heads, [1] * N, dtype, per_edge, sources=N)
        if not per_edge:
            t["src"] = torch.randperm(N, generator=torch.Generator().manual_seed(0)).cuda()
        t["weight"] = torch.logspace(-30, 0, N).cuda()
        got = run(module(layout, dtype, t), t)
        assert torch.equal(got["out"], t["v"] if per_edge else t["v"][t["src"]])
        assert not got["q"].any() and not got["k"].any() and not got["weight"].any()
        assert torch.equal(got["v"] if per_edge else got["v"][t["src"]], t["g"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("per_edge", [False, True])
def test_masked_places_may_hold_anything(layout, per_edge, dtype):
    irreps, heads = LAYOUTS[layout][:2]
    E = 40
    t = make(irreps, heads, [10, 30], dtype, per_edge, sources=E)
    if not per_edge:
        t["src"] = torch.randperm(E, generator=torch.Generator().manual_seed(1)).cuda()
    bad = torch.zeros(E, dtype=torch.bool, device="cuda")
    bad[[0, 3, 11, 25, 39]] = True
    mod = module(layout, dtype, t)
    for mask in ({"weight": torch.where(bad, 0.0, 1.0)}, {"bias": torch.where(bad, -math.inf, 0.0)[:, None].repeat(1, heads)},
                 {"weight": torch.zeros(E, device="cuda")}, {"bias": torch.full((E, heads), -math.inf, device="cuda")}):
        clean = run(mod, {**t, **mask})
        if bool((mask["weight"] == 0).all() if "weight" in mask else (mask["bias"] < 0).all()):      # a row whose mask leaves nothing
            assert not any(x.any() for x in clean.values())
        for value in (float("nan"), float("inf"), -float("inf")):
            x = {**t, **mask, "k": t["k"].clone(), "v": t["v"].clone()}
            rows = bad if per_edge else t["src"][bad]
            x["k"][rows], x["v"][rows] = value, value
            got = run(mod, x)
            assert all(torch.equal(got[n], clean[n]) for n in got)
    low = {**t, "bias": torch.full((E, heads), torch.finfo(torch.float32).min, device="cuda")}      # the type's lowest value everywhere: all alike
    v = t["v"] if per_edge else t["v"][t["src"]]
    mean = torch.stack([v[:10].double().mean(0), v[10:].double().mean(0)])
    err = (run(mod, low)["out"].double() - mean).abs()
    assert (err <= torch.finfo(dtype).eps / 2 * mean.abs() + 100 * 2.0 ** -24 * v.double().abs().max()).all()


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("per_edge", [False, True])
def test_bad_indices_are_reported_and_left_out_of_gradients(layout, per_edge):
    t = make(*LAYOUTS[layout][:2], DEGREES["ragged"], torch.float32, per_edge, "table", True)
    bad = torch.tensor([2, 20, 41, 80], device="cuda")
    t["weight"].fill_(1.0)
    mod = module(layout, torch.float32, t)
    without = {**t, "weight": t["weight"].clone()}
    without["weight"][bad] = 0.0
    want = run(mod, without)
    e3nn_b200.check_status()
    cases = [("buckets", torch.tensor([9, -1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32))]
    if not per_edge:
        cases.append(("src", torch.tensor([23, -1, 2 ** 40, -2 ** 40])))
    for name, values in cases:
        x = {**t, name: t[name].clone()}
        x[name][bad] = values.cuda()
        leaves = {n: x[n].detach().requires_grad_() for n in NAMES if x[n] is not None}
        # (the edges by source of the graph as it should be: building them refuses such a source)
        out = mod(leaves["q"], leaves["k"], leaves["v"], x["rowptr"], x["src"], bias=leaves["bias"], buckets=x["buckets"], edge_weight=leaves["weight"],
                  transpose=None if per_edge else e3nn_b200.csr_from_dst(t["src"], 23))
        got = {"out": out.detach(), **dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), t["g"])))}
        with pytest.raises(IndexError):
            e3nn_b200.check_status()
        assert all(torch.equal(got[n], want[n]) for n in got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_packed_rows_broadcast_rows_and_unaligned_ones(layout, dtype):
    irreps, heads, wide, narrow = LAYOUTS[layout]
    t = make(irreps, heads, DEGREES["ragged"], dtype, False, sources=10)
    D = t["q"].shape[1]
    mod, want = module(layout, dtype, t), None
    want = run(mod, t)
    packed = torch.cat([t["q"], t["k"], t["v"]], 1).requires_grad_()
    out = mod(*packed.split([D, D, D], 1), t["rowptr"], t["src"], transpose=e3nn_b200.csr_from_dst(t["src"], 10))
    (gp,) = torch.autograd.grad(out, packed, t["g"])
    if (3 * D) % (wide if dtype == torch.float32 else narrow) == 0:                        # the same vectors
        assert torch.equal(out, want["out"]) and torch.equal(gp, torch.cat([want["q"], want["k"], want["v"]], 1))
    exact = formula(irreps, irreps, heads, t, dtype)
    odd = torch.zeros(10, 3 * D + 3, dtype=dtype, device="cuda")
    odd[:, 1:3 * D + 1] = packed.detach()
    odd.requires_grad_()
    out = mod(*odd[:, 1:3 * D + 1].split([D, D, D], 1), t["rowptr"], t["src"])
    (go,) = torch.autograd.grad(out, odd, t["g"])
    compare({"out": out.detach(), **dict(zip("qkv", go[:, 1:3 * D + 1].split([D, D, D], 1)))}, exact)
    one = t["q"][:1].expand(10, D)
    got, dense = run(mod, {**t, "q": one}), run(mod, {**t, "q": one.contiguous()})
    assert all(torch.equal(got[n], dense[n]) for n in got)
    shifted = torch.zeros(10 * D + 1, dtype=dtype, device="cuda")[1:].view(10, D).copy_(t["g"])      # a cotangent that is not aligned
    got = run(mod, {**t, "g": shifted})
    assert all(torch.equal(got[n], want[n]) for n in got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("perm", [False, True])
def test_captured_and_replayed(layout, perm, dtype):
    t = make(*LAYOUTS[layout][:2], DEGREES["hub"], dtype, False, "table", True, perm)
    mod = module(layout, dtype, t)
    transpose = e3nn_b200.csr_from_dst(t["src"], 23)
    def step(values):
        leaves = [x.detach().requires_grad_() for x in values]
        out = mod(*leaves[:3], t["rowptr"], t["src"], perm=t["perm"], bias=leaves[3], buckets=t["buckets"], edge_weight=leaves[4], transpose=transpose)
        return (out.detach(), *torch.autograd.grad(out, leaves, t["g"]))
    static = [t[n].clone() for n in NAMES]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        aside = step(static)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(aside, step(static)))
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step(static))
    for s in static[:3]:
        s.mul_(0.75)
    want = step(static)
    for _ in range(2):                                     # (a second replay finds what the first has left)
        graphs[0].replay()
        graphs[1].replay()
        assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want))
    e3nn_b200.check_status()


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("per_edge", [False, True])
@pytest.mark.parametrize("perm", [False, True])
def test_no_rows_and_no_sources(layout, per_edge, perm):
    irreps, heads = LAYOUTS[layout][:2]
    t = make(irreps, heads, [], torch.float32, per_edge, "edges", True, perm, behind=50)      # edges, but no node
    fill_free_memory()
    got = run(bnn.NeighborAttention(irreps, irreps, heads).cuda(), t)
    assert got["out"].shape == (0, t["q"].shape[1]) and not any(got[n].any() for n in got)
    e3nn_b200.check_status()
    if per_edge or perm:
        return
    t = make(irreps, heads, [3, 4], torch.float32, False, None, True)                         # sources out of range: there is none
    mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
    q, k, v = t["q"].requires_grad_(), t["k"][:0].requires_grad_(), t["v"][:0].requires_grad_()
    out = mod(q, k, v, t["rowptr"], t["src"], edge_weight=t["weight"])
    gq, gk, gv = torch.autograd.grad(out, (q, k, v), t["g"])
    with pytest.raises(IndexError):
        e3nn_b200.check_status()
    assert not out.any() and not gq.any() and gk.shape == gv.shape == k.shape


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("per_edge", [False, True])
def test_padding_may_hold_any_bucket(layout, per_edge):
    """Buckets of slots that belong to no row are looked at in neither direction."""
    t = make(*LAYOUTS[layout][:2], DEGREES["ragged"], torch.float32, per_edge, "table", True, front=9, behind=40)
    want = run(module(layout, torch.float32, t), t)
    e3nn_b200.check_status()
    padded = {**t, "buckets": t["buckets"].clone()}
    padded["buckets"][:9], padded["buckets"][-40:] = 2 ** 31 - 1, -1
    got = run(module(layout, torch.float32, t), padded)
    e3nn_b200.check_status()
    assert all(torch.equal(got[n], want[n]) for n in got)


@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_padding_may_hold_any_source(layout):
    """So may the sources of such slots, where the backward pass builds the edges by source itself; a bad source in a row is reported and left out there too."""
    t = make(*LAYOUTS[layout][:2], DEGREES["ragged"], torch.float32, False, "table", True, front=9, behind=40)
    mod = module(layout, torch.float32, t)
    want = run(mod, t)
    padded = {**t, "src": t["src"].clone()}
    padded["src"][:9], padded["src"][-40:-20], padded["src"][-20:] = -1, 23, 2 ** 40
    got = run(mod, padded, transposed=False)
    e3nn_b200.check_status()
    compare(got, formula(*LAYOUTS[layout][:1], *LAYOUTS[layout][:2], t, torch.float32))
    assert all(torch.equal(got[n], want[n]) for n in ("out", "q", "bias", "weight"))
    bad = torch.tensor([12, 30], device="cuda")
    t["weight"][bad] = 1.0
    without = {**t, "weight": t["weight"].clone()}
    without["weight"][bad] = 0.0
    t["src"][bad] = torch.tensor([-1, 23], device="cuda")
    got = run(mod, t, transposed=False)
    with pytest.raises(IndexError):
        e3nn_b200.check_status()
    without["src"] = t["src"].clamp(0, 22)
    want = run(mod, without)
    assert all(torch.equal(got[n], want[n]) for n in got)


@pytest.mark.parametrize("kind", ["per node", "per edge", "per edge, permuted"])
def test_gradients_beyond_32_bit_offsets(kind):
    """Keys and values whose last rows start past 2^31 elements, and their gradients; all rows but forty belong to nothing."""
    irreps, heads, d, E = "256x0e", 8, 256, 40
    S = 2 ** 31 // d + 1000
    gen = torch.Generator().manual_seed(0)
    small = {n: torch.randn(r, d, generator=gen).bfloat16().cuda() for n, r in (("q", 2), ("k", E), ("v", E), ("g", 2))}
    k, v = torch.zeros(S, d, dtype=torch.bfloat16, device="cuda"), torch.zeros(S, d, dtype=torch.bfloat16, device="cuda")
    rows = torch.arange(S - E, S, device="cuda")
    k[rows], v[rows] = small["k"], small["v"]
    q, k, v = small["q"].clone().requires_grad_(), k.requires_grad_(), v.requires_grad_()
    rowptr, perm = torch.tensor([0, 17, E], device="cuda"), None
    if kind == "per edge":
        rowptr = rowptr + S - E
    elif kind == "per edge, permuted":
        perm = torch.arange(S, device="cuda").roll(E)
    mod = bnn.NeighborAttention(irreps, irreps, heads).cuda()
    out = mod(q, k, v, rowptr, rows if kind == "per node" else None, perm=perm)
    gq, gk, gv = torch.autograd.grad(out, (q, k, v), small["g"])
    e3nn_b200.check_status()
    t = {**small, "rowptr": torch.tensor([0, 17, E], device="cuda"), "src": None, "perm": None, "bias": None, "buckets": None, "weight": None}
    compare({"out": out.detach(), "q": gq, "k": gk[-E:], "v": gv[-E:]}, formula(irreps, irreps, heads, t, torch.bfloat16))
    assert not gk[:-E].any() and not gv[:-E].any()
