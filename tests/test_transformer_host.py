"""Host side of the transformer modules: constructors, tables and refusals that need no GPU."""
import pytest
import torch

import e3nn_b200
from e3nn_b200 import nn as bnn
from e3nn_b200 import o3
from e3nn_b200.nn._attention import _head_vectors
from e3nn_b200.nn._norm import _channel_columns, _column_blocks


@pytest.mark.parametrize("irreps,heads", [("8x0e+8x1o+4x2e", 4), ("3x0e+6x1o", 3), ("5x0e", 1), ("4x2e+0x1o+4x0e", 2)])
def test_heads_own_every_column_once(irreps, heads):
    irreps = o3.Irreps(irreps)
    fours = all(mul // heads * ir.dim % 4 == 0 for mul, ir in irreps)
    for vec in (1, 4) if fours else (1,):
        tbl = _head_vectors(irreps, heads, vec).tolist()
        cols = [c + h * run + i for h in range(heads) for c, run in tbl for i in range(vec)]
        assert sorted(cols) == list(range(irreps.dim))
        owner = {c + h * run + i: h for h in range(heads) for c, run in tbl for i in range(vec)}
        at = 0
        for mul, ir in irreps:
            for u in range(mul):
                for m in range(ir.dim):
                    assert owner[at + u * ir.dim + m] == u * heads // mul
            at += mul * ir.dim


def test_columns_blocks_and_channels():
    irreps = o3.Irreps("2x0e+0x3o+3x1o")
    blocks = [(mul, ir.dim) for mul, ir in irreps if mul > 0]
    assert _column_blocks(blocks) == [(0, 0), (0, 1), (1, 2), (1, 2), (1, 2), (1, 3), (1, 3), (1, 3), (1, 4), (1, 4), (1, 4)]
    assert _channel_columns(blocks).tolist() == [[0, 1], [1, 1], [2, 3], [5, 3], [8, 3]]


def test_gate_rows_name_every_column():
    gate = bnn.Gate("4x0e+2x0o", [torch.nn.functional.silu, torch.tanh], "3x0e", [torch.sigmoid], "2x1o+1x2e")
    mod = bnn.NormGateResidual(gate)
    assert mod.irreps_in == gate.irreps_in and mod.irreps_out == gate.irreps_out
    assert mod._in.shape == (gate.irreps_in.dim, 4) and mod._out.shape == (gate.irreps_out.dim, 4)
    for width, narrow in mod._sizes:
        w, n = getattr(mod, f"_wide{width}{narrow}").tolist(), getattr(mod, f"_narrow{width}{narrow}").tolist()
        assert sorted([e[0] + i for e in w for i in range(width)] + [e[1] + i for e in n for i in range(narrow)]) == list(range(gate.irreps_in.dim))
        assert sorted([e[1] + i for e in w for i in range(width)] + [e[2] + i for e in n for i in range(narrow) if e[2] >= 0]) == list(range(gate.irreps_out.dim))
        for e in w:       # gates in the order of the channels they multiply
            for i, slot in enumerate(e[4:]):
                assert slot == (e[1] + i - 6) // 3 if e[1] + i < 12 else slot == 2
    assert (1, 1) in mod._sizes and sum(e[0] == 2 for e in mod._narrow11.tolist()) == 3
    assert set(bnn.NormGateResidual(bnn.Gate("8x0e", [torch.tanh], "16x0e", [torch.sigmoid], "8x1o+8x2e"))._sizes) == {(1, 1), (4, 1), (4, 2), (8, 2)}
    assert mod.weight_post.numel() == gate.irreps_in.num_irreps and mod.scale.numel() == mod.weight_pre.numel() == gate.irreps_out.num_irreps
    assert bnn.NormGateResidual(gate, pre_norm=False).weight_pre is None


@pytest.mark.parametrize("num,r_linear", [(1, None), (2, 1.0), (3, 1.0), (32, None), (33, 0.5), (1024, 2.0)])
def test_lower_ends_ascend(num, r_linear):
    mod = bnn.RelativeBias(num, 2, 5.0, r_linear=r_linear)
    ends = mod.lower_ends
    assert len(ends) == num and ends[0] == 0.0 and all(a < b for a, b in zip(ends, ends[1:])) and ends[-1] < 5.0
    squares = mod._squares.view(torch.float64)
    assert squares.tolist() == [t * t for t in ends[1:]]
    assert mod.half()._squares.dtype == torch.int64


def test_constructors_refuse():
    with pytest.raises(ValueError):
        bnn.RMSNorm("4x0e", eps=-1.0)
    with pytest.raises(NotImplementedError):
        bnn.NormGateResidual(irreps="+".join(f"1x{l}e" for l in range(33)))
    for irreps in ("4097x0e", "4100x0e"):
        with pytest.raises(NotImplementedError):
            bnn.NormGateResidual(irreps=irreps)
    gate = bnn.Gate("4x0e", [torch.tanh], "2x0e", [torch.sigmoid], "2x1o")
    with pytest.raises(ValueError):
        bnn.NormGateResidual()
    with pytest.raises(ValueError):
        bnn.NormGateResidual(gate, irreps="4x0e")
    with pytest.raises(TypeError):
        bnn.NormGateResidual(torch.nn.SiLU())
    for args in ((0, 1, 5.0), (1025, 1, 5.0), (4, 0, 5.0), (4, 1, 0.0), (4, 1, float("inf"))):
        with pytest.raises(ValueError):
            bnn.RelativeBias(*args)
    with pytest.raises(ValueError):
        bnn.RelativeBias(4, 1, 5.0, r_linear=6.0)
    with pytest.raises(ValueError):
        bnn.NeighborAttention("4x0e+2x1o", "4x0e", 4)
    with pytest.raises(ValueError):
        bnn.NeighborAttention("4x0e", "", 2)
    with pytest.raises(ValueError):
        bnn.NeighborAttention("4x0e", "4x0e", 0)
    with pytest.raises(NotImplementedError):
        bnn.NeighborAttention("1100x0e", "4x0e", 1)
    with pytest.raises(ValueError):
        bnn.AttentionBlock("4x1o+4x0e", 2)


def test_host_tensors_are_refused():
    x = torch.randn(4, 16)
    with pytest.raises(NotImplementedError):
        bnn.RMSNorm("4x0e+4x1o")(x)
    with pytest.raises(NotImplementedError):
        bnn.NormGateResidual(irreps="4x0e+4x1o")(x, x)
    idx = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(NotImplementedError):
        bnn.RelativeBias(4, 2, 5.0).buckets(x[:, :3], idx, idx)
    with pytest.raises(NotImplementedError):
        bnn.RelativeBias(4, 2, 5.0)(idx.int())
    with pytest.raises(NotImplementedError):
        bnn.NeighborAttention("4x0e+4x1o", "4x0e+4x1o", 2)(x, x, x, torch.zeros(5, dtype=torch.int64), idx)


def test_calls_that_someone_follows_go_through_autograd():
    import torch.autograd.forward_ad as fw
    from e3nn_b200 import _lib

    x, seen = torch.zeros(2), []
    assert not _lib.wants_function(x, None) and _lib.wants_function(x, torch.zeros(2, requires_grad=True))
    with torch.no_grad():
        assert not _lib.wants_function(torch.zeros(2, requires_grad=True))
        with fw.dual_level():
            assert _lib.wants_function(x)
        def f(t):
            seen.append(_lib.wants_function(t))
            return t + 1
        torch.jit.trace(f, x, check_trace=False)
        torch.func.jvp(f, (x,), (x,))
        torch.func.vmap(f)(x)
    assert seen == [True] * 3 and not _lib.wants_function(x)


def test_tables_are_indexed_in_32_bits():
    with pytest.raises(NotImplementedError, match="entries"):
        bnn.RelativeBias(1024, 2 ** 21, 5.0)


def test_rows_that_no_kernel_takes_are_refused_when_the_norm_is_made():
    for irreps in ("4097x0e", "8196x0e", "9000x0e", "1367x1o", "4095x0e+2x0o"):
        with pytest.raises(e3nn_b200.E3BError, match="columns"):
            bnn.RMSNorm(irreps)
    for irreps in ("4096x0e", "8192x0e", "4095x0e", "4093x0e+1x1o", "4100x0e"):
        assert bnn.RMSNorm(irreps)._dim == o3.Irreps(irreps).dim


def test_modules_are_copied_and_pickled():
    import copy
    import pickle

    gate = bnn.Gate("4x0e", [torch.tanh], "4x0e", [torch.sigmoid], "4x1o")
    for mod in (bnn.RMSNorm("4x0e"), bnn.NormGateResidual(gate), bnn.RelativeBias(4, 2, 5.0), bnn.NeighborAttention("4x0e+4x1o", "4x0e", 2),
                bnn.AttentionBlock("4x0e+4x1o", 2)):
        for other in (copy.deepcopy(mod), pickle.loads(pickle.dumps(mod))):
            assert repr(other) == repr(mod)
            for a, b in zip(list(mod.parameters()) + list(mod.buffers()), list(other.parameters()) + list(other.buffers())):
                assert torch.equal(a, b)
            for name in ("_layouts", "_sizes"):
                for key, value in getattr(mod, name, {}).items():
                    mine, theirs = value if isinstance(value, tuple) else (value,), getattr(other, name)[key]
                    for a, b in zip(mine, theirs if isinstance(theirs, tuple) else (theirs,)):
                        assert (a is None and b is None) or (list(a) == list(b) and a._as_parameter_ != b._as_parameter_)


def test_constants_of_a_gate_in_half_precision():
    for make in (lambda: bnn.Gate("4x0e+2x0o", [torch.nn.functional.silu, torch.tanh], "3x0e", [torch.sigmoid], "2x1o+1x2e"),
                 lambda: bnn.Activation("4x0e+2x0o+4x1o", [torch.nn.functional.silu, torch.abs, None])):
        full, half = bnn.NormGateResidual(make()), bnn.NormGateResidual(make().half())
        assert full._in_channels.tolist() == half._in_channels.tolist()
        for name, value in full.named_buffers():
            assert torch.equal(value, dict(half.named_buffers())[name]), name
        narrow = full._narrow11.tolist()
        for kind, col, _, _, _, act, bits, _ in narrow:
            assert torch.tensor(bits, dtype=torch.int32).view(torch.float32) == make()._in_cst[col]


def test_tables_of_biases_that_the_entry_points_refuse():
    """Refused before anything is launched or read: the addresses are not looked at."""
    from e3nn_b200 import _lib

    core, p, layout = _lib.core(), 256, _lib.HostInts([1, 4, 2, 2, 8, 8])
    def fwd(num_buckets):
        return core.e3b_attention_fwd(p, p, p, 8, 8, 8, p, 0, p, p, p, num_buckets, 0, p, p, layout, 1.0, 1, 1, 1, 0, p, 0, 0, p, 0, p, 0)
    def bwd(num_buckets):
        return core.e3b_attention_bwd(p, p, p, p, 8, 8, 8, p, p, p, 0, p, p, p, num_buckets, 0, p, p, layout, 1.0, 1, 1, 1, 0, p, 0, 0, 0, 0, 0, 0, p, 0, p, 0)
    for call in (fwd, bwd):
        assert call(0) == call(-1) == -1 and call(2 ** 29) == -3
        assert call(2 ** 20) == -1 and b"scratch" in core.e3b_last_error()       # (with such a table the next check is reached)
