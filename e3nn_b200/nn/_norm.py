"""Norms on rows of irreps features and the boundary between two residual blocks.

`RMSNorm` divides every block ``(mul, ir)`` of a row by the root of the mean square of its ``mul * (2l+1)`` columns (a
rotation leaves that number alone) and multiplies every channel by a learned weight; the reference's ``BatchNorm``
(``e3nn/nn/_batchnorm.py:8-50``) with ``normalization='component'`` takes the same mean over a batch and has no form per row.

`NormGateResidual` is the run of steps between the last Linear of one residual block and the first of the next, in one
kernel per direction (``e3b_norm_gate_residual_fwd`` / ``_bwd``)::

    n = RMSNorm(y);  g = gate(n);  z = residual + scale * g;  h = RMSNorm(z)

Rows are fp32, bf16 or fp16; sums, products and parameters are fp32, every output is rounded once (``h`` is taken from ``z``
before ``z`` is rounded).  Gradients are first order and summed in a fixed order.
"""
from __future__ import annotations

import ctypes
from typing import List, Optional, Tuple, Union

import torch

from .. import _lib
from ..o3 import Irreps
from ._activation import Activation
from ._fc import normalize2mom_constant
from ._gate import _ACT_CODE, Gate


def _blocks(irreps: Irreps) -> List[Tuple[int, int]]:
    """``(channels, components)`` of the blocks that have columns."""
    return [(mul, ir.dim) for mul, ir in irreps if mul > 0]


def _column_blocks(blocks) -> List[Tuple[int, int]]:
    """``(block, channel)`` of every column; channels are numbered through the row."""
    out, chan = [], 0
    for b, (mul, d) in enumerate(blocks):
        out += [(b, chan + u) for u in range(mul) for _ in range(d)]
        chan += mul
    return out


def _channel_columns(blocks) -> torch.Tensor:
    """``{first column, components}`` of every channel."""
    out, at = [], 0
    for mul, d in blocks:
        out += [(at + u * d, d) for u in range(mul)]
        at += mul * d
    return torch.tensor(out, dtype=torch.int32).reshape(-1, 2)


def _inverse_counts(blocks) -> torch.Tensor:
    return torch.tensor([1.0 / (mul * d) for mul, d in blocks], dtype=torch.float32)


def _fours(blocks) -> bool:
    """Whether vectors of four columns never straddle two blocks."""
    return all(mul * d % 4 == 0 for mul, d in blocks)


def _float_bits(value: float) -> int:
    return ctypes.c_int32.from_buffer(ctypes.c_float(value)).value


def _fp32(parameter: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if parameter is None or (parameter.dtype == torch.float32 and parameter.is_contiguous()):
        return parameter
    return parameter.to(torch.float32).contiguous()


def _aligned(t: torch.Tensor, width: int) -> torch.Tensor:
    """`t`, or a copy of it where it does not start on a vector of `width` elements."""
    return t if t.data_ptr() % (width * t.element_size()) == 0 else t.clone()


def _aligned_wide(t: torch.Tensor) -> torch.Tensor:
    """Rows of more than 4,096 columns are taken by vectors of four only."""
    return t if t.shape[1] <= 4096 else _aligned(t, 4)


def _flat_rows(x: torch.Tensor, dim: int, name: str) -> torch.Tensor:
    if x.dim() < 1 or x.shape[-1] != dim:
        torch._assert(False, f"Incorrect last dimension for {name}")
    if x.dim() == 2 and x.is_contiguous():
        return x
    return x.reshape(-1, dim).contiguous() if dim > 0 else x.reshape(x.shape[:-1].numel(), 0)


def _on_device_of(x: torch.Tensor, module: torch.nn.Module, table: torch.Tensor, *parameters: Optional[torch.Tensor]) -> None:
    device = x.get_device()
    if table.get_device() != device or any(p is not None and p.get_device() != device for p in parameters):
        raise RuntimeError(f"Expected all tensors to be on the same device, but the input is on {x.device} and {type(module).__name__}'s tables or "
                           "parameters are not (move the module with .to(device))")


def _row_plan(wides, narrows, back, ins, outs, width: int, narrow: int):
    """The items of `_gate_items` as slots of at most 32 neighbours (see ``plan`` of ``e3b_norm_gate_residual_fwd``)."""
    place, length = {}, 0                             # gate column -> place of its copies, one per component
    for c, row in enumerate(back):
        if row[0] == 2:
            length += -length % 4 if c == 0 or back[c - 1][0] != 2 or back[c - 1][2] != row[2] else 0
            place[c] = length
            length += row[2]
    gate_of = {row[3] + m: place[c] + m for c, row in enumerate(back) if row[0] == 2 for m in range(row[2])}
    slots = []
    for c, j, bi, bo, *_ in wides:
        g, last = gate_of.get(c, -1), slots[-1] if slots else None
        n = last[2] if last else 0
        if last and n < 32 and last[:2] == [c - n * width, j - n * width] and last[3:5] == [bi, bo] and last[5] == (g - n * width if g >= 0 else -1):
            last[2] += 1
        else:
            slots.append([c, j, 1, bi, bo, g, 0, 0, 0, 0])
        if (g >= 0 and any(gate_of[c + i] != g + i for i in range(width))) or (g >= 0 and g % min(width, 4)):
            return None
    num_wide = len(slots)
    for kind, c, j, bi, bo, act, bits, _ in narrows:
        comps = back[c][2] if kind == 2 else 0
        at = place[c] if kind == 2 else 0
        if kind == 2 and any(back[c + i][2] != comps or place[c + i] != at + i * comps for i in range(narrow)):
            return None
        last = slots[-1] if len(slots) > num_wide else None
        n = last[3] if last else 0
        if (last and n < 32 and last[0] == kind and last[1] == c - n * narrow and last[2] == (j - n * narrow if j >= 0 else -1)
                and last[4:8] == [bi, bo, act, bits] and last[9] == comps and (kind != 2 or last[8] == at - n * narrow * comps)):
            last[3] += 1
        else:
            slots.append([kind, c, j, 1, bi, bo, act, bits, at, comps])
    din, dout = (sum(mul * d for mul, d in b) for b in (ins, outs))
    flat = [width, narrow, num_wide, len(slots) - num_wide, din, dout, len(ins), len(outs), length]
    flat += [x for slot in slots for x in slot] + [mul * d for mul, d in ins] + [mul * d for mul, d in outs]
    return _lib.HostInts(flat)


def _rms_norm(x, weight, fours: int, eps: float, num_blocks: int, tbl, inv, _channels) -> torch.Tensor:
    h = torch.empty_like(x)
    with _lib.device_of(x):
        rc = _lib.core().e3b_rms_norm_fwd(x.data_ptr(), _lib.address(weight), tbl.data_ptr(), inv.data_ptr(), num_blocks, fours, eps, h.data_ptr(),
                                          x.shape[0], x.shape[1], _lib.element_type(x), _lib.raw_stream(x))
    if rc:
        _lib.check(rc, "e3b_rms_norm_fwd")
    return h


class _RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, module):
        tables, fours, eps = module._tables(), module._fours, module.eps
        # a traced call comes here with its next input: what `RMSNorm.forward` saw was another one.  (No shapes of the tables: to a tracer
        # they are tensors from outside.)
        if x.shape[1] != module._dim:
            torch._assert(False, "Incorrect last dimension for x")
        x = x.contiguous()
        ctx.save_for_backward(x, weight)
        ctx.meta = (tables, fours, eps)
        return _rms_norm(x, weight, fours, eps, module._num_blocks, *tables)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight = ctx.saved_tensors
        (tbl, inv, channels), fours, eps = ctx.meta
        core, (rows, dim), nch = _lib.core(), x.shape, channels.shape[0]
        gx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        gw = scratch = None
        nbytes = 0
        if ctx.needs_input_grad[1]:
            gw = torch.empty(nch, dtype=torch.float32, device=x.device)
            nbytes = core.e3b_norm_scratch_bytes(rows, nch)
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        grad = _aligned_wide(grad.contiguous())
        with _lib.device_of(x):
            rc = core.e3b_rms_norm_bwd(x.data_ptr(), grad.data_ptr(), _lib.address(weight), tbl.data_ptr(), inv.data_ptr(), channels.data_ptr(), nch,
                                       inv.shape[0], fours, eps, _lib.address(gx), _lib.address(gw), _lib.address(scratch), nbytes, rows, dim,
                                       _lib.element_type(x), _lib.raw_stream(x))
        if rc:
            _lib.check(rc, "e3b_rms_norm_bwd")
        return gx, gw, None


class RMSNorm(torch.nn.Module):
    """``h[b, u, m] = weight[b, u] * x[b, u, m] / sqrt(mean_{u, m} x[b, u, m]^2 + eps)`` for every block ``b`` of ``irreps``.

    ``affine=False``: without the weights (one per channel, ones at the start).  Input ``[..., irreps.dim]`` in float32,
    bfloat16 or float16; the output has its type.  Blocks are normalised as they are written: ``"16x0e+16x0e"`` has two.
    At most 4,096 columns, 8,192 where no vector of four straddles two blocks, and 1,808 blocks."""

    def __init__(self, irreps, eps: float = 1e-5, affine: bool = True) -> None:
        super().__init__()
        self.irreps_in = self.irreps_out = Irreps(irreps)
        self.eps = float(eps)
        if not self.eps >= 0.0:
            raise ValueError(f"eps must not be negative, got {eps}")
        blocks = _blocks(self.irreps_in)
        self._dim, self._num_blocks = self.irreps_in.dim, len(blocks)
        self._fours = int(_fours(blocks))
        if self._dim > (8192 if self._fours else 4096):
            raise _lib.E3BError(f"rows of {self._dim} columns are not supported, at most 4096, 8192 where no vector of four straddles two blocks")
        cols = _column_blocks(blocks)
        tbl = torch.tensor([(b, c, 0, 0) for b, c in cols], dtype=torch.int32).reshape(-1, 4)
        self.register_buffer("_tbl", tbl, persistent=False)
        self.register_buffer("_inv_bits", _inverse_counts(blocks).view(torch.int32), persistent=False)
        self.register_buffer("_channels", _channel_columns(blocks), persistent=False)
        if affine:
            self.weight = torch.nn.Parameter(torch.ones(self._channels.shape[0]))
        else:
            self.register_parameter("weight", None)

    def __repr__(self) -> str:
        return f"{self.__class__.__name__}({self.irreps_in}, eps={self.eps})"

    def _tables(self):
        buffers = self._buffers
        return buffers["_tbl"], buffers["_inv_bits"], buffers["_channels"]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not x.is_cuda:
            raise NotImplementedError("RMSNorm runs on CUDA tensors only")
        tables, weight = self._tables(), self.weight
        _on_device_of(x, self, tables[0], weight)
        _lib.element_type(x, "x")
        rows = _aligned_wide(_flat_rows(x, self._dim, "x"))
        _lib.check_earlier(x)
        weight = _fp32(weight)
        if _lib.wants_function(rows, weight):
            out = _RMSNormFunction.apply(rows, weight, self)
        else:
            out = _rms_norm(rows, weight, self._fours, self.eps, self._num_blocks, *tables)
        return out if x.dim() == 2 else out.reshape(x.shape)


def _gate_items(back, const, forth, ins, outs, width: int, narrow: int):
    """The row as wide items of `width` columns and narrow ones of `narrow` (see ``e3b_norm_gate_residual_fwd``), `None` where it does
    not fall into such items.  `back`, `const`: per input column {kind, first output column, count, partner column, activation} and
    constant; `forth`: per output column {input column, gate column or -1, ..}."""
    out_of = {row[0]: j for j, row in enumerate(forth)}                       # input column -> output column
    slot_of = {c: n for n, c in enumerate(c for c, row in enumerate(back) if row[0] == 2)}
    in_blk, out_blk = [b for b, _ in _column_blocks(ins)], [b for b, _ in _column_blocks(outs)]
    if len(back) % width or len(forth) % width:
        return None
    # gated components, and scalars that nothing is applied to, need no activation
    plain = [row[0] == 1 or (row[0] == 0 and row[4] == 3) for row in back]
    wides, narrows, c = [], [], 0
    while c < len(back):
        n = width if plain[c] else narrow
        cols, j = range(c, c + n), out_of.get(c, -1)
        if c % n or c + n > len(back) or (j >= 0 and (j % n or j + n > len(forth) or out_blk[j + n - 1] != out_blk[j])):
            return None
        for x in cols:
            if plain[x] != plain[c] or in_blk[x] != in_blk[c] or out_of.get(x, -1) != (j + x - c if j >= 0 else -1):
                return None
            if not plain[c] and (back[x][0] != back[c][0] or back[x][4] != back[c][4] or const[x] != const[c]):
                return None
        if plain[c]:
            if any(const[x] != 1.0 for x in cols if back[x][0] == 0):
                return None
            wides.append([c, j, in_blk[c], out_blk[j], *(slot_of[forth[out_of[x]][1]] if back[x][0] == 1 else len(slot_of) for x in cols)])
        else:
            kind = back[c][0]
            if kind == 2 and slot_of[c] % n:
                return None
            narrows.append([kind, c, j, in_blk[c], out_blk[j] if j >= 0 else 0, back[c][4] if kind != 3 else 3,
                            _float_bits(const[c] if kind != 3 else 1.0), slot_of[c] if kind == 2 else 0])
        c += n
    return (torch.tensor(wides, dtype=torch.int32).reshape(-1, 4 + width), torch.tensor(narrows, dtype=torch.int32).reshape(-1, 8), len(slot_of))


def _norm_gate(residual, y, w_post, scale, w_pre, shape, eps: float, *tables):
    sizes, plan = shape
    wide, narrow, in_tbl, out_tbl, _, _, in_inv, out_inv = tables
    z = torch.empty_like(residual)
    h = torch.empty_like(residual) if w_pre is not None else None
    with _lib.device_of(y):
        rc = _lib.core().e3b_norm_gate_residual_fwd(
            residual.data_ptr(), y.data_ptr(), w_post.data_ptr(), scale.data_ptr(), _lib.address(w_pre), wide.data_ptr(), narrow.data_ptr(),
            in_tbl.data_ptr(), out_tbl.data_ptr(), in_inv.data_ptr(), out_inv.data_ptr(), sizes.address, 0 if plan is None else plan.address, eps, z.data_ptr(), _lib.address(h), y.shape[0],
            _lib.element_type(y), _lib.raw_stream(y))
    if rc:
        _lib.check(rc, "e3b_norm_gate_residual_fwd")
    return z, h


class _NormGateFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, y, w_post, scale, w_pre, module, key):
        tables, shape, eps = module._tables(key), module._sizes[key], module.eps
        # (a traced call comes here with its next inputs)
        if residual.shape != (y.shape[0], module._dims[1]) or y.shape[1] != module._dims[0] or residual.dtype != y.dtype:
            torch._assert(False, "residual and y do not fit the module")
        residual, y = residual.contiguous(), y.contiguous()
        ctx.save_for_backward(residual, y, w_post, scale, w_pre)
        ctx.meta = (tables, shape, eps)
        ctx.set_materialize_grads(False)
        return _norm_gate(residual, y, w_post, scale, w_pre, shape, eps, *tables)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_z, grad_h):
        residual, y, w_post, scale, w_pre = ctx.saved_tensors
        tables, (sizes, plan), eps = ctx.meta
        if grad_z is None and grad_h is None:
            return (None,) * 7
        core, rows, address = _lib.core(), y.shape[0], _lib.address
        grad_z, grad_h = (None if g is None else _aligned(g.contiguous(), sizes[0]) for g in (grad_z, grad_h))
        g_residual = torch.empty_like(residual) if ctx.needs_input_grad[0] else None
        gy = torch.empty_like(y) if ctx.needs_input_grad[1] else None
        params = scratch = None
        nbytes, n_in, n_out = 0, sizes[9], sizes[10]
        if any(ctx.needs_input_grad[2:5]):
            params = torch.empty(n_in + 2 * n_out, dtype=torch.float32, device=y.device)
            nbytes = core.e3b_norm_scratch_bytes(rows, n_in + 2 * n_out)
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=y.device)
        with _lib.device_of(y):
            rc = core.e3b_norm_gate_residual_bwd(
                residual.data_ptr(), y.data_ptr(), address(grad_z), address(grad_h), w_post.data_ptr(), scale.data_ptr(), address(w_pre),
                *(t.data_ptr() for t in tables), sizes.address, eps, address(g_residual), address(gy), address(params), address(scratch), nbytes, rows,
                _lib.element_type(y), _lib.raw_stream(y))
        if rc:
            _lib.check(rc, "e3b_norm_gate_residual_bwd")
        gw = params.split([n_in, n_out, n_out]) if params is not None else (None, None, None)
        return (g_residual, gy, gw[0], gw[1], gw[2] if w_pre is not None else None, None, None)


class NormGateResidual(torch.nn.Module):
    """``z = residual + scale * gate(norm(y))`` and ``h = norm(z)``: the end of one residual block and the norm before the next.

    ``gate``: a `Gate` or an `Activation`; or ``None`` with ``irreps``, and the row is added as it is.  ``y`` has the
    gate's ``irreps_in``, ``residual``, ``z`` and ``h`` its ``irreps_out``.  Parameters: ``weight_post`` (one per channel
    of ``y``, ones), ``scale`` (one per channel of ``z``, ``scale_init``) and ``weight_pre`` (one per channel of ``z``, ones);
    ``pre_norm=False``: no second norm, ``forward`` returns ``z`` alone.  At most 32 blocks of irreps, and rows of 4,096 columns."""

    def __init__(self, gate: Union[Gate, Activation, None] = None, irreps=None, eps: float = 1e-5, pre_norm: bool = True,
                 scale_init: float = 1.0) -> None:
        super().__init__()
        if (gate is None) == (irreps is None):
            raise ValueError("give either a gate or, without one, the irreps")
        if gate is not None and not isinstance(gate, (Gate, Activation)):
            raise TypeError(f"gate must be a Gate or an Activation, got {type(gate).__name__}")
        self.eps, self.pre_norm = float(eps), bool(pre_norm)
        if not self.eps >= 0.0:
            raise ValueError(f"eps must not be negative, got {eps}")
        self.irreps_in = Irreps(irreps) if gate is None else gate.irreps_in
        self.irreps_out = Irreps(irreps) if gate is None else gate.irreps_out
        ins, outs = _blocks(self.irreps_in), _blocks(self.irreps_out)
        din, dout = self.irreps_in.dim, self.irreps_out.dim
        if gate is None:
            back, const = [[0, j, 1, 0, 3] for j in range(din)], [1.0] * din
            forth = [[j, -1, 3] for j in range(dout)]
        else:
            back, forth = gate._in_tbl.tolist(), gate._out_tbl.tolist()
            # (not the gate's own table of them, which .half() and the like round)
            names = {code: name for name, code in _ACT_CODE.items()}
            constants = {code: 1.0 if names[code] is None else normalize2mom_constant(names[code]) for code in {row[4] for row in back}}
            const = [0.0 if row[0] == 3 else constants[row[4]] for row in back]
        comps = [(row[1], row[2]) if row[0] == 2 else (0, 0) for row in back]
        tables = {"_in": [(*bc, *n) for bc, n in zip(_column_blocks(ins), comps)], "_out": [(*bc, 0, 0) for bc in _column_blocks(outs)]}
        for name, value in tables.items():
            self.register_buffer(name, torch.tensor(value, dtype=torch.int32).reshape(-1, 4), persistent=False)
        self.register_buffer("_in_channels", _channel_columns(ins), persistent=False)
        self.register_buffer("_out_channels", _channel_columns(outs), persistent=False)
        self.register_buffer("_in_inv_bits", _inverse_counts(ins).view(torch.int32), persistent=False)
        self.register_buffer("_out_inv_bits", _inverse_counts(outs).view(torch.int32), persistent=False)
        n_in, n_out = self._in_channels.shape[0], self._out_channels.shape[0]
        self._dims = (din, dout)
        if max(len(ins), len(outs)) > 32:
            raise NotImplementedError(f"at most 32 blocks of irreps are supported, got {self.irreps_in} -> {self.irreps_out}")
        self._sizes, self._table_names = {}, {}
        for width, narrow in ((1, 1), (4, 1), (4, 2), (8, 2)):
            items = _gate_items(back, const, forth, ins, outs, width, narrow)
            if items is not None:
                self.register_buffer(f"_wide{width}{narrow}", items[0], persistent=False)
                self.register_buffer(f"_narrow{width}{narrow}", items[1], persistent=False)
                self._table_names[width, narrow] = (f"_wide{width}{narrow}", f"_narrow{width}{narrow}", "_in", "_out", "_in_channels", "_out_channels",
                                                    "_in_inv_bits", "_out_inv_bits")
                sizes = _lib.HostInts([width, narrow, len(items[0]), len(items[1]), items[2], din, dout, len(ins), len(outs), n_in, n_out])
                pair = 2 if width == 4 else narrow        # by warps, two columns an item where rows are wide enough for it
                rows = items if pair == narrow else _gate_items(back, const, forth, ins, outs, width, pair)
                plan = None if rows is None else _row_plan(rows[0].tolist(), rows[1].tolist(), back, ins, outs, width, pair)
                self._sizes[width, narrow] = (sizes, plan)
        if max(din, dout) > 4096:
            raise NotImplementedError(f"rows of {max(din, dout)} columns are not supported, at most 4096")
        self.weight_post = torch.nn.Parameter(torch.ones(n_in))
        self.scale = torch.nn.Parameter(torch.full((n_out,), float(scale_init)))
        if pre_norm:
            self.weight_pre = torch.nn.Parameter(torch.ones(n_out))
        else:
            self.register_parameter("weight_pre", None)

    def __repr__(self) -> str:
        return f"{self.__class__.__name__}({self.irreps_in} -> {self.irreps_out}, eps={self.eps})"

    def _tables(self, key):
        buffers = self._buffers
        return [buffers[name] for name in self._table_names[key]]

    def forward(self, residual: torch.Tensor, y: torch.Tensor):
        if not (residual.is_cuda and y.is_cuda):
            raise NotImplementedError("NormGateResidual runs on CUDA tensors only")
        if residual.shape[:-1] != y.shape[:-1]:
            torch._assert(False, "residual and y must have the same leading dimensions")
        if residual.dtype != y.dtype:
            raise TypeError(f"residual and y must have one type, got {residual.dtype} and {y.dtype}")
        _lib.element_type(y, "y")
        buffers, parameters = self._buffers, self._parameters
        try:
            w_post, scale, w_pre = parameters["weight_post"], parameters["scale"], parameters["weight_pre"]
        except KeyError:      # provided by something else
            w_post, scale, w_pre = self.weight_post, self.scale, self.weight_pre
        _on_device_of(y, self, buffers["_in"], residual, w_post, scale, w_pre)
        (din, dout), sizes = self._dims, self._sizes
        # vectors of 16 bytes if the row falls into such
        for key in ((4, 1), (1, 1)) if y.dtype == torch.float32 else ((8, 2), (4, 2), (1, 1)):
            if key in sizes:
                break
        r, x = _aligned(_flat_rows(residual, dout, "residual"), key[0]), _aligned(_flat_rows(y, din, "y"), key[0])
        _lib.check_earlier(y)
        args = (r, x, _fp32(w_post), _fp32(scale), _fp32(w_pre))
        if _lib.wants_function(*args):
            z, h = _NormGateFunction.apply(*args, self, key)
        else:
            z, h = _norm_gate(*args, sizes[key], self.eps, *self._tables(key))
        if residual.dim() == 2:
            return (z, h) if self.pre_norm else z
        return (z.reshape(residual.shape), h.reshape(residual.shape)) if self.pre_norm else z.reshape(residual.shape)
