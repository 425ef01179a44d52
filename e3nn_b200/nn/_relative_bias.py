"""Learned bias of attention by distance buckets: ``bias[e, h] = weight[bucket(|edge_vec[e]|), h]``.

The relative position bias of language models with the distance of two atoms in the place of the distance of two tokens
(invariant under rotations, so it may be added to the logits of an equivariant attention).  It has no counterpart in the
reference, whose transformer example weights the exponentials with a cutoff only (``docs/guide/transformer.rst``).

Buckets are lower ends ``t_0 = 0 < t_1 < ...``: linear up to ``r_linear``, logarithmic from there to ``r_max``; the last one takes
all longer distances.  An edge is in the last bucket whose lower end is not above its distance.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib


def _distance_buckets(pos, edge_src, edge_dst, shift, squares):
    E = edge_src.shape[0]
    out = torch.empty(E, dtype=torch.int32, device=pos.device)
    with _lib.device_of(pos):
        rc = _lib.core().e3b_distance_buckets(pos.data_ptr(), edge_src.data_ptr(), edge_dst.data_ptr(), _lib.address(shift), squares.data_ptr(),
                                              squares.shape[0], E, pos.shape[0], out.data_ptr(), _lib.status_address(pos), _lib.raw_stream(pos))
    if rc:
        _lib.check(rc, "e3b_distance_buckets")
    return out


class _DistanceBucketsFunction(torch.autograd.Function):
    """What a tracer records: whole numbers have no derivatives."""

    @staticmethod
    def forward(ctx, pos, edge_src, edge_dst, shift, squares):
        E = edge_src.shape[0]
        if pos.shape[1] != 3 or edge_dst.shape != (E,) or (shift is not None and shift.shape != (E, 3)):      # (of its next graph)
            torch._assert(False, "Incorrect shape for pos, edge_src, edge_dst or shift")
        out = _distance_buckets(pos, edge_src, edge_dst, shift, squares)
        ctx.mark_non_differentiable(out)
        return out

    @staticmethod
    def backward(ctx, grad):
        return (None,) * 5


def _look_up(weight: torch.Tensor, buckets: torch.Tensor) -> torch.Tensor:
    num, heads = weight.shape
    out = torch.empty(buckets.shape[0], heads, dtype=weight.dtype, device=weight.device)
    with _lib.device_of(weight):
        rc = _lib.core().e3b_relative_bias_fwd(weight.data_ptr(), buckets.data_ptr(), num, heads, buckets.shape[0], _lib.element_type(weight), out.data_ptr(),
                                               _lib.status_address(weight), _lib.raw_stream(weight))
    if rc:
        _lib.check(rc, "e3b_relative_bias_fwd")
    return out


class _RelativeBiasFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, buckets):
        ctx.save_for_backward(buckets)
        ctx.meta = (weight.shape[0], weight.dtype)
        return _look_up(weight, buckets)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (buckets,) = ctx.saved_tensors
        return bias_table_grad(grad, buckets, *ctx.meta), None


def bias_table_grad(grad: torch.Tensor, buckets: torch.Tensor, num_buckets: int, dtype: torch.dtype) -> torch.Tensor:
    """``out[b, h] = sum of grad[e, h] over the edges of bucket b`` in fp32, in a fixed order, rounded once to ``dtype``."""
    grad = grad.contiguous()
    if grad.data_ptr() % 16:
        grad = grad.clone()
    edges, heads = grad.shape
    out = torch.empty(num_buckets, heads, dtype=dtype, device=grad.device)
    core = _lib.core()
    nbytes = core.e3b_relative_bias_scratch_bytes(edges, num_buckets, heads)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=grad.device)
    with _lib.device_of(grad):
        rc = core.e3b_relative_bias_bwd(grad.data_ptr(), buckets.data_ptr(), num_buckets, heads, edges, _lib.element_type(grad), _lib.address(out),
                                        _lib.element_type(out), _lib.address(scratch), nbytes, _lib.status_address(grad), _lib.raw_stream(grad))
    if rc:
        _lib.check(rc, "e3b_relative_bias_bwd")
    return out


class RelativeBias(torch.nn.Module):
    """``weight [num_buckets, num_heads]`` (at most 1,024 buckets); ``buckets(...)`` once per graph, ``forward(buckets)`` gives the bias
    ``[E, num_heads]`` in the type of ``weight``.  `NeighborAttention` takes ``bias=module.weight, buckets=buckets`` and looks the bias up itself."""

    def __init__(self, num_buckets: int, num_heads: int, r_max: float, r_linear: Optional[float] = None) -> None:
        super().__init__()
        r_linear = r_max if r_linear is None else r_linear
        if not 1 <= num_buckets <= 1024 or num_heads < 1:
            raise ValueError(f"num_buckets must be 1 .. 1024 and num_heads positive, got {num_buckets} and {num_heads}")
        if num_buckets * num_heads > 2 ** 31 - 33:
            raise NotImplementedError(f"a table has fewer than 2^31 - 32 entries, got {num_buckets} buckets and {num_heads} heads")
        if not 0.0 < r_linear <= r_max < float("inf"):
            raise ValueError(f"0 < r_linear <= r_max is needed, got r_linear={r_linear} and r_max={r_max}")
        self.num_buckets, self.num_heads, self.r_max, self.r_linear = num_buckets, num_heads, float(r_max), float(r_linear)
        n = num_buckets if r_linear >= r_max else (num_buckets + 1) // 2
        ends = [self.r_linear * i / n if i <= n else self.r_linear * (self.r_max / self.r_linear) ** ((i - n) / (num_buckets - n))
                for i in range(1, num_buckets)]
        self.lower_ends = (0.0, *ends)
        # squares in fp64, kept as integers: .half() and the like leave them alone
        self.register_buffer("_squares", torch.tensor([t * t for t in ends], dtype=torch.float64).view(torch.int64), persistent=False)
        self.weight = torch.nn.Parameter(torch.randn(num_buckets, num_heads) * 0.02)

    def __repr__(self) -> str:
        return f"{self.__class__.__name__}({self.num_buckets} buckets, {self.num_heads} heads, linear to {self.r_linear}, r_max={self.r_max})"

    def buckets(self, pos: torch.Tensor, edge_src: torch.Tensor, edge_dst: torch.Tensor, shift: Optional[torch.Tensor] = None) -> torch.Tensor:
        """int32 ``[E]``: bucket of ``|pos[src] - pos[dst] + shift|``, computed in fp64 from the float32 coordinates."""
        if not pos.is_cuda:
            raise NotImplementedError("RelativeBias runs on CUDA tensors only")
        _lib.require_same_device(pos, edge_src, edge_dst, shift)
        squares, E = self._buffers["_squares"], edge_src.shape[0] if edge_src.dim() == 1 else -1
        _lib.require_operand(squares, pos, "RelativeBias's tables (move the module with .to(device))", None, torch.int64)
        if pos.dtype != torch.float32 or (shift is not None and shift.dtype != torch.float32):
            raise TypeError("pos and shift must be float32")
        if edge_src.dtype != torch.int64 or edge_dst.dtype != torch.int64:
            raise TypeError("edge_src and edge_dst must be int64")
        if pos.dim() != 2 or pos.shape[1] != 3:
            torch._assert(False, "Incorrect shape for pos")
        if E < 0 or edge_dst.shape != (E,) or (shift is not None and shift.shape != (E, 3)):
            torch._assert(False, "Incorrect shape for edge_src, edge_dst or shift")
        _lib.check_earlier(pos)
        args = (pos.contiguous(), edge_src.contiguous(), edge_dst.contiguous(), shift.contiguous() if shift is not None else None, squares)
        return _DistanceBucketsFunction.apply(*args) if _lib.is_tracing() else _distance_buckets(*args)

    def forward(self, buckets: torch.Tensor) -> torch.Tensor:
        if not buckets.is_cuda:
            raise NotImplementedError("RelativeBias runs on CUDA tensors only")
        weight = self._parameters.get("weight")
        if weight is None:      # provided by something else
            weight = self.weight
        if weight.get_device() != buckets.get_device():
            raise RuntimeError(f"Expected all tensors to be on the same device, but weight is on {weight.device} and buckets on {buckets.device}")
        if buckets.dtype != torch.int32:
            raise TypeError("buckets must be int32")
        if buckets.dim() != 1:
            torch._assert(False, "Incorrect shape for buckets")
        _lib.element_type(weight, "weight")
        _lib.check_earlier(buckets)
        apply = _RelativeBiasFunction.apply if _lib.wants_function(weight) else _look_up
        return apply(weight.contiguous(), buckets.contiguous())
