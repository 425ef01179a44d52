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


class _RelativeBiasFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, buckets):
        out = torch.empty(buckets.shape[0], weight.shape[1], dtype=weight.dtype, device=weight.device)
        with _lib.device_of(weight):
            rc = _lib.core().e3b_relative_bias_fwd(_lib._ptr(weight), _lib._ptr(buckets), weight.shape[0], weight.shape[1], buckets.shape[0],
                                                   _lib.element_type(weight), _lib._ptr(out), _lib._ptr(_lib.status_word(weight.device)),
                                                   _lib.stream_ptr())
        _lib.check(rc, "e3b_relative_bias_fwd")
        ctx.save_for_backward(buckets)
        ctx.meta = (weight.shape, weight.dtype)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (buckets,) = ctx.saved_tensors
        shape, dtype = ctx.meta
        return bias_table_grad(grad, buckets, shape[0], dtype), None


def bias_table_grad(grad: torch.Tensor, buckets: torch.Tensor, num_buckets: int, dtype: torch.dtype) -> torch.Tensor:
    """``out[b, h] = sum of grad[e, h] over the edges of bucket b`` in fp32, in a fixed order, rounded once to ``dtype``."""
    grad = grad.contiguous()
    edges, heads = grad.shape
    out = torch.empty(num_buckets, heads, dtype=dtype, device=grad.device)
    core = _lib.core()
    nbytes = core.e3b_relative_bias_scratch_bytes(edges, num_buckets, heads)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=grad.device)
    with _lib.device_of(grad):
        rc = core.e3b_relative_bias_bwd(_lib._ptr(grad), _lib._ptr(buckets), num_buckets, heads, edges, _lib.element_type(grad), _lib._ptr(out),
                                        _lib.element_type(out), _lib._ptr(scratch), nbytes, _lib._ptr(_lib.status_word(grad.device)), _lib.stream_ptr())
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
        _lib.require_operand(self._squares, pos, "RelativeBias's tables (move the module with .to(device))", None, torch.int64)
        E = edge_src.numel()
        if pos.dtype != torch.float32 or (shift is not None and shift.dtype != torch.float32):
            raise TypeError("pos and shift must be float32")
        if edge_src.dtype != torch.int64 or edge_dst.dtype != torch.int64:
            raise TypeError("edge_src and edge_dst must be int64")
        torch._assert(pos.dim() == 2 and pos.shape[1] == 3, "Incorrect shape for pos")
        torch._assert(edge_src.shape == edge_dst.shape == (E,), "Incorrect shape for edge_src or edge_dst")
        torch._assert(shift is None or shift.shape == (E, 3), "Incorrect shape for shift")
        _lib.poll_status(pos.device)
        out = torch.empty(E, dtype=torch.int32, device=pos.device)
        pos, edge_src, edge_dst = pos.detach().contiguous(), edge_src.contiguous(), edge_dst.contiguous()
        shift = shift.detach().contiguous() if shift is not None else None
        with _lib.device_of(pos):
            rc = _lib.core().e3b_distance_buckets(_lib._ptr(pos), _lib._ptr(edge_src), _lib._ptr(edge_dst), _lib._ptr(shift), _lib._ptr(self._squares),
                                                  self.num_buckets - 1, E, pos.shape[0], _lib._ptr(out), _lib._ptr(_lib.status_word(pos.device)),
                                                  _lib.stream_ptr())
        _lib.check(rc, "e3b_distance_buckets")
        return out

    def forward(self, buckets: torch.Tensor) -> torch.Tensor:
        if not buckets.is_cuda:
            raise NotImplementedError("RelativeBias runs on CUDA tensors only")
        if self.weight.device != buckets.device:
            raise RuntimeError(f"Expected all tensors to be on the same device, but weight is on {self.weight.device} and buckets on {buckets.device}")
        if buckets.dtype != torch.int32:
            raise TypeError("buckets must be int32")
        torch._assert(buckets.dim() == 1, "Incorrect shape for buckets")
        _lib.element_type(self.weight, "weight")
        _lib.poll_status(buckets.device)
        return _RelativeBiasFunction.apply(self.weight.contiguous(), buckets.contiguous())
