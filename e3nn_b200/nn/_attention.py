"""Multi-head softmax attention over the incoming edges of every node, on irreps features.

The attention of the reference's transformer example (``docs/guide/transformer.rst``: ``exp = cutoff * exp(dot(q, k))``,
``alpha = exp / scatter(exp)``, ``scatter(alpha * v)``) as one pass over a destination-sorted CSR.  The dot product of two rows of
irreps is invariant, so the shares are scalars and the output transforms like the values.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from .. import _lib
from ..message_passing import csr_from_dst
from ..o3 import Irreps, Linear
from ._gate import Gate
from ._norm import NormGateResidual
from ._relative_bias import bias_table_grad

MAX_HEAD_COLUMNS = 1024


def _head_vectors(irreps: Irreps, heads: int, vec: int) -> torch.Tensor:
    """``{column of head 0, columns from one head to the next}`` of every vector of ``vec`` columns of a head."""
    out: List[Tuple[int, int]] = []
    at = 0
    for mul, ir in irreps:
        run = mul // heads * ir.dim
        out += [(at + c, run) for c in range(0, run, vec)]
        at += mul * ir.dim
    return torch.tensor(out, dtype=torch.int32).reshape(-1, 2)


def _fits(t: torch.Tensor, vec: int) -> bool:
    """Whether every row starts on a vector of `vec` elements."""
    return t.data_ptr() % (vec * t.element_size()) == 0 and t.stride(0) % vec == 0


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Rows may lie apart (a slice of a wider tensor, an expanded row); their columns may not."""
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


class _Call:
    """A checked call: its tensors as the kernels take them, and the layout that serves them."""

    __slots__ = ("q", "k", "v", "bias", "weight", "rowptr", "src", "perm", "buckets", "perm_t", "rowptr_t", "vec", "layout", "qk_tbl", "v_tbl", "scale", "edges")


def _attend(c: _Call, keep: bool):
    """The output, and for the backward pass its fp32 form and the statistics of every row."""
    q, k, v = c.q, c.k, c.v
    N, (H, dv), type_code, dev = q.shape[0], (c.layout[1], c.layout[5]), _lib.element_type(q), q.device
    core, address = _lib.core(), _lib.address
    out = torch.empty(N, dv, dtype=q.dtype, device=dev)
    out32 = stats = None
    if keep:
        stats = torch.empty(N, H, 2, dtype=torch.float32, device=dev)
        out32 = torch.empty(N, dv, dtype=torch.float32, device=dev) if type_code else None
    nbytes = core.e3b_attention_scratch_bytes(N, c.edges, H, dv)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    with _lib.device_of(q):
        rc = core.e3b_attention_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), k.stride(0), v.stride(0), c.rowptr.data_ptr(), address(c.perm), address(c.src),
            address(c.bias), address(c.buckets), c.bias.shape[0] if c.buckets is not None else 0, address(c.weight), c.qk_tbl.data_ptr(), c.v_tbl.data_ptr(),
            c.layout.address, c.scale, N, k.shape[0], c.edges, type_code, out.data_ptr(), address(out32), address(stats), scratch.data_ptr(), nbytes,
            _lib.status_address(q), _lib.raw_stream(q))
    if rc:
        _lib.check(rc, "e3b_attention_fwd")
    return out, out32 if out32 is not None else out, stats


class _AttentionFunction(torch.autograd.Function):
    """What the backward pass reads again is saved, so that changes in between are noticed.  ``edges``: rowptr, edge_src, perm, buckets and the
    transpose in one tuple; for a tracer, whose replay brings other graphs, one by one."""

    @staticmethod
    def forward(ctx, module, q, k, v, bias, weight, *edges):
        c = module._checked(q, k, v, bias, weight, *(edges if len(edges) > 1 else edges[0]))
        out, out32, stats = _attend(c, True)
        ctx.save_for_backward(c.q, c.k, c.v, c.bias, c.weight, out32, stats, c.rowptr, c.src, c.perm, c.buckets, c.perm_t, c.rowptr_t)
        ctx.call = (c.vec, c.layout, c.qk_tbl, c.v_tbl, c.scale, c.edges, len(edges))
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, k, v, bias, weight, out32, stats, rowptr, src, perm, buckets, perm_t, rowptr_t = ctx.saved_tensors
        vec, layout, qk_tbl, v_tbl, scale, E, others = ctx.call
        _, H, _, _, dqk, dv = list(layout)
        N, S, dev, type_code, core, address = q.shape[0], k.shape[0], q.device, _lib.element_type(q), _lib.core(), _lib.address
        _, need_k, need_v, need_bias, need_weight = ctx.needs_input_grad[1:6]
        grad = grad.contiguous()
        if not _fits(grad, vec):
            grad = grad.clone()
        per_node = src is not None and (need_k or need_v) and S > 0
        per_edge = src is None and (need_k or need_v)
        gq = torch.empty(N, dqk, dtype=q.dtype, device=dev)
        gk = torch.empty(S, dqk, dtype=q.dtype, device=dev) if need_k or need_v else None
        gv = torch.empty(S, dv, dtype=q.dtype, device=dev) if need_k or need_v else None
        share = torch.empty(E, (H + 1) // 2 * 2, 2, dtype=torch.float32, device=dev) if per_node else None
        da = torch.empty(E, H, dtype=torch.float32, device=dev) if need_bias or need_weight else None
        # with a permutation the call finds the edges of no row by it
        dst = torch.empty(E, dtype=torch.int32, device=dev) if per_node or (perm is not None and (per_edge or da is not None)) else None
        gweight = torch.empty(E, dtype=torch.float32, device=dev) if need_weight else None
        nbytes = core.e3b_attention_bwd_scratch_bytes(N, E, dqk)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        status = _lib.status_address(q)
        with _lib.device_of(q):
            rc = core.e3b_attention_bwd(
                address(q), address(k), address(v), address(grad), q.stride(0), k.stride(0), v.stride(0), address(out32), address(stats),
                address(rowptr), address(perm), address(src), address(bias), address(buckets), bias.shape[0] if buckets is not None else 0, address(weight),
                address(qk_tbl), address(v_tbl), layout.address, scale, N, S, E, type_code, address(gq), address(gk) if per_edge else None,
                address(gv) if per_edge else None, address(share), address(da), address(dst), address(gweight), address(scratch), nbytes, status,
                _lib.raw_stream(q))
        if rc:
            _lib.check(rc, "e3b_attention_bwd")
        if per_node:
            if perm_t is None:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("the edges by source cannot be built while a graph is captured: give NeighborAttention transpose=csr_from_dst(edge_src, k.shape[0])")
                # (slots of no row may name any source, bad ones of rows have been reported: neither adds anything, wherever it is sorted to)
                perm_t, rowptr_t = csr_from_dst(src.clamp(0, S - 1), S)
            nbytes = core.e3b_attention_bwd_src_scratch_bytes(S, E, dqk, dv)
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            with _lib.device_of(q):
                rc = core.e3b_attention_bwd_src(
                    address(q), address(grad), q.stride(0), address(share), address(dst), address(perm_t), address(rowptr_t), address(qk_tbl), address(v_tbl),
                    layout.address, scale, N, S, E, type_code, address(gk), address(gv), address(scratch), nbytes, status, _lib.raw_stream(q))
            if rc:
                _lib.check(rc, "e3b_attention_bwd_src")
        gbias = None
        if need_bias:
            gbias = bias_table_grad(da, buckets, bias.shape[0], torch.float32) if buckets is not None else da
        return None, gq, gk if need_k else None, gv if need_v else None, gbias, gweight, *(None,) * others


class NeighborAttention(torch.nn.Module):
    """``out[n]_h = sum_e share[e, h] v[src_e]_h`` over the edges ``e`` of node ``n``, with
    ``share = softmax_e(scale * <q[n], k[src_e]>_h + bias[e, h] + log(edge_weight[e]))``.

    Head ``h`` owns channels ``h mul / H .. (h+1) mul / H`` of every block of the irreps, so ``num_heads`` divides all
    multiplicities; a head has at most 1,024 columns of each of ``irreps_qk`` and ``irreps_v``.  ``scale`` defaults to the inverse root of
    the columns of a head of ``irreps_qk``.
    """

    def __init__(self, irreps_qk, irreps_v, num_heads: int, scale: Optional[float] = None) -> None:
        super().__init__()
        self.irreps_qk, self.irreps_v, self.num_heads = Irreps(irreps_qk), Irreps(irreps_v), int(num_heads)
        if self.num_heads < 1:
            raise ValueError(f"num_heads must be positive, got {num_heads}")
        for irreps in (self.irreps_qk, self.irreps_v):
            if irreps.dim == 0 or any(mul % self.num_heads for mul, _ in irreps):
                raise ValueError(f"{self.num_heads} heads must divide the multiplicities of {irreps}, which must not be empty")
            if irreps.dim // self.num_heads > MAX_HEAD_COLUMNS:
                raise NotImplementedError(f"{irreps.dim // self.num_heads} columns a head, at most {MAX_HEAD_COLUMNS} are supported")
        self.scale = float(scale) if scale is not None else (self.irreps_qk.dim // self.num_heads) ** -0.5
        self._layouts, self._dims = {}, (self.irreps_qk.dim, self.irreps_v.dim)
        runs = [mul // self.num_heads * ir.dim for irreps in (self.irreps_qk, self.irreps_v) for mul, ir in irreps]
        for vec in (1, 4, 8):
            if any(run % vec for run in runs):
                break
            tables = [_head_vectors(irreps, self.num_heads, vec) for irreps in (self.irreps_qk, self.irreps_v)]
            self.register_buffer(f"_qk{vec}", tables[0], persistent=False)
            self.register_buffer(f"_v{vec}", tables[1], persistent=False)
            self._layouts[vec] = _lib.HostInts([vec, self.num_heads, tables[0].shape[0], tables[1].shape[0], *self._dims])

    def __repr__(self) -> str:
        return f"{self.__class__.__name__}(q, k: {self.irreps_qk}, v: {self.irreps_v}, {self.num_heads} heads)"

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rowptr: torch.Tensor, edge_src: Optional[torch.Tensor] = None,
                perm: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, buckets: Optional[torch.Tensor] = None,
                edge_weight: Optional[torch.Tensor] = None, transpose: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                check_indices: bool = False) -> torch.Tensor:
        """``q [N, irreps_qk.dim]``, ``k`` and ``v`` in one of float32, bfloat16 and float16 -> ``[N, irreps_v.dim]`` in that type.

        Edge slot ``s`` in ``[rowptr[n], rowptr[n+1])`` belongs to node ``n`` and is edge ``perm[s]`` (``s`` itself without ``perm``;
        `e3nn_b200.csr_from_dst` gives both).  ``edge_src [E]``: ``k`` and ``v`` are rows of nodes, edge ``e`` reads row ``edge_src[e]``;
        without it they are rows of edges.  Slots before ``rowptr[0]`` and from ``rowptr[N]`` on belong to no node (``rowptr[a:b+1]`` gives
        the nodes ``a .. b-1`` of a graph alone); their gradients are zero.  A node without edges gets zeros.

        ``bias``: ``[E, num_heads]``, or with ``buckets [E]`` (int32) a table ``[num_buckets, num_heads]`` of any length (`RelativeBias`);
        an entry ``-inf`` of the former masks its edge for that head, whatever ``k`` and ``v`` hold there.  ``edge_weight [E]``
        multiplies the exponentials (a smooth cutoff); an edge with weight zero or below is left out, its rows are not read
        and its gradients, that of the weight included, are zero.  So does an edge whose share is zero in fp32 (below 2^-126): it adds
        nothing to any sum, infinities and NaN in its ``v`` or in the cotangent of its row included.

        Statistics and sums are fp32.  Gradients (first order, fixed order of summation) of ``q``, ``k``, ``v``, ``bias`` and ``edge_weight``;
        those of node-wise ``k`` and ``v`` need the edges by source, ``transpose = csr_from_dst(edge_src, k.shape[0])``,
        which is built in the backward pass (with a synchronisation: not while a graph is captured) if it is not given.
        Indices out of range are reported like those of `conv_uvu` and their edges left out.  ``rowptr`` must not decrease.  ``perm`` may
        leave out edges (their gradients are zero) and name any edge in slots of no node, but none twice in slots of nodes: the
        forward pass would count it twice, the backward pass reports it.
        """
        if transpose is not None and len(transpose) != 2:
            torch._assert(False, "Incorrect shape for transpose")
        edges = (rowptr, edge_src, perm, buckets, *(transpose or (None, None)))
        if _lib.wants_function(q, k, v, bias, edge_weight):
            out = _AttentionFunction.apply(self, q, k, v, bias, edge_weight, *(edges if _lib.is_tracing() else (edges,)))
        else:
            out = _attend(self._checked(q, k, v, bias, edge_weight, *edges), False)[0]
        if check_indices:
            _lib.check_status(q.device, "NeighborAttention")
        return out

    def _checked(self, q, k, v, bias, edge_weight, rowptr, edge_src, perm, buckets, perm_t, rowptr_t) -> _Call:
        buffers = self._buffers
        _lib.require_same_device(q, k, v, rowptr, edge_src, perm, bias, buckets, edge_weight, perm_t, rowptr_t)
        if buffers["_qk1"].get_device() != q.get_device():
            raise RuntimeError(f"Expected all tensors to be on the same device, but NeighborAttention's tables are on {buffers['_qk1'].device} and q is on "
                               f"{q.device} (move the module with .to(device))")
        _lib.element_type(q, "q")
        if not q.dtype == k.dtype == v.dtype:
            raise TypeError(f"q, k and v must have one type, got {q.dtype}, {k.dtype} and {v.dtype}")
        for t, name in ((rowptr, "rowptr"), (edge_src, "edge_src"), (perm, "perm"), (perm_t, "transpose"), (rowptr_t, "transpose")):
            if t is not None and (t.dtype != torch.int64 or t.dim() != 1):
                if t.dtype != torch.int64:
                    raise TypeError(f"{name} must be int64")
                torch._assert(False, f"Incorrect shape for {name}")
        H, dqk, dv = self.num_heads, self._dims[0], self._dims[1]
        N, S = q.shape[0] if q.dim() == 2 else -1, k.shape[0] if k.dim() == 2 else -1
        E = S if edge_src is None else edge_src.shape[0]
        wrong = [name for name, bad in (
            ("q", q.shape != (N, dqk)), ("k", k.shape != (S, dqk)), ("v", v.shape != (S, dv)), ("rowptr", rowptr.shape[0] != N + 1),
            ("perm", perm is not None and perm.shape[0] != E), ("buckets", buckets is not None and buckets.shape != (E,)),
            ("bias", bias is not None and (bias.dim() != 2 or bias.shape[1] != H or (buckets is None and bias.shape[0] != E))),
            ("edge_weight", edge_weight is not None and edge_weight.shape != (E,)),
            ("transpose", (perm_t is None) != (rowptr_t is None) or (perm_t is not None and (perm_t.shape[0] != E or rowptr_t.shape[0] != S + 1)))) if bad]
        if wrong:
            torch._assert(False, f"Incorrect shape for {wrong[0]}")
        if buckets is not None:
            if bias is None:
                raise ValueError("buckets need the table they index: bias=[num_buckets, num_heads]")
            if buckets.dtype != torch.int32:
                raise TypeError("buckets must be int32")
            if bias.shape[0] * H > 2 ** 31 - 33:
                raise NotImplementedError("a table of biases has fewer than 2^31 - 32 entries")
        for t, name in ((bias, "bias"), (edge_weight, "edge_weight")):
            if t is not None:
                _lib.element_type(t, name)
        if max(E, N, S) >= 2 ** 31 - 1:
            raise NotImplementedError("at most 2^31 - 2 edges and rows")
        _lib.check_earlier(q)
        c = _Call()
        c.q, c.k, c.v = _rows(q), _rows(k), _rows(v)
        # vectors of 16 bytes where the layout and the rows allow them, else of four elements, else single elements
        for c.vec in (4, 1) if q.dtype == torch.float32 else (8, 4, 1):
            if c.vec in self._layouts and _fits(c.q, c.vec) and _fits(c.k, c.vec) and _fits(c.v, c.vec):
                break
        c.layout, c.qk_tbl, c.v_tbl = self._layouts[c.vec], buffers[f"_qk{c.vec}"], buffers[f"_v{c.vec}"]
        c.scale, c.edges = self.scale, E
        c.rowptr, c.src, c.perm, c.buckets, c.perm_t, c.rowptr_t = (t if t is None or t.is_contiguous() else t.contiguous()
                                                                    for t in (rowptr, edge_src, perm, buckets, perm_t, rowptr_t))
        c.bias = None if bias is None else bias.to(torch.float32).contiguous()
        c.weight = None if edge_weight is None else edge_weight.to(torch.float32).contiguous()
        return c


class AttentionBlock(torch.nn.Module):
    """One residual attention block on node features, from the modules of this package::

        q, k, v = Linear(h)
        y       = Linear(NeighborAttention(q, k, v))
        x', h'  = NormGateResidual(gate)(x, y)            h' = norm(x') is the next block's input

    ``h`` is ``x`` after a norm: `RMSNorm` before the first block, the previous block's second output after it.  Scalars
    of ``irreps_node`` are activated with ``act`` and all other channels gated with ``gate_act``."""

    def __init__(self, irreps_node, num_heads: int, irreps_key=None, act=torch.nn.functional.silu, gate_act=torch.sigmoid,
                 linear_math_mode: str = "tf32x3", eps: float = 1e-5, scale_init: float = 1.0) -> None:
        super().__init__()
        self.irreps_node = Irreps(irreps_node)
        self.irreps_key = Irreps(irreps_key) if irreps_key is not None else self.irreps_node
        scalars = Irreps([(mul, ir) for mul, ir in self.irreps_node if ir.l == 0])
        gated = Irreps([(mul, ir) for mul, ir in self.irreps_node if ir.l > 0])
        gates = Irreps([(mul, "0e") for mul, _ in gated])
        gate = Gate(scalars, [act] * len(scalars), gates, [gate_act] * len(gates), gated)
        if gate.irreps_out != self.irreps_node:
            raise ValueError(f"irreps_node must be sorted, scalars first, and keep its parities under the activations: got {self.irreps_node}, "
                             f"the gate gives {gate.irreps_out}")
        self.attention = NeighborAttention(self.irreps_key, self.irreps_node, num_heads)
        self.lin_qkv = Linear(self.irreps_node, self.irreps_key + self.irreps_key + self.irreps_node, math_mode=linear_math_mode)
        self.lin_out = Linear(self.irreps_node, gate.irreps_in, math_mode=linear_math_mode)
        self.post = NormGateResidual(gate, eps=eps, scale_init=scale_init)

    def forward(self, x: torch.Tensor, h: torch.Tensor, rowptr: torch.Tensor, edge_src: torch.Tensor, **edges) -> Tuple[torch.Tensor, torch.Tensor]:
        """``x`` and ``h`` ``[N, irreps_node.dim]`` float32; ``edges`` are the keyword arguments of `NeighborAttention`
        (``perm``, ``bias``, ``buckets``, ``edge_weight``, ``transpose``)."""
        dk = self.irreps_key.dim
        q, k, v = self.lin_qkv(h).split([dk, dk, self.irreps_node.dim], dim=-1)
        return self.post(x, self.lin_out(self.attention(q, k, v, rowptr, edge_src, **edges)))
