// Attention over the incoming edges of every node: gradients along the rows of destinations.
//
// With p = softmax(a) (computed again from q, k and the kept maximum and sum), g the cotangent of the output:
//   dp[e, h] = <g[dst], v[src]>_h     delta[n, h] = <g[n], out[n]>_h     da = p (dp - delta)
//   grad_q[n] = scale sum_e da k[src]      grad_k = scale da q[dst]      grad_v = p g[dst]      grad bias = da
// delta is taken from the unrounded fp32 output: dp - delta cancels, and in a row with one edge it is exactly zero.
// k and v per edge: their gradients are written here, row by row.  k and v per node: p and da of every edge are kept and
// attention_bwd_src.cu adds the terms of every source over its outgoing edges.  Like the forward kernel with three products
// a column in place of two: 425,984 edges of 1,024 columns in bf16 450 us = 3.9 TB/s of gathered rows (latency and shared-memory reads at 42 %
// of the issue slots: the registers, q, g and the sums of q's gradient, allow twelve warps an SM), in fp32 1,127 us; 150,001 edges with k and v per edge, 180 columns in fp32, 102 us (432 MB read and written).
#include "attention.cuh"

namespace e3b {
namespace {

struct BwdArgs {
    const void *q, *k, *v, *grad_out;
    int64_t q_stride, k_stride, v_stride;
    const float *out32, *stats;
    void *grad_q, *grad_k, *grad_v;      // grad_k, grad_v: per edge, or null
    float2* share;                       // [edges, even(heads)] {p, da} or null
    float* da;                           // [edges, heads] or null
    int32_t* dst;                        // [edges] or null: destination of every edge; with a permutation below zero beforehand
    float scale;
    Heads h;
    Edges e;
    Rows r;
    Partials parts;
    bool merge;
    RingSource ring;
    int depth;
    uint32_t warp_smem;
    __device__ __forceinline__ float2* share_of(int64_t edge) const { return share + edge * ((h.heads + 1) & ~1); }
};

// q, cotangent and statistics of a row; returns delta.  The output enters unrounded, in the order of the dots g v of the kernel (PAIRS: of
// dot_row): an edge alone in its row gives the same number.
template <bool PAIRS, typename T, int VEC, int V>
__device__ __forceinline__ float open_row(const BwdArgs& a, int64_t n, const int (&cq)[V], const int (&cv)[V], int head, bool live, float (&qf)[V][VEC],
                                          float (&gf)[V][VEC], float* top, float* inv) {
    load_row_f<T, VEC, V>(qf, static_cast<const T*>(a.q), n, a.q_stride, cq);
    load_row_f<T, VEC, V>(gf, static_cast<const T*>(a.grad_out), n, a.h.dv, cv);
    float d = 0.0f, o[V][VEC];
    load_row_f<float, VEC, V>(o, a.out32, n, a.h.dv, cv);
    if constexpr (PAIRS) {
        float2 pair = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < VEC; i += 2) pair = fma2(make_float2(gf[j][i], gf[j][i + 1]), make_float2(o[j][i], o[j][i + 1]), pair);
        d = pair.x + pair.y;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) d = fmaf(gf[j][i], o[j][i], d);
    }
    if (live) {
        *top = a.stats[(n * a.h.heads + head) * 2];
        *inv = a.stats[(n * a.h.heads + head) * 2 + 1];
    }
    return head_sum(d, a.h.lanes);
}

// Slots in front of the first row and behind the last take part in nothing: their gradients are zero.  With a permutation the
// edges that no row has visited are cleared afterwards (clear_unvisited_kernel): slots outside may name any edge, and not every
// edge need be named.
template <typename T, int VEC, int V>
__device__ __forceinline__ void clear_outside(const BwdArgs& a, int part, const int (&cq)[V], const int (&cv)[V], int head, bool leads) {
    if (a.e.perm || (a.r.num > 0 && a.r.begin(0) == 0 && a.r.end(a.r.num - 1) == a.r.edges)) return;
    const Part range = find_part(a.r, part);      // (found again: kept from the walk it costs registers there)
    float zero[V][VEC];
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) zero[j][i] = 0.0f;
    auto clear = [&](int64_t from, int64_t to) {
        for (int64_t e = from; e < to; ++e) {
            if (a.dst && blockIdx.y == 0 && (threadIdx.x & 31) == 0) a.dst[e] = -1;
            if (leads && a.share) a.share_of(e)[head] = make_float2(0.0f, 0.0f);
            if (leads && a.da) a.da[e * a.h.heads + head] = 0.0f;
            if (a.grad_k) {
                store_row<T, VEC, V>(static_cast<T*>(a.grad_k), e, a.h.dqk, cq, zero, 0.0f);
                store_row<T, VEC, V>(static_cast<T*>(a.grad_v), e, a.h.dv, cv, zero, 0.0f);
            }
        }
    };
    clear(range.first, range.e0);
    clear(range.behind, range.e1);
}

template <typename T, int VEC, int V>
__global__ void __launch_bounds__(256) attn_bwd_dst_kernel(const BwdArgs a) {
    extern __shared__ float smem[];
    constexpr int U = edges_in_flight(V, words_of<T, VEC>(), 64);
    const int lane = threadIdx.x & 31, part = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int head = blockIdx.y * (32 / a.h.lanes) + lane / a.h.lanes;
    const bool live = head < a.h.heads, leads = live && (lane & (a.h.lanes - 1)) == 0;
    int cq[V], cv[V];
    lane_columns<V>(a.h.qk, a.h.nqk, a.h.lanes, head, live, cq);
    lane_columns<V>(a.h.v, a.h.nv, a.h.lanes, head, live, cv);
    const T* k = static_cast<const T*>(a.k);
    const T* v = static_cast<const T*>(a.v);
    Sums<VEC, V, 1, false> s;
    s.clear();
    int64_t goes_on = -1;
    int ended = -1;
    if (part < a.r.parts) {
        float qf[V][VEC], gf[V][VEC], delta = 0.0f, top = 0.0f, inv = 0.0f;
        int row_now = 0;
        const Part range = find_part(a.r, part);
        walk_rows(
            a.r, range,
            [&](int64_t n) {
                row_now = static_cast<int>(n);
                delta = open_row<false, T, VEC, V>(a, n, cq, cv, head, live, qf, gf, &top, &inv);
                s.clear();
            },
            [&](int64_t first, int64_t last) {
                for (int64_t base = first; base < last; base += 32) {
                    EdgeMeta meta;
                    meta.load(a.e, base + lane, last);
                    if (a.dst && blockIdx.y == 0 && meta.edge >= 0) a.dst[meta.edge] = row_now;
                    const int count = static_cast<int>(min(last - base, int64_t{32}));
                    for (int u0 = 0; u0 < count; u0 += U) {
                        Packed<T, VEC> kk[U][V], vv[U][V];
                        float bias[U];
                        int edge[U];
                        bool use[U];
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            const int row = __shfl_sync(kAll, meta.row, u0 + u);
                            edge[u] = __shfl_sync(kAll, meta.edge, u0 + u);
                            use[u] = row >= 0;
                            bias[u] = 0.0f;
                            if (a.e.buckets) {
                                const int b = __shfl_sync(kAll, meta.bucket, u0 + u);
                                if (live) bias[u] = a.e.bias[b * a.h.heads + head];
                            } else if (a.e.bias) {
                                if (live && edge[u] >= 0) bias[u] = a.e.bias[static_cast<int64_t>(edge[u]) * a.h.heads + head];
                                use[u] = use[u] && bias[u] != -INFINITY;
                            }
                            load_row<T, VEC, V>(kk[u], k, row, a.k_stride, cq, use[u]);
                            load_row<T, VEC, V>(vv[u], v, row, a.v_stride, cv, use[u]);
                        }
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            float d = 0.0f, dp = 0.0f, kf[V][VEC];
#pragma unroll
                            for (int j = 0; j < V; ++j) {
                                float vf[VEC];
                                kk[u][j].unpack(kf[j]);
                                vv[u][j].unpack(vf);
#pragma unroll
                                for (int i = 0; i < VEC; ++i) {
                                    d = fmaf(qf[j][i], kf[j][i], d);
                                    dp = fmaf(gf[j][i], vf[i], dp);
                                }
                            }
                            const float x = logit(head_sum(d, a.h.lanes), a.scale, bias[u], a.e.weight ? __shfl_sync(kAll, meta.log_weight, u0 + u) : 0.0f);
                            dp = head_sum(dp, a.h.lanes);
                            float p = 0.0f, da = 0.0f;
                            if (use[u]) {
                                p = __expf(x - top) * inv;
                                da = p == 0.0f ? 0.0f : p * (dp - delta);
                            }
                            if (da != 0.0f) {
#pragma unroll
                                for (int j = 0; j < V; ++j)
#pragma unroll
                                    for (int i = 0; i < VEC; ++i) s.a[0][j][i] = fmaf(da, kf[j][i], s.a[0][j][i]);
                            }
                            if (edge[u] < 0) continue;
                            if (leads && a.share) a.share_of(edge[u])[head] = make_float2(p, da);
                            if (leads && a.da) a.da[static_cast<int64_t>(edge[u]) * a.h.heads + head] = da;
                            if (a.grad_k) {
                                store_row<T, VEC, V, true>(static_cast<T*>(a.grad_k), edge[u], a.h.dqk, cq, qf, a.scale * da);
                                store_row<T, VEC, V, true>(static_cast<T*>(a.grad_v), edge[u], a.h.dv, cv, gf, p);
                            }
                        }
                    }
                }
            },
            [&](int64_t n, bool started, bool ends) {
                if (!ends) {
                    goes_on = n;
                } else if (started) {
                    if (a.grad_q) store_row<T, VEC, V>(static_cast<T*>(a.grad_q), n, a.h.dqk, cq, s.a[0], a.scale);
                } else {
                    s.save(a.parts.at(part, 0), a.h, cq, cv, head, leads);
                    ended = static_cast<int>(n);
                }
            });
        clear_outside<T, VEC, V>(a, part, cq, cv, head, leads);
        if (blockIdx.y == 0 && lane == 0) a.parts.ended[part] = ended;
    }
    leave_part(a.merge, s, goes_on, part, a.r.parts, a.parts, a.h, cq, cv, head, leads, smem);
}

// The same with k and v through the ring.
template <typename T, int VEC, int V>
__global__ void __launch_bounds__(384, 1) attn_bwd_dst_ring_kernel(const BwdArgs a) {
    extern __shared__ __align__(128) uint8_t memory[];
    constexpr int U = edges_together(V * VEC);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = blockIdx.x * (blockDim.x >> 5) + warp;
    const int head = lane / a.h.lanes;
    const bool live = head < a.h.heads, leads = live && (lane & (a.h.lanes - 1)) == 0;
    int cq[V], cv[V];
    lane_columns<V>(a.h.qk, a.h.nqk, a.h.lanes, head, live, cq);
    lane_columns<V>(a.h.v, a.h.nv, a.h.lanes, head, live, cv);
    Sums<VEC, V, 1, false> s;
    s.clear();
    int64_t goes_on = -1;
    int ended = -1;
    if (part < a.r.parts) {
        const Part range = find_part(a.r, part);
        Ring<U, EdgeMeta> ring(a.ring, memory + warp * a.warp_smem, a.depth);
        float qf[V][VEC], gf[V][VEC], delta = 0.0f, top = 0.0f, inv = 0.0f, bias[U];
        int edge[U], row_now = 0;
        bool use[U];
        walk_ring(
            a.r, range, ring, a.e.status, [&](EdgeMeta& m, int i) { m.load(a.e, range.e0 + i, range.behind); },
            [&](int64_t n) {
                row_now = static_cast<int>(n);
                delta = open_row<true, T, VEC, V>(a, n, cq, cv, head, live, qf, gf, &top, &inv);
                s.clear();
            },
            [&](const EdgeMeta& meta, int at, int m) {
                if (a.dst && lane >= at && lane < at + m && meta.edge >= 0) a.dst[meta.edge] = row_now;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int from = (at + u) & 31;
                    edge[u] = __shfl_sync(kAll, meta.edge, from);
                    if (u >= m) edge[u] = -1;
                    use[u] = __shfl_sync(kAll, meta.row, from) >= 0 && edge[u] >= 0;
                    bias[u] = 0.0f;
                    if (a.e.buckets) {
                        const int b = __shfl_sync(kAll, meta.bucket, from);
                        if (live) bias[u] = a.e.bias[b * a.h.heads + head];
                    } else if (a.e.bias) {
                        if (live && use[u]) bias[u] = a.e.bias[static_cast<int64_t>(edge[u]) * a.h.heads + head];
                        use[u] = use[u] && bias[u] != -INFINITY;
                    }
                }
            },
            [&](const uint8_t* const (&slot)[U], const EdgeMeta& meta, int at, int m) {
                float x[2 * U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    x[u] = dot_columns<T, VEC, V>(slot[u], qf, cq);
                    x[U + u] = dot_columns<T, VEC, V>(slot[u] + a.ring.a_bytes, gf, cv);
                }
                head_sums<2 * U>(x, a.h.lanes);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float lw = a.e.weight ? __shfl_sync(kAll, meta.log_weight, (at + u) & 31) : 0.0f;
                    if (edge[u] < 0) continue;
                    float p = 0.0f, da = 0.0f;
                    if (use[u]) {
                        p = __expf(logit(x[u], a.scale, bias[u], lw) - top) * inv;
                        da = p == 0.0f ? 0.0f : p * (x[U + u] - delta);
                    }
                    if (da != 0.0f) add_columns<T, VEC, V>(slot[u], da, s.a[0], cq);
                    if (leads && a.share) a.share_of(edge[u])[head] = make_float2(p, da);
                    if (leads && a.da) a.da[static_cast<int64_t>(edge[u]) * a.h.heads + head] = da;
                    if (a.grad_k) {
                        store_row<T, VEC, V, true>(static_cast<T*>(a.grad_k), edge[u], a.h.dqk, cq, qf, a.scale * da);
                        store_row<T, VEC, V, true>(static_cast<T*>(a.grad_v), edge[u], a.h.dv, cv, gf, p);
                    }
                }
            },
            [&](int64_t n, bool started, bool ends) {
                if (!ends) {
                    goes_on = n;
                } else if (started) {
                    store_row<T, VEC, V>(static_cast<T*>(a.grad_q), n, a.h.dqk, cq, s.a[0], a.scale);
                } else {
                    s.save(a.parts.at(part, 0), a.h, cq, cv, head, leads);
                    ended = static_cast<int>(n);
                }
            });
        clear_outside<T, VEC, V>(a, part, cq, cv, head, leads);
        if (lane == 0) a.parts.ended[part] = ended;
    }
    leave_part(a.merge, s, goes_on, part, a.r.parts, a.parts, a.h, cq, cv, head, leads, reinterpret_cast<float*>(memory));
}

template <typename T, int VEC, int V>
__global__ void __launch_bounds__(512) attn_bwd_dst_join_kernel(const BwdArgs a) {
    extern __shared__ float smem[];
    const int lane = threadIdx.x & 31;
    const int head = blockIdx.y * (32 / a.h.lanes) + lane / a.h.lanes;
    const bool live = head < a.h.heads;
    int cq[V];
    lane_columns<V>(a.h.qk, a.h.nqk, a.h.lanes, head, live, cq);
    Sums<VEC, V, 1, false> s;
    int64_t n;
    if (join_parts(s, a.r, blockIdx.x, a.parts, a.h, cq, cq, head, live, smem, &n)) store_row<T, VEC, V>(static_cast<T*>(a.grad_q), n, a.h.dqk, cq, s.a[0], a.scale);
}

// With a permutation, before the rows are walked: every edge that a slot of a row names is claimed (-1 -> -2).  One that is named twice would
// get its gradients from two rows.  (An exchange in the kernel that walks the rows costs it 2 % without a permutation too.)
__global__ void __launch_bounds__(256) claim_edges_kernel(const Rows r, const int64_t* __restrict__ perm, int32_t* __restrict__ dst, int32_t* status) {
    const int64_t last = r.num > 0 ? r.end(r.num - 1) : 0;
    for (int64_t s = (r.num > 0 ? r.begin(0) : 0) + static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; s < last; s += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t e = perm[s];
        if (e >= 0 && e < r.edges && atomicCAS(dst + e, -1, -2) != -1) *status = 4;
    }
}

// Gradients of the edges that no row has visited (dst below zero) are zero.  A warp looks at 32 edges.
template <typename T>
__global__ void __launch_bounds__(256) clear_unvisited_kernel(const int32_t* __restrict__ dst, int64_t edges, int heads, int dqk, int dv, float* __restrict__ da,
                                                              T* __restrict__ grad_k, T* __restrict__ grad_v) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
    for (int64_t base = (static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5)) * 32; base < edges; base += warps * 32) {
        unsigned left = __ballot_sync(kAll, base + lane < edges && dst[base + lane] < 0);
        for (; left; left &= left - 1) {
            const int64_t e = base + __ffs(left) - 1;
            if (da)
                for (int i = lane; i < heads; i += 32) da[e * heads + i] = 0.0f;
            if (!grad_k) continue;
            for (int i = lane; i < dqk; i += 32) grad_k[e * dqk + i] = from_float<T>(0.0f);
            for (int i = lane; i < dv; i += 32) grad_v[e * dv + i] = from_float<T>(0.0f);
        }
    }
}

// Gradient of the weight of every edge: share / weight = exp(logit without it) / sum, so it is sum_h da / weight; an edge that was
// left out has none.
__global__ void __launch_bounds__(256) attn_weight_grad_kernel(const float* __restrict__ da, const float* __restrict__ weight, int heads,
                                                               int64_t edges, float* __restrict__ grad) {
    for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < edges; e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const float w = weight[e];
        float s = 0.0f;
        for (int h = 0; h < heads; ++h) s += da[e * heads + h];
        grad[e] = w <= 0.0f || s == 0.0f ? 0.0f : s / w;      // (s = 0: also an edge of no row, whatever its weight)
    }
}

int dq_slot(int dqk) { return static_cast<int>(ceil_div(dqk, 4) * 4); }

}  // namespace
}  // namespace e3b

using namespace e3b;

extern "C" int64_t e3b_attention_bwd_scratch_bytes(int64_t num_dst, int64_t num_edges, int dim_qk) {
    if (num_dst < 0 || num_edges < 0) return 0;
    return partial_bytes(most_parts(num_dst, num_edges), dq_slot(dim_qk));
}

extern "C" int e3b_attention_bwd(const void* q, const void* k, const void* v, const void* grad_out, int64_t q_stride, int64_t k_stride,
                                 int64_t v_stride, const float* out32, const float* stats, const int64_t* rowptr, const int64_t* perm,
                                 const int64_t* edge_src, const float* bias, const int32_t* buckets, int num_buckets,
                                 const float* edge_weight, const int32_t* qk_table, const int32_t* v_table, const int32_t* layout,
                                 float scale, int64_t num_dst, int64_t num_src, int64_t num_edges, int type, void* grad_q, void* grad_k,
                                 void* grad_v, float* share, float* grad_logit, int32_t* edge_dst, float* grad_weight, void* scratch,
                                 int64_t scratch_bytes, int32_t* status, void* stream) {
    if (!layout || num_dst < 0 || num_src < 0 || num_edges < 0 || num_edges >= INT32_MAX || num_dst >= INT32_MAX || num_src >= INT32_MAX || !known_type(type))
        return fail(E3B_ERR_ARG, "attention_bwd: bad size or type");
    const int vec = layout[0], heads = layout[1], nqk = layout[2], nv = layout[3], dqk = layout[4], dv = layout[5];
    if (heads < 1 || (vec != 1 && vec != 4 && (vec != 8 || type == kFloat32))) return fail(E3B_ERR_ARG, "attention_bwd: bad head layout");
    if (buckets && num_buckets < 1) return fail(E3B_ERR_ARG, "attention_bwd: an empty table of biases");      // (the kernels read its first row in the place of a bad one)
    if (buckets && static_cast<int64_t>(num_buckets) * heads > INT32_MAX - 32)
        return fail(E3B_ERR_UNSUPPORTED, "attention_bwd: a table of %d buckets and %d heads", num_buckets, heads);
    if (num_dst == 0 && num_edges == 0) return E3B_OK;
    if ((num_dst > 0 && (!q || !grad_out || !out32 || !stats || !grad_q)) || !rowptr || (num_edges > 0 && num_src > 0 && (!k || !v)) || !qk_table ||
        !v_table || !scratch || !status || (share && !aligned_to(share, 16)) || (buckets && !bias) || !grad_k != !grad_v || (grad_weight && (!edge_weight || !grad_logit)) ||
        (perm && num_edges > 0 && (share || grad_logit || grad_k) && !edge_dst))
        return fail(E3B_ERR_ARG, "attention_bwd: null pointer");
    if (scratch_bytes < e3b_attention_bwd_scratch_bytes(num_dst, num_edges, dqk))
        return fail(E3B_ERR_ARG, "attention_bwd: scratch of %lld bytes is too small", static_cast<long long>(scratch_bytes));
    const int size = element_size(type);
    const RingSource rows{static_cast<const char*>(k), static_cast<const char*>(v), nullptr, k_stride * size, v_stride * size,
                          static_cast<uint32_t>(dqk * size), static_cast<uint32_t>(dv * size), 0};
    Plan p;
    const int planned = plan(&p, "attention_bwd", type, vec, heads, std::max(nqk, nv), num_dst, num_edges, rows, 3, 4, true);
    if (planned != E3B_OK) return planned;
    const Split& s = p.s;
    BwdArgs a{q, k, v, grad_out, q_stride, k_stride, v_stride, out32, stats, grad_q, grad_k, grad_v, reinterpret_cast<float2*>(share), grad_logit,
              edge_dst, scale, {qk_table, v_table, heads, nqk, nv, dqk, dv, p.lanes},
              {perm, edge_src, bias, buckets, edge_weight, num_buckets, num_src, num_edges, status},
              {rowptr, num_dst, num_edges, s.per_part, s.parts}, partials_in(scratch, s.parts, dq_slot(dqk)), s.merge, rows, p.depth,
              static_cast<uint32_t>(p.warp_smem)};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned edge_grid = static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(ceil_div(num_edges, 256), kNumSMs * 8)));
    if (perm && edge_dst) {
        E3B_CUDA_TRY(cudaMemsetAsync(edge_dst, 0xff, sizeof(int32_t) * num_edges, st));      // all -1
        claim_edges_kernel<<<edge_grid, 256, 0, st>>>(a.r, perm, edge_dst, status);
        const int claimed = check_launch("attention_bwd edges");
        if (claimed != E3B_OK) return claimed;
    }
    const int rc = by_type_and_vectors(type, vec, p.v, [&](auto t0, auto vec0, auto v0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(vec0)::value, V = decltype(v0)::value;
        using S = Sums<VEC, V, 1, false>;
        const unsigned blocks = static_cast<unsigned>(ceil_div(s.parts, s.warps));
        const size_t merge_smem = s.merge ? sizeof(float) * 32 * S::kFloats * s.warps : 0;
        int r = E3B_OK;
        if constexpr (VEC * sizeof(T) == 16) {
            if (p.ring) {
                const size_t smem = std::max(p.warp_smem * s.warps, merge_smem);
                if ((r = allow_smem(attn_bwd_dst_ring_kernel<T, VEC, V>, smem)) != E3B_OK) return r;
                attn_bwd_dst_ring_kernel<T, VEC, V><<<blocks, 32 * s.warps, smem, st>>>(a);
            }
        }
        if (!p.ring) {
            if ((r = allow_smem(attn_bwd_dst_kernel<T, VEC, V>, merge_smem)) != E3B_OK) return r;
            attn_bwd_dst_kernel<T, VEC, V><<<dim3(blocks, p.groups), 32 * s.warps, merge_smem, st>>>(a);
        }
        if ((r = check_launch("attention_bwd")) != E3B_OK || s.parts == 1) return r;
        const size_t smem = s.join_warps > 1 ? sizeof(float) * 32 * S::kFloats * s.join_warps : 0;
        if ((r = allow_smem(attn_bwd_dst_join_kernel<T, VEC, V>, smem)) != E3B_OK) return r;
        attn_bwd_dst_join_kernel<T, VEC, V><<<dim3(s.parts, p.groups), 32 * s.join_warps, smem, st>>>(a);
        return check_launch("attention_bwd join");
    });
    if (rc != E3B_OK || num_edges == 0) return rc;
    if (perm && (grad_logit || grad_k)) {
        auto clear = [&](auto t0) {
            using T = decltype(t0);
            clear_unvisited_kernel<T><<<edge_grid, 256, 0, st>>>(edge_dst, num_edges, heads, dqk, dv, grad_logit, static_cast<T*>(grad_k), static_cast<T*>(grad_v));
        };
        if (type == kFloat32) clear(float());
        else if (type == kBFloat16) clear(__nv_bfloat16());
        else clear(__half());
        const int cleared = check_launch("attention_bwd edges of no row");
        if (cleared != E3B_OK) return cleared;
    }
    if (!grad_weight) return E3B_OK;
    attn_weight_grad_kernel<<<edge_grid, 256, 0, st>>>(
        grad_logit, edge_weight, heads, num_edges, grad_weight);
    return check_launch("attention_bwd weights");
}
