// Attention over the incoming edges of every node: gradients of keys and values that are rows of nodes.
//
//   grad_k[s] = scale sum_e da[e] q[dst(e)]      grad_v[s] = sum_e p[e] g[dst(e)]      over the outgoing edges e of node s
// with p and da from attention_bwd.cu.  The edges of a source come from the CSR by source (perm, rowptr: the stable sort of
// edge_src), so every row is summed in a fixed order, without atomics (which would move two rows an edge twice, read and
// written).  The same parts, lanes and ring as in the forward kernel, with the edge's p and da as a third copy: 425,984 edges of
// 1,024 columns in bf16 211 us = 8.3 TB/s of gathered rows, in fp32 432 us.
#include "attention.cuh"

namespace e3b {
namespace {

struct SrcArgs {
    const void *q, *grad_out;
    int64_t q_stride;
    const float2* share;          // [edges, even(heads)] {p, da}
    const int32_t* dst;           // [edges], -1: no destination
    const int64_t* perm;          // [edges] edges in the order of their sources
    void *grad_k, *grad_v;        // [num_src, dqk], [num_src, dv]
    int64_t num_dst;
    float scale;
    Heads h;
    Rows r;
    Partials parts;
    int32_t* status;
    bool merge;
    RingSource ring;
    int depth;
    uint32_t warp_smem;
};

// The 32 slots from `base` on, one a lane: edge and its destination (-1: the edge is left out).
struct SourceMeta {
    int edge, row;
    __device__ __forceinline__ void load(const SrcArgs& a, int64_t slot, int64_t last) {
        edge = row = -1;
        if (slot >= last) return;
        const int64_t e = a.perm[slot];
        if (e < 0 || e >= a.r.edges) {
            *a.status = 2;
            return;
        }
        edge = static_cast<int>(e);
        row = a.dst[e];
        if (row >= a.num_dst) row = -1;
    }
};

template <typename T, int VEC, int V>
__global__ void __launch_bounds__(256) attn_bwd_src_kernel(const SrcArgs a) {
    extern __shared__ float smem[];
    constexpr int U = edges_in_flight(V, words_of<T, VEC>(), 80);
    const int lane = threadIdx.x & 31, part = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int head = blockIdx.y * (32 / a.h.lanes) + lane / a.h.lanes;
    const bool live = head < a.h.heads, leads = live && (lane & (a.h.lanes - 1)) == 0;
    int cq[V], cv[V];
    lane_columns<V>(a.h.qk, a.h.nqk, a.h.lanes, head, live, cq);
    lane_columns<V>(a.h.v, a.h.nv, a.h.lanes, head, live, cv);
    const T* q = static_cast<const T*>(a.q);
    const T* g = static_cast<const T*>(a.grad_out);
    Sums<VEC, V, 2, false> s;
    s.clear();
    int64_t goes_on = -1;
    int ended = -1;
    if (part < a.r.parts) {
        const Part range = find_part(a.r, part);
        walk_rows(
            a.r, range, [&](int64_t) { s.clear(); },
            [&](int64_t first, int64_t last) {
                for (int64_t base = first; base < last; base += 32) {
                    SourceMeta meta;
                    meta.load(a, base + lane, last);
                    const int count = static_cast<int>(min(last - base, int64_t{32}));
                    for (int u0 = 0; u0 < count; u0 += U) {
                        Packed<T, VEC> qq[U][V], gg[U][V];
                        float p[U], da[U];
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            const int edge = __shfl_sync(kAll, meta.edge, u0 + u), dst = __shfl_sync(kAll, meta.row, u0 + u);
                            const bool use = dst >= 0;
                            const float2 x = use && live ? a.share[static_cast<int64_t>(edge) * ((a.h.heads + 1) & ~1) + head] : make_float2(0.0f, 0.0f);
                            p[u] = x.x;
                            da[u] = x.y;
                            load_row<T, VEC, V>(qq[u], q, dst, a.q_stride, cq, use);
                            load_row<T, VEC, V>(gg[u], g, dst, a.h.dv, cv, use);
                        }
#pragma unroll
                        for (int u = 0; u < U; ++u) {
#pragma unroll
                            for (int j = 0; j < V; ++j) {
                                float x[VEC], y[VEC];
                                qq[u][j].unpack(x);
                                gg[u][j].unpack(y);
#pragma unroll
                                for (int i = 0; i < VEC; ++i) {      // (a share of zero adds nothing, whatever q and the cotangent hold)
                                    if (da[u] != 0.0f) s.a[0][j][i] = fmaf(da[u], x[i], s.a[0][j][i]);
                                    if (p[u] != 0.0f) s.a[1][j][i] = fmaf(p[u], y[i], s.a[1][j][i]);
                                }
                            }
                        }
                    }
                }
            },
            [&](int64_t n, bool started, bool ends) {
                if (!ends) {
                    goes_on = n;
                } else if (started) {
                    store_row<T, VEC, V>(static_cast<T*>(a.grad_k), n, a.h.dqk, cq, s.a[0], a.scale);
                    store_row<T, VEC, V>(static_cast<T*>(a.grad_v), n, a.h.dv, cv, s.a[1], 1.0f);
                } else {
                    s.save(a.parts.at(part, 0), a.h, cq, cv, head, leads);
                    ended = static_cast<int>(n);
                }
            });
        if (blockIdx.y == 0 && lane == 0) a.parts.ended[part] = ended;
    }
    leave_part(a.merge, s, goes_on, part, a.r.parts, a.parts, a.h, cq, cv, head, leads, smem);
}

// The same with the rows of q and g, and the shares of the edge, through the ring.
template <typename T, int VEC, int V>
__global__ void __launch_bounds__(512, 1) attn_bwd_src_ring_kernel(const SrcArgs a) {
    extern __shared__ __align__(128) uint8_t memory[];
    constexpr int U = edges_together(V * VEC);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = blockIdx.x * (blockDim.x >> 5) + warp;
    const int head = lane / a.h.lanes;
    const bool live = head < a.h.heads, leads = live && (lane & (a.h.lanes - 1)) == 0;
    int cq[V], cv[V];
    lane_columns<V>(a.h.qk, a.h.nqk, a.h.lanes, head, live, cq);
    lane_columns<V>(a.h.v, a.h.nv, a.h.lanes, head, live, cv);
    uint32_t pq[V], pv[V];
    slot_places<T, V>(cq, 0, a.ring.zeros(), pq);
    slot_places<T, V>(cv, a.ring.a_bytes, a.ring.zeros(), pv);
    Sums<VEC, V, 2, false> s;
    s.clear();
    int64_t goes_on = -1;
    int ended = -1;
    if (part < a.r.parts) {
        const Part range = find_part(a.r, part);
        Ring<U, SourceMeta> ring(a.ring, memory + warp * a.warp_smem, a.depth);
        bool use[U];
        walk_ring(
            a.r, range, ring, a.status, [&](SourceMeta& m, int i) { m.load(a, range.e0 + i, range.behind); }, [&](int64_t) { s.clear(); },
            [&](const SourceMeta& meta, int at, int m) {
#pragma unroll
                for (int u = 0; u < U; ++u) use[u] = u < m && __shfl_sync(kAll, meta.row, (at + u) & 31) >= 0;
            },
            [&](const uint8_t* const (&slot)[U], const SourceMeta&, int, int) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (!use[u] || !live) continue;
                    const float2 x = reinterpret_cast<const float2*>(slot[u] + a.ring.a_bytes + a.ring.b_bytes)[head];
                    if (x.y != 0.0f) add_row<T, VEC, V>(slot[u], x.y, s.a[0], pq);
                    if (x.x != 0.0f) add_row<T, VEC, V>(slot[u], x.x, s.a[1], pv);
                }
            },
            [&](int64_t n, bool started, bool ends) {
                if (!ends) {
                    goes_on = n;
                } else if (started) {
                    store_row<T, VEC, V>(static_cast<T*>(a.grad_k), n, a.h.dqk, cq, s.a[0], a.scale);
                    store_row<T, VEC, V>(static_cast<T*>(a.grad_v), n, a.h.dv, cv, s.a[1], 1.0f);
                } else {
                    s.save(a.parts.at(part, 0), a.h, cq, cv, head, leads);
                    ended = static_cast<int>(n);
                }
            });
        if (lane == 0) a.parts.ended[part] = ended;
    }
    leave_part(a.merge, s, goes_on, part, a.r.parts, a.parts, a.h, cq, cv, head, leads, reinterpret_cast<float*>(memory));
}

template <typename T, int VEC, int V>
__global__ void __launch_bounds__(512) attn_bwd_src_join_kernel(const SrcArgs a) {
    extern __shared__ float smem[];
    const int lane = threadIdx.x & 31;
    const int head = blockIdx.y * (32 / a.h.lanes) + lane / a.h.lanes;
    const bool live = head < a.h.heads;
    int cq[V], cv[V];
    lane_columns<V>(a.h.qk, a.h.nqk, a.h.lanes, head, live, cq);
    lane_columns<V>(a.h.v, a.h.nv, a.h.lanes, head, live, cv);
    Sums<VEC, V, 2, false> s;
    int64_t n;
    if (!join_parts(s, a.r, blockIdx.x, a.parts, a.h, cq, cv, head, live, smem, &n)) return;
    store_row<T, VEC, V>(static_cast<T*>(a.grad_k), n, a.h.dqk, cq, s.a[0], a.scale);
    store_row<T, VEC, V>(static_cast<T*>(a.grad_v), n, a.h.dv, cv, s.a[1], 1.0f);
}

int dkv_slot(int dqk, int dv) { return static_cast<int>(ceil_div(dqk + dv, 4) * 4); }

}  // namespace
}  // namespace e3b

using namespace e3b;

extern "C" int64_t e3b_attention_bwd_src_scratch_bytes(int64_t num_src, int64_t num_edges, int dim_qk, int dim_v) {
    if (num_src < 0 || num_edges < 0) return 0;
    return partial_bytes(most_parts(num_src, num_edges), dkv_slot(dim_qk, dim_v));
}

extern "C" int e3b_attention_bwd_src(const void* q, const void* grad_out, int64_t q_stride, const float* share,
                                     const int32_t* edge_dst, const int64_t* src_perm, const int64_t* src_rowptr, const int32_t* qk_table,
                                     const int32_t* v_table, const int32_t* layout, float scale, int64_t num_dst, int64_t num_src,
                                     int64_t num_edges, int type, void* grad_k, void* grad_v, void* scratch, int64_t scratch_bytes,
                                     int32_t* status, void* stream) {
    if (!layout || num_dst < 0 || num_src < 0 || num_edges < 0 || num_edges >= INT32_MAX || num_dst >= INT32_MAX || num_src >= INT32_MAX || !known_type(type))
        return fail(E3B_ERR_ARG, "attention_bwd_src: bad size or type");
    const int vec = layout[0], heads = layout[1], nqk = layout[2], nv = layout[3], dqk = layout[4], dv = layout[5];
    if (heads < 1 || (vec != 1 && vec != 4 && (vec != 8 || type == kFloat32))) return fail(E3B_ERR_ARG, "attention_bwd_src: bad head layout");
    if (num_src == 0) return E3B_OK;
    if ((num_edges > 0 && num_dst > 0 && (!q || !grad_out)) || (num_edges > 0 && (!share || !aligned_to(share, 16) || !edge_dst || !src_perm)) || !src_rowptr ||
        !qk_table || !v_table || !grad_k || !grad_v || !scratch || !status)
        return fail(E3B_ERR_ARG, "attention_bwd_src: null pointer");
    if (scratch_bytes < e3b_attention_bwd_src_scratch_bytes(num_src, num_edges, dqk, dv))
        return fail(E3B_ERR_ARG, "attention_bwd_src: scratch of %lld bytes is too small", static_cast<long long>(scratch_bytes));
    const int size = element_size(type);
    const RingSource rows{static_cast<const char*>(q), static_cast<const char*>(grad_out), reinterpret_cast<const char*>(share), q_stride * size,
                          static_cast<int64_t>(dv) * size, static_cast<uint32_t>(dqk * size), static_cast<uint32_t>(dv * size),
                          static_cast<uint32_t>(((heads + 1) & ~1) * sizeof(float2))};
    Plan p;
    const int planned = plan(&p, "attention_bwd_src", type, vec, heads, std::max(nqk, nv), num_src, num_edges, rows, 4, 3, true);
    if (planned != E3B_OK) return planned;
    const Split& s = p.s;
    SrcArgs a{q, grad_out, q_stride, reinterpret_cast<const float2*>(share), edge_dst, src_perm, grad_k, grad_v, num_dst, scale,
              {qk_table, v_table, heads, nqk, nv, dqk, dv, p.lanes}, {src_rowptr, num_src, num_edges, s.per_part, s.parts},
              partials_in(scratch, s.parts, dkv_slot(dqk, dv)), status, s.merge, rows, p.depth, static_cast<uint32_t>(p.warp_smem)};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_type_and_vectors(type, vec, p.v, [&](auto t0, auto vec0, auto v0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(vec0)::value, V = decltype(v0)::value;
        using S = Sums<VEC, V, 2, false>;
        const unsigned blocks = static_cast<unsigned>(ceil_div(s.parts, s.warps));
        const size_t merge_smem = s.merge ? sizeof(float) * 32 * S::kFloats * s.warps : 0;
        int r = E3B_OK;
        if constexpr (VEC * sizeof(T) == 16) {
            if (p.ring) {
                const size_t smem = std::max(p.warp_smem * s.warps, merge_smem);
                if ((r = allow_smem(attn_bwd_src_ring_kernel<T, VEC, V>, smem)) != E3B_OK) return r;
                attn_bwd_src_ring_kernel<T, VEC, V><<<blocks, 32 * s.warps, smem, st>>>(a);
            }
        }
        if (!p.ring) {
            if ((r = allow_smem(attn_bwd_src_kernel<T, VEC, V>, merge_smem)) != E3B_OK) return r;
            attn_bwd_src_kernel<T, VEC, V><<<dim3(blocks, p.groups), 32 * s.warps, merge_smem, st>>>(a);
        }
        if ((r = check_launch("attention_bwd_src")) != E3B_OK || s.parts == 1) return r;
        const size_t smem = s.join_warps > 1 ? sizeof(float) * 32 * S::kFloats * s.join_warps : 0;
        if ((r = allow_smem(attn_bwd_src_join_kernel<T, VEC, V>, smem)) != E3B_OK) return r;
        attn_bwd_src_join_kernel<T, VEC, V><<<dim3(s.parts, p.groups), 32 * s.join_warps, smem, st>>>(a);
        return check_launch("attention_bwd_src join");
    });
}
