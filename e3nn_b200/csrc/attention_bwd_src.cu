// Attention over the incoming edges of every node: gradients of keys and values that are rows of nodes.
//
//   grad_k[s] = scale sum_e da[e] q[dst(e)]      grad_v[s] = sum_e p[e] g[dst(e)]      over the outgoing edges e of node s
// with p and da from attention_bwd.cu.  The edges of a source come from the CSR by source (perm, rowptr: the stable sort of
// edge_src), so every row is summed in a fixed order, without atomics (which would move two rows an edge twice, read and
// written).  Bound by the gather of q and g: the same parts, lanes and loads in flight as in the forward kernel.
#include "attention.cuh"

namespace e3b {
namespace {

struct SrcArgs {
    const void *q, *grad_out;
    int64_t q_stride;
    const float *p, *da;          // [edges, heads]
    const int32_t* dst;           // [edges], -1: no destination
    const int64_t* perm;          // [edges] edges in the order of their sources
    void *grad_k, *grad_v;        // [num_src, dqk], [num_src, dv]
    int64_t num_dst;
    float scale;
    Heads h;
    Rows r;
    Partials parts;
    int32_t* status;
};

template <typename T, int VEC, int V, bool MERGE>
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
        walk_rows(
            a.r, part, [&](int64_t) { s.clear(); },
            [&](int64_t first, int64_t last) {
                for (int64_t base = first; base < last; base += 32) {
                    int my_edge = -1, my_dst = -1;
                    if (base + lane < last) {
                        const int64_t e = a.perm[base + lane];
                        if (e >= 0 && e < a.r.edges) {
                            my_edge = static_cast<int>(e);
                            my_dst = a.dst[e];
                            if (my_dst >= a.num_dst) my_dst = -1;
                        } else {
                            *a.status = 2;
                        }
                    }
                    const int count = static_cast<int>(min(last - base, int64_t{32}));
                    for (int u0 = 0; u0 < count; u0 += U) {
                        Packed<T, VEC> qq[U][V], gg[U][V];
                        float p[U], da[U];
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            const int edge = __shfl_sync(kAll, my_edge, u0 + u), dst = __shfl_sync(kAll, my_dst, u0 + u);
                            const bool use = dst >= 0;
                            p[u] = use && live ? a.p[static_cast<int64_t>(edge) * a.h.heads + head] : 0.0f;
                            da[u] = use && live ? a.da[static_cast<int64_t>(edge) * a.h.heads + head] : 0.0f;
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
                                for (int i = 0; i < VEC; ++i) {
                                    s.a[0][j][i] = fmaf(da[u], x[i], s.a[0][j][i]);
                                    s.a[1][j][i] = fmaf(p[u], y[i], s.a[1][j][i]);
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
            },
            [](int64_t, int64_t) {});
        if (blockIdx.y == 0 && lane == 0) a.parts.ended[part] = ended;
    }
    leave_part<MERGE>(s, goes_on, part, a.r.parts, a.parts, a.h, cq, cv, head, leads, smem);
}

template <typename T, int VEC, int V>
__global__ void __launch_bounds__(256) attn_bwd_src_join_kernel(const SrcArgs a) {
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
    return partial_bytes(split_rows(num_src, num_edges).parts, dkv_slot(dim_qk, dim_v));
}

extern "C" int e3b_attention_bwd_src(const void* q, const void* grad_out, int64_t q_stride, const float* share, const float* grad_logit,
                                     const int32_t* edge_dst, const int64_t* src_perm, const int64_t* src_rowptr, const int32_t* qk_table,
                                     const int32_t* v_table, const int32_t* layout, float scale, int64_t num_dst, int64_t num_src,
                                     int64_t num_edges, int type, void* grad_k, void* grad_v, void* scratch, int64_t scratch_bytes,
                                     int32_t* status, void* stream) {
    if (!layout || num_dst < 0 || num_src < 0 || num_edges < 0 || num_edges >= INT32_MAX || num_dst >= INT32_MAX || num_src >= INT32_MAX || !known_type(type))
        return fail(E3B_ERR_ARG, "attention_bwd_src: bad size or type");
    const int vec = layout[0], heads = layout[1], nqk = layout[2], nv = layout[3], dqk = layout[4], dv = layout[5];
    if (heads < 1 || (vec != 1 && vec != 4)) return fail(E3B_ERR_ARG, "attention_bwd_src: bad head layout");
    const int most = vec == 4 ? 8 : 32, lanes = lanes_of_head(heads, std::max(nqk, nv), most);
    if (lanes == 0) return fail(E3B_ERR_UNSUPPORTED, "attention_bwd_src: a head of %d columns (at most 1024)", vec * std::max(nqk, nv));
    if (num_src == 0) return E3B_OK;
    const Split s = split_rows(num_src, num_edges);
    if ((num_edges > 0 && num_dst > 0 && (!q || !grad_out)) || (num_edges > 0 && (!share || !grad_logit || !edge_dst || !src_perm)) || !src_rowptr ||
        !qk_table || !v_table || !grad_k || !grad_v || !scratch || !status)
        return fail(E3B_ERR_ARG, "attention_bwd_src: null pointer");
    if (scratch_bytes < e3b_attention_bwd_src_scratch_bytes(num_src, num_edges, dqk, dv))
        return fail(E3B_ERR_ARG, "attention_bwd_src: scratch of %lld bytes is too small", static_cast<long long>(scratch_bytes));
    SrcArgs a{q, grad_out, q_stride, share, grad_logit, edge_dst, src_perm, grad_k, grad_v, num_dst, scale,
              {qk_table, v_table, heads, nqk, nv, dqk, dv, lanes}, {src_rowptr, num_src, num_edges, s.per_part, s.parts},
              partials_in(scratch, s.parts, dkv_slot(dqk, dv)), status};
    const int groups = static_cast<int>(ceil_div(heads, 32 / lanes));
    const int v_lane = compiled_vectors(vec, static_cast<int>(ceil_div(std::max(nqk, nv), lanes)));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_type_and_vectors(type, vec, v_lane, [&](auto t0, auto vec0, auto v0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(vec0)::value, V = decltype(v0)::value;
        using S = Sums<VEC, V, 2, false>;
        const dim3 grid(static_cast<unsigned>(ceil_div(s.parts, s.warps)), groups);
        int r = E3B_OK;
        if (s.merge) {
            const size_t smem = sizeof(float) * 32 * S::kFloats * s.warps;
            if ((r = allow_smem(attn_bwd_src_kernel<T, VEC, V, true>, smem)) != E3B_OK) return r;
            attn_bwd_src_kernel<T, VEC, V, true><<<grid, 32 * s.warps, smem, st>>>(a);
        } else {
            attn_bwd_src_kernel<T, VEC, V, false><<<grid, 32 * s.warps, 0, st>>>(a);
        }
        if ((r = check_launch("attention_bwd_src")) != E3B_OK || s.parts == 1) return r;
        const size_t smem = s.join_warps > 1 ? sizeof(float) * 32 * S::kFloats * s.join_warps : 0;
        if ((r = allow_smem(attn_bwd_src_join_kernel<T, VEC, V>, smem)) != E3B_OK) return r;
        attn_bwd_src_join_kernel<T, VEC, V><<<dim3(s.parts, groups), 32 * s.join_warps, smem, st>>>(a);
        return check_launch("attention_bwd_src join");
    });
}
