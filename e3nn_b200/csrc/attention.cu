// Attention over the incoming edges of every node, forward.
//
//   a[e, h] = scale <q[dst], k[src]>_h + bias[e, h] + log weight[e]
//   out[n]_h = sum_e softmax_e(a[e, h]) v[src]_h           over the edges e of row n; a row without edges is zero
//
// One pass: the maximum and the sum of a row run along with the sum of the values.  k and v are rows of nodes (gathered by src) or of
// edges.  An edge moves (dqk + dv) elements from L2 or HBM and costs 2 (dqk + dv) operations.  All edges of a row share its q, but each has a
// row of k and of v of its own, gathered for a few operations an element, so these run on the FP32 pipe.  What counts is bytes in flight in
// fp32; in 16 bits latency at 12 to 16 warps an SM (42 to 45 % of the issue slots are used) and reads of the ring: a row of 1,024 columns in
// bf16 and 8 heads takes 36 shared-memory wavefronts where 16 are the least, one of 576 in fp32 36 for 18.
// Layout of heads, ring, split into parts and their joining: attention.cuh.  Logits, statistics and sums are fp32; the output is
// rounded once.  2,097,152 edges over 65,536 nodes, 576 columns, 8 heads: fp32 1,126 us = 8.6 TB/s of gathered rows (302 MB of k and v, L2
// holds 126 MB), bf16 890 us; 425,984 edges of 1,024 columns in bf16 265 us = 6.6 TB/s; one query over 50,021 edges of 576 columns in bf16
// 33 us and 22 us for the join, in fp32 55 and 26 us.
#include "attention.cuh"

namespace e3b {
namespace {

struct FwdArgs {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    void* out;               // [rows, dv]
    float* out32;            // the same in fp32, or null (kept for the gradient of 16-bit types)
    float* stats;            // [rows, heads, 2] maximum and reciprocal of the sum, or null
    float scale;
    Heads h;
    Edges e;
    Rows r;
    Partials p;
    bool merge;
    RingSource ring;
    int depth;
    uint32_t warp_smem;
};

template <typename T, int VEC, int V>
__device__ __forceinline__ void finish_row(const FwdArgs& a, const Sums<VEC, V, 1, true>& s, int64_t n, const int (&cv)[V], int head, bool leads) {
    const float inv = s.l == 0.0f ? 0.0f : 1.0f / s.l;      // (NaN stays NaN)
    store_row<T, VEC, V>(static_cast<T*>(a.out), n, a.h.dv, cv, s.a[0], inv);
    if (a.out32) store_row<float, VEC, V>(a.out32, n, a.h.dv, cv, s.a[0], inv);
    if (a.stats && leads) {
        a.stats[(n * a.h.heads + head) * 2] = s.m == -INFINITY ? 0.0f : s.m;
        a.stats[(n * a.h.heads + head) * 2 + 1] = inv;
    }
}

// Rows by loads into registers, for rows that cannot be copied in units of 16 bytes and for heads of several warps: the k and v rows of
// several edges (about 80 registers) are under way before the first is used.  425,984 edges of 576 columns on 16 heads (four channels a head)
// in bf16 507 us where the ring takes 192 us for twice the bytes in fp32: latency.
template <typename T, int VEC, int V>
__global__ void __launch_bounds__(256) attn_fwd_kernel(const FwdArgs a) {
    extern __shared__ float smem[];
    constexpr int U = edges_in_flight(V, words_of<T, VEC>(), 80);
    const int lane = threadIdx.x & 31, part = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int head = blockIdx.y * (32 / a.h.lanes) + lane / a.h.lanes;
    const bool live = head < a.h.heads, leads = live && (lane & (a.h.lanes - 1)) == 0;
    int cq[V], cv[V];
    lane_columns<V>(a.h.qk, a.h.nqk, a.h.lanes, head, live, cq);
    lane_columns<V>(a.h.v, a.h.nv, a.h.lanes, head, live, cv);
    const T* q = static_cast<const T*>(a.q);
    const T* k = static_cast<const T*>(a.k);
    const T* v = static_cast<const T*>(a.v);
    Sums<VEC, V, 1, true> s;
    s.clear();
    int64_t goes_on = -1;
    int ended = -1;
    if (part < a.r.parts) {
        float qf[V][VEC];
        const Part range = find_part(a.r, part);
        walk_rows(
            a.r, range,
            [&](int64_t n) {
                load_row_f<T, VEC, V>(qf, q, n, a.q_stride, cq);
                s.clear();
            },
            [&](int64_t first, int64_t last) {
                for (int64_t base = first; base < last; base += 32) {
                    EdgeMeta meta;
                    meta.load(a.e, base + lane, last);
                    const int count = static_cast<int>(min(last - base, int64_t{32}));
                    for (int u0 = 0; u0 < count; u0 += U) {
                        Packed<T, VEC> kk[U][V], vv[U][V];
                        float bias[U], dot[U];
                        bool use[U];
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            const int row = __shfl_sync(kAll, meta.row, u0 + u);
                            use[u] = row >= 0;
                            bias[u] = 0.0f;
                            if (a.e.buckets) {
                                const int b = __shfl_sync(kAll, meta.bucket, u0 + u);
                                if (live) bias[u] = a.e.bias[b * a.h.heads + head];
                            } else if (a.e.bias) {
                                const int e = __shfl_sync(kAll, meta.edge, u0 + u);
                                if (live && e >= 0) bias[u] = a.e.bias[static_cast<int64_t>(e) * a.h.heads + head];
                                use[u] = use[u] && bias[u] != -INFINITY;      // masked: whatever k and v hold there
                            }
                            load_row<T, VEC, V>(kk[u], k, row, a.k_stride, cq, use[u]);
                            load_row<T, VEC, V>(vv[u], v, row, a.v_stride, cv, use[u]);
                        }
                        float top = s.m;
                        bool nan = false;
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            float d = 0.0f;
#pragma unroll
                            for (int j = 0; j < V; ++j) {
                                float f[VEC];
                                kk[u][j].unpack(f);
#pragma unroll
                                for (int i = 0; i < VEC; ++i) d = fmaf(qf[j][i], f[i], d);
                            }
                            dot[u] = logit(head_sum(d, a.h.lanes), a.scale, bias[u], a.e.weight ? __shfl_sync(kAll, meta.log_weight, u0 + u) : 0.0f);
                            if (!use[u]) dot[u] = -INFINITY;
                            nan = nan || dot[u] != dot[u];
                            top = fmaxf(top, dot[u]);
                        }
                        if (nan) top = NAN;
                        const float ref = top == -INFINITY ? 0.0f : top;
                        const float keep = __expf(s.m - ref);
                        s.m = top;
                        s.l *= keep;
#pragma unroll
                        for (int j = 0; j < V; ++j)
#pragma unroll
                            for (int i = 0; i < VEC; ++i) s.a[0][j][i] *= keep;
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            const float w = __expf(dot[u] - ref);
                            if (w == 0.0f) continue;      // as in the ring: it adds nothing, whatever v holds
                            s.l += w;
#pragma unroll
                            for (int j = 0; j < V; ++j) {
                                float f[VEC];
                                vv[u][j].unpack(f);
#pragma unroll
                                for (int i = 0; i < VEC; ++i) s.a[0][j][i] = fmaf(w, f[i], s.a[0][j][i]);
                            }
                        }
                    }
                }
            },
            [&](int64_t n, bool started, bool ends) {
                if (!ends) {
                    goes_on = n;
                } else if (started) {
                    finish_row<T, VEC, V>(a, s, n, cv, head, leads);
                } else {
                    s.save(a.p.at(part, 0), a.h, cq, cv, head, leads);
                    ended = static_cast<int>(n);
                }
            });
        if (blockIdx.y == 0 && lane == 0) a.p.ended[part] = ended;
    }
    leave_part(a.merge, s, goes_on, part, a.r.parts, a.p, a.h, cq, cv, head, leads, smem);
}

// The same with k and v through the ring: the registers hold q, the sums and the row in hand, so more warps fit and all copies that
// fit in shared memory are under way (about 200 KB an SM).
template <typename T, int VEC, int V>
__global__ void __launch_bounds__(512, 1) attn_fwd_ring_kernel(const FwdArgs a) {
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
    Sums<VEC, V, 1, true> s;
    s.clear();
    int64_t goes_on = -1;
    int ended = -1;
    if (part < a.r.parts) {
        const Part range = find_part(a.r, part);
        Ring<U, EdgeMeta> ring(a.ring, memory + warp * a.warp_smem, a.depth);
        float qf[V][VEC], bias[U];
        bool use[U];
        walk_ring(
            a.r, range, ring, a.e.status, [&](EdgeMeta& m, int i) { m.load(a.e, range.e0 + i, range.behind); },
            [&](int64_t n) {
                load_row_f<T, VEC, V>(qf, static_cast<const T*>(a.q), n, a.q_stride, cq);
                s.clear();
            },
            [&](const EdgeMeta& meta, int at, int m) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int from = (at + u) & 31;
                    use[u] = u < m && __shfl_sync(kAll, meta.row, from) >= 0;
                    bias[u] = 0.0f;
                    if (a.e.buckets) {
                        const int b = __shfl_sync(kAll, meta.bucket, from);
                        if (live) bias[u] = a.e.bias[b * a.h.heads + head];
                    } else if (a.e.bias) {
                        const int e = __shfl_sync(kAll, meta.edge, from);
                        if (live && use[u]) bias[u] = a.e.bias[static_cast<int64_t>(e) * a.h.heads + head];
                        use[u] = use[u] && bias[u] != -INFINITY;      // masked: whatever k and v hold there
                    }
                }
            },
            [&](const uint8_t* const (&slot)[U], const EdgeMeta& meta, int at, int m) {
                float x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) x[u] = dot_row<T, VEC, V>(slot[u], qf, pq);
                head_sums<U>(x, a.h.lanes);
                float top = s.m;
                bool nan = false;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    x[u] = logit(x[u], a.scale, bias[u], a.e.weight ? __shfl_sync(kAll, meta.log_weight, (at + u) & 31) : 0.0f);
                    if (!use[u]) x[u] = -INFINITY;
                    nan = nan || x[u] != x[u];
                    top = fmaxf(top, x[u]);
                }
                if (nan) top = NAN;
                if (top != s.m) {         // a new maximum: rare after the first edges of a row
                    const float keep = __expf(s.m - (top == -INFINITY ? 0.0f : top));
                    s.m = top;
                    s.l *= keep;
#pragma unroll
                    for (int j = 0; j < V; ++j)
#pragma unroll
                        for (int i = 0; i < VEC; ++i) s.a[0][j][i] *= keep;
                }
                const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float w = __expf(x[u] - ref);
                    if (w == 0.0f) continue;      // left out, or too small to count: its slot may hold anything
                    s.l += w;
                    add_row<T, VEC, V>(slot[u], w, s.a[0], pv);
                }
            },
            [&](int64_t n, bool started, bool ends) {
                if (!ends) {
                    goes_on = n;
                } else if (started) {
                    finish_row<T, VEC, V>(a, s, n, cv, head, leads);
                } else {
                    s.save(a.p.at(part, 0), a.h, cq, cv, head, leads);
                    ended = static_cast<int>(n);
                }
            });
        if (lane == 0) a.p.ended[part] = ended;
    }
    leave_part(a.merge, s, goes_on, part, a.r.parts, a.p, a.h, cq, cv, head, leads, reinterpret_cast<float*>(memory));
}

template <typename T, int VEC, int V>
__global__ void __launch_bounds__(512) attn_fwd_join_kernel(const FwdArgs a) {
    extern __shared__ float smem[];
    const int lane = threadIdx.x & 31;
    const int head = blockIdx.y * (32 / a.h.lanes) + lane / a.h.lanes;
    const bool live = head < a.h.heads, leads = live && (lane & (a.h.lanes - 1)) == 0;
    int cv[V];
    lane_columns<V>(a.h.v, a.h.nv, a.h.lanes, head, live, cv);
    Sums<VEC, V, 1, true> s;
    int64_t n;
    if (join_parts(s, a.r, blockIdx.x, a.p, a.h, cv, cv, head, live, smem, &n)) finish_row<T, VEC, V>(a, s, n, cv, head, leads);
}

int fwd_slot(int heads, int dv) { return static_cast<int>(ceil_div(dv + 2 * heads, 4) * 4); }

}  // namespace
}  // namespace e3b

using namespace e3b;

extern "C" int64_t e3b_attention_scratch_bytes(int64_t num_dst, int64_t num_edges, int num_heads, int dim_v) {
    if (num_dst < 0 || num_edges < 0) return 0;
    return partial_bytes(most_parts(num_dst, num_edges), fwd_slot(num_heads, dim_v));
}

extern "C" int e3b_attention_fwd(const void* q, const void* k, const void* v, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                 const int64_t* rowptr, const int64_t* perm, const int64_t* edge_src, const float* bias,
                                 const int32_t* buckets, int num_buckets, const float* edge_weight, const int32_t* qk_table,
                                 const int32_t* v_table, const int32_t* layout, float scale, int64_t num_dst, int64_t num_src,
                                 int64_t num_edges, int type, void* out, float* out32, float* stats, void* scratch,
                                 int64_t scratch_bytes, int32_t* status, void* stream) {
    if (!layout || num_dst < 0 || num_src < 0 || num_edges < 0 || num_edges >= INT32_MAX || num_dst >= INT32_MAX || num_src >= INT32_MAX || !known_type(type))
        return fail(E3B_ERR_ARG, "attention_fwd: bad size or type");
    const int vec = layout[0], heads = layout[1], nqk = layout[2], nv = layout[3], dqk = layout[4], dv = layout[5];
    if (num_dst == 0) return E3B_OK;
    if (heads < 1 || (vec != 1 && vec != 4 && (vec != 8 || type == kFloat32))) return fail(E3B_ERR_ARG, "attention_fwd: bad head layout");
    if (buckets && num_buckets < 1) return fail(E3B_ERR_ARG, "attention_fwd: an empty table of biases");      // (the kernels read its first row in the place of a bad one)
    if (buckets && static_cast<int64_t>(num_buckets) * heads > INT32_MAX - 32)
        return fail(E3B_ERR_UNSUPPORTED, "attention_fwd: a table of %d buckets and %d heads", num_buckets, heads);
    if (!q || !rowptr || (num_edges > 0 && num_src > 0 && (!k || !v)) || !qk_table || !v_table || !out || !scratch || !status || (buckets && !bias))
        return fail(E3B_ERR_ARG, "attention_fwd: null pointer");
    const int size = element_size(type);
    const RingSource rows{static_cast<const char*>(k), static_cast<const char*>(v), nullptr, k_stride * size, v_stride * size,
                          static_cast<uint32_t>(dqk * size), static_cast<uint32_t>(dv * size), 0};
    Plan p;
    const int planned = plan(&p, "attention_fwd", type, vec, heads, std::max(nqk, nv), num_dst, num_edges, rows, 4, 3, true);
    if (planned != E3B_OK) return planned;
    if (scratch_bytes < e3b_attention_scratch_bytes(num_dst, num_edges, heads, dv))
        return fail(E3B_ERR_ARG, "attention_fwd: scratch of %lld bytes is too small", static_cast<long long>(scratch_bytes));
    const Split& s = p.s;
    FwdArgs a{q, k, v, q_stride, k_stride, v_stride, out, out32, stats, scale, {qk_table, v_table, heads, nqk, nv, dqk, dv, p.lanes},
              {perm, edge_src, bias, buckets, edge_weight, num_buckets, num_src, num_edges, status},
              {rowptr, num_dst, num_edges, s.per_part, s.parts}, partials_in(scratch, s.parts, fwd_slot(heads, dv)), s.merge, rows, p.depth,
              static_cast<uint32_t>(p.warp_smem)};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_type_and_vectors(type, vec, p.v, [&](auto t0, auto vec0, auto v0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(vec0)::value, V = decltype(v0)::value;
        using S = Sums<VEC, V, 1, true>;
        const unsigned blocks = static_cast<unsigned>(ceil_div(s.parts, s.warps));
        const size_t merge_smem = s.merge ? sizeof(float) * 32 * S::kFloats * s.warps : 0;
        int rc = E3B_OK;
        if constexpr (VEC * sizeof(T) == 16) {
            if (p.ring) {
                const size_t smem = std::max(p.warp_smem * s.warps, merge_smem);
                if ((rc = allow_smem(attn_fwd_ring_kernel<T, VEC, V>, smem)) != E3B_OK) return rc;
                attn_fwd_ring_kernel<T, VEC, V><<<blocks, 32 * s.warps, smem, st>>>(a);
            }
        }
        if (!p.ring) {
            if ((rc = allow_smem(attn_fwd_kernel<T, VEC, V>, merge_smem)) != E3B_OK) return rc;
            attn_fwd_kernel<T, VEC, V><<<dim3(blocks, p.groups), 32 * s.warps, merge_smem, st>>>(a);
        }
        if ((rc = check_launch("attention_fwd")) != E3B_OK || s.parts == 1) return rc;
        const size_t smem = s.join_warps > 1 ? sizeof(float) * 32 * S::kFloats * s.join_warps : 0;
        if ((rc = allow_smem(attn_fwd_join_kernel<T, VEC, V>, smem)) != E3B_OK) return rc;
        attn_fwd_join_kernel<T, VEC, V><<<dim3(s.parts, p.groups), 32 * s.join_warps, smem, st>>>(a);
        return check_launch("attention_fwd join");
    });
}
