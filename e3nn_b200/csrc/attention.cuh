// What the kernels of the neighbour attention share: how heads lie in a row of irreps features, how the edges of all rows
// are split into equal parts, and how the sums of a row that several parts have worked on are joined.
//
// Heads.  Head h of a row of irreps features owns mul_b / H channels of every block b, so its columns are one run of
// (mul_b / H) d_b elements per block.  A warp gives `lanes` (a power of two) neighbouring lanes to a head and holds
// 32 / lanes heads; a lane owns every lanes-th vector of its head: the products q k of all heads of an edge are reduced together
// by log2(lanes) shuffles, the softmax of all heads runs side by side, and every load instruction covers whole sectors.
// The host's table gives, per vector of a head, {column of head 0, distance between heads}.
//
// Parts.  Rows differ in length (an isolated atom, a hub, one query over a long list), so the unit is not the row: the edges of row
// n followed by one item for its end, row after row, are numbered, item (rowptr[n + 1] + n) being the end of row n, and
// every warp takes `per_part` consecutive items.  A row that lies inside one part is finished there.  Of a longer row each part
// leaves its sums in scratch memory (slot 1: the row goes on in the next part; slot 0: it ended here) and a second
// kernel adds them in the order of the parts.  The split depends on the sizes alone, so results do not depend on scheduling.
#pragma once
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "typed.cuh"

namespace e3b {
namespace {

constexpr unsigned kAll = 0xffffffffu;

// One row space (destinations of the edges, or their sources) and its split.
struct Rows {
    const int64_t* rowptr;   // [num + 1]; values are clamped to [0, edges], rowptr[0] is taken as 0
    int64_t num, edges;
    int64_t per_part;        // items a warp takes
    int parts;
    __device__ __forceinline__ int64_t begin(int64_t n) const { return n == 0 ? 0 : min(max(rowptr[n], int64_t{0}), edges); }
    __device__ __forceinline__ int64_t end(int64_t n) const { return min(max(rowptr[n + 1], int64_t{0}), edges); }
};

// First row whose end lies at item d or later (num: none); 32 probes a step.
__device__ __forceinline__ int64_t find_row(const Rows& r, int64_t d) {
    const int lane = threadIdx.x & 31;
    int64_t lo = 0, hi = r.num;
    while (lo < hi) {
        const int64_t step = (hi - lo + 31) / 32, i = lo + lane * step;
        const unsigned before = __ballot_sync(kAll, i < hi && r.end(i) + i < d);
        const int c = before == kAll ? 32 : __ffs(~before) - 1;
        if (c == 0) break;
        hi = min(hi, lo + c * step);
        lo += (c - 1) * step + 1;
    }
    return lo;
}

// The rows of part p: open(n), edges(first, last), close(n, started here, ended here); rest(first, last) are edge slots behind
// the last row.
template <typename Open, typename Edges, typename Close, typename Rest>
__device__ __forceinline__ void walk_rows(const Rows& r, int part, Open&& open, Edges&& edges, Close&& close, Rest&& rest) {
    int64_t d = part * r.per_part;
    const int64_t d1 = min(d + r.per_part, r.num + r.edges);
    int64_t n = find_row(r, d);
    while (d < d1 && n < r.num) {
        const int64_t first = r.begin(n), last = r.end(n);
        const bool ends = last + n < d1;
        const int64_t e0 = min(max(d - n, first), last), e1 = ends ? last : min(d1 - n, last);
        open(n);
        edges(e0, e1);
        close(n, e0 == first, ends);
        d = max(d + 1, last + n + 1);
        ++n;
    }
    if (n >= r.num && d < d1) rest(d - r.num, d1 - r.num);
}

struct Heads {
    const int32_t* qk;       // [nqk][2], [nv][2] {column of head 0, columns from one head to the next} of each vector
    const int32_t* v;
    int heads, nqk, nv, dqk, dv;
    int lanes;               // of a head
};

// Columns of this lane's vectors (-1: none) and its head.
template <int V>
__device__ __forceinline__ void lane_columns(const int32_t* __restrict__ tbl, int n, int lanes, int head, bool live, int (&col)[V]) {
    const int g = (threadIdx.x & 31) & (lanes - 1);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int i = j * lanes + g;
        col[j] = live && i < n ? tbl[2 * i] + head * tbl[2 * i + 1] : -1;
    }
}

__device__ __forceinline__ float head_sum(float v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
}

// Logit of an edge, with the same roundings in the forward and the backward kernel: a row with one edge has exactly the share 1.
__device__ __forceinline__ float logit(float dot, float scale, float bias, float log_weight) {
    return __fadd_rn(__fmaf_rn(dot, scale, bias), log_weight);
}

// What the attention reads per edge.
struct Edges {
    const int64_t* perm;        // slot -> edge, or null: the same
    const int64_t* src;         // row of k and v, or null: the edge itself
    const float* bias;          // [edges, heads], or the table [num_buckets, heads] if buckets is given, or null
    const int32_t* buckets;
    const float* weight;        // [edges] or null
    int num_buckets;
    int64_t num_src, edges;
    int32_t* status;
};

// The 32 slots from `base` on, one a lane: edge, row of k and v (-1: the edge is left out), bucket, logarithm of the weight.
struct EdgeMeta {
    int edge, row, bucket;
    float log_weight;
    __device__ __forceinline__ void load(const Edges& a, int64_t slot, int64_t last) {
        edge = row = -1;
        bucket = 0;
        log_weight = 0.0f;
        if (slot >= last) return;
        const int64_t e = a.perm ? a.perm[slot] : slot;
        if (e < 0 || e >= a.edges) {
            *a.status = 2;
            return;
        }
        edge = static_cast<int>(e);
        const int64_t n = a.src ? a.src[edge] : e;
        row = static_cast<int>(n);
        if (n < 0 || n >= a.num_src) {
            *a.status = 2;
            row = -1;
        }
        if (a.buckets) {
            bucket = a.buckets[edge];
            if (bucket < 0 || bucket >= a.num_buckets) {
                *a.status = 2;
                row = -1;
                bucket = 0;
            }
        }
        if (a.weight) {
            const float w = a.weight[edge];
            if (w <= 0.0f) row = -1;
            else log_weight = logf(w);
        }
    }
};

// Edges loaded together: their two rows of V vectors of `words` registers each fill at most `budget` registers.
__host__ __device__ constexpr int edges_in_flight(int v, int words, int budget) {
    const int n = budget / (2 * v * words);
    return n >= 8 ? 8 : n >= 4 ? 4 : n >= 2 ? 2 : 1;
}
template <typename T, int VEC> __host__ __device__ constexpr int words_of() { return VEC == 1 ? 1 : VEC * static_cast<int>(sizeof(T)) / 4; }

template <typename T, int VEC, int V>
__device__ __forceinline__ void load_row(Packed<T, VEC> (&p)[V], const T* __restrict__ base, int64_t row, int64_t stride, const int (&col)[V], bool use) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (use && col[j] >= 0) p[j].load(base + row * stride + col[j]);
        else p[j].zero();
    }
}
template <typename T, int VEC, int V>
__device__ __forceinline__ void load_row_f(float (&f)[V][VEC], const T* __restrict__ base, int64_t row, int64_t stride, const int (&col)[V]) {
    Packed<T, VEC> p[V];
    load_row<T, VEC, V>(p, base, row, stride, col, true);
#pragma unroll
    for (int j = 0; j < V; ++j) p[j].unpack(f[j]);
}
template <typename T, int VEC, int V>
__device__ __forceinline__ void store_row(T* __restrict__ base, int64_t row, int64_t stride, const int (&col)[V], const float (&f)[V][VEC], float by) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (col[j] < 0) continue;
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = f[j][i] * by;
        Packed<T, VEC>::store(base + row * stride + col[j], o);
    }
}

// ---------------------------------------------------------------------------------------------- sums shared by several parts
// Scratch memory: per part two slots of `slot` floats (slot 1: the row goes on, slot 0: it ended here), the row that ended here
// (-1: none) and whether slot 1 holds anything.
struct Partials {
    float* sums;
    int32_t* ended;      // [parts]
    int32_t* goes_on;    // [parts]
    int slot;
    __device__ __forceinline__ float* at(int part, int which) const { return sums + (static_cast<int64_t>(part) * 2 + which) * slot; }
};

inline int64_t partial_floats(int parts, int slot) { return static_cast<int64_t>(parts) * 2 * slot; }
inline int64_t partial_bytes(int parts, int slot) { return 4 * (partial_floats(parts, slot) + 2 * static_cast<int64_t>(parts) + 8); }
inline Partials partials_in(void* scratch, int parts, int slot) {
    float* sums = static_cast<float*>(scratch);
    int32_t* ints = reinterpret_cast<int32_t*>(sums + partial_floats(parts, slot));
    return {sums, ints, ints + parts, slot};
}

// The running sums of a row: NA accumulators (0: over the columns of q and k, 1: over those of v) and, in the softmax, the
// maximum and the sum of each head.
template <int VEC, int V, int NA, bool SOFTMAX>
struct Sums {
    float a[NA][V][VEC];
    float m, l;
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int n = 0; n < NA; ++n)
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) a[n][j][i] = 0.0f;
    }
    // this * own + other * theirs, the factors bringing both to the common maximum
    __device__ __forceinline__ void factors(float om, float ol, float* own, float* theirs) {
        *own = *theirs = 1.0f;
        if (!SOFTMAX) return;
        const float top = fmaxf(m, om), base = top == -INFINITY ? 0.0f : top;
        *own = __expf(m - base);
        *theirs = __expf(om - base);
        l = l * *own + ol * *theirs;
        m = (m != m || om != om) ? NAN : top;      // (fmaxf drops a NaN)
    }
    __device__ __forceinline__ void save(float* p, const Heads& h, const int (&cq)[V], const int (&cv)[V], int head, bool leads) const {
        const int base1 = NA == 2 ? h.dqk : 0;
#pragma unroll
        for (int n = 0; n < NA; ++n) {
            const bool over_v = NA == 2 ? n == 1 : SOFTMAX;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int c = over_v ? cv[j] : cq[j];
                if (c >= 0) Packed<float, VEC>::store(p + (n == 1 ? base1 : 0) + c, a[n][j]);
            }
        }
        if (SOFTMAX && leads) {
            p[h.dv + head] = m;
            p[h.dv + h.heads + head] = l;
        }
    }
    __device__ __forceinline__ void add(const float* p, const Heads& h, const int (&cq)[V], const int (&cv)[V], int head, bool live) {
        const int base1 = NA == 2 ? h.dqk : 0;
        float own = 1.0f, theirs = 1.0f;
        if (SOFTMAX) factors(live ? p[h.dv + head] : -INFINITY, live ? p[h.dv + h.heads + head] : 0.0f, &own, &theirs);
#pragma unroll
        for (int n = 0; n < NA; ++n) {
            const bool over_v = NA == 2 ? n == 1 : SOFTMAX;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int c = over_v ? cv[j] : cq[j];
                if (c < 0) continue;
                Packed<float, VEC> x;
                float f[VEC];
                x.load(p + (n == 1 ? base1 : 0) + c);
                x.unpack(f);
#pragma unroll
                for (int i = 0; i < VEC; ++i) a[n][j][i] = SOFTMAX ? fmaf(f[i], theirs, a[n][j][i] * own) : a[n][j][i] + f[i];
            }
        }
    }
    static constexpr int kFloats = NA * V * VEC + 2;     // a lane's share in shared memory
    __device__ __forceinline__ void put(float* lane0) const {
        float* p = lane0 + (threadIdx.x & 31);
#pragma unroll
        for (int n = 0; n < NA; ++n)
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) p[32 * ((n * V + j) * VEC + i)] = a[n][j][i];
        p[32 * (kFloats - 2)] = m;
        p[32 * (kFloats - 1)] = l;
    }
    __device__ __forceinline__ void take(const float* lane0) {
        const float* p = lane0 + (threadIdx.x & 31);
        float own, theirs;
        factors(p[32 * (kFloats - 2)], p[32 * (kFloats - 1)], &own, &theirs);
#pragma unroll
        for (int n = 0; n < NA; ++n)
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float f = p[32 * ((n * V + j) * VEC + i)];
                    a[n][j][i] = SOFTMAX ? fmaf(f, theirs, a[n][j][i] * own) : a[n][j][i] + f;
                }
    }
};

// The end of a part: `sums` are those of the row that goes on (row, -1: none).  Where all warps of the block are inside one
// row (MERGE: long rows only) their sums are added up here, in the order of the warps, and the first keeps them.
template <bool MERGE, typename S, int V>
__device__ __forceinline__ void leave_part(S& sums, int64_t row, int part, int parts, const Partials& out, const Heads& h, const int (&cq)[V],
                                           const int (&cv)[V], int head, bool leads, float* smem) {
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    bool keeps = row >= 0;
    if (MERGE) {
        __shared__ int64_t row_of[32];
        if ((threadIdx.x & 31) == 0) row_of[warp] = row;
        __syncthreads();
        bool same = row_of[0] >= 0;
        for (int w = 1; w < warps; ++w) same = same && row_of[w] == row_of[0];
        if (same) {
            if (warp > 0) sums.put(smem + warp * 32 * S::kFloats);
            __syncthreads();
            if (warp == 0)
                for (int w = 1; w < warps; ++w) sums.take(smem + w * 32 * S::kFloats);
            keeps = warp == 0;
        }
    }
    if (part >= parts) return;
    if (keeps) sums.save(out.at(part, 1), h, cq, cv, head, leads);
    if (blockIdx.y == 0 && (threadIdx.x & 31) == 0) out.goes_on[part] = keeps ? 1 : 0;
}

// Sums of the row that ended in part p with slots of earlier parts: slot 1 of the parts from the row's first on, then slot 0 of
// p.  The warps of the block take 32 parts each in turn and are added in order.  False: nothing to do, or not the warp that goes on.
template <typename S, int V>
__device__ __forceinline__ bool join_parts(S& sums, const Rows& r, int part, const Partials& in, const Heads& h, const int (&cq)[V],
                                           const int (&cv)[V], int head, bool live, float* smem, int64_t* row) {
    const int64_t n = in.ended[part];
    if (n < 0) return false;
    *row = n;
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    const int from = static_cast<int>((r.begin(n) + n) / r.per_part);
    sums.clear();
    for (int p0 = from + warp * 32; p0 < part; p0 += warps * 32) {
        unsigned held = __ballot_sync(kAll, p0 + lane < part && in.goes_on[p0 + lane] != 0);
        while (held) {
            const int i = __ffs(held) - 1;
            held &= held - 1;
            sums.add(in.at(p0 + i, 1), h, cq, cv, head, live);
        }
    }
    if (warps > 1) {
        if (warp > 0) sums.put(smem + warp * 32 * S::kFloats);
        __syncthreads();
        if (warp > 0) return false;
        for (int w = 1; w < warps; ++w) sums.take(smem + w * 32 * S::kFloats);
    }
    sums.add(in.at(part, 0), h, cq, cv, head, live);
    return true;
}

// ------------------------------------------------------------------------------------------------------------- host side
struct Split {
    int64_t per_part;
    int parts, warps;       // of a block
    bool merge;             // rows are longer than a block's parts
    int join_warps;
};

// About four waves of warps; at least 32 items a part (a part costs a search for its row and up to two slots).
inline Split split_rows(int64_t num, int64_t edges) {
    Split s;
    const int64_t items = std::max<int64_t>(num + edges, 1);
    s.per_part = std::min<int64_t>(256, std::max<int64_t>(32, ceil_div(items, static_cast<int64_t>(kNumSMs) * 16 * 4)));
    s.parts = static_cast<int>(ceil_div(items, s.per_part));
    s.warps = s.parts >= kNumSMs * 8 ? 8 : 2;
    const int64_t longest = num > 0 ? edges / num : 0;
    s.merge = longest > s.per_part * s.warps;
    s.join_warps = longest > 4 * s.per_part ? 8 : 1;
    return s;
}

// Lanes a head gets and vectors a lane then owns; 0: the head is too wide.
inline int lanes_of_head(int heads, int vectors, int most) {
    int lanes = 32;
    while (lanes > 1 && 32 / lanes < heads && vectors <= (lanes / 2) * most) lanes /= 2;
    return vectors <= lanes * most ? lanes : 0;
}

struct Launch {
    Heads h;
    Rows r;
    Split s;
    int vec, v, groups;     // vector width, vectors a lane, head groups (grid.y)
};

// Vectors a lane that are compiled: the next one up is taken.
inline int compiled_vectors(int vec, int v) {
    if (vec == 4) return v <= 6 ? v : 8;
    return v <= 4 ? 4 : v <= 8 ? 8 : v <= 16 ? 16 : 32;
}

template <typename T, typename F>
int by_vectors(int vec, int v, F&& f) {
    if (vec == 4) {
        switch (v) {
            case 1: return f(T(), Int<4>(), Int<1>());
            case 2: return f(T(), Int<4>(), Int<2>());
            case 3: return f(T(), Int<4>(), Int<3>());
            case 4: return f(T(), Int<4>(), Int<4>());
            case 5: return f(T(), Int<4>(), Int<5>());
            case 6: return f(T(), Int<4>(), Int<6>());
            default: return f(T(), Int<4>(), Int<8>());
        }
    }
    switch (v) {
        case 4: return f(T(), Int<1>(), Int<4>());
        case 8: return f(T(), Int<1>(), Int<8>());
        case 16: return f(T(), Int<1>(), Int<16>());
        default: return f(T(), Int<1>(), Int<32>());
    }
}
template <typename F>
int by_type_and_vectors(int type, int vec, int v, F&& f) {
    if (type == kFloat32) return by_vectors<float>(vec, v, f);
    if (type == kBFloat16) return by_vectors<__nv_bfloat16>(vec, v, f);
    return by_vectors<__half>(vec, v, f);
}

template <typename K>
int allow_smem(K kernel, size_t smem) {
    if (smem > 48 * 1024) E3B_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    return E3B_OK;
}

}  // namespace
}  // namespace e3b
