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
// n followed by one item for its end, row after row, are numbered (slots in front of the first row with it), item (rowptr[n + 1] + n) being the end of row n, and
// every warp takes `per_part` consecutive items.  A row that lies inside one part is finished there.  Of a longer row each part
// leaves its sums in scratch memory (slot 1: the row goes on in the next part; slot 0: it ended here) and a second
// kernel adds them in the order of the parts.  The split depends on the sizes alone, so results do not depend on scheduling.  How many warps
// join a row, and whether a block first adds its own parts, goes by the mean length: a row far longer than the mean is joined by one warp, a part
// after another (65,535 rows of 8 edges and one of 65,536, 576 columns in fp32: 382 us, and 397 us for that join).
#pragma once
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "tc_common.cuh"
#include "typed.cuh"

namespace e3b {
namespace {

constexpr unsigned kAll = 0xffffffffu;

// One row space (destinations of the edges, or their sources) and its split.
struct Rows {
    const int64_t* rowptr;   // [num + 1]; values are clamped to [0, edges]
    int64_t num, edges;
    int64_t per_part;        // items a warp takes
    int parts;
    __device__ __forceinline__ int64_t begin(int64_t n) const { return min(max(rowptr[n], int64_t{0}), edges); }
    __device__ __forceinline__ int64_t end(int64_t n) const { return min(max(rowptr[n + 1], int64_t{0}), edges); }
};

// The slots and rows of one part: rows n0 .. n1 - 1 end in it, row n1 (if there is one) goes on; slots first .. e1 - 1, of which those
// before e0 lie in front of the first row (a row pointer may start anywhere: a range of rows of a larger graph) and those from
// `behind` on behind the last.
struct Part {
    int64_t n0, n1, first, e0, e1, behind;
};

// First rows whose end lies at item d0 or later, and at d1 or later (num: none).  Half a warp looks for each, 16 probes a step.
__device__ __forceinline__ Part find_part(const Rows& r, int part) {
    const int lane = threadIdx.x & 31, probe = lane & 15;
    const int64_t d0 = part * r.per_part, d1 = min(d0 + r.per_part, r.num + r.edges), d = lane < 16 ? d0 : d1;
    int64_t lo = 0, hi = r.num;
    while (__any_sync(kAll, lo < hi)) {
        const int64_t step = max((hi - lo + 15) / 16, int64_t{1}), i = lo + probe * step;
        const unsigned before = (__ballot_sync(kAll, i < hi && r.end(i) + i < d) >> (lane & 16)) & 0xffffu;
        const int c = __ffs(~before) - 1;           // probes in front of the row (16: all)
        hi = c == 0 ? lo : min(hi, lo + c * step);
        if (c > 0) lo += (c - 1) * step + 1;
    }
    Part p;
    p.n0 = __shfl_sync(kAll, lo, 0);
    p.n1 = max(__shfl_sync(kAll, lo, 16), p.n0);
    p.first = min(max(d0 - p.n0, int64_t{0}), r.edges);
    p.e1 = min(max(d1 - p.n1, p.first), r.edges);
    p.e0 = r.num > 0 && p.n0 == 0 ? min(max(p.first, r.begin(0)), p.e1) : p.first;
    p.behind = p.n1 < r.num ? p.e1 : min(max(r.num > 0 ? r.end(r.num - 1) : 0, p.e0), p.e1);
    return p;
}

// The rows of a part in order: open(n), edges(first, last), close(n, started here, ended here).
template <typename Open, typename Edges, typename Close>
__device__ __forceinline__ void walk_rows(const Rows& r, const Part& p, Open&& open, Edges&& edges, Close&& close) {
    int64_t s = p.e0;
    for (int64_t n = p.n0; n < r.num && (n < p.n1 || s < p.behind); ++n) {
        const bool ends = n < p.n1, started = n > p.n0 || r.begin(n) == p.e0;
        const int64_t last = ends ? min(max(r.end(n), s), p.behind) : p.behind;
        open(n);
        edges(s, last);
        s = last;
        close(n, started, ends);
        if (!ends) break;
    }
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
// SHARE: a factor of zero gives zeros, whatever the row holds.
template <typename T, int VEC, int V, bool SHARE = false>
__device__ __forceinline__ void store_row(T* __restrict__ base, int64_t row, int64_t stride, const int (&col)[V], const float (&f)[V][VEC], float by) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (col[j] < 0) continue;
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = SHARE && by == 0.0f ? 0.0f : f[j][i] * by;
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
// row (looked for where rows are long) their sums are added up here, in the order of the warps, and the first keeps them.
template <typename S, int V>
__device__ __forceinline__ void leave_part(bool merge, S& sums, int64_t row, int part, int parts, const Partials& out, const Heads& h, const int (&cq)[V],
                                           const int (&cv)[V], int head, bool leads, float* smem) {
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    bool keeps = row >= 0;
    if (merge) {
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

// ------------------------------------------------------------------------------------------------- rows through shared memory
// The two rows of every edge arrive by bulk copies (cp.async.bulk) in a ring of `depth` slots that belongs to one warp: one copy
// instruction a row, issued by the lane that holds the edge's number, no registers and no address arithmetic of the other lanes
// while it is under way.  The ring runs ahead over the ends of rows; a slot is refilled as soon as its edges have been used.
// Every wait is bounded: one that gives up reports status 3, waits (bounded again) for the copies under way and ends the part.
struct RingSource {
    const char *a, *b, *c;               // rows by EdgeMeta::row (a, b) and by EdgeMeta::edge (c, may be null)
    int64_t a_stride, b_stride;          // bytes
    uint32_t a_bytes, b_bytes, c_bytes;  // of a row, multiples of 16
    __host__ __device__ uint32_t zeros() const { return a_bytes + b_bytes + c_bytes; }      // a slot ends with 16 bytes of zeros (and no padding: it would cost a slot of wide rows)
    __host__ __device__ uint32_t slot() const { return zeros() + 16; }
};

__device__ __forceinline__ void bulk_copy(void* smem, const void* global, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc::smem_u32(smem)),
                 "l"(__cvta_generic_to_global(global)), "r"(bytes), "r"(tc::smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t parity) {
    for (uint32_t it = 0; it < 400000u; ++it) {
        if (tc::mbar_try_wait(bar, parity)) return true;
        if ((it & 63u) == 63u) __nanosleep(64);
    }
    return false;
}

// Edges used together.  (Four everywhere: 5 to 15 % slower on rows of 26 to 32 edges of 576 and 1,024 columns, whose last group is
// then half empty and whose ring holds few more.)
__host__ __device__ constexpr int edges_together(int columns) { return columns <= 12 ? 4 : 2; }

template <int U, typename Meta>
struct Ring {
    const RingSource src;
    uint8_t* smem;
    uint64_t* full;
    int depth, total;             // slots; edges of the part
    int used, issued;             // edges handed out, edges under way or there
    int used_at, issued_at;       // their slots
    uint32_t parity;              // of the slots from used_at on
    Meta now, next;               // 32 edges each: those of the batch that is being used, and of the one after it

    __device__ __forceinline__ Ring(const RingSource& source, uint8_t* memory, int slots) : src(source), smem(memory), depth(slots) {
        full = reinterpret_cast<uint64_t*>(memory + static_cast<size_t>(slots) * source.slot());
        const int lane = threadIdx.x & 31;
        for (int i = lane; i < depth; i += 32) {
            tc::mbar_init(&full[i], 1);
            *reinterpret_cast<uint4*>(memory + static_cast<uint32_t>(i) * source.slot() + source.zeros()) = make_uint4(0u, 0u, 0u, 0u);
        }
        tc::mbar_init_fence();
        __syncwarp();
    }
    // copies of the next m edges (one lane each)
    __device__ __forceinline__ void issue(int m) {
        const int lane = threadIdx.x & 31, t = (lane - issued) & 31, i = issued + t;
        m = min(m, total - issued);
        if (t < m) {
            const bool same = (i >> 5) == (used >> 5);
            const int64_t row = same ? now.row : next.row, edge = same ? now.edge : next.edge;
            int at = issued_at + t;
            if (at >= depth) at -= depth;
            uint64_t* bar = &full[at];
            if (row >= 0) {
                uint8_t* slot = smem + static_cast<uint32_t>(at) * src.slot();
                tc::fence_proxy_async_smem();
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_u32(bar)), "r"(src.zeros()) : "memory");
                bulk_copy(slot, src.a + row * src.a_stride, src.a_bytes, bar);
                bulk_copy(slot + src.a_bytes, src.b + row * src.b_stride, src.b_bytes, bar);
                if (src.c) bulk_copy(slot + src.a_bytes + src.b_bytes, src.c + edge * src.c_bytes, src.c_bytes, bar);
            } else {
                tc::mbar_arrive(bar);
            }
        }
        issued += m;
        issued_at += m;
        if (issued_at >= depth) issued_at -= depth;
    }
    // `load(meta, i)` fetches what lane i & 31 has to know about edge i of the part (nothing from `count` on)
    template <typename Load>
    __device__ __forceinline__ void start(int count, Load&& load) {
        total = count;
        used = issued = used_at = issued_at = 0;
        parity = 0;
        const int lane = threadIdx.x & 31;
        load(now, lane);
        load(next, lane + 32);
        __syncwarp();
        issue(depth);
    }
    // The next m <= U edges, all of one batch: waits for their slots.  False: a wait gave up.
    __device__ __forceinline__ bool wait(int m, const uint8_t* (&slot)[U]) {
        bool ok = true;
        int at = used_at;
        uint32_t p = parity;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            slot[u] = smem + static_cast<uint32_t>(at) * src.slot();
            if (u < m) {
                ok = bounded_wait(&full[at], p) && ok;
                if (++at == depth) { at = 0; p ^= 1u; }
            }
        }
        return __all_sync(kAll, ok);
    }
    // They have been used: their slots take the next edges.
    template <typename Load>
    __device__ __forceinline__ void release(int m, Load&& load) {
        __syncwarp();
        const int batch = used >> 5;
        used += m;
        used_at += m;
        if (used_at >= depth) { used_at -= depth; parity ^= 1u; }
        if ((used >> 5) != batch) {
            now = next;
            load(next, ((used >> 5) + 1) * 32 + (threadIdx.x & 31));
        }
        if (issued < total) issue(m);
    }
    // After a wait that gave up: the copies under way must not outlive this warp's shared memory.
    __device__ __forceinline__ void abandon(int32_t* status) {
        if ((threadIdx.x & 31) == 0) *status = 3;
        for (int i = used; i < issued; ++i) {
            bounded_wait(&full[used_at], parity);
            if (++used_at == depth) { used_at = 0; parity ^= 1u; }
        }
        used = issued = total;
    }
};

// walk_rows over a ring: before(meta, lane of the first edge, m) runs ahead of the wait, group(slots, meta, lane, m) uses the edges.
template <int U, typename Meta, typename Load, typename Open, typename Before, typename Group, typename Close>
__device__ __forceinline__ void walk_ring(const Rows& r, const Part& p, Ring<U, Meta>& ring, int32_t* status, Load&& load, Open&& open, Before&& before,
                                          Group&& group, Close&& close) {
    ring.start(static_cast<int>(p.behind - p.e0), load);
    bool failed = false;
    walk_rows(
        r, p, open,
        [&](int64_t first, int64_t last) {
            int left = static_cast<int>(last - first);
            while (left > 0 && !failed) {
                const int at = ring.used & 31, m = min(min(min(U, left), 32 - at), ring.issued - ring.used);
                const uint8_t* slot[U];
                before(ring.now, at, m);
                failed = !ring.wait(m, slot);
                if (failed) break;
                group(slot, ring.now, at, m);
                ring.release(m, load);
                left -= m;
            }
        },
        [&](int64_t n, bool started, bool ends) {
            if (!failed) close(n, started, ends);
        });
    if (failed) ring.abandon(status);
}

// Places of a lane's vectors in a slot, in bytes; vectors that it does not have are the zeros at the slot's end, so that no product
// has to be left out (a multiplication by zero would not do: what lies in the row belongs to another head and may be anything).
template <typename T, int V>
__device__ __forceinline__ void slot_places(const int (&col)[V], uint32_t row, uint32_t zeros, uint32_t (&place)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) place[j] = col[j] >= 0 ? row + static_cast<uint32_t>(col[j]) * static_cast<uint32_t>(sizeof(T)) : zeros;
}
// Dots with the lane's columns of a row in a slot, and products added to a lane's sums; two columns an instruction.
template <typename T, int VEC, int V>
__device__ __forceinline__ float dot_row(const uint8_t* slot, const float (&f)[V][VEC], const uint32_t (&place)[V]) {
    static_assert(VEC % 2 == 0, "rows in shared memory are read in vectors of 16 bytes");
    float2 d = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        Packed<T, VEC> p;
        float x[VEC];
        p.load(reinterpret_cast<const T*>(slot + place[j]));
        p.unpack(x);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) d = fma2(make_float2(f[j][i], f[j][i + 1]), make_float2(x[i], x[i + 1]), d);
    }
    return d.x + d.y;
}
template <typename T, int VEC, int V>
__device__ __forceinline__ void add_row(const uint8_t* slot, float by, float (&sum)[V][VEC], const uint32_t (&place)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        Packed<T, VEC> p;
        float x[VEC];
        p.load(reinterpret_cast<const T*>(slot + place[j]));
        p.unpack(x);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const float2 s = fma2(make_float2(by, by), make_float2(x[i], x[i + 1]), make_float2(sum[j][i], sum[j][i + 1]));
            sum[j][i] = s.x;
            sum[j][i + 1] = s.y;
        }
    }
}
// The same by columns, testing each: for the kernel whose registers have no room for the places (with them, 700 us in place of 470
// on 425,984 edges of 1,024 columns in bf16: it spills).  Same order of additions.
template <typename T, int VEC, int V>
__device__ __forceinline__ float dot_columns(const uint8_t* row, const float (&f)[V][VEC], const int (&col)[V]) {
    float2 d = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (col[j] < 0) continue;
        Packed<T, VEC> p;
        float x[VEC];
        p.load(reinterpret_cast<const T*>(row) + col[j]);
        p.unpack(x);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) d = fma2(make_float2(f[j][i], f[j][i + 1]), make_float2(x[i], x[i + 1]), d);
    }
    return d.x + d.y;
}
template <typename T, int VEC, int V>
__device__ __forceinline__ void add_columns(const uint8_t* row, float by, float (&sum)[V][VEC], const int (&col)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if (col[j] < 0) continue;
        Packed<T, VEC> p;
        float x[VEC];
        p.load(reinterpret_cast<const T*>(row) + col[j]);
        p.unpack(x);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const float2 s = fma2(make_float2(by, by), make_float2(x[i], x[i + 1]), make_float2(sum[j][i], sum[j][i + 1]));
            sum[j][i] = s.x;
            sum[j][i + 1] = s.y;
        }
    }
}
// Sums over the lanes of a head of U numbers side by side.
template <int U>
__device__ __forceinline__ void head_sums(float (&v)[U], int lanes) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        if (o >= lanes) continue;
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] += __shfl_xor_sync(kAll, v[u], o);
    }
}

// ------------------------------------------------------------------------------------------------------------- host side
struct Split {
    int64_t per_part;
    int parts, warps;       // of a block
    bool merge;             // rows are longer than a block's parts
    int join_warps;
};

// Parts of equal size over whole waves of warps (`per_sm` run at a time on an SM), at most about 1,024 items each; at least 16 items a
// part (a part costs a search for its row and up to two slots).
inline Split split_rows(int64_t num, int64_t edges, int per_sm) {
    Split s;
    const int64_t items = std::max<int64_t>(num + edges, 1), wave = static_cast<int64_t>(kNumSMs) * per_sm;
    const int64_t waves = std::max<int64_t>(1, ceil_div(items, wave * 1024));
    s.per_part = std::max<int64_t>(16, ceil_div(items, wave * waves));
    s.parts = static_cast<int>(ceil_div(items, s.per_part));
    s.warps = s.parts >= kNumSMs * 4 ? 4 : 1;
    const int64_t longest = num > 0 ? edges / num : 0;
    // rows longer than the parts of an SM: all its warps are one block, which leaves one sum
    s.merge = s.warps > 1 && longest > s.per_part * per_sm;
    if (s.merge) s.warps = per_sm;
    s.join_warps = longest > 4 * s.per_part ? 16 : 1;
    return s;
}

// Lanes a head gets and vectors a lane then owns; 0: the head is too wide.
inline int lanes_of_head(int heads, int vectors, int most) {
    int lanes = 32;
    while (lanes > 1 && 32 / lanes < heads && vectors <= (lanes / 2) * most) lanes /= 2;
    return vectors <= lanes * most ? lanes : 0;
}

// Vectors a lane that are compiled: the next one up is taken.
inline int compiled_vectors(int vec, int v) {
    if (vec > 1) return v <= 6 ? v : 8;
    return v <= 4 ? 4 : v <= 8 ? 8 : v <= 16 ? 16 : 32;
}

constexpr int kWarpsPerSm[] = {16, 12, 8, 4};    // that the kernels may be launched with
inline int most_parts(int64_t num, int64_t edges) {
    int parts = 1;
    for (int w : kWarpsPerSm) parts = std::max(parts, split_rows(num, edges, w).parts);
    return parts;
}

// How a kernel is launched: through the ring where the rows can be copied in bulk (16-byte rows, strides and addresses, vectors of 16
// bytes) and one warp holds all heads, else by loads into registers.
struct Plan {
    int lanes, v, groups;      // lanes of a head, vectors of a lane, head groups (grid.y)
    bool ring;
    int depth;
    size_t warp_smem;          // of the ring
    Split s;
};

// Slots of a warp's ring: as many blocks of four warps on an SM as leave `least` slots to a warp (fewer, deeper rings below that).
inline bool ring_fits(uint32_t slot, int most_blocks, int least, int* blocks, int* depth) {
    for (*blocks = most_blocks; *blocks >= 1; --*blocks) {
        const int budget = (227 * 1024 / *blocks - 1024) / 4 - 128;
        *depth = std::min<int>(16, budget / static_cast<int>(slot + 8));
        if (*depth >= (*blocks > 1 ? least : 2)) return true;
    }
    return false;
}

inline int most_vectors(int vec) { return vec == 8 ? 4 : vec == 4 ? 8 : 32; }

inline int plan(Plan* p, const char* what, int type, int vec, int heads, int vectors, int64_t num, int64_t edges, const RingSource& rows,
                int most_blocks, int least, bool may_ring) {
    p->lanes = lanes_of_head(heads, vectors, most_vectors(vec));
    if (p->lanes == 0) return fail(E3B_ERR_UNSUPPORTED, "%s: a head of %d columns (at most 1024)", what, vec * vectors);
    p->groups = static_cast<int>(ceil_div(heads, 32 / p->lanes));
    p->v = compiled_vectors(vec, static_cast<int>(ceil_div(vectors, p->lanes)));
    int blocks = 2;
    p->ring = may_ring && vec * element_size(type) == 16 && p->groups == 1 && ((rows.a_bytes | rows.b_bytes | rows.c_bytes) & 15) == 0 &&
              ((rows.a_stride | rows.b_stride) & 15) == 0 && aligned_to(rows.a, 16) && aligned_to(rows.b, 16) && aligned_to(rows.c, 16) &&
              ring_fits(rows.slot(), most_blocks, least, &blocks, &p->depth);
    p->s = split_rows(num, edges, p->ring ? 4 * blocks : 8);
    if (p->ring) {
        if (p->s.warps > 4) p->depth = std::min(p->depth, (226 * 1024 / p->s.warps - 128) / static_cast<int>(rows.slot() + 8));
        if (p->s.warps == 1) p->depth = std::min<int>(16, (200 * 1024) / static_cast<int>(rows.slot() + 8));
        p->warp_smem = ceil_div(static_cast<int64_t>(p->depth) * (rows.slot() + 8), 128) * 128;
    }
    return E3B_OK;
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
    if constexpr (sizeof(T) == 2) {
        if (vec == 8) {
            switch (v) {
                case 1: return f(T(), Int<8>(), Int<1>());
                case 2: return f(T(), Int<8>(), Int<2>());
                case 3: return f(T(), Int<8>(), Int<3>());
                default: return f(T(), Int<8>(), Int<4>());
            }
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

}  // namespace
}  // namespace e3b
