// The boundary between two residual blocks, shared by its two directions:
//   n = norm(y; w_post),  g = gate(n),  z = residual + scale * g,  h = norm(z; w_pre)      (norm as in norm.cu, gate as in gate.cu)
//
// A thread block takes one row at a time and walks the rows.  The columns fall into two sorts of items, and a thread owns the same
// K + M items of every row, so that weights, table entries and the sums of the parameter gradients stay in its registers:
//   wide    VEC columns that are multiplied by gates (or by nothing): the output columns together with the input columns they
//           come from, so y and residual meet in one thread
//   narrow  NW columns that pass through an activation: scalars, and the gates themselves.  The exponentials are most of the
//           arithmetic; narrow items spread them over all threads (as part of wide items they kept one warp busy while
//           the others waited at the next barrier: 262,144 rows in bf16 1,443 -> 1,080 us).
// Only the activated gates, and backward the products whose sums are the gates' gradients, go through shared memory.
#pragma once
#include <cstring>

#include "norm.cuh"

namespace e3b {
namespace {

enum NarrowKind { kScalar = 0, kGates = 2, kUnused = 3 };      // (codes of the gate tables)
constexpr int kWideWords = 4;        // {input column, output column, input block, output block}, then the gate slot of each column
constexpr int kNarrowWords = 8;      // {kind, input column, output column or -1, blocks of both, activation, constant (bits), first gate slot}

struct GateRow {
    const int32_t* wide;       // [num_wide][kWideWords + VEC]; slot num_gates holds 1 (a column without a gate)
    const int32_t* narrow;     // [num_narrow][kNarrowWords]
    const int32_t* in_tbl;     // [din][4]  {irreps block, channel, first output column, count}: the last two of a gate's components
    const int32_t* out_tbl;    // [dout][4] {irreps block, channel, -, -}
    const int32_t* in_chan;    // [nchan_in][2]  {first column, components}
    const int32_t* out_chan;   // [nchan_out][2]
    const float* in_inv;       // [nblk_in]  1 / n_b
    const float* out_inv;      // [nblk_out]
    int num_wide, num_narrow, num_gates, din, dout, nblk_in, nblk_out, nchan_in, nchan_out, nw;
};

// The items of this thread; first column -1: none.  in_blocks, out_blocks: bit b set where this warp touches irreps block b.
template <int VEC, int NW, int K, int M>
struct Items {
    int win[K], wout[K], wbi[K], wbo[K], gate[K][VEC];
    int kind[M], nin[M], nout[M], nbi[M], nbo[M], act[M], slot[M];
    float cst[M];
    unsigned in_blocks, out_blocks;
    __device__ __forceinline__ void init(const GateRow& t) {
        in_blocks = out_blocks = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int n = k * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x);
            win[k] = wout[k] = -1;
            wbi[k] = wbo[k] = 0;
#pragma unroll
            for (int i = 0; i < VEC; ++i) gate[k][i] = t.num_gates;
            if (n >= t.num_wide) continue;
            const int32_t* e = t.wide + n * (kWideWords + VEC);
            win[k] = e[0];
            wout[k] = e[1];
            wbi[k] = e[2];
            wbo[k] = e[3];
#pragma unroll
            for (int i = 0; i < VEC; ++i) gate[k][i] = e[kWideWords + i];
            in_blocks |= 1u << wbi[k];
            out_blocks |= 1u << wbo[k];
        }
#pragma unroll
        for (int j = 0; j < M; ++j) {
            const int n = j * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x);
            kind[j] = nin[j] = nout[j] = -1;
            nbi[j] = nbo[j] = slot[j] = 0;
            act[j] = 3;
            cst[j] = 1.0f;
            if (n >= t.num_narrow) continue;
            const int32_t* e = t.narrow + n * kNarrowWords;
            kind[j] = e[0];
            nin[j] = e[1];
            nout[j] = e[2];
            nbi[j] = e[3];
            nbo[j] = e[4];
            act[j] = e[5];
            cst[j] = __int_as_float(e[6]);
            slot[j] = e[7];
            in_blocks |= 1u << nbi[j];
            if (nout[j] >= 0) out_blocks |= 1u << nbo[j];
        }
        in_blocks = __reduce_or_sync(0xffffffffu, in_blocks);
        out_blocks = __reduce_or_sync(0xffffffffu, out_blocks);
    }
};

// The next rows of A arrays on their way: by cp.async to shared memory, two rows in front of the one in hand (one where a thread has eight items).  Every thread
// fetches its own columns and reads nothing else, so the only wait is for its own copies.  Single 16-bit columns are too
// small for such a copy: they are loaded into registers, one row in front.
__host__ __device__ constexpr int rows_ahead(int bytes, int items) { return bytes >= 4 && items < 8 ? 2 : 1; }      // (eight items: one, for their shared memory)
template <typename T, int WIDTH, int N, int A, int AHEAD>
struct RowAhead {
    static constexpr int kBytes = WIDTH * static_cast<int>(sizeof(T));
    static constexpr bool kAsync = kBytes >= 4;
    static constexpr int kThread = kAsync ? AHEAD * A * N * kBytes : 0;      // bytes a thread
    char* mine;            // this thread's place: [rows ahead][A][N] of kBytes, a block of threads apart
    Packed<T, WIDTH> reg[kAsync ? 1 : A][kAsync ? 1 : N];
    __device__ __forceinline__ explicit RowAhead(void* smem) : mine(static_cast<char*>(smem) + threadIdx.x * kBytes) {}
    __device__ __forceinline__ char* at(int stage, int a, int n) const { return mine + ((stage * A + a) * N + n) * static_cast<int>(blockDim.x) * kBytes; }
    __device__ __forceinline__ void fetch(int stage, int a, int n, const T* from) {
        if constexpr (kAsync) {
            const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(at(stage, a, n)));
            if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(__cvta_generic_to_global(from)) : "memory");
            else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(__cvta_generic_to_global(from)), "n"(kBytes) : "memory");
        } else {
            reg[a][n].load(from);
        }
    }
    __device__ __forceinline__ void read(int stage, int a, int n, float (&f)[WIDTH]) const {
        if constexpr (kAsync) {
            Packed<T, WIDTH> p;
            p.load(reinterpret_cast<const T*>(at(stage, a, n)));
            p.unpack(f);
        } else {
            reg[a][n].unpack(f);
        }
    }
};
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int AHEAD>
__device__ __forceinline__ void wait_for_row() { asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory"); }

// ------------------------------------------------------------------------------------------------- one warp a row
// Rows of ordinary width are taken by one warp each: no barriers, sums by shuffles, and the work that does not depend on the
// width (sums, roots, addresses) is done once a row and not once a warp of it.  The columns fall into slots of 32 items that lie
// side by side in the input and in the output row and belong to one irreps block, so everything about a slot but the lane's place in it
// is the same for all lanes and comes from the kernel's parameters.
constexpr int kMaxWide = 9, kMaxNarrow = 8, kMaxBlocks = 8;
struct WideSlot {
    int in, out, count;        // first columns, items
    int bi, bo;                // irreps blocks
    int gates;                 // place of the first column's gate in the row of gates per column, -1: no gate
};
struct NarrowSlot {
    int kind, in, out, count, bi, bo, act;
    float cst;
    int spread, comps;         // gates: place of the first gate's copies, copies of each (components of its channel)
};
struct RowPlan {
    WideSlot w[kMaxWide];
    NarrowSlot n[kMaxNarrow];
    int num_wide, num_narrow, din, dout, nblk_in, nblk_out, num_spread;      // num_spread: length of the row of gates per column
    float inv_in[kMaxBlocks], inv_out[kMaxBlocks];           // 1 / columns, in the order in which the slots come to the blocks
    unsigned wide_in_ends, narrow_in_ends, wide_out_ends, narrow_out_ends;
};
constexpr int kPlanHead = 9, kPlanSlot = 10;     // host array: {vec, narrow, wide slots, narrow slots, din, dout, blocks in, blocks out, spread}, slots

// The kernel's parameters from the host's array.  False: more slots or blocks than a warp's registers take.
inline bool row_plan(const int32_t* host, const int32_t* in_count, const int32_t* out_count, RowPlan* p) {
    *p = {};
    p->num_wide = host[2];
    p->num_narrow = host[3];
    p->din = host[4];
    p->dout = host[5];
    p->nblk_in = host[6];
    p->nblk_out = host[7];
    p->num_spread = host[8];
    if (p->num_wide > kMaxWide || p->num_narrow > kMaxNarrow || p->nblk_in > kMaxBlocks || p->nblk_out > kMaxBlocks) return false;
    const int32_t* s = host + kPlanHead;
    for (int i = 0; i < p->num_wide; ++i, s += kPlanSlot) p->w[i] = {s[0], s[1], s[2], s[3], s[4], s[5]};
    for (int i = 0; i < p->num_narrow; ++i, s += kPlanSlot) {
        float cst;
        memcpy(&cst, &s[7], sizeof(cst));
        p->n[i] = {s[0], s[1], s[2], s[3], s[4], s[5], s[6], cst, s[8], s[9]};
    }
    // blocks numbered in the order of the slots; a block whose slots do not come together is not for this kernel
    int in_seen[32], out_seen[32], n_in = 0, n_out = 0;
    auto visit = [](int block, int* seen, int* n) {
        if (*n > 0 && seen[*n - 1] == block) return true;
        for (int i = 0; i < *n; ++i)
            if (seen[i] == block) return false;
        seen[(*n)++] = block;
        return true;
    };
    int last_in = -1, last_out = -1;          // slot (narrow ones from 0, wide ones from kMaxNarrow on) that ends the present block
    auto mark = [](int slot, unsigned* narrow, unsigned* wide) {
        if (slot < 0) return;
        if (slot < kMaxNarrow) *narrow |= 1u << slot;
        else *wide |= 1u << (slot - kMaxNarrow);
    };
    auto slot = [&](int number, int* bi, int* bo, bool has_out) {
        const int before_in = n_in, before_out = n_out;
        if (!visit(*bi, in_seen, &n_in) || (has_out && !visit(*bo, out_seen, &n_out))) return false;
        if (n_in != before_in) mark(last_in, &p->narrow_in_ends, &p->wide_in_ends);
        last_in = number;
        *bi = n_in - 1;
        if (has_out) {
            if (n_out != before_out) mark(last_out, &p->narrow_out_ends, &p->wide_out_ends);
            last_out = number;
            *bo = n_out - 1;
        }
        return true;
    };
    for (int j = 0; j < p->num_narrow; ++j)
        if (!slot(j, &p->n[j].bi, &p->n[j].bo, p->n[j].out >= 0)) return false;
    for (int k = 0; k < p->num_wide; ++k)
        if (!slot(kMaxNarrow + k, &p->w[k].bi, &p->w[k].bo, true)) return false;
    mark(last_in, &p->narrow_in_ends, &p->wide_in_ends);
    mark(last_out, &p->narrow_out_ends, &p->wide_out_ends);
    for (int i = 0; i < n_in; ++i) p->inv_in[i] = 1.0f / static_cast<float>(in_count[in_seen[i]]);
    for (int i = 0; i < n_out; ++i) p->inv_out[i] = 1.0f / static_cast<float>(out_count[out_seen[i]]);
    return true;
}

// Activations of a narrow item: silu and sigmoid on the hardware's exponential and division, the others as in gate_act (which costs five times the
// instructions, and whose last bits differ).  From the documented errors (__expf 2 + 1.173 |x| ulp, __fdividef 2 ulp for divisors to 2^126,
// an ulp at most 2^-23) and the three roundings around them: relative error below (6 + 1.2 |x|) 2^-23 for x > -87; below that, where a
// sigmoid is less than 2^-125, the result may be zero.
template <int N>
__device__ __forceinline__ void activate(int act, float cst, const float (&x)[N], float (&y)[N]) {
    if (act == kGSilu || act == kGSigmoid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float s = cst * __fdividef(1.0f, 1.0f + __expf(-x[i]));
            y[i] = act == kGSilu ? x[i] * s : s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = cst * gate_act(act, x[i]);
    }
}

// The same with the derivative (y may be x).
template <int N>
__device__ __forceinline__ void activate_and_derive(int act, float cst, const float (&x)[N], float (&y)[N], float (&dy)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float v = x[i];
        if (act == kGSilu || act == kGSigmoid) {
            const float s = __fdividef(1.0f, 1.0f + __expf(-v)), ds = s * (1.0f - s);
            y[i] = cst * (act == kGSilu ? v * s : s);
            dy[i] = cst * (act == kGSilu ? fmaf(v, ds, s) : ds);
        } else {
            y[i] = cst * gate_act(act, v);
            dy[i] = cst * gate_act_grad(act, v);
        }
    }
}

// Sums over the irreps blocks of a row.  The slots come block by block, the narrow ones of a block before the wide ones: bit j of
// narrow_ends (k of wide_ends) is set where a block ends with slot j (k); out receives the blocks in that order:
// rsqrt(sum * inv + eps) or, with MEAN, sum * inv.  In shared memory of the warp.
template <bool MEAN, int K, int M>
__device__ __forceinline__ void row_sums(const float (&wv)[K], const float (&nv)[M], unsigned wide_ends, unsigned narrow_ends, const float* inv, float eps,
                                         float* out) {
    float s = 0.0f;
    int b = 0;
    auto end = [&]() {
        s = warp_sum(s);
        if ((threadIdx.x & 31) == 0) out[b] = MEAN ? s * inv[b] : rsqrtf(fmaf(s, inv[b], eps));
        s = 0.0f;
        ++b;
    };
#pragma unroll
    for (int j = 0; j < M; ++j) {
        s += nv[j];
        if (narrow_ends >> j & 1u) end();
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        s += wv[k];
        if (wide_ends >> k & 1u) end();
    }
    __syncwarp();
}

// N gates into the row of gates per column, each for the components of its channel
template <int COMPS, int N>
__device__ __forceinline__ void spread_gates(float* to, const float (&g)[N], int comps) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (COMPS > 0) {
#pragma unroll
            for (int m = 0; m < COMPS; ++m) to[i * COMPS + m] = g[i];
        } else {
            for (int m = 0; m < comps; ++m) to[i * comps + m] = g[i];
        }
    }
}
template <int N>
__device__ __forceinline__ void spread_gates(float* row, int lane, const float (&g)[N], int comps) {
    float* to = row + lane * N * comps;
    switch (comps) {
        case 3: spread_gates<3, N>(to, g, comps); break;
        case 5: spread_gates<5, N>(to, g, comps); break;
        case 7: spread_gates<7, N>(to, g, comps); break;
        default: spread_gates<0, N>(to, g, comps); break;
    }
}

// ----------------------------------------------------------------------------------------------------------- host side
constexpr int kMostColumns = 4096;      // of a row: what the registers and the shared memory of 512 threads take in both directions
struct RowShape {
    int vec, narrow, k, m, threads;
};

// f(element type, widths of wide and narrow items, items of a thread, threads of a block at most) with all as types
template <typename T, typename F>
int by_items(const RowShape& s, F&& f) {
    auto with_km = [&](auto v0, auto n0) -> int {
        if (s.k == 1 && s.m == 1) {
            if (s.threads <= 128) return f(T(), v0, n0, Int<1>(), Int<1>(), Int<128>());
            if (s.threads <= 256) return f(T(), v0, n0, Int<1>(), Int<1>(), Int<256>());
        }
        if (s.k == 1) return f(T(), v0, n0, Int<1>(), Int<2>(), Int<512>());
        if constexpr (decltype(v0)::value == 1) {
            if (s.k == 8) return f(T(), v0, n0, Int<8>(), Int<8>(), Int<512>());
        }
        if (s.m == 8) return f(T(), v0, n0, Int<2>(), Int<8>(), Int<512>());
        return f(T(), v0, n0, Int<2>(), Int<4>(), Int<512>());
    };
    if constexpr (sizeof(T) == 2) {
        if (s.vec == 8) return with_km(Int<8>(), Int<2>());
        if (s.vec == 4) return with_km(Int<4>(), Int<2>());
    } else {
        if (s.vec == 4) return with_km(Int<4>(), Int<1>());
    }
    return with_km(Int<1>(), Int<1>());
}
template <typename F>
int by_type_and_items(int type, const RowShape& s, F&& f) {
    if (type == kFloat32) return by_items<float>(s, f);
    if (type == kBFloat16) return by_items<__nv_bfloat16>(s, f);
    return by_items<__half>(s, f);
}

// sizes: host array {vec, narrow, num_wide, num_narrow, gates, din, dout, blocks in, blocks out, channels in, channels out}
inline int gate_row(const char* what, int type, const int32_t* sizes, const int32_t* wide, const int32_t* narrow, const int32_t* in_tbl,
                    const int32_t* out_tbl, const int32_t* in_chan, const int32_t* out_chan, const float* in_inv, const float* out_inv, GateRow* t,
                    RowShape* s) {
    *t = {wide, narrow, in_tbl, out_tbl, in_chan, out_chan, in_inv, out_inv, sizes[2], sizes[3], sizes[4], sizes[5], sizes[6], sizes[7], sizes[8], sizes[9], sizes[10], 0};
    s->vec = sizes[0];
    s->narrow = sizes[1];
    const bool known = (s->vec == 1 && s->narrow == 1) || (type == kFloat32 ? s->vec == 4 && s->narrow == 1 : (s->vec == 4 || s->vec == 8) && s->narrow == 2);
    if (!known) return fail(E3B_ERR_ARG, "%s: items of %d and %d columns", what, s->vec, s->narrow);
    if (t->nblk_in > 32 || t->nblk_out > 32) return fail(E3B_ERR_UNSUPPORTED, "%s: %d irreps blocks, at most 32", what, std::max(t->nblk_in, t->nblk_out));
    // one item of each sort a thread while that takes up to 256 threads, then more
    const int n = t->num_wide, m = t->num_narrow;
    s->k = s->m = 1;
    if (std::max(n, m) > 256) s->m = 2;
    if (n > kMaxThreads || m > 2 * kMaxThreads) s->k = 2, s->m = 4;
    if (m > 4 * kMaxThreads) s->m = 8;
    if (n > 2 * kMaxThreads) s->k = s->m = 8;
    if (std::max(t->din, t->dout) > kMostColumns) return fail(E3B_ERR_UNSUPPORTED, "%s: rows of %d columns, at most %d", what, std::max(t->din, t->dout), kMostColumns);
    s->threads = static_cast<int>(std::max<int64_t>(1, ceil_div(std::max(ceil_div(n, s->k), ceil_div(m, s->m)), 32)) * 32);
    t->nw = warps_pow2(s->threads);
    return E3B_OK;
}

}  // namespace
}  // namespace e3b
