// The boundary between two residual blocks, shared by its two directions:
//   n = norm(y; w_post),  g = gate(n),  z = residual + scale * g,  h = norm(z; w_pre)      (norm as in norm.cu, gate as in gate.cu)
//
// A thread block takes one row at a time and walks the rows.  The columns fall into two sorts of items, and a thread owns the same
// K + M items of every row, so that weights, table entries and the sums of the parameter gradients stay in its registers:
//   wide    VEC columns that are multiplied by gates (or by nothing): the output columns together with the input columns they
//           come from, so y and residual meet in one thread
//   narrow  NW columns that pass through an activation: scalars, and the gates themselves.  The exponentials are most of the
//           arithmetic; narrow items spread them over all threads (as part of wide items they kept one warp busy while
//           the others waited at the next barrier: 1,443 us of 262,144 rows in bf16 against what norm_gate.cu states).
// Only the activated gates, and backward the products whose sums are the gates' gradients, go through shared memory.
#pragma once
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

// The next rows of A arrays on their way to shared memory (cp.async), kAhead rows in front of the one in hand.  Every thread
// fetches its own columns and reads nothing else, so the only wait is for its own copies.  Single 16-bit columns are too
// small for such a copy: they are loaded when they are needed.
constexpr int kAhead = 2;
template <typename T, int WIDTH, int N, int A>
struct RowAhead {
    static constexpr int kBytes = WIDTH * static_cast<int>(sizeof(T));
    static constexpr bool kAsync = kBytes >= 4;
    static constexpr int kThread = kAsync ? kAhead * A * N * kBytes : 0;      // bytes a thread
    char* mine;            // this thread's place: [kAhead][A][N] of kBytes, a block of threads apart
    __device__ __forceinline__ explicit RowAhead(void* smem) : mine(static_cast<char*>(smem) + threadIdx.x * kBytes) {}
    __device__ __forceinline__ char* at(int stage, int a, int n) const { return mine + ((stage * A + a) * N + n) * static_cast<int>(blockDim.x) * kBytes; }
    __device__ __forceinline__ void fetch(int stage, int a, int n, const T* from) const {
        if constexpr (kAsync) {
            const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(at(stage, a, n)));
            if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(__cvta_generic_to_global(from)) : "memory");
            else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(__cvta_generic_to_global(from)), "n"(kBytes) : "memory");
        }
    }
    __device__ __forceinline__ void read(int stage, int a, int n, const T* from, float (&f)[WIDTH]) const {
        Packed<T, WIDTH> p;
        if constexpr (kAsync) p.load(reinterpret_cast<const T*>(at(stage, a, n)));
        else p.load(from);
        p.unpack(f);
    }
};
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void wait_for_row() { asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory"); }

// ----------------------------------------------------------------------------------------------------------- host side
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
        if (s.k == 2) return f(T(), v0, n0, Int<2>(), Int<4>(), Int<512>());
        return f(T(), v0, n0, Int<8>(), Int<8>(), Int<512>());
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
    if (n > 2 * kMaxThreads || m > 4 * kMaxThreads) s->k = s->m = 8;
    if (std::max(n, m) > 8 * kMaxThreads) return fail(E3B_ERR_UNSUPPORTED, "%s: %d items, at most %d", what, std::max(n, m), 8 * kMaxThreads);
    s->threads = static_cast<int>(std::max<int64_t>(1, ceil_div(std::max(ceil_div(n, s->k), ceil_div(m, s->m)), 32)) * 32);
    t->nw = s->threads / 32;
    return E3B_OK;
}

}  // namespace
}  // namespace e3b
