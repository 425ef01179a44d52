// Norms on rows of irreps features and the boundary between two residual blocks.
//
// A row is a list of blocks, block b with mul_b channels of d_b = 2l+1 components (n_b = mul_b d_b columns):
//   norm(x)[b, u, m] = w[b, u] * x[b, u, m] * s_b(x),   s_b(x) = (sum_{u,m} x[b, u, m]^2 / n_b + eps)^(-1/2)
// e3b_rms_norm:       h = norm(x; w)                                       the norm before a block
// e3b_norm_gate_residual:  n = norm(y; w_post),  g = gate(n)               the norm after it, Gate (gate.cu),
//                     z = residual + scale * g,  h = norm(z; w_pre)        residual, norm before the next block
// Gradient of norm: with t = g w (cotangent times weight), gx = s (t - x s^2 mean_b(t x)), gw = sum over rows and m of g x s.
//
// Every row is read once and written once in its own type; sums, products and the row between the steps are fp32 (h is taken
// from z before z is rounded).  A thread block takes one to four rows at a time and walks the rows; thread t owns the same columns of every
// row, so weights and table entries stay in registers and the sums of the parameter gradients too.
// Sums over a block of the irreps: a warp reduces per irreps block (its columns touch one to three), the warps' sums are
// added in the order of the warps.
#include <algorithm>

#include "common.cuh"
#include "gate_act.cuh"
#include "typed.cuh"

namespace e3b {
namespace {

constexpr int kMaxThreads = 512;

// Columns this thread owns on one side (input or output row) and what belongs to them.
template <int VEC, int K>
struct Columns {
    int col[K];      // first column, -1: none
    int blk[K];      // irreps block (VEC columns never straddle two)
    int b0, b1;      // irreps blocks this warp touches
    __device__ __forceinline__ void init(const int32_t* __restrict__ tbl, int dim) {
        b0 = 1 << 30;
        b1 = -1;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * VEC;
            col[k] = c < dim ? c : -1;
            blk[k] = c < dim ? tbl[4 * c] : -1;
            if (c < dim) { b0 = min(b0, blk[k]); b1 = max(b1, blk[k]); }
        }
        b0 = __reduce_min_sync(0xffffffffu, b0);
        b1 = __reduce_max_sync(0xffffffffu, b1);
    }
};

// Sums of v over the irreps blocks: each warp leaves its share in red[b * nw + warp] (entries of blocks it does not touch
// stay zero from the start of the kernel).
template <int VEC, int K>
__device__ __forceinline__ void warp_shares(const Columns<VEC, K>& c, const float (&v)[K], float* red, int nw) {
    for (int b = c.b0; b <= c.b1; ++b) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) s += c.blk[k] == b ? v[k] : 0.0f;
        s = warp_sum(s);
        if ((threadIdx.x & 31) == 0) red[b * nw + (threadIdx.x >> 5)] = s;
    }
}
__device__ __forceinline__ float add_shares(const float* red, int nw) {       // nw: a multiple of 4
    float s = 0.0f;
    for (int w = 0; w < nw; w += 4) {
        const float4 a = *reinterpret_cast<const float4*>(red + w);
        s += (a.x + a.y) + (a.z + a.w);
    }
    return s;
}

// ------------------------------------------------------------------------------------------------------------- norm
template <typename T, int VEC, int K>
__global__ void __launch_bounds__(kMaxThreads) rms_fwd_kernel(const T* __restrict__ x, const float* __restrict__ weight,
                                                              const int32_t* __restrict__ tbl, const float* __restrict__ inv_n,
                                                              float eps, T* __restrict__ h, int64_t rows, int dim, int nblk, int nw) {
    extern __shared__ float red[];      // [2][nblk][nw]: two rows' shares in turn
    Columns<VEC, K> c;
    c.init(tbl, dim);
    float w[K][VEC], inv[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        inv[k] = c.col[k] >= 0 ? inv_n[c.blk[k]] : 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[k][i] = c.col[k] >= 0 ? (weight ? weight[tbl[4 * (c.col[k] + i) + 1]] : 1.0f) : 0.0f;
    }
    for (int i = threadIdx.x; i < 2 * nblk * nw; i += blockDim.x) red[i] = 0.0f;
    __syncthreads();
    Packed<T, VEC> next[K];
    int64_t z = blockIdx.x;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (c.col[k] >= 0) next[k].load(x + z * dim + c.col[k]);
    for (int turn = 0; z < rows; z += gridDim.x, turn ^= 1) {
        float v[K][VEC], sq[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = 0.0f;
            if (c.col[k] < 0) continue;
            next[k].unpack(v[k]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) sq[k] = fmaf(v[k][i], v[k][i], sq[k]);
            if (z + gridDim.x < rows) next[k].load(x + (z + gridDim.x) * dim + c.col[k]);
        }
        float* r = red + turn * nblk * nw;
        warp_shares<VEC, K>(c, sq, r, nw);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (c.col[k] < 0) continue;
            const float s = rsqrtf(fmaf(add_shares(r + c.blk[k] * nw, nw), inv[k], eps));
            float o[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) o[i] = v[k][i] * s * w[k][i];
            Packed<T, VEC>::store(h + z * dim + c.col[k], o);
        }
    }
}

// Sums over the columns of a channel, then this thread block's partial row of the parameter gradient.
template <int VEC, int K>
__device__ __forceinline__ void store_channels(const Columns<VEC, K>& c, const float (&acc)[K][VEC], const int32_t* __restrict__ chan,
                                               int nchan, float* buf, float* __restrict__ partial) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (c.col[k] < 0) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) buf[c.col[k] + i] = acc[k][i];
    }
    __syncthreads();
    for (int u = threadIdx.x; u < nchan; u += blockDim.x) {
        float s = 0.0f;
        const int first = chan[2 * u], n = chan[2 * u + 1];
        for (int m = 0; m < n; ++m) s += buf[first + m];
        partial[u] = s;
    }
}

template <typename T, int VEC, int K>
__global__ void __launch_bounds__(kMaxThreads) rms_bwd_kernel(const T* __restrict__ x, const T* __restrict__ gh, const float* __restrict__ weight,
                                                              const int32_t* __restrict__ tbl, const float* __restrict__ inv_n,
                                                              const int32_t* __restrict__ chan, int nchan, float eps, T* __restrict__ gx,
                                                              float* __restrict__ partial, int64_t rows, int dim, int nblk, int nw) {
    extern __shared__ float smem[];
    float* red = smem;                           // [2 turns][2 sums][nblk][nw]
    float* buf = smem + 4 * nblk * nw;           // [dim]
    Columns<VEC, K> c;
    c.init(tbl, dim);
    float w[K][VEC], inv[K], acc[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        inv[k] = c.col[k] >= 0 ? inv_n[c.blk[k]] : 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            w[k][i] = c.col[k] >= 0 ? (weight ? weight[tbl[4 * (c.col[k] + i) + 1]] : 1.0f) : 0.0f;
            acc[k][i] = 0.0f;
        }
    }
    for (int i = threadIdx.x; i < 4 * nblk * nw; i += blockDim.x) red[i] = 0.0f;
    __syncthreads();
    Packed<T, VEC> nx[K], ng[K];
    int64_t z = blockIdx.x;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (c.col[k] >= 0) { nx[k].load(x + z * dim + c.col[k]); ng[k].load(gh + z * dim + c.col[k]); }
    for (int turn = 0; z < rows; z += gridDim.x, turn ^= 1) {
        float v[K][VEC], g[K][VEC], sq[K], dot[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = dot[k] = 0.0f;
            if (c.col[k] < 0) continue;
            nx[k].unpack(v[k]);
            ng[k].unpack(g[k]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                sq[k] = fmaf(v[k][i], v[k][i], sq[k]);
                dot[k] = fmaf(g[k][i] * w[k][i], v[k][i], dot[k]);
            }
            if (z + gridDim.x < rows) {
                nx[k].load(x + (z + gridDim.x) * dim + c.col[k]);
                ng[k].load(gh + (z + gridDim.x) * dim + c.col[k]);
            }
        }
        float* r0 = red + turn * 2 * nblk * nw;
        float* r1 = r0 + nblk * nw;
        warp_shares<VEC, K>(c, sq, r0, nw);
        warp_shares<VEC, K>(c, dot, r1, nw);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (c.col[k] < 0) continue;
            const float s = rsqrtf(fmaf(add_shares(r0 + c.blk[k] * nw, nw), inv[k], eps));
            const float mean = add_shares(r1 + c.blk[k] * nw, nw) * inv[k] * s * s;
            float o[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                o[i] = s * (g[k][i] * w[k][i] - v[k][i] * mean);
                acc[k][i] = fmaf(g[k][i], v[k][i] * s, acc[k][i]);
            }
            if (gx) Packed<T, VEC>::store(gx + z * dim + c.col[k], o);
        }
    }
    if (partial) store_channels<VEC, K>(c, acc, chan, nchan, buf, partial + static_cast<int64_t>(blockIdx.x) * nchan);
}

// Parameter gradient: the thread blocks' partial rows added in a fixed order.  32 channels a block, 32 slices of the rows.
__global__ void __launch_bounds__(1024) add_partials_kernel(const float* __restrict__ partial, int n, int parts, float* __restrict__ out) {
    __shared__ float s[32][33];
    const int u = blockIdx.x * 32 + threadIdx.x;
    float a = 0.0f;
    if (u < n) {
#pragma unroll 4
        for (int p = threadIdx.y; p < parts; p += 32) a += partial[static_cast<int64_t>(p) * n + u];
    }
    s[threadIdx.x][threadIdx.y] = a;
    __syncthreads();
    const float t = warp_sum(s[threadIdx.y][threadIdx.x]);      // channel threadIdx.y, its slices across the lanes
    if (threadIdx.x == 0 && blockIdx.x * 32 + threadIdx.y < n) out[blockIdx.x * 32 + threadIdx.y] = t;
}

// ------------------------------------------------------------------------------------------------- norm, gate, residual, norm
// A thread's item: VEC output columns together with the VEC input columns they come from (scalars and gated components), or VEC
// gates.  So y and residual meet in the registers of one thread, and only the activated gates (and, backward, the products whose
// sums are the gradients of the gates) go through shared memory.  Items are in the order of their input columns.
enum ItemKind { kScalar = 0, kGated = 1, kGates = 2, kUnused = 3 };
constexpr int kItemWords = 8;      // {kind, input column, output column, input block, output block, activation, constant (bits), gate slot}

struct GateRow {
    const int32_t* items;      // [num_items][kItemWords + VEC]: behind the words, the gate slot of each column (gated)
    const int32_t* in_tbl;     // [din][4]  {irreps block, channel, first output column, count}: the last two of a gate's components
    const int32_t* out_tbl;    // [dout][4] {irreps block, channel, -, -}
    const int32_t* in_chan;    // [nchan_in][2]  {first column, components}
    const int32_t* out_chan;   // [nchan_out][2]
    const float* in_inv;       // [nblk_in]  1 / n_b
    const float* out_inv;      // [nblk_out]
    int num_items, num_gates, din, dout, nblk_in, nblk_out, nchan_in, nchan_out, nw;
};

template <int VEC, int K>
struct Items {
    int kind[K], in[K], out[K], bi[K], bo[K], act[K], slot[K];     // slot: the first of its gates' slots
    float cst[K];
    int gate[K][VEC];                                              // slot of each column's gate
    int i0, i1, o0, o1;                                            // irreps blocks this warp touches
    __device__ __forceinline__ void init(const GateRow& t) {
        i0 = o0 = 1 << 30;
        i1 = o1 = -1;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int n = k * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x);
            kind[k] = -1;
            in[k] = out[k] = bi[k] = bo[k] = -1;
            act[k] = 3;
            slot[k] = 0;
            cst[k] = 1.0f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) gate[k][i] = 0;
            if (n >= t.num_items) continue;
            const int32_t* e = t.items + n * (kItemWords + VEC);
            kind[k] = e[0];
            in[k] = e[1];
            out[k] = e[2];
            bi[k] = e[3];
            bo[k] = e[4];
            act[k] = e[5];
            cst[k] = __int_as_float(e[6]);
            slot[k] = e[7];
#pragma unroll
            for (int i = 0; i < VEC; ++i) gate[k][i] = e[kItemWords + i];
            i0 = min(i0, bi[k]);
            i1 = max(i1, bi[k]);
            if (bo[k] >= 0) { o0 = min(o0, bo[k]); o1 = max(o1, bo[k]); }
        }
        i0 = __reduce_min_sync(0xffffffffu, i0);
        i1 = __reduce_max_sync(0xffffffffu, i1);
        o0 = __reduce_min_sync(0xffffffffu, o0);
        o1 = __reduce_max_sync(0xffffffffu, o1);
    }
};

// Sums over the irreps blocks of a row by the warps that touch a block.  share: [nblk][nw]; span: [nblk][2] first and last of those
// warps (warps between them that do not touch the block leave the zero from the start of the kernel).
struct BlockSums {
    float* share;
    int* span;
    int nblk, nw;
    __device__ __forceinline__ void clear() const {
        for (int i = threadIdx.x; i < nblk * nw; i += blockDim.x) share[i] = 0.0f;
        for (int i = threadIdx.x; i < nblk; i += blockDim.x) { span[2 * i] = 1 << 30; span[2 * i + 1] = -1; }
    }
    __device__ __forceinline__ void touch(int b0, int b1) const {
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0)
            for (int b = b0; b <= b1; ++b) { atomicMin(&span[2 * b], warp); atomicMax(&span[2 * b + 1], warp); }
    }
    template <int K>
    __device__ __forceinline__ void add(const float (&v)[K], const int (&blk)[K], int b0, int b1) const {
        for (int b = b0; b <= b1; ++b) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) s += blk[k] == b ? v[k] : 0.0f;
            s = warp_sum(s);
            if ((threadIdx.x & 31) == 0) share[b * nw + (threadIdx.x >> 5)] = s;
        }
    }
    __device__ __forceinline__ float get(int b) const {
        const int w1 = span[2 * b + 1];
        float s = 0.0f;
        for (int w = span[2 * b]; w <= w1; ++w) s += share[b * nw + w];
        return s;
    }
    __host__ __device__ static int floats(int nblk, int nw) { return (nblk * nw + 2 * nblk + 3) / 4 * 4; }
};
__device__ __forceinline__ BlockSums block_sums_at(float*& p, int nblk, int nw) {
    BlockSums b{p, reinterpret_cast<int*>(p + nblk * nw), nblk, nw};
    p += BlockSums::floats(nblk, nw);
    return b;
}

// The next rows of A arrays on their way to shared memory (cp.async), kAhead rows in front of the one in hand.  Every thread
// fetches its own columns and reads nothing else, so the only wait is for its own copies.  Single 16-bit columns are too
// small for such a copy: they are loaded when they are needed.
constexpr int kAhead = 2;
template <typename T, int VEC, int K, int A>
struct RowAhead {
    static constexpr int kBytes = VEC * static_cast<int>(sizeof(T));
    static constexpr bool kAsync = kBytes >= 4;
    static constexpr int kStage = kAsync ? A * K * kBytes : 0;      // bytes a thread and row
    char* mine;            // this thread's place: [kAhead][A][K] of kBytes, a block of threads apart
    __device__ __forceinline__ RowAhead(void* smem) : mine(static_cast<char*>(smem) + threadIdx.x * kBytes) {}
    __device__ __forceinline__ char* at(int stage, int a, int k) const { return mine + ((stage * A + a) * K + k) * static_cast<int>(blockDim.x) * kBytes; }
    __device__ __forceinline__ void fetch(int stage, int a, int k, const T* from) const {
        if constexpr (kAsync) {
            const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(at(stage, a, k)));
            if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(__cvta_generic_to_global(from)) : "memory");
            else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(__cvta_generic_to_global(from)), "n"(kBytes) : "memory");
        }
    }
    static __device__ __forceinline__ void commit() {
        if constexpr (kAsync) asm volatile("cp.async.commit_group;" ::: "memory");
    }
    static __device__ __forceinline__ void wait() {
        if constexpr (kAsync) asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    }
    __device__ __forceinline__ void read(int stage, int a, int k, const T* from, float (&f)[VEC]) const {
        Packed<T, VEC> p;
        if constexpr (kAsync) p.load(reinterpret_cast<const T*>(at(stage, a, k)));
        else p.load(from);
        p.unpack(f);
    }
};

// MAXT, BLOCKS: threads of a block at most, and blocks on an SM that the registers must allow.
template <typename T, int VEC, int K, int MAXT, int BLOCKS>
__global__ void __launch_bounds__(MAXT, BLOCKS) norm_gate_fwd_kernel(const T* __restrict__ residual, const T* __restrict__ y,
                                                                     const float* __restrict__ w_post, const float* __restrict__ scale,
                                                                     const float* __restrict__ w_pre, const GateRow t, float eps,
                                                                     T* __restrict__ z_out, T* __restrict__ h_out, int64_t rows) {
    extern __shared__ __align__(16) float smem[];
    float* at = smem;
    const BlockSums in = block_sums_at(at, t.nblk_in, t.nw), outs = block_sums_at(at, t.nblk_out, t.nw);
    float* gates = at;                                   // [num_gates]
    const RowAhead<T, VEC, K, 2> ahead(gates + (t.num_gates + 3) / 4 * 4);
    Items<VEC, K> it;
    it.init(t);
    auto fetch = [&](int64_t z, int stage) {
        if (z < rows) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (it.kind[k] >= 0) ahead.fetch(stage, 0, k, y + z * t.din + it.in[k]);
                if (it.out[k] >= 0) ahead.fetch(stage, 1, k, residual + z * t.dout + it.out[k]);
            }
        }
        ahead.commit();
    };
    int64_t z = blockIdx.x;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch(z + static_cast<int64_t>(i) * gridDim.x, i);
    in.clear();
    outs.clear();
    __syncthreads();
    in.touch(it.i0, it.i1);
    outs.touch(it.o0, it.o1);
    // a gated column: z = residual + y s (w_post scale) gate
    float cy[K][VEC], sc[K][VEC], wn[K][VEC], inv_i[K], inv_o[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        inv_i[k] = it.kind[k] >= 0 ? t.in_inv[it.bi[k]] : 0.0f;
        inv_o[k] = it.out[k] >= 0 ? t.out_inv[it.bo[k]] : 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            cy[k][i] = it.kind[k] >= 0 ? w_post[t.in_tbl[4 * (it.in[k] + i) + 1]] : 0.0f;
            sc[k][i] = wn[k][i] = 0.0f;
            if (it.out[k] >= 0) {
                const int ch = t.out_tbl[4 * (it.out[k] + i) + 1];
                sc[k][i] = scale[ch] * it.cst[k];
                wn[k][i] = w_pre ? w_pre[ch] : 0.0f;
                if (it.kind[k] == kGated) cy[k][i] *= scale[ch];
            }
        }
    }
    __syncthreads();
    for (int stage = 0; z < rows; z += gridDim.x, stage = stage + 1 == kAhead ? 0 : stage + 1) {
        float v[K][VEC], o[K][VEC], sq[K];
        ahead.wait();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = 0.0f;
            if (it.kind[k] >= 0) {
                ahead.read(stage, 0, k, y + z * t.din + it.in[k], v[k]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) sq[k] = fmaf(v[k][i], v[k][i], sq[k]);
            }
            if (it.out[k] >= 0) ahead.read(stage, 1, k, residual + z * t.dout + it.out[k], o[k]);
        }
        fetch(z + static_cast<int64_t>(kAhead) * gridDim.x, stage);
        in.add<K>(sq, it.bi, it.i0, it.i1);
        __syncthreads();
        float s_in[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (it.kind[k] < 0) continue;
            s_in[k] = rsqrtf(fmaf(in.get(it.bi[k]), inv_i[k], eps));
            if (it.kind[k] != kGates) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[k][i] = it.cst[k] * gate_act(it.act[k], v[k][i] * s_in[k] * cy[k][i]);
            Packed<float, VEC>::store(gates + it.slot[k], v[k]);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = 0.0f;
            if (it.out[k] < 0) continue;
            if (it.kind[k] == kGated) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[k][i] = fmaf(v[k][i] * cy[k][i], s_in[k] * gates[it.gate[k][i]], o[k][i]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[k][i] = fmaf(sc[k][i], gate_act(it.act[k], v[k][i] * s_in[k] * cy[k][i]), o[k][i]);
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) sq[k] = fmaf(o[k][i], o[k][i], sq[k]);
            Packed<T, VEC>::store(z_out + z * t.dout + it.out[k], o[k]);
        }
        if (h_out) outs.add<K>(sq, it.bo, it.o0, it.o1);
        __syncthreads();
        if (h_out) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (it.out[k] < 0) continue;
                const float s = rsqrtf(fmaf(outs.get(it.bo[k]), inv_o[k], eps));
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[k][i] *= s * wn[k][i];
                Packed<T, VEC>::store(h_out + z * t.dout + it.out[k], o[k]);
            }
        }
    }
}

// The row is computed again from residual and y (their two statistics included); gz and gh may be null.
template <typename T, int VEC, int K, int MAXT, int BLOCKS>
__global__ void __launch_bounds__(MAXT, BLOCKS) norm_gate_bwd_kernel(const T* __restrict__ residual, const T* __restrict__ y,
                                                                     const T* __restrict__ gz, const T* __restrict__ gh,
                                                                     const float* __restrict__ w_post, const float* __restrict__ scale,
                                                                     const float* __restrict__ w_pre, const GateRow t, float eps,
                                                                     T* __restrict__ g_residual, T* __restrict__ gy,
                                                                     float* __restrict__ partial, int64_t rows) {
    extern __shared__ __align__(16) float smem[];
    float* at = smem;
    const BlockSums in = block_sums_at(at, t.nblk_in, t.nw), dots = block_sums_at(at, t.nblk_in, t.nw);
    const BlockSums outs = block_sums_at(at, t.nblk_out, t.nw), ghs = block_sums_at(at, t.nblk_out, t.nw);
    float* gates = at;                                        // [num_gates] activated gates
    float* prod = gates + (t.num_gates + 3) / 4 * 4;          // [dout] cotangent of the gated row times the normalised row
    const RowAhead<T, VEC, K, 4> ahead(prod + (t.dout + 3) / 4 * 4);
    Items<VEC, K> it;
    it.init(t);
    auto fetch = [&](int64_t z, int stage) {
        if (z < rows) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int64_t o = z * t.dout + it.out[k];
                if (it.kind[k] >= 0) ahead.fetch(stage, 0, k, y + z * t.din + it.in[k]);
                if (it.out[k] >= 0) {
                    ahead.fetch(stage, 1, k, residual + o);
                    if (gz) ahead.fetch(stage, 2, k, gz + o);
                    if (gh) ahead.fetch(stage, 3, k, gh + o);
                }
            }
        }
        ahead.commit();
    };
    int64_t z = blockIdx.x;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch(z + static_cast<int64_t>(i) * gridDim.x, i);
    in.clear();
    dots.clear();
    outs.clear();
    ghs.clear();
    __syncthreads();
    in.touch(it.i0, it.i1);
    dots.touch(it.i0, it.i1);
    outs.touch(it.o0, it.o1);
    ghs.touch(it.o0, it.o1);
    float wp[K][VEC], sc[K][VEC], wn[K][VEC], inv_i[K], inv_o[K];
    float a_post[K][VEC], a_scale[K][VEC], a_pre[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        inv_i[k] = it.kind[k] >= 0 ? t.in_inv[it.bi[k]] : 0.0f;
        inv_o[k] = it.out[k] >= 0 ? t.out_inv[it.bo[k]] : 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            a_post[k][i] = a_scale[k][i] = a_pre[k][i] = 0.0f;
            wp[k][i] = it.kind[k] >= 0 ? w_post[t.in_tbl[4 * (it.in[k] + i) + 1]] : 0.0f;
            sc[k][i] = wn[k][i] = 0.0f;
            if (it.out[k] >= 0) {
                const int ch = t.out_tbl[4 * (it.out[k] + i) + 1];
                sc[k][i] = scale[ch];
                wn[k][i] = w_pre ? w_pre[ch] : 0.0f;
            }
        }
    }
    __syncthreads();
    for (int stage = 0; z < rows; z += gridDim.x, stage = stage + 1 == kAhead ? 0 : stage + 1) {
        float v[K][VEC], x[K][VEC], g0[K][VEC], g1[K][VEC], sq[K], dot[K];     // v: y, then normalised; x: residual, then z
        ahead.wait();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = 0.0f;
            const int64_t o = z * t.dout + it.out[k];
            if (it.kind[k] >= 0) {
                ahead.read(stage, 0, k, y + z * t.din + it.in[k], v[k]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) sq[k] = fmaf(v[k][i], v[k][i], sq[k]);
            }
            if (it.out[k] >= 0) {
                ahead.read(stage, 1, k, residual + o, x[k]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) g0[k][i] = g1[k][i] = 0.0f;
                if (gz) ahead.read(stage, 2, k, gz + o, g0[k]);
                if (gh) ahead.read(stage, 3, k, gh + o, g1[k]);
            }
        }
        fetch(z + static_cast<int64_t>(kAhead) * gridDim.x, stage);
        in.add<K>(sq, it.bi, it.i0, it.i1);
        __syncthreads();
        float s_in[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (it.kind[k] < 0) continue;
            s_in[k] = rsqrtf(fmaf(in.get(it.bi[k]), inv_i[k], eps));
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[k][i] *= s_in[k];
            if (it.kind[k] != kGates) continue;
            float g[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) g[i] = it.cst[k] * gate_act(it.act[k], v[k][i] * wp[k][i]);
            Packed<float, VEC>::store(gates + it.slot[k], g);
        }
        __syncthreads();
        float val[K][VEC];      // the gated row; gated columns: the gate
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = dot[k] = 0.0f;
            if (it.out[k] < 0) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float n = v[k][i] * wp[k][i];
                if (it.kind[k] == kGated) {
                    val[k][i] = gates[it.gate[k][i]];
                    x[k][i] = fmaf(sc[k][i], n * val[k][i], x[k][i]);
                } else {
                    val[k][i] = it.cst[k] * gate_act(it.act[k], n);
                    x[k][i] = fmaf(sc[k][i], val[k][i], x[k][i]);
                }
                sq[k] = fmaf(x[k][i], x[k][i], sq[k]);
                dot[k] = fmaf(g1[k][i] * wn[k][i], x[k][i], dot[k]);
            }
        }
        if (gh) {
            outs.add<K>(sq, it.bo, it.o0, it.o1);
            ghs.add<K>(dot, it.bo, it.o0, it.o1);
            __syncthreads();
        }
        // cotangent of z, then of the normalised row (kept in g1), which for the gates needs the products of their channels
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (it.out[k] < 0) continue;
            if (gh) {
                const float s = rsqrtf(fmaf(outs.get(it.bo[k]), inv_o[k], eps)), mean = ghs.get(it.bo[k]) * inv_o[k] * s * s;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    a_pre[k][i] = fmaf(g1[k][i], x[k][i] * s, a_pre[k][i]);
                    g0[k][i] = fmaf(s, g1[k][i] * wn[k][i] - x[k][i] * mean, g0[k][i]);
                }
            }
            if (g_residual) Packed<T, VEC>::store(g_residual + z * t.dout + it.out[k], g0[k]);
            float pr[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float n = v[k][i] * wp[k][i], gv = g0[k][i] * sc[k][i];
                if (it.kind[k] == kGated) {
                    a_scale[k][i] = fmaf(g0[k][i], n * val[k][i], a_scale[k][i]);
                    g1[k][i] = gv * val[k][i];
                    pr[i] = gv * n;
                } else {
                    a_scale[k][i] = fmaf(g0[k][i], val[k][i], a_scale[k][i]);
                    g1[k][i] = gv * it.cst[k] * gate_act_grad(it.act[k], n);
                    pr[i] = 0.0f;
                }
            }
            if (it.kind[k] == kGated) Packed<float, VEC>::store(prod + it.out[k], pr);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            dot[k] = 0.0f;
            if (it.kind[k] < 0) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (it.kind[k] >= kGates) {
                    const int32_t* e = t.in_tbl + 4 * (it.in[k] + i);
                    float g = 0.0f;
                    for (int m = 0; m < e[3]; ++m) g += prod[e[2] + m];
                    g1[k][i] = it.kind[k] == kGates ? g * it.cst[k] * gate_act_grad(it.act[k], v[k][i] * wp[k][i]) : 0.0f;
                }
                a_post[k][i] = fmaf(g1[k][i], v[k][i], a_post[k][i]);
                g1[k][i] *= wp[k][i];
                dot[k] = fmaf(g1[k][i], v[k][i], dot[k]);
            }
        }
        if (gy) {
            dots.add<K>(dot, it.bi, it.i0, it.i1);
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (it.kind[k] < 0) continue;
                const float mean = dots.get(it.bi[k]) * inv_i[k];
#pragma unroll
                for (int i = 0; i < VEC; ++i) g1[k][i] = s_in[k] * (g1[k][i] - v[k][i] * mean);
                Packed<T, VEC>::store(gy + z * t.din + it.in[k], g1[k]);
            }
        }
    }
    if (partial) {
        Columns<VEC, K> ci, co;
#pragma unroll
        for (int k = 0; k < K; ++k) { ci.col[k] = it.kind[k] >= 0 ? it.in[k] : -1; co.col[k] = it.out[k]; }
        float* mine = partial + static_cast<int64_t>(blockIdx.x) * (t.nchan_in + 2 * t.nchan_out);
        store_channels<VEC, K>(ci, a_post, t.in_chan, t.nchan_in, smem, mine);
        store_channels<VEC, K>(co, a_scale, t.out_chan, t.nchan_out, smem, mine + t.nchan_in);
        store_channels<VEC, K>(co, a_pre, t.out_chan, t.nchan_out, smem, mine + t.nchan_in + t.nchan_out);
    }
}

// ----------------------------------------------------------------------------------------------------------- launches
struct Shape {
    int vec, k, threads, nw;
};

// Vectors of four where the irreps blocks and the pointers allow them, else single columns; up to 512 threads a row.
Shape row_shape(int widest, bool vec4) {
    Shape s;
    s.vec = vec4 ? 4 : 1;
    const int n = static_cast<int>(ceil_div(widest, s.vec));
    s.k = 1;
    while (s.k < 8 && n > s.k * kMaxThreads) s.k *= 2;
    s.threads = static_cast<int>(ceil_div(ceil_div(n, s.k), 32)) * 32;
    s.nw = static_cast<int>(ceil_div(s.threads / 32, 4)) * 4;
    return s;
}

template <typename F>
int resident_blocks(F kernel, int threads, size_t smem, int64_t rows, int* grid) {
    if (smem > 48 * 1024) E3B_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    int per_sm = 0;
    E3B_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem));
    if (per_sm < 1) return fail(E3B_ERR_UNSUPPORTED, "norm: the row does not fit a thread block");
    *grid = static_cast<int>(std::min<int64_t>(rows, static_cast<int64_t>(per_sm) * kNumSMs));
    return E3B_OK;
}

// f(element type, vector width, vectors a thread) with the three as types
template <typename T, typename F>
int by_shape(const Shape& s, F&& f) {
    if (s.vec == 4) {
        if (s.k == 1) return f(T(), Int<4>(), Int<1>());
        if (s.k == 2) return f(T(), Int<4>(), Int<2>());
        return f(T(), Int<4>(), Int<4>());
    }
    if (s.k == 1) return f(T(), Int<1>(), Int<1>());
    if (s.k == 2) return f(T(), Int<1>(), Int<2>());
    if (s.k == 4) return f(T(), Int<1>(), Int<4>());
    return f(T(), Int<1>(), Int<8>());
}
template <typename F>
int by_type(int type, const Shape& s, F&& f) {
    if (type == kFloat32) return by_shape<float>(s, f);
    if (type == kBFloat16) return by_shape<__nv_bfloat16>(s, f);
    return by_shape<__half>(s, f);
}

bool row_fits(int widest, bool vec4) { return widest <= (vec4 ? 4 * 4 : 8) * kMaxThreads; }      // of RMSNorm

int max_parts(int64_t rows) { return static_cast<int>(std::min<int64_t>(rows, 32 * kNumSMs)); }

}  // namespace
}  // namespace e3b

using namespace e3b;

extern "C" int e3b_norm_max_columns(int aligned) { return (aligned ? 4 * 4 : 8) * kMaxThreads; }

extern "C" int e3b_rms_norm_fwd(const void* x, const float* weight, const int32_t* table, const float* inv_count, int num_blocks,
                                int vec4, float eps, void* h, int64_t rows, int dim, int type, void* stream) {
    if (rows < 0 || dim < 0 || num_blocks < 0 || !known_type(type)) return fail(E3B_ERR_ARG, "rms_norm_fwd: bad size or type");
    if (rows == 0 || dim == 0) return E3B_OK;
    if (!x || !table || !inv_count || !h) return fail(E3B_ERR_ARG, "rms_norm_fwd: null pointer");
    const bool v4 = vec4 && dim % 4 == 0 && aligned_to(x, 4 * element_size(type)) && aligned_to(h, 4 * element_size(type));
    if (!row_fits(dim, v4)) return fail(E3B_ERR_UNSUPPORTED, "rms_norm_fwd: %d columns", dim);
    const Shape s = row_shape(dim, v4);
    const size_t smem = sizeof(float) * 2 * num_blocks * s.nw;
    return by_type(type, s, [&](auto t0, auto v0, auto k0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(v0)::value, K = decltype(k0)::value;
        int grid = 0;
        const int rc = resident_blocks(rms_fwd_kernel<T, VEC, K>, s.threads, smem, rows, &grid);
        if (rc != E3B_OK) return rc;
        rms_fwd_kernel<T, VEC, K><<<grid, s.threads, smem, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(x), weight, table, inv_count, eps, static_cast<T*>(h), rows, dim, num_blocks, s.nw);
        return check_launch("rms_norm_fwd");
    });
}

extern "C" int64_t e3b_norm_scratch_bytes(int64_t rows, int num_params) {
    return rows < 0 || num_params < 0 ? 0 : sizeof(float) * static_cast<int64_t>(max_parts(rows)) * num_params;
}

extern "C" int e3b_rms_norm_bwd(const void* x, const void* grad_h, const float* weight, const int32_t* table, const float* inv_count,
                                const int32_t* channels, int num_channels, int num_blocks, int vec4, float eps, void* grad_x,
                                float* grad_weight, void* scratch, int64_t scratch_bytes, int64_t rows, int dim, int type, void* stream) {
    if (rows < 0 || dim < 0 || num_blocks < 0 || num_channels < 0 || !known_type(type)) return fail(E3B_ERR_ARG, "rms_norm_bwd: bad size or type");
    if (dim == 0) return E3B_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        if (grad_weight) E3B_CUDA_TRY(cudaMemsetAsync(grad_weight, 0, sizeof(float) * num_channels, st));
        return E3B_OK;
    }
    if (!x || !grad_h || !table || !inv_count || !channels || (!grad_x && !grad_weight)) return fail(E3B_ERR_ARG, "rms_norm_bwd: null pointer");
    if (grad_weight && (!scratch || scratch_bytes < e3b_norm_scratch_bytes(rows, num_channels)))
        return fail(E3B_ERR_ARG, "rms_norm_bwd: scratch of %lld bytes is too small", static_cast<long long>(scratch_bytes));
    const int bytes = 4 * element_size(type);
    const bool v4 = vec4 && dim % 4 == 0 && aligned_to(x, bytes) && aligned_to(grad_h, bytes) && aligned_to(grad_x, bytes);
    if (!row_fits(dim, v4)) return fail(E3B_ERR_UNSUPPORTED, "rms_norm_bwd: %d columns", dim);
    const Shape s = row_shape(dim, v4);
    const size_t smem = sizeof(float) * (4 * num_blocks * s.nw + dim);
    int grid = 0;
    const int rc = by_type(type, s, [&](auto t0, auto v0, auto k0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(v0)::value, K = decltype(k0)::value;
        const int r = resident_blocks(rms_bwd_kernel<T, VEC, K>, s.threads, smem, rows, &grid);
        if (r != E3B_OK) return r;
        rms_bwd_kernel<T, VEC, K><<<grid, s.threads, smem, st>>>(
            static_cast<const T*>(x), static_cast<const T*>(grad_h), weight, table, inv_count, channels, num_channels, eps,
            static_cast<T*>(grad_x), grad_weight ? static_cast<float*>(scratch) : nullptr, rows, dim, num_blocks, s.nw);
        return check_launch("rms_norm_bwd");
    });
    if (rc != E3B_OK || !grad_weight || num_channels == 0) return rc;
    add_partials_kernel<<<static_cast<unsigned>(ceil_div(num_channels, 32)), dim3(32, 32), 0, st>>>(static_cast<const float*>(scratch),
                                                                                                   num_channels, grid, grad_weight);
    return check_launch("rms_norm_bwd sums");
}

namespace {
// f(element type, vector width, items a thread, threads of a block at most) with the four as types
template <typename T, typename F>
int by_items(const Shape& s, F&& f) {
    auto with_k = [&](auto v0) -> int {
        if (s.k == 1 && s.threads <= 160) return f(T(), v0, Int<1>(), Int<160>());
        if (s.k == 1 && s.threads <= 320) return f(T(), v0, Int<1>(), Int<320>());
        if (s.k == 1) return f(T(), v0, Int<1>(), Int<512>());
        if (s.k == 2) return f(T(), v0, Int<2>(), Int<512>());
        if constexpr (decltype(v0)::value == 1) {
            if (s.k == 8) return f(T(), v0, Int<8>(), Int<512>());
        }
        return f(T(), v0, Int<4>(), Int<512>());
    };
    if constexpr (sizeof(T) == 2) {
        if (s.vec == 8) return with_k(Int<8>());
    }
    return s.vec == 1 ? with_k(Int<1>()) : with_k(Int<4>());
}
template <typename F>
int by_type_and_items(int type, const Shape& s, F&& f) {
    if (type == kFloat32) return by_items<float>(s, f);
    if (type == kBFloat16) return by_items<__nv_bfloat16>(s, f);
    return by_items<__half>(s, f);
}

// Everything both directions check and derive.
int gate_row(const char* what, int type, const int32_t* sizes, const int32_t* items, const int32_t* in_tbl, const int32_t* out_tbl, const int32_t* in_chan,
             const int32_t* out_chan, const float* in_inv, const float* out_inv, GateRow* t, Shape* s) {
    *t = {items, in_tbl, out_tbl, in_chan, out_chan, in_inv, out_inv, sizes[1], sizes[2], sizes[3], sizes[4], sizes[5], sizes[6], sizes[7], sizes[8], 0};
    s->vec = sizes[0];
    if (s->vec != 1 && s->vec != 4 && (s->vec != 8 || type == kFloat32)) return fail(E3B_ERR_ARG, "%s: items of %d columns", what, s->vec);
    const int most = (s->vec == 1 ? 8 : 4) * kMaxThreads;
    if (t->num_items > most) return fail(E3B_ERR_UNSUPPORTED, "%s: %d items of %d columns, at most %d", what, t->num_items, s->vec, most);
    s->k = t->num_items <= kMaxThreads ? 1 : t->num_items <= 2 * kMaxThreads ? 2 : t->num_items <= 4 * kMaxThreads ? 4 : 8;
    s->threads = static_cast<int>(ceil_div(ceil_div(t->num_items, s->k), 32)) * 32;
    s->nw = t->nw = s->threads / 32;
    return E3B_OK;
}
}  // namespace

extern "C" int e3b_norm_gate_residual_fwd(const void* residual, const void* y, const float* weight_post, const float* scale,
                                          const float* weight_pre, const int32_t* items, const int32_t* in_table, const int32_t* out_table,
                                          const float* in_inv, const float* out_inv, const int32_t* sizes, float eps, void* z, void* h,
                                          int64_t rows, int type, void* stream) {
    if (!sizes || rows < 0 || !known_type(type)) return fail(E3B_ERR_ARG, "norm_gate_residual_fwd: bad size or type");
    if (rows == 0 || sizes[4] == 0) return E3B_OK;
    if (!residual || !y || !weight_post || !scale || !items || !in_table || !out_table || !in_inv || !out_inv || !z || (h && !weight_pre))
        return fail(E3B_ERR_ARG, "norm_gate_residual_fwd: null pointer");
    const int bytes = sizes[0] * element_size(type);
    if (!aligned_to(residual, bytes) || !aligned_to(y, bytes) || !aligned_to(z, bytes) || !aligned_to(h, bytes))
        return fail(E3B_ERR_ARG, "norm_gate_residual_fwd: rows must start on %d bytes", bytes);
    GateRow t;
    Shape s;
    const int rc = gate_row("norm_gate_residual_fwd", type, sizes, items, in_table, out_table, nullptr, nullptr, in_inv, out_inv, &t, &s);
    if (rc != E3B_OK) return rc;
    const int64_t floats = BlockSums::floats(t.nblk_in, t.nw) + BlockSums::floats(t.nblk_out, t.nw) + ceil_div(t.num_gates, 4) * 4;
    return by_type_and_items(type, s, [&](auto t0, auto v0, auto k0, auto m0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(v0)::value, K = decltype(k0)::value, MAXT = decltype(m0)::value, BLOCKS = MAXT == 160 ? 5 : MAXT == 320 ? 3 : 1;
        const size_t smem = sizeof(float) * floats + static_cast<size_t>(kAhead) * RowAhead<T, VEC, K, 2>::kStage * s.threads;
        int grid = 0;
        const int e = resident_blocks(norm_gate_fwd_kernel<T, VEC, K, MAXT, BLOCKS>, s.threads, smem, rows, &grid);
        if (e != E3B_OK) return e;
        norm_gate_fwd_kernel<T, VEC, K, MAXT, BLOCKS><<<grid, s.threads, smem, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(residual), static_cast<const T*>(y), weight_post, scale, weight_pre, t, eps, static_cast<T*>(z),
            static_cast<T*>(h), rows);
        return check_launch("norm_gate_residual_fwd");
    });
}

extern "C" int e3b_norm_gate_residual_bwd(const void* residual, const void* y, const void* grad_z, const void* grad_h,
                                          const float* weight_post, const float* scale, const float* weight_pre, const int32_t* items,
                                          const int32_t* in_table, const int32_t* out_table, const int32_t* in_channels,
                                          const int32_t* out_channels, const float* in_inv, const float* out_inv, const int32_t* sizes,
                                          float eps, void* grad_residual, void* grad_y, float* grad_params, void* scratch,
                                          int64_t scratch_bytes, int64_t rows, int type, void* stream) {
    if (!sizes || rows < 0 || !known_type(type)) return fail(E3B_ERR_ARG, "norm_gate_residual_bwd: bad size or type");
    const int params = sizes[7] + 2 * sizes[8];
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0 || sizes[4] == 0) {
        if (grad_params) E3B_CUDA_TRY(cudaMemsetAsync(grad_params, 0, sizeof(float) * params, st));
        return E3B_OK;
    }
    if (!residual || !y || (!grad_z && !grad_h) || !weight_post || !scale || !items || !in_table || !out_table || !in_channels || !out_channels ||
        !in_inv || !out_inv || (grad_h && !weight_pre))
        return fail(E3B_ERR_ARG, "norm_gate_residual_bwd: null pointer");
    if (grad_params && (!scratch || scratch_bytes < e3b_norm_scratch_bytes(rows, params)))
        return fail(E3B_ERR_ARG, "norm_gate_residual_bwd: scratch of %lld bytes is too small", static_cast<long long>(scratch_bytes));
    const int bytes = sizes[0] * element_size(type);
    if (!aligned_to(residual, bytes) || !aligned_to(y, bytes) || !aligned_to(grad_z, bytes) || !aligned_to(grad_h, bytes) ||
        !aligned_to(grad_residual, bytes) || !aligned_to(grad_y, bytes))
        return fail(E3B_ERR_ARG, "norm_gate_residual_bwd: rows must start on %d bytes", bytes);
    GateRow t;
    Shape s;
    const int bad = gate_row("norm_gate_residual_bwd", type, sizes, items, in_table, out_table, in_channels, out_channels, in_inv, out_inv, &t, &s);
    if (bad != E3B_OK) return bad;
    const int64_t floats = 2 * BlockSums::floats(t.nblk_in, t.nw) + 2 * BlockSums::floats(t.nblk_out, t.nw) + ceil_div(t.num_gates, 4) * 4 + ceil_div(t.dout, 4) * 4;
    int grid = 0;
    const int rc = by_type_and_items(type, s, [&](auto t0, auto v0, auto k0, auto m0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(v0)::value, K = decltype(k0)::value, MAXT = decltype(m0)::value, BLOCKS = MAXT == 160 ? 3 : MAXT == 320 ? 2 : 1;
        const size_t smem = std::max<size_t>(sizeof(float) * floats + static_cast<size_t>(kAhead) * RowAhead<T, VEC, K, 4>::kStage * s.threads, sizeof(float) * t.din);
        const int e = resident_blocks(norm_gate_bwd_kernel<T, VEC, K, MAXT, BLOCKS>, s.threads, smem, rows, &grid);
        if (e != E3B_OK) return e;
        norm_gate_bwd_kernel<T, VEC, K, MAXT, BLOCKS><<<grid, s.threads, smem, st>>>(
            static_cast<const T*>(residual), static_cast<const T*>(y), static_cast<const T*>(grad_z), static_cast<const T*>(grad_h), weight_post,
            scale, weight_pre, t, eps, static_cast<T*>(grad_residual), static_cast<T*>(grad_y), grad_params ? static_cast<float*>(scratch) : nullptr, rows);
        return check_launch("norm_gate_residual_bwd");
    });
    if (rc != E3B_OK || !grad_params || params == 0) return rc;
    add_partials_kernel<<<static_cast<unsigned>(ceil_div(params, 32)), dim3(32, 32), 0, st>>>(static_cast<const float*>(scratch), params,
                                                                                             grid, grad_params);
    return check_launch("norm_gate_residual_bwd sums");
}
