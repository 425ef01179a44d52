// RMSNorm on rows of irreps features.
//
// A row is a list of blocks, block b with mul_b channels of d_b = 2l+1 components (n_b = mul_b d_b columns):
//   h[b, u, m] = w[b, u] x[b, u, m] s_b,   s_b = (sum_{u,m} x[b, u, m]^2 / n_b + eps)^(-1/2)
// Gradient: with t = g w (cotangent times weight), gx = s (t - x s^2 mean_b(t x)), gw = sum over rows and m of g x s.
//
// Every row is read once and written once in its own type, sums and products are fp32.  One thread block per
// row at a time (blocks walk the rows), thread t owns the same columns of every row, so weights and the sums of their gradient
// stay in registers.  Sums over a block of the irreps: a warp reduces per irreps block (its columns touch one to three), the
// warps' sums are added in the order of the warps.  The next row is loaded before the present one is reduced.
// 262,144 rows of 576 columns in fp32: 232 us forward (5.2 TB/s, 79 % of a copy), 422 us gradient (4.3 TB/s); in bf16 264 and 510 us for half the
// bytes: there the work of a row, its sums and its barrier bound it.  Rows of single columns (17x0e+9x1o+5x2e, 69 columns): 132 and 208 us in
// fp32 and in bf16 alike.  4,001 rows of 288 columns in fp32: 5.5 us forward, 7.5 us gradient and 6.2 us for the sums of the thread blocks' weight
// gradients (9 and 14 MB moved: the latency of a few dependent rows).
#include "norm.cuh"

namespace e3b {
namespace {

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

template <typename T, int VEC, int K>
__global__ void __launch_bounds__(kMaxThreads) rms_bwd_kernel(const T* __restrict__ x, const T* __restrict__ gh, const float* __restrict__ weight,
                                                              const int32_t* __restrict__ tbl, const float* __restrict__ inv_n,
                                                              const int32_t* __restrict__ chan, int nchan, float eps, T* __restrict__ gx,
                                                              float* __restrict__ partial, int64_t rows, int dim, int nblk, int nw, int turns) {
    extern __shared__ float smem[];
    // two rows' shares in turn; of rows with so many blocks that they do not fit twice one row's, which the weights' sums replace at the end
    float* red = smem;                                            // [turns][2 sums][nblk][nw]
    float* buf = smem + (turns == 2 ? 4 * nblk * nw : 0);         // [dim]
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
    for (int i = threadIdx.x; i < turns * 2 * nblk * nw; i += blockDim.x) red[i] = 0.0f;
    __syncthreads();
    Packed<T, VEC> nx[K], ng[K];
    int64_t z = blockIdx.x;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (c.col[k] >= 0) { nx[k].load(x + z * dim + c.col[k]); ng[k].load(gh + z * dim + c.col[k]); }
    for (int turn = 0; z < rows; z += gridDim.x, turn ^= turns - 1) {
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
        if (turns == 1) __syncthreads();
    }
    if (!partial) return;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (c.col[k] < 0) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) buf[c.col[k] + i] = acc[k][i];
    }
    __syncthreads();
    store_channels(buf, chan, nchan, partial + static_cast<int64_t>(blockIdx.x) * nchan);
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

constexpr size_t kMostSmem = 226 * 1024;      // that allow_smem allows
bool row_fits(int widest, bool vec4) { return widest <= (vec4 ? 4 * 4 : 8) * kMaxThreads; }      // of RMSNorm

}  // namespace
}  // namespace e3b

using namespace e3b;

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

extern "C" int64_t e3b_norm_scratch_bytes(int64_t rows, int num_params) { return norm_scratch_bytes(rows, num_params); }

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
    // what the forward kernel takes fits here too: with one row's shares at a time, as many bytes as two rows' there
    const size_t twice = sizeof(float) * (4 * static_cast<size_t>(num_blocks) * s.nw + dim);
    const int turns = twice <= kMostSmem ? 2 : 1;
    const size_t smem = turns == 2 ? twice : std::max(sizeof(float) * 2 * static_cast<size_t>(num_blocks) * s.nw, sizeof(float) * static_cast<size_t>(dim));
    int grid = 0;
    const int rc = by_type(type, s, [&](auto t0, auto v0, auto k0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(v0)::value, K = decltype(k0)::value;
        const int r = resident_blocks(rms_bwd_kernel<T, VEC, K>, s.threads, smem, rows, &grid);
        if (r != E3B_OK) return r;
        rms_bwd_kernel<T, VEC, K><<<grid, s.threads, smem, st>>>(
            static_cast<const T*>(x), static_cast<const T*>(grad_h), weight, table, inv_count, channels, num_channels, eps,
            static_cast<T*>(grad_x), grad_weight ? static_cast<float*>(scratch) : nullptr, rows, dim, num_blocks, s.nw, turns);
        return check_launch("rms_norm_bwd");
    });
    if (rc != E3B_OK || !grad_weight || num_channels == 0) return rc;
    add_partials_kernel<<<static_cast<unsigned>(ceil_div(num_channels, 32)), dim3(32, 32), 0, st>>>(static_cast<const float*>(scratch),
                                                                                                   num_channels, grid, grad_weight);
    return check_launch("rms_norm_bwd sums");
}

