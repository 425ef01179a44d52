// Shared by the norm kernels: sums over the blocks of the irreps, parameter gradients, launches.
#pragma once
#include <algorithm>

#include "common.cuh"
#include "gate_act.cuh"
#include "typed.cuh"

namespace e3b {
namespace {

constexpr int kMaxThreads = 512;

// Sums over the irreps blocks of a row by the warps that touch a block.  share: [nblk][nw], nw the number of warps rounded up to a power
// of two; what a warp does not touch stays at the zero from the start of the kernel.
struct BlockSums {
    float* share;
    int nblk, nw;
    __device__ __forceinline__ void clear() const {
        for (int i = threadIdx.x; i < nblk * nw; i += blockDim.x) share[i] = 0.0f;
    }
    // shares of this warp's items: K values of the blocks vb, M of the blocks wb (0 where there is no item); `blocks`: what it touches
    template <int K, int M>
    __device__ __forceinline__ void add(unsigned blocks, const float (&v)[K], const int (&vb)[K], const float (&w)[M], const int (&wb)[M]) const {
        for (; blocks; blocks &= blocks - 1) {
            const int b = __ffs(blocks) - 1;
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) s += vb[k] == b ? v[k] : 0.0f;
#pragma unroll
            for (int j = 0; j < M; ++j) s += wb[j] == b ? w[j] : 0.0f;
            s = warp_sum(s);
            if ((threadIdx.x & 31) == 0) share[b * nw + (threadIdx.x >> 5)] = s;
        }
    }
    // sums of the blocks vb and wb (whole warps; after a barrier): 32 / nw blocks at a time, nw lanes each
    template <int K, int M>
    __device__ __forceinline__ void get(const int (&vb)[K], float (&v)[K], const int (&wb)[M], float (&w)[M]) const {
        const int lane = threadIdx.x & 31, at_once = 32 / nw;
        for (int b0 = 0; b0 < nblk; b0 += at_once) {
            const int i = b0 * nw + lane;
            float s = i < nblk * nw ? share[i] : 0.0f;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1)
                if (o < nw) s += __shfl_xor_sync(0xffffffffu, s, o);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const float t = __shfl_sync(0xffffffffu, s, (vb[k] - b0) * nw & 31);
                if (vb[k] >= b0 && vb[k] < b0 + at_once) v[k] = t;
            }
#pragma unroll
            for (int j = 0; j < M; ++j) {
                const float t = __shfl_sync(0xffffffffu, s, (wb[j] - b0) * nw & 31);
                if (wb[j] >= b0 && wb[j] < b0 + at_once) w[j] = t;
            }
        }
    }
    __host__ __device__ static int floats(int nblk, int nw) { return (nblk * nw + 3) / 4 * 4; }
};
inline int warps_pow2(int threads) {
    int n = 1;
    while (n * 32 < threads) n *= 2;
    return n;
}
__device__ __forceinline__ BlockSums block_sums_at(float*& p, int nblk, int nw) {
    BlockSums b{p, nblk, nw};
    p += BlockSums::floats(nblk, nw);
    return b;
}

// A thread block's row of the parameter gradients: columns already summed over its rows lie in `columns`, channel u has
// chan[2u + 1] of them from chan[2u] on.
__device__ __forceinline__ void store_channels(const float* columns, const int32_t* __restrict__ chan, int nchan, float* __restrict__ partial) {
    for (int u = threadIdx.x; u < nchan; u += blockDim.x) {
        float s = 0.0f;
        const int first = chan[2 * u], n = chan[2 * u + 1];
        for (int m = 0; m < n; ++m) s += columns[first + m];
        partial[u] = s;
    }
}

// Parameter gradient: the thread blocks' partial rows added in a fixed order.  32 channels a block, 32 slices of the rows.
static __global__ void __launch_bounds__(1024) add_partials_kernel(const float* __restrict__ partial, int n, int parts, float* __restrict__ out) {
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

// Thread blocks of a persistent launch: all that fit on the GPU, at most one a row.  The query of the last shape is kept, one
// per kernel and host thread (it costs about as much as the launch).
template <typename F>
int resident_blocks(F kernel, int threads, size_t smem, int64_t rows, int* grid) {
    struct Last {
        F kernel;
        int threads, per_sm, device;
        size_t smem;
    };
    static thread_local Last last[8] = {};
    static thread_local int next = 0;
    int device = 0;
    E3B_CUDA_TRY(cudaGetDevice(&device));
    const Last* hit = nullptr;
    for (const Last& l : last)
        if (l.kernel == kernel && l.threads == threads && l.smem == smem && l.device == device) hit = &l;
    if (!hit) {
        int per_sm = 0;
        const int rc = allow_smem(kernel, smem);
        if (rc != E3B_OK) return rc;
        E3B_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem));
        if (per_sm < 1) return fail(E3B_ERR_UNSUPPORTED, "norm: the row does not fit a thread block");
        last[next] = {kernel, threads, per_sm, device, smem};
        hit = &last[next];
        next = (next + 1) % 8;
    }
    *grid = static_cast<int>(std::min<int64_t>(rows, static_cast<int64_t>(hit->per_sm) * kNumSMs));
    return E3B_OK;
}

inline int max_parts(int64_t rows) { return static_cast<int>(std::min<int64_t>(rows, 32 * kNumSMs)); }
inline int64_t norm_scratch_bytes(int64_t rows, int num_params) {
    return rows < 0 || num_params < 0 ? 0 : sizeof(float) * static_cast<int64_t>(max_parts(rows)) * num_params;
}

}  // namespace
}  // namespace e3b
