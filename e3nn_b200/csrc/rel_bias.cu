// Learned bias by distance buckets (the relative position bias of attention, on distances of atoms).
//
//   bucket[e] = number of thresholds t_i with t_i <= |pos[src[e]] - pos[dst[e]] + shift[e]|
//   bias[e, h] = table[bucket[e], h];     grad_table[b, h] = sum over the edges of bucket b of grad[e, h]
//
// Buckets: squared distances and squared thresholds are compared in fp64, where the fp32 inputs and their differences are
// exact to 2^-53, so that a distance next to a border falls on the side that it is on.  28 bytes of edge data in, 4 out, and two
// positions from L2 that wait for the indices: 2,097,152 edges 27 us (67 MB, 2.5 TB/s), bound by those dependent loads.
// Bias: writes 4 H bytes an edge (2 H in 16 bits): 2,097,152 edges of 16 heads in fp32 36 us = 4.0 TB/s, in bf16 36 us too: a table entry is
// looked up per output.
// Gradient: every thread keeps its heads and walks edges of its own; it adds into cells of a table in shared memory that no other
// thread touches, so the order of the additions is fixed by the grid; slices, then thread blocks, are added in order.  No atomics.
// Bound by the loads in flight: a table per slice limits the threads, sixteen 16-byte loads each make up for it: 2,097,152 edges, 16 heads, 64 buckets
// in fp32 60 us = 2.4 TB/s (one head a thread: 98 us), in bf16 54 us; 8 heads, 256 buckets in bf16, where only 26 slices fit, 79 us.  Tables that do
// not fit (more than 1,664 buckets of 32 heads) are taken in windows of buckets, each of which reads all edges.
#include <algorithm>

#include "common.cuh"
#include "typed.cuh"

namespace e3b {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBuckets = 1024;      // of the distance buckets (their thresholds lie in shared memory); a table may have more
constexpr int64_t kMostCells = INT32_MAX - 32;      // of a table
constexpr int kSumThreads = 512;       // of a block of the table gradient, at most

__global__ void __launch_bounds__(kThreads) distance_buckets_kernel(const float* __restrict__ pos, const int64_t* __restrict__ src,
                                                                    const int64_t* __restrict__ dst, const float* __restrict__ shift,
                                                                    const double* __restrict__ thresholds2, int num, int64_t edges,
                                                                    int64_t nodes, int32_t* __restrict__ buckets, int32_t* status) {
    __shared__ double t2[kMaxBuckets];
    for (int i = threadIdx.x; i < num; i += kThreads) t2[i] = thresholds2[i];
    __syncthreads();
    constexpr int U = 2;       // edges a thread looks at side by side
    const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t e0 = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; e0 < edges; e0 += U * stride) {
        double r2[U];
        bool bad[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t e = min(e0 + u * stride, edges - 1);
            int64_t a = src[e], b = dst[e];
            bad[u] = a < 0 || a >= nodes || b < 0 || b >= nodes;
            if (bad[u]) a = b = -1;
            r2[u] = 0.0;
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                double d = bad[u] ? 0.0 : static_cast<double>(pos[3 * a + i]) - static_cast<double>(pos[3 * b + i]);
                if (shift) d += static_cast<double>(shift[3 * e + i]);
                r2[u] = __dadd_rn(r2[u], __dmul_rn(d, d));
            }
        }
        int lo[U], hi[U];                           // thresholds below lo are <= r, from hi on they are > r
#pragma unroll
        for (int u = 0; u < U; ++u) { lo[u] = 0; hi[u] = num; }
        for (int left = num; left > 0; left >>= 1) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (lo[u] >= hi[u]) continue;
                const int mid = (lo[u] + hi[u]) >> 1;
                if (t2[mid] <= r2[u]) lo[u] = mid + 1; else hi[u] = mid;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t e = e0 + u * stride;
            if (e >= edges) continue;
            buckets[e] = bad[u] ? 0 : lo[u];
            if (bad[u]) *status = 2;
        }
    }
}

// VEC outputs of the flat [edges * heads] array a thread.  INDEX: 32 bits where they hold it (a division of 64-bit numbers costs more than the rest).
template <typename T, int VEC, typename INDEX>
__global__ void __launch_bounds__(kThreads) bias_fwd_kernel(const T* __restrict__ table, const int32_t* __restrict__ buckets, int num_buckets,
                                                            int heads, int64_t total, T* __restrict__ out, int32_t* status) {
    const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads * VEC;
    for (int64_t i0 = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * VEC; i0 < total; i0 += stride) {
        float v[VEC];
        int64_t e = static_cast<INDEX>(i0) / static_cast<INDEX>(heads);
        int h = static_cast<int>(i0 - e * heads);
        int b = buckets[e];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if (i > 0 && ++h == heads) {
                h = 0;
                ++e;
                if (i0 + i < total) b = buckets[e];
            }
            const bool ok = b >= 0 && b < num_buckets;
            if (!ok && i0 + i < total) *status = 2;
            v[i] = ok ? to_float(table[b * heads + h]) : 0.0f;
        }
        if (VEC == 1 || i0 + VEC <= total) {
            Packed<T, VEC>::store(out + i0, v);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (i0 + i < total) out[i0 + i] = from_float<T>(v[i]);
        }
    }
}

// Thread t of a block: HV heads from HV (t % lanes) on (lanes = width / HV), slice t / lanes; its block's edges in turns of `slices`.
// Shared memory: [slices][window][width]: the buckets from blockIdx.z * window on (all of them, unless the table is large).
template <typename T, int HV, bool WINDOWS>
__global__ void __launch_bounds__(kSumThreads, 1) bias_bwd_kernel(const T* __restrict__ grad, const int32_t* __restrict__ buckets, int num_buckets,
                                                                  int window, int heads, int width, int slices, int64_t edges, int64_t edges_per_block,
                                                                  float* __restrict__ partial, int32_t* status) {
    extern __shared__ __align__(16) float acc[];
    const int lanes = width / HV, h = threadIdx.x % lanes * HV, slice = threadIdx.x / lanes, head = blockIdx.y * width + h;
    const int first = WINDOWS ? blockIdx.z * window : 0, here = WINDOWS ? min(window, num_buckets - first) : num_buckets, cells = here * width;
    for (int i = threadIdx.x; i < slices * cells; i += blockDim.x) acc[i] = 0.0f;
    __syncthreads();
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * edges_per_block;
    const int count = static_cast<int>(min(edges_per_block, edges - begin));
    if (head < heads && slice < slices) {
        float* mine = acc + slice * cells + h;
        const T* from = grad + begin * heads + head;
        const int32_t* which = buckets + begin;
        constexpr int U = 16;       // edges in flight a thread
        bool bad = false;
        for (int e0 = slice; e0 < count; e0 += U * slices) {
            int b[U];
            Packed<T, HV> g[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int e = min(e0 + u * slices, count - 1);
                b[u] = which[e];
                g[u].load(from + static_cast<int64_t>(e) * heads);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (e0 + u * slices >= count) break;
                const int at = b[u] - first;
                float x[HV], y[HV];
                if (at < 0 || at >= here) {      // bad, if there is anything to add: slots of no row may name any bucket
                    g[u].unpack(y);
#pragma unroll
                    for (int i = 0; i < HV; ++i) bad = bad || (y[i] != 0.0f && (!WINDOWS || b[u] < 0 || b[u] >= num_buckets));
                    continue;
                }
                Packed<float, HV> sum;
                sum.load(mine + at * width);
                sum.unpack(x);
                g[u].unpack(y);
#pragma unroll
                for (int i = 0; i < HV; ++i) x[i] += y[i];
                Packed<float, HV>::store(mine + at * width, x);
            }
        }
        if (bad) *status = 2;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < cells; i += blockDim.x) {
        const int b = i / width, hh = i % width;
        if (static_cast<int>(blockIdx.y) * width + hh >= heads) continue;
        float s = 0.0f;
        for (int k = 0; k < slices; ++k) s += acc[k * cells + i];
        partial[(static_cast<int64_t>(blockIdx.x) * num_buckets + first + b) * heads + blockIdx.y * width + hh] = s;
    }
}

// 32 cells a block, 32 slices of the thread blocks' partial tables.
template <typename T>
__global__ void __launch_bounds__(1024) bias_sum_kernel(const float* __restrict__ partial, int cells, int parts, T* __restrict__ out) {
    __shared__ float s[32][33];
    const int i = blockIdx.x * 32 + threadIdx.x;
    float a = 0.0f;
    if (i < cells) {
#pragma unroll 4
        for (int p = threadIdx.y; p < parts; p += 32) a += partial[static_cast<int64_t>(p) * cells + i];
    }
    s[threadIdx.x][threadIdx.y] = a;
    __syncthreads();
    const float t = warp_sum(s[threadIdx.y][threadIdx.x]);
    const int cell = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && cell < cells) out[cell] = from_float<T>(t);
}

// How the table gradient is split: heads a thread and a block take, buckets and slices of edges of a block, thread blocks.  The tables of the
// slices fill the shared memory of an SM; a wide vector of heads a thread keeps the loads in flight when that leaves few threads.
struct BiasSplit {
    int vec, width, slices, groups, parts, window;
    int64_t per_block;
    size_t smem;
};
BiasSplit bias_split(int64_t edges, int heads, int num_buckets, int element) {
    BiasSplit s;
    constexpr size_t kMostSmem = 208 * 1024;
    s.vec = element == 2 && heads % 8 == 0 ? 8 : heads % 4 == 0 ? 4 : 1;
    s.width = std::min(heads, 32);
    s.window = static_cast<int>(std::min<size_t>(num_buckets, kMostSmem / (sizeof(float) * s.width)));      // every block reads the buckets of its edges, whatever its window
    const size_t table = sizeof(float) * s.window * s.width;
    s.groups = static_cast<int>(ceil_div(heads, s.width));
    // a block clears, sums and writes its tables: every slice takes at least some edges
    const int64_t a_block = ceil_div(edges, kNumSMs);
    s.slices = static_cast<int>(std::max<size_t>(1, std::min<size_t>(kSumThreads * s.vec / s.width, kMostSmem / table)));
    s.slices = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(s.slices, ceil_div(a_block, 16))));
    while (s.vec > 1 && s.slices * s.width / s.vec < 128) s.vec = s.vec == 8 ? 4 : 1;      // few slices: more threads, each with fewer heads
    s.smem = table * s.slices;
    const int64_t least = std::max<int64_t>(16 * s.slices, num_buckets / 4);
    s.parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ceil_div(edges, least), kNumSMs)));
    s.per_block = ceil_div(std::max<int64_t>(edges, 1), s.parts);
    return s;
}

int flat_grid(int64_t items) { return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ceil_div(items, kThreads), kNumSMs * 16))); }

template <typename T>
int bias_fwd(const void* table, const int32_t* buckets, int num_buckets, int heads, int64_t edges, void* out, int32_t* status, cudaStream_t st) {
    const int64_t total = edges * heads;
    const bool v4 = aligned_to(out, 4 * sizeof(T));
    const T* tab = static_cast<const T*>(table);
    T* o = static_cast<T*>(out);
    const int grid = flat_grid(v4 ? ceil_div(total, 4) : total);
    if (v4 && total < UINT32_MAX) bias_fwd_kernel<T, 4, uint32_t><<<grid, kThreads, 0, st>>>(tab, buckets, num_buckets, heads, total, o, status);
    else if (v4) bias_fwd_kernel<T, 4, int64_t><<<grid, kThreads, 0, st>>>(tab, buckets, num_buckets, heads, total, o, status);
    else bias_fwd_kernel<T, 1, int64_t><<<grid, kThreads, 0, st>>>(tab, buckets, num_buckets, heads, total, o, status);
    return check_launch("relative_bias_fwd");
}

template <typename T>
int bias_bwd(const void* grad, const int32_t* buckets, int num_buckets, int heads, int64_t edges, void* grad_table, float* partial,
             int table_type, int32_t* status, cudaStream_t st) {
    const BiasSplit s = bias_split(edges, heads, num_buckets, sizeof(T));
    auto launch = [&](auto v0) -> int {
        constexpr int HV = decltype(v0)::value;
        const unsigned windows = static_cast<unsigned>(ceil_div(num_buckets, s.window));
        const auto kernel = windows > 1 ? bias_bwd_kernel<T, HV, true> : bias_bwd_kernel<T, HV, false>;      // (with windows 64 in the place of 60 us on the case above)
        const int allowed = allow_smem(kernel, s.smem);
        if (allowed != E3B_OK) return allowed;
        if (windows > 65535 || s.groups > 65535) return fail(E3B_ERR_UNSUPPORTED, "relative_bias_bwd: a table of %d buckets and %d heads", num_buckets, heads);
        kernel<<<dim3(s.parts, s.groups, windows), s.width / HV * s.slices, s.smem, st>>>(
            static_cast<const T*>(grad), buckets, num_buckets, s.window, heads, s.width, s.slices, edges, s.per_block, partial, status);
        return check_launch("relative_bias_bwd");
    };
    if (!aligned_to(grad, s.vec * sizeof(T))) return fail(E3B_ERR_ARG, "relative_bias_bwd: the gradient must start on %d bytes", static_cast<int>(s.vec * sizeof(T)));
    int rc;
    if constexpr (sizeof(T) == 2) rc = s.vec == 8 ? launch(Int<8>()) : s.vec == 4 ? launch(Int<4>()) : launch(Int<1>());
    else rc = s.vec == 4 ? launch(Int<4>()) : launch(Int<1>());
    if (rc != E3B_OK) return rc;
    const int cells = num_buckets * heads;
    const dim3 block(32, 32);
    const int grid = (cells + 31) / 32;
    if (table_type == kFloat32) bias_sum_kernel<<<grid, block, 0, st>>>(partial, cells, s.parts, static_cast<float*>(grad_table));
    else if (table_type == kBFloat16) bias_sum_kernel<<<grid, block, 0, st>>>(partial, cells, s.parts, static_cast<__nv_bfloat16*>(grad_table));
    else bias_sum_kernel<<<grid, block, 0, st>>>(partial, cells, s.parts, static_cast<__half*>(grad_table));
    return check_launch("relative_bias_bwd sums");
}

}  // namespace
}  // namespace e3b

using namespace e3b;

extern "C" int e3b_distance_buckets(const float* pos, const int64_t* edge_src, const int64_t* edge_dst, const float* shift,
                                    const double* thresholds_squared, int num_thresholds, int64_t num_edges, int64_t num_nodes,
                                    int32_t* buckets, int32_t* status, void* stream) {
    if (num_edges < 0 || num_nodes < 0 || num_thresholds < 0 || num_thresholds >= kMaxBuckets) return fail(E3B_ERR_ARG, "distance_buckets: bad size");
    if (num_edges == 0) return E3B_OK;
    if ((num_nodes > 0 && !pos) || !edge_src || !edge_dst || (num_thresholds > 0 && !thresholds_squared) || !buckets || !status)
        return fail(E3B_ERR_ARG, "distance_buckets: null pointer");
    distance_buckets_kernel<<<flat_grid(ceil_div(num_edges, 2)), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        pos, edge_src, edge_dst, shift, thresholds_squared, num_thresholds, num_edges, num_nodes, buckets, status);
    return check_launch("distance_buckets");
}

extern "C" int e3b_relative_bias_fwd(const void* table, const int32_t* buckets, int num_buckets, int num_heads, int64_t num_edges, int type,
                                     void* bias, int32_t* status, void* stream) {
    if (num_edges < 0 || num_buckets < 1 || num_heads < 1 || !known_type(type)) return fail(E3B_ERR_ARG, "relative_bias_fwd: bad size or type");
    if (static_cast<int64_t>(num_buckets) * num_heads > kMostCells) return fail(E3B_ERR_UNSUPPORTED, "relative_bias_fwd: a table of %d buckets and %d heads", num_buckets, num_heads);
    if (num_edges == 0) return E3B_OK;
    if (!table || !buckets || !bias || !status) return fail(E3B_ERR_ARG, "relative_bias_fwd: null pointer");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (type == kFloat32) return bias_fwd<float>(table, buckets, num_buckets, num_heads, num_edges, bias, status, st);
    if (type == kBFloat16) return bias_fwd<__nv_bfloat16>(table, buckets, num_buckets, num_heads, num_edges, bias, status, st);
    return bias_fwd<__half>(table, buckets, num_buckets, num_heads, num_edges, bias, status, st);
}

extern "C" int64_t e3b_relative_bias_scratch_bytes(int64_t num_edges, int num_buckets, int num_heads) {
    if (num_edges < 0 || num_buckets < 1 || num_heads < 1) return 0;
    const int parts = std::max(bias_split(num_edges, num_heads, num_buckets, 2).parts, bias_split(num_edges, num_heads, num_buckets, 4).parts);
    return sizeof(float) * static_cast<int64_t>(parts) * num_buckets * num_heads;
}

extern "C" int e3b_relative_bias_bwd(const void* grad_bias, const int32_t* buckets, int num_buckets, int num_heads, int64_t num_edges, int type,
                                     void* grad_table, int table_type, void* scratch, int64_t scratch_bytes, int32_t* status, void* stream) {
    if (num_edges < 0 || num_buckets < 1 || num_heads < 1 || !known_type(type) || !known_type(table_type))
        return fail(E3B_ERR_ARG, "relative_bias_bwd: bad size or type");
    if (static_cast<int64_t>(num_buckets) * num_heads > kMostCells) return fail(E3B_ERR_UNSUPPORTED, "relative_bias_bwd: a table of %d buckets and %d heads", num_buckets, num_heads);
    if (!grad_table) return fail(E3B_ERR_ARG, "relative_bias_bwd: null pointer");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (num_edges == 0) {
        E3B_CUDA_TRY(cudaMemsetAsync(grad_table, 0, static_cast<size_t>(element_size(table_type)) * num_buckets * num_heads, st));
        return E3B_OK;
    }
    if (!grad_bias || !buckets || !scratch || !status) return fail(E3B_ERR_ARG, "relative_bias_bwd: null pointer");
    if (scratch_bytes < e3b_relative_bias_scratch_bytes(num_edges, num_buckets, num_heads)) return fail(E3B_ERR_ARG, "relative_bias_bwd: scratch of %lld bytes is too small", static_cast<long long>(scratch_bytes));
    float* partial = static_cast<float*>(scratch);
    if (type == kFloat32) return bias_bwd<float>(grad_bias, buckets, num_buckets, num_heads, num_edges, grad_table, partial, table_type, status, st);
    if (type == kBFloat16) return bias_bwd<__nv_bfloat16>(grad_bias, buckets, num_buckets, num_heads, num_edges, grad_table, partial, table_type, status, st);
    return bias_bwd<__half>(grad_bias, buckets, num_buckets, num_heads, num_edges, grad_table, partial, table_type, status, st);
}
