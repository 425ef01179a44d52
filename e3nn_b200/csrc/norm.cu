// Norms on rows of irreps features and the boundary between two residual blocks.
//
// A row is a list of blocks, block b with mul_b channels of d_b = 2l+1 components (n_b = mul_b d_b columns):
//   norm(x)[b, u, m] = w[b, u] * x[b, u, m] * s_b(x),   s_b(x) = (sum_{u,m} x[b, u, m]^2 / n_b + eps)^(-1/2)
// e3b_rms_norm:       h = norm(x; w)                                       the norm before a block
// e3b_norm_gate_residual:  n = norm(y; w_post),  g = gate(n)               the norm after it, Gate (gate.cu),
//                     z = residual + scale * g,  h = norm(z; w_pre)        residual, norm before the next block
// Gradient of norm: with t = g w (cotangent times weight), gx = s (t - x s^2 mean_b(t x)), gw = sum over rows and m of g x s.
//
// Bound by HBM: every row is read once and written once in its own type; sums, products and the row between the steps are
// fp32 (h is taken from z before z is rounded).  One thread block per row at a time (blocks walk the rows), thread t owns the
// same VEC columns of every row, so weights and table entries stay in registers and the sums of the parameter gradients
// too; the normalised row goes through shared memory because a gated column reads its gate from another part of it.
// Sums over a block of the irreps: a warp reduces per irreps block (its columns touch one to three), the warps' sums are
// added in the order of the warps.  The next row is loaded before the present one is reduced.
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
struct GateRow {
    const int32_t* in_tbl;     // [din][4]  {irreps block, channel, activation, constant (bits)}
    const int32_t* out_tbl;    // [dout][4] {irreps block, channel, input column, gate column or -1}
    const int32_t* back_tbl;   // [din][4]  {0 scalar / 1 gated / 2 gate / 3 unused, first output column, count, partner column}
    const int32_t* in_chan;    // [nchan_in][2]  {first column, components}
    const int32_t* out_chan;   // [nchan_out][2]
    const float* in_inv;       // [nblk_in]  1 / n_b
    const float* out_inv;      // [nblk_out]
    int din, dout, nblk_in, nblk_out, nchan_in, nchan_out, nw;
};

template <typename T, int VEC, int K>
__global__ void __launch_bounds__(kMaxThreads) norm_gate_fwd_kernel(const T* __restrict__ residual, const T* __restrict__ y,
                                                                    const float* __restrict__ w_post, const float* __restrict__ scale,
                                                                    const float* __restrict__ w_pre, GateRow t, float eps,
                                                                    T* __restrict__ z_out, T* __restrict__ h_out, int64_t rows) {
    extern __shared__ float smem[];
    float* red_in = smem;                                // [nblk_in][nw]
    float* red_out = red_in + t.nblk_in * t.nw;          // [nblk_out][nw]
    float* val = red_out + t.nblk_out * t.nw;            // [din] normalised row, scalars and gates activated
    Columns<VEC, K> ci, co;
    ci.init(t.in_tbl, t.din);
    co.init(t.out_tbl, t.dout);
    float wp[K][VEC], cst[K][VEC], sc[K][VEC], wn[K][VEC], inv_i[K], inv_o[K];
    int act[K][VEC], src[K][VEC], gate[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        inv_i[k] = ci.col[k] >= 0 ? t.in_inv[ci.blk[k]] : 0.0f;
        inv_o[k] = co.col[k] >= 0 ? t.out_inv[co.blk[k]] : 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if (ci.col[k] >= 0) {
                const int32_t* e = t.in_tbl + 4 * (ci.col[k] + i);
                wp[k][i] = w_post[e[1]];
                act[k][i] = e[2];
                cst[k][i] = __int_as_float(e[3]);
            }
            if (co.col[k] >= 0) {
                const int32_t* e = t.out_tbl + 4 * (co.col[k] + i);
                sc[k][i] = scale[e[1]];
                wn[k][i] = w_pre ? w_pre[e[1]] : 0.0f;
                src[k][i] = e[2];
                gate[k][i] = e[3];
            }
        }
    }
    for (int i = threadIdx.x; i < (t.nblk_in + t.nblk_out) * t.nw; i += blockDim.x) smem[i] = 0.0f;
    __syncthreads();
    Packed<T, VEC> ny[K], nr[K];
    int64_t z = blockIdx.x;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (ci.col[k] >= 0) ny[k].load(y + z * t.din + ci.col[k]);
        if (co.col[k] >= 0) nr[k].load(residual + z * t.dout + co.col[k]);
    }
    for (; z < rows; z += gridDim.x) {
        const int64_t zn = z + gridDim.x;
        float v[K][VEC], o[K][VEC], sq[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = 0.0f;
            if (ci.col[k] >= 0) {
                ny[k].unpack(v[k]);
#pragma unroll
                for (int i = 0; i < VEC; ++i) sq[k] = fmaf(v[k][i], v[k][i], sq[k]);
                if (zn < rows) ny[k].load(y + zn * t.din + ci.col[k]);
            }
            if (co.col[k] >= 0) {
                nr[k].unpack(o[k]);
                if (zn < rows) nr[k].load(residual + zn * t.dout + co.col[k]);
            }
        }
        warp_shares<VEC, K>(ci, sq, red_in, t.nw);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (ci.col[k] < 0) continue;
            const float s = rsqrtf(fmaf(add_shares(red_in + ci.blk[k] * t.nw, t.nw), inv_i[k], eps));
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[k][i] = cst[k][i] * gate_act(act[k][i], v[k][i] * s * wp[k][i]);
            Packed<float, VEC>::store(val + ci.col[k], v[k]);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = 0.0f;
            if (co.col[k] < 0) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float g = val[src[k][i]] * (gate[k][i] >= 0 ? val[gate[k][i]] : 1.0f);
                o[k][i] = fmaf(sc[k][i], g, o[k][i]);
                sq[k] = fmaf(o[k][i], o[k][i], sq[k]);
            }
            Packed<T, VEC>::store(z_out + z * t.dout + co.col[k], o[k]);
        }
        if (h_out) warp_shares<VEC, K>(co, sq, red_out, t.nw);
        __syncthreads();
        if (h_out) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (co.col[k] < 0) continue;
                const float s = rsqrtf(fmaf(add_shares(red_out + co.blk[k] * t.nw, t.nw), inv_o[k], eps));
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[k][i] *= s * wn[k][i];
                Packed<T, VEC>::store(h_out + z * t.dout + co.col[k], o[k]);
            }
        }
    }
}

// The row is computed again from residual and y (their two statistics included); gz and gh may be null.
template <typename T, int VEC, int K>
__global__ void __launch_bounds__(kMaxThreads) norm_gate_bwd_kernel(const T* __restrict__ residual, const T* __restrict__ y,
                                                                    const T* __restrict__ gz, const T* __restrict__ gh,
                                                                    const float* __restrict__ w_post, const float* __restrict__ scale,
                                                                    const float* __restrict__ w_pre, GateRow t, float eps,
                                                                    T* __restrict__ g_residual, T* __restrict__ gy,
                                                                    float* __restrict__ partial, int64_t rows) {
    extern __shared__ float smem[];
    float* red_in = smem;                                // [nblk_in][nw]
    float* red_dot = red_in + t.nblk_in * t.nw;          // [nblk_in][nw]
    float* red_sq = red_dot + t.nblk_in * t.nw;          // [nblk_out][nw]
    float* red_gh = red_sq + t.nblk_out * t.nw;          // [nblk_out][nw]
    float* val = red_gh + t.nblk_out * t.nw;             // [din] normalised row, scalars and gates activated
    float* gval = val + (t.din + 3) / 4 * 4;             // [dout] cotangent of the gated row
    Columns<VEC, K> ci, co;
    ci.init(t.in_tbl, t.din);
    co.init(t.out_tbl, t.dout);
    float wp[K][VEC], sc[K][VEC], wn[K][VEC], inv_i[K], inv_o[K];
    float a_post[K][VEC], a_scale[K][VEC], a_pre[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        inv_i[k] = ci.col[k] >= 0 ? t.in_inv[ci.blk[k]] : 0.0f;
        inv_o[k] = co.col[k] >= 0 ? t.out_inv[co.blk[k]] : 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            a_post[k][i] = a_scale[k][i] = a_pre[k][i] = 0.0f;
            if (ci.col[k] >= 0) wp[k][i] = w_post[t.in_tbl[4 * (ci.col[k] + i) + 1]];
            if (co.col[k] >= 0) {
                const int ch = t.out_tbl[4 * (co.col[k] + i) + 1];
                sc[k][i] = scale[ch];
                wn[k][i] = w_pre ? w_pre[ch] : 0.0f;
            }
        }
    }
    for (int i = threadIdx.x; i < 2 * (t.nblk_in + t.nblk_out) * t.nw; i += blockDim.x) smem[i] = 0.0f;
    __syncthreads();
    for (int64_t z = blockIdx.x; z < rows; z += gridDim.x) {
        float v[K][VEC], r[K][VEC], g0[K][VEC], g1[K][VEC], sq[K], dot[K], s_in[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = 0.0f;
            Packed<T, VEC> p;
            if (ci.col[k] >= 0) {
                p.load(y + z * t.din + ci.col[k]);
                p.unpack(v[k]);
            }
            if (co.col[k] >= 0) {
                Packed<T, VEC> q0, q1;
                p.load(residual + z * t.dout + co.col[k]);
                q0.zero();
                q1.zero();
                if (gz) q0.load(gz + z * t.dout + co.col[k]);
                if (gh) q1.load(gh + z * t.dout + co.col[k]);
                p.unpack(r[k]);
                q0.unpack(g0[k]);
                q1.unpack(g1[k]);
            }
            if (ci.col[k] >= 0) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) sq[k] = fmaf(v[k][i], v[k][i], sq[k]);
            }
        }
        warp_shares<VEC, K>(ci, sq, red_in, t.nw);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (ci.col[k] < 0) continue;
            s_in[k] = rsqrtf(fmaf(add_shares(red_in + ci.blk[k] * t.nw, t.nw), inv_i[k], eps));
            float a[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int32_t* e = t.in_tbl + 4 * (ci.col[k] + i);
                a[i] = __int_as_float(e[3]) * gate_act(e[2], v[k][i] * s_in[k] * wp[k][i]);
            }
            Packed<float, VEC>::store(val + ci.col[k], a);
        }
        __syncthreads();
        float gated[K][VEC];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = dot[k] = 0.0f;
            if (co.col[k] < 0) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int32_t* e = t.out_tbl + 4 * (co.col[k] + i);
                gated[k][i] = val[e[2]] * (e[3] >= 0 ? val[e[3]] : 1.0f);
                r[k][i] = fmaf(sc[k][i], gated[k][i], r[k][i]);
                sq[k] = fmaf(r[k][i], r[k][i], sq[k]);
                dot[k] = fmaf(g1[k][i] * wn[k][i], r[k][i], dot[k]);
            }
        }
        if (gh) {
            warp_shares<VEC, K>(co, sq, red_sq, t.nw);
            warp_shares<VEC, K>(co, dot, red_gh, t.nw);
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (co.col[k] < 0) continue;
            if (gh) {
                const float s = rsqrtf(fmaf(add_shares(red_sq + co.blk[k] * t.nw, t.nw), inv_o[k], eps));
                const float mean = add_shares(red_gh + co.blk[k] * t.nw, t.nw) * inv_o[k] * s * s;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    a_pre[k][i] = fmaf(g1[k][i], r[k][i] * s, a_pre[k][i]);
                    g0[k][i] = fmaf(s, g1[k][i] * wn[k][i] - r[k][i] * mean, g0[k][i]);
                }
            }
            float gv[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                a_scale[k][i] = fmaf(g0[k][i], gated[k][i], a_scale[k][i]);
                gv[i] = g0[k][i] * sc[k][i];
            }
            if (g_residual) Packed<T, VEC>::store(g_residual + z * t.dout + co.col[k], g0[k]);
            Packed<float, VEC>::store(gval + co.col[k], gv);
        }
        __syncthreads();
        float gn[K][VEC];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            dot[k] = 0.0f;
            if (ci.col[k] < 0) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int c = ci.col[k] + i;
                const int32_t* b = t.back_tbl + 4 * c;
                const int kind = b[0];
                const float n = v[k][i] * s_in[k];
                float g = 0.0f;
                if (kind == 1) {
                    g = gval[b[1]] * val[b[3]];
                } else if (kind != 3) {
                    if (kind == 0) {
                        g = gval[b[1]];
                    } else {
                        for (int m = 0; m < b[2]; ++m) g = fmaf(gval[b[1] + m], val[b[3] + m], g);
                    }
                    const int32_t* e = t.in_tbl + 4 * c;
                    g *= __int_as_float(e[3]) * gate_act_grad(e[2], n * wp[k][i]);
                }
                a_post[k][i] = fmaf(g, n, a_post[k][i]);
                gn[k][i] = g * wp[k][i];
                dot[k] = fmaf(gn[k][i], v[k][i], dot[k]);
            }
        }
        warp_shares<VEC, K>(ci, dot, red_dot, t.nw);
        __syncthreads();
        if (gy) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (ci.col[k] < 0) continue;
                const float mean = add_shares(red_dot + ci.blk[k] * t.nw, t.nw) * inv_i[k] * s_in[k] * s_in[k];
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[i] = s_in[k] * (gn[k][i] - v[k][i] * mean);
                Packed<T, VEC>::store(gy + z * t.din + ci.col[k], o);
            }
        }
    }
    if (partial) {
        float* mine = partial + static_cast<int64_t>(blockIdx.x) * (t.nchan_in + 2 * t.nchan_out);
        store_channels<VEC, K>(ci, a_post, t.in_chan, t.nchan_in, val, mine);
        store_channels<VEC, K>(co, a_scale, t.out_chan, t.nchan_out, gval, mine + t.nchan_in);
        store_channels<VEC, K>(co, a_pre, t.out_chan, t.nchan_out, gval, mine + t.nchan_in + t.nchan_out);
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

bool row_fits(int widest, bool vec4) { return widest <= (vec4 ? 4 * 4 : 8) * kMaxThreads; }

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
// The integer description of a gate row: host array of 7 sizes.
GateRow gate_row(const int32_t* in_tbl, const int32_t* out_tbl, const int32_t* back_tbl, const int32_t* in_chan, const int32_t* out_chan,
                 const float* in_inv, const float* out_inv, const int32_t* sizes, int nw) {
    return {in_tbl, out_tbl, back_tbl, in_chan, out_chan, in_inv, out_inv, sizes[0], sizes[1], sizes[2], sizes[3], sizes[4], sizes[5], nw};
}
}  // namespace

extern "C" int e3b_norm_gate_residual_fwd(const void* residual, const void* y, const float* weight_post, const float* scale,
                                          const float* weight_pre, const int32_t* in_table, const int32_t* out_table,
                                          const float* in_inv, const float* out_inv, const int32_t* sizes, int vec4, float eps,
                                          void* z, void* h, int64_t rows, int type, void* stream) {
    if (!sizes || rows < 0 || !known_type(type)) return fail(E3B_ERR_ARG, "norm_gate_residual_fwd: bad size or type");
    const int din = sizes[0], dout = sizes[1];
    if (rows == 0 || dout == 0) return E3B_OK;
    if (!residual || !y || !weight_post || !scale || !in_table || !out_table || !in_inv || !out_inv || !z || (h && !weight_pre))
        return fail(E3B_ERR_ARG, "norm_gate_residual_fwd: null pointer");
    const int bytes = 4 * element_size(type);
    const bool v4 = vec4 && din % 4 == 0 && dout % 4 == 0 && aligned_to(residual, bytes) && aligned_to(y, bytes) && aligned_to(z, bytes) && aligned_to(h, bytes);
    if (!row_fits(std::max(din, dout), v4)) return fail(E3B_ERR_UNSUPPORTED, "norm_gate_residual_fwd: %d columns", std::max(din, dout));
    const Shape s = row_shape(std::max(din, dout), v4);
    const GateRow t = gate_row(in_table, out_table, nullptr, nullptr, nullptr, in_inv, out_inv, sizes, s.nw);
    const size_t smem = sizeof(float) * ((t.nblk_in + t.nblk_out) * s.nw + din);
    return by_type(type, s, [&](auto t0, auto v0, auto k0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(v0)::value, K = decltype(k0)::value;
        int grid = 0;
        const int rc = resident_blocks(norm_gate_fwd_kernel<T, VEC, K>, s.threads, smem, rows, &grid);
        if (rc != E3B_OK) return rc;
        norm_gate_fwd_kernel<T, VEC, K><<<grid, s.threads, smem, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(residual), static_cast<const T*>(y), weight_post, scale, weight_pre, t, eps, static_cast<T*>(z),
            static_cast<T*>(h), rows);
        return check_launch("norm_gate_residual_fwd");
    });
}

extern "C" int e3b_norm_gate_residual_bwd(const void* residual, const void* y, const void* grad_z, const void* grad_h,
                                          const float* weight_post, const float* scale, const float* weight_pre, const int32_t* in_table,
                                          const int32_t* out_table, const int32_t* back_table, const int32_t* in_channels,
                                          const int32_t* out_channels, const float* in_inv, const float* out_inv, const int32_t* sizes,
                                          int vec4, float eps, void* grad_residual, void* grad_y, float* grad_params, void* scratch,
                                          int64_t scratch_bytes, int64_t rows, int type, void* stream) {
    if (!sizes || rows < 0 || !known_type(type)) return fail(E3B_ERR_ARG, "norm_gate_residual_bwd: bad size or type");
    const int din = sizes[0], dout = sizes[1], params = sizes[4] + 2 * sizes[5];
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0 || dout == 0) {
        if (grad_params) E3B_CUDA_TRY(cudaMemsetAsync(grad_params, 0, sizeof(float) * params, st));
        return E3B_OK;
    }
    if (!residual || !y || (!grad_z && !grad_h) || !weight_post || !scale || !in_table || !out_table || !back_table || !in_channels ||
        !out_channels || !in_inv || !out_inv || (grad_h && !weight_pre))
        return fail(E3B_ERR_ARG, "norm_gate_residual_bwd: null pointer");
    if (grad_params && (!scratch || scratch_bytes < e3b_norm_scratch_bytes(rows, params)))
        return fail(E3B_ERR_ARG, "norm_gate_residual_bwd: scratch of %lld bytes is too small", static_cast<long long>(scratch_bytes));
    const int bytes = 4 * element_size(type);
    const bool v4 = vec4 && din % 4 == 0 && dout % 4 == 0 && aligned_to(residual, bytes) && aligned_to(y, bytes) && aligned_to(grad_z, bytes) &&
                    aligned_to(grad_h, bytes) && aligned_to(grad_residual, bytes) && aligned_to(grad_y, bytes);
    if (!row_fits(std::max(din, dout), v4)) return fail(E3B_ERR_UNSUPPORTED, "norm_gate_residual_bwd: %d columns", std::max(din, dout));
    const Shape s = row_shape(std::max(din, dout), v4);
    const GateRow t = gate_row(in_table, out_table, back_table, in_channels, out_channels, in_inv, out_inv, sizes, s.nw);
    const size_t smem = sizeof(float) * (2 * (t.nblk_in + t.nblk_out) * s.nw + ceil_div(din, 4) * 4 + dout);
    int grid = 0;
    const int rc = by_type(type, s, [&](auto t0, auto v0, auto k0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(v0)::value, K = decltype(k0)::value;
        const int r = resident_blocks(norm_gate_bwd_kernel<T, VEC, K>, s.threads, smem, rows, &grid);
        if (r != E3B_OK) return r;
        norm_gate_bwd_kernel<T, VEC, K><<<grid, s.threads, smem, st>>>(
            static_cast<const T*>(residual), static_cast<const T*>(y), static_cast<const T*>(grad_z), static_cast<const T*>(grad_h), weight_post,
            scale, weight_pre, t, eps, static_cast<T*>(grad_residual), static_cast<T*>(grad_y), grad_params ? static_cast<float*>(scratch) : nullptr, rows);
        return check_launch("norm_gate_residual_bwd");
    });
    if (rc != E3B_OK || !grad_params || params == 0) return rc;
    add_partials_kernel<<<static_cast<unsigned>(ceil_div(params, 32)), dim3(32, 32), 0, st>>>(static_cast<const float*>(scratch), params,
                                                                                             grid, grad_params);
    return check_launch("norm_gate_residual_bwd sums");
}
