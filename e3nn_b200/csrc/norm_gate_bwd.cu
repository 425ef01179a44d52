// Norm, gate, residual and norm, gradients (norm_gate.cuh: the formula and the layout of a row).
//
// With r = s_z (1 / root mean square of z) and t = gh w_pre:  gz' = gz + r (t - z r^2 mean(t z)) is the cotangent of residual;
// gg = gz' scale goes through the gate (a gate's cotangent is the sum of gg n over its components, times the derivative of its activation),
// then through the first norm like the second.  z and both statistics are computed again from residual and y: that costs no traffic,
// and z is not rounded.  Parameter gradients are summed over the rows of a thread block in registers, one entry a column,
// added up per channel at its end and over the thread blocks in their order.  Bound by the five barriers a row and the latency between
// them (one row takes 8 warps about 800 instructions each, under half of the issue slots): 16,384 rows of 1,216 + 1,024 columns in fp32 231 us = 1.9 TB/s, in bf16 204 us.  Measured
// and not taken: two items a thread with half the threads (402 us: twelve warps an SM no longer hide the barriers).
#include "norm_gate.cuh"

namespace e3b {
namespace {

template <typename T, int VEC, int NW, int K, int M, int MAXT, int BLOCKS>
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
    float* gates = at;                                        // [num_gates + 1] activated gates
    float* prod = gates + (t.num_gates + 4) / 4 * 4;          // [dout] cotangent of the gated row times the normalised row
    constexpr int AHEAD = rows_ahead(NW * sizeof(T), K > M ? K : M);
    RowAhead<T, VEC, K, 4, AHEAD> wide(prod + (t.dout + 3) / 4 * 4);
    RowAhead<T, NW, M, 4, AHEAD> narrow(wide.mine - threadIdx.x * wide.kBytes + static_cast<int>(blockDim.x) * wide.kThread);
    Items<VEC, NW, K, M> it;
    it.init(t);
    auto fetch = [&](int64_t z, int stage) {
        if (z < rows) {
            const int64_t zi = z * t.din, zo = z * t.dout;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (it.win[k] < 0) continue;
                wide.fetch(stage, 0, k, y + zi + it.win[k]);
                wide.fetch(stage, 1, k, residual + zo + it.wout[k]);
                if (gz) wide.fetch(stage, 2, k, gz + zo + it.wout[k]);
                if (gh) wide.fetch(stage, 3, k, gh + zo + it.wout[k]);
            }
#pragma unroll
            for (int j = 0; j < M; ++j) {
                if (it.nin[j] >= 0) narrow.fetch(stage, 0, j, y + zi + it.nin[j]);
                if (it.nout[j] < 0) continue;
                narrow.fetch(stage, 1, j, residual + zo + it.nout[j]);
                if (gz) narrow.fetch(stage, 2, j, gz + zo + it.nout[j]);
                if (gh) narrow.fetch(stage, 3, j, gh + zo + it.nout[j]);
            }
        }
        commit_copies();
    };
    int64_t z = blockIdx.x;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch(z + static_cast<int64_t>(i) * gridDim.x, i);
    in.clear();
    dots.clear();
    outs.clear();
    ghs.clear();
    if (threadIdx.x == 0) gates[t.num_gates] = 1.0f;
    __syncthreads();
    float wp[K][VEC], sc[K][VEC], wn[K][VEC], w_inv_i[K], w_inv_o[K];
    float n_wp[M][NW], n_sc[M][NW], n_wn[M][NW], n_inv_i[M], n_inv_o[M];
    float a_post[K][VEC], a_scale[K][VEC], a_pre[K][VEC], n_post[M][NW], n_scale[M][NW], n_pre[M][NW];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        w_inv_i[k] = t.in_inv[it.wbi[k]];
        w_inv_o[k] = t.out_inv[it.wbo[k]];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            a_post[k][i] = a_scale[k][i] = a_pre[k][i] = wp[k][i] = sc[k][i] = wn[k][i] = 0.0f;
            if (it.win[k] < 0) continue;
            const int ch = t.out_tbl[4 * (it.wout[k] + i) + 1];
            wp[k][i] = w_post[t.in_tbl[4 * (it.win[k] + i) + 1]];
            sc[k][i] = scale[ch];
            wn[k][i] = w_pre ? w_pre[ch] : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < M; ++j) {
        n_inv_i[j] = t.in_inv[it.nbi[j]];
        n_inv_o[j] = t.out_inv[it.nbo[j]];
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            n_post[j][i] = n_scale[j][i] = n_pre[j][i] = n_sc[j][i] = n_wn[j][i] = 0.0f;
            n_wp[j][i] = it.nin[j] >= 0 ? w_post[t.in_tbl[4 * (it.nin[j] + i) + 1]] : 0.0f;
            if (it.nout[j] < 0) continue;
            const int ch = t.out_tbl[4 * (it.nout[j] + i) + 1];
            n_sc[j][i] = scale[ch];
            n_wn[j][i] = w_pre ? w_pre[ch] : 0.0f;
        }
    }
    __syncthreads();
    for (int stage = 0; z < rows; z += gridDim.x, stage = stage + 1 == AHEAD ? 0 : stage + 1) {
        const int64_t zi = z * t.din, zo = z * t.dout;
        // v: y, then normalised; x: residual, then z; g0: cotangent of z; g1: of h, then of the normalised row
        float v[K][VEC], x[K][VEC], g0[K][VEC], g1[K][VEC], sq[K], dot[K];
        float nv[M][NW], nx[M][NW], n0[M][NW], n1[M][NW], nsq[M], ndot[M];
        wait_for_row<AHEAD>();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = 0.0f;
            if (it.win[k] < 0) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) g0[k][i] = g1[k][i] = 0.0f;
            wide.read(stage, 0, k, v[k]);
            wide.read(stage, 1, k, x[k]);
            if (gz) wide.read(stage, 2, k, g0[k]);
            if (gh) wide.read(stage, 3, k, g1[k]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) sq[k] = fmaf(v[k][i], v[k][i], sq[k]);
        }
#pragma unroll
        for (int j = 0; j < M; ++j) {
            nsq[j] = 0.0f;
            if (it.nin[j] < 0) continue;
#pragma unroll
            for (int i = 0; i < NW; ++i) n0[j][i] = n1[j][i] = nx[j][i] = 0.0f;
            narrow.read(stage, 0, j, nv[j]);
            if (it.nout[j] >= 0) {
                narrow.read(stage, 1, j, nx[j]);
                if (gz) narrow.read(stage, 2, j, n0[j]);
                if (gh) narrow.read(stage, 3, j, n1[j]);
            }
#pragma unroll
            for (int i = 0; i < NW; ++i) nsq[j] = fmaf(nv[j][i], nv[j][i], nsq[j]);
        }
        fetch(z + static_cast<int64_t>(AHEAD) * gridDim.x, stage);
        in.add(it.in_blocks, sq, it.wbi, nsq, it.nbi);
        __syncthreads();
        float s_in[K], ns_in[M], act[M][NW], slope[M][NW];       // activated columns of the narrow items and their derivatives
        in.get(it.wbi, s_in, it.nbi, ns_in);
#pragma unroll
        for (int j = 0; j < M; ++j) {
            nsq[j] = ndot[j] = 0.0f;
            if (it.nin[j] < 0) continue;
            ns_in[j] = rsqrtf(fmaf(ns_in[j], n_inv_i[j], eps));
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                nv[j][i] *= ns_in[j];
                act[j][i] = nv[j][i] * n_wp[j][i];
            }
            activate_and_derive<NW>(it.act[j], it.cst[j], act[j], act[j], slope[j]);
            if (it.kind[j] == kGates) Packed<float, NW>::store(gates + it.slot[j], act[j]);
            if (it.nout[j] < 0) continue;
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                nx[j][i] = fmaf(n_sc[j][i], act[j][i], nx[j][i]);
                nsq[j] = fmaf(nx[j][i], nx[j][i], nsq[j]);
                ndot[j] = fmaf(n1[j][i] * n_wn[j][i], nx[j][i], ndot[j]);
            }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (it.win[k] < 0) continue;
            s_in[k] = rsqrtf(fmaf(s_in[k], w_inv_i[k], eps));
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[k][i] *= s_in[k];
        }
        __syncthreads();
        float gate[K][VEC];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = dot[k] = 0.0f;
            if (it.win[k] < 0) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                gate[k][i] = gates[it.gate[k][i]];
                x[k][i] = fmaf(sc[k][i], v[k][i] * wp[k][i] * gate[k][i], x[k][i]);
                sq[k] = fmaf(x[k][i], x[k][i], sq[k]);
                dot[k] = fmaf(g1[k][i] * wn[k][i], x[k][i], dot[k]);
            }
        }
        if (gh) {
            outs.add(it.out_blocks, sq, it.wbo, nsq, it.nbo);
            ghs.add(it.out_blocks, dot, it.wbo, ndot, it.nbo);
            __syncthreads();
            outs.get(it.wbo, sq, it.nbo, nsq);
            ghs.get(it.wbo, dot, it.nbo, ndot);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (it.win[k] < 0) continue;
            if (gh) {
                const float s = rsqrtf(fmaf(sq[k], w_inv_o[k], eps)), mean = dot[k] * w_inv_o[k] * s * s;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    a_pre[k][i] = fmaf(g1[k][i], x[k][i] * s, a_pre[k][i]);
                    g0[k][i] = fmaf(s, g1[k][i] * wn[k][i] - x[k][i] * mean, g0[k][i]);
                }
            }
            if (g_residual) Packed<T, VEC>::store(g_residual + zo + it.wout[k], g0[k]);
            float pr[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float n = v[k][i] * wp[k][i], gv = g0[k][i] * sc[k][i];
                a_scale[k][i] = fmaf(g0[k][i], n * gate[k][i], a_scale[k][i]);
                g1[k][i] = gv * gate[k][i];
                pr[i] = gv * n;
            }
            Packed<float, VEC>::store(prod + it.wout[k], pr);
        }
#pragma unroll
        for (int j = 0; j < M; ++j) {
            if (it.nout[j] < 0) continue;
            if (gh) {
                const float s = rsqrtf(fmaf(nsq[j], n_inv_o[j], eps)), mean = ndot[j] * n_inv_o[j] * s * s;
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    n_pre[j][i] = fmaf(n1[j][i], nx[j][i] * s, n_pre[j][i]);
                    n0[j][i] = fmaf(s, n1[j][i] * n_wn[j][i] - nx[j][i] * mean, n0[j][i]);
                }
            }
            if (g_residual) Packed<T, NW>::store(g_residual + zo + it.nout[j], n0[j]);
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                n_scale[j][i] = fmaf(n0[j][i], act[j][i], n_scale[j][i]);
                n1[j][i] = n0[j][i] * n_sc[j][i];       // cotangent of the activated column
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < M; ++j) {
            ndot[j] = 0.0f;
            if (it.nin[j] < 0) continue;
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                if (it.kind[j] == kGates) {
                    const int32_t* e = t.in_tbl + 4 * (it.nin[j] + i);
                    n1[j][i] = 0.0f;
                    for (int m = 0; m < e[3]; ++m) n1[j][i] += prod[e[2] + m];
                }
                n1[j][i] = it.kind[j] == kUnused ? 0.0f : n1[j][i] * slope[j][i];
                n_post[j][i] = fmaf(n1[j][i], nv[j][i], n_post[j][i]);
                n1[j][i] *= n_wp[j][i];
                ndot[j] = fmaf(n1[j][i], nv[j][i], ndot[j]);
            }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            dot[k] = 0.0f;
            if (it.win[k] < 0) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                a_post[k][i] = fmaf(g1[k][i], v[k][i], a_post[k][i]);
                g1[k][i] *= wp[k][i];
                dot[k] = fmaf(g1[k][i], v[k][i], dot[k]);
            }
        }
        if (gy) {
            dots.add(it.in_blocks, dot, it.wbi, ndot, it.nbi);
            __syncthreads();
            dots.get(it.wbi, dot, it.nbi, ndot);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (it.win[k] < 0) continue;
                const float mean = dot[k] * w_inv_i[k];
#pragma unroll
                for (int i = 0; i < VEC; ++i) g1[k][i] = s_in[k] * (g1[k][i] - v[k][i] * mean);
                Packed<T, VEC>::store(gy + zi + it.win[k], g1[k]);
            }
#pragma unroll
            for (int j = 0; j < M; ++j) {
                if (it.nin[j] < 0) continue;
                const float mean = ndot[j] * n_inv_i[j];
#pragma unroll
                for (int i = 0; i < NW; ++i) n1[j][i] = ns_in[j] * (n1[j][i] - nv[j][i] * mean);
                Packed<T, NW>::store(gy + zi + it.nin[j], n1[j]);
            }
        }
    }
    if (!partial) return;
    // columns through shared memory, channels from there: three gradients one after the other
    float* mine = partial + static_cast<int64_t>(blockIdx.x) * (t.nchan_in + 2 * t.nchan_out);
    auto columns = [&](const float (&w)[K][VEC], const float (&n)[M][NW], const int (&wc)[K], const int (&nc)[M]) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (wc[k] >= 0) smem[wc[k] + i] = w[k][i];
#pragma unroll
        for (int j = 0; j < M; ++j)
#pragma unroll
            for (int i = 0; i < NW; ++i)
                if (nc[j] >= 0) smem[nc[j] + i] = n[j][i];
        __syncthreads();
    };
    columns(a_post, n_post, it.win, it.nin);
    store_channels(smem, t.in_chan, t.nchan_in, mine);
    columns(a_scale, n_scale, it.wout, it.nout);
    store_channels(smem, t.out_chan, t.nchan_out, mine + t.nchan_in);
    columns(a_pre, n_pre, it.wout, it.nout);
    store_channels(smem, t.out_chan, t.nchan_out, mine + t.nchan_in + t.nchan_out);
}

}  // namespace
}  // namespace e3b

using namespace e3b;

extern "C" int e3b_norm_gate_residual_bwd(const void* residual, const void* y, const void* grad_z, const void* grad_h,
                                          const float* weight_post, const float* scale, const float* weight_pre, const int32_t* wide,
                                          const int32_t* narrow, const int32_t* in_table, const int32_t* out_table, const int32_t* in_channels,
                                          const int32_t* out_channels, const float* in_inv, const float* out_inv, const int32_t* sizes,
                                          float eps, void* grad_residual, void* grad_y, float* grad_params, void* scratch,
                                          int64_t scratch_bytes, int64_t rows, int type, void* stream) {
    if (!sizes || rows < 0 || !known_type(type)) return fail(E3B_ERR_ARG, "norm_gate_residual_bwd: bad size or type");
    const int params = sizes[9] + 2 * sizes[10];
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0 || sizes[6] == 0) {
        if (grad_params) E3B_CUDA_TRY(cudaMemsetAsync(grad_params, 0, sizeof(float) * params, st));
        return E3B_OK;
    }
    if (!residual || !y || (!grad_z && !grad_h) || !weight_post || !scale || (sizes[2] > 0 && !wide) || (sizes[3] > 0 && !narrow) || !in_table || !out_table || !in_channels ||
        !out_channels || !in_inv || !out_inv || (grad_h && !weight_pre))
        return fail(E3B_ERR_ARG, "norm_gate_residual_bwd: null pointer");
    if (grad_params && (!scratch || scratch_bytes < norm_scratch_bytes(rows, params)))
        return fail(E3B_ERR_ARG, "norm_gate_residual_bwd: scratch of %lld bytes is too small", static_cast<long long>(scratch_bytes));
    const int bytes = sizes[0] * element_size(type);
    if (!aligned_to(residual, bytes) || !aligned_to(y, bytes) || !aligned_to(grad_z, bytes) || !aligned_to(grad_h, bytes) ||
        !aligned_to(grad_residual, bytes) || !aligned_to(grad_y, bytes))
        return fail(E3B_ERR_ARG, "norm_gate_residual_bwd: rows must start on %d bytes", bytes);
    GateRow t;
    RowShape s;
    const int bad = gate_row("norm_gate_residual_bwd", type, sizes, wide, narrow, in_table, out_table, in_channels, out_channels, in_inv, out_inv, &t, &s);
    if (bad != E3B_OK) return bad;
    const int64_t floats = 2 * BlockSums::floats(t.nblk_in, t.nw) + 2 * BlockSums::floats(t.nblk_out, t.nw) + (t.num_gates + 4) / 4 * 4 + ceil_div(t.dout, 4) * 4;
    int grid = 0;
    const int rc = by_type_and_items(type, s, [&](auto t0, auto v0, auto n0, auto k0, auto m0, auto x0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(v0)::value, NW = decltype(n0)::value, K = decltype(k0)::value, M = decltype(m0)::value, MAXT = decltype(x0)::value, AHEAD = rows_ahead(NW * sizeof(T), K > M ? K : M);
        constexpr int BLOCKS = MAXT == 128 ? 4 : MAXT == 256 ? 2 : 1;
        const size_t smem = std::max<size_t>(sizeof(float) * floats + static_cast<size_t>(RowAhead<T, VEC, K, 4, AHEAD>::kThread + RowAhead<T, NW, M, 4, AHEAD>::kThread) * s.threads,
                                             sizeof(float) * std::max(t.din, t.dout));
        const int e = resident_blocks(norm_gate_bwd_kernel<T, VEC, NW, K, M, MAXT, BLOCKS>, s.threads, smem, rows, &grid);
        if (e != E3B_OK) return e;
        norm_gate_bwd_kernel<T, VEC, NW, K, M, MAXT, BLOCKS><<<grid, s.threads, smem, st>>>(
            static_cast<const T*>(residual), static_cast<const T*>(y), static_cast<const T*>(grad_z), static_cast<const T*>(grad_h), weight_post,
            scale, weight_pre, t, eps, static_cast<T*>(grad_residual), static_cast<T*>(grad_y), grad_params ? static_cast<float*>(scratch) : nullptr, rows);
        return check_launch("norm_gate_residual_bwd");
    });
    if (rc != E3B_OK || !grad_params || params == 0) return rc;
    add_partials_kernel<<<static_cast<unsigned>(ceil_div(params, 32)), dim3(32, 32), 0, st>>>(static_cast<const float*>(scratch), params,
                                                                                             grid, grad_params);
    return check_launch("norm_gate_residual_bwd sums");
}
