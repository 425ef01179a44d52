// Norm, gate, residual and norm, forward (norm_gate.cuh: the formula and the layout of a row).
//
// Bound by instructions in 16-bit types, by HBM in fp32: a row of 1,216 + 1,024 columns is read once and written twice.  Two rows
// are under way per thread block while one is computed; three barriers a row.
#include "norm_gate.cuh"

namespace e3b {
namespace {

// MAXT, BLOCKS: threads of a block at most, and blocks on an SM that the registers must allow.
template <typename T, int VEC, int NW, int K, int M, int MAXT, int BLOCKS>
__global__ void __launch_bounds__(MAXT, BLOCKS) norm_gate_fwd_kernel(const T* __restrict__ residual, const T* __restrict__ y,
                                                                     const float* __restrict__ w_post, const float* __restrict__ scale,
                                                                     const float* __restrict__ w_pre, const GateRow t, float eps,
                                                                     T* __restrict__ z_out, T* __restrict__ h_out, int64_t rows) {
    extern __shared__ __align__(16) float smem[];
    float* at = smem;
    const BlockSums in = block_sums_at(at, t.nblk_in, t.nw), outs = block_sums_at(at, t.nblk_out, t.nw);
    float* gates = at;                                   // [num_gates + 1]
    const RowAhead<T, VEC, K, 2> wide(gates + (t.num_gates + 4) / 4 * 4);
    const RowAhead<T, NW, M, 2> narrow(wide.mine - threadIdx.x * wide.kBytes + static_cast<int>(blockDim.x) * wide.kThread);
    Items<VEC, NW, K, M> it;
    it.init(t);
    auto fetch = [&](int64_t z, int stage) {
        if (z < rows) {
            const T *yr = y + z * t.din, *rr = residual + z * t.dout;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (it.win[k] < 0) continue;
                wide.fetch(stage, 0, k, yr + it.win[k]);
                wide.fetch(stage, 1, k, rr + it.wout[k]);
            }
#pragma unroll
            for (int j = 0; j < M; ++j) {
                if (it.nin[j] >= 0) narrow.fetch(stage, 0, j, yr + it.nin[j]);
                if (it.nout[j] >= 0) narrow.fetch(stage, 1, j, rr + it.nout[j]);
            }
        }
        commit_copies();
    };
    int64_t z = blockIdx.x;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch(z + static_cast<int64_t>(i) * gridDim.x, i);
    in.clear();
    outs.clear();
    if (threadIdx.x == 0) gates[t.num_gates] = 1.0f;
    __syncthreads();
    in.touch(it.in_blocks);
    outs.touch(it.out_blocks);
    // a wide column: z = residual + y s (w_post scale) gate
    float cy[K][VEC], wn[K][VEC], w_inv_i[K], w_inv_o[K];
    float n_cy[M][NW], n_sc[M][NW], n_wn[M][NW], n_inv_i[M], n_inv_o[M];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        w_inv_i[k] = t.in_inv[it.wbi[k]];
        w_inv_o[k] = t.out_inv[it.wbo[k]];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            cy[k][i] = wn[k][i] = 0.0f;
            if (it.win[k] < 0) continue;
            const int ch = t.out_tbl[4 * (it.wout[k] + i) + 1];
            cy[k][i] = w_post[t.in_tbl[4 * (it.win[k] + i) + 1]] * scale[ch];
            wn[k][i] = w_pre ? w_pre[ch] : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < M; ++j) {
        n_inv_i[j] = t.in_inv[it.nbi[j]];
        n_inv_o[j] = t.out_inv[it.nbo[j]];
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            n_cy[j][i] = it.nin[j] >= 0 ? w_post[t.in_tbl[4 * (it.nin[j] + i) + 1]] : 0.0f;
            n_sc[j][i] = it.cst[j];
            n_wn[j][i] = 0.0f;
            if (it.nout[j] < 0) continue;
            const int ch = t.out_tbl[4 * (it.nout[j] + i) + 1];
            n_sc[j][i] = it.cst[j] * scale[ch];
            n_wn[j][i] = w_pre ? w_pre[ch] : 0.0f;
        }
    }
    __syncthreads();
    for (int stage = 0; z < rows; z += gridDim.x, stage = stage + 1 == kAhead ? 0 : stage + 1) {
        float v[K][VEC], o[K][VEC], nv[M][NW], no[M][NW], sq[K], nsq[M];
        const T *yr = y + z * t.din, *rr = residual + z * t.dout;
        wait_for_row();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = 0.0f;
            if (it.win[k] < 0) continue;
            wide.read(stage, 0, k, yr + it.win[k], v[k]);
            wide.read(stage, 1, k, rr + it.wout[k], o[k]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) sq[k] = fmaf(v[k][i], v[k][i], sq[k]);
        }
#pragma unroll
        for (int j = 0; j < M; ++j) {
            nsq[j] = 0.0f;
            if (it.nin[j] < 0) continue;
            narrow.read(stage, 0, j, yr + it.nin[j], nv[j]);
            if (it.nout[j] >= 0) narrow.read(stage, 1, j, rr + it.nout[j], no[j]);
#pragma unroll
            for (int i = 0; i < NW; ++i) nsq[j] = fmaf(nv[j][i], nv[j][i], nsq[j]);
        }
        fetch(z + static_cast<int64_t>(kAhead) * gridDim.x, stage);
        in.add(it.in_blocks, sq, it.wbi, nsq, it.nbi);
        __syncthreads();
        // the activations: gates for the wide items, scalars for the row itself
#pragma unroll
        for (int j = 0; j < M; ++j) {
            nsq[j] = 0.0f;
            if (it.kind[j] < 0 || it.kind[j] == kUnused) continue;
            const float s = rsqrtf(fmaf(in.get(it.nbi[j]), n_inv_i[j], eps));
#pragma unroll
            for (int i = 0; i < NW; ++i) nv[j][i] = n_sc[j][i] * gate_act(it.act[j], nv[j][i] * s * n_cy[j][i]);
            if (it.kind[j] == kGates) {
                Packed<float, NW>::store(gates + it.slot[j], nv[j]);
            } else {
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    no[j][i] += nv[j][i];
                    nsq[j] = fmaf(no[j][i], no[j][i], nsq[j]);
                }
                Packed<T, NW>::store(z_out + z * t.dout + it.nout[j], no[j]);
            }
        }
        float s_in[K];
#pragma unroll
        for (int k = 0; k < K; ++k) s_in[k] = it.win[k] >= 0 ? rsqrtf(fmaf(in.get(it.wbi[k]), w_inv_i[k], eps)) : 0.0f;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = 0.0f;
            if (it.win[k] < 0) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                o[k][i] = fmaf(v[k][i] * cy[k][i], s_in[k] * gates[it.gate[k][i]], o[k][i]);
                sq[k] = fmaf(o[k][i], o[k][i], sq[k]);
            }
            Packed<T, VEC>::store(z_out + z * t.dout + it.wout[k], o[k]);
        }
        if (h_out) outs.add(it.out_blocks, sq, it.wbo, nsq, it.nbo);
        __syncthreads();
        if (h_out) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (it.win[k] < 0) continue;
                const float s = rsqrtf(fmaf(outs.get(it.wbo[k]), w_inv_o[k], eps));
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[k][i] *= s * wn[k][i];
                Packed<T, VEC>::store(h_out + z * t.dout + it.wout[k], o[k]);
            }
#pragma unroll
            for (int j = 0; j < M; ++j) {
                if (it.nout[j] < 0) continue;
                const float s = rsqrtf(fmaf(outs.get(it.nbo[j]), n_inv_o[j], eps));
#pragma unroll
                for (int i = 0; i < NW; ++i) no[j][i] *= s * n_wn[j][i];
                Packed<T, NW>::store(h_out + z * t.dout + it.nout[j], no[j]);
            }
        }
    }
}

}  // namespace
}  // namespace e3b

using namespace e3b;

extern "C" int e3b_norm_gate_residual_fwd(const void* residual, const void* y, const float* weight_post, const float* scale,
                                          const float* weight_pre, const int32_t* wide, const int32_t* narrow, const int32_t* in_table,
                                          const int32_t* out_table, const float* in_inv, const float* out_inv, const int32_t* sizes, float eps,
                                          void* z, void* h, int64_t rows, int type, void* stream) {
    if (!sizes || rows < 0 || !known_type(type)) return fail(E3B_ERR_ARG, "norm_gate_residual_fwd: bad size or type");
    if (rows == 0 || sizes[6] == 0) return E3B_OK;
    if (!residual || !y || !weight_post || !scale || (sizes[2] > 0 && !wide) || (sizes[3] > 0 && !narrow) || !in_table || !out_table || !in_inv || !out_inv || !z || (h && !weight_pre))
        return fail(E3B_ERR_ARG, "norm_gate_residual_fwd: null pointer");
    const int bytes = sizes[0] * element_size(type);
    if (!aligned_to(residual, bytes) || !aligned_to(y, bytes) || !aligned_to(z, bytes) || !aligned_to(h, bytes))
        return fail(E3B_ERR_ARG, "norm_gate_residual_fwd: rows must start on %d bytes", bytes);
    GateRow t;
    RowShape s;
    const int rc = gate_row("norm_gate_residual_fwd", type, sizes, wide, narrow, in_table, out_table, nullptr, nullptr, in_inv, out_inv, &t, &s);
    if (rc != E3B_OK) return rc;
    const int64_t floats = BlockSums::floats(t.nblk_in, t.nw) + BlockSums::floats(t.nblk_out, t.nw) + (t.num_gates + 4) / 4 * 4;
    return by_type_and_items(type, s, [&](auto t0, auto v0, auto n0, auto k0, auto m0, auto x0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(v0)::value, NW = decltype(n0)::value, K = decltype(k0)::value, M = decltype(m0)::value, MAXT = decltype(x0)::value;
        constexpr int BLOCKS = MAXT == 128 ? 6 : MAXT == 256 ? 3 : 1;
        const size_t smem = sizeof(float) * floats + static_cast<size_t>(RowAhead<T, VEC, K, 2>::kThread + RowAhead<T, NW, M, 2>::kThread) * s.threads;
        int grid = 0;
        const int e = resident_blocks(norm_gate_fwd_kernel<T, VEC, NW, K, M, MAXT, BLOCKS>, s.threads, smem, rows, &grid);
        if (e != E3B_OK) return e;
        norm_gate_fwd_kernel<T, VEC, NW, K, M, MAXT, BLOCKS><<<grid, s.threads, smem, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(residual), static_cast<const T*>(y), weight_post, scale, weight_pre, t, eps, static_cast<T*>(z),
            static_cast<T*>(h), rows);
        return check_launch("norm_gate_residual_fwd");
    });
}
