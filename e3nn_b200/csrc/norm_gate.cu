// Norm, gate, residual and norm, forward (norm_gate.cuh: the formula and the layout of a row).
//
// A row of 1,216 + 1,024 columns is read once and written twice; sums per irreps block, conversions and activations take about 2,000 warp
// instructions a row, which fill about half of the issue slots.  The rest is latency: at most 16 warps an SM by warps, each with two row
// sums after one another, and barriers by thread blocks.  By thread blocks: two rows are under way per block while
// one is computed, three barriers a row.  By warps (below): 262,144 rows of 1,216 + 1,024 columns in bf16 858 us = 2.6 TB/s (by thread blocks
// 1,080), 16,384 rows in fp32 85 us = 3.3 TB/s (105).
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
    constexpr int AHEAD = rows_ahead(NW * sizeof(T), K > M ? K : M);
    RowAhead<T, VEC, K, 2, AHEAD> wide(gates + (t.num_gates + 4) / 4 * 4);
    RowAhead<T, NW, M, 2, AHEAD> narrow(wide.mine - threadIdx.x * wide.kBytes + static_cast<int>(blockDim.x) * wide.kThread);
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
    for (int i = 0; i < AHEAD; ++i) fetch(z + static_cast<int64_t>(i) * gridDim.x, i);
    in.clear();
    outs.clear();
    if (threadIdx.x == 0) gates[t.num_gates] = 1.0f;
    __syncthreads();
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
    for (int stage = 0; z < rows; z += gridDim.x, stage = stage + 1 == AHEAD ? 0 : stage + 1) {
        float v[K][VEC], o[K][VEC], nv[M][NW], no[M][NW], sq[K], nsq[M];
        wait_for_row<AHEAD>();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            sq[k] = 0.0f;
            if (it.win[k] < 0) continue;
            wide.read(stage, 0, k, v[k]);
            wide.read(stage, 1, k, o[k]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) sq[k] = fmaf(v[k][i], v[k][i], sq[k]);
        }
#pragma unroll
        for (int j = 0; j < M; ++j) {
            nsq[j] = 0.0f;
            if (it.nin[j] < 0) continue;
            narrow.read(stage, 0, j, nv[j]);
            if (it.nout[j] >= 0) narrow.read(stage, 1, j, no[j]);
#pragma unroll
            for (int i = 0; i < NW; ++i) nsq[j] = fmaf(nv[j][i], nv[j][i], nsq[j]);
        }
        fetch(z + static_cast<int64_t>(AHEAD) * gridDim.x, stage);
        in.add(it.in_blocks, sq, it.wbi, nsq, it.nbi);
        __syncthreads();
        // the activations: gates for the wide items, scalars for the row itself
        float s_in[K], ns_in[M];
        in.get(it.wbi, s_in, it.nbi, ns_in);
#pragma unroll
        for (int j = 0; j < M; ++j) {
            nsq[j] = 0.0f;
            if (it.kind[j] < 0 || it.kind[j] == kUnused) continue;
            const float s = rsqrtf(fmaf(ns_in[j], n_inv_i[j], eps));
#pragma unroll
            for (int i = 0; i < NW; ++i) nv[j][i] *= s * n_cy[j][i];
            activate<NW>(it.act[j], 1.0f, nv[j], nv[j]);
#pragma unroll
            for (int i = 0; i < NW; ++i) nv[j][i] *= n_sc[j][i];
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
#pragma unroll
        for (int k = 0; k < K; ++k) s_in[k] = rsqrtf(fmaf(s_in[k], w_inv_i[k], eps));
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
            float so[K], nso[M];
            outs.get(it.wbo, so, it.nbo, nso);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (it.win[k] < 0) continue;
                const float s = rsqrtf(fmaf(so[k], w_inv_o[k], eps));
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[k][i] *= s * wn[k][i];
                Packed<T, VEC>::store(h_out + z * t.dout + it.wout[k], o[k]);
            }
#pragma unroll
            for (int j = 0; j < M; ++j) {
                if (it.nout[j] < 0) continue;
                const float s = rsqrtf(fmaf(nso[j], n_inv_o[j], eps));
#pragma unroll
                for (int i = 0; i < NW; ++i) no[j][i] *= s * n_wn[j][i];
                Packed<T, NW>::store(h_out + z * t.dout + it.nout[j], no[j]);
            }
        }
    }
}

// One warp a row (norm_gate.cuh).  Shared memory: per block w_post (times scale for wide columns), scale and w_pre by column; per warp
// the gates of every column, two arrays of block sums and the next row of y and residual.
constexpr int row_warps(int vec, int k) { return vec == 4 && k == 9 ? 6 : 8; }      // of a block: the registers of two blocks fit an SM
template <typename T, int VEC, int NW, int K, int M>
__global__ void __launch_bounds__(32 * row_warps(VEC, K), 2) norm_gate_fwd_row_kernel(const T* __restrict__ residual, const T* __restrict__ y,
                                                                   const float* __restrict__ w_post, const float* __restrict__ scale,
                                                                   const float* __restrict__ w_pre, const int32_t* __restrict__ in_tbl,
                                                                   const int32_t* __restrict__ out_tbl, const __grid_constant__ RowPlan t, float eps,
                                                                   T* __restrict__ z_out, T* __restrict__ h_out, int64_t rows) {
    extern __shared__ __align__(16) float smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int din4 = (t.din + 3) & ~3, dout4 = (t.dout + 3) & ~3, spread4 = (t.num_spread + 3) & ~3;
    float* wp = smem;                  // [din]
    float* sc = wp + din4;             // [dout]
    float* wn = sc + dout4;            // [dout]
    constexpr bool kAsync = NW * sizeof(T) >= 4 && VEC * sizeof(T) >= 4;
    constexpr int kStage = kAsync ? 2 * (K * VEC + M * NW) * 32 * static_cast<int>(sizeof(T)) : 0;      // bytes of the next row
    float* mine = wn + dout4 + warp * (spread4 + 2 * kMaxBlocks + kStage / 4);
    float* gates = mine;               // [num_spread]
    float* s_in = mine + spread4;      // [kMaxBlocks] x 2
    float* s_out = s_in + kMaxBlocks;
    char* stage = reinterpret_cast<char*>(s_out + kMaxBlocks);
    for (int c = threadIdx.x; c < t.din; c += blockDim.x) wp[c] = w_post[in_tbl[4 * c + 1]];
    for (int j = threadIdx.x; j < t.dout; j += blockDim.x) {
        sc[j] = scale[out_tbl[4 * j + 1]];
        wn[j] = w_pre ? w_pre[out_tbl[4 * j + 1]] : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (k < t.num_wide)
            for (int i = threadIdx.x; i < t.w[k].count * VEC; i += blockDim.x) wp[t.w[k].in + i] *= sc[t.w[k].out + i];
    __syncthreads();
    // the lane's places in the stage: y of the wide slots, residual of them, y of the narrow ones, residual of those
    auto wide_at = [&](int a, int k) { return reinterpret_cast<T*>(stage) + ((a * K + k) * 32 + lane) * VEC; };
    auto narrow_at = [&](int a, int j) { return reinterpret_cast<T*>(stage) + 2 * K * 32 * VEC + ((a * M + j) * 32 + lane) * NW; };
    auto copy = [&](T* to, const T* from, auto width) {
        constexpr int kBytes = decltype(width)::value * static_cast<int>(sizeof(T));
        const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to));
        if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(__cvta_generic_to_global(from)) : "memory");
        else if constexpr (kBytes >= 4) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(__cvta_generic_to_global(from)), "n"(kBytes) : "memory");
    };
    unsigned wide_has = 0, narrow_has = 0, out_has = 0;       // slots in which this lane has columns, narrow ones with output columns
#pragma unroll
    for (int k = 0; k < K; ++k) wide_has |= k < t.num_wide && lane < t.w[k].count ? 1u << k : 0u;
#pragma unroll
    for (int j = 0; j < M; ++j) narrow_has |= j < t.num_narrow && lane < t.n[j].count ? 1u << j : 0u;
#pragma unroll
    for (int j = 0; j < M; ++j) out_has |= (narrow_has >> j & 1u) && t.n[j].out >= 0 ? 1u << j : 0u;
    auto fetch = [&](int64_t z) {
        if (kAsync && z < rows) {
            const T *yr = y + z * t.din + lane * VEC, *rr = residual + z * t.dout + lane * VEC;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!(wide_has >> k & 1u)) continue;
                copy(wide_at(0, k), yr + t.w[k].in, Int<VEC>());
                copy(wide_at(1, k), rr + t.w[k].out, Int<VEC>());
            }
            yr = y + z * t.din + lane * NW;
            rr = residual + z * t.dout + lane * NW;
#pragma unroll
            for (int j = 0; j < M; ++j) {
                if (!(narrow_has >> j & 1u)) continue;
                copy(narrow_at(0, j), yr + t.n[j].in, Int<NW>());
                if (t.n[j].out >= 0) copy(narrow_at(1, j), rr + t.n[j].out, Int<NW>());
            }
        }
        commit_copies();
    };
    const int64_t step = static_cast<int64_t>(gridDim.x) * warps;
    int64_t z = static_cast<int64_t>(blockIdx.x) * warps + warp;
    fetch(z);
    for (; z < rows; z += step) {
        Packed<T, VEC> py[K], pr[K];
        float nv[M][NW], no[M][NW], wsq[K], nsq[M];
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int k = 0; k < K; ++k) {
            wsq[k] = 0.0f;
            if (!(wide_has >> k & 1u)) continue;
            py[k].load(kAsync ? wide_at(0, k) : y + z * t.din + t.w[k].in + lane * VEC);
            pr[k].load(kAsync ? wide_at(1, k) : residual + z * t.dout + t.w[k].out + lane * VEC);
            float v[VEC];
            py[k].unpack(v);
            wsq[k] = dot_n<VEC>(v, v);
        }
#pragma unroll
        for (int j = 0; j < M; ++j) {
            nsq[j] = 0.0f;
            if (!(narrow_has >> j & 1u)) continue;
            Packed<T, NW> p;
            p.load(kAsync ? narrow_at(0, j) : y + z * t.din + t.n[j].in + lane * NW);
            p.unpack(nv[j]);
            if (t.n[j].out >= 0) {
                p.load(kAsync ? narrow_at(1, j) : residual + z * t.dout + t.n[j].out + lane * NW);
                p.unpack(no[j]);
            }
#pragma unroll
            for (int i = 0; i < NW; ++i) nsq[j] = fmaf(nv[j][i], nv[j][i], nsq[j]);
        }
        fetch(z + step);
        row_sums<false, K, M>(wsq, nsq, t.wide_in_ends, t.narrow_in_ends, t.inv_in, eps, s_in);
#pragma unroll
        for (int j = 0; j < M; ++j) {
            nsq[j] = 0.0f;
            if (!(narrow_has >> j & 1u) || t.n[j].kind == kUnused) continue;
            const float s = s_in[t.n[j].bi];
#pragma unroll
            for (int i = 0; i < NW; ++i) nv[j][i] *= s * wp[t.n[j].in + lane * NW + i];
            activate<NW>(t.n[j].act, t.n[j].cst, nv[j], nv[j]);
            if (t.n[j].kind == kGates) {
                spread_gates<NW>(gates + t.n[j].spread, lane, nv[j], t.n[j].comps);
            } else {
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    no[j][i] = fmaf(sc[t.n[j].out + lane * NW + i], nv[j][i], no[j][i]);
                    nsq[j] = fmaf(no[j][i], no[j][i], nsq[j]);
                }
                Packed<T, NW>::store(z_out + z * t.dout + t.n[j].out + lane * NW, no[j]);
            }
        }
        __syncwarp();
        float o[K][VEC];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            wsq[k] = 0.0f;
            if (!(wide_has >> k & 1u)) continue;
            const float s = s_in[t.w[k].bi];
            float v[VEC], c[VEC];
            py[k].unpack(v);
            pr[k].unpack(o[k]);
            load_n<VEC>(wp + t.w[k].in + lane * VEC, c);
            mul_n<VEC>(v, c, v);
            if (t.w[k].gates >= 0) {
                load_n<VEC>(gates + t.w[k].gates + lane * VEC, c);
                scale_n<VEC>(c, s, c);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) c[i] = s;
            }
            fma_n<VEC>(v, c, o[k], o[k]);
            wsq[k] = dot_n<VEC>(o[k], o[k]);
            Packed<T, VEC>::store(z_out + z * t.dout + t.w[k].out + lane * VEC, o[k]);
        }
        if (!h_out) {
            __syncwarp();
            continue;
        }
        row_sums<false, K, M>(wsq, nsq, t.wide_out_ends, t.narrow_out_ends, t.inv_out, eps, s_out);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!(wide_has >> k & 1u)) continue;
            const float s = s_out[t.w[k].bo];
            float c[VEC];
            load_n<VEC>(wn + t.w[k].out + lane * VEC, c);
            scale_n<VEC>(c, s, c);
            mul_n<VEC>(o[k], c, o[k]);
            Packed<T, VEC>::store(h_out + z * t.dout + t.w[k].out + lane * VEC, o[k]);
        }
#pragma unroll
        for (int j = 0; j < M; ++j) {
            if (!(out_has >> j & 1u)) continue;
            const float s = s_out[t.n[j].bo];
#pragma unroll
            for (int i = 0; i < NW; ++i) no[j][i] *= s * wn[t.n[j].out + lane * NW + i];
            Packed<T, NW>::store(h_out + z * t.dout + t.n[j].out + lane * NW, no[j]);
        }
        __syncwarp();
    }
}

}  // namespace
}  // namespace e3b

using namespace e3b;

extern "C" int e3b_norm_gate_residual_fwd(const void* residual, const void* y, const float* weight_post, const float* scale,
                                          const float* weight_pre, const int32_t* wide, const int32_t* narrow, const int32_t* in_table,
                                          const int32_t* out_table, const float* in_inv, const float* out_inv, const int32_t* sizes,
                                          const int32_t* plan, float eps, void* z, void* h, int64_t rows, int type, void* stream) {
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
    // One warp a row where its columns fit the registers of a warp and there are rows for eight warps an SM.  (64 rows of 384 + 288
    // columns: 12 us by warps, 5 us by thread blocks; 262,144 rows of 1,216 + 1,024 columns in bf16: 858 against 1,080 us.)
    RowPlan rp;
    const int* counts = plan ? plan + kPlanHead + kPlanSlot * (plan[2] + plan[3]) : nullptr;
    if (plan && row_plan(plan, counts, counts + plan[6], &rp)) {
        const int size = rp.num_wide <= 3 && rp.num_narrow <= 3 ? 3 : rp.num_wide <= 5 && rp.num_narrow <= 4 ? 5 : 9, vec = plan[0];
        const int padded = (rp.din + 3) / 4 * 4 + 2 * ((rp.dout + 3) / 4 * 4), spread = (rp.num_spread + 3) / 4 * 4 + 2 * kMaxBlocks;
        auto launch = [&](auto t0, auto v0, auto n0, auto k0, auto m0) -> int {
            using T = decltype(t0);
            constexpr int VEC = decltype(v0)::value, NW = decltype(n0)::value, K = decltype(k0)::value, M = decltype(m0)::value;
            constexpr int kStage = NW * sizeof(T) >= 4 ? 2 * (K * VEC + M * NW) * 32 * static_cast<int>(sizeof(T)) : 0;
            const int64_t per_warp = 4 * spread + kStage;
            int warps = static_cast<int>(std::min<int64_t>(row_warps(VEC, K), (112 * 1024 - 4 * padded) / per_warp));      // two blocks an SM
            if (warps < 1) warps = 1;
            const size_t smem = 4 * padded + warps * per_warp;
            int grid = 0;
            const int e = resident_blocks(norm_gate_fwd_row_kernel<T, VEC, NW, K, M>, 32 * warps, smem, ceil_div(rows, warps), &grid);
            if (e != E3B_OK) return e;
            norm_gate_fwd_row_kernel<T, VEC, NW, K, M><<<grid, 32 * warps, smem, static_cast<cudaStream_t>(stream)>>>(
                static_cast<const T*>(residual), static_cast<const T*>(y), weight_post, scale, weight_pre, in_table, out_table, rp, eps,
                static_cast<T*>(z), static_cast<T*>(h), rows);
            return check_launch("norm_gate_residual_fwd");
        };
        auto by_size = [&](auto t0, auto v0, auto n0, auto most) -> int {
            if (size == 3) return launch(t0, v0, n0, Int<3>(), Int<3>());
            if (size == 5) return launch(t0, v0, n0, Int<5>(), Int<4>());
            return launch(t0, v0, n0, Int<9>(), most);
        };
        auto by_width = [&](auto t0) -> int {
            if constexpr (sizeof(t0) == 2) {
                if (vec == 8) return size == 3 ? launch(t0, Int<8>(), Int<2>(), Int<3>(), Int<3>()) : launch(t0, Int<8>(), Int<2>(), Int<5>(), Int<4>());
            }
            if (vec == 4) return by_size(t0, Int<4>(), Int<2>(), Int<4>());
            return by_size(t0, Int<1>(), Int<1>(), Int<8>());
        };
        const bool known = vec == 1 ? plan[1] == 1 : plan[1] == 2 && (vec == 4 || (vec == 8 && type != kFloat32));
        if (known && vec <= s.vec && rows >= 8 * kNumSMs && (size < 9 || (vec < 8 && (vec == 1 || rp.num_narrow <= 4)))) {
            if (type == kFloat32) return by_width(float());
            return type == kBFloat16 ? by_width(__nv_bfloat16()) : by_width(__half());
        }
    }
    const int64_t floats = BlockSums::floats(t.nblk_in, t.nw) + BlockSums::floats(t.nblk_out, t.nw) + (t.num_gates + 4) / 4 * 4;
    return by_type_and_items(type, s, [&](auto t0, auto v0, auto n0, auto k0, auto m0, auto x0) -> int {
        using T = decltype(t0);
        constexpr int VEC = decltype(v0)::value, NW = decltype(n0)::value, K = decltype(k0)::value, M = decltype(m0)::value, MAXT = decltype(x0)::value, AHEAD = rows_ahead(NW * sizeof(T), K > M ? K : M);
        constexpr int BLOCKS = MAXT == 128 ? 6 : MAXT == 256 ? 3 : 1;
        const size_t smem = sizeof(float) * floats + static_cast<size_t>(RowAhead<T, VEC, K, 2, AHEAD>::kThread + RowAhead<T, NW, M, 2, AHEAD>::kThread) * s.threads;
        int grid = 0;
        const int e = resident_blocks(norm_gate_fwd_kernel<T, VEC, NW, K, M, MAXT, BLOCKS>, s.threads, smem, rows, &grid);
        if (e != E3B_OK) return e;
        norm_gate_fwd_kernel<T, VEC, NW, K, M, MAXT, BLOCKS><<<grid, s.threads, smem, static_cast<cudaStream_t>(stream)>>>(
            static_cast<const T*>(residual), static_cast<const T*>(y), weight_post, scale, weight_pre, t, eps, static_cast<T*>(z),
            static_cast<T*>(h), rows);
        return check_launch("norm_gate_residual_fwd");
    });
}
