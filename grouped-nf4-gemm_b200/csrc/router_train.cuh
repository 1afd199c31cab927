// Top-k routing for training: selection and weights as route_topk_kernel (ep_kernels.cuh) has them, with per-expert
// counts, the balance loss and the z loss in the same pass, and the gradient of all of it in a second one.
//
//   p = softmax(l),  lse = log sum exp l,  idx = the k largest (ties to the lower index),  w = p[idx] or renormalised
//   over the n tokens that count (token_mask, at least one logit above -inf):
//     counts_e = tokens that chose e,  f_e = counts_e / (n k),  P_e = mean p_e
//     balance = E sum_e f_e P_e          z = mean lse^2
//   dl_e = p_e (G_e - sum_j p_j G_j) + 2 g_z lse p_e / n,   G_e = [e = idx_j] g_w_j + g_b E f_e / n
//   (f is piecewise constant; renormalised weights instead give w_j (g_j - sum_i w_i g_i) at idx_j)
//
// One warp per token, the row in registers (lane = expert mod 32), so the logits are read once forward and once
// backward and nothing of size [T, E] is written but the gradient.  Forward keeps each warp's probability sums and
// counts in registers over all its tokens; warps of a CTA, then CTAs, are added in a fixed order: no floating-point
// atomics, the same bits on every run.
#pragma once

#include "common.cuh"

namespace gnf4b {

constexpr int kRtMaxExperts = 1024;
constexpr int kRtMaxK = 32;

// Order-preserving integer of a float: NaN 1, then -inf .. +inf; 0 is left for "no expert here" and "already taken".
__device__ __forceinline__ uint32_t rt_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);                 // -0 and +0 tie
    if ((b & 0x7fffffffu) > 0x7f800000u) return 1u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float rt_value(uint32_t key) {
    if (key == 1u) return __uint_as_float(0x7fc00000u);
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

template <int LT>      // 0 bf16, 1 fp16, 2 fp32
__device__ __forceinline__ float rt_load(const void* p, int64_t i) {
    if (LT == 2) return __ldg(static_cast<const float*>(p) + i);
    const unsigned short b = __ldg(static_cast<const unsigned short*>(p) + i);
    return LT == 0 ? bf16_bits_to_float(b) : __half2float(__ushort_as_half(b));
}
template <int LT>
__device__ __forceinline__ void rt_store(void* p, int64_t i, float v) {
    if (LT == 2) static_cast<float*>(p)[i] = v;
    else if (LT == 0) static_cast<uint16_t*>(p)[i] = f32_to_bf16_bits(v);
    else static_cast<unsigned short*>(p)[i] = __half_as_ushort(__float2half_rn(v));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct RouteTrainArgs {
    const void* logits;
    int64_t T, stride;           // elements between rows
    int32_t E, k, mode, norm;
    const uint8_t* mask;         // optional, nonzero = counts
    int64_t* idx;
    float* w;
    float* lse;
    int32_t* counts;
    float* balance;
    float* z;
    float* n_tokens;
    float* part_p;               // [grid][E]
    int32_t* part_c;             // [grid][E]
    float* part_zn;              // [grid][2]
};

// sums over the CTAs' parts (or the one CTA's own) -> counts, losses; all threads of one CTA
__device__ __forceinline__ void rt_finish(const RouteTrainArgs& a, int parts, const float* part_p, const int32_t* part_c,
                                          const float* part_zn, float* s_red) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, warps = blockDim.x >> 5;
    float z = 0.f, n = 0.f;
    if (t < 32) {                                    // one warp: part t, t + 32, ... then a fixed tree
        for (int c = t; c < parts; c += 32) { z += part_zn[2 * c]; n += part_zn[2 * c + 1]; }
        z = warp_sum(z);
        n = warp_sum(n);
        if (t == 0) { s_red[64] = z; s_red[65] = n; }
    }
    float bal = 0.f;
    for (int e = t; e < a.E; e += blockDim.x) {
        float p = 0.f;
        int32_t c = 0;
#pragma unroll 8
        for (int q = 0; q < parts; ++q) {
            p += part_p[(int64_t)q * a.E + e];
            c += part_c[(int64_t)q * a.E + e];
        }
        a.counts[e] = c;
        bal += (float)c * p;
    }
    bal = warp_sum(bal);
    if (lane == 0) s_red[warp] = bal;
    __syncthreads();
    if (t == 0) {
        float sum = 0.f;
        for (int v = 0; v < warps; ++v) sum += s_red[v];
        const float nt = s_red[65];
        *a.n_tokens = nt;
        *a.balance = nt > 0.f ? (float)a.E * (sum / (nt * (float)a.k)) / nt : 0.f;
        *a.z = nt > 0.f ? s_red[64] / nt : 0.f;
    }
}

template <int LT, int NE, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
route_train_fwd_kernel(const RouteTrainArgs a) {
    extern __shared__ float s_mem[];                 // [WARPS][E] probability sums, then as many counts
    __shared__ float s_zn[WARPS][2];
    __shared__ float s_red[66];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    pdl_launch_dependents();
    float psum[NE];
    int32_t cnt[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) { psum[i] = 0.f; cnt[i] = 0; }
    float zsum = 0.f, ntok = 0.f;
    const int64_t step = (int64_t)gridDim.x * WARPS;
    int64_t t = (int64_t)blockIdx.x * WARPS + warp;
    float v[NE];
    auto load = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int e = lane + 32 * i;
            v[i] = (row < a.T && e < a.E) ? rt_load<LT>(a.logits, row * a.stride + e) : 0.f;
        }
    };
    load(t);
    for (; t < a.T; t += step) {
        uint32_t key[NE];
        float x[NE];
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            x[i] = v[i];
            key[i] = lane + 32 * i < a.E ? rt_key(x[i]) : 0u;
        }
        const bool masked = a.mask && __ldg(a.mask + t) == 0;
        load(t + step);                              // the next row is on its way while this one is worked on
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < NE; ++i) best = max(best, key[i]);
        const uint32_t top_key = __reduce_max_sync(0xffffffffu, best);
        const float top = rt_value(top_key);
        const bool dead = top == -INFINITY;          // nothing to choose from: no weight, no loss, no count
        const bool counted = !masked && !dead;
        float ex[NE], z = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            ex[i] = (!dead && lane + 32 * i < a.E) ? expf(x[i] - top) : 0.f;
            z += ex[i];
        }
        z = warp_sum(z);
        const float lse = dead ? -INFINITY : top + logf(z);
        if (counted) {
            const float rz = 1.0f / z;
#pragma unroll
            for (int i = 0; i < NE; ++i) psum[i] += ex[i] * rz;
            zsum += lse * lse;
            ntok += 1.f;
        }
        // the k largest, one after the other: the largest key left, and of its holders the lowest expert
        float sel = 0.f;
        int32_t sel_e = 0;
        uint32_t m = top_key;
        for (int j = 0; j < a.k; ++j) {
            if (j) m = __reduce_max_sync(0xffffffffu, best);
            int at = NE;
#pragma unroll
            for (int i = NE - 1; i >= 0; --i)
                if (key[i] == m) at = i;
            const uint32_t e = __reduce_min_sync(0xffffffffu, at < NE ? (uint32_t)(lane + 32 * at) : 0xffffffffu);
            if (lane == j) { sel = rt_value(m); sel_e = (int32_t)e; }
            const int gone = (int)(e & 31u) == lane ? (int)(e >> 5) : -1;
            best = 0;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                if (i == gone) { key[i] = 0; cnt[i] += counted ? 1 : 0; }
                best = max(best, key[i]);
            }
        }
        float wj = (lane < a.k && !dead) ? expf(sel - top) : 0.f;
        if (a.mode == 1 || a.norm) z = warp_sum(wj);
        wj = dead ? 0.f : wj / z;
        if (lane < a.k) {
            a.idx[t * a.k + lane] = sel_e;
            a.w[t * a.k + lane] = wj;
        }
        if (lane == 0) a.lse[t] = lse;
    }
    float* s_p = s_mem;
    int32_t* s_c = reinterpret_cast<int32_t*>(s_mem + WARPS * a.E);
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int e = lane + 32 * i;
        if (e < a.E) { s_p[warp * a.E + e] = psum[i]; s_c[warp * a.E + e] = cnt[i]; }
    }
    if (lane == 0) { s_zn[warp][0] = zsum; s_zn[warp][1] = ntok; }
    __syncthreads();
    if (gridDim.x == 1) {                            // a small batch: this CTA has everything
        rt_finish(a, WARPS, s_p, s_c, &s_zn[0][0], s_red);
        return;
    }
    for (int e = threadIdx.x; e < a.E; e += WARPS * 32) {
        float p = 0.f;
        int32_t c = 0;
        for (int q = 0; q < WARPS; ++q) { p += s_p[q * a.E + e]; c += s_c[q * a.E + e]; }
        a.part_p[(int64_t)blockIdx.x * a.E + e] = p;
        a.part_c[(int64_t)blockIdx.x * a.E + e] = c;
    }
    if (threadIdx.x == 0) {
        float z = 0.f, n = 0.f;
        for (int q = 0; q < WARPS; ++q) { z += s_zn[q][0]; n += s_zn[q][1]; }
        a.part_zn[2 * blockIdx.x] = z;
        a.part_zn[2 * blockIdx.x + 1] = n;
    }
}

static __global__ void __launch_bounds__(1024) route_train_finish_kernel(const RouteTrainArgs a, int parts) {
    __shared__ float s_red[66];
    pdl_wait();
    pdl_launch_dependents();
    rt_finish(a, parts, a.part_p, a.part_c, a.part_zn, s_red);
}

struct RouteTrainBwdArgs {
    const void* logits;
    int64_t T, stride;
    int32_t E, k, mode, norm;
    const uint8_t* mask;
    const int64_t* idx;
    const float* w;
    const float* lse;
    const int32_t* counts;
    const float* n_tokens;
    const float* g_w;            // [T, k], optional
    const float* g_balance;      // scalars on the device, optional
    const float* g_z;
    void* grad;                  // [T, E] contiguous, the logits' type
};

template <int LT, int NE, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
route_train_bwd_kernel(const RouteTrainBwdArgs a) {
    extern __shared__ float s_sel[];                 // [WARPS][E]: what the weights' gradient adds at the chosen experts
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float* mine = s_sel + warp * a.E;
    for (int e = lane; e < a.E; e += 32) mine[e] = 0.f;
    pdl_wait();
    pdl_launch_dependents();
    __syncwarp();
    const float n = __ldg(a.n_tokens);
    const float gb = (a.g_balance && n > 0.f) ? __ldg(a.g_balance) * (float)a.E / (n * n * (float)a.k) : 0.f;
    const float gz = (a.g_z && n > 0.f) ? 2.f * __ldg(a.g_z) / n : 0.f;
    float push[NE];                                  // d balance / d p_e of one token
#pragma unroll
    for (int i = 0; i < NE; ++i) push[i] = lane + 32 * i < a.E ? gb * (float)__ldg(a.counts + lane + 32 * i) : 0.f;
    const bool renorm = a.mode == 1 || a.norm;
    for (int64_t t = (int64_t)blockIdx.x * WARPS + warp; t < a.T; t += (int64_t)gridDim.x * WARPS) {
        float x[NE];
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int e = lane + 32 * i;
            x[i] = e < a.E ? rt_load<LT>(a.logits, t * a.stride + e) : 0.f;
        }
        const float lse = __ldg(a.lse + t);
        const bool dead = lse == -INFINITY;
        const bool counted = !dead && !(a.mask && __ldg(a.mask + t) == 0);
        int64_t e_sel = 0;
        float w = 0.f, g = 0.f;
        const bool has = a.g_w && lane < a.k;
        if (has) {
            e_sel = __ldg(a.idx + t * a.k + lane);
            w = __ldg(a.w + t * a.k + lane);
            g = __ldg(a.g_w + t * a.k + lane);
        }
        // nothing comes back through this token's weights (padding, or weights that are not used): no term, whatever its
        // logits are -- a NaN in a masked token stays out
        const bool through_w = __any_sync(0xffffffffu, g != 0.f);
        const float gw = warp_sum(g * w);
        if (has && e_sel >= 0 && e_sel < a.E) mine[e_sel] = renorm ? w * (g - gw) : g;
        __syncwarp();
        float p[NE], ap = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            p[i] = (!dead && lane + 32 * i < a.E) ? expf(x[i] - lse) : 0.f;
            ap += p[i] * push[i];
        }
        ap = warp_sum(ap);
        const float zc = gz * lse;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int e = lane + 32 * i;
            if (e < a.E) {
                const float s = mine[e];
                float d = (dead || !through_w) ? 0.f : renorm ? s : p[i] * (s - gw);
                if (counted) d += p[i] * (push[i] - ap + zc);
                rt_store<LT>(a.grad, t * a.E + e, d);
            }
        }
        __syncwarp();
        if (has && e_sel >= 0 && e_sel < a.E) mine[e_sel] = 0.f;
        __syncwarp();
    }
}

}  // namespace gnf4b
