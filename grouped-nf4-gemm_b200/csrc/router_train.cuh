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
// One warp per token, the row in registers (16-byte loads: lane l holds V neighbouring experts of every 32 V), so the
// logits are read once forward and once backward and nothing of size [T, E] is written but the gradient.
//
// The k largest: the k-th largest of the lanes' own maxima bounds the k-th largest of the row from below, and in the mean
// only a few more than k elements reach that bound.  They are gathered in shared memory, one per lane, and each lane
// counts how many of them are larger than its own, and only where two are equal how many of those have a lower index: that
// is its place.  From k = 17 on the mean number that reaches the bound passes 32 (about 130 for k = 32): the bound is then
// taken from two maxima a lane, and up to 64 candidates are ranked two a lane (16384 x 1024, top 32: 625 -> 102 us).
// Where still more reach the bound (many equal logits) the k are picked one after the other.  Picking alone, a scan of
// the lane's registers per choice, costs about three times the instructions, and instructions are what bounds this pass.
//
// ex2, lg2 and rcp are the approximate ones (two units of the last fp32 place and less): what is summed stays fp32, and a
// row's sum of E terms is rounded by more than that.
//
// Forward keeps each warp's probability sums in registers over all its tokens and the counts as integers in shared
// memory.  The warps of a CTA are added in a fixed order, the CTAs by integer atomics: counts as they are, probability
// sums as 64-bit fixed-point numbers in steps of 2^-32 (a sum is at most 2^31; a step is far below the fp32 sums' own
// rounding), so that the order in which CTAs arrive cannot change a bit.  The last CTA to arrive computes the losses.
//
// Measured at 65536 tokens x 256 experts, top 8, fp32 (67 MB of logits, 10 us of reading): forward 51 us, about 500
// instructions a token at 71 % of the issue slots and 10 us of launches and joining (115 us with k scans, and 27 to 66 us more for
// a second kernel over the CTAs' sums); backward 35 us, about 320 instructions a token (42 us with 24 instead of 32 warps per
// SM; 20 us would be the bytes; 34 without the sum that corrects lse).  65536 x 32 bf16, top 4: 28.7 and 13.4 us (12.3 without).
#pragma once

#include "common.cuh"

namespace gnf4b {

constexpr int kRtMaxExperts = 1024;
constexpr int kRtMaxK = 32;
constexpr int kRtFewK = 16;          // up to here one maximum a lane bounds the k-th largest closely enough

// Order-preserving integer of a float: -NaN .. -inf .. +inf .. +NaN; a NaN is to come last, see rt_fix_nan.
constexpr uint32_t kRtKeyInf = 0xff800000u, kRtKeyNegInf = 0x007fffffu;
__device__ __forceinline__ uint32_t rt_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);                 // -0 and +0 tie
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint32_t rt_fix_nan(uint32_t key) { return key > kRtKeyInf || key < kRtKeyNegInf ? 1u : key; }
__device__ __forceinline__ float rt_value(uint32_t key) {
    if (key == 1u) return __uint_as_float(0x7fc00000u);
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
__device__ __forceinline__ float rt_exp(float x) {                // e^x, x <= 0 but for NaN: a few units of 2^-24 times (1 + |x|)
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
    return r;
}

// The row of NE elements per lane: element i of a lane is expert rt_expert(lane, i).  LT 0 bf16, 1 fp16, 2 fp32.
template <int LT, int NE>
struct RtRow {
    static constexpr int V = LT == 2 ? (NE < 4 ? NE : 4) : (NE < 8 ? NE : 8);
    static constexpr int kWords = V * (LT == 2 ? 4 : 2) / 4;      // 32-bit words of a vector; 0: one 16-bit element
    __device__ __forceinline__ static int expert(int lane, int i) { return (i / V) * (32 * V) + lane * V + (i % V); }
    // experts >= E read as -inf.  vec: rows and E allow whole vectors
    __device__ __forceinline__ static void load(const void* row, int lane, int E, bool vec, float* x) {
#pragma unroll
        for (int g = 0; g < NE / V; ++g) {
            const int e0 = g * 32 * V + lane * V;
            if (kWords > 0 && vec) {
                uint32_t w[kWords > 0 ? kWords : 1];
                const uint8_t* p = static_cast<const uint8_t*>(row) + (int64_t)e0 * (LT == 2 ? 4 : 2);
                const bool in = e0 < E;
                constexpr uint32_t none = LT == 2 ? 0xff800000u : LT == 0 ? 0xff80ff80u : 0xfc00fc00u;       // -inf
                if (kWords == 4) {
                    uint4 q = make_uint4(none, none, none, none);
                    if (in) q = __ldcs(reinterpret_cast<const uint4*>(p));
                    w[0] = q.x;
                    if (kWords > 1) w[kWords > 1 ? 1 : 0] = q.y;
                    if (kWords > 2) { w[kWords > 2 ? 2 : 0] = q.z; w[kWords > 3 ? 3 : 0] = q.w; }
                } else if (kWords == 2) {
                    uint2 q = make_uint2(none, none);
                    if (in) q = __ldcs(reinterpret_cast<const uint2*>(p));
                    w[0] = q.x;
                    w[kWords > 1 ? 1 : 0] = q.y;
                } else {
                    w[0] = in ? __ldcs(reinterpret_cast<const uint32_t*>(p)) : none;
                }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (LT == 2) {
                        x[g * V + j] = __uint_as_float(w[j < kWords ? j : 0]);
                    } else {
                        const uint32_t h = (w[(j >> 1) < kWords ? (j >> 1) : 0] >> (16 * (j & 1))) & 0xffffu;
                        x[g * V + j] = LT == 0 ? bf16_bits_to_float(h) : __half2float(__ushort_as_half((unsigned short)h));
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float v = -INFINITY;
                    if (e0 + j < E) {
                        if (LT == 2) v = __ldg(static_cast<const float*>(row) + e0 + j);
                        else {
                            const unsigned short h = __ldg(static_cast<const unsigned short*>(row) + e0 + j);
                            v = LT == 0 ? bf16_bits_to_float(h) : __half2float(__ushort_as_half(h));
                        }
                    }
                    x[g * V + j] = v;
                }
            }
        }
    }
    __device__ __forceinline__ static uint32_t bits(float v) {
        return LT == 2 ? __float_as_uint(v) : LT == 0 ? (uint32_t)f32_to_bf16_bits(v) : (uint32_t)__half_as_ushort(__float2half_rn(v));
    }
    __device__ __forceinline__ static void store(void* row, int lane, int E, bool vec, const float* x) {
#pragma unroll
        for (int g = 0; g < NE / V; ++g) {
            const int e0 = g * 32 * V + lane * V;
            if (kWords > 0 && vec) {
                uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if (LT == 2) w[j & 3] = bits(x[g * V + j]);
                    else w[(j >> 1) & 3] |= bits(x[g * V + j]) << (16 * (j & 1));
                }
                uint8_t* p = static_cast<uint8_t*>(row) + (int64_t)e0 * (LT == 2 ? 4 : 2);
                if (e0 < E) {
                    if (kWords == 4) __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
                    else if (kWords == 2) __stcs(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[1]));
                    else __stcs(reinterpret_cast<uint32_t*>(p), w[0]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (e0 + j < E) {
                        if (LT == 2) static_cast<float*>(row)[e0 + j] = x[g * V + j];
                        else static_cast<uint16_t*>(row)[e0 + j] = (uint16_t)bits(x[g * V + j]);
                    }
            }
        }
    }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ float warp_max(float v) {              // of what is not NaN
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

__device__ __forceinline__ float rt_log(float x) {                // ln x, 1 <= x: off by at most 2^-22 or two units in the last place
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r * 0.6931471805599453f;
}
__device__ __forceinline__ float rt_rcp(float x) {                // 1 / x to one unit in the last place
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

struct RouteTrainArgs {
    const void* logits;
    int64_t T, stride;           // elements between rows
    int32_t E, k, mode, norm;
    int32_t vec;                 // rows and E allow 16-byte loads
    const uint8_t* mask;         // optional, nonzero = counts
    int64_t* idx;
    float* w;
    float* lse;
    int32_t* counts;
    float* balance;
    float* z;
    float* n_tokens;
    // scratch of several CTAs, zero before the launch but for part_zn
    unsigned long long* sum_p;   // [E], steps of 2^-32
    uint32_t* sum_c;             // [E]
    uint32_t* arrived;
    uint32_t* not_finite;        // a probability sum was NaN
    float* part_zn;              // [grid][2]
};
__host__ __device__ inline size_t rt_zeroed_bytes(int32_t E) { return (size_t)E * 12 + 8; }

// MANY: k > kRtFewK
template <int LT, int NE, int WARPS, bool MANY>
__global__ void __launch_bounds__(WARPS * 32, NE <= 8 ? 2 : 1)
route_train_fwd_kernel(const __grid_constant__ RouteTrainArgs a) {
    using Row = RtRow<LT, NE>;
    constexpr int kRtCand = MANY ? 64 : 32;          // candidates for the k places that are ranked together
    extern __shared__ __align__(16) float s_mem[];   // [WARPS][E] probability sums, then [E] counts
    __shared__ __align__(16) float s_val[WARPS][kRtCand];
    __shared__ __align__(16) int32_t s_exp[WARPS][kRtCand];
    __shared__ float s_zn[WARPS][2];
    __shared__ float s_tot[34];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int32_t* s_c = reinterpret_cast<int32_t*>(s_mem + WARPS * a.E);
    for (int e = threadIdx.x; e < a.E; e += WARPS * 32) s_c[e] = 0;
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    float psum[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) psum[i] = 0.f;
    float zsum = 0.f, ntok = 0.f;
    const int64_t step = (int64_t)gridDim.x * WARPS;
    const int64_t item = LT == 2 ? 4 : 2;
    const uint8_t* base = static_cast<const uint8_t*>(a.logits);
    const bool vec = a.vec != 0, renorm = a.mode == 1 || a.norm;
    int64_t t = (int64_t)blockIdx.x * WARPS + warp;
    float v[NE];
    if (t < a.T) Row::load(base + t * a.stride * item, lane, a.E, vec, v);
    for (; t < a.T; t += step) {
        float r[NE], x[NE], best = -INFINITY;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            r[i] = v[i];
            best = fmaxf(best, r[i]);
        }
        const bool masked = a.mask && __ldg(a.mask + t) == 0;
        if (t + step < a.T) Row::load(base + (t + step) * a.stride * item, lane, a.E, vec, v);     // on its way meanwhile
        float top = warp_max(best), z = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            x[i] = rt_exp(r[i] - top);
            z += x[i];
        }
        z = warp_sum(z);
        bool dead = false;                           // nothing to choose from: no weight, no loss, no count
        const bool plain = z == z;
        if (!plain) {                                // a NaN, an infinity or nothing but -inf: rare
            bool nan = false;
            uint32_t top_key = 0;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const uint32_t key = rt_key(r[i]), fixed = rt_fix_nan(key);
                nan |= fixed != key;
                top_key = max(top_key, Row::expert(lane, i) < a.E ? fixed : 0u);
            }
            top_key = __reduce_max_sync(0xffffffffu, top_key);
            top = rt_value(top_key);
            dead = !__any_sync(0xffffffffu, nan) && top_key == kRtKeyNegInf;
            if (dead) {
#pragma unroll
                for (int i = 0; i < NE; ++i) x[i] = 0.f;
            }
        }
        const bool counted = !masked && !dead;
        const float lse = dead ? -INFINITY : top + rt_log(z);
        if (counted) {
            const float rz = rt_rcp(z);
#pragma unroll
            for (int i = 0; i < NE; ++i) psum[i] = fmaf(x[i], rz, psum[i]);
            zsum += lse * lse;
            ntok += 1.f;
        }
        // the k largest
        float sel = 0.f;
        int32_t sel_e = 0, place = 32;
        int found = kRtCand + 1;
        if (plain) {
            float bound = top;
            if (!MANY) {
                float left = best;
#pragma unroll 4
                for (int j = 1; j < a.k; ++j) {
                    if (left == bound) left = -INFINITY;
                    bound = warp_max(left);
                }
            } else {                                 // two maxima a lane: of the first and of the second half of its elements
                float left0 = r[0], left1 = r[NE / 2];
#pragma unroll
                for (int i = 1; i < NE / 2; ++i) {
                    left0 = fmaxf(left0, r[i]);
                    left1 = fmaxf(left1, r[NE / 2 + i]);
                }
                for (int j = 1; j < a.k; ++j) {
                    if (left0 == bound) left0 = -INFINITY;
                    if (left1 == bound) left1 = -INFINITY;
                    bound = warp_max(fmaxf(left0, left1));
                }
            }
            // (a bound of -inf would take in the experts >= E: one after the other then)
            if (bound > -INFINITY) {
                int n = 0;
#pragma unroll
                for (int i = 0; i < NE; ++i) n += r[i] >= bound ? 1 : 0;
                // candidates of the lanes before this one and of all, bit by bit of the count
                const uint32_t before = (1u << lane) - 1u;
                int at = 0;
                found = 0;
#pragma unroll
                for (int b = 0; (1 << b) <= NE; ++b) {
                    const uint32_t who = __ballot_sync(0xffffffffu, n >> b & 1);
                    at += __popc(who & before) << b;
                    found += __popc(who) << b;
                }
                if (found <= kRtCand) {
#pragma unroll
                    for (int i = 0; i < NE; ++i)
                        if (r[i] >= bound) {
                            s_val[warp][at] = r[i];
                            s_exp[warp][at] = Row::expert(lane, i);
                            ++at;
                        }
                    // the ranking reads four at a time
                    for (int j = lane; j < ((found + 3) & ~3) || j < 32; j += 32)
                        if (j >= found) {
                            s_val[warp][j] = -INFINITY;
                            s_exp[warp][j] = INT32_MAX;
                        }
                }
            }
        }
        const auto ranked = [&](float val, int32_t e) {       // candidates before this one
            int before = 0;
            for (int j = 0; j < found; j += 4) {
                const float4 ov = *reinterpret_cast<const float4*>(&s_val[warp][j]);
                const int4 oe = *reinterpret_cast<const int4*>(&s_exp[warp][j]);
                before += (ov.x > val || (ov.x == val && oe.x < e)) ? 1 : 0;
                before += (ov.y > val || (ov.y == val && oe.y < e)) ? 1 : 0;
                before += (ov.z > val || (ov.z == val && oe.z < e)) ? 1 : 0;
                before += (ov.w > val || (ov.w == val && oe.w < e)) ? 1 : 0;
            }
            return before;
        };
        if (found <= 32) {
            __syncwarp();
            sel = s_val[warp][lane];
            sel_e = s_exp[warp][lane];
            place = 0;
            for (int j = 0; j < found; j += 4) {
                const float4 ov = *reinterpret_cast<const float4*>(&s_val[warp][j]);
                place += (ov.x > sel) + (ov.y > sel) + (ov.z > sel) + (ov.w > sel);
            }
            // equal ones share a place: once more with the index
            if (__popc(__reduce_or_sync(0xffffffffu, lane < found ? 1u << place : 0u)) != found) place = ranked(sel, sel_e);
            if (lane >= found) place = 32;
        } else if (MANY && found <= kRtCand) {       // two a lane; the k then go to their places
            __syncwarp();
            const bool second = lane + 32 < found;
            const int two = lane + (MANY ? 32 : 0);
            const float v0 = s_val[warp][lane], v1 = second ? s_val[warp][two] : -INFINITY;
            const int32_t e0 = s_exp[warp][lane], e1 = second ? s_exp[warp][two] : INT32_MAX;
            const int p0 = ranked(v0, e0), p1 = second ? ranked(v1, e1) : kRtCand;
            __syncwarp();
            if (p0 < a.k) { s_val[warp][p0] = v0; s_exp[warp][p0] = e0; }
            if (p1 < a.k) { s_val[warp][p1] = v1; s_exp[warp][p1] = e1; }
            __syncwarp();
            if (lane < a.k) {
                sel = s_val[warp][lane];
                sel_e = s_exp[warp][lane];
                place = lane;
            }
        } else {
            // one after the other: the largest key left, and of its holders the lowest expert
            uint32_t mask = 0;                       // this lane's elements that are taken
            for (int j = 0; j < a.k; ++j) {
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < NE; ++i)
                    if (!(mask >> i & 1u) && Row::expert(lane, i) < a.E) m = max(m, rt_fix_nan(rt_key(r[i])));
                m = __reduce_max_sync(0xffffffffu, m);
                uint32_t e = 0xffffffffu;
#pragma unroll
                for (int i = 0; i < NE; ++i)
                    if (!(mask >> i & 1u) && rt_fix_nan(rt_key(r[i])) == m && Row::expert(lane, i) < a.E) e = min(e, (uint32_t)Row::expert(lane, i));
                e = __reduce_min_sync(0xffffffffu, e);
#pragma unroll
                for (int i = 0; i < NE; ++i)
                    if ((uint32_t)Row::expert(lane, i) == e) mask |= 1u << i;
                if (lane == j) { sel = rt_value(m); sel_e = (int32_t)e; place = j; }
            }
        }
        const bool chosen = place < a.k;
        const float ej = (chosen && !dead) ? rt_exp(sel - top) : 0.f;
        // renormalised probabilities of a row with a NaN are NaN like the probabilities; mode 1 has only the chosen logits
        if (renorm) z = warp_sum(ej) + (a.mode == 0 && !plain && !dead ? z : 0.f);
        if (chosen) {
            a.idx[t * a.k + place] = sel_e;
            a.w[t * a.k + place] = dead ? 0.f : ej * rt_rcp(z);
            if (counted) atomicAdd(s_c + sel_e, 1);
        }
        if (lane == 0) a.lse[t] = lse;
        __syncwarp();                                // before the candidates' slots are written again
    }
    __syncthreads();
    float* s_p = s_mem;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int e = Row::expert(lane, i);
        if (e < a.E) s_p[warp * a.E + e] = psum[i];
    }
    if (lane == 0) { s_zn[warp][0] = zsum; s_zn[warp][1] = ntok; }
    __syncthreads();
    const bool only = gridDim.x == 1;
    for (int e = threadIdx.x; e < a.E; e += WARPS * 32) {
        float p = 0.f;
        for (int q = 0; q < WARPS; ++q) p += s_p[q * a.E + e];
        s_p[e] = p;                                  // its own column: no other thread reads it
        if (!only) {
            if (p == p) atomicAdd(a.sum_p + e, (unsigned long long)((double)p * 4294967296.0));
            else atomicOr(a.not_finite, 1u);
            if (s_c[e]) atomicAdd(a.sum_c + e, (uint32_t)s_c[e]);
        }
    }
    float z = 0.f, n = 0.f;
    if (threadIdx.x == 0) {
        for (int q = 0; q < WARPS; ++q) { z += s_zn[q][0]; n += s_zn[q][1]; }
        s_tot[32] = z;
        s_tot[33] = n;
        if (!only) {
            a.part_zn[2 * blockIdx.x] = z;
            a.part_zn[2 * blockIdx.x + 1] = n;
        }
    }
    __shared__ uint32_t s_last;
    if (!only) {
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) s_last = atomicAdd(a.arrived, 1u) == gridDim.x - 1;
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        if (warp == 0) {                             // part lane, lane + 32, ... then a fixed tree
            z = 0.f;
            n = 0.f;
            for (int c = lane; c < (int)gridDim.x; c += 32) { z += __ldcg(a.part_zn + 2 * c); n += __ldcg(a.part_zn + 2 * c + 1); }
            z = warp_sum(z);
            n = warp_sum(n);
            if (lane == 0) { s_tot[32] = z; s_tot[33] = n; }
        }
        const bool bad = __ldcg(a.not_finite) != 0;
        for (int e = threadIdx.x; e < a.E; e += WARPS * 32) {
            s_c[e] = (int32_t)__ldcg(a.sum_c + e);
            s_p[e] = bad ? __uint_as_float(0x7fc00000u) : (float)((double)__ldcg(a.sum_p + e) * (1.0 / 4294967296.0));
        }
    }
    float bal = 0.f;                                 // each thread its own columns of s_c and s_p
    for (int e = threadIdx.x; e < a.E; e += WARPS * 32) {
        a.counts[e] = s_c[e];
        bal += (float)s_c[e] * s_p[e];
    }
    bal = warp_sum(bal);
    if (lane == 0) s_tot[warp] = bal;
    __syncthreads();
    if (threadIdx.x == 0) {
        float sum = 0.f;
        for (int q = 0; q < WARPS; ++q) sum += s_tot[q];
        const float nt = s_tot[33];
        *a.n_tokens = nt;
        *a.balance = nt > 0.f ? (float)a.E * (sum / (nt * (float)a.k)) / nt : 0.f;
        *a.z = nt > 0.f ? s_tot[32] / nt : 0.f;
    }
}

struct RouteTrainBwdArgs {
    const void* logits;
    int64_t T, stride;
    int32_t E, k, mode, norm;
    int32_t vec, vec_grad;       // rows and E allow 16-byte loads / stores
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
__global__ void __launch_bounds__(WARPS * 32, NE <= 8 ? 4 : NE == 16 ? 2 : 1)
route_train_bwd_kernel(const __grid_constant__ RouteTrainBwdArgs a) {
    using Row = RtRow<LT, NE>;
    __shared__ __align__(16) float s_sel[WARPS][NE * 32];        // what the weights' gradient adds at the chosen experts
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float* mine = s_sel[warp];
#pragma unroll
    for (int i = 0; i < NE; ++i) mine[lane + 32 * i] = 0.f;
    pdl_wait();
    pdl_launch_dependents();
    __syncwarp();
    const float n = __ldg(a.n_tokens);
    const float gb = (a.g_balance && n > 0.f) ? __ldg(a.g_balance) * (float)a.E / (n * n * (float)a.k) : 0.f;
    const float gz = (a.g_z && n > 0.f) ? 2.f * __ldg(a.g_z) / n : 0.f;
    const bool losses = gb != 0.f || gz != 0.f;      // else no term of theirs: a NaN logit times nothing is not NaN
    float push[NE];                                  // d balance / d p_e of one token
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int e = Row::expert(lane, i);
        push[i] = e < a.E ? gb * (float)__ldg(a.counts + e) : 0.f;
    }
    const bool renorm = a.mode == 1 || a.norm, vec = a.vec != 0, vec_grad = a.vec_grad != 0;
    const int64_t item = LT == 2 ? 4 : 2;
    const int64_t step = (int64_t)gridDim.x * WARPS;
    int64_t t = (int64_t)blockIdx.x * WARPS + warp;
    // a token's loads are issued while the one before it is worked on
    float v[NE], lse_n = 0.f, w_n = 0.f, g_n = 0.f;
    int64_t e_n = -1;
    bool keep_n = true;
    auto load = [&](int64_t row) {
        Row::load(static_cast<const uint8_t*>(a.logits) + row * a.stride * item, lane, a.E, vec, v);
        lse_n = __ldg(a.lse + row);
        if (a.mask) keep_n = __ldg(a.mask + row) != 0;
        if (a.g_w && lane < a.k) {
            e_n = __ldg(a.idx + row * a.k + lane);
            w_n = __ldg(a.w + row * a.k + lane);
            g_n = __ldg(a.g_w + row * a.k + lane);
        }
    };
    if (t < a.T) load(t);
    for (; t < a.T; t += step) {
        const float lse = lse_n, w = w_n, g = g_n;
        const int64_t e_sel = e_n;
        const bool dead = lse == -INFINITY;
        const bool counted = losses && !dead && keep_n;
        const bool has = e_sel >= 0 && e_sel < a.E;
        // lse in one fp32 number is off by up to half its last place, 5e-4 where the logits are around 10000, and by the same
        // for every expert of the token: dividing by the sum of what it gives, which lies near 1, takes that factor out
        float p[NE], ap = 0.f, z = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            p[i] = dead ? 0.f : rt_exp(v[i] - lse);
            z += p[i];
            ap = fmaf(p[i], push[i], ap);
        }
        if (t + step < a.T) load(t + step);
        // nothing comes back through this token's weights (padding, or weights that are not used): no term, whatever its
        // logits are -- a NaN in a masked token stays out
        const bool through_w = __any_sync(0xffffffffu, g != 0.f) && !dead;
        float gw = g * w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            gw += __shfl_xor_sync(0xffffffffu, gw, o);
            ap += __shfl_xor_sync(0xffffffffu, ap, o);
            z += __shfl_xor_sync(0xffffffffu, z, o);
        }
        const float rz = dead ? 0.f : rt_rcp(z);
        ap *= rz;
#pragma unroll
        for (int i = 0; i < NE; ++i) p[i] *= rz;
        if (through_w && has) mine[e_sel] = renorm ? w * (g - gw) : g;
        __syncwarp();
        const float zc = gz * lse - ap;
        float d[NE];
#pragma unroll
        for (int i = 0; i < NE; ++i) d[i] = counted ? p[i] * (push[i] + zc) : 0.f;
        if (through_w) {
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const float s = mine[Row::expert(lane, i)];
                d[i] += renorm ? s : p[i] * (s - gw);
            }
        }
        Row::store(static_cast<uint8_t*>(a.grad) + t * a.E * item, lane, a.E, vec_grad, d);
        __syncwarp();
        if (has) mine[e_sel] = 0.f;
        __syncwarp();
    }
}

}  // namespace gnf4b
