// The GLU between an expert's two products, for training: forward also writes its input in 8 bits, backward reads only
// that and the incoming gradient.
//
//   forward   out = act(gate, up) in fp32, one rounding to bf16;
//             per 64 gate values and per 64 up values of a row: step = max|v| / 127, code = rint(v * (127 / max|v|))
//   backward  gate' = code * step, up' likewise;  d gate = g * d act / d gate, d up = g * d act / d up at (gate', up'),
//             fp32, one rounding to bf16
//     silu:     act = gate s(gate) up,                      s the logistic function
//     gpt-oss:  act = (up~ + 1) gate~ s(1.702 gate~), gate~ = min(gate, 7), up~ = clamp(up, -7, 7); no gradient beyond
//
// A step of the block's maximum / 127 costs at most half a step, 0.4 % of the block's largest magnitude, and halves what
// a layer keeps between the passes (2 bytes + 1/8 instead of 4 per pair).  A block whose maximum is below 2^-100 is kept
// as zeros (127 / max would leave the fp32 range); one with an infinity or a NaN restores to non-finite values.
//
// Both passes are bound by memory: eight pairs per thread, eight neighbouring lanes per block, 16-byte loads and
// stores, codes of a block side by side ([row][block][gate 64 | up 64], so any h is aligned).  sigmoid from ex2.approx
// and rcp.approx: two to three units in the last fp32 place, far below the bf16 rounding behind it; the exact
// division and expf would make the arithmetic, not the memory, the bound.
#pragma once

#include "common.cuh"

namespace gnf4b {

constexpr int kCkBlock = 64;
constexpr int kCkThreads = 256;

__device__ __forceinline__ float ck_sigmoid(float x) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}

// Eight pairs of row r from column c on; columns >= h read as zero.  ACT 0: halves, ACT 1: interleaved.
template <int ACT, bool VEC>
__device__ __forceinline__ void ck_load_pairs(const uint16_t* __restrict__ gu, int64_t r, int64_t c, int64_t h, float* g, float* u) {
    const uint16_t* p = gu + r * 2 * h + (ACT == 0 ? c : 2 * c);
    const uint16_t* q = ACT == 0 ? p + h : p + 8;
    uint32_t a[4] = {0, 0, 0, 0}, b[4] = {0, 0, 0, 0};
    if (c < h) {
        if (VEC) {
            const uint4 va = __ldcs(reinterpret_cast<const uint4*>(p)), vb = __ldcs(reinterpret_cast<const uint4*>(q));
            a[0] = va.x; a[1] = va.y; a[2] = va.z; a[3] = va.w;
            b[0] = vb.x; b[1] = vb.y; b[2] = vb.z; b[3] = vb.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // element j of the first and of the second group of eight
                const bool in_a = ACT == 0 ? c + j < h : c + (j >> 1) < h;
                const bool in_b = ACT == 0 ? c + j < h : c + 4 + (j >> 1) < h;
                if (in_a) a[j >> 1] |= (uint32_t)__ldg(p + j) << (16 * (j & 1));
                if (in_b) b[j >> 1] |= (uint32_t)__ldg(q + j) << (16 * (j & 1));
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float a0 = __uint_as_float(a[j] << 16), a1 = __uint_as_float(a[j] & 0xffff0000u);
        const float b0 = __uint_as_float(b[j] << 16), b1 = __uint_as_float(b[j] & 0xffff0000u);
        if (ACT == 0) {
            g[2 * j] = a0; g[2 * j + 1] = a1;
            u[2 * j] = b0; u[2 * j + 1] = b1;
        } else {
            g[j] = a0; u[j] = a1;
            g[4 + j] = b0; u[4 + j] = b1;
        }
    }
}

// codes of eight values and the block's step; eight lanes share the block
__device__ __forceinline__ uint2 ck_codes(const float* v, float* step) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);      // NaN compares above infinity
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float top = __uint_as_float(m);
    float inv = 0.f;
    *step = 0.f;
    if (!(top < 0x1p-100f)) {
        inv = __fdiv_rn(127.0f, top);
        *step = __fdiv_rn(top, 127.0f);
    }
    uint32_t b[8];
    // 1.5 * 2^23 + x leaves rint(x) in the low byte (two's complement)
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = __float_as_uint(__fmaf_rn(v[j], inv, 12582912.0f));
    const uint32_t lo = prmt(prmt(b[0], b[1], 0x0040u), prmt(b[2], b[3], 0x0040u), 0x5410u);
    const uint32_t hi = prmt(prmt(b[4], b[5], 0x0040u), prmt(b[6], b[7], 0x0040u), 0x5410u);
    return make_uint2(lo, hi);
}
__device__ __forceinline__ void ck_values(uint2 c, float step, float* v) {
    const uint32_t w[2] = {c.x ^ 0x80808080u, c.y ^ 0x80808080u};                     // code + 128
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t f = prmt(w[j >> 2], 0x4b000000u, 0x7440u | (uint32_t)(j & 3)); // 2^23 + code + 128
        v[j] = __fmul_rn(__uint_as_float(f) - 8388736.0f, step);
    }
}

template <int ACT>
__device__ __forceinline__ float ck_act(float g, float u) {
    if (ACT == 0) return g * ck_sigmoid(g) * u;
    const float gc = g > 7.0f ? 7.0f : g, uc = u > 7.0f ? 7.0f : u < -7.0f ? -7.0f : u;          // a NaN stays one
    return (uc + 1.0f) * gc * ck_sigmoid(1.702f * gc);
}

template <int ACT, bool VEC, bool KEEP>
__global__ void __launch_bounds__(kCkThreads)
glu_ckpt8_fwd_kernel(const uint16_t* __restrict__ gu, int64_t rows, int64_t h, const uint16_t* __restrict__ bias,
                     const int32_t* __restrict__ row_expert, int32_t E, uint16_t* __restrict__ out, uint2* __restrict__ codes,
                     float2* __restrict__ steps, int32_t* status) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t nb = (h + kCkBlock - 1) / kCkBlock;
    const int64_t i = (int64_t)blockIdx.x * kCkThreads + threadIdx.x;         // (row, block, eighth of the block)
    const int64_t rb = i >> 3;
    const int64_t r = rb / nb;
    const int64_t c = (rb - r * nb) * kCkBlock + (i & 7) * 8;
    const bool in = r < rows;
    float g[8], u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = u[j] = 0.f;
    if (in) {
        ck_load_pairs<ACT, VEC>(gu, r, c, h, g, u);
        if (ACT == 1 && bias) {
            const int32_t e = __ldg(row_expert + r);
            if (e >= 0 && e < E) {
                const uint16_t* b = bias + (int64_t)e * 2 * h + 2 * c;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j < h) {
                        g[j] += bf16_bits_to_float(__ldg(b + 2 * j));
                        u[j] += bf16_bits_to_float(__ldg(b + 2 * j + 1));
                    }
            } else if (status) {
                atomicOr(status, GNF4B_ST_BAD_EXPERT);
            }
        }
    }
    if (KEEP) {
        float sg, su;
        const uint2 cg = ck_codes(g, &sg), cu = ck_codes(u, &su);
        if (in) {
            codes[rb * 16 + (i & 7)] = cg;
            codes[rb * 16 + 8 + (i & 7)] = cu;
            if ((i & 7) == 0) steps[rb] = make_float2(sg, su);
        }
    }
    if (!in || c >= h) return;
    uint16_t* o = out + r * h + c;
    if (VEC) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w[j] = (uint32_t)f32_to_bf16_bits(ck_act<ACT>(g[2 * j], u[2 * j])) |
                   ((uint32_t)f32_to_bf16_bits(ck_act<ACT>(g[2 * j + 1], u[2 * j + 1])) << 16);
        *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < h) o[j] = f32_to_bf16_bits(ck_act<ACT>(g[j], u[j]));
    }
}

template <int ACT, bool VEC>
__global__ void __launch_bounds__(kCkThreads)
glu_ckpt8_bwd_kernel(const uint16_t* __restrict__ grad, const uint2* __restrict__ codes, const float2* __restrict__ steps,
                     int64_t rows, int64_t h, uint16_t* __restrict__ out) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t nb = (h + kCkBlock - 1) / kCkBlock;
    const int64_t i = (int64_t)blockIdx.x * kCkThreads + threadIdx.x;
    const int64_t rb = i >> 3;
    const int64_t r = rb / nb;
    const int64_t c = (rb - r * nb) * kCkBlock + (i & 7) * 8;
    if (r >= rows || c >= h) return;
    float go[8];
    const uint16_t* p = grad + r * h + c;
    if (VEC) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            go[2 * j] = __uint_as_float(w[j] << 16);
            go[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) go[j] = c + j < h ? bf16_bits_to_float(__ldg(p + j)) : 0.f;
    }
    const float2 st = __ldg(steps + rb);
    float g[8], u[8];
    ck_values(__ldcs(codes + rb * 16 + (i & 7)), st.x, g);
    ck_values(__ldcs(codes + rb * 16 + 8 + (i & 7)), st.y, u);
    uint32_t dg[8], du[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float a, b;
        if (ACT == 0) {
            const float s = ck_sigmoid(g[j]);
            a = go[j] * u[j] * s * (1.0f + g[j] * (1.0f - s));
            b = go[j] * g[j] * s;
        } else {
            const float gc = g[j] > 7.0f ? 7.0f : g[j], uc = u[j] > 7.0f ? 7.0f : u[j] < -7.0f ? -7.0f : u[j];
            const float s = ck_sigmoid(1.702f * gc);
            a = g[j] > 7.0f ? 0.f : go[j] * (uc + 1.0f) * s * (1.0f + 1.702f * gc * (1.0f - s));
            b = fabsf(u[j]) > 7.0f ? 0.f : go[j] * gc * s;
        }
        dg[j] = f32_to_bf16_bits(a);
        du[j] = f32_to_bf16_bits(b);
    }
    uint16_t* o = out + r * 2 * h + (ACT == 0 ? c : 2 * c);
    uint16_t* q = ACT == 0 ? o + h : o + 8;
    if (VEC) {
        if (ACT == 0) {
            __stcs(reinterpret_cast<uint4*>(o), make_uint4(dg[0] | (dg[1] << 16), dg[2] | (dg[3] << 16), dg[4] | (dg[5] << 16), dg[6] | (dg[7] << 16)));
            __stcs(reinterpret_cast<uint4*>(q), make_uint4(du[0] | (du[1] << 16), du[2] | (du[3] << 16), du[4] | (du[5] << 16), du[6] | (du[7] << 16)));
        } else {
            __stcs(reinterpret_cast<uint4*>(o), make_uint4(dg[0] | (du[0] << 16), dg[1] | (du[1] << 16), dg[2] | (du[2] << 16), dg[3] | (du[3] << 16)));
            __stcs(reinterpret_cast<uint4*>(q), make_uint4(dg[4] | (du[4] << 16), dg[5] | (du[5] << 16), dg[6] | (du[6] << 16), dg[7] | (du[7] << 16)));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < h) {
                o[ACT == 0 ? j : 2 * j] = (uint16_t)dg[j];
                (ACT == 0 ? q : o + 1)[ACT == 0 ? j : 2 * j] = (uint16_t)du[j];
            }
    }
}

}  // namespace gnf4b
