// MXFP4 on the way in and out: rows of bf16 / fp16 / fp32 -> packed e2m1 elements and one e8m0 exponent per 32, the
// reverse, and the GLU between an expert's two products with its result packed at once.
//
//   e    = the least integer >= -69 with max|x| <= 6 * 2^e over the block; exponent byte e + 127
//   code = the e2m1 value nearest to x / 2^e, the one of lower magnitude on a tie, +0 for everything that rounds to 0
//
// the rule of quantize_pack_mxfp4 in mxfp4_pack_ref.py (its floor of 1e-20 under the block's maximum gives the -69),
// byte for byte.  A block with an infinity or a NaN has no such exponent: its byte is 255 and every code +-6, so that
// neither reading of the byte 255 (NaN, or 2^128) turns it into finite numbers.
//
// All three are bound by memory: four neighbouring lanes share a block, eight elements each, so loads are 16 bytes and
// code stores 4 bytes a lane, both contiguous over the warp; the block maximum takes two shuffles.  Measured at 32768 x
// 2880 bf16: quantise 45 us (5.3 TB/s; one, two and four items in flight per thread: 52, 47, 45), dequantise 38 us
// (6.4 TB/s; one item per thread: 54); both in turn 72 us, 6.6 TB/s, as fast as a copy.  8192 x 7168 fp32: 38 and 41 us, 7.0 and
// 6.4 TB/s.  The GLU with its result packed is bound by instructions (one item a thread, a 64-bit division, the exact
// exponential and division of the activation): 32768 x 2880 136 us (SiLU), 237 (gpt-oss), 243 with bias; its bytes are 65.
#pragma once

#include "common.cuh"

namespace gnf4b {

constexpr int kMxThreads = 256;

// e2m1 codes of eight numbers already divided by the block scale, element 0 in the low nibble.  cvt.rn rounds ties to
// the even code; the callers hand in magnitudes shrunk by less than the distance of any two of their values, which
// puts exact ties below the tie and moves nothing else across one.
__device__ __forceinline__ uint32_t e2m1_codes(const float* v) {
    uint32_t w;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(w)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    const uint32_t mag = w & 0x77777777u;
    const uint32_t nonzero = (mag | (mag >> 1) | (mag >> 2)) & 0x11111111u;
    return mag | (w & (nonzero << 3));                // a negative number that rounds to zero is +0
}

// exponent e of a block whose largest magnitude is `top` (finite)
__device__ __forceinline__ int mx_exponent(float top) {
    const uint32_t b = __float_as_uint(fmaxf(top, 1e-20f));
    return (int)(b >> 23) - 127 - 2 + ((b & 0x7fffffu) > 0x400000u ? 1 : 0);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }      // -126 <= e <= 127

// Codes and exponent byte for this lane's eight numbers, given as sign-magnitude words: `top_bits` the block's largest
// magnitude as fp32 bits, `shrink` the factor that breaks ties (see e2m1_codes).
__device__ __forceinline__ uint32_t mx_pack8(float* f, uint32_t top_bits, float shrink, uint32_t* exp_byte) {
    if (top_bits >= 0x7f800000u) {
        *exp_byte = 255;
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) w |= (7u | (__float_as_uint(f[j]) >> 31 << 3)) << (4 * j);
        return w;
    }
    const int e = mx_exponent(__uint_as_float(top_bits));
    *exp_byte = (uint32_t)(e + 127);
    const float s = __fmul_rn(pow2f(-e), shrink);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __fmul_rn(f[j], s);
    return e2m1_codes(f);
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }

// Eight 16-bit floats in four words -> codes.  Magnitudes compare as integers (NaN above infinity).
// shrink: 1 - 2^-12 (bf16, 8 significant bits: product of 20 bits is exact) or 1 - 2^-13 (fp16: 24 bits, exact).
template <bool FP16>
__device__ __forceinline__ uint32_t mx_quant16(const uint32_t* w, uint32_t* exp_byte) {
    uint32_t m = max_u16x2(max_u16x2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), max_u16x2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
    m = max_u16x2(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max_u16x2(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const uint32_t top16 = max(m & 0xffffu, m >> 16);
    float f[8];
    uint32_t top;
    if (FP16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 p = __half22float2(*reinterpret_cast<const __half2*>(w + j));
            f[2 * j] = p.x;
            f[2 * j + 1] = p.y;
        }
        top = __float_as_uint(__half2float(__ushort_as_half((unsigned short)top16)));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[2 * j] = __uint_as_float(w[j] << 16);
            f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
        top = top16 << 16;
    }
    return mx_pack8(f, top, FP16 ? 1.0f - 0x1p-13f : 1.0f - 0x1p-12f, exp_byte);
}

// fp32 has too many bits for one factor: the low 12 are first gathered into one sticky bit, which keeps every number on
// its side of every tie (ties have at most two significant bits), and the rest is treated like a 13-bit number.
__device__ __forceinline__ uint32_t mx_quant32(const uint32_t* w, uint32_t* exp_byte) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, w[j] & 0x7fffffffu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __uint_as_float((w[j] & 0xfffff000u) | ((w[j] & 0xfffu) ? 0x800u : 0u));
    return mx_pack8(f, m, 1.0f - 0x1p-14f, exp_byte);
}

// x: rows of K elements, `stride` elements apart (XT: 0 bf16, 1 fp16, 2 fp32).  VEC: rows start on 16 bytes.
// Item i = eight elements; items of one block sit in four neighbouring lanes (K is a multiple of 32 and so is the
// number of items per warp).  U items per thread are in flight.
template <int XT, bool VEC, int U>
__global__ void __launch_bounds__(kMxThreads)
mx_quantize_kernel(const void* __restrict__ x, int64_t items, int64_t per_row, int64_t stride, uint32_t* __restrict__ codes,
                   uint8_t* __restrict__ scales) {
    constexpr int kWords = XT == 2 ? 8 : 4;
    pdl_wait();
    pdl_launch_dependents();
    const int64_t first = (int64_t)blockIdx.x * (kMxThreads * U) + threadIdx.x;
    uint32_t w[U][kWords];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = first + u * kMxThreads;
#pragma unroll
        for (int j = 0; j < kWords; ++j) w[u][j] = 0;
        if (i >= items) continue;
        int64_t at = i * 8;
        if (stride != per_row * 8) {
            const int64_t r = i / per_row;
            at = r * stride + (i - r * per_row) * 8;
        }
        if (VEC) {
            const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x) + at * (XT == 2 ? 4 : 2));
#pragma unroll
            for (int v = 0; v < kWords / 4; ++v) {
                const uint4 q = __ldcs(p + v);
                w[u][4 * v] = q.x; w[u][4 * v + 1] = q.y; w[u][4 * v + 2] = q.z; w[u][4 * v + 3] = q.w;
            }
        } else if (XT == 2) {
#pragma unroll
            for (int j = 0; j < kWords; ++j) w[u][j] = __ldg(static_cast<const uint32_t*>(x) + at + j);
        } else {
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                const unsigned short* p = static_cast<const unsigned short*>(x) + at + 2 * j;
                w[u][j] = (uint32_t)__ldg(p) | ((uint32_t)__ldg(p + 1) << 16);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = first + u * kMxThreads;
        uint32_t eb;
        const uint32_t c = XT == 2 ? mx_quant32(w[u], &eb) : mx_quant16<XT == 1>(w[u], &eb);
        if (i < items) {
            codes[i] = c;
            if ((i & 3) == 0) scales[i >> 2] = (uint8_t)eb;
        }
    }
}

__device__ __forceinline__ float2 e2m1x2_to_float2(uint32_t byte) {
    uint32_t h;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;\n\t}" : "=r"(h) : "r"(byte));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// items of eight elements -> OT (0 bf16, 1 fp16, 2 fp32), contiguous.  Exact in bf16 and fp32; the exponent byte 255
// reads as 2^128 (a zero stays zero), as everywhere in this library but in the product of two MXFP4 operands.
template <int OT, int U>
__global__ void __launch_bounds__(kMxThreads)
mx_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t items, void* __restrict__ out) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t first = (int64_t)blockIdx.x * (kMxThreads * U) + threadIdx.x;
    uint32_t c[U];
    float sc[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const int64_t i = first + k * kMxThreads;
        c[k] = i < items ? __ldcs(codes + i) : 0u;
        sc[k] = i < items ? load_scale<GNF4B_S_E8M0>(scales, i >> 2) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const int64_t i = first + k * kMxThreads;
        if (OT != 2 && i >= items) break;
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 p = e2m1x2_to_float2((c[k] >> (8 * j)) & 0xffu);
            f[2 * j] = __fmul_rn(p.x + p.x, sc[k]);
            f[2 * j + 1] = __fmul_rn(p.y + p.y, sc[k]);
        }
        if (OT == 2) {
            // two lanes hold 16 numbers and store one lane's eight after the other's, so that a store writes whole
            // 32-byte sectors (1237 x 7168: 11.8 us with half sectors)
            const bool odd = threadIdx.x & 1;
            float g[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) g[j] = __shfl_xor_sync(0xffffffffu, odd ? f[j] : f[4 + j], 1);
            if (i < items) {                          // items come in fours: both lanes or none
                float4* o = static_cast<float4*>(out) + 2 * (i - odd) + odd;
                __stcs(o, odd ? make_float4(g[0], g[1], g[2], g[3]) : make_float4(f[0], f[1], f[2], f[3]));
                __stcs(o + 2, odd ? make_float4(f[4], f[5], f[6], f[7]) : make_float4(g[0], g[1], g[2], g[3]));
            }
        } else {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (OT == 0) {
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[j]) : "f"(f[2 * j + 1]), "f"(f[2 * j]));
                } else {
                    const __half2 h = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
                    w[j] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
            __stcs(static_cast<uint4*>(out) + i, make_uint4(w[0], w[1], w[2], w[3]));
        }
    }
}

// gate_up [rows, 2h] bf16 -> MXFP4 rows of the GLU's bf16 result, h a multiple of 32: the bits of gnf4b_silu_glu
// (ACT 0) or gnf4b_glu_gpt_oss (ACT 1, optional bias bf16 [E, 2h] by row_expert) followed by the quantiser, without
// the pass over the result in memory.  A row whose expert id is outside [0, E) gets no bias and raises
// GNF4B_ST_BAD_EXPERT.
template <int ACT, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
mx_glu_quantize_kernel(const uint16_t* __restrict__ gu, int64_t items, int64_t h, const uint16_t* __restrict__ bias,
                       const int32_t* __restrict__ row_expert, int32_t E, uint32_t* __restrict__ codes,
                       uint8_t* __restrict__ scales, int32_t* status) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t i = (int64_t)blockIdx.x * kMxThreads + threadIdx.x;
    uint32_t w[4] = {0, 0, 0, 0};
    if (i < items) {
        const int64_t per_row = h / 8;
        const int64_t r = i / per_row, c = (i - r * per_row) * 8;
        uint32_t a[4], b[4];                   // ACT 0: gate and up words; ACT 1: eight interleaved pairs
        const uint16_t* p = gu + r * 2 * h + (ACT == 0 ? c : 2 * c);
        const uint16_t* q = ACT == 0 ? p + h : p + 8;
        if (VEC) {
            const uint4 va = __ldg(reinterpret_cast<const uint4*>(p)), vb = __ldg(reinterpret_cast<const uint4*>(q));
            a[0] = va.x; a[1] = va.y; a[2] = va.z; a[3] = va.w;
            b[0] = vb.x; b[1] = vb.y; b[2] = vb.z; b[3] = vb.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a[j] = (uint32_t)__ldg(p + 2 * j) | ((uint32_t)__ldg(p + 2 * j + 1) << 16);
                b[j] = (uint32_t)__ldg(q + 2 * j) | ((uint32_t)__ldg(q + 2 * j + 1) << 16);
            }
        }
        if (ACT == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float g0 = __uint_as_float(a[j] << 16), g1 = __uint_as_float(a[j] & 0xffff0000u);
                const float u0 = __uint_as_float(b[j] << 16), u1 = __uint_as_float(b[j] & 0xffff0000u);
                w[j] = (uint32_t)f32_to_bf16_bits(__fmul_rn(silu_f32(g0), u0)) |
                       ((uint32_t)f32_to_bf16_bits(__fmul_rn(silu_f32(g1), u1)) << 16);
            }
        } else {
            const uint16_t* brow = nullptr;
            if (bias) {
                const int32_t e = __ldg(row_expert + r);
                if (e >= 0 && e < E) brow = bias + (int64_t)e * 2 * h + 2 * c;
                else if (status) atomicOr(status, GNF4B_ST_BAD_EXPERT);
            }
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t pair = j < 4 ? a[j] : b[j - 4];
                float g = __uint_as_float(pair << 16), u = __uint_as_float(pair & 0xffff0000u);
                if (brow) {
                    g = bf16_round(__fadd_rn(g, bf16_bits_to_float(__ldg(brow + 2 * j))));
                    u = bf16_round(__fadd_rn(u, bf16_bits_to_float(__ldg(brow + 2 * j + 1))));
                }
                o[j] = glu_gpt_oss(g, u);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = (uint32_t)f32_to_bf16_bits(o[2 * j]) | ((uint32_t)f32_to_bf16_bits(o[2 * j + 1]) << 16);
        }
    }
    uint32_t eb;
    const uint32_t code = mx_quant16<false>(w, &eb);
    if (i < items) {
        codes[i] = code;
        if ((i & 3) == 0) scales[i >> 2] = (uint8_t)eb;
    }
}

}  // namespace gnf4b
