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
// The product v * (127 / max|v|) is taken exactly before it is rounded to a whole number.  Where a value lies half way
// between two codes (half of the block's maximum is 63.5 steps) the rounding of 127 / max decides, so that another way to
// write the same formula may take the other of the two, which is as near.
//
// A step of the block's maximum / 127 costs at most half a step, 0.4 % of the block's largest magnitude, and halves what
// a layer keeps between the passes (2 bytes + 1/8 instead of 4 per pair).  A block whose maximum is below 2^-100 is kept
// as zeros (127 / max would leave the fp32 range); one with an infinity or a NaN restores to non-finite values.
//
// Both passes want to be bound by memory (4 + 2 + 2 bytes a pair each), and at 8 bytes a pair the instructions are just as
// scarce: eight pairs per thread, eight neighbouring lanes per block, 16-byte loads and stores, codes of a block side by
// side ([row][block][gate 64 | up 64], so any h is aligned).  The maxima of gate and up travel through the shuffles as
// one word of two bf16 magnitudes; of the four divisions a block needs, even lanes make the gate's and odd ones the
// up's; row and column come from a multiplication; the sigmoid is ex2.approx and rcp.approx: two to three units in the
// last fp32 place, far below the bf16 rounding behind it.  Measured at 32768 x 2880 (gpt-oss form, 755 MB each way):
// forward 125 us, 6.0 TB/s, backward 130 us, 5.8 TB/s (158 and 165 us before the index, the maxima and the
// divisions were made cheaper); forward with a bias, loaded two bytes at a time, 252 us.
#pragma once

#include "common.cuh"

namespace gnf4b {

constexpr int kCkBlock = 64;
constexpr int kCkThreads = 256;

// 1 / (1 + 2^x)
__device__ __forceinline__ float ck_sigmoid2(float x) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}
__device__ __forceinline__ uint32_t ck_pack(float lo, float hi) {     // bf16 pair
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
constexpr float kCkLog2e = 1.4426950408889634f;
constexpr float kCkAlpha = 1.702f;

// Where this thread works: block rb (row r, columns c ..), eighth of the block
struct CkPlace {
    uint32_t rb;
    int64_t r;
    int c, sub;
};
__device__ __forceinline__ CkPlace ck_place(const FastDiv& nb) {
    CkPlace p;
    p.rb = blockIdx.x * (kCkThreads / 8) + (threadIdx.x >> 3);
    p.sub = threadIdx.x & 7;
    const uint32_t r = nb.div(p.rb);
    p.r = r;
    p.c = (int)(p.rb - r * nb.d) * kCkBlock + p.sub * 8;
    return p;
}

// Words of eight pairs of row r from column c on; what lies behind column h is zero.
//   ACT 0 (halves): a = 8 gates, b = 8 ups;  ACT 1 (interleaved): a, b = four pairs each, gate in the low half
template <int ACT, bool VEC>
__device__ __forceinline__ void ck_load_pairs(const uint16_t* __restrict__ gu, const CkPlace& at, int h, uint32_t* a, uint32_t* b) {
    const uint16_t* p = gu + at.r * 2 * h + (ACT == 0 ? at.c : 2 * at.c);
    const uint16_t* q = ACT == 0 ? p + h : p + 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = b[j] = 0;
    if (VEC) {
        const uint4 va = __ldcs(reinterpret_cast<const uint4*>(p)), vb = __ldcs(reinterpret_cast<const uint4*>(q));
        a[0] = va.x; a[1] = va.y; a[2] = va.z; a[3] = va.w;
        b[0] = vb.x; b[1] = vb.y; b[2] = vb.z; b[3] = vb.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool in_a = ACT == 0 ? at.c + j < h : at.c + (j >> 1) < h;
            const bool in_b = ACT == 0 ? at.c + j < h : at.c + 4 + (j >> 1) < h;
            if (in_a) a[j >> 1] |= (uint32_t)__ldg(p + j) << (16 * (j & 1));
            if (in_b) b[j >> 1] |= (uint32_t)__ldg(q + j) << (16 * (j & 1));
        }
    }
}
template <int ACT>
__device__ __forceinline__ void ck_unpack(const uint32_t* a, const uint32_t* b, float* g, float* u) {
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

// Largest magnitudes of the block's gates and ups as fp32 bits (integer order: a NaN is above infinity); eight lanes share
// the block.  Without a bias the values are bf16 and both maxima fit one word.
template <int ACT>
__device__ __forceinline__ void ck_tops_bf16(const uint32_t* a, const uint32_t* b, uint32_t* top_g, uint32_t* top_u) {
    constexpr uint32_t k = 0x7fff7fffu;
    uint32_t ma = __vmaxu2(__vmaxu2(a[0] & k, a[1] & k), __vmaxu2(a[2] & k, a[3] & k));
    const uint32_t mb = __vmaxu2(__vmaxu2(b[0] & k, b[1] & k), __vmaxu2(b[2] & k, b[3] & k));
    uint32_t m;                                       // up's maximum above, gate's below
    if (ACT == 0) m = max(ma & 0xffffu, ma >> 16) | (max(mb & 0xffffu, mb >> 16) << 16);
    else m = __vmaxu2(ma, mb);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    *top_g = m << 16;
    *top_u = m & 0xffff0000u;
}
__device__ __forceinline__ uint32_t ck_top_f32(const float* v) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}
__device__ __forceinline__ uint2 ck_codes(const float* v, float inv) {
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
    if (ACT == 0) return g * ck_sigmoid2(g * -kCkLog2e) * u;
    const float gc = min_nan(g, 7.0f), uc = max_nan(min_nan(u, 7.0f), -7.0f);
    return (uc + 1.0f) * (gc * ck_sigmoid2(gc * (-kCkAlpha * kCkLog2e)));
}

template <int ACT, bool VEC, bool KEEP, bool BIAS>
__global__ void __launch_bounds__(kCkThreads)
glu_ckpt8_fwd_kernel(const uint16_t* __restrict__ gu, uint32_t blocks, FastDiv nb, int h, const uint16_t* __restrict__ bias,
                     const int32_t* __restrict__ row_expert, int32_t E, uint16_t* __restrict__ out, uint2* __restrict__ codes,
                     float2* __restrict__ steps, int32_t* status) {
    pdl_wait();
    pdl_launch_dependents();
    const CkPlace at = ck_place(nb);
    const bool in = at.rb < blocks, some = in && at.c < h;
    uint32_t a[4] = {0, 0, 0, 0}, b[4] = {0, 0, 0, 0};
    if (some) ck_load_pairs<ACT, VEC>(gu, at, h, a, b);
    float g[8], u[8];
    ck_unpack<ACT>(a, b, g, u);
    if (BIAS && some) {
        const int32_t e = __ldg(row_expert + at.r);
        if (e >= 0 && e < E) {
            const uint16_t* p = bias + ((int64_t)e * h + at.c) * 2;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (at.c + j < h) {
                    g[j] += bf16_bits_to_float(__ldg(p + 2 * j));
                    u[j] += bf16_bits_to_float(__ldg(p + 2 * j + 1));
                }
        } else if (status) {
            atomicOr(status, GNF4B_ST_BAD_EXPERT);
        }
    }
    if (KEEP) {
        uint32_t tg, tu;
        if (BIAS) {
            tg = ck_top_f32(g);
            tu = ck_top_f32(u);
        } else {
            ck_tops_bf16<ACT>(a, b, &tg, &tu);
        }
        // even lanes divide for the gates, odd ones for the ups
        const bool odd = threadIdx.x & 1;
        const float top = __uint_as_float(odd ? tu : tg);
        const bool held = !(top < 0x1p-100f);
        const float inv = held ? __fdiv_rn(127.0f, top) : 0.f, step = held ? __fdiv_rn(top, 127.0f) : 0.f;
        const float inv_o = __shfl_xor_sync(0xffffffffu, inv, 1), step_o = __shfl_xor_sync(0xffffffffu, step, 1);
        const uint2 cg = ck_codes(g, odd ? inv_o : inv), cu = ck_codes(u, odd ? inv : inv_o);
        if (in) {
            uint2* p = codes + (int64_t)at.rb * 16 + at.sub;
            p[0] = cg;
            p[8] = cu;
            if (at.sub == 0) steps[at.rb] = make_float2(step, step_o);
        }
    }
    if (!some) return;
    uint16_t* o = out + at.r * h + at.c;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = ck_pack(ck_act<ACT>(g[2 * j], u[2 * j]), ck_act<ACT>(g[2 * j + 1], u[2 * j + 1]));
    if (VEC) {
        *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (at.c + j < h) o[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
}

template <int ACT, bool VEC>
__global__ void __launch_bounds__(kCkThreads)
glu_ckpt8_bwd_kernel(const uint16_t* __restrict__ grad, const uint2* __restrict__ codes, const float2* __restrict__ steps,
                     uint32_t blocks, FastDiv nb, int h, uint16_t* __restrict__ out) {
    pdl_wait();
    pdl_launch_dependents();
    const CkPlace at = ck_place(nb);
    if (at.rb >= blocks || at.c >= h) return;
    float go[8];
    const uint16_t* p = grad + at.r * h + at.c;
    const uint2 cg = __ldcs(codes + (int64_t)at.rb * 16 + at.sub), cu = __ldcs(codes + (int64_t)at.rb * 16 + 8 + at.sub);
    const float2 st = __ldg(steps + at.rb);
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
        for (int j = 0; j < 8; ++j) go[j] = at.c + j < h ? bf16_bits_to_float(__ldg(p + j)) : 0.f;
    }
    float g[8], u[8];
    ck_values(cg, st.x, g);
    ck_values(cu, st.y, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (ACT == 0) {
            const float s = ck_sigmoid2(g[j] * -kCkLog2e), gs = go[j] * s;
            const float dg = gs * u[j] * fmaf(g[j], 1.0f - s, 1.0f);
            u[j] = gs * g[j];
            g[j] = dg;
        } else {
            const float gc = min_nan(g[j], 7.0f), uc = max_nan(min_nan(u[j], 7.0f), -7.0f);
            const float s = ck_sigmoid2(gc * (-kCkAlpha * kCkLog2e)), gs = go[j] * s;
            const float dg = gs * (uc + 1.0f) * fmaf(kCkAlpha * gc, 1.0f - s, 1.0f);
            u[j] = fabsf(u[j]) > 7.0f ? 0.f : gs * gc;      // beyond a clamp: no gradient (a NaN is not beyond)
            g[j] = g[j] > 7.0f ? 0.f : dg;
        }
    }
    uint16_t* o = out + at.r * 2 * h + (ACT == 0 ? at.c : 2 * at.c);
    uint16_t* q = ACT == 0 ? o + h : o + 8;
    uint32_t wo[4], wq[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        wo[j] = ACT == 0 ? ck_pack(g[2 * j], g[2 * j + 1]) : ck_pack(g[j], u[j]);
        wq[j] = ACT == 0 ? ck_pack(u[2 * j], u[2 * j + 1]) : ck_pack(g[4 + j], u[4 + j]);
    }
    if (VEC) {
        __stcs(reinterpret_cast<uint4*>(o), make_uint4(wo[0], wo[1], wo[2], wo[3]));
        __stcs(reinterpret_cast<uint4*>(q), make_uint4(wq[0], wq[1], wq[2], wq[3]));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool in_o = ACT == 0 ? at.c + j < h : at.c + (j >> 1) < h;
            const bool in_q = ACT == 0 ? at.c + j < h : at.c + 4 + (j >> 1) < h;
            if (in_o) o[j] = (uint16_t)(wo[j >> 1] >> (16 * (j & 1)));
            if (in_q) q[j] = (uint16_t)(wq[j >> 1] >> (16 * (j & 1)));
        }
    }
}

}  // namespace gnf4b
