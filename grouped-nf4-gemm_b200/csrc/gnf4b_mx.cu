// C entry points of the MXFP4 quantiser and of the product of two MXFP4 operands (include/gnf4b.h).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "api_internal.h"
#include "common.cuh"
#include "mx_quant.cuh"
#include "w4a4_kernel.cuh"

using namespace gnf4b;

namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <int XT>
cudaError_t launch_quantize(const void* x, int64_t rows, int64_t K, int64_t stride, uint8_t* blocks, uint8_t* scales, cudaStream_t st) {
    const int64_t items = rows * (K / 8);
    const bool vec = aligned(x, 16) && (stride * (XT == 2 ? 4 : 2)) % 16 == 0;
    uint32_t* codes = reinterpret_cast<uint32_t*>(blocks);
    constexpr int U = XT == 2 ? 2 : 4;
    // one item per thread while that does not even fill the GPU: latency is all there is
    if (items <= 148 * 2048) {
        const unsigned grid = (unsigned)ceil_div(items, kMxThreads);
        return vec ? launch_pdl(mx_quantize_kernel<XT, true, 1>, grid, (unsigned)kMxThreads, st, x, items, K / 8, stride, codes, scales)
                   : launch_pdl(mx_quantize_kernel<XT, false, 1>, grid, (unsigned)kMxThreads, st, x, items, K / 8, stride, codes, scales);
    }
    const unsigned grid = (unsigned)ceil_div(items, kMxThreads * U);
    return vec ? launch_pdl(mx_quantize_kernel<XT, true, U>, grid, (unsigned)kMxThreads, st, x, items, K / 8, stride, codes, scales)
               : launch_pdl(mx_quantize_kernel<XT, false, U>, grid, (unsigned)kMxThreads, st, x, items, K / 8, stride, codes, scales);
}

constexpr int64_t kMaxItems = (int64_t)INT32_MAX * kMxThreads;      // grid limit of the one-item-per-thread kernels

}  // namespace

extern "C" {

int gnf4b_quantize_mxfp4(const void* x, int x_dtype, int64_t rows, int64_t K, int64_t x_stride, uint8_t* blocks, uint8_t* scales,
                         void* cuda_stream) {
    if (rows < 0 || x_dtype < GNF4B_X_BF16 || x_dtype > GNF4B_X_FP32) return GNF4B_EINVAL;
    if (K <= 0 || K % 32) return GNF4B_ESHAPE;
    if (rows == 0) return GNF4B_OK;
    if (!x || !blocks || !scales || !aligned(blocks, 4) || !aligned(x, x_dtype == GNF4B_X_FP32 ? 4 : 2) || x_stride < 0) return GNF4B_EINVAL;
    if (rows > kMaxItems / (K / 8)) return GNF4B_ETOOBIG;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
    const cudaError_t e = x_dtype == GNF4B_X_BF16 ? launch_quantize<0>(x, rows, K, x_stride, blocks, scales, st)
                          : x_dtype == GNF4B_X_FP16 ? launch_quantize<1>(x, rows, K, x_stride, blocks, scales, st)
                                                    : launch_quantize<2>(x, rows, K, x_stride, blocks, scales, st);
    return e == cudaSuccess ? GNF4B_OK : cuda_fail(e, "quantize_mxfp4 launch");
}

int gnf4b_dequantize_mxfp4(const uint8_t* blocks, const uint8_t* scales, int64_t n_blocks, int out_dtype, void* out, void* cuda_stream) {
    if (n_blocks < 0 || out_dtype < GNF4B_X_BF16 || out_dtype > GNF4B_X_FP32) return GNF4B_EINVAL;
    if (n_blocks == 0) return GNF4B_OK;
    if (!blocks || !scales || !out || !aligned(blocks, 4) || !aligned(out, 16)) return GNF4B_EINVAL;
    if (n_blocks > kMaxItems / 4) return GNF4B_ETOOBIG;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
    const int64_t items = n_blocks * 4;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(blocks);
    const bool few = items <= 148 * 2048;
    const unsigned grid = (unsigned)ceil_div(items, few ? kMxThreads : kMxThreads * 4);
#define GNF4B_DQ(T) (few ? launch_pdl(mx_dequantize_kernel<T, 1>, grid, (unsigned)kMxThreads, st, codes, scales, items, out) \
                         : launch_pdl(mx_dequantize_kernel<T, 4>, grid, (unsigned)kMxThreads, st, codes, scales, items, out))
    const cudaError_t e = out_dtype == GNF4B_X_BF16 ? GNF4B_DQ(0) : out_dtype == GNF4B_X_FP16 ? GNF4B_DQ(1) : GNF4B_DQ(2);
#undef GNF4B_DQ
    return e == cudaSuccess ? GNF4B_OK : cuda_fail(e, "dequantize_mxfp4 launch");
}

int gnf4b_glu_quantize_mxfp4(const void* gate_up, int64_t rows, int64_t h, int act, const void* bias, const int32_t* row_expert,
                             int32_t E, uint8_t* blocks, uint8_t* scales, int32_t* status_word, void* cuda_stream) {
    if (rows < 0 || (act != GNF4B_ACT_SILU_GLU && act != GNF4B_ACT_GPT_OSS_GLU)) return GNF4B_EINVAL;
    if (h <= 0 || h % 32) return GNF4B_ESHAPE;
    if (bias && (act != GNF4B_ACT_GPT_OSS_GLU || !row_expert || E <= 0)) return GNF4B_EINVAL;
    if (rows == 0) return GNF4B_OK;
    if (!gate_up || !blocks || !scales || !aligned(blocks, 4) || !aligned(gate_up, 2)) return GNF4B_EINVAL;
    if (rows > kMaxItems / (h / 8)) return GNF4B_ETOOBIG;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
    const int64_t items = rows * (h / 8);
    const unsigned grid = (unsigned)ceil_div(items, kMxThreads);
    const bool vec = aligned(gate_up, 16);                       // h % 32: every row and half row then starts on 16 bytes
    const uint16_t* gu = static_cast<const uint16_t*>(gate_up);
    const uint16_t* b = static_cast<const uint16_t*>(bias);
    uint32_t* codes = reinterpret_cast<uint32_t*>(blocks);
    cudaError_t e;
#define GNF4B_GLUQ(A, V) launch_pdl(mx_glu_quantize_kernel<A, V>, grid, (unsigned)kMxThreads, st, gu, items, h, b, row_expert, E, codes, scales, status_word)
    if (act == GNF4B_ACT_SILU_GLU) e = vec ? GNF4B_GLUQ(0, true) : GNF4B_GLUQ(0, false);
    else e = vec ? GNF4B_GLUQ(1, true) : GNF4B_GLUQ(1, false);
#undef GNF4B_GLUQ
    return e == cudaSuccess ? GNF4B_OK : cuda_fail(e, "glu_quantize_mxfp4 launch");
}

int gnf4b_w4a4_plan(int64_t T, int32_t G, int64_t N, int64_t K, int32_t max_rows, int32_t sm_count, int32_t smem_optin,
                    int32_t* plan) {
    if (T <= 0 || G <= 0 || sm_count <= 0 || smem_optin <= 0 || !plan) return GNF4B_EINVAL;
    if (N <= 0 || K <= 0 || K % 32) return GNF4B_ESHAPE;
    if (T > INT32_MAX - 256 || N > INT32_MAX - 256 || K > INT32_MAX) return GNF4B_ETOOBIG;
    const W4A4Plan p = w4a4_plan(T, G, N, K, max_rows, sm_count, smem_optin);
    if (p.stages < 2) return GNF4B_EUNSUPPORTED;
    const int32_t fields[GNF4B_W4A4_PLAN_FIELDS] = {p.pair, p.rows_w, p.tok_cap, p.xbox, p.x_bytes, p.x_blocks, p.stages, p.acc_bufs,
                                                    (int32_t)p.smem};
    std::copy(fields, fields + GNF4B_W4A4_PLAN_FIELDS, plan);
    return GNF4B_OK;
}

int gnf4b_gemm_grouped_w4a4(const uint8_t* x_blocks, const uint8_t* x_scales, int64_t T, const uint8_t* W, int64_t w_stride_e,
                            int64_t w_stride_n, const uint8_t* S, int64_t s_stride_e, int64_t s_stride_n, const int32_t* group_offsets,
                            const int32_t* expert_ids, int32_t G, int32_t E, int64_t N, int64_t K, int32_t max_rows, void* out,
                            int32_t* status_word, void* cuda_stream) {
    if (T < 0 || G < 0) return GNF4B_EINVAL;
    if (E <= 0 || N <= 0 || K <= 0 || K % 32) return GNF4B_ESHAPE;
    // row and column numbers, tiles included that reach beyond the end, are 32-bit coordinates of the loads
    if (T > INT32_MAX - 256 || N > INT32_MAX - 256 || K > INT32_MAX) return GNF4B_ETOOBIG;
    if (T == 0 || G == 0) return GNF4B_OK;
    if (!x_blocks || !x_scales || !W || !S || !group_offsets || !expert_ids || !out) return GNF4B_EINVAL;
    if (s_stride_e < 0 || s_stride_n < 0) return GNF4B_EINVAL;
    if (!aligned(out, 4)) return GNF4B_EINVAL;
    // TMA: 16-byte aligned bases and positive strides in multiples of 16 bytes (K / 2 is one: K is a multiple of 32); the
    // stride of a dimension of one is not used
    if (!aligned(x_blocks, 16) || !aligned(W, 16) || (N > 1 && (w_stride_n <= 0 || w_stride_n % 16)) ||
        (E > 1 && (w_stride_e <= 0 || w_stride_e % 16)))
        return GNF4B_EUNSUPPORTED;
    DevInfo di;
    const int rc = device_info(&di);
    if (rc) return rc;
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return GNF4B_EUNSUPPORTED;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
    const W4A4Plan p = w4a4_plan(T, G, N, K, max_rows, di.sm_count, di.smem_optin);
    if (p.stages < 2) return GNF4B_EUNSUPPORTED;
    // items are numbered in 31 bits (a group adds at most one chunk beyond its share)
    if ((ceil_div(T, 16) + G) * ceil_div(N, p.rows_w) > INT32_MAX) return GNF4B_ETOOBIG;
    W4A4Args a;
    a.xs = x_scales;
    a.ws = S;
    a.status = status_word;
    a.out = static_cast<uint16_t*>(out);
    a.ws_se = s_stride_e;
    a.ws_sn = s_stride_n;
    a.T = T;
    a.N = N;
    a.K = K;
    a.E = E;
    a.rows_w = p.rows_w;
    a.n_tiles = FastDiv::of((uint32_t)ceil_div(N, p.pair ? 256 : p.rows_w));
    a.k_stages = (int32_t)ceil_div(K, kQStageK);
    a.tok_cap = p.tok_cap;
    a.xbox = p.xbox;
    a.x_bytes = p.x_bytes;
    a.x_blocks = p.x_blocks;
    a.stages = p.stages;
    a.acc_bufs = p.acc_bufs;
    CUtensorMap x_map, w_map;
    const cuuint32_t ones[3] = {1, 1, 1};
    {
        const cuuint64_t dims[2] = {(cuuint64_t)(K / 2), (cuuint64_t)T};
        const cuuint64_t strides[1] = {(cuuint64_t)(K / 2)};
        const cuuint32_t box[2] = {(cuuint32_t)kQRowBytes, (cuuint32_t)p.xbox};
        if (enc(&x_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(x_blocks), dims, strides, box, ones,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return GNF4B_EUNSUPPORTED;
    }
    {
        const cuuint64_t dims[3] = {(cuuint64_t)(K / 2), (cuuint64_t)N, (cuuint64_t)E};
        const cuuint64_t sn = (cuuint64_t)(N > 1 ? w_stride_n : K / 2);
        const cuuint64_t strides[2] = {sn, (cuuint64_t)(E > 1 ? w_stride_e : (int64_t)sn * N)};
        const cuuint32_t box[3] = {(cuuint32_t)kQRowBytes, (cuuint32_t)p.rows_w, 1};
        if (enc(&w_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(W), dims, strides, box, ones,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return GNF4B_EUNSUPPORTED;
    }
    static int granted[64], granted_pair[64];
    cudaError_t e = p.pair ? ensure_smem(w4a4_kernel<2>, p.smem, granted_pair) : ensure_smem(w4a4_kernel<1>, p.smem, granted);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(w4a4)");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.pair ? di.sm_count & ~1 : di.sm_count));
    cfg.blockDim = dim3(kQThreads);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.pair ? 2 : 1;
    // a launch's group table lives in shared memory: longer lists take several launches (the offsets are absolute)
    for (int32_t g0 = 0; g0 < G; g0 += kQMaxGroups) {
        a.off = group_offsets + g0;
        a.eids = expert_ids + g0;
        a.G = std::min<int32_t>(kQMaxGroups, G - g0);
        e = p.pair ? cudaLaunchKernelEx(&cfg, w4a4_kernel<2>, a, x_map, w_map) : cudaLaunchKernelEx(&cfg, w4a4_kernel<1>, a, x_map, w_map);
        if (e != cudaSuccess) return cuda_fail(e, "w4a4 launch");
    }
    return GNF4B_OK;
}

}  // extern "C"
