// C entry points of the training operators: routing with its losses, the GLU with an 8-bit checkpoint (include/gnf4b.h).
#include <cuda_runtime.h>

#include <algorithm>

#include "api_internal.h"
#include "common.cuh"
#include "glu_ckpt8.cuh"
#include "router_train.cuh"

using namespace gnf4b;

namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int kRtWarps = 8;

// Warps of a forward CTA: as many as their registers let share an SM (a row of up to 512 experts: 16 per CTA)
constexpr int rt_fwd_warps(int ne) { return ne <= 16 ? 16 : 8; }
int rt_fwd_warps_of(int32_t E) { return rt_fwd_warps(E <= 512 ? 16 : 32); }

// CTAs of the forward pass: one while a warp then has few tokens, else up to two per SM
int rt_grid(int64_t T, int32_t E, int sm_count) {
    const int warps = rt_fwd_warps_of(E);
    if (T <= warps * 8) return 1;
    return (int)std::min<int64_t>(ceil_div(T, warps * 2), (int64_t)sm_count * 2);
}

size_t rt_scratch_bytes(int grid, int32_t E) { return grid == 1 ? 0 : rt_zeroed_bytes(E) + (size_t)grid * 8; }

// whole 16-byte vectors (or as many experts as a lane holds) from every row start on
bool rt_vec(const void* p, int64_t stride, int32_t E, int dtype) {
    const int size = dtype == GNF4B_X_FP32 ? 4 : 2;
    return aligned(p, 16) && (stride * size) % 16 == 0 && (E * size) % 16 == 0;
}

int rt_check(int dtype, int64_t T, int64_t stride, int32_t E, int32_t k, int32_t mode, int32_t norm) {
    if (dtype < GNF4B_X_BF16 || dtype > GNF4B_X_FP32 || T < 0 || mode < 0 || mode > 1 || norm < 0 || norm > 1) return GNF4B_EINVAL;
    if (E <= 0 || k <= 0 || k > E || stride < 0) return GNF4B_ESHAPE;
    if (E > kRtMaxExperts || k > kRtMaxK || T > INT32_MAX) return GNF4B_ETOOBIG;
    return GNF4B_OK;
}

template <int LT, int NE>
cudaError_t rt_fwd(const RouteTrainArgs& a, int grid, cudaStream_t st) {
    constexpr int W = rt_fwd_warps(NE);
    const size_t smem = (size_t)(W + 1) * a.E * 4;
    constexpr bool kTwo = NE > 1;                    // a row of up to 32 experts has one candidate a lane whatever k is
    const bool many = kTwo && a.k > kRtFewK;
    auto kfn = many ? route_train_fwd_kernel<LT, NE, W, kTwo> : route_train_fwd_kernel<LT, NE, W, false>;
    static int granted[2][64];
    cudaError_t e = ensure_smem(kfn, smem, granted[many]);
    if (e != cudaSuccess) return e;
    if (grid > 1) {
        e = cudaMemsetAsync(a.sum_p, 0, rt_zeroed_bytes(a.E), st);
        if (e != cudaSuccess) return e;
    }
    return launch_pdl_smem(kfn, (unsigned)grid, (unsigned)(W * 32), smem, st, a);
}
template <int LT, int NE>
cudaError_t rt_bwd(const RouteTrainBwdArgs& a, int grid, cudaStream_t st) {
    return launch_pdl(route_train_bwd_kernel<LT, NE, kRtWarps>, (unsigned)grid, (unsigned)(kRtWarps * 32), st, a);
}

template <typename F2, typename F4, typename F8, typename F16, typename F32, typename F1>
cudaError_t by_experts(int32_t E, F1 f1, F2 f2, F4 f4, F8 f8, F16 f16, F32 f32) {
    return E <= 32 ? f1() : E <= 64 ? f2() : E <= 128 ? f4() : E <= 256 ? f8() : E <= 512 ? f16() : f32();
}

}  // namespace

extern "C" {

size_t gnf4b_route_train_scratch_bytes(int64_t T, int32_t E) {
    DevInfo di;
    if (T <= 0 || E <= 0 || device_info(&di)) return 0;
    const int grid = rt_grid(T, E, di.sm_count);
    return rt_scratch_bytes(grid, E);
}

int gnf4b_route_train_fwd(const void* logits, int dtype, int64_t T, int64_t stride, int32_t E, int32_t k, int32_t mode, int32_t norm,
                          const uint8_t* token_mask, int64_t* idx, float* weights, float* lse, int32_t* counts, float* balance_loss,
                          float* z_loss, float* n_tokens, void* scratch, size_t scratch_bytes, void* cuda_stream) {
    int rc = rt_check(dtype, T, stride, E, k, mode, norm);
    if (rc) return rc;
    if (!counts || !balance_loss || !z_loss || !n_tokens || (T > 0 && (!logits || !idx || !weights || !lse))) return GNF4B_EINVAL;
    DevInfo di;
    rc = device_info(&di);
    if (rc) return rc;
    const int grid = rt_grid(T, E, di.sm_count);
    if (grid > 1 && (!scratch || !aligned(scratch, 8) || scratch_bytes < rt_scratch_bytes(grid, E))) return GNF4B_EWORKSPACE;
    RouteTrainArgs a;
    a.logits = logits; a.T = T; a.stride = stride; a.E = E; a.k = k; a.mode = mode; a.norm = norm;
    a.mask = token_mask; a.idx = idx; a.w = weights; a.lse = lse; a.counts = counts;
    a.balance = balance_loss; a.z = z_loss; a.n_tokens = n_tokens;
    a.sum_p = static_cast<unsigned long long*>(scratch);
    a.sum_c = reinterpret_cast<uint32_t*>(a.sum_p + E);
    a.arrived = a.sum_c + E;
    a.not_finite = a.arrived + 1;
    a.part_zn = reinterpret_cast<float*>(a.not_finite + 1);
    a.vec = rt_vec(logits, stride, E, dtype);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
#define GNF4B_RT(L) by_experts(E, [&] { return rt_fwd<L, 1>(a, grid, st); }, [&] { return rt_fwd<L, 2>(a, grid, st); }, \
        [&] { return rt_fwd<L, 4>(a, grid, st); }, [&] { return rt_fwd<L, 8>(a, grid, st); }, [&] { return rt_fwd<L, 16>(a, grid, st); }, \
        [&] { return rt_fwd<L, 32>(a, grid, st); })
    const cudaError_t e = dtype == GNF4B_X_BF16 ? GNF4B_RT(0) : dtype == GNF4B_X_FP16 ? GNF4B_RT(1) : GNF4B_RT(2);
#undef GNF4B_RT
    return e == cudaSuccess ? GNF4B_OK : cuda_fail(e, "route_train_fwd launch");
}

int gnf4b_route_train_bwd(const void* logits, int dtype, int64_t T, int64_t stride, int32_t E, int32_t k, int32_t mode, int32_t norm,
                          const uint8_t* token_mask, const int64_t* idx, const float* weights, const float* lse, const int32_t* counts,
                          const float* n_tokens, const float* g_weights, const float* g_balance, const float* g_z, void* grad,
                          void* cuda_stream) {
    int rc = rt_check(dtype, T, stride, E, k, mode, norm);
    if (rc) return rc;
    if (T == 0) return GNF4B_OK;
    if (!logits || !idx || !weights || !lse || !counts || !n_tokens || !grad) return GNF4B_EINVAL;
    DevInfo di;
    rc = device_info(&di);
    if (rc) return rc;
    RouteTrainBwdArgs a;
    a.logits = logits; a.T = T; a.stride = stride; a.E = E; a.k = k; a.mode = mode; a.norm = norm;
    a.mask = token_mask; a.idx = idx; a.w = weights; a.lse = lse; a.counts = counts; a.n_tokens = n_tokens;
    a.vec = rt_vec(logits, stride, E, dtype);
    a.vec_grad = rt_vec(grad, E, E, dtype);
    a.g_w = g_weights; a.g_balance = g_balance; a.g_z = g_z; a.grad = grad;
    const int grid = (int)std::min<int64_t>(ceil_div(T, kRtWarps), (int64_t)di.sm_count * 8);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
#define GNF4B_RT(L) by_experts(E, [&] { return rt_bwd<L, 1>(a, grid, st); }, [&] { return rt_bwd<L, 2>(a, grid, st); }, \
        [&] { return rt_bwd<L, 4>(a, grid, st); }, [&] { return rt_bwd<L, 8>(a, grid, st); }, [&] { return rt_bwd<L, 16>(a, grid, st); }, \
        [&] { return rt_bwd<L, 32>(a, grid, st); })
    const cudaError_t e = dtype == GNF4B_X_BF16 ? GNF4B_RT(0) : dtype == GNF4B_X_FP16 ? GNF4B_RT(1) : GNF4B_RT(2);
#undef GNF4B_RT
    return e == cudaSuccess ? GNF4B_OK : cuda_fail(e, "route_train_bwd launch");
}

int gnf4b_glu_ckpt8_fwd(const void* gate_up, int64_t rows, int64_t h, int act, const void* bias, const int32_t* row_expert, int32_t E,
                        void* out, int8_t* codes, float* steps, int32_t* status_word, void* cuda_stream) {
    if (rows < 0 || (act != GNF4B_ACT_SILU_GLU && act != GNF4B_ACT_GPT_OSS_GLU)) return GNF4B_EINVAL;
    if (h <= 0) return GNF4B_ESHAPE;
    if (bias && (act != GNF4B_ACT_GPT_OSS_GLU || !row_expert || E <= 0)) return GNF4B_EINVAL;
    if ((codes == nullptr) != (steps == nullptr)) return GNF4B_EINVAL;
    if (rows == 0) return GNF4B_OK;
    if (!gate_up || !out || !aligned(gate_up, 2) || !aligned(out, 2) || !aligned(codes, 8) || !aligned(steps, 8)) return GNF4B_EINVAL;
    const int64_t nb = ceil_div(h, kCkBlock);
    if (h > INT32_MAX / 4 || rows > INT32_MAX / nb) return GNF4B_ETOOBIG;       // block numbers of 31 bits
    const uint32_t blocks = (uint32_t)(rows * nb);
    const unsigned grid = (unsigned)ceil_div(blocks, kCkThreads / 8);
    const bool vec = h % 8 == 0 && aligned(gate_up, 16) && aligned(out, 16);
    const bool keep = codes != nullptr;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
    cudaError_t e;
#define GNF4B_CK(A, V, K, B) launch_pdl(glu_ckpt8_fwd_kernel<A, V, K, B>, grid, (unsigned)kCkThreads, st, static_cast<const uint16_t*>(gate_up), \
        blocks, FastDiv::of((uint32_t)nb), (int)h, static_cast<const uint16_t*>(bias), row_expert, E, static_cast<uint16_t*>(out), \
        reinterpret_cast<uint2*>(codes), reinterpret_cast<float2*>(steps), status_word)
    if (act == GNF4B_ACT_SILU_GLU)
        e = keep ? (vec ? GNF4B_CK(0, true, true, false) : GNF4B_CK(0, false, true, false))
                 : (vec ? GNF4B_CK(0, true, false, false) : GNF4B_CK(0, false, false, false));
    else if (bias)
        e = keep ? (vec ? GNF4B_CK(1, true, true, true) : GNF4B_CK(1, false, true, true))
                 : (vec ? GNF4B_CK(1, true, false, true) : GNF4B_CK(1, false, false, true));
    else
        e = keep ? (vec ? GNF4B_CK(1, true, true, false) : GNF4B_CK(1, false, true, false))
                 : (vec ? GNF4B_CK(1, true, false, false) : GNF4B_CK(1, false, false, false));
#undef GNF4B_CK
    return e == cudaSuccess ? GNF4B_OK : cuda_fail(e, "glu_ckpt8_fwd launch");
}

int gnf4b_glu_ckpt8_bwd(const void* grad_out, const int8_t* codes, const float* steps, int64_t rows, int64_t h, int act,
                        void* grad_gate_up, void* cuda_stream) {
    if (rows < 0 || (act != GNF4B_ACT_SILU_GLU && act != GNF4B_ACT_GPT_OSS_GLU)) return GNF4B_EINVAL;
    if (h <= 0) return GNF4B_ESHAPE;
    if (rows == 0) return GNF4B_OK;
    if (!grad_out || !codes || !steps || !grad_gate_up || !aligned(grad_out, 2) || !aligned(grad_gate_up, 2) || !aligned(codes, 8) ||
        !aligned(steps, 8))
        return GNF4B_EINVAL;
    const int64_t nb = ceil_div(h, kCkBlock);
    if (h > INT32_MAX / 4 || rows > INT32_MAX / nb) return GNF4B_ETOOBIG;
    const uint32_t blocks = (uint32_t)(rows * nb);
    const unsigned grid = (unsigned)ceil_div(blocks, kCkThreads / 8);
    const bool vec = h % 8 == 0 && aligned(grad_out, 16) && aligned(grad_gate_up, 16);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
    cudaError_t e;
#define GNF4B_CK(A, V) launch_pdl(glu_ckpt8_bwd_kernel<A, V>, grid, (unsigned)kCkThreads, st, static_cast<const uint16_t*>(grad_out), \
        reinterpret_cast<const uint2*>(codes), reinterpret_cast<const float2*>(steps), blocks, FastDiv::of((uint32_t)nb), (int)h, \
        static_cast<uint16_t*>(grad_gate_up))
    if (act == GNF4B_ACT_SILU_GLU) e = vec ? GNF4B_CK(0, true) : GNF4B_CK(0, false);
    else e = vec ? GNF4B_CK(1, true) : GNF4B_CK(1, false);
#undef GNF4B_CK
    return e == cudaSuccess ? GNF4B_OK : cuda_fail(e, "glu_ckpt8_bwd launch");
}

}  // extern "C"
