// State and device helpers of the token operators (token_fc, token_norm, token_gate, log_probs).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "token_check.h"

namespace enn_b200 {

struct NormParams {
    int32_t c;
    int32_t norm, post_norm;
    int32_t gate_tokens;
    float eps, post_eps, residual_scale;
    const float *weight, *bias, *post_weight, *post_bias;      // null: ones / zeros; each four times, copy i at i * stride + i
    int32_t stride;
    int64_t pitch;                                              // bytes from row to row of byte rows
};

struct GateParams {
    int32_t c, act;
    int64_t in_stride;      // elements from row to row of the gates and of the values
    int64_t pitch;
};

struct LogProbsParams {
    int32_t vocab, given, top;
    float scale;
    int64_t pitch;          // logits from row to row
};

struct TokenFcDirect {      // what the general kernel takes
    int32_t k, n;
    int64_t in_pitch, w_pitch;
    const int8_t *w;
    const float *channel_scale, *bias;
};
struct TokenFcParams {
    int32_t k, n;
    int64_t in_pitch, w_pitch;
    const int8_t *w;        // [n][w_pitch], zero beyond k
    const float *channel_scale, *bias;
    CUtensorMap map_w;
    int32_t *err_host, *err_dev;      // pinned word in which a kernel that gave up on a wait leaves a code
    bool starve_next;                 // the next call is a self-test of that
    bool gave_up() const { return err_host && *static_cast<volatile const int32_t *>(err_host) != 0; }
    TokenFcDirect direct() const { return {k, n, in_pitch, w_pitch, w, channel_scale, bias}; }
};

// Everything a prepared token operator holds; deleted by the operator's release.
struct TokenState {
    TokenCall call;
    int32_t in_dtype = 0, out_dtype = 0;
    int32_t sms = 0;        // what launches are sized for (option grid_cap when the operator was prepared, else all): the persistent kernels,
                            // pairs of token_fc, norms and log_probs of many rows, keep to as many CTAs as they hold; the others have a CTA per tile
    bool residual = false, packed = false;
    NormParams norm{};
    GateParams gate{};
    LogProbsParams log_probs{};
    TokenFcParams fc{};
};

// The launch for `rows` > 0 rows on the context's stream; pointers in the descriptor's order.
cudaError_t token_norm_launch(const enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs);
cudaError_t token_gate_launch(const enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs);
cudaError_t log_probs_launch(const enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs);
cudaError_t token_fc_launch(enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs);
cudaError_t token_fc_plan(enn_b200_op *op);
cudaError_t launch_pad_rows(const void *src, int32_t width, int32_t height, int64_t pitch, void *dst, cudaStream_t stream);

#ifdef __CUDACC__
namespace {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Rounded once, to nearest even.
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Scale of a quantised row and what its values are multiplied with, from the bits of the largest magnitude.  Magnitudes compare as
// integers, with infinities above all numbers and NaN above those: a maximum over the bits does not lose a NaN as fmaxf does.
struct RowScale {
    float scale, inv;
};
__device__ __forceinline__ RowScale row_scale(uint32_t largest_bits) {
    const float largest = __uint_as_float(largest_bits);
    RowScale r;
    if (largest_bits >= 0x7f800000u) {               // a NaN or an infinity in the row
        r.scale = __uint_as_float(0x7fffffffu);
        r.inv = 0.f;
    } else if (largest_bits < 0x0d800000u) {         // 2^-100: 127 / largest would overflow further down
        r.scale = 0.f;
        r.inv = 0.f;
    } else {
        r.scale = __fdiv_rn(largest, 127.f);
        r.inv = __fdiv_rn(127.f, largest);
    }
    return r;
}
// The factors are a few roundings off, so |v * inv| <= 127 (1 + 2^-21) and rounds to 127 at most; where inv is 0 the product is 0 or NaN, and
// the conversion turns NaN into 0.
__device__ __forceinline__ int32_t quantise(float v, float inv) { return __float2int_rn(__fmul_rn(v, inv)); }
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

}  // namespace
#endif

}  // namespace enn_b200
