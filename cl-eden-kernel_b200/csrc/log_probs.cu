// log_probs: log probabilities of given ids, entropy and the largest alternatives of rows of logits.
#include <math_constants.h>

#include "token_ops.h"

namespace enn_b200 {
namespace {

constexpr int kThreads = 256;

// Order of the logits as unsigned integers: NaN above +inf, -0 equal to +0; the lower index first among equals.
__device__ __forceinline__ uint64_t order_key(float v, int32_t index) {
    uint32_t b = __float_as_uint(v + 0.f);
    if (v != v) b = 0x7fffffffu;
    b = b & 0x80000000u ? ~b : b | 0x80000000u;
    return static_cast<uint64_t>(b) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}

template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, V *scratch, F join) {
    for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[threadIdx.x & (kThreads / 32 - 1)];
    for (int o = kThreads / 64; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) log_probs_kernel(LogProbsParams p, const T *logits, const int32_t *ids, float *given, float *entropy, int32_t *top_ids, float *top) {
    __shared__ float scratch[kThreads / 32];
    __shared__ uint64_t scratch64[kThreads / 32];
    pdl_wait();
    pdl_trigger();
    const int64_t t = blockIdx.x;
    const T *row = logits + t * p.pitch;
    float largest = -CUDART_INF_F;
    for (int i = threadIdx.x; i < p.vocab; i += kThreads) largest = fmaxf(largest, to_float(row[i]) * p.scale);
    largest = block_reduce(largest, scratch, [](float a, float b) { return fmaxf(a, b); });
    // With d = z - largest: S = sum e^d, U = sum d e^d; lse = largest + log S, entropy = log S - U / S.
    float s = 0.f, u = 0.f;
    for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
        const float d = to_float(row[i]) * p.scale - largest, e = expf(d);
        s += e;
        u += d == -CUDART_INF_F ? 0.f : d * e;
    }
    s = block_reduce(s, scratch, [](float a, float b) { return a + b; });
    u = block_reduce(u, scratch, [](float a, float b) { return a + b; });
    const float log_s = logf(s);
    if (threadIdx.x == 0) entropy[t] = log_s - u / s;
    for (int j = threadIdx.x; j < p.given; j += kThreads) {
        const int32_t id = ids[t * p.given + j];
        given[t * p.given + j] = id < 0 ? 0.f : (id >= p.vocab ? CUDART_NAN_F : (to_float(row[id]) * p.scale - largest) - log_s);
    }
    uint64_t below = ~0ull;
    for (int j = 0; j < p.top; ++j) {
        uint64_t best = 0;
        for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
            const uint64_t k = order_key(to_float(row[i]), i);
            if (k < below && k > best) best = k;
        }
        best = block_reduce(best, scratch64, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
        below = best;
        const int32_t id = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(best));
        if (threadIdx.x == 0) {
            top_ids[t * p.top + j] = id;
            top[t * p.top + j] = (to_float(row[id]) * p.scale - largest) - log_s;
        }
    }
}

template <typename T>
cudaError_t launch_typed(const TokenState &t, int32_t rows, const void *const *ins, void *const *outs, cudaStream_t stream) {
    const LogProbsParams &p = t.log_probs;
    int o = 0;
    const int32_t *ids = p.given ? static_cast<const int32_t *>(ins[1]) : nullptr;
    float *given = p.given ? static_cast<float *>(outs[o++]) : nullptr;
    float *entropy = static_cast<float *>(outs[o++]);
    int32_t *top_ids = p.top ? static_cast<int32_t *>(outs[o++]) : nullptr;
    float *top = p.top ? static_cast<float *>(outs[o++]) : nullptr;
    return launch_pdl(log_probs_kernel<T>, dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, stream, p, static_cast<const T *>(ins[0]), ids, given, entropy, top_ids, top);
}

}  // namespace

cudaError_t log_probs_launch(const enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs) {
    const TokenState &t = *op->token;
    const cudaStream_t stream = op->ctx->stream;
    switch (t.in_dtype) {
        case ENN_B200_F32: return launch_typed<float>(t, rows, ins, outs, stream);
        case ENN_B200_F16: return launch_typed<__half>(t, rows, ins, outs, stream);
        case ENN_B200_BF16: return launch_typed<__nv_bfloat16>(t, rows, ins, outs, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace enn_b200
