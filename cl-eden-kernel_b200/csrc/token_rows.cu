// token_norm and token_gate: row-wise operators around the 8-bit products of a block.
#include "token_ops.h"

namespace enn_b200 {
namespace {

constexpr int kThreads = 256;

template <typename F>
__device__ __forceinline__ float block_reduce(float v, float *scratch, F join) {
    for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[threadIdx.x & (kThreads / 32 - 1)];
    for (int o = kThreads / 64; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float block_sum(float v, float *scratch) {
    return block_reduce(v, scratch, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ uint32_t block_max_bits(uint32_t v, float *scratch) {
    return __float_as_uint(block_reduce(__uint_as_float(v), scratch, [](float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }));
}

// row[0..c) = norm(row)
__device__ void norm_row(float *row, int c, int kind, float eps, const float *weight, const float *bias, float *scratch) {
    if (kind == ENN_B200_NORM_NONE) return;
    float mean = 0.f;
    if (kind == ENN_B200_NORM_LAYER) {
        float s = 0.f;
        for (int i = threadIdx.x; i < c; i += kThreads) s += row[i];
        mean = block_sum(s, scratch) / static_cast<float>(c);
    }
    float s = 0.f;
    for (int i = threadIdx.x; i < c; i += kThreads) s += (row[i] - mean) * (row[i] - mean);
    const float r = rsqrtf(block_sum(s, scratch) / static_cast<float>(c) + eps);
    for (int i = threadIdx.x; i < c; i += kThreads) row[i] = (row[i] - mean) * r * (weight ? weight[i] : 1.f) + (bias ? bias[i] : 0.f);
}

template <typename T, typename O>
__global__ void __launch_bounds__(kThreads) token_norm_kernel(NormParams p, const T *x, const T *residual, const T *gate, T *stream, O *y, float *scale) {
    extern __shared__ float row[];
    __shared__ float scratch[kThreads / 32];
    pdl_wait();
    pdl_trigger();
    const int64_t t = blockIdx.x, at = t * p.c;
    for (int i = threadIdx.x; i < p.c; i += kThreads) row[i] = to_float(x[at + i]);
    norm_row(row, p.c, p.post_norm, p.post_eps, p.post_weight, p.post_bias, scratch);
    for (int i = threadIdx.x; i < p.c; i += kThreads) {
        float v = row[i];
        if (gate) v *= to_float(gate[t / p.gate_tokens * p.c + i]);
        v *= p.residual_scale;
        if (residual) {
            v += to_float(residual[at + i]);
            stream[at + i] = from_float<T>(v);
        }
        row[i] = v;
    }
    norm_row(row, p.c, p.norm, p.eps, p.weight, p.bias, scratch);
    if constexpr (sizeof(O) == 1) {
        uint32_t largest = 0;
        for (int i = threadIdx.x; i < p.c; i += kThreads) largest = max(largest, magnitude(row[i]));
        const RowScale rs = row_scale(block_max_bits(largest, scratch));
        for (int64_t i = threadIdx.x; i < p.pitch; i += kThreads) y[t * p.pitch + i] = i < p.c ? static_cast<O>(quantise(row[i], rs.inv)) : O(0);
        if (threadIdx.x == 0) scale[t] = rs.scale;
    } else {
        for (int i = threadIdx.x; i < p.c; i += kThreads) y[at + i] = from_float<O>(row[i]);
    }
}

// 1 / (1 + e^-g) from an exponential that does not overflow.
__device__ __forceinline__ float sigmoid(float g) {
    const float e = expf(-fabsf(g));
    return (g >= 0.f ? 1.f : e) / (1.f + e);
}

__device__ __forceinline__ float gate_act(float g, int act) {
    switch (act) {
        case ENN_B200_GATE_SILU: return g * sigmoid(g);
        case ENN_B200_GATE_GELU: return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
        case ENN_B200_GATE_GELU_TANH: return 0.5f * g * (1.f + tanhf(0.79788456080286536f * (g + 0.044715f * g * g * g)));
        case ENN_B200_GATE_RELU: return g < 0.f ? 0.f : g;
        default: return sigmoid(g);
    }
}

template <typename T, typename O>
__global__ void __launch_bounds__(kThreads) token_gate_kernel(GateParams p, const T *gates, const T *values, O *y, float *scale) {
    __shared__ float scratch[kThreads / 32];
    pdl_wait();
    pdl_trigger();
    const int64_t t = blockIdx.x;
    const T *g = gates + t * p.in_stride, *u = values + t * p.in_stride;
    auto at = [&](int64_t i) { return gate_act(to_float(g[i]), p.act) * to_float(u[i]); };
    if constexpr (sizeof(O) == 1) {
        uint32_t largest = 0;
        for (int i = threadIdx.x; i < p.c; i += kThreads) largest = max(largest, magnitude(at(i)));
        const RowScale rs = row_scale(block_max_bits(largest, scratch));
        for (int64_t i = threadIdx.x; i < p.pitch; i += kThreads) y[t * p.pitch + i] = i < p.c ? static_cast<O>(quantise(at(i), rs.inv)) : O(0);
        if (threadIdx.x == 0) scale[t] = rs.scale;
    } else {
        for (int i = threadIdx.x; i < p.c; i += kThreads) y[t * p.c + i] = from_float<O>(at(i));
    }
}

// f(T{}) with the element type of `dtype`.
template <typename F>
cudaError_t with_type(int32_t dtype, F f) {
    switch (dtype) {
        case ENN_B200_F32: return f(float{});
        case ENN_B200_F16: return f(__half{});
        case ENN_B200_BF16: return f(__nv_bfloat16{});
        case ENN_B200_S8: return f(int8_t{});
    }
    return cudaErrorInvalidValue;
}

template <typename T, typename O>
cudaError_t norm_typed(const TokenState &t, int32_t rows, const void *const *ins, void *const *outs, cudaStream_t stream) {
    int i = 0, o = 0;
    const T *x = static_cast<const T *>(ins[i++]);
    const T *residual = t.residual ? static_cast<const T *>(ins[i++]) : nullptr;
    const T *gate = t.norm.gate_tokens ? static_cast<const T *>(ins[i++]) : nullptr;
    T *h = t.residual ? static_cast<T *>(outs[o++]) : nullptr;
    O *y = static_cast<O *>(outs[o++]);
    float *scale = sizeof(O) == 1 ? static_cast<float *>(outs[o++]) : nullptr;
    const size_t smem = sizeof(float) * static_cast<size_t>(t.norm.c);
    if (smem > 32 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(token_norm_kernel<T, O>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(token_norm_kernel<T, O>, dim3(static_cast<unsigned>(rows)), dim3(kThreads), smem, stream, t.norm, x, residual, gate, h, y, scale);
}

template <typename T, typename O>
cudaError_t gate_typed(const TokenState &t, int32_t rows, const void *const *ins, void *const *outs, cudaStream_t stream) {
    const T *g = static_cast<const T *>(ins[0]), *u = t.packed ? g + t.gate.c : static_cast<const T *>(ins[1]);
    return launch_pdl(token_gate_kernel<T, O>, dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, stream, t.gate, g, u, static_cast<O *>(outs[0]),
                      sizeof(O) == 1 ? static_cast<float *>(outs[1]) : nullptr);
}

}  // namespace

cudaError_t token_norm_launch(const TokenState &t, int32_t rows, const void *const *ins, void *const *outs, cudaStream_t stream) {
    return with_type(t.in_dtype, [&](auto in) {
        return with_type(t.out_dtype, [&](auto out) {
            if constexpr (sizeof(in) == 1) return cudaErrorInvalidValue;
            else return norm_typed<decltype(in), decltype(out)>(t, rows, ins, outs, stream);
        });
    });
}

cudaError_t token_gate_launch(const TokenState &t, int32_t rows, const void *const *ins, void *const *outs, cudaStream_t stream) {
    return with_type(t.in_dtype, [&](auto in) {
        return with_type(t.out_dtype, [&](auto out) {
            if constexpr (sizeof(in) == 1) return cudaErrorInvalidValue;
            else return gate_typed<decltype(in), decltype(out)>(t, rows, ins, outs, stream);
        });
    });
}

}  // namespace enn_b200
