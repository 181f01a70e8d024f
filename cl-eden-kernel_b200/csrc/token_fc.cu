// token_fc: byte rows times byte weights, with a scale per token and per channel.
#include "token_ops.h"

namespace enn_b200 {
namespace {

// (acc * token scale) * channel scale + bias, rounded once.  The integer sum is rounded to 24 bits first where it is longer.
__device__ __forceinline__ float scaled(int32_t acc, float token, float channel, float bias) {
    return __fmaf_rn(__fmul_rn(static_cast<float>(acc), token), channel, bias);
}

// ---- general kernel: any address and pitch.  64 tokens x 64 channels per CTA, four by four per thread, dp4a on words that are put
//      together from single bytes when they are brought into shared memory ----
constexpr int kTile = 64, kWords = 16, kDirectThreads = 256;

template <typename O>
__global__ void __launch_bounds__(kDirectThreads) token_fc_direct_kernel(TokenFcParams p, int32_t rows, const int8_t *q, const float *token_scale, O *out) {
    __shared__ int32_t sa[kWords][kTile + 1], sw[kWords][kTile + 1];
    pdl_wait();
    pdl_trigger();
    const int64_t m0 = static_cast<int64_t>(blockIdx.x) * kTile;
    const int n0 = blockIdx.y * kTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int32_t acc[4][4] = {};
    for (int k0 = 0; k0 < p.k; k0 += 4 * kWords) {
        for (int i = threadIdx.x; i < kTile * kWords; i += kDirectThreads) {
            const int r = i / kWords, w = i % kWords, k = k0 + 4 * w;
            uint32_t a = 0, b = 0;
            for (int j = 0; j < 4; ++j) {
                if (k + j >= p.k) break;
                if (m0 + r < rows) a |= static_cast<uint32_t>(static_cast<uint8_t>(q[(m0 + r) * p.in_pitch + k + j])) << (8 * j);
                if (n0 + r < p.n) b |= static_cast<uint32_t>(static_cast<uint8_t>(p.w[(n0 + r) * p.w_pitch + k + j])) << (8 * j);
            }
            sa[w][r] = static_cast<int32_t>(a);
            sw[w][r] = static_cast<int32_t>(b);
        }
        __syncthreads();
        for (int w = 0; w < kWords; ++w)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(sa[w][ty + 16 * i], sw[w][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + ty + 16 * i;
        if (m >= rows) continue;
        const float ts = token_scale[m];
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + tx + 16 * j;
            if (n < p.n) out[m * p.n + n] = from_float<O>(scaled(acc[i][j], ts, p.channel_scale[n], p.bias ? p.bias[n] : 0.f));
        }
    }
}

template <typename O>
cudaError_t launch_typed(const TokenState &t, int32_t rows, const void *const *ins, void *const *outs, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>((rows + kTile - 1) / kTile), static_cast<unsigned>((t.fc.n + kTile - 1) / kTile));
    return launch_pdl(token_fc_direct_kernel<O>, grid, dim3(kDirectThreads), 0, stream, t.fc, rows, static_cast<const int8_t *>(ins[0]),
                      static_cast<const float *>(ins[1]), static_cast<O *>(outs[0]));
}

}  // namespace

cudaError_t token_fc_launch(const TokenState &t, int32_t rows, const void *const *ins, void *const *outs, cudaStream_t stream) {
    switch (t.out_dtype) {
        case ENN_B200_F32: return launch_typed<float>(t, rows, ins, outs, stream);
        case ENN_B200_F16: return launch_typed<__half>(t, rows, ins, outs, stream);
        case ENN_B200_BF16: return launch_typed<__nv_bfloat16>(t, rows, ins, outs, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace enn_b200
