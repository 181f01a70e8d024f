// token_fc: byte rows times byte weights, with a scale per token and per channel.
#include <algorithm>
#include <cstdio>

#include "per_device.h"
#include "tc_host.h"
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
__global__ void __launch_bounds__(kDirectThreads) token_fc_direct_kernel(TokenFcDirect p, int32_t rows, const int8_t *q, const float *token_scale, O *out) {
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

// ---- tensor-core kernel: one tile of 128 channels x bn tokens per CTA, the reduction split over a cluster.
// The channels are the rows of the matrix instruction (always 128), the tokens its columns (16 .. 256), so that a call of few tokens
// wastes nothing but its 16th columns and is bound by reading the weights.  A cluster of `splits` CTAs shares a tile: each multiplies
// its part of k, and the exact 32-bit partial sums meet through distributed shared memory; no atomics, no workspace, the same result for
// every split.
//   warp 0, lane 0   copies the weight tiles.  Weights are constants of the operator, so their copies start before the kernel ahead in
//                    the stream has finished (programmatic launch): a decode step's products overlap what is in front of them.
//   warp 1, lane 0   copies the token tiles
//   warp 2, lane 0   issues the matrix instructions
//   warps 2 .. 5     bring the accumulators from tensor memory into shared memory, which the operands no longer need
//   all              add the partial sums, scale and store
constexpr int kChannels = kBM;
constexpr int kTcThreads = 192;
constexpr int kMaxTokens = kMaxBN;
constexpr int kMaxSplits = 8;       // portable cluster size
constexpr int kMaxStages = 12;

struct TcCall {
    int32_t rows, n;
    int32_t kb_total;               // k-blocks of 128 bytes
    int32_t splits, m_tiles, bn, stages;
    uint32_t idesc, tmem_cols;
    const float *token_scale, *channel_scale, *bias;
    int32_t *err;
    int32_t starve;                 // self-test of the bounded waits: nothing is copied, the waits give up early
    int32_t vec;                    // four outputs at once: n and the address allow it
};

__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
__device__ __forceinline__ int4 ld_cluster(uint32_t addr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

// Four neighbouring results; the address is a multiple of four elements.
__device__ __forceinline__ void store4(float *p, const float (&v)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(__half *p, const float (&v)[4]) {
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, const float (&v)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

template <typename O>
__global__ void __launch_bounds__(kTcThreads) token_fc_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q, const TcCall p, O *out) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 * kMaxStages + 1];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    volatile int *abort_flag = &abort_word;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nst = p.stages;
    const uint32_t w_bytes = kChannels * kBK, q_bytes = static_cast<uint32_t>(p.bn) * kBK, stage_bytes = w_bytes + q_bytes;
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages, tfull = empty0 + 8 * kMaxStages;
    const uint32_t ring = smem_u32(smem);
    const int split = static_cast<int>(blockIdx.x) % p.splits, tile = static_cast<int>(blockIdx.x) / p.splits;
    const int tm = tile % p.m_tiles, tn = tile / p.m_tiles;      // the token tiles of a weight tile run together
    const int64_t m0 = static_cast<int64_t>(tm) * p.bn;
    const int n0 = tn * kChannels;
    const int kb0 = static_cast<int>(static_cast<int64_t>(p.kb_total) * split / p.splits);
    const int kbs = static_cast<int>(static_cast<int64_t>(p.kb_total) * (split + 1) / p.splits) - kb0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < nst; ++s) {
            mbar_init(full0 + 8 * s, 2);        // an expect-tx arrival of either producer
            mbar_init(empty0 + 8 * s, 1);
        }
        mbar_init(tfull, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) tmem_alloc(smem_u32(&tmem_slot), p.tmem_cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_trigger();

    uint32_t stage = 0, phase = 0;      // a producer's next fill, the issuer's next k-block
    if (warp < 2) {
        if (lane == 0 && !p.starve) {
            if (warp == 1) pdl_wait();          // the tokens are what the kernel before this one writes
            const CUtensorMap *map = warp ? &map_q : &map_w;
            const uint32_t dst = ring + (warp ? w_bytes : 0), bytes = warp ? q_bytes : w_bytes;
            const int row = warp ? static_cast<int>(m0) : n0;
            for (int kb = 0; kb < kbs; ++kb) {
                if (kb >= nst && !mbar_test_wait(empty0 + 8 * stage, phase ^ 1) && !mbar_wait_fast(empty0 + 8 * stage, phase ^ 1, abort_flag, p.err, 1)) break;
                mbar_expect_tx(full0 + 8 * stage, bytes);
                tma_load_2d(dst + stage * stage_bytes, map, full0 + 8 * stage, (kb0 + kb) * kBK, row);
                if (++stage == static_cast<uint32_t>(nst)) { stage = 0; phase ^= 1; }
            }
        }
    } else {
        if (warp == 2 && lane == 0) {
            const uint32_t desc_hi = static_cast<uint32_t>(make_smem_desc(0) >> 32);
            const uint32_t looks = p.starve ? 64u : (kSpinLimit >> 7);
            for (int kb = 0; kb < kbs; ++kb) {
                if (!mbar_test_wait(full0 + 8 * stage, phase) && !mbar_wait_fast(full0 + 8 * stage, phase, abort_flag, p.err, 2, looks)) break;
                const uint32_t lo = (ring + stage * stage_bytes) >> 4;
                umma_i8_run<false, 4>(tmem, desc_hi, lo, lo + (w_bytes >> 4), p.idesc, kb != 0);
                umma_commit(empty0 + 8 * stage);
                if (++stage == static_cast<uint32_t>(nst)) { stage = 0; phase ^= 1; }
            }
            if (!*abort_flag) umma_commit(tfull);
        }
        __syncwarp();
        if (mbar_wait(tfull, 0, abort_flag, p.err, 3)) {
            // Every matrix instruction has read its operands: their memory takes the sums, [token][channel].
            tc_fence_after();
            const int q = warp & 3;
            const uint32_t t_row = tmem + (static_cast<uint32_t>(q * 32) << 16);
            const uint32_t dst = ring + (q * 32 + lane) * 4;
            for (int c = 0; c < p.bn; c += 16) {
                uint32_t r[16];
                tmem_ld16(t_row + c, r);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + (c + i) * (kChannels * 4)), "r"(r[i]) : "memory");
            }
        }
        tc_fence_before();
    }
    __syncwarp();
    if (p.splits > 1) cluster_sync_all();
    else __syncthreads();
    if (*abort_flag) {
        if (warp < 2 && lane == 0 && !p.starve) drain_stages(full0, nst, stage, phase);      // no copy may land in memory that is given back
    } else {
        // The CTAs of the cluster take the tokens in turn; a warp stores the 128 channels of a token, a lane four of them.
        pdl_wait();
        const int n = n0 + lane * 4;
        float cs[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cs[i] = n + i < p.n ? p.channel_scale[n + i] : 0.f;
            b[i] = p.bias && n + i < p.n ? p.bias[n + i] : 0.f;
        }
        const int tokens = static_cast<int>(min(static_cast<int64_t>(p.bn), p.rows - m0));
        for (int j = split + p.splits * warp; j < tokens; j += p.splits * (kTcThreads / 32)) {
            const float ts = p.token_scale[m0 + j];
            const uint32_t at = ring + j * (kChannels * 4) + lane * 16;
            int4 a = make_int4(0, 0, 0, 0);
            if (p.splits == 1) {
                a = ld_cluster(at);
            } else {
                for (int s = 0; s < p.splits; s += 2) {
                    const int4 x = ld_cluster(mapa_rank(at, s)), y = ld_cluster(mapa_rank(at, s + 1));
                    a.x += x.x + y.x; a.y += x.y + y.y; a.z += x.z + y.z; a.w += x.w + y.w;
                }
            }
            const float v[4] = {scaled(a.x, ts, cs[0], b[0]), scaled(a.y, ts, cs[1], b[1]), scaled(a.z, ts, cs[2], b[2]), scaled(a.w, ts, cs[3], b[3])};
            O *o = out + (m0 + j) * p.n + n;
            if (p.vec && n < p.n) {
                store4(o, v);
            } else if (!p.vec) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.n) o[i] = from_float<O>(v[i]);
            }
        }
    }
    if (p.splits > 1) cluster_sync_all();       // nobody leaves while its sums are still read
    else __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, p.tmem_cols);
    }
}

template <typename O>
cudaError_t kernel_init(int device) {
    static PerDeviceInit once;
    return once.run(device, [] { return cudaFuncSetAttribute(token_fc_kernel<O>, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024); });
}

constexpr uint32_t kSignedBytes = (2u << 4) | (1u << 7) | (1u << 10);      // s32 sums of s8 x s8

template <typename O>
cudaError_t launch_tc(enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs) {
    TokenState &t = *op->token;
    enn_b200_context *ctx = op->ctx;
    TcCall c{};
    c.rows = rows;
    c.n = t.fc.n;
    c.kb_total = (t.fc.k + kBK - 1) / kBK;
    c.m_tiles = (rows + kMaxTokens - 1) / kMaxTokens;
    c.bn = ((rows + c.m_tiles - 1) / c.m_tiles + 15) / 16 * 16;
    const int64_t n_tiles = (t.fc.n + kChannels - 1) / kChannels, tiles = n_tiles * c.m_tiles;
    // Two CTAs share an SM while their rings fit (up to 128 tokens).
    const int per_sm = c.bn <= 128 ? 2 : 1;
    const int slots = per_sm * ctx->launch_sms();
    c.splits = 1;
    while (c.splits < kMaxSplits && tiles * c.splits * 2 <= slots && c.kb_total >= 4 * c.splits) c.splits *= 2;
    const int stage_bytes = (kChannels + c.bn) * kBK, budget = (per_sm == 2 ? 111 : 222) * 1024;
    c.stages = std::min({budget / stage_bytes, (c.kb_total + c.splits - 1) / c.splits, kMaxStages});
    const size_t smem = 1024 + static_cast<size_t>(std::max(c.stages * stage_bytes, c.bn * kChannels * 4));
    c.tmem_cols = 32;
    while (c.tmem_cols < static_cast<uint32_t>(c.bn)) c.tmem_cols *= 2;
    c.idesc = kSignedBytes | (static_cast<uint32_t>(c.bn >> 3) << 17) | (static_cast<uint32_t>(kChannels >> 4) << 24);
    c.token_scale = static_cast<const float *>(ins[1]);
    c.channel_scale = t.fc.channel_scale;
    c.bias = t.fc.bias;
    c.err = t.fc.err_dev;
    c.starve = t.fc.starve_next;
    t.fc.starve_next = false;
    c.vec = t.fc.n % 4 == 0 && reinterpret_cast<uintptr_t>(outs[0]) % (4 * sizeof(O)) == 0;
    CUtensorMap map_q;
    if (!encode_2d(ctx, &map_q, ins[0], static_cast<uint64_t>(t.fc.k), static_cast<uint64_t>(rows), static_cast<uint64_t>(t.fc.in_pitch), kBK, static_cast<uint32_t>(c.bn)))
        return cudaErrorInvalidValue;
    const cudaError_t e = kernel_init<O>(ctx->device);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * c.splits));
    cfg.blockDim = dim3(kTcThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(c.splits);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, token_fc_kernel<O>, t.fc.map_w, map_q, c, static_cast<O *>(outs[0]));
}

template <typename O>
cudaError_t launch_typed(enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs) {
    const TokenState &t = *op->token;
    // The tensor copies want 16-byte lines; other addresses and pitches take the general kernel.
    if (op->impl == ENN_B200_IMPL_TCGEN05 && reinterpret_cast<uintptr_t>(ins[0]) % 16 == 0 && t.fc.in_pitch % 16 == 0) return launch_tc<O>(op, rows, ins, outs);
    const dim3 grid(static_cast<unsigned>((rows + kTile - 1) / kTile), static_cast<unsigned>((t.fc.n + kTile - 1) / kTile));
    return launch_pdl(token_fc_direct_kernel<O>, grid, dim3(kDirectThreads), 0, op->ctx->stream, t.fc.direct(), rows, static_cast<const int8_t *>(ins[0]),
                      static_cast<const float *>(ins[1]), static_cast<O *>(outs[0]));
}

}  // namespace

// The part of the plan that does not depend on a call: the weights' tensor map and the error word.
cudaError_t token_fc_plan(enn_b200_op *op) {
    TokenFcParams &f = op->token->fc;
    if (!encode_2d(op->ctx, &f.map_w, f.w, static_cast<uint64_t>(f.k), static_cast<uint64_t>(f.n), static_cast<uint64_t>(f.w_pitch), kBK, kChannels)) return cudaErrorInvalidValue;
    cudaError_t e = cudaHostAlloc(reinterpret_cast<void **>(&f.err_host), sizeof(int32_t), cudaHostAllocMapped);
    if (e != cudaSuccess) {
        f.err_host = nullptr;
        return e;
    }
    *f.err_host = 0;
    return cudaHostGetDevicePointer(reinterpret_cast<void **>(&f.err_dev), f.err_host, 0);
}

cudaError_t token_fc_launch(enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs) {
    const TokenFcParams &f = op->token->fc;
    if (f.err_host && *reinterpret_cast<volatile int32_t *>(f.err_host) != 0) return cudaErrorLaunchFailure;
    switch (op->token->out_dtype) {
        case ENN_B200_F32: return launch_typed<float>(op, rows, ins, outs);
        case ENN_B200_F16: return launch_typed<__half>(op, rows, ins, outs);
        case ENN_B200_BF16: return launch_typed<__nv_bfloat16>(op, rows, ins, outs);
    }
    return cudaErrorInvalidValue;
}

}  // namespace enn_b200
