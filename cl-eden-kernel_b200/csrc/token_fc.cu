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
// The channels are the rows of the matrix instruction (always 128), the tokens its columns (16 .. 128), so that a call of few tokens
// multiplies at most 15 columns for nothing and is bound by reading the weights.  A cluster of `splits` CTAs shares a tile: each multiplies
// its part of k, and the exact 32-bit partial sums meet through distributed shared memory; no atomics, no workspace, the same result for
// every split.
//   warp 0, lane 0   copies the weight tiles.  Weights are constants of the operator, so their copies start before the kernel ahead in
//                    the stream has finished (programmatic launch): a decode step's products overlap what is in front of them.
//   warp 1, lane 0   copies the token tiles
//   warp 2, lane 0   issues the matrix instructions
//   warps 2 .. 5     bring the accumulators from tensor memory into shared memory, which the operands no longer need
//   all              add the partial sums, scale and store
// 16 tokens x 8192 -> 16384: 24.4 us, 5.5 TB/s of weights; 1 x 4096 -> 4096 5.6 us, of which 2.6 are the weights and the rest one
// dependent step after the other (launch, first tiles, cluster, store).  Weights in tiles of 16 KB instead of rows made no difference.
constexpr int kChannels = kBM;
constexpr int kTcThreads = 192;
constexpr int kTcTokens = 128;      // most tokens of a tile
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
    __shared__ float scales[kTcTokens];         // of the tile's tokens
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

    // A lane of the write-out has four channels; their constants and the tokens' scales are on the way while the tile is multiplied.
    const int n = n0 + lane * 4, tokens = static_cast<int>(min(static_cast<int64_t>(p.bn), p.rows - m0));
    float cs[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        cs[i] = n + i < p.n ? p.channel_scale[n + i] : 0.f;
        b[i] = p.bias && n + i < p.n ? p.bias[n + i] : 0.f;
    }
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
        pdl_wait();
        const int mine = static_cast<int>(threadIdx.x) - 64;      // warps 2 .. 5: 128 threads
        if (mine < tokens) scales[mine] = p.token_scale[m0 + mine];
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
        const int per = p.splits * (kTcThreads / 32);
#pragma unroll 2
        for (int j = split + p.splits * warp; j < tokens && n < p.n; j += per) {
            const float ts = scales[j];
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
            if (p.vec) {
                store4(o, v);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.n) o[i] = from_float<O>(v[i]);
            }
        }
    }
    // Nobody leaves while its sums are still read.  The arrival is relaxed, so that it does not wait for the results' stores; it has no need to order
    // memory: a lane reads sums of other CTAs only where it stores what it makes of them, and its loads have returned by then.
    __syncwarp();
    if (p.splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
    else __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, p.tmem_cols);
    }
}

// ---- tensor-core kernel for large products: persistent pairs of CTAs (cta_group::2), 256 channels x bn tokens per tile.
// A CTA of the pair holds 128 channels of the weights and half of the tokens of every k-block, so that each operand byte comes from L2 once
// per pair, and the accumulators of its 128 channels.  Two accumulators of up to 256 columns take all of tensor memory: one is multiplied
// into while the other is scaled and stored, 32 channels x 32 tokens at a time by a warp of the epilogue.  16-bit results are transposed
// on their way through shared memory and leave in 16-byte pieces, 64 bytes of a token; others (n not a multiple of eight, 32-bit
// results) leave straight from the accumulators' layout, where a thread has one channel: 32 neighbouring channels of a token per instruction.
// 8192 x 4096 -> 8192: 178 us in a short run (3.1 POPS, tensor pipe 78 % busy), 207 us under the power limit of a long one.  The width of the
// token tiles follows the rounds (512 x 4096 -> 4096: 13.0 us in 64 tiles of 128, 14.8 us on single CTAs).  Below kPairRows tokens
// single CTAs with a split reduction are quicker where the weights are few, and about as quick where they are many (pairs in parentheses):
// 160 x 4096 -> 4096 10.2 us (12.4), 64 x 8192 -> 16384 26.4 us (27.5), 128 x 8192 -> 16384 29.2 us (28.3).  From there pairs lose less than
// they gain: 200 x 4096 -> 4096 11.2 us (12.2), 256 x 4096 -> 4096 12.1 us (12.3), 200 x 8192 -> 16384 38.6 us (30.4), 300 x 1024 -> 4096 9.6 us (7.2).
//   warp 0           copies the weight tiles, of both CTAs
//   warp 1           issues the matrix instructions in the first CTA; allocates in both
//   warps 2 .. 9     epilogue: lane quarter warp & 3, every other group of 32 tokens
//   warp 10          copies the token tiles
constexpr int kPairStages = 6;
constexpr int kPairEpiWarps = 8;
constexpr int kPairThreads = (kPairEpiWarps + 3) * 32;
constexpr int kPairStageBytes = (kBM + kMaxBN / 2) * kBK;
constexpr int kPairRows = 192;
// What a tile costs beside its columns, in columns; found by trying.  Less takes tiles that are too narrow (512 x 4096 -> 4096 13.0 us, 17.0 with 0, 14.9 with
// 24; 2048 x 4096 -> 6144 38 us, 99 with 0), more some that are too wide (256 x 4096 -> 4096 12.3 us, 15.9 with 96; 8192 x 512 -> 4096 23.4, 24.1).
constexpr int kTileCost = 48;
constexpr int kPairOutBytes = 32 * 32 * 2;      // results of a warp on their way out

struct PairCall {
    int32_t rows, n, kb_total;
    int32_t tiles_c, tiles_t, bn;       // channel tiles of 256, token tiles of bn
    int32_t band;                       // channel tiles that are walked together: their operands stay in L2
    uint32_t idesc;
    const float *token_scale, *channel_scale, *bias;
    int32_t *err;
    int32_t starve;
    int32_t vec;                        // 16-bit results in pieces of eight channels: n and the address allow it
};

__device__ __forceinline__ uint32_t pack_results(float a, float b, __half) {
    const __half2 p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ uint32_t pack_results(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&p);
}
// Four 8 x 8 matrices of 16-bit values, transposed: lane i gives the address of row i % 8 of matrix i / 8.
__device__ __forceinline__ void store_matrices_transposed(uint32_t addr, const uint32_t (&r)[4]) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
                 "%23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
                   "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}

// Tile number -> channel tile and token tile: bands of channel tiles, the channel tile running fastest within a band.
__device__ __forceinline__ void pair_tile(const PairCall &p, int tile, int &tc, int &tt) {
    const int per = p.band * p.tiles_t, b = tile / per, r = tile - b * per, width = min(p.band, p.tiles_c - b * p.band);
    tt = r / width;
    tc = b * p.band + (r - tt * width);
}

// Gives an accumulator back without a release, which would wait for the results' stores as well.  What has to be over is the reading of
// tensor memory alone, and it is: tcgen05.wait::ld has brought the values of every load into registers, and the tcgen05 fence before the arrival
// with the one that the issuer takes after its wait orders these loads before the next matrix instructions.  Nothing else passes from here to the issuer.
__device__ __forceinline__ void arrive_relaxed(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

template <typename O>
__global__ void __launch_bounds__(kPairThreads, 1) token_fc_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_q, const PairCall p,
                                                                         O *out) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bars[2 * kPairStages + 4];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    volatile int *abort_flag = &abort_word;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kPairStages, tfull0 = empty0 + 8 * kPairStages, tempty0 = tfull0 + 16;
    const uint32_t ring = smem_u32(smem), w_bytes = kBM * kBK, q_bytes = static_cast<uint32_t>(p.bn / 2) * kBK;
    const int first = static_cast<int>(blockIdx.x >> 1), step = static_cast<int>(gridDim.x >> 1), total = p.tiles_c * p.tiles_t;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) {
            mbar_init(full0 + 8 * s, 2);        // an expect-tx arrival of either producer of the first CTA
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(tfull0 + 8 * b, 1);
            mbar_init(tempty0 + 8 * b, 2 * kPairEpiWarps);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc_pair(smem_u32(&tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                         // the peer's barriers exist before anything signals them
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_trigger();

    // A role that gives up stops its own CTA and the peer.
    const auto give_up = [&] { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_rank(smem_u32(&abort_word), rank ^ 1)), "r"(1) : "memory"); };
    uint32_t stage = 0, phase = 0;
    if (warp == 0 || warp == kPairEpiWarps + 2) {
        // Two lanes take the k-blocks in turn (a thread issues a tensor copy in about the time a k-block is multiplied); a stage keeps its lane.
        if (lane < 2 && !p.starve) {
            const bool is_w = warp == 0;
            if (!is_w) pdl_wait();
            const CUtensorMap *map = is_w ? &map_w : &map_q;
            const uint32_t bytes = is_w ? w_bytes : q_bytes, dst = ring + (is_w ? 0 : w_bytes);
            const int tiles = first < total ? (total - first + step - 1) / step : 0;
            int t = 0, t_row = -1, kb = lane, row = 0;
            stage = lane;
            while (kb >= p.kb_total) { kb -= p.kb_total; ++t; }
            while (t < tiles) {
                if (t != t_row) {
                    t_row = t;
                    int tc, tt;
                    pair_tile(p, first + t * step, tc, tt);
                    row = is_w ? (tc * 2 + static_cast<int>(rank)) * kBM : tt * p.bn + static_cast<int>(rank) * (p.bn / 2);
                }
                if (!mbar_test_wait(empty0 + 8 * stage, phase ^ 1) && !mbar_wait_fast(empty0 + 8 * stage, phase ^ 1, abort_flag, p.err, 1)) {
                    give_up();
                    break;
                }
                if (rank == 0) mbar_expect_tx(full0 + 8 * stage, 2 * bytes);      // of both CTAs; every copy reports to the first
                tma_load_2d_pair(dst + stage * kPairStageBytes, map, mapa_rank(full0 + 8 * stage, 0), kb * kBK, row);
                stage += 2;
                if (stage >= kPairStages) { stage -= kPairStages; phase ^= 1; }
                kb += 2;
                while (kb >= p.kb_total) { kb -= p.kb_total; ++t; }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t desc_hi = static_cast<uint32_t>(make_smem_desc(0) >> 32);
            int it = 0;
            for (int tile = first; tile < total; tile += step, ++it) {
                const uint32_t ab = it & 1, use = it >> 1;
                if (!mbar_wait_fast(tempty0 + 8 * ab, (use & 1) ^ 1, abort_flag, p.err, 2)) { give_up(); break; }
                asm volatile("fence.acq_rel.cluster;" ::: "memory");      // half of the arrivals came from the peer
                tc_fence_after();
                if (p.starve) {      // self-test: nothing was copied, so that this wait runs out
                    mbar_wait_fast(full0, 0, abort_flag, p.err, 3, 64u);
                    give_up();
                    break;
                }
                if (!mma_tile_d6<true>(tmem + ab * kMaxBN, p.kb_total, stage, phase, full0, empty0, desc_hi, ring >> 4, kPairStageBytes >> 4, w_bytes >> 4, p.idesc, abort_flag,
                                       p.err)) {
                    give_up();
                    break;
                }
                umma_commit_pair(tfull0 + 8 * ab);
            }
        }
    } else {
        const int q = warp & 3, half = (warp - 2) >> 2;
        const uint32_t stage_out = ring + kPairStages * kPairStageBytes + (warp - 2) * kPairOutBytes;
        pdl_wait();
        int it = 0;
        for (int tile = first; tile < total; tile += step, ++it) {
            int tc, tt;
            pair_tile(p, tile, tc, tt);
            const uint32_t ab = it & 1, use = it >> 1;
            const int n_warp = (tc * 2 + static_cast<int>(rank)) * kBM + q * 32;
            float cs[4], b[4];      // of channels 8 k + lane / 4, or of channel lane
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int n = n_warp + (p.vec ? 8 * k + (lane >> 2) : lane);
                cs[k] = n < p.n ? p.channel_scale[n] : 0.f;
                b[k] = p.bias && n < p.n ? p.bias[n] : 0.f;
            }
            float scales[kMaxBN / 64];      // of the tokens of this warp's groups, a lane one of each
#pragma unroll
            for (int g = 0; g < kMaxBN / 64; ++g) {
                const int c = half * 32 + 64 * g + lane;
                const int64_t m = static_cast<int64_t>(tt) * p.bn + c;
                scales[g] = c < p.bn && m < p.rows ? p.token_scale[m] : 0.f;
            }
            if (!mbar_wait(tfull0 + 8 * ab, use & 1, abort_flag, p.err, 4)) {
                if (lane == 0) give_up();
                break;
            }
            tc_fence_after();
            const uint32_t t_row = tmem + ab * kMaxBN + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll
            for (int g = 0; g < kMaxBN / 64; ++g) {
                const int c = half * 32 + 64 * g;
                if (c >= p.bn) break;
                const int64_t m = static_cast<int64_t>(tt) * p.bn + c;
                if (m >= p.rows) break;
                const int tokens = static_cast<int>(min(static_cast<int64_t>(min(32, p.bn - c)), p.rows - m));
                if (sizeof(O) == 2 && p.vec) {
                    if constexpr (sizeof(O) == 2) {
                        uint32_t r[2][16];      // [channels 16 h ..][4 j + 2 i + s]: channel lane / 4 + 8 i, token 8 j + 2 (lane & 3) + s
                        tmem_ld_16x256<4>(t_row + c, r[0]);
                        tmem_ld_16x256<4>(t_row + c + (16u << 16), r[1]);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float s0 = __shfl_sync(0xffffffffu, scales[g], 8 * j + 2 * (lane & 3)), s1 = __shfl_sync(0xffffffffu, scales[g], 8 * j + 2 * (lane & 3) + 1);
                            uint32_t v[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) {      // channels 8 k + lane / 4
                                const uint32_t *a = r[k >> 1] + 4 * j + 2 * (k & 1);
                                v[k] = pack_results(scaled(static_cast<int32_t>(a[0]), s0, cs[k], b[k]), scaled(static_cast<int32_t>(a[1]), s1, cs[k], b[k]), O{});
                            }
                            const int token = 8 * j + (lane & 7);      // 64 bytes each; the pieces of neighbours change places, for the banks
                            store_matrices_transposed(stage_out + token * 64 + (((lane >> 3) ^ (token >> 1)) & 3) * 16, v);
                        }
                        __syncwarp();
                        O *o = out + (m + (lane >> 2)) * p.n + n_warp + (lane & 3) * 8;
                        const bool mine = n_warp + (lane & 3) * 8 < p.n;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int token = 8 * i + (lane >> 2);
                            uint4 v;
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                         : "r"(stage_out + token * 64 + (((lane & 3) ^ (token >> 1)) & 3) * 16) : "memory");
                            if (mine && token < tokens) *reinterpret_cast<uint4 *>(o) = v;
                            o += 8 * static_cast<int64_t>(p.n);
                        }
                        __syncwarp();
                    }
                } else {
                    uint32_t r[32];
                    tmem_ld32(t_row + c, r);
                    O *o = out + m * p.n + n_warp + lane;
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float s = __shfl_sync(0xffffffffu, scales[g], j);
                        if (n_warp + lane < p.n && j < tokens) *o = from_float<O>(scaled(static_cast<int32_t>(r[j]), s, cs[0], b[0]));
                        o += p.n;
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_relaxed(mapa_rank(tempty0 + 8 * ab, 0));
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    // No copy may land in memory that is given back (a pair's copies report to the first CTA).
    if (*abort_flag && rank == 0 && (warp == 0 || warp == kPairEpiWarps + 2) && lane < 2 && !p.starve) drain_stages(full0, kPairStages, stage, phase, lane, 2);
    __syncwarp();
    cluster_sync_all();                         // no signal may reach a CTA that has left
    tc_fence_after();
    if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

template <typename O>
cudaError_t kernel_init(int device) {
    static PerDeviceInit once;
    return once.run(device, [] {
        const cudaError_t e = cudaFuncSetAttribute(token_fc_kernel<O>, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
        return e != cudaSuccess ? e : cudaFuncSetAttribute(token_fc_pair_kernel<O>, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
    });
}

constexpr uint32_t kSignedBytes = (2u << 4) | (1u << 7) | (1u << 10);      // s32 sums of s8 x s8

template <typename K, typename... Args>
cudaError_t launch_clusters(K kernel, unsigned grid, unsigned threads, size_t smem, unsigned cluster, cudaStream_t stream, const Args &...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Token tiles of at most `most` tokens, as even as multiples of `unit` allow.
void token_tiles(int32_t rows, int32_t most, int32_t unit, int32_t *tiles, int32_t *bn) {
    *tiles = (rows + most - 1) / most;
    *bn = ((rows + *tiles - 1) / *tiles + unit - 1) / unit * unit;
}

template <typename O>
cudaError_t launch_tc(enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs) {
    TokenState &t = *op->token;
    enn_b200_context *ctx = op->ctx;
    const TokenFcParams &f = t.fc;
    const cudaError_t e = kernel_init<O>(ctx->device);
    if (e != cudaSuccess) return e;
    const int32_t kb_total = (f.k + kBK - 1) / kBK;
    const float *token_scale = static_cast<const float *>(ins[1]);
    O *out = static_cast<O *>(outs[0]);
    const int32_t starve = t.fc.starve_next;
    t.fc.starve_next = false;
    CUtensorMap map_q;
    const auto encode = [&](int32_t box) {
        return encode_2d(ctx, &map_q, ins[0], static_cast<uint64_t>(f.k), static_cast<uint64_t>(rows), static_cast<uint64_t>(f.in_pitch), kBK, static_cast<uint32_t>(box));
    };
    const int pairs = t.sms / 2;

    // Large products: pairs of CTAs.  The width of the token tiles is the one whose rounds over the device take least, a tile costing its
    // columns and about as much as kTileCost more.
    PairCall c2{};
    c2.tiles_c = (f.n + 2 * kBM - 1) / (2 * kBM);
    int64_t least = INT64_MAX, tiles2 = 0;
    for (int32_t bn = kMaxBN; bn >= 64 && pairs > 0; bn -= 32) {
        const int32_t tiles_t = (rows + bn - 1) / bn;
        const int64_t tiles = static_cast<int64_t>(c2.tiles_c) * tiles_t, cost = (tiles + pairs - 1) / pairs * (bn + kTileCost);
        if (cost < least) {
            least = cost;
            tiles2 = tiles;
            c2.tiles_t = tiles_t;
            c2.bn = bn;
        }
    }
    if (rows >= kPairRows && pairs > 0 && tiles2 * 2 >= pairs) {
        c2.rows = rows; c2.n = f.n; c2.kb_total = kb_total;
        c2.band = std::min(16, c2.tiles_c);
        c2.idesc = kSignedBytes | (static_cast<uint32_t>(c2.bn >> 3) << 17) | (static_cast<uint32_t>(2 * kBM >> 4) << 24);
        c2.token_scale = token_scale; c2.channel_scale = f.channel_scale; c2.bias = f.bias;
        c2.err = f.err_dev; c2.starve = starve;
        c2.vec = sizeof(O) == 2 && f.n % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
        if (!encode(c2.bn / 2)) return cudaErrorInvalidValue;
        return launch_clusters(token_fc_pair_kernel<O>, static_cast<unsigned>(2 * std::min<int64_t>(tiles2, pairs)), kPairThreads, 1024 + kPairStages * kPairStageBytes + kPairEpiWarps * kPairOutBytes, 2, ctx->stream,
                               f.map_w, map_q, c2, out);
    }

    // (CTAs of clusters wait for one another, so that none may wait for tensor memory that a CTA of another cluster holds.  A split leaves two
    // stages at least, 54 KB with more than 64 tokens: an SM holds four such CTAs at most, which have 128 of its 512 columns each.)
    // Two CTAs share an SM: while one waits for its first tiles or stores its results, the other keeps the SM busy.
    TcCall c{};
    c.rows = rows; c.n = f.n; c.kb_total = kb_total;
    token_tiles(rows, kTcTokens, 16, &c.m_tiles, &c.bn);
    const int64_t tiles = static_cast<int64_t>((f.n + kChannels - 1) / kChannels) * c.m_tiles;
    c.splits = 1;
    while (c.splits < kMaxSplits && tiles * c.splits * 2 <= 2 * t.sms && kb_total >= 4 * c.splits) c.splits *= 2;
    const int stage_bytes = (kChannels + c.bn) * kBK;
    c.stages = std::min({111 * 1024 / stage_bytes, (kb_total + c.splits - 1) / c.splits, kMaxStages});
    const size_t smem = 1024 + static_cast<size_t>(std::max(c.stages * stage_bytes, c.bn * kChannels * 4));
    c.tmem_cols = 32;
    while (c.tmem_cols < static_cast<uint32_t>(c.bn)) c.tmem_cols *= 2;
    c.idesc = kSignedBytes | (static_cast<uint32_t>(c.bn >> 3) << 17) | (static_cast<uint32_t>(kChannels >> 4) << 24);
    c.token_scale = token_scale; c.channel_scale = f.channel_scale; c.bias = f.bias;
    c.err = f.err_dev; c.starve = starve;
    c.vec = f.n % 4 == 0 && reinterpret_cast<uintptr_t>(out) % (4 * sizeof(O)) == 0;
    if (!encode(c.bn)) return cudaErrorInvalidValue;
    return launch_clusters(token_fc_kernel<O>, static_cast<unsigned>(tiles * c.splits), kTcThreads, smem, static_cast<unsigned>(c.splits), ctx->stream, f.map_w, map_q, c, out);
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

__global__ void pad_rows_kernel(const int8_t *src, int32_t width, int64_t pitch, int64_t total, int8_t *dst) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t r = i / pitch, c = i - r * pitch;
        dst[i] = c < width ? src[r * width + c] : int8_t{0};
    }
}

}  // namespace

// Dense rows into rows `pitch` bytes apart, zeros beyond the width.
cudaError_t launch_pad_rows(const void *src, int32_t width, int32_t height, int64_t pitch, void *dst, cudaStream_t stream) {
    const int64_t total = pitch * height;
    pad_rows_kernel<<<static_cast<unsigned>(std::min<int64_t>(total / 2048 + 1, 4096)), 256, 0, stream>>>(static_cast<const int8_t *>(src), width, pitch, total,
                                                                                                           static_cast<int8_t *>(dst));
    return cudaGetLastError();
}

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
    switch (op->token->out_dtype) {
        case ENN_B200_F32: return launch_typed<float>(op, rows, ins, outs);
        case ENN_B200_F16: return launch_typed<__half>(op, rows, ins, outs);
        case ENN_B200_BF16: return launch_typed<__nv_bfloat16>(op, rows, ins, outs);
    }
    return cudaErrorInvalidValue;
}

}  // namespace enn_b200
