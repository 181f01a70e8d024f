// log_probs: log probabilities of given ids, entropy and the largest alternatives of rows of logits.
//
// Bound by reading the logits, which happens once: with k = scale * log2(e), m the running maximum and d = k (l - m), a thread keeps
//   S = sum 2^d   and   U = sum d 2^d,
// rescaled whenever m grows (S' = c S, U' = c (U + d S) with d = k (m - m'), c = 2^d).  Then
//   log p = scale (l - m) - ln S,   entropy = ln S - ln 2 U / S.
// The alternatives come from the same pass: a thread remembers where its largest logit was.  A value that n of the threads' maxima reach
// bounds the n-th largest logit from below, so that what is above it lies with those threads, and their logits alone are looked at again.
// A row is split over a cluster of up to eight CTAs where the rows alone do not occupy the device; the parts meet in the first CTA's
// shared memory, without atomics or workspace.  All orders are total (value, then index), so that results do not depend on timing.
// 2048x65536 f32 with one id and one alternative 106 us (5.1 TB/s), 93 us without both; 1x131072 8.1 us, half of it the search.  16-bit rows are bound by
// instructions (8 a logit, one of them 2^x, of which an SM does 16 a cycle): 2048x65536 bf16 48 us without alternatives (5.6 TB/s).
#include <math_constants.h>

#include <algorithm>
#include <type_traits>

#include "per_device.h"
#include "tc_common.cuh"
#include "token_ops.h"

namespace enn_b200 {
namespace {

constexpr int kMaxTop = ENN_B200_LOG_PROBS_MAX_TOP;
constexpr int kMaxSegments = 8;
constexpr int kChunk = 4;               // 16-byte pieces a thread works on at a time
constexpr int kDepth = 2;               // chunks a thread asks for ahead
constexpr int kCandidates = 1024;
// Threads of a CTA, and the CTAs an SM is to hold.  kLong; kShort for short rows that are more than the device holds CTAs of kLong, whose time is that of
// the reductions and of the search, one step after the other: more rows side by side (bf16 with five alternatives: 450x2000 9.0 us with kLong,
// 6.1 us so, 4000x2000 42 and 18 us, with 20: 450x8000 10.2 and 11.7 us, 1000x8000 16.4 and 14.3 us; below, 440x2000 6.9 us with kLong, 6.2 us with kShort,
// 440x8000 7.4 and 11.3 us).  kLongest where the stream is most of it (f32 with 20 alternatives, kLong and kLongest: 1000x24576 28.3 and 34.0 us,
// 800x40000 33.6 and 37.8 us, 600x49152 34.6 and 31.6 us, 2048x65536 118 and 109 us).  16-bit rows of these bytes have twice the logits and gain
// nothing (1000x98304 bf16 54 and 60 us, 2048x131072 bf16 126 and 128 us).
constexpr int kLongest = 512, kLong = 256, kShort = 64;
constexpr int kShortBytes = 16 << 10, kLongestBytes = 192 << 10;       // rows of up to, segments of at least
constexpr int blocks_of(int threads) { return threads == kLongest ? 2 : (threads == kLong ? 3 : 8); }
constexpr int kLookers = 8;             // threads that look at one thread's logits again
constexpr float kNothing = -1e4f;       // 2^-10000 is 0; keeps the products d 2^d away from infinity times 0
constexpr float kLowest = -3.402823466e38f;

// Order of the logits as unsigned integers: NaN above +inf, -0 equal to +0; the lower index first among equals.  0 is below all keys.
__device__ __forceinline__ uint64_t order_key(float v, int32_t index) {
    uint32_t b = __float_as_uint(v + 0.f);
    if (v != v) b = 0x7fffffffu;
    b = b & 0x80000000u ? ~b : b | 0x80000000u;
    return static_cast<uint64_t>(b) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ int32_t key_index(uint64_t key) { return static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key)); }
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t b = static_cast<uint32_t>(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

__device__ __forceinline__ float exp2_fast(float x) {      // two units in the last place; 0 below 2^-126
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {      // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// A segment [begin, end) of a row as 16-byte pieces at 16-byte addresses: piece g holds the logits begin - skip + g E .. + E, of which
// those outside the segment (in the first and the last piece) read as -inf and are not loaded.
template <typename T>
struct Segment {
    static constexpr int E = 16 / sizeof(T);
    const T *row;
    int32_t begin, end, skip, pieces;
    int32_t whole_begin, whole_end;      // the whole pieces
    __device__ __forceinline__ Segment(const T *r, int32_t b, int32_t e) : row(r), begin(b), end(e) {
        skip = static_cast<int32_t>((reinterpret_cast<uintptr_t>(r + b) & 15) / sizeof(T));
        pieces = e > b ? (e - b + skip + E - 1) / E : 0;
        whole_begin = skip ? 1 : 0;
        whole_end = e > b ? (e - b + skip) / E : 0;
    }
    // Pieces [g, g + n) lie in the segment as a whole.
    __device__ __forceinline__ bool inside(int32_t g, int32_t n) const { return g + n <= whole_end && g >= whole_begin; }
    __device__ __forceinline__ int32_t first(int32_t g) const { return begin - skip + g * E; }
    __device__ __forceinline__ bool whole(int32_t g) const { return g >= whole_begin && g < whole_end; }
    __device__ __forceinline__ uint4 load(int32_t g) const {
        uint4 v;
        if (whole(g)) {
            asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(row + first(g)));
        } else {
            T t[E];
#pragma unroll
            for (int i = 0; i < E; ++i) t[i] = holds(first(g) + i) ? row[first(g) + i] : from_float<T>(-CUDART_INF_F);
            __builtin_memcpy(&v, t, 16);
        }
        return v;
    }
    // The key of logit i of piece g, 0 outside the segment.
    __device__ __forceinline__ uint64_t key(int32_t g, int i, float v) const { return holds(first(g) + i) ? order_key(v, first(g) + i) : 0; }
    __device__ __forceinline__ bool holds(int32_t index) const { return index >= begin && index < end; }
};

__device__ __forceinline__ void unpack(uint4 v, float (&x)[4], float) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <typename T> __device__ __forceinline__ void unpack(uint4 v, float (&x)[8], T) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2(w[i], T{});
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
template <typename T> __device__ __forceinline__ uint4 nothing() {      // a piece of -inf
    const float2 f = make_float2(-CUDART_INF_F, -CUDART_INF_F);
    if constexpr (sizeof(T) == 4) return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
    T t[2] = {from_float<T>(f.x), from_float<T>(f.y)};
    uint32_t w;
    __builtin_memcpy(&w, t, 4);
    return make_uint4(w, w, w, w);
}

// Largest of a few pieces; NaN is passed over.
template <int N> __device__ __forceinline__ float largest_of(const uint4 (&v)[N], float) {
    float m = -CUDART_INF_F;
#pragma unroll
    for (int c = 0; c < N; ++c) {
        float x[4];
        unpack(v[c], x, float{});
        m = fmaxf(m, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    }
    return m;
}
template <typename T2, int N> __device__ __forceinline__ float largest_of2(const uint4 (&v)[N]) {
    T2 m;
#pragma unroll
    for (int c = 0; c < N; ++c) {
        T2 t[4];
        __builtin_memcpy(t, &v[c], 16);
        const T2 of = __hmax2(__hmax2(t[0], t[1]), __hmax2(t[2], t[3]));
        m = c ? __hmax2(m, of) : of;
    }
    return fmaxf(to_float(m.x), to_float(m.y));
}
template <int N> __device__ __forceinline__ float largest_of(const uint4 (&v)[N], __half) { return largest_of2<__half2>(v); }
template <int N> __device__ __forceinline__ float largest_of(const uint4 (&v)[N], __nv_bfloat16) { return largest_of2<__nv_bfloat162>(v); }

// Two floats in one register pair, for the instructions that work on both.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
    return p;
}
__device__ __forceinline__ float2 unpair(uint64_t p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

struct Stats {
    float m, s, u;
    __device__ __forceinline__ void rescale(float to, float k) {
        const float d = fmaxf((m - to) * k, kNothing), c = exp2_fast(d);
        u = c * fmaf(d, s, u);
        s *= c;
        m = to;
    }
};

__device__ __forceinline__ uint64_t warp_largest(uint64_t key) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(key >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(key >> 32) == hi ? static_cast<uint32_t>(key) : 0u);
    return static_cast<uint64_t>(hi) << 32 | lo;
}

// The `n` largest keys of up to 32 lists in descending order, 0 past their ends; one warp, lane i walks list i.
__device__ __forceinline__ void take_largest(const uint64_t *lists, int n_lists, int length, int stride, int n, uint64_t *out) {
    const int lane = threadIdx.x & 31;
    int at = 0;
    uint64_t head = lane < n_lists && length ? lists[lane * stride] : 0;
    for (int i = 0; i < n; ++i) {
        const uint64_t key = warp_largest(head);
        if (lane == 0) out[i] = key;
        if (key && head == key) head = ++at < length ? lists[lane * stride + at] : 0;
    }
}

template <int kThreads>
struct Shared {
    static constexpr int kWarps = kThreads / 32;
    float part[3][kWarps];
    uint64_t of_warp[kWarps];
    uint64_t firsts[kWarps * (kMaxTop / kWarps + 2)], bound;
    int32_t n_lookups;
    int32_t lookups[kThreads];                  // threads whose logits are looked at again
    uint64_t candidates[kCandidates];
    int32_t n_candidates;
    uint64_t sorted[kMaxTop];                   // the largest of this segment
    Stats stats[kMaxSegments];                  // of the first CTA: what the segments found
    uint64_t merged[kMaxSegments][kMaxTop];
};

template <typename V, typename F>
__device__ __forceinline__ V warp_join(V v, F join) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Round by round over the whole segment: for rows with NaN or +inf, and where more candidates turn up than there is room for.
template <int kThreads, typename T>
__device__ __noinline__ void largest_by_rounds(const Segment<T> &seg, int top, Shared<kThreads> &sh) {
    constexpr int kWarps = kThreads / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t below = ~0ull;
    for (int r = 0; r < top; ++r) {
        uint64_t best = 0;
        for (int32_t g = threadIdx.x; g < seg.pieces; g += kThreads) {
            float x[Segment<T>::E];
            unpack(seg.load(g), x, T{});
            for (int i = 0; i < Segment<T>::E; ++i) {
                const uint64_t k = seg.key(g, i, x[i]);
                if (k < below && k > best) best = k;
            }
        }
        best = warp_join(best, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
        __syncthreads();
        if (lane == 0) sh.of_warp[warp] = best;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) best = sh.of_warp[w] > best ? sh.of_warp[w] : best;
        if (threadIdx.x == 0) sh.sorted[r] = best;
        below = best;
    }
    __syncthreads();
}

// The logits of the threads whose maximum reaches `least`, as far as they reach it themselves, into sh.candidates.  `mine`: a key of the
// thread's maximum.  Returns their number, which may be above what there is room for.
template <int kThreads, typename T>
__device__ __forceinline__ int collect(const Segment<T> &seg, uint64_t mine, uint64_t least, Shared<kThreads> &sh) {
    if (threadIdx.x == 0) sh.n_candidates = sh.n_lookups = 0;
    __syncthreads();
    if (mine && mine >= least) sh.lookups[atomicAdd(&sh.n_lookups, 1)] = threadIdx.x;
    __syncthreads();
    const float reach = least ? key_value(least) : -CUDART_INF_F;
    const int n = sh.n_lookups;
    for (int w = threadIdx.x / kLookers; w < n; w += kThreads / kLookers)      // a few threads look at the logits of each of them
        for (int32_t g = sh.lookups[w] + kThreads * static_cast<int32_t>(threadIdx.x % kLookers); g < seg.pieces; g += kThreads * kLookers) {
            float x[Segment<T>::E];
            unpack(seg.load(g), x, T{});
#pragma unroll
            for (int i = 0; i < Segment<T>::E; ++i)
                if (x[i] >= reach) {
                    const uint64_t k = seg.key(g, i, x[i]);
                    if (k && k >= least) {
                        const int32_t slot = atomicAdd(&sh.n_candidates, 1);
                        if (slot < kCandidates) sh.candidates[slot] = k;
                    }
                }
        }
    __syncthreads();
    return sh.n_candidates;
}

// A key that `top` of the keys `mine` of the threads reach, 0 if fewer of them have one: the top-th largest among the first few of every
// warp, two more than would do, so that hardly more threads than `top` reach it.
template <int kThreads>
__device__ __forceinline__ uint64_t reached_by(uint64_t mine, int top, Shared<kThreads> &sh) {
    constexpr int kWarps = kThreads / 32;
    const int rounds = min(top, (top + kWarps - 1) / kWarps + 2), n = rounds * kWarps;
    __syncthreads();
    for (int r = 0; r < rounds; ++r) {
        const uint64_t found = warp_largest(mine);
        const uint32_t holders = __ballot_sync(0xffffffffu, mine == found);
        if (static_cast<int>(threadIdx.x & 31) == __ffs(holders) - 1) {      // equal ones one after the other
            sh.firsts[r * kWarps + (threadIdx.x >> 5)] = found;
            mine = 0;
        }
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < n) {      // at most 64 keys, and never more than threads
        const uint64_t k = sh.firsts[threadIdx.x];
        int place = 0;
        for (int j = 0; j < n; ++j) {
            const uint64_t other = sh.firsts[j];
            place += other > k || (other == k && j < static_cast<int>(threadIdx.x));
        }
        if (place == top - 1) sh.bound = k;
    }
    __syncthreads();
    return sh.bound;
}

// sh.sorted[0 .. top): the largest keys of a segment without NaN.  `best`: the thread's largest logit.
template <int kThreads, typename T>
__device__ __forceinline__ void largest_of_segment(const Segment<T> &seg, float best, int top, Shared<kThreads> &sh) {
    const bool has = static_cast<int32_t>(threadIdx.x) < seg.pieces;
    // By value first: all that equal the bound are candidates.
    uint64_t mine = has ? order_key(best, -1) : 0;
    uint64_t least = reached_by(mine, top, sh);
    int n = collect(seg, mine, least & 0xffffffff00000000ull, sh);
    if (n > kCandidates) {
        // Many equal logits (a vocabulary with few left and the others at one value): the threads' maxima with their indexes.
        mine = 0;
        for (int32_t g = threadIdx.x; g < seg.pieces && !mine; g += kThreads) {
            float x[Segment<T>::E];
            unpack(seg.load(g), x, T{});
#pragma unroll
            for (int i = Segment<T>::E - 1; i >= 0; --i)
                if (x[i] == best && seg.holds(seg.first(g) + i)) mine = order_key(best, seg.first(g) + i);
        }
        least = reached_by(mine, top, sh);
        n = collect(seg, mine, least, sh);
        if (n > kCandidates) {
            largest_by_rounds(seg, top, sh);
            return;
        }
    }
    if (threadIdx.x < top) sh.sorted[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {      // its place is the number of larger ones
        const uint64_t k = sh.candidates[i];
        int place = 0;
        for (int j = 0; j < n; ++j) place += sh.candidates[j] > k;
        if (place < top) sh.sorted[place] = k;
    }
    __syncthreads();
}

// Grid: rows x segments, the segments of a row being a cluster.  Where rows have one segment a CTA takes several of them, and the copies
// of the next row's first chunks are under way while the alternatives of this one are sorted out.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, blocks_of(kThreads)) log_probs_kernel(LogProbsParams p, int32_t rows, int32_t seg_size, const T *logits, const int32_t *ids, float *given,
                                                                      float *entropy, int32_t *top_ids, float *top) {
    extern __shared__ __align__(16) uint8_t ring[];      // [kDepth][kChunk][kThreads] pieces: a thread reads what it copied itself
    __shared__ Shared<kThreads> sh;
    constexpr int kWarps = kThreads / 32;
    constexpr int E = Segment<T>::E;
    constexpr int kStep = kThreads * kChunk;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int segs = gridDim.y, rank = blockIdx.y;
    if (segs > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // waited for before the first CTA's memory is written
    const auto segment = [&](int64_t t) { return Segment<T>(logits + t * p.pitch, rank * seg_size, min(p.vocab, (rank + 1) * seg_size)); };
    const float k = p.scale * 1.4426950408889634f;
    const uint32_t mine0 = smem_u32(ring) + threadIdx.x * 16;
    constexpr uint32_t kPiece = kThreads * 16, kSlot = kChunk * kPiece;      // bytes from piece to piece of a thread, from chunk to chunk
    pdl_wait();
    pdl_trigger();

    // What is copied next: piece g_next (of thread 0) of row t_next.
    int64_t t_next = blockIdx.x;
    int32_t g_next = 0;
    Segment<T> ahead = segment(min(t_next, static_cast<int64_t>(rows) - 1));
    const T *from = ahead.row + ahead.first(threadIdx.x);
    const auto fetch = [&](uint32_t at) {
        const auto copy = [&](int c) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + c * kPiece), "l"(from + c * (kThreads * E)) : "memory"); };
        if (t_next < rows) {
            if (ahead.inside(g_next, kStep)) {      // of every thread: no tests in the middle of a row
#pragma unroll
                for (int c = 0; c < kChunk; ++c) copy(c);
            } else {
#pragma unroll
                for (int c = 0; c < kChunk; ++c)
                    if (ahead.whole(g_next + c * kThreads + static_cast<int32_t>(threadIdx.x))) copy(c);
            }
            g_next += kStep;
            from += kStep * E;
            if (g_next >= ahead.pieces) {
                g_next = 0;
                t_next += gridDim.x;
                if (t_next < rows) {
                    ahead = segment(t_next);
                    from = ahead.row + ahead.first(threadIdx.x);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int s = 0; s < kDepth; ++s) fetch(mine0 + s * kSlot);
    uint32_t at = mine0;      // the chunk that is worked on
    bool careful = false;

    for (int64_t t = blockIdx.x; t < rows; t += gridDim.x) {
        const Segment<T> seg = segment(t);
        Stats a{kLowest, 0.f, 0.f};
        float best = -CUDART_INF_F;
        for (int32_t g0 = 0; g0 < seg.pieces; g0 += kStep) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
            uint4 raw[kChunk];
            const auto take = [&](int c) {
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(raw[c].x), "=r"(raw[c].y), "=r"(raw[c].z), "=r"(raw[c].w) : "r"(at + c * kPiece) : "memory");
            };
            if (seg.inside(g0, kStep)) {
#pragma unroll
                for (int c = 0; c < kChunk; ++c) take(c);
            } else {
#pragma unroll
                for (int c = 0; c < kChunk; ++c) {
                    const int32_t g = g0 + c * kThreads + static_cast<int32_t>(threadIdx.x);
                    raw[c] = nothing<T>();
                    if (seg.whole(g)) take(c);
                    else if (g < seg.pieces) raw[c] = seg.load(g);
                }
            }
            fetch(at);
            at = at == mine0 + (kDepth - 1) * kSlot ? mine0 : at + kSlot;
            const float largest = largest_of(raw, T{});
            best = fmaxf(best, largest);
            // m is the maximum, and not a value near it: the largest logit then counts as exactly 1 and 0, and log p and the entropy of a row
            // that is all but certain are not what is left of two larger numbers.  (Moving m only by factors of 2^20 was no quicker.)
            if (largest > a.m) a.rescale(largest, k);
            // Two at a time.  What is ruled out makes 0 times -inf of d 2^d, seen in U: the chunk is then done again with care, as are those
            // after it (a vocabulary is ruled out all over).
            const uint64_t minus_m = pair(-a.m, -a.m), k2 = pair(k, k);
            const auto sum = [&](auto limit) {
                uint64_t s2 = 0, u2 = 0;      // of the chunk: no long chain of additions
#pragma unroll
                for (int c = 0; c < kChunk; ++c) {
                    float x[E];
                    unpack(raw[c], x, T{});
#pragma unroll
                    for (int i = 0; i < E; i += 2) {
                        const uint64_t d2 = limit(mul2(add2(pair(x[i], x[i + 1]), minus_m), k2));
                        const float2 d = unpair(d2);
                        const uint64_t e2 = pair(exp2_fast(d.x), exp2_fast(d.y));
                        s2 = add2(s2, e2);
                        u2 = fma2(d2, e2, u2);
                    }
                }
                const float2 s = unpair(s2), u = unpair(u2);
                return make_float2(s.x + s.y, u.x + u.y);
            };
            float2 su;
            if (!careful) {
                su = sum([](uint64_t d2) { return d2; });
                careful = su.y != su.y;
            }
            if (careful)
                su = sum([](uint64_t d2) {
                    const float2 d = unpair(d2);
                    return pair(max_nan(d.x, kNothing), max_nan(d.y, kNothing));
                });
            a.s += su.x;
            a.u += su.y;
        }

        // The statistics of the segment, the same in every thread.
        float m = warp_join(a.m, [](float x, float y) { return fmaxf(x, y); });
        if (lane == 0) sh.part[0][warp] = m;
        __syncthreads();
        m = warp_join(sh.part[0][lane % kWarps], [](float x, float y) { return fmaxf(x, y); });
        a.rescale(m, k);
        const auto plus = [](float x, float y) { return x + y; };
        a.s = warp_join(a.s, plus);
        a.u = warp_join(a.u, plus);
        if (lane == 0) {
            sh.part[1][warp] = a.s;
            sh.part[2][warp] = a.u;
        }
        __syncthreads();
        a.s = warp_join(lane < kWarps ? sh.part[1][lane] : 0.f, plus);
        a.u = warp_join(lane < kWarps ? sh.part[2][lane] : 0.f, plus);

        if (p.top) {
            if (a.s != a.s) {
                largest_by_rounds(seg, p.top, sh);
            } else {
                largest_of_segment(seg, best, p.top, sh);
            }
        }
        if (segs > 1) {
            asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
            if (threadIdx.x < p.top) {
                const uint64_t key = sh.sorted[threadIdx.x];
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_rank(smem_u32(&sh.merged[rank][threadIdx.x]), 0)), "l"(key) : "memory");
            }
            if (threadIdx.x == 0) {
                const uint32_t at = mapa_rank(smem_u32(&sh.stats[rank]), 0);
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(a.m) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 4), "f"(a.s) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 8), "f"(a.u) : "memory");
            }
            cluster_sync_all();
            if (rank != 0) return;      // a cluster has one row
            a = sh.stats[0];
            for (int s = 1; s < segs; ++s) {
                Stats b = sh.stats[s];
                const float to = fmaxf(a.m, b.m);
                a.rescale(to, k);
                b.rescale(to, k);
                a.s += b.s;
                a.u += b.u;
            }
            if (warp == 0 && p.top) take_largest(&sh.merged[0][0], segs, p.top, kMaxTop, p.top, sh.sorted);
            __syncthreads();
        }
        // A row that is ruled out as a whole has no exponentials at all.
        const float log_s = a.s == 0.f ? CUDART_NAN_F : logf(a.s);
        const auto log_p = [&](float l) { return (l - a.m) * p.scale - log_s; };
        if (threadIdx.x == 0) entropy[t] = log_s - 0.69314718055994531f * (a.u / a.s);
        for (int j = threadIdx.x; j < p.given; j += kThreads) {
            const int32_t id = ids[t * p.given + j];
            given[t * p.given + j] = id < 0 ? 0.f : (id >= p.vocab ? CUDART_NAN_F : log_p(to_float(seg.row[id])));
        }
        if (threadIdx.x < p.top) {
            const uint64_t key = sh.sorted[threadIdx.x];
            top_ids[t * p.top + threadIdx.x] = key_index(key);
            top[t * p.top + threadIdx.x] = log_p(key_value(key));
        }
    }
}

template <typename T>
cudaError_t launch_typed(const enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs) {
    const LogProbsParams &p = op->token->log_probs;
    int o = 0;
    const int32_t *ids = p.given ? static_cast<const int32_t *>(ins[1]) : nullptr;
    float *given = p.given ? static_cast<float *>(outs[o++]) : nullptr;
    float *entropy = static_cast<float *>(outs[o++]);
    int32_t *top_ids = p.top ? static_cast<int32_t *>(outs[o++]) : nullptr;
    float *top = p.top ? static_cast<float *>(outs[o++]) : nullptr;
    // Segments while the device has room for them and a segment keeps a chunk for every thread.
    const int64_t sms = op->token->sms;
    int segs = 1;
    while (segs < kMaxSegments && static_cast<int64_t>(rows) * segs * 2 <= blocks_of(kLong) * sms && p.vocab / (segs * 2) >= 4096) segs *= 2;
    const int32_t seg_size = (p.vocab + segs - 1) / segs;
    const auto run = [&](auto threads) {
        constexpr int kThreads = decltype(threads)::value, kRing = kDepth * kChunk * kThreads * 16;
        constexpr auto kernel = log_probs_kernel<T, kThreads>;
        static PerDeviceInit once;
        const cudaError_t e = once.run(op->ctx->device, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing); });
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(static_cast<unsigned>(segs > 1 ? rows : std::min<int64_t>(rows, blocks_of(kThreads) * sms)), static_cast<unsigned>(segs));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = kRing;
        cfg.stream = op->ctx->stream;
        cudaLaunchAttribute attr[2] = {};
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = attr[1].val.clusterDim.z = 1;
        attr[1].val.clusterDim.y = static_cast<unsigned>(segs);
        cfg.attrs = attr;
        cfg.numAttrs = segs > 1 ? 2 : 1;
        return cudaLaunchKernelEx(&cfg, kernel, p, rows, seg_size, static_cast<const T *>(ins[0]), ids, given, entropy, top_ids, top);
    };
    if (rows > blocks_of(kLong) * sms && p.vocab * static_cast<int64_t>(sizeof(T)) <= kShortBytes) return run(std::integral_constant<int, kShort>{});
    if (seg_size * static_cast<int64_t>(sizeof(T)) >= kLongestBytes) return run(std::integral_constant<int, kLongest>{});
    return run(std::integral_constant<int, kLong>{});
}

}  // namespace

cudaError_t log_probs_launch(const enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs) {
    switch (op->token->in_dtype) {
        case ENN_B200_F32: return launch_typed<float>(op, rows, ins, outs);
        case ENN_B200_F16: return launch_typed<__half>(op, rows, ins, outs);
        case ENN_B200_BF16: return launch_typed<__nv_bfloat16>(op, rows, ins, outs);
    }
    return cudaErrorInvalidValue;
}

}  // namespace enn_b200
