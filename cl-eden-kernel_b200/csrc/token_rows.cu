// token_norm and token_gate: row-wise operators around the 8-bit products of a block.
//
// Both are bound by memory: a row is read once, stays in registers as floats while its statistics are reduced, and is written once.
// A row belongs to a warp (up to 1024 channels), a CTA, or for quantised gates a cluster; a thread holds up to eight groups of eight
// neighbouring channels, 16 bytes of a 16-bit type.  Constant vectors come from L1, which they share with nothing: rows are loaded and
// stored past it (those of gates between lines, which have no such vectors, through it).  Measured in queued passes: gates 8192x12288
// bf16 92 us (6.6 TB/s), norms on both sides of a block with the stream 8192x5120 bf16 65 us (5.2 TB/s; half of the issue slots busy, 28
// instructions a channel, the rest the latency of three reductions a row).
#include <algorithm>
#include <type_traits>

#include "per_device.h"
#include "tc_common.cuh"
#include "token_ops.h"

namespace enn_b200 {
namespace {

constexpr int kGroup = 8;           // channels a thread handles together

__device__ __forceinline__ uint4 ld_stream(const void *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
// Zeros where `on` does not hold, without a branch that the loads after it would have to wait for.  It is for lines that two groups
// share, so L1 keeps them (4096x4099, of gates and values: 26.2 us, 27.4 us where it does not).
__device__ __forceinline__ uint4 ld_if(const void *p, bool on) {
    uint4 v;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t"
        "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
        "@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
        : "l"(p), "r"(static_cast<uint32_t>(on))
        : "memory");
    return v;
}
// Eight channels as they lie in memory.
template <typename T> struct Raw { uint4 v[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ Raw<T> ld8(const T *p) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) r.v[i] = ld_stream(reinterpret_cast<const uint4 *>(p) + i);
    return r;
}
__device__ __forceinline__ void widen(const Raw<float> &r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f[4 * i] = __uint_as_float(r.v[i].x); f[4 * i + 1] = __uint_as_float(r.v[i].y);
        f[4 * i + 2] = __uint_as_float(r.v[i].z); f[4 * i + 3] = __uint_as_float(r.v[i].w);
    }
}
__device__ __forceinline__ float2 widen2(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
__device__ __forceinline__ float2 widen2(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <typename T> __device__ __forceinline__ void widen(const Raw<T> &r, float (&f)[8]) {
    const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = widen2(w[i], T{});
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ void st8(float *p, const float (&f)[8]) {
    __stcs(reinterpret_cast<float4 *>(p), make_float4(f[0], f[1], f[2], f[3]));
    __stcs(reinterpret_cast<float4 *>(p) + 1, make_float4(f[4], f[5], f[6], f[7]));
}
template <typename T> __device__ __forceinline__ void st8(T *p, const float (&f)[8]) {
    __stcs(reinterpret_cast<uint4 *>(p), make_uint4(pack2(f[0], f[1], T{}), pack2(f[2], f[3], T{}), pack2(f[4], f[5], T{}), pack2(f[6], f[7], T{})));
}
__device__ __forceinline__ uint32_t pack4_s8(const float *f, float inv) {
    uint32_t hi, d;
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(hi) : "r"(quantise(f[3], inv)), "r"(quantise(f[2], inv)));
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(quantise(f[1], inv)), "r"(quantise(f[0], inv)), "r"(hi));
    return d;
}

// Lines that a group which begins inside one touches.
template <typename T> constexpr int kLinesOf = static_cast<int>(sizeof(T)) / 2 + 1;
// The part of a row that a group of `nt` threads holds: channels [0, n) of a segment in groups of eight neighbours, NV per thread.
// LINES: every group is whole and lies on 16-byte lines (n, every address and every pitch allow it).  Else the groups are shifted
// by `skip` channels, so that they lie on the lines of the tensor they were laid out for; the first and the last may reach over the
// row's ends, where nothing outside counts or is written; a tensor with other lines is read from two of its own and written channel by channel.
template <int NV, bool LINES>
struct Row {
    int n, tid, nt, skip;
    int low, high;      // channels, counted from the row's first, that are the tensor's: those of its neighbours count
    __device__ __forceinline__ int at(int v, int j = 0) const { return (v * nt + tid) * kGroup + j - (LINES ? 0 : skip); }
    __device__ __forceinline__ bool any(int v) const { return at(v) < n; }
    __device__ __forceinline__ bool whole(int v) const { return LINES ? any(v) : at(v) >= 0 && at(v) + kGroup <= n; }
    __device__ __forceinline__ bool inside(int v, int j) const { return LINES ? any(v) : at(v, j) >= 0 && at(v, j) < n; }
    // The group's line may be read as a whole.
    __device__ __forceinline__ bool readable(int v) const { return LINES ? any(v) : any(v) && at(v) >= low && at(v) + kGroup <= high; }
    // Nothing counts outside the row.
    __device__ __forceinline__ void clear_outside(int v, float (&f)[8]) const {
        if constexpr (!LINES) {
            if (whole(v)) return;
#pragma unroll
            for (int j = 0; j < kGroup; ++j) f[j] = inside(v, j) ? f[j] : 0.f;
        }
    }
    // The groups lie on lines of the tensor whose row begins at p.
    template <typename T> __device__ __forceinline__ bool lined(const T *p) const { return LINES || ((reinterpret_cast<uintptr_t>(p) - skip * sizeof(T)) & 15) == 0; }
    // Lays the groups out on the lines of the row at p.
    template <typename T> __device__ __forceinline__ void lay_out(const T *p) {
        if (!LINES) skip = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    }
    // Channels of the tensor before the row's first and after its last.  (Where the stream is updated in place, another block may be
    // writing a neighbour's channels on a shared line: what is read of them is not used.)
    __device__ __forceinline__ void bound(int64_t before, int64_t after) {
        if (LINES) return;
        low = -static_cast<int>(min(static_cast<int64_t>(2 * kGroup), before));
        high = n + static_cast<int>(min(static_cast<int64_t>(2 * kGroup), after));
    }
    // A group that lies across lines: put together from those, or channel by channel (0 outside) where they are not the tensor's.
    template <typename T> __device__ __forceinline__ int offset(const T *p, int v) const { return static_cast<int>(reinterpret_cast<uintptr_t>(p + at(v)) & 15); }
    template <typename T> __device__ __forceinline__ bool lines_readable(int v, int off) const {
        const int first = at(v) - off / static_cast<int>(sizeof(T));
        return first >= low && first + kLinesOf<T> * 16 / static_cast<int>(sizeof(T)) <= high;
    }
    template <typename T> __device__ __forceinline__ Raw<T> join(const uint4 (&q)[kLinesOf<T>], int off) const {
        constexpr int L = kLinesOf<T>, W = static_cast<int>(sizeof(T)) * 2;      // W: words of a group
        uint32_t w[4 * L], out[W];
#pragma unroll
        for (int i = 0; i < L; ++i) { w[4 * i] = q[i].x; w[4 * i + 1] = q[i].y; w[4 * i + 2] = q[i].z; w[4 * i + 3] = q[i].w; }
#pragma unroll
        for (int i = 0; i < 4 * L - 2; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
        for (int i = 0; i < 4 * L - 3; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
#pragma unroll
        for (int i = 0; i < W; ++i) out[i] = sizeof(T) == 2 ? __funnelshift_r(w[i], w[i + 1], off & 2 ? 16 : 0) : w[i];
        Raw<T> r;
        __builtin_memcpy(&r, out, sizeof(out));
        return r;
    }
    template <typename T> __device__ __forceinline__ Raw<T> gather(const T *p, int v) const {
        T e[kGroup];
#pragma unroll
        for (int j = 0; j < kGroup; ++j) e[j] = inside(v, j) ? p[at(v, j)] : from_float<T>(0.f);
        Raw<T> r;
        __builtin_memcpy(&r, e, sizeof(e));
        return r;
    }
    template <typename T> __device__ __forceinline__ Raw<T> across(const T *p, int v) const {
        const int off = offset(p, v);
        if (!lines_readable<T>(v, off)) return gather(p, v);
        uint4 q[kLinesOf<T>];
#pragma unroll
        for (int i = 0; i < kLinesOf<T>; ++i) q[i] = ld_stream(reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(p + at(v)) - off) + i);
        return join<T>(q, off);
    }
    // Two tensors whose groups lie across lines, all loads ahead of their first use (4096x4099, of gates and values: bf16 34.0 us group
    // by group, 26.2 us so; f32 42.9 and 39.9 us).  Four groups of a 32-bit type and more would not fit the registers.
    template <typename T> __device__ __forceinline__ void load_two(const T *a, const T *b, Raw<T> (&ra)[NV], Raw<T> (&rb)[NV]) const {
        const int oa = offset(a, 0), ob = offset(b, 0);     // a group's length is a multiple of a line's
        uint4 qa[NV][kLinesOf<T>], qb[NV][kLinesOf<T>];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const bool on_a = any(v) && lines_readable<T>(v, oa), on_b = any(v) && lines_readable<T>(v, ob);
#pragma unroll
            for (int i = 0; i < kLinesOf<T>; ++i) {
                qa[v][i] = ld_if(reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(a + at(v)) - oa) + i, on_a);
                qb[v][i] = ld_if(reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(b + at(v)) - ob) + i, on_b);
            }
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            ra[v] = join<T>(qa[v], oa);
            rb[v] = join<T>(qb[v], ob);
            if (any(v) && !lines_readable<T>(v, oa)) ra[v] = gather(a, v);
            if (any(v) && !lines_readable<T>(v, ob)) rb[v] = gather(b, v);
        }
    }
    // Past the row's ends what lies there; nothing where the thread has no channels.
    template <typename T> __device__ __forceinline__ void load(const T *p, Raw<T> (&held)[NV]) const {
        const bool on_lines = lined(p);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            held[v] = Raw<T>{};
            if (on_lines && readable(v)) held[v] = ld8(p + at(v));
            else if (!LINES && any(v)) held[v] = across(p, v);
        }
    }
    // f(channel value, constant) over the thread's channels; nothing where the constant vector is not given.  A vector is kept four
    // times, `stride` floats apart, each a float further along and zeros around it, so that the groups of any row lie on 16-byte lines of one.
    template <typename F> __device__ __forceinline__ void with(const float *p, int stride, float (&f)[NV][8], F apply) const {
        if (!p) return;
        const float *q = LINES ? p : p + (skip & 3) * stride + (skip & 3);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (any(v)) {
                const float4 a = __ldg(reinterpret_cast<const float4 *>(q + at(v))), b = __ldg(reinterpret_cast<const float4 *>(q + at(v)) + 1);
                const float w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int j = 0; j < kGroup; ++j) f[v][j] = apply(f[v][j], w[j]);
            }
        }
    }
    template <typename T> __device__ __forceinline__ void store(T *p, const float (&f)[NV][8]) const {
        const bool on_lines = lined(p);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (whole(v) && on_lines) {
                st8(p + at(v), f[v]);
            } else if (!LINES) {
                if (whole(v)) {
#pragma unroll
                    for (int j = 0; j < kGroup; ++j) p[at(v) + j] = from_float<T>(f[v][j]);
                } else {
#pragma unroll
                    for (int j = 0; j < kGroup; ++j)
                        if (inside(v, j)) p[at(v, j)] = from_float<T>(f[v][j]);
                }
            }
        }
    }
    __device__ __forceinline__ void store_bytes(int8_t *p, const float (&f)[NV][8], float inv) const {
        const bool words = LINES || ((reinterpret_cast<uintptr_t>(p) - skip) & 7) == 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (whole(v) && words) {
                *reinterpret_cast<uint2 *>(p + at(v)) = make_uint2(pack4_s8(f[v], inv), pack4_s8(f[v] + 4, inv));
            } else if (!LINES) {
                if (whole(v)) {
#pragma unroll
                    for (int j = 0; j < kGroup; ++j) p[at(v) + j] = static_cast<int8_t>(quantise(f[v][j], inv));
                } else {
#pragma unroll
                    for (int j = 0; j < kGroup; ++j)
                        if (inside(v, j)) p[at(v, j)] = static_cast<int8_t>(quantise(f[v][j], inv));
                }
            }
        }
    }
    __device__ __forceinline__ void store_as(int dtype, void *out, int64_t offset, const float (&f)[NV][8]) const {
        if (dtype == ENN_B200_BF16) store(static_cast<__nv_bfloat16 *>(out) + offset, f);
        else if (dtype == ENN_B200_F16) store(static_cast<__half *>(out) + offset, f);
        else store(static_cast<float *>(out) + offset, f);
    }
};

// Sums and maxima over the threads of a row: a warp, or the whole block.  Two sets of scratch words in turn, so that one barrier per
// reduction is enough.
__device__ __forceinline__ float warp_sum(float s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}
struct Reduce {
    float2 (*scratch)[32];
    int nt, turn;
    __device__ __forceinline__ float2 exchange(float2 v) {
        const int lane = threadIdx.x & 31;
        if (lane == 0) scratch[turn][threadIdx.x >> 5] = v;
        __syncthreads();
        v = lane < nt >> 5 ? scratch[turn][lane] : make_float2(0.f, 0.f);
        turn ^= 1;
        return v;
    }
    __device__ __forceinline__ float sum(float s) {
        s = warp_sum(s);
        return nt == 32 ? s : warp_sum(exchange(make_float2(s, 0.f)).x);
    }
    __device__ __forceinline__ uint32_t largest(uint32_t m) {
        m = __reduce_max_sync(0xffffffffu, m);
        return nt == 32 ? m : __reduce_max_sync(0xffffffffu, __float_as_uint(exchange(make_float2(0.f, __uint_as_float(m))).y));
    }
    __device__ __forceinline__ void both(float &s, uint32_t &m) {
        s = warp_sum(s);
        m = __reduce_max_sync(0xffffffffu, m);
        if (nt == 32) return;
        const float2 v = exchange(make_float2(s, __uint_as_float(m)));
        s = warp_sum(v.x);
        m = __reduce_max_sync(0xffffffffu, __float_as_uint(v.y));
    }
};

template <int NV>
__device__ __forceinline__ float sum_of_squares(const float (&f)[NV][8]) {
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < kGroup; ++j) s = fmaf(f[v][j], f[v][j], s);
    return s;
}
template <int NV>
__device__ __forceinline__ uint32_t largest_of(const float (&f)[NV][8]) {
    uint32_t m = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < kGroup; ++j) m = max(m, magnitude(f[v][j]));
    return m;
}
template <int NV>
__device__ __forceinline__ void multiply(float (&f)[NV][8], float by) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < kGroup; ++j) f[v][j] *= by;
}

// f = norm(f).  Channels past the row's end are 0 before and after.  With `largest` the bits of the largest magnitude of the result
// come back too; for an RMS norm without a bias they ride on the sum of squares, since max |f r w| = r max |f w|.
template <int NV, bool LINES>
__device__ __forceinline__ void norm_row(const Row<NV, LINES> &row, float (&f)[NV][8], int c, int kind, float eps, const float *weight, const float *bias, int stride,
                                         Reduce &reduce, uint32_t *largest) {
    const auto times = [](float a, float w) { return a * w; };
    if (kind != ENN_B200_NORM_NONE) {
        const float over = 1.f / static_cast<float>(c);
        if (kind == ENN_B200_NORM_LAYER) {
            float s = 0.f;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < kGroup; ++j) s += f[v][j];
            const float mean = reduce.sum(s) * over;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < kGroup; ++j) f[v][j] = row.inside(v, j) ? f[v][j] - mean : 0.f;
        }
        float s = sum_of_squares(f);
        if (largest && kind == ENN_B200_NORM_RMS && !bias) {
            row.with(weight, stride, f, times);
            uint32_t m = largest_of(f);
            reduce.both(s, m);
            const float r = rsqrtf(fmaf(s, over, eps));
            multiply(f, r);
            *largest = magnitude(__uint_as_float(m) * r);
            return;
        }
        multiply(f, rsqrtf(fmaf(reduce.sum(s), over, eps)));
        row.with(weight, stride, f, times);
        row.with(bias, stride, f, [](float a, float b) { return a + b; });
    }
    if (largest) *largest = reduce.largest(largest_of(f));
}

// Threads that the registers of NV groups a thread leave an SM: 64 registers each, 80 with four groups, 96 with eight.  One block may
// have them all, so that eight groups, which spill, remain for rows above 24576 channels (2048x10240 bf16 with a stream: 46 us in eight
// groups, 29 us in four; 33x10241 bf16 to bytes with a stream: 12.9 us, 6.5 us in two).
constexpr int norm_threads(int nv) { return nv <= 2 ? 1024 : (nv == 4 ? 768 : 544); }

// A thread's own ring in shared memory: `depth` rows ahead, each with `streams` tensors, filled by asynchronous copies.  A thread reads
// what it copied itself, so that no barrier is needed; the bytes in flight do not depend on how long a row's reductions take.
template <typename T, int NV>
struct Ahead {
    static constexpr int kPieces = sizeof(T) / 2;      // 16-byte pieces of a group
    uint32_t base;                                     // of this thread
    uint32_t piece;                                    // bytes from piece to piece: 16 for each thread of the block
    int streams, depth, slot;
    __device__ __forceinline__ uint32_t at(int s, int stream, int v, int i) const { return base + static_cast<uint32_t>(((s * streams + stream) * NV + v) * kPieces + i) * piece; }
    template <bool LINES> __device__ __forceinline__ void fetch(const Row<NV, LINES> &row, int s, int stream, const T *p) const {
        if (!row.lined(p)) return;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (row.readable(v))
#pragma unroll
                for (int i = 0; i < kPieces; ++i)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at(s, stream, v, i)), "l"(reinterpret_cast<const uint4 *>(p + row.at(v)) + i) : "memory");
    }
    template <bool LINES> __device__ __forceinline__ void read(const Row<NV, LINES> &row, int stream, const T *p, Raw<T> (&held)[NV]) const {
        const bool copied = row.lined(p);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (row.readable(v) && copied) {
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    uint4 &q = held[v].v[i];
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(at(slot, stream, v, i)) : "memory");
                }
            } else {
                held[v] = Raw<T>{};
                if (!LINES && row.any(v)) held[v] = row.across(p, v);
            }
        }
    }
};
__device__ __forceinline__ void ahead_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the `pending` youngest groups have arrived.
__device__ __forceinline__ void ahead_wait(int pending) {
    if (pending >= 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
    else if (pending == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (pending == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
}
constexpr int kMaxDepth = 4;
constexpr int kRingBytes = 216 * 1024;      // at most
// Of an SM: what they take, L1 lacks for the constant vectors (the same tensors pass after pass: 8192x5120 bf16, both norms and a stream, 67 us with
// all of it, 61 us so; 2048x12289 bf16 to bytes with a stream 88 and 83 us; 2048x8192 f32, both norms and a stream, 72 us either way).
constexpr int kRingShare = 112 * 1024;

// BYTES: the result is quantised.  A kernel of its own, since one for both overflows the instruction cache (with a stream: 2048x4097 bf16 to bytes
// 27.1 us, 25.1 us so; 8192x1001 bf16 20.7 and 18.4 us).
template <typename T, int NV, bool LINES, bool BYTES>
__global__ void __launch_bounds__(norm_threads(NV), 1) token_norm_kernel(NormParams p, int32_t rows, int32_t out_dtype, int32_t depth, const T *x,
                                                                                       const T *residual, const T *gate, T *stream, void *out, float *scale) {
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ float2 scratch[2][32];
    const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.y;
    Row<NV, LINES> row{p.c, static_cast<int>(threadIdx.x), static_cast<int>(blockDim.x), 0, 0, p.c};
    const int64_t gate_rows = gate ? (rows - 1) / p.gate_tokens + 1 : 0;
    Reduce reduce{scratch, row.nt, 0};
    pdl_wait();
    pdl_trigger();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    const uint32_t threads = blockDim.x * blockDim.y;
    Ahead<T, NV> ahead{smem_u32(ring) + 16 * (threadIdx.y * blockDim.x + threadIdx.x), 16 * threads, 1 + (residual != nullptr) + (gate != nullptr), depth, 0};
    auto fetch = [&](int s, int64_t t) {
        if (depth == 0) return;
        if (t < rows) {
            Row<NV, LINES> r = row;
            r.lay_out(x + t * p.c);
            r.bound(t * p.c, (rows - 1 - t) * p.c);
            ahead.fetch(r, s, 0, x + t * p.c);
            if (residual) ahead.fetch(r, s, 1, residual + t * p.c);
            if (gate) {
                const int64_t tg = t / p.gate_tokens;
                r.bound(tg * p.c, (gate_rows - 1 - tg) * p.c);
                ahead.fetch(r, s, ahead.streams - 1, gate + tg * p.c);
            }
        }
        ahead_commit();
    };
    auto take = [&](const Row<NV, LINES> &r, int which, const T *p_row, float (&f)[NV][8]) {
        Raw<T> held[NV];
        if (depth) ahead.read(r, which, p_row, held);
        else r.load(p_row, held);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            widen(held[v], f[v]);
            r.clear_outside(v, f[v]);
        }
    };
    for (int s = 0; s < depth; ++s) fetch(s, first + s * step);
    for (int64_t t = first; t < rows; t += step) {      // t is the same for a whole warp, and for the whole block where a row has several warps
        float f[NV][8];
        row.lay_out(x + t * p.c);
        row.bound(t * p.c, (rows - 1 - t) * p.c);
        if (depth) ahead_wait(depth - 1);
        take(row, 0, x + t * p.c, f);
        norm_row(row, f, p.c, p.post_norm, p.post_eps, p.post_weight, p.post_bias, p.stride, reduce, nullptr);
        if (gate) {
            float g[NV][8];
            const int64_t tg = t / p.gate_tokens;
            Row<NV, LINES> r = row;
            r.bound(tg * p.c, (gate_rows - 1 - tg) * p.c);
            take(r, ahead.streams - 1, gate + tg * p.c, g);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < kGroup; ++j) f[v][j] *= g[v][j];
        }
        if (residual) {
            float r[NV][8];
            take(row, 1, residual + t * p.c, r);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < kGroup; ++j) f[v][j] = fmaf(f[v][j], p.residual_scale, r[v][j]);
        } else if (p.residual_scale != 1.f) {
            multiply(f, p.residual_scale);
        }
        fetch(ahead.slot, t + depth * step);        // this row's memory has been read
        if (++ahead.slot >= depth) ahead.slot = 0;
        if (residual) row.store(stream + t * p.c, f);
        if constexpr (!BYTES) {
            norm_row(row, f, p.c, p.norm, p.eps, p.weight, p.bias, p.stride, reduce, nullptr);
            row.store_as(out_dtype, out, t * p.c, f);
        } else {
            uint32_t largest;
            norm_row(row, f, p.c, p.norm, p.eps, p.weight, p.bias, p.stride, reduce, &largest);
            const RowScale rs = row_scale(largest);
            int8_t *q = static_cast<int8_t *>(out) + t * p.pitch;
            row.store_bytes(q, f, rs.inv);
            for (int64_t i = p.c + row.tid; i < p.pitch; i += row.nt) q[i] = 0;
            if (row.tid == 0) scale[t] = rs.scale;
        }
    }
}

// 2^(-|g| log2(e) / 2), the root of e^-|g|: below 2^-126 only where its square is nothing to any result.  The instructions for 2^x and
// the reciprocal are a unit or two off in the last place.
__device__ __forceinline__ float root_exp(float g) {
    float h;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(fabsf(g) * -0.72134752044448170f));
    return h;
}
__device__ __forceinline__ float reciprocal(float a) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
    return r;
}
// a / (1 + e^-g) from an exponential that does not overflow.
__device__ __forceinline__ float times_sigmoid(float a, float g) {
    const float h = root_exp(g), e = h * h;
    return (g >= 0.f ? a : a * e) * reciprocal(1.f + e);
}
template <int ACT>
__device__ __forceinline__ float gate_act(float g) {
    if (ACT == ENN_B200_GATE_SILU) return times_sigmoid(g, g);
    if (ACT == ENN_B200_GATE_GELU) return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
    if (ACT == ENN_B200_GATE_GELU_TANH) return times_sigmoid(g, 2.f * 0.79788456080286536f * fmaf(0.044715f * g * g, g, g));      // (1 + tanh v) / 2 is the sigmoid of 2 v
    if (ACT == ENN_B200_GATE_RELU) return g < 0.f ? 0.f : g;
    return times_sigmoid(1.f, g);
}

// f = act(gates) * values of the thread's channels.
template <typename T, int NV, bool LINES>
__device__ __forceinline__ void gate_row(const Row<NV, LINES> &row, const T *gates, const T *values, int act, float (&f)[NV][8]) {
    Raw<T> rg[NV], ru[NV];
    if (!LINES && (sizeof(T) == 2 || (NV <= 2 && !(row.lined(gates) && row.lined(values))))) {
        row.load_two(gates, values, rg, ru);
    } else {
        row.load(gates, rg);
        row.load(values, ru);
    }
    auto apply = [&](auto which) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float g[8], u[8];
            widen(rg[v], g);
            widen(ru[v], u);
            row.clear_outside(v, u);
            row.clear_outside(v, g);
#pragma unroll
            for (int j = 0; j < kGroup; ++j) f[v][j] = gate_act<decltype(which)::value>(g[j]) * u[j];
        }
    };
    switch (act) {
        case ENN_B200_GATE_SILU: apply(std::integral_constant<int, ENN_B200_GATE_SILU>{}); break;
        case ENN_B200_GATE_GELU: apply(std::integral_constant<int, ENN_B200_GATE_GELU>{}); break;
        case ENN_B200_GATE_GELU_TANH: apply(std::integral_constant<int, ENN_B200_GATE_GELU_TANH>{}); break;
        case ENN_B200_GATE_RELU: apply(std::integral_constant<int, ENN_B200_GATE_RELU>{}); break;
        default: apply(std::integral_constant<int, ENN_B200_GATE_SIGMOID>{});
    }
}

constexpr int gate_threads(int nv) { return nv == 1 ? 1024 : 512; }

// Grid: rows x segments of `seg` channels.  Floats leave at once.  Bytes need the row's largest magnitude first: the
// segments of a row are then the CTAs of a cluster, which tell each other theirs.
template <typename T, int NV, bool LINES>
__global__ void __launch_bounds__(gate_threads(NV)) token_gate_kernel(GateParams p, int32_t rows, int32_t seg, int32_t out_dtype, const T *gates, const T *values,
                                                                 void *out, float *scale) {
    __shared__ float2 scratch[2][32];
    __shared__ uint32_t of_cluster[8];
    const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    const int32_t segs = static_cast<int32_t>(gridDim.y), rank = static_cast<int32_t>(blockIdx.y), c0 = rank * seg;
    Row<NV, LINES> row{min(seg, p.c - c0), static_cast<int>(threadIdx.x), static_cast<int>(blockDim.x), 0, 0, 0};
    // Seen by the others of the cluster before they write here: waited for below.
    const bool clustered = segs > 1 && out_dtype == ENN_B200_S8;
    if (clustered) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    pdl_wait();
    pdl_trigger();
    if (t >= rows) return;      // a whole warp, and then the block has no barrier
    float f[NV][8];
    // Groups on the lines of the results, which are stored as a whole; gates and values are put together where theirs are others.
    if (out_dtype == ENN_B200_S8) row.skip = static_cast<int>(reinterpret_cast<uintptr_t>(static_cast<int8_t *>(out) + t * p.pitch + c0) & 7);
    else if (out_dtype == ENN_B200_F32) row.lay_out(static_cast<float *>(out) + t * p.c + c0);
    else row.lay_out(static_cast<uint16_t *>(out) + t * p.c + c0);
    row.bound(t * p.in_stride + c0, (rows - 1 - t) * p.in_stride + (p.c - c0 - row.n));      // of the gates or of the values, whichever is less
    gate_row(row, gates + t * p.in_stride + c0, values + t * p.in_stride + c0, p.act, f);
    if (out_dtype != ENN_B200_S8) {
        row.store_as(out_dtype, out, t * p.c + c0, f);
        return;
    }
    Reduce reduce{scratch, row.nt, 0};
    uint32_t largest = reduce.largest(largest_of(f));      // 0 past the segment's end
    if (clustered) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (row.tid < segs) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_rank(smem_u32(of_cluster + rank), row.tid)), "r"(largest) : "memory");
        cluster_sync_all();     // the only writes to other CTAs come before it: nobody has to wait for them at the end
        for (int s = 0; s < segs; ++s) largest = max(largest, of_cluster[s]);
    }
    const RowScale rs = row_scale(largest);
    int8_t *q = static_cast<int8_t *>(out) + t * p.pitch;
    row.store_bytes(q + c0, f, rs.inv);
    if (rank == 0) {
        for (int64_t i = p.c + row.tid; i < p.pitch; i += row.nt) q[i] = 0;
        if (row.tid == 0) scale[t] = rs.scale;
    }
}

bool aligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Threads of a row and groups per thread for `n` channels.  `spread`: as many threads as there are groups (few rows: latency), else
// four groups each (many rows: what a row costs whatever its length, reductions and addresses, is shared by more channels), up to
// `most(groups)` threads; `two`: two, where four are too many (the code for shifted groups then overflows the instruction cache: 2048x4097 bf16 to
// bytes with a stream 30 us, 27 us with two, gates of 4096x4099 bf16 35 us, 26 us; the rows of 32-bit types in flight leave L1 nothing:
// 2048x8192 f32, both norms and a stream, 82 us, 72 us with two).
struct Shape {
    int nt, nv, per_block;
};
Shape row_shape(int n, bool lines, bool spread, bool two, int (*most)(int)) {
    const int groups = (n + (lines ? 0 : kGroup - 1) + kGroup - 1) / kGroup;      // one more where they are shifted
    auto threads = [&](int nv) { return ((groups + nv - 1) / nv + 31) / 32 * 32; };
    Shape s;
    if (groups <= 32 || (spread && groups <= most(1))) s.nv = 1;
    else if (groups <= 64 || ((two || spread) && groups <= 2 * most(2))) s.nv = 2;
    else s.nv = groups <= 4 * most(4) ? 4 : 8;
    s.nt = threads(s.nv);
    s.per_block = s.nt == 32 ? 8 : 1;
    return s;
}

template <int MOST, typename F>
cudaError_t with_shape(int nv, bool lines, F f) {
    auto groups = [&](auto v) {
        switch (nv) {
            case 1: return f(std::integral_constant<int, 1>{}, v);
            case 2: return f(std::integral_constant<int, 2>{}, v);
            case 4: return f(std::integral_constant<int, 4>{}, v);
            default: return f(std::integral_constant<int, MOST>{}, v);
        }
    };
    return lines ? groups(std::true_type{}) : groups(std::false_type{});
}

template <typename T>
cudaError_t norm_typed(const enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs) {
    const TokenState &t = *op->token;
    const NormParams &p = t.norm;
    int i = 0, o = 0;
    const T *x = static_cast<const T *>(ins[i++]);
    const T *residual = t.residual ? static_cast<const T *>(ins[i++]) : nullptr;
    const T *gate = p.gate_tokens ? static_cast<const T *>(ins[i++]) : nullptr;
    T *stream = t.residual ? static_cast<T *>(outs[o++]) : nullptr;
    void *y = outs[o++];
    float *scale = t.out_dtype == ENN_B200_S8 ? static_cast<float *>(outs[o++]) : nullptr;
    const bool lines = p.c % kGroup == 0 && aligned(x, 16) && aligned(residual, 16) && aligned(gate, 16) && aligned(stream, 16) && aligned(y, scale ? 8 : 16);
    const Shape s = row_shape(p.c, lines, rows <= 2 * op->token->sms, !lines || sizeof(T) == 4, norm_threads);
    // As many blocks as an SM holds, each taking rows in turn, and rings of up to four rows in what shared memory
    // that leaves them; the widest rows of 32-bit types do without.
    const int threads = s.nt * s.per_block;
    const int blocks = norm_threads(s.nv) / threads;
    const int ahead_bytes = threads * s.nv * kGroup * static_cast<int>(sizeof(T)) * (1 + (residual != nullptr) + (gate != nullptr));
    const int depth = ahead_bytes > kRingBytes ? 0 : std::min(kMaxDepth, std::max(1, kRingShare / blocks / ahead_bytes));
    const int64_t want = (static_cast<int64_t>(rows) + s.per_block - 1) / s.per_block, most = static_cast<int64_t>(t.sms) * blocks;
    const dim3 grid(static_cast<unsigned>(std::min(want, most))), block(static_cast<unsigned>(s.nt), static_cast<unsigned>(s.per_block));
    return with_shape<8>(s.nv, lines, [&](auto nv, auto v) {
        auto launch = [&](auto kernel, PerDeviceInit &once) {
            const cudaError_t e = once.run(op->ctx->device, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes); });
            if (e != cudaSuccess) return e;
            return launch_pdl(kernel, grid, block, static_cast<size_t>(depth) * ahead_bytes, op->ctx->stream, p, rows, t.out_dtype, depth, x, residual, gate, stream, y, scale);
        };
        static PerDeviceInit bytes, floats;
        constexpr int NV = decltype(nv)::value;
        constexpr bool LINES = decltype(v)::value;
        return scale ? launch(token_norm_kernel<T, NV, LINES, true>, bytes) : launch(token_norm_kernel<T, NV, LINES, false>, floats);
    });
}

template <typename T>
cudaError_t gate_typed(const enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs) {
    const TokenState &t = *op->token;
    const GateParams &p = t.gate;
    const T *g = static_cast<const T *>(ins[0]), *u = t.packed ? g + p.c : static_cast<const T *>(ins[1]);
    const bool bytes = t.out_dtype == ENN_B200_S8;
    const bool lines = p.c % kGroup == 0 && aligned(g, 16) && aligned(u, 16) && aligned(outs[0], bytes ? 8 : 16);
    // Segments: of up to 8192 channels.  Of bytes one for up to 16384 channels (the exchange in a cluster costs more than it brings:
    // 8192x12288 99 us in two, 96 us in one; 2048x24576 53 us in four, 63 us in two), then up to eight, and more where the rows alone do not
    // occupy the device.
    int segs = 1;
    if (!bytes) segs = (p.c + 8191) / 8192;
    else
        while (segs < 8 && (p.c > (segs == 1 ? 16384 - (lines ? 0 : kGroup) : 8192 * segs) || (static_cast<int64_t>(rows) * segs * 2 <= 2 * op->token->sms && p.c >= 2048 * segs))) segs *= 2;
    const int seg = segs == 1 ? p.c : ((p.c + segs - 1) / segs + kGroup - 1) / kGroup * kGroup;
    if (!bytes) segs = (p.c + seg - 1) / seg;
    const Shape s = row_shape(seg, lines, static_cast<int64_t>(rows) * segs <= 2 * op->token->sms, !lines, gate_threads);      // at most four groups: segments end before
    const int per_block = segs > 1 && bytes ? 1 : s.per_block;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((static_cast<int64_t>(rows) + per_block - 1) / per_block), static_cast<unsigned>(segs));
    cfg.blockDim = dim3(static_cast<unsigned>(s.nt), static_cast<unsigned>(per_block));
    cfg.stream = op->ctx->stream;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = attr[1].val.clusterDim.z = 1;
    attr[1].val.clusterDim.y = static_cast<unsigned>(segs);
    cfg.attrs = attr;
    cfg.numAttrs = bytes && segs > 1 ? 2 : 1;
    return with_shape<4>(s.nv, lines, [&](auto nv, auto v) {
        return cudaLaunchKernelEx(&cfg, token_gate_kernel<T, decltype(nv)::value, decltype(v)::value>, p, rows, seg, t.out_dtype, g, u, outs[0],
                                  bytes ? static_cast<float *>(outs[1]) : nullptr);
    });
}

}  // namespace

cudaError_t token_norm_launch(const enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs) {
    switch (op->token->in_dtype) {
        case ENN_B200_F32: return norm_typed<float>(op, rows, ins, outs);
        case ENN_B200_F16: return norm_typed<__half>(op, rows, ins, outs);
        case ENN_B200_BF16: return norm_typed<__nv_bfloat16>(op, rows, ins, outs);
    }
    return cudaErrorInvalidValue;
}

cudaError_t token_gate_launch(const enn_b200_op *op, int32_t rows, const void *const *ins, void *const *outs) {
    switch (op->token->in_dtype) {
        case ENN_B200_F32: return gate_typed<float>(op, rows, ins, outs);
        case ENN_B200_F16: return gate_typed<__half>(op, rows, ins, outs);
        case ENN_B200_BF16: return gate_typed<__nv_bfloat16>(op, rows, ins, outs);
    }
    return cudaErrorInvalidValue;
}

}  // namespace enn_b200
