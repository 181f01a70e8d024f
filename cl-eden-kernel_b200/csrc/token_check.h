// Checks of the token operators' descriptors and calls, and the sizes that follow from them.  Host code without CUDA, so that the
// refusals are tested without a device.
#pragma once
#include <stdint.h>

#include <cmath>

#include "../../include/enn_b200.h"

namespace enn_b200 {

// Rows in memory: `row` bytes each, `stride` bytes from one to the next; `group` tokens share a row.
struct RowLayout {
    int64_t row = 0, stride = 0;
    int32_t group = 1;
    int64_t span(int32_t tokens) const {
        const int64_t rows = tokens / group + (tokens % group ? 1 : 0);
        return rows ? (rows - 1) * stride + row : 0;
    }
    // Whether `bytes` > 0 bytes at `other` reach into the rows of the tokens; what lies between rows is not theirs.
    bool reached_by(const void *at, int32_t tokens, const void *other, int64_t bytes) const {
        const uintptr_t a = reinterpret_cast<uintptr_t>(at), o = reinterpret_cast<uintptr_t>(other);
        if (o < a) return static_cast<uint64_t>(bytes) > a - o;
        if (o - a >= static_cast<uint64_t>(span(tokens))) return false;
        const int64_t within = static_cast<int64_t>((o - a) % static_cast<uint64_t>(stride));
        return within < row || within + bytes > stride;
    }
};

// What a call of a prepared token operator is checked against.
struct TokenCall {
    static constexpr int kMaxIns = 3, kMaxOuts = 4;
    int32_t m = 0;
    int32_t n_in = 0, n_out = 0;
    RowLayout in[kMaxIns], out[kMaxOuts];
    int64_t in_bytes[kMaxIns] = {}, out_bytes[kMaxOuts] = {};      // of all m rows
    int32_t in_align[kMaxIns] = {}, out_align[kMaxOuts] = {};      // element sizes
    bool in_place = false;                                          // out 0 may be the memory of in 1 (token_norm's stream)

    void add_in(int64_t row, int64_t stride, int32_t align, int32_t group = 1) {
        in[n_in] = RowLayout{row, stride, group};
        in_align[n_in] = align;
        in_bytes[n_in] = in[n_in].span(m);
        ++n_in;
    }
    void add_out(int64_t row, int32_t align) {
        out[n_out] = RowLayout{row, row, 1};
        out_align[n_out] = align;
        out_bytes[n_out] = out[n_out].span(m);
        ++n_out;
    }
};

constexpr int32_t kMostRows = 1 << 30;

inline int32_t float_size(int32_t dtype) {
    return dtype == ENN_B200_F32 ? 4 : (dtype == ENN_B200_F16 || dtype == ENN_B200_BF16 ? 2 : 0);
}

// Most bytes a tensor may span: far above any device's memory, and far enough below 2^63 for the sums over an operator's tensors.
constexpr int64_t kMostBytes = int64_t{1} << 60;
// Rows of `row` bytes, `stride` bytes from one to the next.
inline bool rows_fit(int32_t m, int64_t stride, int64_t row) { return m <= 1 || stride <= (kMostBytes - row) / (m - 1); }

// Multiply-accumulates of a product, the largest number where they are more.
inline int64_t token_macs(int32_t m, int32_t k, int32_t n) {
    const int64_t mn = static_cast<int64_t>(m) * n;
    return mn > INT64_MAX / k ? INT64_MAX : mn * k;
}

inline int64_t token_pitch(int32_t c) { return (static_cast<int64_t>(c) + 15) & ~int64_t{15}; }

// The check_* return null and fill `call`, or what is wrong with the descriptor.
inline const char *check_token_fc(const enn_b200_token_fc_desc &d, TokenCall *call) {
    if (d.m < 0 || d.m > kMostRows || d.k <= 0 || d.n <= 0 || d.n > (1 << 21)) return "token_fc: bad shape (n is 1 .. 2^21)";
    if (d.k >= 131072) return "token_fc: k must be below 131072 (sums of products are 32-bit)";
    const int32_t e = float_size(d.out_dtype);
    if (!e) return "token_fc: out_dtype must be F32, F16 or BF16";
    if (d.in_pitch != 0 && d.in_pitch < d.k) return "token_fc: rows overlap (in_pitch < k)";
    if (d.in_pitch > (int64_t{1} << 38)) return "token_fc: in_pitch is too large";
    const int64_t pitch = d.in_pitch ? d.in_pitch : token_pitch(d.k);
    if (!rows_fit(d.m, pitch, d.k)) return "token_fc: rows span more than 2^60 bytes";
    call->m = d.m;
    call->add_in(d.k, pitch, 1);
    call->add_in(4, 4, 4);
    call->add_out(static_cast<int64_t>(d.n) * e, e);
    return nullptr;
}

inline bool token_out(TokenCall *call, int32_t c, int32_t dtype) {
    if (dtype == ENN_B200_S8) {
        call->add_out(token_pitch(c), 1);
        call->add_out(4, 4);
        return true;
    }
    const int32_t e = float_size(dtype);
    call->add_out(static_cast<int64_t>(c) * e, e);
    return e != 0;
}

inline const char *check_token_norm(const enn_b200_token_norm_desc &d, TokenCall *call) {
    if (d.m < 0 || d.m > kMostRows || d.c <= 0) return "token_norm: bad shape";
    if (d.c > 32768) return "token_norm: c must be at most 32768";
    if (d.norm < ENN_B200_NORM_NONE || d.norm > ENN_B200_NORM_LAYER || d.post_norm < ENN_B200_NORM_NONE || d.post_norm > ENN_B200_NORM_LAYER)
        return "token_norm: unknown norm";
    const int32_t e = float_size(d.io_dtype);
    if (!e) return "token_norm: io_dtype must be F32, F16 or BF16";
    if (d.gate_tokens < 0) return "token_norm: gate_tokens must not be negative";
    if (!(d.eps >= 0.f) || !(d.post_eps >= 0.f) || std::isinf(d.eps) || std::isinf(d.post_eps)) return "token_norm: eps must be finite and not negative";
    if (!std::isfinite(d.residual_scale)) return "token_norm: residual_scale must be finite";
    const int64_t row = static_cast<int64_t>(d.c) * e;
    call->m = d.m;
    call->add_in(row, row, e);
    if (d.residual) call->add_in(row, row, e);
    if (d.gate_tokens) call->add_in(row, row, e, d.gate_tokens);
    if (d.residual) call->add_out(row, e);
    call->in_place = d.residual != 0;
    return token_out(call, d.c, d.out_dtype) ? nullptr : "token_norm: out_dtype must be F32, F16, BF16 or S8";
}

inline const char *check_token_gate(const enn_b200_token_gate_desc &d, TokenCall *call) {
    if (d.m < 0 || d.m > kMostRows || d.c <= 0) return "token_gate: bad shape";
    if (d.c > 65536) return "token_gate: c must be at most 65536";
    if (d.act < ENN_B200_GATE_SILU || d.act > ENN_B200_GATE_SIGMOID) return "token_gate: unknown activation";
    const int32_t e = float_size(d.in_dtype);
    if (!e) return "token_gate: in_dtype must be F32, F16 or BF16";
    const int64_t row = static_cast<int64_t>(d.c) * e;
    call->m = d.m;
    call->add_in(row * (d.packed ? 2 : 1), row * (d.packed ? 2 : 1), e);
    if (!d.packed) call->add_in(row, row, e);
    return token_out(call, d.c, d.out_dtype) ? nullptr : "token_gate: out_dtype must be F32, F16, BF16 or S8";
}

inline const char *check_log_probs(const enn_b200_log_probs_desc &d, TokenCall *call) {
    if (d.m < 0 || d.m > kMostRows || d.vocab <= 0 || d.vocab > (1 << 24)) return "log_probs: bad shape (vocab is 1 .. 2^24)";
    const int32_t e = float_size(d.in_dtype);
    if (!e) return "log_probs: in_dtype must be F32, F16 or BF16";
    if (d.given < 0 || d.given > 1024) return "log_probs: given must be within 0 .. 1024";
    if (d.top < 0 || d.top > ENN_B200_LOG_PROBS_MAX_TOP || d.top > d.vocab) return "log_probs: top must be within 0 .. min(vocab, 32)";
    if (!(d.scale > 0.f) || d.scale > 0x1p127f) return "log_probs: scale must be positive and at most 2^127";      // scale * log2(e) is a float
    if (d.in_pitch != 0 && d.in_pitch < d.vocab) return "log_probs: rows overlap (in_pitch < vocab)";
    if (d.in_pitch > (int64_t{1} << 38)) return "log_probs: in_pitch is too large";
    const int64_t pitch = d.in_pitch ? d.in_pitch : d.vocab;
    if (!rows_fit(d.m, pitch * e, int64_t{e} * d.vocab)) return "log_probs: rows span more than 2^60 bytes";
    call->m = d.m;
    call->add_in(int64_t{e} * d.vocab, pitch * e, e);
    if (d.given) call->add_in(int64_t{4} * d.given, int64_t{4} * d.given, 4);
    if (d.given) call->add_out(int64_t{4} * d.given, 4);
    call->add_out(4, 4);
    if (d.top) {
        call->add_out(int64_t{4} * d.top, 4);
        call->add_out(int64_t{4} * d.top, 4);
    }
    return nullptr;
}

// A call of enn_b200_op_execute_rows: null, or what is wrong with it.
inline const char *check_rows_call(const TokenCall &c, int32_t rows, const void *const *ins, int32_t n_in, void *const *outs, int32_t n_out) {
    if (rows < 0 || rows > c.m) return "rows must be within 0 and the prepared m";
    if (n_in != c.n_in || n_out != c.n_out || !ins || !outs) return "wrong number of inputs or outputs for this operator";
    if (rows == 0) return nullptr;      // nothing is touched: empty tensors have no address
    for (int i = 0; i < n_in; ++i) {
        if (!ins[i]) return "null device pointer";
        if (reinterpret_cast<uintptr_t>(ins[i]) % c.in_align[i]) return "an input is not aligned to its element type";
    }
    for (int o = 0; o < n_out; ++o) {
        if (!outs[o]) return "null device pointer";
        if (reinterpret_cast<uintptr_t>(outs[o]) % c.out_align[o]) return "an output is not aligned to its element type";
        for (int i = 0; i < n_in; ++i)
            if (outs[o] == ins[i] && !(c.in_place && o == 0 && i == 1)) return "an output must not be an input's memory";
        for (int p = 0; p < o; ++p)
            if (outs[o] == outs[p]) return "two outputs must not be the same memory";
    }
    return nullptr;
}

// The memory of a call that check_rows_call has passed: null, or what is wrong with it.
inline const char *check_rows_memory(const TokenCall &c, int32_t rows, const void *const *ins, void *const *outs) {
    for (int o = 0; o < c.n_out && rows > 0; ++o) {
        const int64_t bytes = c.out[o].span(rows);
        for (int i = 0; i < c.n_in; ++i)
            if (c.in[i].reached_by(ins[i], rows, outs[o], bytes) && !(c.in_place && o == 0 && i == 1 && outs[o] == ins[i]))
                return "an output must not share memory with an input";
        for (int p = 0; p < o; ++p)
            if (c.out[p].reached_by(outs[p], rows, outs[o], bytes)) return "two outputs must not share memory";
    }
    return nullptr;
}

}  // namespace enn_b200
