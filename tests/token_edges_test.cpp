// Sizes and calls of the token operators at their limits (csrc/token_check.h), without a device.
#include "token_check.h"

#include <cmath>
#include <cstdio>
#include <cstring>
#include <initializer_list>

using namespace enn_b200;

static int failures = 0;
static void expect(bool ok, const char *what) {
    if (ok) return;
    std::printf("FAILED: %s\n", what);
    ++failures;
}

static void sizes() {
    const int32_t most = 1 << 30;
    const int64_t widest = int64_t{1} << 38;
    TokenCall c;
    expect(!check_token_fc({1, 33, 1, ENN_B200_F32, widest}, &c) && c.in_bytes[0] == 33, "one row of any pitch");
    c = TokenCall();
    expect(!check_token_fc({most, 33, 1, ENN_B200_F32, 48}, &c) && c.in_bytes[0] == (int64_t{1} << 30) * 48 - 15, "many rows");
    c = TokenCall();
    expect(!check_token_fc({most, 16, 1 << 21, ENN_B200_F32, int64_t{1} << 29}, &c) && c.in_bytes[0] == (((int64_t{1} << 30) - 1) << 29) + 16 && c.out_bytes[0] == int64_t{1} << 53, "rows that fit");
    expect(check_token_fc({most, 16, 1, ENN_B200_F32, widest}, &c), "fc: more bytes than 64 bits count");
    expect(check_token_fc({most, 16, 1, ENN_B200_F32, int64_t{1} << 33}, &c) && check_token_fc({most, 16, 1, ENN_B200_F32, int64_t{1} << 31}, &c), "fc: more bytes than there can be");
    c = TokenCall();
    enn_b200_log_probs_desc d{most, 1000, ENN_B200_F32, 0, 0, 1.f, int64_t{1} << 27};
    expect(!check_log_probs(d, &c) && c.in_bytes[0] == ((((int64_t{1} << 30) - 1) << 27) + 1000) * 4, "log_probs: rows that fit");
    for (int64_t pitch : {int64_t{1} << 29, int64_t{1} << 31, int64_t{1} << 32, int64_t{1} << 33, widest}) {
        d.in_pitch = pitch;
        expect(check_log_probs(d, &c), "log_probs: more bytes than there can be");
    }
    d.in_dtype = ENN_B200_BF16;
    d.in_pitch = widest;
    expect(check_log_probs(d, &c), "log_probs: 16-bit logits");
    expect(token_macs(3, 5, 7) == 105 && token_macs(0, 5, 7) == 0 && token_macs(most, 131071, 1 << 21) == INT64_MAX, "multiply-accumulates stay at the largest number");
}

// Every place of an output against a count byte by byte.
static void overlaps() {
    static char buf[4096];
    char *const base = buf + 1024;
    const auto shares = [&](const RowLayout &in, int32_t tokens, int64_t at, int64_t bytes) {
        const int64_t rows = (tokens + in.group - 1) / in.group;
        for (int64_t r = 0; r < rows; ++r)
            for (int64_t j = 0; j < in.row; ++j)
                if (r * in.stride + j >= at && r * in.stride + j < at + bytes) return true;
        return false;
    };
    for (const RowLayout &in : {RowLayout{8, 8, 1}, RowLayout{8, 24, 1}, RowLayout{4, 32, 3}})
        for (int32_t tokens : {1, 3, 4, 7})
            for (int64_t bytes : {1, 4, 16, 24, 40, 300})
                for (int64_t at = -320; at < 320; ++at)
                    if (in.reached_by(base, tokens, base + at, bytes) != shares(in, tokens, at, bytes)) {
                        std::printf("row %d stride %d group %d tokens %d bytes %d at %d\n", static_cast<int>(in.row), static_cast<int>(in.stride), in.group, tokens, static_cast<int>(bytes), static_cast<int>(at));
                        expect(false, "overlap");
                        return;
                    }
}

static void calls() {
    static char buf[16384];
    TokenCall n;      // 4 rows of 40 16-bit channels, a row of gates for 3 tokens, to bytes (48 a row) and scales
    expect(!check_token_norm({4, 40, ENN_B200_NORM_RMS, ENN_B200_NORM_NONE, 1, 3, ENN_B200_BF16, ENN_B200_S8, 1e-6f, 0.f, 1.f}, &n), "a norm");
    char *x = buf, *r = buf + 640, *g = buf + 1280, *h = buf + 2048, *q = buf + 2560, *s = buf + 4096;
    const auto norm = [&](int32_t rows, char *ho, char *qo, char *so) {
        const void *ins[] = {x, r, g};
        void *outs[] = {ho, qo, so};
        return !check_rows_call(n, rows, ins, 3, outs, 3) && !check_rows_memory(n, rows, ins, outs);
    };
    expect(norm(4, h, q, s) && norm(4, r, q, s), "memory of their own, the stream in place");
    expect(!norm(4, r + 2, q, s) && !norm(4, r - 80, q, s) && !norm(4, r + 80, q, s) && !norm(4, r + 318, q, s), "the stream shifted");
    expect(norm(4, r + 320, q, s) && norm(4, r - 320, q, s), "the stream beside its input");
    expect(norm(1, r + 80, q, s) && !norm(2, r + 80, q, s), "rows past the call's do not count");
    expect(!norm(4, x + 16, q, s) && !norm(4, h, x + 300, s) && norm(4, h, x + 320, s), "over the block's output");
    expect(!norm(4, h, g - 64, s) && !norm(4, h, q, g + 156) && norm(4, h, q, g + 160) && norm(3, h, q, g + 80), "over the gates");
    expect(!norm(4, h, h + 16, s) && !norm(4, h, h - 16, s) && !norm(4, h, q, q + 188) && norm(4, h, q, q + 192), "over another output");
    expect(!norm(4, r, r + 16, s), "bytes over the stream in place");

    TokenCall l;      // 3 rows of 10 logits, 16 apart
    enn_b200_log_probs_desc d{3, 10, ENN_B200_F32, 0, 0, 1.f, 16};
    expect(!check_log_probs(d, &l), "log_probs");
    const auto probs = [&](int32_t rows, char *out) {
        const void *ins[] = {x};
        void *outs[] = {out};
        return !check_rows_call(l, rows, ins, 1, outs, 1) && !check_rows_memory(l, rows, ins, outs);
    };
    expect(!probs(3, x + 36) && probs(3, x + 40) && !probs(3, x + 56) && probs(1, x + 56) && !probs(3, x + 64), "between the rows of the logits");

    TokenCall f;      // 100 rows of 33 bytes, dense
    expect(!check_token_fc({100, 33, 7, ENN_B200_F32, 33}, &f), "fc");
    const auto fc = [&](int32_t rows, char *scale, char *out) {
        const void *ins[] = {x, scale};
        void *outs[] = {out};
        return !check_rows_call(f, rows, ins, 2, outs, 1) && !check_rows_memory(f, rows, ins, outs);
    };
    char *far = buf + 8192;
    expect(fc(100, far, far + 400) && !fc(100, far, far + 396) && !fc(100, far, far - 2796) && fc(100, far, far - 2800) && !fc(100, far, x + 3296) && fc(100, far, x + 3300), "fc");
}

static void scales() {
    for (float scale : {1e-45f, 1.f, 0x1p126f, 0x1p127f}) {
        TokenCall c;
        expect(!check_log_probs({2, 100, ENN_B200_F32, 1, 5, scale, 0}, &c), "a scale whose product with log2(e) is a float");
    }
    for (float scale : {std::nextafterf(0x1p127f, INFINITY), 3.402823466e38f, INFINITY, -1.f, -0.f}) {
        TokenCall c;
        expect(check_log_probs({2, 100, ENN_B200_F32, 1, 5, scale, 0}, &c), "a scale whose product with log2(e) is none");
    }
}

int main(int argc, char **argv) {
    const char *which = argc > 1 ? argv[1] : "";
    if (!std::strcmp(which, "sizes")) sizes();
    else if (!std::strcmp(which, "overlaps")) overlaps();
    else if (!std::strcmp(which, "calls")) calls();
    else if (!std::strcmp(which, "scales")) scales();
    else expect(false, "which test?");
    return failures ? 1 : 0;
}
