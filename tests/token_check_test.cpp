// Refusals and sizes of the token operators (csrc/token_check.h), without a device.
#include "token_check.h"

#include <cmath>
#include <cstdio>

using namespace enn_b200;

static int failures = 0;
static void expect(bool ok, const char *what) {
    if (ok) return;
    std::printf("FAILED: %s\n", what);
    ++failures;
}

static bool fc(int32_t m, int32_t k, int32_t n, int32_t out, int64_t pitch, TokenCall *c = nullptr) {
    TokenCall t;
    return !check_token_fc({m, k, n, out, pitch}, c ? c : &t);
}
static enn_b200_token_norm_desc norm_desc() {
    return {4, 40, ENN_B200_NORM_RMS, ENN_B200_NORM_NONE, 1, 3, ENN_B200_BF16, ENN_B200_S8, 1e-6f, 0.f, 1.f};
}
template <typename F>
static bool norm(F change, TokenCall *c = nullptr) {
    TokenCall t;
    auto d = norm_desc();
    change(d);
    return !check_token_norm(d, c ? c : &t);
}
template <typename F>
static bool log_probs(F change, TokenCall *c = nullptr) {
    TokenCall t;
    enn_b200_log_probs_desc d{2, 100, ENN_B200_F32, 1, 5, 1.f, 0};
    change(d);
    return !check_log_probs(d, c ? c : &t);
}

int main() {
    TokenCall c;
    expect(fc(3, 33, 7, ENN_B200_F16, 0, &c) && c.in_bytes[0] == 2 * 48 + 33 && c.in_bytes[1] == 12 && c.out_bytes[0] == 42 && c.n_in == 2 && c.n_out == 1, "fc sizes");
    expect(fc(0, 1, 1, ENN_B200_F32, 0), "no rows");
    expect(!fc(-1, 1, 1, ENN_B200_F32, 0) && !fc(1, 0, 1, ENN_B200_F32, 0) && !fc(1, 1, 0, ENN_B200_F32, 0) && !fc(1, 1, (1 << 21) + 1, ENN_B200_F32, 0), "fc shape");
    expect(fc(1, 131071, 1, ENN_B200_F32, 0) && !fc(1, 131072, 1, ENN_B200_F32, 0), "fc reduction that fits 32 bits");
    expect(!fc(1, 1, 1, ENN_B200_S8, 0) && !fc(1, 1, 1, 2, 0), "fc result type");
    expect(fc(1, 33, 1, ENN_B200_F32, 33) && !fc(1, 33, 1, ENN_B200_F32, 32) && !fc(1, 33, 1, ENN_B200_F32, -16), "fc pitch");

    expect(fc(1 << 30, 1, 1, ENN_B200_F32, 0) && !fc((1 << 30) + 1, 1, 1, ENN_B200_F32, 0), "most rows");

    TokenCall n;
    expect(norm([](auto &) {}, &n) && n.n_in == 3 && n.n_out == 3 && n.in_bytes[2] == 2 * 40 * 2 && n.out_bytes[1] == 4 * 48 && n.in_place, "norm sizes");
    TokenCall n2;
    expect(norm([](auto &d) { d.residual = d.gate_tokens = 0; d.out_dtype = ENN_B200_F32; }, &n2) && n2.n_in == 1 && n2.n_out == 1 && !n2.in_place && n2.out_bytes[0] == 640, "norm alone");
    expect(norm([](auto &d) { d.c = 32768; }) && !norm([](auto &d) { d.c = 32769; }) && !norm([](auto &d) { d.c = 0; }) && !norm([](auto &d) { d.m = -1; }), "norm shape");
    expect(!norm([](auto &d) { d.norm = 3; }) && !norm([](auto &d) { d.post_norm = -1; }), "norm kind");
    expect(!norm([](auto &d) { d.io_dtype = ENN_B200_S8; }) && !norm([](auto &d) { d.out_dtype = ENN_B200_U8; }), "norm types");
    expect(!norm([](auto &d) { d.eps = -1.f; }) && !norm([](auto &d) { d.post_eps = NAN; }) && !norm([](auto &d) { d.eps = INFINITY; }), "norm eps");
    expect(!norm([](auto &d) { d.residual_scale = NAN; }) && !norm([](auto &d) { d.residual_scale = INFINITY; }) && !norm([](auto &d) { d.gate_tokens = -1; }), "norm scale and gates");

    TokenCall g;
    expect(!check_token_gate({5, 30, ENN_B200_GATE_GELU, 1, ENN_B200_F32, ENN_B200_S8}, &g) && g.n_in == 1 && g.in_bytes[0] == 1200 && g.out_bytes[0] == 160 && g.out_bytes[1] == 20, "gate sizes");
    TokenCall x;
    expect(check_token_gate({5, 30, 5, 1, ENN_B200_F32, ENN_B200_S8}, &x) && check_token_gate({5, 65537, 0, 1, ENN_B200_F32, ENN_B200_S8}, &x) &&
               check_token_gate({5, 30, 0, 1, ENN_B200_S8, ENN_B200_S8}, &x) && check_token_gate({5, 30, 0, 1, ENN_B200_F32, 7}, &x), "gate refusals");

    TokenCall l;
    expect(log_probs([](auto &) {}, &l) && l.n_in == 2 && l.n_out == 4 && l.out_bytes[2] == 40, "log_probs sizes");
    TokenCall l2;
    expect(log_probs([](auto &d) { d.given = d.top = 0; d.in_pitch = 128; }, &l2) && l2.n_in == 1 && l2.n_out == 1 && l2.in_bytes[0] == 4 * 228, "entropy alone");
    expect(!log_probs([](auto &d) { d.top = 33; }) && !log_probs([](auto &d) { d.vocab = 4; }) && !log_probs([](auto &d) { d.given = -1; }) && !log_probs([](auto &d) { d.given = 1025; }), "log_probs counts");
    expect(!log_probs([](auto &d) { d.scale = 0.f; }) && !log_probs([](auto &d) { d.scale = NAN; }) && !log_probs([](auto &d) { d.scale = INFINITY; }), "log_probs scale");
    expect(!log_probs([](auto &d) { d.vocab = 0; }) && !log_probs([](auto &d) { d.vocab = (1 << 24) + 1; }) && !log_probs([](auto &d) { d.in_pitch = 99; }) && !log_probs([](auto &d) { d.in_dtype = ENN_B200_S8; }), "log_probs shape");

    char buf[256];
    const void *a = buf, *b = buf + 32, *odd = buf + 1;
    void *o0 = buf + 64, *o1 = buf + 96, *o2 = buf + 128;
    const void *ins[] = {a, b, buf + 48};
    void *outs[] = {o0, o1, o2};
    expect(!check_rows_call(n, 4, ins, 3, outs, 3) && !check_rows_call(n, 1, ins, 3, outs, 3), "a call");
    expect(!check_rows_call(n, 0, ins, 3, outs, 3), "no rows in a call");
    expect(check_rows_call(n, 5, ins, 3, outs, 3) && check_rows_call(n, -1, ins, 3, outs, 3), "rows out of range");
    expect(check_rows_call(n, 1, ins, 2, outs, 3) && check_rows_call(n, 1, ins, 3, outs, 2) && check_rows_call(n, 1, nullptr, 3, outs, 3) && check_rows_call(n, 1, ins, 3, nullptr, 3), "counts");
    const void *with_null[] = {a, nullptr, b}, *with_odd[] = {odd, b, buf + 48};
    expect(check_rows_call(n, 1, with_null, 3, outs, 3) && check_rows_call(n, 1, with_odd, 3, outs, 3), "pointers");
    void *in_place[] = {buf + 32, o1, o2}, *over_x[] = {buf, o1, o2}, *y_over_r[] = {o0, buf + 32, o2}, *twice[] = {o0, o1, o1};
    expect(!check_rows_call(n, 1, ins, 3, in_place, 3), "the stream in place");
    expect(check_rows_call(n, 1, ins, 3, over_x, 3) && check_rows_call(n, 1, ins, 3, y_over_r, 3) && check_rows_call(n, 1, ins, 3, twice, 3), "shared memory");
    void *odd_scale[] = {o0, o1, buf + 129};
    expect(check_rows_call(n, 1, ins, 3, odd_scale, 3), "scales not aligned");
    expect(token_pitch(1) == 16 && token_pitch(16) == 16 && token_pitch(4097) == 4112, "pitch");
    return failures ? 1 : 0;
}
