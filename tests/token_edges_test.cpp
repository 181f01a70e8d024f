// Sizes and calls of the token operators at their limits (csrc/token_check.h), without a device.
#include "token_check.h"

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

int main(int argc, char **argv) {
    const char *which = argc > 1 ? argv[1] : "";
    if (!std::strcmp(which, "sizes")) sizes();
    else expect(false, "which test?");
    return failures ? 1 : 0;
}
