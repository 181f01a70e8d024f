// C entry points of the token operators: prepare, and enn_b200_op_execute_rows.
#include <new>

#include "token_ops.h"

using namespace enn_b200;

namespace {

int32_t tfail(enn_b200_context *ctx, int32_t st, const char *msg) {
    if (ctx) ctx->last_error = msg;
    return st;
}

int32_t cfail(enn_b200_context *ctx, cudaError_t e) {
    if (ctx) ctx->last_error = std::string("token operator: ") + cudaGetErrorString(e);
    return ENN_B200_CUDA_FAILURE;
}

// The device of the context for the length of a call; the caller's current device is put back.
class OnDevice {
  public:
    explicit OnDevice(int device) {
        if (cudaGetDevice(&before_) != cudaSuccess) before_ = device;
        ok_ = before_ == device || cudaSetDevice(device) == cudaSuccess;
        changed_ = ok_ && before_ != device;
    }
    ~OnDevice() {
        if (changed_) cudaSetDevice(before_);
    }
    bool ok() const { return ok_; }

  private:
    int before_ = 0;
    bool ok_ = false, changed_ = false;
};

// A prepared operator under construction, released unless it is handed out.
struct Building {
    enn_b200_op *op = nullptr;
    ~Building() {
        if (op) enn_b200_op_release(op);
    }
    bool start(enn_b200_context *ctx, int kind, const TokenCall &call) {
        op = new (std::nothrow) enn_b200_op();
        if (!op) return false;
        op->ctx = ctx;
        op->kind = kind;
        op->impl = op->info.impl = ENN_B200_IMPL_ELTWISE;
        op->info.kernel_launches = 1;
        op->token = new (std::nothrow) TokenState();
        if (!op->token) return false;
        op->token->call = call;
        op->token->sms = ctx->launch_sms();
        for (int i = 0; i < call.n_in; ++i) op->info.in_bytes += call.in_bytes[i];
        for (int o = 0; o < call.n_out; ++o) op->info.out_bytes += call.out_bytes[o];
        op->info.algorithmic_bytes = op->info.in_bytes + op->info.out_bytes;
        op->info.out_n = call.m;
        op->info.out_h = op->info.out_w = 1;
        return true;
    }
    // `width` bytes of each of `height` rows, from host or device memory, into an allocation of the operator with `pitch` bytes per row,
    // zeros beyond the width.  (A two-dimensional copy of odd widths takes milliseconds for a few thousand rows.)
    cudaError_t rows(const void *src, int32_t width, int32_t height, int64_t pitch, void **dst) {
        const size_t bytes = static_cast<size_t>(width) * height;
        cudaError_t e = cudaMalloc(dst, static_cast<size_t>(pitch) * height);
        if (e != cudaSuccess) return e;
        op->owned.push_back(*dst);
        if (width == pitch) return cudaMemcpyAsync(*dst, src, bytes, cudaMemcpyDefault, op->ctx->stream);
        void *dense = nullptr;
        if ((e = cudaMalloc(&dense, bytes)) != cudaSuccess) return e;
        e = cudaMemcpyAsync(dense, src, bytes, cudaMemcpyDefault, op->ctx->stream);
        if (e == cudaSuccess) e = launch_pad_rows(dense, width, height, pitch, *dst, op->ctx->stream);
        const cudaError_t done = cudaStreamSynchronize(op->ctx->stream);
        cudaFree(dense);
        return e == cudaSuccess ? done : e;
    }
    // `copies` times, copy i shifted by i floats within `stride`, zeros around each.
    cudaError_t vector(const float *src, int32_t n, const float **dst, int copies = 1, int32_t stride = 0) {
        if (!src) return cudaSuccess;
        op->info.algorithmic_bytes += int64_t{4} * n;
        const size_t bytes = sizeof(float) * static_cast<size_t>(n);
        float *d = nullptr;
        const size_t around = copies > 1 ? 16 : 0, all = bytes + sizeof(float) * (static_cast<size_t>(stride) * (copies - 1) + copies + 2 * around);
        cudaError_t e = cudaMalloc(&d, all);
        if (e != cudaSuccess) return e;
        op->owned.push_back(d);
        e = cudaMemsetAsync(d, 0, all, op->ctx->stream);
        d += around;
        for (int i = 0; i < copies && e == cudaSuccess; ++i)
            e = cudaMemcpyAsync(d + static_cast<size_t>(i) * stride + i, src, bytes, cudaMemcpyDefault, op->ctx->stream);
        *dst = d;
        return e;
    }
    // Hands the operator out once its constants have arrived: their sources may go then.
    int32_t finish(enn_b200_op **out) {
        const cudaError_t e = op->owned.empty() ? cudaSuccess : cudaStreamSynchronize(op->ctx->stream);
        if (e != cudaSuccess) return cfail(op->ctx, e);
        *out = op;
        op = nullptr;
        return ENN_B200_SUCCESS;
    }
};

}  // namespace

namespace enn_b200 {
bool tc_available(const enn_b200_context *ctx);      // gemm_tc.cu
void token_release(enn_b200_op *op) {
    if (op->token->fc.err_host) cudaFreeHost(op->token->fc.err_host);
    delete op->token;
    op->token = nullptr;
}
}  // namespace enn_b200

extern "C" {

int64_t enn_b200_token_pitch(int32_t c) { return c > 0 ? token_pitch(c) : 0; }

int32_t enn_b200_token_fc_prepare(enn_b200_context *ctx, const enn_b200_token_fc_desc *d, const int8_t *weights, const float *channel_scales,
                                  const float *bias, enn_b200_op **out) {
    if (!ctx || !d || !weights || !channel_scales || !out) return tfail(ctx, ENN_B200_INVALID_PARAMS, "null argument");
    *out = nullptr;
    TokenCall call;
    if (const char *wrong = check_token_fc(*d, &call)) return tfail(ctx, ENN_B200_INVALID_PARAMS, wrong);
    OnDevice dev(ctx->device);
    if (!dev.ok()) return tfail(ctx, ENN_B200_CUDA_FAILURE, "the context's device cannot be selected");
    Building b;
    if (!b.start(ctx, OP_TOKEN_FC, call)) return tfail(ctx, ENN_B200_FAILURE, "out of host memory");
    TokenState &t = *b.op->token;
    t.out_dtype = d->out_dtype;
    t.fc.k = d->k;
    t.fc.n = d->n;
    t.fc.in_pitch = d->in_pitch ? d->in_pitch : token_pitch(d->k);
    t.fc.w_pitch = token_pitch(d->k);
    void *w = nullptr;
    cudaError_t e = b.rows(weights, d->k, d->n, t.fc.w_pitch, &w);
    t.fc.w = static_cast<const int8_t *>(w);
    if (e == cudaSuccess) e = b.vector(channel_scales, d->n, &t.fc.channel_scale);
    if (e == cudaSuccess) e = b.vector(bias, d->n, &t.fc.bias);
    if (e != cudaSuccess) return cfail(ctx, e);
    if (tc_available(ctx) && (e = token_fc_plan(b.op)) != cudaSuccess) return cfail(ctx, e);
    b.op->impl = b.op->info.impl = t.fc.err_dev ? ENN_B200_IMPL_TCGEN05 : ENN_B200_IMPL_DIRECT;
    b.op->info.macs = token_macs(d->m, d->k, d->n);
    b.op->info.algorithmic_bytes += static_cast<int64_t>(d->n) * d->k;
    b.op->info.out_c = d->n;
    return b.finish(out);
}

int32_t enn_b200_token_norm_prepare(enn_b200_context *ctx, const enn_b200_token_norm_desc *d, const float *weight, const float *bias,
                                    const float *post_weight, const float *post_bias, enn_b200_op **out) {
    if (!ctx || !d || !out) return tfail(ctx, ENN_B200_INVALID_PARAMS, "null argument");
    *out = nullptr;
    TokenCall call;
    if (const char *wrong = check_token_norm(*d, &call)) return tfail(ctx, ENN_B200_INVALID_PARAMS, wrong);
    if ((d->norm == ENN_B200_NORM_NONE && (weight || bias)) || (d->post_norm == ENN_B200_NORM_NONE && (post_weight || post_bias)))
        return tfail(ctx, ENN_B200_INVALID_PARAMS, "token_norm: a weight or bias without its norm");
    OnDevice dev(ctx->device);
    if (!dev.ok()) return tfail(ctx, ENN_B200_CUDA_FAILURE, "the context's device cannot be selected");
    Building b;
    if (!b.start(ctx, OP_TOKEN_NORM, call)) return tfail(ctx, ENN_B200_FAILURE, "out of host memory");
    TokenState &t = *b.op->token;
    t.in_dtype = d->io_dtype;
    t.out_dtype = d->out_dtype;
    t.residual = d->residual != 0;
    NormParams &p = t.norm;
    p.c = d->c;
    p.norm = d->norm; p.post_norm = d->post_norm;
    p.gate_tokens = d->gate_tokens;
    p.eps = d->eps; p.post_eps = d->post_eps; p.residual_scale = d->residual_scale;
    p.pitch = token_pitch(d->c);
    p.stride = (d->c + 3) / 4 * 4 + 16;
    cudaError_t e = b.vector(weight, d->c, &p.weight, 4, p.stride);
    if (e == cudaSuccess) e = b.vector(bias, d->c, &p.bias, 4, p.stride);
    if (e == cudaSuccess) e = b.vector(post_weight, d->c, &p.post_weight, 4, p.stride);
    if (e == cudaSuccess) e = b.vector(post_bias, d->c, &p.post_bias, 4, p.stride);
    if (e != cudaSuccess) return cfail(ctx, e);
    b.op->info.out_c = d->c;
    return b.finish(out);
}

int32_t enn_b200_token_gate_prepare(enn_b200_context *ctx, const enn_b200_token_gate_desc *d, enn_b200_op **out) {
    if (!ctx || !d || !out) return tfail(ctx, ENN_B200_INVALID_PARAMS, "null argument");
    *out = nullptr;
    TokenCall call;
    if (const char *wrong = check_token_gate(*d, &call)) return tfail(ctx, ENN_B200_INVALID_PARAMS, wrong);
    Building b;
    if (!b.start(ctx, OP_TOKEN_GATE, call)) return tfail(ctx, ENN_B200_FAILURE, "out of host memory");
    TokenState &t = *b.op->token;
    t.in_dtype = d->in_dtype;
    t.out_dtype = d->out_dtype;
    t.packed = d->packed != 0;
    t.gate = GateParams{d->c, d->act, static_cast<int64_t>(d->c) * (d->packed ? 2 : 1), token_pitch(d->c)};
    b.op->info.out_c = d->c;
    return b.finish(out);
}

int32_t enn_b200_log_probs_prepare(enn_b200_context *ctx, const enn_b200_log_probs_desc *d, enn_b200_op **out) {
    if (!ctx || !d || !out) return tfail(ctx, ENN_B200_INVALID_PARAMS, "null argument");
    *out = nullptr;
    TokenCall call;
    if (const char *wrong = check_log_probs(*d, &call)) return tfail(ctx, ENN_B200_INVALID_PARAMS, wrong);
    Building b;
    if (!b.start(ctx, OP_LOG_PROBS, call)) return tfail(ctx, ENN_B200_FAILURE, "out of host memory");
    TokenState &t = *b.op->token;
    t.in_dtype = d->in_dtype;
    t.log_probs = LogProbsParams{d->vocab, d->given, d->top, d->scale, d->in_pitch ? d->in_pitch : static_cast<int64_t>(d->vocab)};
    b.op->info.out_c = d->given + 1 + 2 * d->top;
    return b.finish(out);
}

int32_t enn_b200_op_execute_rows(enn_b200_op *op, int32_t rows, const void *const *ins, int32_t n_in, void *const *outs, int32_t n_out) {
    if (!op) return ENN_B200_INVALID_PARAMS;
    enn_b200_context *ctx = op->ctx;
    if (!op->token) return tfail(ctx, ENN_B200_INVALID_PARAMS, "not a token operator");
    const TokenState &t = *op->token;
    if (const char *wrong = check_rows_call(t.call, rows, ins, n_in, outs, n_out)) return tfail(ctx, ENN_B200_INVALID_PARAMS, wrong);
    if (const char *wrong = check_rows_memory(t.call, rows, ins, outs)) return tfail(ctx, ENN_B200_INVALID_PARAMS, wrong);
    if (t.fc.gave_up()) return tfail(ctx, ENN_B200_CUDA_FAILURE, "token_fc: the kernel gave up on a barrier wait earlier");
    if (rows == 0) return ENN_B200_SUCCESS;
    OnDevice dev(ctx->device);
    if (!dev.ok()) return tfail(ctx, ENN_B200_CUDA_FAILURE, "the context's device cannot be selected");
    cudaError_t e = cudaErrorInvalidValue;
    switch (op->kind) {
        case OP_TOKEN_FC: e = token_fc_launch(op, rows, ins, outs); break;
        case OP_TOKEN_NORM: e = token_norm_launch(op, rows, ins, outs); break;
        case OP_TOKEN_GATE: e = token_gate_launch(op, rows, ins, outs); break;
        case OP_LOG_PROBS: e = log_probs_launch(op, rows, ins, outs); break;
    }
    return e == cudaSuccess ? ENN_B200_SUCCESS : cfail(ctx, e);
}

}  // extern "C"
