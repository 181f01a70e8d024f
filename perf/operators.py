"""Performance cases of the operators around an 8-bit product whose activations are quantised token by token.

A block of a language model served in 8-bit integers runs: token_norm (residual stream, norm, bytes and a scale per
token), token_fc (byte products, a scale per token and per channel), token_gate (gated activation, bytes and scales),
token_fc again; and log_probs reads what the last product answers.  `run` computes a case in plain torch operations, or
through this repository's operators where `own` is true.
"""
import functools
import importlib
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
ROW_ZERO = 2.0 ** -100      # rows whose largest magnitude is below this are quantised to zero


def _fc(name, m, k, n, out, bias):
    """Byte tokens [m][k] with a scale each, times weights [n][k] with a scale per channel; `out`: type of the result."""
    case = dict(op="fc", m=m, k=k, n=n, out=out, bias=bias)
    return dict(case, name=name) if name else case


def _norm(name, m, c, io, norm, post, residual, gate_tokens, n=0):
    """norm / post: none | rms | layer, the norm of the stream and the one of the block's output; gate_tokens: tokens
    that share a row of gates (0: no gates); n > 0: the result is quantised and multiplied with weights [n][c]."""
    case = dict(op="norm_fc" if n else "norm", m=m, c=c, io=io, norm=norm, post=post, residual=residual, gate_tokens=gate_tokens, n=n)
    return dict(case, name=name) if name else case


def _gate(name, m, c, io, act, packed, n=0):
    """act: silu | gelu | gelu_tanh | relu | sigmoid; packed: gates and values are the halves of one row; n as above."""
    case = dict(op="gate_fc" if n else "gate", m=m, c=c, io=io, act=act, packed=packed, n=n)
    return dict(case, name=name) if name else case


def _log_probs(name, m, vocab, io, given, top, masked, scale=1.0):
    """given: token ids per row; top: alternatives per row; masked: part of the vocabulary is ruled out (-inf)."""
    case = dict(op="log_probs", m=m, vocab=vocab, io=io, given=given, top=top, masked=masked, scale=scale)
    return dict(case, name=name) if name else case


def listed():
    return [
        # One token of one request through a square projection: weight streaming at its shortest, latency counts.
        _fc("fc_1x4096x4096", 1, 4096, 4096, "bf16", False),
        # A decode step of 16 requests through a wide projection: 134 MB of weights, all from memory.
        _fc("fc_16x8192x16384", 16, 8192, 16384, "bf16", False),
        # Sizes that fill no tile and no 16-byte line, with a bias and full-precision results (a classifier's head).
        _fc("fc_777x1365x3001", 777, 1365, 3001, "f32", True),
        # Prompt processing: a large product that is bound by the tensor cores.
        _fc("fc_8192x4096x8192", 8192, 4096, 8192, "bf16", False),
        # One token's layer norm: the shortest call.
        _norm("norm_1x8192", 1, 8192, "f16", "layer", "none", False, 0),
        # Between two blocks of a prompt: the block's output is normalised, gated and scaled into the stream, the stream normalised.
        _norm("norm_8192x5120", 8192, 5120, "bf16", "rms", "rms", True, 0),
        # A conditioned block, a row of gates for each sequence of 256 tokens, odd width, straight into the next 8-bit product.
        _norm("norm_fc_2048x4097x6144", 2048, 4097, "bf16", "rms", "none", True, 256, n=6144),
        # The gate of a prompt's feed-forward part, both halves in one row.
        _gate("gate_8192x12288", 8192, 12288, "bf16", "silu", True),
        # A small decode batch: gate, bytes, and the product back to the stream's width.
        _gate("gate_fc_33x10240x4096", 33, 10240, "f16", "gelu_tanh", False, n=4096),
        # One step of a sampler that reports 20 alternatives.
        _log_probs("log_probs_1x131072", 1, 131072, "bf16", 1, 20, False),
        # A decode batch with part of the vocabulary ruled out; odd vocabulary, so that rows begin at any address.
        _log_probs("log_probs_300x50001", 300, 50001, "f16", 1, 5, True, scale=1.25),
        # Scoring a long text: full-precision logits.
        _log_probs("log_probs_2048x65536", 2048, 65536, "f32", 1, 1, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """Widths as models have them, multiples of 64 mostly; now and then any number."""
    w = _log(rng, lo, hi)
    return w if rng.random() < 0.2 else max(lo, w // 64 * 64)


MOST_FLOPS = 2 * 8192 * 4096 * 8192
MOST_BYTES = 500e6


def draw(rng):
    while True:
        kind = rng.choice(["fc", "fc", "norm", "norm", "norm_fc", "gate", "gate", "gate_fc", "log_probs", "log_probs"])
        m, io = _log(rng, 1, 16384), rng.choice(["bf16", "bf16", "f16", "f32"])
        n = _width(rng, 64, 16384)
        if kind == "fc":
            case = _fc(None, m, _width(rng, 64, 16384), n, io, rng.random() < 0.4)
        elif kind in ("norm", "norm_fc"):
            io = rng.choice(["bf16", "f16"]) if kind == "norm_fc" else io
            residual = rng.random() < 0.7
            case = _norm(None, m, _width(rng, 64, 16384), io, rng.choice(["rms", "rms", "layer"]), rng.choice(["none", "none", "rms", "layer"]),
                         residual, rng.choice([0, 0, 1, 77, 1024]), n if kind == "norm_fc" else 0)
        elif kind in ("gate", "gate_fc"):
            io = rng.choice(["bf16", "f16"]) if kind == "gate_fc" else io
            case = _gate(None, m, _width(rng, 64, 24576), io, rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu", "sigmoid"]), rng.random() < 0.6,
                         n if kind == "gate_fc" else 0)
        else:
            vocab = _log(rng, 1000, 262144)
            case = _log_probs(None, _log(rng, 1, 4096), vocab if rng.random() < 0.4 else vocab // 64 * 64, io, rng.choice([0, 1, 1, 1, 4]),
                              rng.choice([0, 1, 5, 20, 20]), rng.random() < 0.3, rng.choice([1.0, 1.0, 0.7, 1.25]))
            if case["given"] == 0 and case["top"] == 0:
                continue
        w = work(case)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES:
            return case


def work(case):
    """Each input and weight read once, each output written once; what lies between two operators of a case does not count."""
    m, op = case["m"], case["op"]
    if op == "log_probs":
        e = SIZES[case["io"]]
        return {"bytes": m * case["vocab"] * e + m * (8 * case["given"] + 4 + 8 * case["top"]), "flops": 6 * m * case["vocab"]}
    if op == "fc":
        k, n, e = case["k"], case["n"], SIZES[case["out"]]
        return {"bytes": m * k + n * k + 4 * m + (8 if case["bias"] else 4) * n + m * n * e, "flops": 2 * m * k * n}
    c, n, e = case["c"], case["n"], SIZES[case["io"]]
    product = n * c + 4 * n + m * n * e
    if op in ("gate", "gate_fc"):
        return {"bytes": 2 * m * c * e + (product if n else m * c * e), "flops": 10 * m * c + 2 * m * c * n}
    weights = 4 * c * ((1, 2)[case["norm"] == "layer"] + {"none": 0, "rms": 1, "layer": 2}[case["post"]])
    gates = -(-m // case["gate_tokens"]) * c * e if case["gate_tokens"] else 0
    stream = (3 if case["residual"] else 1) * m * c * e      # the block's output, and the stream read and written
    return {"bytes": stream + gates + weights + (product if n else m * c * e), "flops": 16 * m * c + 2 * m * c * n}


# ---- states -----------------------------------------------------------------------------------------------------------

class _State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    return gen


def _activations(gen, m, c):
    """Activations as transformer blocks have them: normal, a few channels twenty times as large."""
    x = torch.randn(m, c, device="cuda", generator=gen)
    loud = torch.rand(c, device="cuda", generator=gen) < 0.002
    return x * (1 + 19 * loud)


def _byte_weights(gen, n, k):
    """Weights quantised per channel: bytes over the channel's range, scales that give products of about one."""
    w = (torch.randn(n, k, device="cuda", generator=gen) * 32).round_().clamp_(-127, 127).to(torch.int8)
    scale = torch.exp(torch.empty(n, device="cuda").uniform_(math.log(0.5), math.log(2.0), generator=gen)) / (32 * math.sqrt(k))
    return w, scale


def prepare(case, seed):
    if own:
        _use_the_operators_stream()
    gen = _generator(seed)
    m, op = case["m"], case["op"]
    s = _State(case=case)
    if op == "log_probs":
        v, io = case["vocab"], TYPES[case["io"]]
        logits = torch.randn(m, v, device="cuda", generator=gen) * 3
        if case["masked"]:
            logits.masked_fill_(torch.rand(v, device="cuda", generator=gen) < 0.3, -math.inf)
        s.logits = logits.to(io)
        s.ids = torch.randint(0, v, (m, case["given"]), device="cuda", generator=gen, dtype=torch.int32)
    elif op == "fc":
        k, n = case["k"], case["n"]
        pitch = -(-k // 16) * 16      # byte rows begin at multiples of 16
        rows = torch.zeros(m, pitch, dtype=torch.int8, device="cuda")
        rows[:, :k] = (torch.randn(m, k, device="cuda", generator=gen) * 32).round_().clamp_(-127, 127).to(torch.int8)
        s.rows = rows
        s.token_scale = torch.exp(torch.empty(m, device="cuda").uniform_(math.log(0.2), math.log(5.0), generator=gen)) / 32
        s.w, s.channel_scale = _byte_weights(gen, n, k)
        s.bias = torch.randn(n, device="cuda", generator=gen) if case["bias"] else None
    else:
        c, n, io = case["c"], case["n"], TYPES[case["io"]]
        if op in ("gate", "gate_fc"):
            both = torch.cat([torch.randn(m, c, device="cuda", generator=gen) * 2, _activations(gen, m, c)], dim=1).to(io)
            s.ins = [both] if case["packed"] else [both[:, :c].contiguous(), both[:, c:].contiguous()]
        else:
            s.x = _activations(gen, m, c).to(io)
            s.residual = (4 * _activations(gen, m, c)).to(io) if case["residual"] else None
            rows = -(-m // case["gate_tokens"]) if case["gate_tokens"] else 0
            s.gates = torch.randn(rows, c, device="cuda", generator=gen).to(io) if rows else None
            s.weight = 1 + 0.2 * torch.randn(c, device="cuda", generator=gen)
            s.bias = 0.1 * torch.randn(c, device="cuda", generator=gen) if case["norm"] == "layer" else None
            s.post_weight = 1 + 0.2 * torch.randn(c, device="cuda", generator=gen) if case["post"] != "none" else None
            s.post_bias = 0.1 * torch.randn(c, device="cuda", generator=gen) if case["post"] == "layer" else None
            s.residual_scale = 0.75 if case["residual"] else 1.0
        if n:
            s.w, s.channel_scale = _byte_weights(gen, n, c)
    if own:
        _prepare_own(s)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------

EPS = 1e-6


def _plain_norm(x, kind, weight, bias):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    return y if bias is None else y + bias


def _plain_act(g, act):
    if act == "relu":
        return g.clamp(min=0)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-g))
    if act == "silu":
        return g / (1 + torch.exp(-g))
    if act == "gelu":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))


def _plain_quantise(y):
    largest = y.abs().amax(-1, keepdim=True)
    zero = largest < ROW_ZERO
    q = torch.round(y * (127 / largest.clamp(min=ROW_ZERO)))
    return torch.where(zero, 0.0, q), torch.where(zero, 0.0, largest / 127)


def _plain_product(q, token_scale, w, channel_scale, bias, out):
    y = torch.matmul(q.float(), w.float().t()) * token_scale.reshape(-1, 1) * channel_scale
    return (y if bias is None else y + bias).to(out)


def _plain(s):
    case = s.case
    m, op = case["m"], case["op"]
    if op == "fc":
        return _plain_product(s.rows[:, :case["k"]], s.token_scale, s.w, s.channel_scale, s.bias, TYPES[case["out"]])
    if op == "log_probs":
        z = s.logits.float() * case["scale"]
        largest = z.amax(-1, keepdim=True)
        e = torch.exp(z - largest)
        total = e.sum(-1, keepdim=True)
        lse = largest + torch.log(total)
        # -inf has probability zero and takes no part in the entropy
        entropy = lse.squeeze(-1) - torch.where(e > 0, e * z, 0.0).sum(-1) / total.squeeze(-1)
        out = {"entropy": entropy}
        if case["given"]:
            out["given"] = torch.gather(z, 1, s.ids.long()) - lse
        if case["top"]:
            # order of the logits as integers, the lower index first among equals
            bits = (s.logits.float() + 0.0).view(torch.int32)
            order = (bits ^ ((bits >> 31) & 0x7fffffff)).long()
            index = torch.arange(case["vocab"], device=z.device)
            ids = (1 << 32) - 1 - ((order << 32) + ((1 << 32) - 1 - index)).topk(case["top"], dim=-1).values.remainder(1 << 32)
            out["top_ids"] = ids.to(torch.int32)
            out["top"] = torch.gather(z, 1, ids) - lse
        return out
    io = TYPES[case["io"]]
    stream = None
    if op in ("gate", "gate_fc"):
        gate, value = (s.ins[0][:, :case["c"]], s.ins[0][:, case["c"]:]) if case["packed"] else s.ins
        y = _plain_act(gate.float(), case["act"]) * value.float()
    else:
        y = _plain_norm(s.x.float(), case["post"], s.post_weight, s.post_bias)
        if s.gates is not None:
            y = y * s.gates.float().repeat_interleave(case["gate_tokens"], 0)[:m]
        y = y * s.residual_scale
        if s.residual is not None:
            y = s.residual.float() + y
            stream = y.to(io)
        y = _plain_norm(y, case["norm"], s.weight, s.bias)
    out = {"y": _plain_product(*_plain_quantise(y), s.w, s.channel_scale, None, io) if case["n"] else y.to(io)}
    return out if stream is None else dict(out, stream=stream)


# ---- through the operators --------------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _library():
    enn = importlib.import_module("cl-eden-kernel_b200")
    ctx = enn.Context(torch.cuda.current_device())
    return enn, ctx, torch.cuda.ExternalStream(ctx.stream)


def _use_the_operators_stream():
    """The program's torch work runs on the stream of the operators, so that inputs, calls, what reads their results, and memory that is
    given back and used again are in order without events or waits."""
    _, ctx, stream = _library()
    if torch.cuda.current_stream().cuda_stream != ctx.stream:
        torch.cuda.synchronize()
        torch.cuda.set_stream(stream)


class _Op:
    """A prepared operator, released with its last user."""

    def __init__(self, op):
        self.op = op

    def __del__(self):
        self.op.release()


def _prepare_own(s):
    """Prepares the operators on their weights and allocates their results, as a program does before its first call."""
    enn, ctx, _ = _library()
    types = {"f32": enn.F32, "f16": enn.F16, "bf16": enn.BF16}
    norms = {"none": enn.NORM_NONE, "rms": enn.NORM_RMS, "layer": enn.NORM_LAYER}
    acts = {"silu": enn.GATE_SILU, "gelu": enn.GATE_GELU, "gelu_tanh": enn.GATE_GELU_TANH, "relu": enn.GATE_RELU, "sigmoid": enn.GATE_SIGMOID}
    case = s.case
    m, op = case["m"], case["op"]

    def new(shape, dtype):
        return torch.empty(shape, dtype=dtype, device="cuda")

    s.calls = []

    def call(prepared, ins, outs):
        s.calls.append((_Op(prepared), [t.data_ptr() for t in ins], [t.data_ptr() for t in outs]))

    def product(rows, token_scale, k, n, out, bias):
        y = new((m, n), TYPES[out])
        call(enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=k, n=n, out_dtype=types[out]), s.w.data_ptr(), s.channel_scale.data_ptr(),
                          bias.data_ptr() if bias is not None else None), [rows, token_scale], [y])
        return y

    if op == "log_probs":
        d = enn.LogProbsDesc(m=m, vocab=case["vocab"], in_dtype=types[case["io"]], given=case["given"], top=case["top"], scale=case["scale"])
        s.out = {"entropy": new((m,), torch.float32)}
        if case["given"]:
            s.out["given"] = new((m, case["given"]), torch.float32)
        if case["top"]:
            s.out["top_ids"], s.out["top"] = new((m, case["top"]), torch.int32), new((m, case["top"]), torch.float32)
        call(enn.log_probs(ctx, d), [s.logits] + ([s.ids] if case["given"] else []),
             [s.out[k] for k in ("given", "entropy", "top_ids", "top") if k in s.out])
        return
    if op == "fc":
        s.out = product(s.rows, s.token_scale, case["k"], case["n"], case["out"], s.bias)
        return
    c, io = case["c"], TYPES[case["io"]]
    s.out = {}
    if case["n"]:      # bytes and scales between the two operators
        s.bytes, s.scales = new((m, enn.token_pitch(c)), torch.int8), new((m,), torch.float32)
        outs, out_dtype = [s.bytes, s.scales], enn.S8
    else:
        s.out["y"] = new((m, c), io)
        outs, out_dtype = [s.out["y"]], types[case["io"]]
    if op in ("gate", "gate_fc"):
        d = enn.TokenGateDesc(m=m, c=c, act=acts[case["act"]], packed=int(case["packed"]), in_dtype=types[case["io"]], out_dtype=out_dtype)
        call(enn.token_gate(ctx, d), s.ins, outs)
    else:
        d = enn.TokenNormDesc(m=m, c=c, norm=norms[case["norm"]], post_norm=norms[case["post"]], residual=int(case["residual"]),
                              gate_tokens=case["gate_tokens"], io_dtype=types[case["io"]], out_dtype=out_dtype, eps=EPS, post_eps=EPS,
                              residual_scale=s.residual_scale)
        if case["residual"]:
            s.out["stream"] = new((m, c), io)
            outs = [s.out["stream"]] + outs
        vectors = [v.data_ptr() if v is not None else None for v in (s.weight, s.bias, s.post_weight, s.post_bias)]
        call(enn.token_norm(ctx, d, *vectors), [t for t in (s.x, s.residual, s.gates) if t is not None], outs)
    if case["n"]:
        s.out["y"] = product(s.bytes, s.scales, c, case["n"], case["io"], None)


def run(state):
    if not own:
        return _plain(state)
    for op, ins, outs in state.calls:
        op.op.execute_rows(state.case["m"], ins, outs)
    return state.out


# ---- 64 bits ----------------------------------------------------------------------------------------------------------

def _exact_norm(x, kind, weight, bias):
    if kind == "none":
        return x
    mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    variance = ((x - mean) ** 2).mean(-1, keepdim=True)
    y = (x - mean) / torch.sqrt(variance + EPS) * weight.double()
    return y if bias is None else y + bias.double()


def _exact_gate(g, act):
    return {"silu": lambda: g * torch.special.expit(g), "sigmoid": lambda: torch.special.expit(g), "relu": lambda: torch.maximum(g, torch.zeros_like(g)),
            "gelu": lambda: g * torch.special.ndtr(g),
            "gelu_tanh": lambda: g * torch.special.expit(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))}[act]()


def exact(case, seed):
    s = prepare(case, seed)
    m, op = case["m"], case["op"]

    def product(q, scale, bias=None):
        y = (q @ s.w.double().T) * scale[:, None] * s.channel_scale.double()
        return y if bias is None else y + bias.double()

    if op == "fc":
        return product(s.rows[:, :case["k"]].double(), s.token_scale.double(), s.bias)
    if op == "log_probs":
        z = s.logits.double() * case["scale"]
        lse = torch.logsumexp(z, -1)
        p = torch.exp(z - lse[:, None])
        out = {"entropy": lse - torch.nan_to_num(p * z, nan=0.0).sum(-1)}
        if case["given"]:
            out["given"] = torch.gather(z, 1, s.ids.long()) - lse[:, None]
        if case["top"]:
            values, ids = torch.sort(s.logits, dim=-1, descending=True, stable=True)
            out["top_ids"] = ids[:, :case["top"]].to(torch.int32)
            out["top"] = values[:, :case["top"]].double() * case["scale"] - lse[:, None]
        return out
    stream = None
    if op in ("gate", "gate_fc"):
        halves = torch.cat(s.ins, 1).double()
        y = _exact_gate(halves[:, :case["c"]], case["act"]) * halves[:, case["c"]:]
    else:
        y = _exact_norm(s.x.double(), case["post"], s.post_weight, s.post_bias) * s.residual_scale
        if s.gates is not None:
            y = y * s.gates.double()[torch.arange(m, device="cuda") // case["gate_tokens"]]
        if s.residual is not None:
            y = stream = s.residual.double() + y
        y = _exact_norm(y, case["norm"], s.weight, s.bias)
    if case["n"]:
        scale = y.abs().amax(-1) / 127
        y = product(torch.round(y / scale[:, None]), scale)
    return {"y": y} if stream is None else {"y": y, "stream": stream}
