"""GPU tests of the token operators against plain forms in 64 bits.

Tolerances count roundings, u = 2^-24 for a float operation and half an eps for the final rounding; each is derived beside
its test and holds for any order of the sums with chains of up to SERIAL additions.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SERIAL = 200      # additions one after the other in any partial sum, with those that join the partial sums
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GUARD = 3         # rows past the last that must stay as they were


def code(enn, name):
    return {"f32": enn.F32, "f16": enn.F16, "bf16": enn.BF16, "s8": enn.S8}[name]


def half_eps(name):
    return torch.finfo(TYPES[name]).eps / 2


def rand(seed, *shape):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=gen)


def guarded(rows, cols, dtype, offset=0):
    """A buffer of rows + GUARD rows filled with a pattern, `offset` elements into its allocation."""
    size = (rows + GUARD) * cols + offset
    flat = (torch.arange(size, device="cuda") % 97).to(dtype)
    return flat[offset:].view(rows + GUARD, cols)


def untouched(buf, rows):
    flat = buf.reshape(buf.shape[0], -1)
    want = guarded(buf.shape[0] - GUARD, flat.shape[1], buf.dtype)
    return torch.equal(flat[rows:].float(), want[rows:].float())


def execute(op, rows, ins, outs):
    torch.cuda.synchronize()
    op.execute_rows(rows, [t.data_ptr() for t in ins], [t.data_ptr() for t in outs])
    op.ctx.sync()


# ---- token_fc ---------------------------------------------------------------------------------------------------------

def fc_inputs(seed, m, k, n, pitch=0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    q = torch.randint(-127, 128, (m, pitch or -(-k // 16) * 16), device="cuda", generator=gen).to(torch.int8)
    w = torch.randint(-127, 128, (n, k), device="cuda", generator=gen).to(torch.int8)
    s = torch.rand(m, device="cuda", generator=gen) * 0.05
    sw = torch.rand(n, device="cuda", generator=gen) * 0.01
    bias = torch.randn(n, device="cuda", generator=gen) * 50
    return q, w, s, sw, bias


def fc_check(got, q, w, s, sw, bias, out, k):
    acc = torch.round(q[:, :k].double() @ w.double().T)         # exact: below 2^53
    prod = acc * s.double()[:, None] * sw.double()
    want = prod if bias is None else prod + bias.double()
    # the sum rounded to 24 bits, two products, one sum; then the result's rounding
    tol = 4 * U * (prod.abs() + want.abs()) + half_eps(out) * want.abs() * (1 + 8 * U) + (2.0 ** -25 if out == "f16" else 1e-40)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{float((err / tol).max())} of the tolerance"


FC_SHAPES = [(1, 1, 1), (1, 64, 64), (1, 4096, 256), (2, 16, 17), (7, 33, 130), (16, 512, 128), (17, 129, 255), (33, 1000, 96), (64, 64, 512),
             (65, 640, 321), (127, 95, 63), (128, 128, 128), (129, 144, 129), (200, 1365, 301), (256, 2048, 256), (257, 272, 520), (300, 16, 1000),
             (513, 384, 767), (1024, 256, 1030)]


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k,n", FC_SHAPES)
def test_token_fc(enn, ctx, m, k, n, out):
    q, w, s, sw, bias = fc_inputs(m * 1000 + n, m, k, n)
    for b in (None, bias):
        op = enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=k, n=n, out_dtype=code(enn, out)), w.cpu().numpy(), sw.cpu().numpy(), None if b is None else b.cpu().numpy())
        y = guarded(m, n, TYPES[out])
        execute(op, m, [q, s], [y])
        fc_check(y[:m], q, w, s, sw, b, out, k)
        assert untouched(y, m)
        op.release()


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k,n", [(129, 64, 19000), (300, 129, 9001), (1000, 200, 4000), (1037, 1365, 5003), (2500, 16, 2000), (2049, 900, 1795), (4097, 1040, 2304)])
def test_token_fc_large_products(enn, ctx, m, k, n, out):
    """Products whose tiles occupy the device, ragged in every direction."""
    q, w, s, sw, bias = fc_inputs(m + n, m, k, n)
    for b in (None, bias):
        op = enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=k, n=n, out_dtype=code(enn, out)), w.data_ptr(), sw.data_ptr(), None if b is None else b.data_ptr())
        y = guarded(m, n, TYPES[out])
        execute(op, m, [q, s], [y])
        fc_check(y[:m], q, w, s, sw, b, out, k)
        assert untouched(y, m)
        op.release()


def test_token_fc_large_product_with_fewer_rows_and_any_address(enn, ctx):
    m, k, n = 2000, 300, 4100
    q, w, s, sw, _ = fc_inputs(3, m, k, n)
    s[1234:] = math.nan
    op = enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=k, n=n, out_dtype=enn.F16), w.data_ptr(), sw.data_ptr())
    y = guarded(m, n, torch.float16)
    execute(op, 1234, [q, s], [y])
    fc_check(y[:1234], q[:1234], w, s[:1234], sw, None, "f16", k)
    assert untouched(y, 1234)
    y = guarded(m, n, torch.float16, 1)
    execute(op, 1234, [q, s], [y])
    fc_check(y[:1234], q[:1234], w, s[:1234], sw, None, "f16", k)
    op.release()


@pytest.mark.parametrize("rows", [0, 1, 5, 31, 64, 100, 190, 300])
def test_token_fc_fewer_rows_than_prepared(enn, ctx, rows):
    """One handle serves decode steps and prompts: rows past the given number are neither read nor written."""
    m, k, n = 300, 320, 200
    q, w, s, sw, _ = fc_inputs(5, m, k, n)
    s[rows:] = math.nan
    op = enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=k, n=n, out_dtype=enn.BF16), w.data_ptr(), sw.data_ptr())
    y = guarded(m, n, torch.bfloat16)
    execute(op, rows, [q, s], [y])
    assert untouched(y, rows)
    fc_check(y[:rows], q[:rows], w, s[:rows], sw, None, "bf16", k)
    op.release()


@pytest.mark.parametrize("m,k,n", [(1, 131071, 3), (3, 65536, 20), (130, 65552, 140)])
def test_token_fc_largest_sums(enn, ctx, m, k, n):
    """Every product 127 * 127 or -127 * 127: sums of up to 2.1e9 without a wrap."""
    q = torch.full((m, -(-k // 16) * 16), 127, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), 127, dtype=torch.int8, device="cuda")
    w[1::2] = -127
    s, sw = torch.full((m,), 1e-3, device="cuda"), torch.full((n,), 1e-3, device="cuda")
    op = enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=k, n=n, out_dtype=enn.F32), w.data_ptr(), sw.data_ptr())
    y = guarded(m, n, torch.float32)
    execute(op, m, [q, s], [y])
    fc_check(y[:m], q, w, s, sw, None, "f32", k)
    op.release()


@pytest.mark.parametrize("m", [1, 20, 150])
@pytest.mark.parametrize("q_offset,pitch,out_offset", [(0, 101, 0), (1, 112, 0), (0, 208, 1), (3, 150, 3), (16, 112, 8)])
def test_token_fc_addresses_and_pitches(enn, ctx, m, q_offset, pitch, out_offset):
    k, n = 100, 72
    q, w, s, sw, _ = fc_inputs(9, m, k, n, pitch)
    flat = torch.zeros(q.numel() + 64, dtype=torch.int8, device="cuda")
    moved = flat[q_offset:q_offset + q.numel()].view(q.shape)
    moved.copy_(q)
    op = enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=k, n=n, out_dtype=enn.F16, in_pitch=pitch), w.data_ptr(), sw.data_ptr())
    y = guarded(m, n, torch.float16, out_offset)
    execute(op, m, [moved, s], [y])
    fc_check(y[:m], q, w, s, sw, None, "f16", k)
    op.release()


def test_token_fc_bytes_past_the_row_do_not_count(enn, ctx):
    """What lies between k and the pitch may be anything, the byte -128 too."""
    for m in (1, 40, 200):
        q, w, s, sw, _ = fc_inputs(11, m, 90, 150, 96)
        q[:, 90:] = -128
        op = enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=90, n=150, out_dtype=enn.F32), w.data_ptr(), sw.data_ptr())
        y = guarded(m, 150, torch.float32)
        execute(op, m, [q, s], [y])
        fc_check(y[:m], q, w, s, sw, None, "f32", 90)
        op.release()


def test_token_fc_rows_that_stand_for_nothing(enn, ctx):
    """Scale 0 gives the bias, scale NaN gives NaN, and neither reaches another row."""
    m, k, n = 70, 128, 96
    q, w, s, sw, bias = fc_inputs(12, m, k, n)
    s[3], s[50], q[3], q[50] = 0.0, math.nan, 0, 0
    op = enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=k, n=n, out_dtype=enn.F32), w.data_ptr(), sw.data_ptr(), bias.data_ptr())
    y = guarded(m, n, torch.float32)
    execute(op, m, [q, s], [y])
    assert torch.equal(y[3], bias) and bool(torch.isnan(y[50]).all())
    keep = torch.tensor([i for i in range(m) if i != 50], device="cuda")
    fc_check(y[:m][keep], q[keep], w, s[keep], sw, bias, "f32", k)
    op.release()


def test_token_fc_implementations_agree(enn, ctx):
    """The direct kernel is the second implementation: equal bits, since the sums are exact and the rest is the same arithmetic."""
    for m, k, n in [(1, 300, 90), (40, 1000, 260), (300, 528, 384)]:
        q, w, s, sw, bias = fc_inputs(13, m, k, n)
        op = enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=k, n=n, out_dtype=enn.F32), w.data_ptr(), sw.data_ptr(), bias.data_ptr())
        a, b = guarded(m, n, torch.float32), guarded(m, n, torch.float32)
        execute(op, m, [q, s], [a])
        op.set_impl(enn.IMPL_DIRECT)
        execute(op, m, [q, s], [b])
        assert torch.equal(a, b)
        op.release()


def test_token_fc_that_gives_up_on_a_wait(enn, ctx):
    """A kernel whose wait ran out leaves a code; later calls fail until it is cleared, and then run as before."""
    for m, n in ((3, 256), (300, 256), (2000, 4096)):
        q, w, s, sw, _ = fc_inputs(14, m, 4096, n)
        op = enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=4096, n=n, out_dtype=enn.F32), w.data_ptr(), sw.data_ptr())
        assert op.info.impl == enn.IMPL_TCGEN05
        y = guarded(m, n, torch.float32)
        op.test_starve_next()
        execute(op, m, [q, s], [y])
        with pytest.raises(enn.EnnError) as e:
            execute(op, m, [q, s], [y])
        assert e.value.status == enn.CUDA_FAILURE and "gave up" in str(e.value)
        op.clear_error()
        execute(op, m, [q, s], [y])
        fc_check(y[:m], q, w, s, sw, None, "f32", 4096)
        op.release()


# ---- token_norm -------------------------------------------------------------------------------------------------------

def norm64(x, kind, eps, weight, bias):
    """norm(x) in 64 bits, the magnitude of its terms, and r."""
    if kind == "none":
        return x, x.abs(), torch.ones_like(x[:, :1])
    mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    r = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    w = torch.ones(x.shape[1], device="cuda", dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    return (x - mean) * r * w + b, (x.abs() + mean.abs()) * r * w.abs() + b.abs(), r * w.abs()


def norm_error(size, x, x_err, kind, eps, weight, bias):
    """Bound of the error of norm(x) in float, given a bound of the error of x: the inputs' errors and the roundings of the
    sums move the row's mean and its root of squares, each by a share of the row's largest relative size."""
    y, terms, gain = norm64(x, kind, eps, weight, bias)
    if kind == "none":
        return y, x_err
    n = SERIAL + 20
    mean_err = (n * U * x.abs().mean(-1, keepdim=True) + x_err.mean(-1, keepdim=True)) if kind == "layer" else 0
    mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    d_err = x_err + mean_err + 2 * U * (x.abs() + mean.abs())
    ms = ((x - mean) ** 2).mean(-1, keepdim=True)
    ms_err = 2 * ((x - mean).abs() * d_err).mean(-1, keepdim=True) + (d_err ** 2).mean(-1, keepdim=True) + n * U * ms
    r_rel = ms_err / (ms + eps) + 8 * U            # half of it, with room for the second order
    y_err = d_err * gain + r_rel * (x - mean).abs() * gain + 6 * U * terms
    return y, y_err


def norm_reference(case, x, r, gate, vectors, residual_scale, eps):
    w, b, pw, pb = vectors
    x = x.double()
    y, err = norm_error(x.shape[1], x, torch.zeros_like(x), case["post"], eps, pw, pb)
    if gate is not None:
        g = gate.double()[torch.arange(x.shape[0], device="cuda") // case["gate_tokens"]]
        y, err = y * g, err * g.abs() + U * (y * g).abs()
    y, err = y * residual_scale, err * abs(residual_scale) + U * (y * residual_scale).abs()
    stream = None
    if r is not None:
        y = y + r.double()
        err = err + U * y.abs()
        stream = (y, err)
    return stream, norm_error(x.shape[1], y, err, case["norm"], eps, w, b)


def check_close(got, want, err, name):
    tiny = {"f32": 1e-38, "bf16": 1e-38, "f16": 2.0 ** -25}[name]
    tol = err * (1 + half_eps(name)) + half_eps(name) * want.abs() + tiny
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), f"{float((off / tol).max())} of the tolerance"


def check_bytes(q, s, want, err, c):
    """Byte rows: half a step off at most, with the errors of the values and of the scale."""
    largest = want.abs().amax(-1)
    worst = err.amax(-1)
    assert bool(((s.double() - largest / 127).abs() <= worst / 127 + 2 * U * largest / 127).all())
    step = s.double()[:, None]
    off = (q[:, :c].double() * step - want).abs()
    tol = 0.5 * step * (1 + 300 * U) + err + worst[:, None] + 4 * U * want.abs()
    assert bool((off <= tol).all()), f"{float((off / tol.clamp(min=1e-300)).max())} of the tolerance"
    assert bool((q[:, c:] == 0).all()) and int(q[:, :c].abs().max()) <= 127


def run_norm(enn, ctx, case, seed=1, rows=None, eps=1e-6, residual_scale=0.7, x=None, r=None):
    m, c, io, out = case["m"], case["c"], case["io"], case["out"]
    rows = m if rows is None else rows
    x = (rand(seed, m, c) * 2 + 0.3).to(TYPES[io]) if x is None else x
    r = (rand(seed + 1, m, c) * 3).to(TYPES[io]) if r is None and case["residual"] else r
    gt = case["gate_tokens"]
    gate = rand(seed + 2, -(-m // gt), c).to(TYPES[io]) if gt else None
    vec = lambda k, on: 1 + 0.3 * rand(seed + k, c) if on else None      # noqa: E731
    vectors = (vec(3, case["norm"] != "none"), vec(4, case["norm"] == "layer"), vec(5, case["post"] != "none"), vec(6, case["post"] == "layer"))
    kinds = {"none": enn.NORM_NONE, "rms": enn.NORM_RMS, "layer": enn.NORM_LAYER}
    d = enn.TokenNormDesc(m=m, c=c, norm=kinds[case["norm"]], post_norm=kinds[case["post"]], residual=int(case["residual"]), gate_tokens=gt,
                          io_dtype=code(enn, io), out_dtype=code(enn, out), eps=eps, post_eps=eps, residual_scale=residual_scale)
    op = enn.token_norm(ctx, d, *[None if v is None else v.cpu().numpy() for v in vectors])
    ins = [x] + ([r] if case["residual"] else []) + ([gate] if gt else [])
    pitch = enn.token_pitch(c)
    outs = [guarded(m, c, TYPES[io])] if case["residual"] else []
    outs += [guarded(m, pitch, torch.int8), guarded(m, 1, torch.float32)] if out == "s8" else [guarded(m, c, TYPES[out])]
    execute(op, rows, ins, outs)
    op.release()
    for o in outs:
        assert untouched(o, rows)
    if rows == 0:
        return
    stream, (y, err) = norm_reference(case, x[:rows], r[:rows] if r is not None else None, gate, vectors, float(np.float32(residual_scale)), float(np.float32(eps)))
    if case["residual"]:
        check_close(outs[0][:rows], *stream, io)
    if out == "s8":
        check_bytes(outs[-2][:rows], outs[-1][:rows, 0], y, err, c)
    else:
        check_close(outs[-1][:rows], y, err, out)


def norm_case(m, c, io="bf16", out="bf16", norm="rms", post="none", residual=True, gate_tokens=0):
    return dict(m=m, c=c, io=io, out=out, norm=norm, post=post, residual=residual, gate_tokens=gate_tokens)


@pytest.mark.parametrize("out", ["f32", "f16", "bf16", "s8"])
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,c", [(1, 1), (3, 8), (5, 64), (2, 100), (9, 513), (4, 1024), (3, 4096), (2, 4097), (2, 8192), (1, 12288)])
def test_token_norm_types_and_widths(enn, ctx, m, c, io, out):
    run_norm(enn, ctx, norm_case(m, c, io, out, "rms", "none", True))
    run_norm(enn, ctx, norm_case(m, c, io, out, "layer", "layer", True, 2))


@pytest.mark.parametrize("out", ["bf16", "s8"])
@pytest.mark.parametrize("gate_tokens", [0, 1, 7, 1000])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("post", ["none", "rms", "layer"])
@pytest.mark.parametrize("norm", ["none", "rms", "layer"])
def test_token_norm_forms(enn, ctx, norm, post, residual, gate_tokens, out):
    run_norm(enn, ctx, norm_case(20, 264, "bf16", out, norm, post, residual, gate_tokens))


@pytest.mark.parametrize("c", [16384, 20000, 32761, 32768])
@pytest.mark.parametrize("out", ["f16", "s8"])
def test_token_norm_widest_rows(enn, ctx, c, out):
    run_norm(enn, ctx, norm_case(3, c, "f16", out, "rms", "rms", True, 2))
    run_norm(enn, ctx, norm_case(3, c, "f32", out, "layer", "none", False))


@pytest.mark.parametrize("m", [2, 300])
@pytest.mark.parametrize("c", [8185, 8192, 8193, 16376, 16377, 16384, 16385, 24569, 24576, 24577])
def test_token_norm_widths_around_a_block_s(enn, ctx, m, c):
    run_norm(enn, ctx, norm_case(m, c, "bf16", "s8", "rms", "none", True))
    run_norm(enn, ctx, norm_case(m, c, "f32", "f32", "layer", "rms", True, 3))


@pytest.mark.parametrize("rows", [0, 1, 16, 37])
def test_token_norm_fewer_rows_than_prepared(enn, ctx, rows):
    for out in ("bf16", "s8"):
        run_norm(enn, ctx, norm_case(40, 520, "bf16", out, "rms", "rms", True, 3), rows=rows)


@pytest.mark.parametrize("io,out", [("bf16", "bf16"), ("f16", "s8"), ("f32", "f32"), ("bf16", "f32"), ("f32", "s8")])
@pytest.mark.parametrize("m,c", [(700, 4097), (900, 1001), (3000, 67), (400, 6150), (300, 9), (650, 2044), (310, 12301)])
def test_token_norm_odd_widths_many_rows(enn, ctx, m, c, io, out):
    run_norm(enn, ctx, norm_case(m, c, io, out, "layer", "rms", True, 50))
    run_norm(enn, ctx, norm_case(m, c, io, out, "rms", "none", False))


@pytest.mark.parametrize("x_off,r_off,g_off,h_off,y_off", [(1, 0, 0, 0, 0), (0, 3, 0, 0, 0), (5, 5, 5, 5, 5), (2, 2, 1, 2, 7), (0, 0, 0, 4, 0), (0, 0, 0, 0, 1)])
def test_token_norm_tensors_on_different_lines(enn, ctx, x_off, r_off, g_off, h_off, y_off):
    """Every tensor at an address of its own, rows of odd and even widths."""
    for m, c, io, out in ((400, 515, "bf16", "bf16"), (30, 1024, "f16", "s8"), (310, 4096, "bf16", "s8"), (3, 32768, "f32", "f16")):
        place = lambda t, off: torch.zeros(t.numel() + 16, dtype=t.dtype, device="cuda")[off:off + t.numel()].view(t.shape).copy_(t)      # noqa: E731
        x, r, g = place(rand(1, m, c).to(TYPES[io]), x_off), place(rand(2, m, c).to(TYPES[io]), r_off), place(rand(3, -(-m // 7), c).to(TYPES[io]), g_off)
        vectors = tuple(1 + 0.3 * rand(k, c) for k in range(4))
        torch.cuda.synchronize()
        d = enn.TokenNormDesc(m=m, c=c, norm=enn.NORM_LAYER, post_norm=enn.NORM_LAYER, residual=1, gate_tokens=7, io_dtype=code(enn, io), out_dtype=code(enn, out), eps=1e-6,
                              post_eps=1e-6, residual_scale=0.5)
        op = enn.token_norm(ctx, d, *[v.data_ptr() for v in vectors])
        h = guarded(m, c, TYPES[io], h_off)
        outs = [h, guarded(m, enn.token_pitch(c), torch.int8, y_off), guarded(m, 1, torch.float32)] if out == "s8" else [h, guarded(m, c, TYPES[out], y_off)]
        execute(op, m, [x, r, g], outs)
        op.release()
        stream, (y, err) = norm_reference(norm_case(m, c, io, out, "layer", "layer", True, 7), x, r, g, vectors, 0.5, float(np.float32(1e-6)))
        check_close(h[:m], *stream, io)
        if out == "s8":
            check_bytes(outs[1][:m], outs[2][:m, 0], y, err, c)
        else:
            check_close(outs[1][:m], y, err, out)


def test_token_norm_many_rows(enn, ctx):
    run_norm(enn, ctx, norm_case(5000, 72, "f32", "s8", "layer", "none", True, 64))
    run_norm(enn, ctx, norm_case(3000, 1536, "bf16", "bf16", "rms", "rms", True))
    run_norm(enn, ctx, norm_case(1500, 2056, "f16", "s8", "rms", "none", True))


def test_token_norm_stream_in_place(enn, ctx):
    m, c = 33, 1000
    x, r = rand(1, m, c).bfloat16(), rand(2, m, c).bfloat16()
    d = enn.TokenNormDesc(m=m, c=c, norm=enn.NORM_RMS, residual=1, io_dtype=enn.BF16, out_dtype=enn.BF16, eps=1e-6, residual_scale=1.0)
    op = enn.token_norm(ctx, d)
    h, y, y2 = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    execute(op, m, [x, r], [h, y])
    execute(op, m, [x, r], [r, y2])
    assert torch.equal(r, h) and torch.equal(y, y2)
    op.release()


@pytest.mark.parametrize("c", [40, 4104])
def test_token_norm_rows_of_zeros_infinities_and_nan(enn, ctx, c):
    """Zero rows: finite with eps > 0 and scale 0; tiny rows count as zero; a NaN or infinity stays in its row."""
    x = torch.zeros(6, c, device="cuda")
    x[1, 3], x[2, c - 1], x[3, 0] = math.inf, math.nan, 1e-32
    x[4], x[5] = rand(3, c), -3e38
    d = enn.TokenNormDesc(m=6, c=c, norm=enn.NORM_NONE, io_dtype=enn.F32, out_dtype=enn.S8, residual_scale=1.0)
    op = enn.token_norm(ctx, d)
    q, s = guarded(6, enn.token_pitch(c), torch.int8), guarded(6, 1, torch.float32)
    execute(op, 6, [x], [q, s])
    op.release()
    s = s[:6, 0]
    assert s[0] == 0 and s[3] == 0 and bool(torch.isnan(s[1:3]).all())
    assert bool((q[:4] == 0).all()) and bool((q[5, :c] == -127).all())
    check_bytes(q[4:6], s[4:6], x[4:6].double(), torch.zeros_like(x[4:6]).double(), c)
    d = enn.TokenNormDesc(m=6, c=c, norm=enn.NORM_RMS, io_dtype=enn.F32, out_dtype=enn.F32, eps=1e-5, residual_scale=1.0)
    op = enn.token_norm(ctx, d)
    y = guarded(6, c, torch.float32)
    execute(op, 6, [x], [y])
    op.release()
    assert bool((y[0] == 0).all()) and bool(torch.isnan(y[1, 3])) and bool(torch.isnan(y[2]).all()) and bool(torch.isfinite(y[4]).all())


@pytest.mark.parametrize("offset", [1, 2, 4])
def test_token_norm_any_address(enn, ctx, offset):
    """Rows that begin between 16-byte lines, inputs and outputs alike."""
    m, c = 5, 768
    for out in ("bf16", "s8"):
        flat = torch.zeros(2, m * c + 8, dtype=torch.bfloat16, device="cuda")
        x, r = flat[0, offset:offset + m * c].view(m, c), flat[1, offset:offset + m * c].view(m, c)
        x.copy_(rand(1, m, c))
        r.copy_(rand(2, m, c))
        d = enn.TokenNormDesc(m=m, c=c, norm=enn.NORM_LAYER, residual=1, io_dtype=enn.BF16, out_dtype=code(enn, out), eps=1e-6, residual_scale=1.0)
        op = enn.token_norm(ctx, d)
        h = guarded(m, c, torch.bfloat16, offset)
        outs = [h, guarded(m, c, torch.int8, offset), guarded(m, 1, torch.float32)] if out == "s8" else [h, guarded(m, c, torch.bfloat16, offset)]
        execute(op, m, [x, r], outs)
        op.release()
        case = norm_case(m, c, "bf16", out, "layer")
        stream, (y, err) = norm_reference(case, x, r, None, (None,) * 4, 1.0, float(np.float32(1e-6)))
        check_close(h[:m], *stream, "bf16")
        if out == "s8":
            check_bytes(outs[1][:m], outs[2][:m, 0], y, err, c)
        else:
            check_close(outs[1][:m], y, err, "bf16")


# ---- token_gate -------------------------------------------------------------------------------------------------------

def act64(g, act):
    """act(g) in 64 bits, and a bound of its error in float: the exponential's argument is at most a few roundings off, the error
    and hyperbolic tangent functions a few roundings of one."""
    if act == "relu":
        return torch.where(g < 0, 0.0, g), torch.zeros_like(g)
    sig = torch.special.expit(g)
    if act == "sigmoid":
        return sig, U * sig * (8 + 4 * g.abs() * (1 - sig))
    if act == "silu":
        return g * sig, U * (g * sig).abs() * (10 + 4 * g.abs() * (1 - sig))
    if act == "gelu":
        return g * torch.special.ndtr(g), U * g.abs() * 6
    v = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    sig = torch.special.expit(v)
    return g * sig, U * g.abs() * 6


def run_gate(enn, ctx, m, c, io, out, act, packed, rows=None, seed=1, spread=3.0):
    rows = m if rows is None else rows
    g, u = (rand(seed, m, c) * spread).to(TYPES[io]), rand(seed + 1, m, c).to(TYPES[io])
    ins = [torch.cat([g, u], 1)] if packed else [g, u]
    acts = {"silu": enn.GATE_SILU, "gelu": enn.GATE_GELU, "gelu_tanh": enn.GATE_GELU_TANH, "relu": enn.GATE_RELU, "sigmoid": enn.GATE_SIGMOID}
    op = enn.token_gate(ctx, enn.TokenGateDesc(m=m, c=c, act=acts[act], packed=int(packed), in_dtype=code(enn, io), out_dtype=code(enn, out)))
    outs = [guarded(m, enn.token_pitch(c), torch.int8), guarded(m, 1, torch.float32)] if out == "s8" else [guarded(m, c, TYPES[out])]
    execute(op, rows, ins, outs)
    op.release()
    a, err = act64(g[:rows].double(), act)
    want = a * u[:rows].double()
    err = err * u[:rows].double().abs() + U * want.abs()
    for o in outs:
        assert untouched(o, rows)
    if rows and out == "s8":
        check_bytes(outs[0][:rows], outs[1][:rows, 0], want, err, c)
    elif rows:
        check_close(outs[0][:rows], want, err, out)


@pytest.mark.parametrize("out", ["f32", "f16", "bf16", "s8"])
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,c,packed", [(1, 1, True), (3, 9, False), (2, 64, True), (4, 1000, True), (5, 2047, True), (3, 2048, False), (2, 11008, True), (1, 24576, False)])
def test_token_gate_types_and_widths(enn, ctx, m, c, packed, io, out):
    run_gate(enn, ctx, m, c, io, out, "silu", packed)


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("out", ["f32", "s8"])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"])
def test_token_gate_activations(enn, ctx, act, out, packed):
    run_gate(enn, ctx, 17, 520, "f32", out, act, packed)
    run_gate(enn, ctx, 3, 520, "f32", out, act, packed, spread=30.0)


@pytest.mark.parametrize("c", [32768, 50001, 65536])
@pytest.mark.parametrize("out", ["bf16", "s8"])
def test_token_gate_widest_rows(enn, ctx, c, out):
    run_gate(enn, ctx, 2, c, "bf16", out, "silu", True)


@pytest.mark.parametrize("m", [2, 300])
@pytest.mark.parametrize("out", ["bf16", "s8"])
@pytest.mark.parametrize("c", [8185, 8193, 16376, 16377, 16383, 16384, 16385])
def test_token_gate_widths_around_a_segment_s(enn, ctx, m, c, out):
    run_gate(enn, ctx, m, c, "bf16", out, "silu", True)
    run_gate(enn, ctx, m, c, "f32", out, "relu", False)


@pytest.mark.parametrize("out", ["bf16", "s8"])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("m,c", [(700, 4099), (900, 1001), (2500, 67), (300, 9), (650, 2044), (40, 8193), (5, 40001)])
def test_token_gate_odd_widths_many_rows(enn, ctx, m, c, packed, out):
    run_gate(enn, ctx, m, c, "bf16", out, "silu", packed)
    run_gate(enn, ctx, min(m, 100), c, "f32", out, "gelu_tanh", packed)


@pytest.mark.parametrize("g_off,u_off,y_off", [(1, 0, 0), (0, 3, 0), (0, 0, 1), (5, 5, 5), (2, 6, 3), (4, 0, 4)])
def test_token_gate_tensors_on_different_lines(enn, ctx, g_off, u_off, y_off):
    """Gates, values and results at addresses of their own, NaN before and behind what is read."""
    def place(t, off):
        flat = torch.full((t.numel() + 16,), float("nan"), dtype=t.dtype, device="cuda")
        flat[off:off + t.numel()] = t.reshape(-1)
        return flat[off:off + t.numel()].view(t.shape)
    for m, c, io, out in ((400, 515, "bf16", "bf16"), (400, 516, "f32", "f32"), (30, 1024, "f16", "s8"), (310, 4096, "f32", "s8"), (310, 4099, "bf16", "f32"), (1, 7, "f16", "f16"), (3, 20000, "f32", "bf16")):
        g, u = place((rand(1, m, c) * 3).to(TYPES[io]), g_off), place(rand(2, m, c).to(TYPES[io]), u_off)
        op = enn.token_gate(ctx, enn.TokenGateDesc(m=m, c=c, act=enn.GATE_SILU, packed=0, in_dtype=code(enn, io), out_dtype=code(enn, out)))
        outs = [guarded(m, enn.token_pitch(c), torch.int8, y_off), guarded(m, 1, torch.float32)] if out == "s8" else [guarded(m, c, TYPES[out], y_off)]
        execute(op, m, [g, u], outs)
        op.release()
        a, err = act64(g.double(), "silu")
        want = a * u.double()
        err = err * u.double().abs() + U * want.abs()
        assert torch.equal(outs[0][m:], guarded(m, outs[0].shape[1], outs[0].dtype, y_off)[m:])
        if out == "s8":
            check_bytes(outs[0][:m], outs[1][:m, 0], want, err, c)
        else:
            check_close(outs[0][:m], want, err, out)


def test_token_gate_many_rows(enn, ctx):
    run_gate(enn, ctx, 4000, 200, "bf16", "s8", "silu", True)
    run_gate(enn, ctx, 700, 4000, "f16", "s8", "gelu_tanh", False)
    run_gate(enn, ctx, 700, 4000, "bf16", "bf16", "gelu", True)


@pytest.mark.parametrize("rows", [0, 1, 29])
def test_token_gate_fewer_rows_than_prepared(enn, ctx, rows):
    for out in ("f16", "s8"):
        run_gate(enn, ctx, 30, 264, "f16", out, "silu", True, rows=rows)


def test_token_gate_far_values(enn, ctx):
    """Large gates of either sign: no overflow of the exponential reaches the result, a NaN stays in its row."""
    g = torch.tensor([[-1e4, -100.0, -88.0, 0.0, 88.0, 100.0, 1e4, -1e30]] * 3, device="cuda")
    u = torch.ones_like(g)
    u[2, 5] = math.nan
    for act, want in ((enn.GATE_SILU, [0, 0, 0, 0, 88, 100, 1e4, 0]), (enn.GATE_GELU, [0, 0, 0, 0, 88, 100, 1e4, 0]), (enn.GATE_GELU_TANH, [0, 0, 0, 0, 88, 100, 1e4, 0]),
                      (enn.GATE_SIGMOID, [0, 0, 0, 0.5, 1, 1, 1, 0]), (enn.GATE_RELU, [0, 0, 0, 0, 88, 100, 1e4, 0])):
        op = enn.token_gate(ctx, enn.TokenGateDesc(m=3, c=8, act=act, in_dtype=enn.F32, out_dtype=enn.F32))
        y = guarded(3, 8, torch.float32)
        execute(op, 3, [g, u], [y])
        op.release()
        want = torch.tensor(want, device="cuda", dtype=torch.float32)
        assert torch.allclose(y[0], want, rtol=1e-6, atol=1e-30) and torch.allclose(y[1], want, rtol=1e-6, atol=1e-30)
        assert torch.equal(torch.isnan(y[2]), torch.isnan(u[2]))
        op = enn.token_gate(ctx, enn.TokenGateDesc(m=3, c=8, act=act, in_dtype=enn.F32, out_dtype=enn.S8))
        q, s = guarded(3, 16, torch.int8), guarded(3, 1, torch.float32)
        execute(op, 3, [g, u], [q, s])
        op.release()
        assert bool(torch.isnan(s[2, 0])) and bool((q[2] == 0).all()) and int(q[0].max()) == 127


# ---- log_probs --------------------------------------------------------------------------------------------------------

def run_log_probs(enn, ctx, logits, ids, top, scale=1.0, pitch=0, rows=None):
    """Runs the operator on [m][vocab] logits (rows `pitch` apart) and returns given, entropy, top_ids, top of all rows."""
    m, v = logits.shape
    io = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}[logits.dtype]
    if pitch:
        store = torch.full((m, pitch), 1e4, dtype=logits.dtype, device="cuda")
        store[:, :v] = logits
    else:
        store = logits.contiguous()
    given = 0 if ids is None else ids.shape[1]
    op = enn.log_probs(ctx, enn.LogProbsDesc(m=m, vocab=v, in_dtype=code(enn, io), given=given, top=top, scale=scale, in_pitch=pitch))
    outs = ([guarded(m, given, torch.float32)] if given else []) + [guarded(m, 1, torch.float32)]
    outs += [guarded(m, top, torch.int32), guarded(m, top, torch.float32)] if top else []
    rows = m if rows is None else rows
    execute(op, rows, [store] + ([ids] if given else []), outs)
    op.release()
    for o in outs:
        assert untouched(o, rows)
    it = iter(outs)
    return (next(it)[:m] if given else None, next(it)[:m, 0], next(it)[:m] if top else None, next(it)[:m] if top else None)


def check_log_probs(logits, ids, top, got, scale=1.0):
    """With z = scale * l rounded once and d = z - max rounded once, e^d is off by its own roundings and those of its argument,
    sums by SERIAL roundings: log p by the sum of the two."""
    given, entropy, top_ids, top_lp = got
    z = logits.double() * float(np.float32(scale))
    lse = torch.logsumexp(z, -1, keepdim=True)
    lp = z - lse
    p = torch.exp(lp)
    reach = torch.where(torch.isinf(z), 0.0, z.abs()).amax(-1, keepdim=True)
    arg = 2 * U * (2 * reach)                   # of the argument of an exponential that counts
    tol = (SERIAL + 20) * U + 2 * arg + 4 * U * (reach + lse.abs())
    want = torch.where(p > 0, -p * lp, 0.0).sum(-1)
    mean_d = torch.where(p > 0, p * (z.amax(-1, keepdim=True) - z), 0.0).sum(-1, keepdim=True)
    assert bool(((entropy.double() - want).abs() <= ((tol + 2 * arg) * (1 + 2 * mean_d)).squeeze(-1)).all())
    if given is not None:
        w = torch.gather(lp, 1, ids.long())
        ok = (given.double() - w).abs() <= tol + 2 * U * torch.where(torch.isinf(w), 0.0, w.abs())
        assert bool((ok | (given.double() == w)).all())
    if top:
        order = torch.sort(logits.double(), dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(top_ids.long(), order)
        w = torch.gather(lp, 1, order)
        ok = (top_lp.double() - w).abs() <= tol + 2 * U * torch.where(torch.isinf(w), 0.0, w.abs())
        assert bool((ok | (top_lp.double() == w)).all())


@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,v,top", [(1, 1, 1), (2, 2, 2), (3, 31, 5), (1, 32, 32), (5, 255, 7), (2, 1000, 20), (4, 1024, 1), (7, 4099, 32), (2, 32000, 20), (3, 50001, 5),
                                      (2, 131072, 32), (1, 262143, 3), (33, 8192, 20)])
def test_log_probs(enn, ctx, m, v, top, io):
    logits = (rand(v, m, v) * 3).to(TYPES[io])
    ids = torch.randint(0, v, (m, 2), device="cuda", dtype=torch.int32)
    check_log_probs(logits, ids, top, run_log_probs(enn, ctx, logits, ids, top))
    check_log_probs(logits, ids, top, run_log_probs(enn, ctx, logits, ids, top, scale=0.7), scale=0.7)


@pytest.mark.parametrize("given,top", [(0, 0), (1, 0), (0, 1), (300, 2)])
def test_log_probs_forms(enn, ctx, given, top):
    logits = rand(4, 6, 2222) * 2
    ids = torch.randint(0, 2222, (6, given), device="cuda", dtype=torch.int32) if given else None
    check_log_probs(logits, ids, top, run_log_probs(enn, ctx, logits, ids, top))


@pytest.mark.parametrize("pitch", [1001, 1008, 1500])
@pytest.mark.parametrize("io", ["f16", "f32"])
def test_log_probs_pitch(enn, ctx, pitch, io):
    """What lies between the rows is not looked at."""
    logits = (rand(6, 9, 1001) * 3).to(TYPES[io])
    ids = torch.randint(0, 1001, (9, 1), device="cuda", dtype=torch.int32)
    check_log_probs(logits, ids, 20, run_log_probs(enn, ctx, logits, ids, 20, pitch=pitch))


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("v", [100, 5000, 70000])
def test_log_probs_ties_go_to_the_lower_index(enn, ctx, v, io):
    logits = torch.zeros(6, v, device="cuda", dtype=TYPES[io])
    logits[1] = (rand(1, v) * 2).round()                              # few distinct values
    logits[2, ::2] = -0.0                                             # equal to +0
    logits[3] = torch.arange(v, device="cuda").to(TYPES[io]) / 1000   # ascending: every later one is larger
    logits[4] = -torch.arange(v, device="cuda").to(TYPES[io]) / 1000
    logits[5, v // 2:] = 1
    ids = torch.randint(0, v, (6, 1), device="cuda", dtype=torch.int32)
    check_log_probs(logits, ids, 32, run_log_probs(enn, ctx, logits, ids, 32))


def test_log_probs_clusters_of_large_values(enn, ctx):
    """The alternatives all in one place: next to each other, and at distances that make one thread or block see them all."""
    v = 65536
    for step in (1, 2, 8, 64, 256, 512, 1024, 2048):
        logits = rand(step, 3, v)
        at = (torch.arange(32, device="cuda") * step + 7 * step) % v
        logits[0, at] = 20 + rand(3, 32)
        logits[1, at] = 20.0
        logits[2] = logits[2].half().float()
        ids = torch.randint(0, v, (3, 1), device="cuda", dtype=torch.int32)
        check_log_probs(logits, ids, 32, run_log_probs(enn, ctx, logits, ids, 32))


@pytest.mark.parametrize("m,v,io,top", [(600, 3000, "bf16", 20), (500, 1001, "f16", 5), (450, 8000, "bf16", 32), (700, 37, "f32", 32), (3000, 500, "f32", 1),
                                        (230, 49500, "f32", 20), (250, 100001, "bf16", 7), (500, 20000, "f16", 20)])
def test_log_probs_many_rows(enn, ctx, m, v, io, top):
    """Many rows of every length, among them rows of equal logits, rows with little left and rows with none."""
    logits = (rand(m + v, m, v) * 3).to(TYPES[io])
    logits[1] = 0
    logits[2, 3:] = -math.inf
    logits[3] = torch.finfo(TYPES[io]).min
    logits[3, 5] = 1
    logits[m - 1] = (rand(3, v) * 2).round().to(TYPES[io])
    ids = torch.randint(0, v, (m, 1), device="cuda", dtype=torch.int32)
    got = run_log_probs(enn, ctx, logits, ids, top)
    check_log_probs(logits, ids, top, got)


def test_log_probs_masked_vocabulary(enn, ctx):
    v = 3001
    logits = rand(8, 5, v) * 4
    logits[0, 1:] = -math.inf                 # one left: log p 0, entropy 0
    logits[1, ::2] = -math.inf
    logits[2, 5:] = -math.inf                 # fewer left than alternatives asked for
    logits[3] = torch.finfo(torch.float32).min      # the type's lowest value throughout: equal shares
    logits[4, 7:] = torch.finfo(torch.float32).min
    ids = torch.tensor([[0], [1], [4], [9], [3]], device="cuda", dtype=torch.int32)
    got = run_log_probs(enn, ctx, logits, ids, 10)
    assert got[0][0, 0] == 0 and got[1][0] == 0
    assert got[2][0].tolist() == list(range(10)) and bool((got[3][0, 1:] == -math.inf).all())
    assert got[2][2, 5:].tolist() == [5, 6, 7, 8, 9] and bool((got[3][2, 5:] == -math.inf).all())
    assert abs(float(got[0][3, 0]) + math.log(v)) < 1e-4 and abs(float(got[1][3]) - math.log(v)) < 1e-4
    keep = [0, 1, 2]
    check_log_probs(logits[keep], ids[keep], 10, tuple(x[keep] for x in got))
    few = logits[4:5, :7]
    alone = run_log_probs(enn, ctx, few.contiguous(), ids[4:5], 7)
    check_log_probs(few, ids[4:5], 7, alone)
    assert abs(float(got[1][4]) - float(alone[1][0])) < 1e-5 and abs(float(got[0][4, 0]) - float(alone[0][0, 0])) < 1e-5


def test_log_probs_rows_without_a_distribution(enn, ctx):
    """All ruled out, a NaN, +inf: NaN there and nowhere else; ids still ordered, NaN above all."""
    for v in (50, 9000):
        logits = rand(9, 4, v)
        logits[0] = -math.inf
        logits[1, 17], logits[1, 30] = math.nan, math.inf
        logits[2, 21] = math.inf
        ids = torch.tensor([[3], [3], [3], [3]], device="cuda", dtype=torch.int32)
        given, entropy, top_ids, top = run_log_probs(enn, ctx, logits, ids, 4)
        assert bool(torch.isnan(given[:3]).all()) and bool(torch.isnan(entropy[:3]).all()) and bool(torch.isnan(top[:3]).all())
        assert top_ids[0].tolist() == [0, 1, 2, 3] and top_ids[1, :2].tolist() == [17, 30] and int(top_ids[2, 0]) == 21
        check_log_probs(logits[3:], ids[3:], 4, (given[3:], entropy[3:], top_ids[3:], top[3:]))


def test_log_probs_ids_outside_the_vocabulary(enn, ctx):
    logits = rand(10, 2, 500)
    ids = torch.tensor([[-1, 500, 499], [-2 ** 31, 2 ** 31 - 1, 0]], device="cuda", dtype=torch.int32)
    given = run_log_probs(enn, ctx, logits, ids, 0)[0]
    assert bool((given[:, 0] == 0).all()) and bool(torch.isnan(given[:, 1]).all())
    check_log_probs(logits, ids[:, 2:], 0, (given[:, 2:], run_log_probs(enn, ctx, logits, None, 0)[1], None, None))


@pytest.mark.parametrize("rows", [0, 1, 6])
def test_log_probs_fewer_rows_than_prepared(enn, ctx, rows):
    logits = rand(11, 7, 640)
    ids = torch.randint(0, 640, (7, 1), device="cuda", dtype=torch.int32)
    got = run_log_probs(enn, ctx, logits, ids, 3, rows=rows)
    if rows:
        check_log_probs(logits[:rows], ids[:rows], 3, tuple(x[:rows] for x in got))


def test_log_probs_rows_past_32_bits(enn, ctx):
    """Rows that begin more than 2^31 elements into the logits."""
    v, pitch, m = 1000, 1 << 28, 10
    store = torch.empty((m - 1) * pitch + v, dtype=torch.bfloat16, device="cuda")
    logits = (rand(12, m, v) * 3).bfloat16()
    for t in range(m):
        store[t * pitch:t * pitch + v] = logits[t]
    op = enn.log_probs(ctx, enn.LogProbsDesc(m=m, vocab=v, in_dtype=enn.BF16, given=0, top=4, scale=1.0, in_pitch=pitch))
    outs = [guarded(m, 1, torch.float32), guarded(m, 4, torch.int32), guarded(m, 4, torch.float32)]
    execute(op, m, [store], outs)
    op.release()
    check_log_probs(logits, None, 4, (None, outs[0][:m, 0], outs[1][:m], outs[2][:m]))


# ---- together ---------------------------------------------------------------------------------------------------------

def block(enn, ctx, m, c, f, v, seed=1):
    """A feed-forward block and a head as a program prepares them: norm -> product -> gate -> product -> norm with the stream -> product ->
    log probabilities.  Returns the operators and their weights."""
    w1, s1 = torch.randint(-127, 128, (2 * f, c), device="cuda").to(torch.int8), torch.full((2 * f,), 0.4 / math.sqrt(c) / 64, device="cuda")
    w2, s2 = torch.randint(-127, 128, (c, f), device="cuda").to(torch.int8), torch.full((c,), 1 / math.sqrt(f) / 64, device="cuda")
    w3, s3 = torch.randint(-127, 128, (v, c), device="cuda").to(torch.int8), torch.full((v,), 1 / math.sqrt(c) / 64, device="cuda")
    g1, g2 = 1 + 0.1 * rand(seed, c), 1 + 0.1 * rand(seed + 1, c)
    torch.cuda.synchronize()
    ops = dict(
        norm1=enn.token_norm(ctx, enn.TokenNormDesc(m=m, c=c, norm=enn.NORM_RMS, io_dtype=enn.BF16, out_dtype=enn.S8, eps=1e-6, residual_scale=1.0), g1.data_ptr()),
        up=enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=c, n=2 * f, out_dtype=enn.BF16), w1.data_ptr(), s1.data_ptr()),
        gate=enn.token_gate(ctx, enn.TokenGateDesc(m=m, c=f, act=enn.GATE_SILU, packed=1, in_dtype=enn.BF16, out_dtype=enn.S8)),
        down=enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=f, n=c, out_dtype=enn.BF16), w2.data_ptr(), s2.data_ptr()),
        norm2=enn.token_norm(ctx, enn.TokenNormDesc(m=m, c=c, norm=enn.NORM_RMS, residual=1, io_dtype=enn.BF16, out_dtype=enn.S8, eps=1e-6, residual_scale=1.0), g2.data_ptr()),
        head=enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=c, n=v, out_dtype=enn.F32), w3.data_ptr(), s3.data_ptr()),
        probs=enn.log_probs(ctx, enn.LogProbsDesc(m=m, vocab=v, in_dtype=enn.F32, given=1, top=5, scale=1.0)))
    return ops, (w1, s1, w2, s2, w3, s3, g1, g2)


def block_buffers(enn, m, c, f, v):
    new = lambda *shape, dtype=torch.bfloat16: torch.empty(*shape, dtype=dtype, device="cuda")      # noqa: E731
    return dict(q1=new(m, enn.token_pitch(c), dtype=torch.int8), t1=new(m, dtype=torch.float32), up=new(m, 2 * f), q2=new(m, enn.token_pitch(f), dtype=torch.int8),
                t2=new(m, dtype=torch.float32), down=new(m, c), h=new(m, c), q3=new(m, enn.token_pitch(c), dtype=torch.int8), t3=new(m, dtype=torch.float32),
                logits=new(m, v, dtype=torch.float32), given=new(m, 1, dtype=torch.float32), entropy=new(m, dtype=torch.float32),
                top_ids=new(m, 5, dtype=torch.int32), top=new(m, 5, dtype=torch.float32))


BLOCK_CALLS = [("norm1", ["x"], ["q1", "t1"]), ("up", ["q1", "t1"], ["up"]), ("gate", ["up"], ["q2", "t2"]), ("down", ["q2", "t2"], ["down"]),
               ("norm2", ["down", "x"], ["h", "q3", "t3"]), ("head", ["q3", "t3"], ["logits"]), ("probs", ["logits", "ids"], ["given", "entropy", "top_ids", "top"])]


def run_block(ops, bufs, rows):
    for name, ins, outs in BLOCK_CALLS:
        ops[name].execute_rows(rows, [bufs[i].data_ptr() for i in ins], [bufs[o].data_ptr() for o in outs])


def check_block(bufs, weights, rows, c, f):
    """Every operator of the run against 64 bits on the inputs it saw."""
    w1, s1, w2, s2, w3, s3, g1, g2 = weights
    b = {k: t[:rows] for k, t in bufs.items()}
    eps = float(np.float32(1e-6))
    check_bytes(b["q1"], b["t1"], *norm_error(c, b["x"].double(), torch.zeros(rows, c, device="cuda").double(), "rms", eps, g1, None), c)
    fc_check(b["up"], b["q1"], w1, b["t1"], s1, None, "bf16", c)
    a, err = act64(b["up"][:, :f].double(), "silu")
    u = b["up"][:, f:].double()
    check_bytes(b["q2"], b["t2"], a * u, err * u.abs() + U * (a * u).abs(), f)
    fc_check(b["down"], b["q2"], w2, b["t2"], s2, None, "bf16", f)
    stream, (y, err) = norm_reference(norm_case(rows, c), b["down"], b["x"], None, (g2, None, None, None), 1.0, eps)
    check_close(b["h"], *stream, "bf16")
    check_bytes(b["q3"], b["t3"], y, err, c)
    fc_check(b["logits"], b["q3"], w3, b["t3"], s3, None, "f32", c)
    check_log_probs(b["logits"], b["ids"], 5, (b["given"], b["entropy"], b["top_ids"], b["top"]))


@pytest.mark.parametrize("m,rows", [(1, 1), (40, 40), (40, 7), (300, 300)])
def test_a_block_as_a_program_runs_it(enn, ctx, m, rows):
    c, f, v = 520, 1360, 5003
    ops, weights = block(enn, ctx, m, c, f, v)
    bufs = block_buffers(enn, m, c, f, v)
    bufs["x"] = (rand(3, m, c) * 2).bfloat16()
    bufs["ids"] = torch.randint(0, v, (m, 1), device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    run_block(ops, bufs, rows)
    ctx.sync()
    check_block(bufs, weights, rows, c, f)
    for op in ops.values():
        op.release()


def test_a_block_in_an_operator_list(enn, ctx):
    """The same operators as a list: one graph, tensors placed by the list; equal to the calls one by one, call after call."""
    m, c, f, v = 24, 256, 704, 2000
    ops, weights = block(enn, ctx, m, c, f, v)
    bufs = block_buffers(enn, m, c, f, v)
    bufs["x"] = (rand(5, m, c) * 2).bfloat16()
    bufs["ids"] = torch.randint(0, v, (m, 1), device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    run_block(ops, bufs, m)
    ctx.sync()
    check_block(bufs, weights, m, c, f)
    ol = enn.OpList(ctx)
    size = {k: t.numel() * t.element_size() for k, t in bufs.items()}
    tid = {k: ol.tensor(n) for k, n in size.items()}
    for name, ins, outs in BLOCK_CALLS:
        ol.add_n(ops[name], [tid[i] for i in ins], [tid[o] for o in outs])
    results = ["h", "given", "entropy", "top_ids", "top"]
    ol.set_io([tid["x"], tid["ids"]], [tid[r] for r in results], [size[r] for r in results])
    ol.finalize()
    assert [k for _, k, _ in ol.nodes()] == [12, 11, 13, 11, 12, 11, 14]
    assert ol.stats()["device_bytes"] < sum(size.values()) * 2
    assert len(ol.profile(2)) == 7
    x_host, ids_host = bufs["x"].cpu(), bufs["ids"].cpu()
    for _ in range(3):
        got = [torch.zeros(bufs[r].shape, dtype=bufs[r].dtype) for r in results]
        ol.execute_host_ptrs([x_host.data_ptr(), ids_host.data_ptr()], [t.data_ptr() for t in got])
        for r, t in zip(results, got):
            assert torch.equal(t, bufs[r].cpu()), r
    for _ in range(3):
        got = [torch.zeros(bufs[r].shape, dtype=bufs[r].dtype).pin_memory() for r in results]
        ol.submit_host_ptrs([x_host.data_ptr(), ids_host.data_ptr()], [t.data_ptr() for t in got])
        ol.wait()
        for r, t in zip(results, got):
            assert torch.equal(t, bufs[r].cpu()), r
    ol.destroy()


def test_a_block_captured_and_replayed(enn):
    """Captured on the context's stream by the caller, replayed on new inputs, with plain calls of the same operators in between."""
    ctx = enn.Context(0)
    m, c, f, v = 5, 384, 1024, 1500
    ops, weights = block(enn, ctx, m, c, f, v)
    bufs = block_buffers(enn, m, c, f, v)
    bufs["x"] = (rand(5, m, c) * 2).bfloat16()
    bufs["ids"] = torch.randint(0, v, (m, 1), device="cuda", dtype=torch.int32)
    stream = torch.cuda.ExternalStream(ctx.stream)
    torch.cuda.synchronize()
    run_block(ops, bufs, m)
    ctx.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run_block(ops, bufs, m)
    for seed in (6, 7):
        bufs["x"].copy_((rand(seed, m, c) * 2).bfloat16())
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.sync()
        check_block(bufs, weights, m, c, f)
        first = {k: t.clone() for k, t in bufs.items()}
        torch.cuda.synchronize()
        run_block(ops, bufs, m)
        ctx.sync()
        assert all(torch.equal(first[k], bufs[k]) for k in bufs)
    del graph
    for op in ops.values():
        op.release()
    ctx.close()


def test_two_graphs_of_the_same_operators_at_once(enn):
    """Graphs of the same handles on other tensors, replayed on two streams at the same time: the operators share no memory."""
    ctx = enn.Context(0)
    m, c, f, v = 33, 512, 1400, 6000
    ops, weights = block(enn, ctx, m, c, f, v)
    stream = torch.cuda.ExternalStream(ctx.stream)
    graphs, sets = [], []
    for i in range(2):
        bufs = block_buffers(enn, m, c, f, v)
        bufs["x"] = (rand(40 + i, m, c) * 2).bfloat16()
        bufs["ids"] = torch.randint(0, v, (m, 1), device="cuda", dtype=torch.int32)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run_block(ops, bufs, m)
        graphs.append(graph)
        sets.append(bufs)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for bufs in sets:
        check_block(bufs, weights, m, c, f)
    del graph, graphs
    for op in ops.values():
        op.release()
    ctx.close()


def test_calls_of_two_contexts_at_once(enn):
    """The same shapes on two contexts' streams at the same time, many calls in flight: nothing is shared."""
    m, c, f, v = 17, 640, 1200, 4001
    lanes = []
    for i in range(2):
        ctx = enn.Context(0)
        ops, weights = block(enn, ctx, m, c, f, v, seed=20 + i)
        bufs = block_buffers(enn, m, c, f, v)
        bufs["x"] = (rand(30 + i, m, c) * 2).bfloat16()
        bufs["ids"] = torch.randint(0, v, (m, 1), device="cuda", dtype=torch.int32)
        lanes.append((ctx, ops, weights, bufs))
    torch.cuda.synchronize()
    for _ in range(50):
        for _, ops, _, bufs in lanes:
            run_block(ops, bufs, m)
    for ctx, ops, weights, bufs in lanes:
        ctx.sync()
        check_block(bufs, weights, m, c, f)
        for op in ops.values():
            op.release()
        ctx.close()


def test_results_do_not_change_from_call_to_call(enn, ctx):
    m, c, f, v = 9, 1000, 2000, 30000
    ops, _ = block(enn, ctx, m, c, f, v)
    bufs = block_buffers(enn, m, c, f, v)
    bufs["x"] = rand(8, m, c).bfloat16()
    bufs["ids"] = torch.randint(0, v, (m, 1), device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    run_block(ops, bufs, m)
    ctx.sync()
    first = {k: t.clone() for k, t in bufs.items()}
    for _ in range(20):
        run_block(ops, bufs, m)
    ctx.sync()
    assert all(torch.equal(first[k], bufs[k]) for k in bufs)
    for op in ops.values():
        op.release()


# ---- refusals ---------------------------------------------------------------------------------------------------------

def refused(enn, f, *args):
    with pytest.raises(enn.EnnError) as e:
        f(*args)
    assert e.value.status == enn.INVALID_PARAMS and str(e.value)


def test_token_operators_refuse_bad_calls(enn, ctx):
    one = np.ones(64, np.float32)
    refused(enn, enn.token_fc, ctx, enn.TokenFcDesc(m=1, k=131072, n=1, out_dtype=enn.F32), np.zeros(131072, np.int8), one[:1])
    refused(enn, enn.token_norm, ctx, enn.TokenNormDesc(m=1, c=64, norm=enn.NORM_NONE, io_dtype=enn.F32, out_dtype=enn.F32, residual_scale=1.0), one)
    refused(enn, enn.token_gate, ctx, enn.TokenGateDesc(m=1, c=64, act=9, in_dtype=enn.F32, out_dtype=enn.F32))
    refused(enn, enn.log_probs, ctx, enn.LogProbsDesc(m=1, vocab=8, in_dtype=enn.F32, top=9, scale=1.0))
    op = enn.token_fc(ctx, enn.TokenFcDesc(m=2, k=32, n=16, out_dtype=enn.F32), np.zeros((16, 32), np.int8), one[:16])
    q, s, y = torch.zeros(2, 32, dtype=torch.int8, device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(2, 16, device="cuda")
    a = [q.data_ptr(), s.data_ptr()]
    refused(enn, op.execute_rows, 3, a, [y.data_ptr()])
    refused(enn, op.execute_rows, -1, a, [y.data_ptr()])
    refused(enn, op.execute_rows, 1, a[:1], [y.data_ptr()])
    refused(enn, op.execute_rows, 1, a, [])
    refused(enn, op.execute_rows, 1, [a[0], None], [y.data_ptr()])
    refused(enn, op.execute_rows, 1, [a[0], a[1] + 2], [y.data_ptr()])
    refused(enn, op.execute_rows, 1, a, [a[1]])
    refused(enn, op.execute, q.data_ptr(), y.data_ptr())              # the one-tensor form
    op.execute_rows(0, [None, None], [None])                          # nothing to do
    ol = enn.OpList(ctx)
    t = [ol.tensor(n) for n in (64, 8, 128, 16)]
    refused(enn, ol.add_n, op, [t[0], t[1]], [t[3]])                  # too small
    refused(enn, ol.add_n, op, [t[0]], [t[2]])
    refused(enn, ol.add_n, op, [t[0], t[1]], [t[1]])
    refused(enn, ol.add, op, [t[0], t[1]], 99)
    ol.add(op, [t[0], t[1]], t[2])
    ol.destroy()
    mean = enn.mean(ctx, enn.mean_desc((1, 2, 2, 8), (1, 2)))
    refused(enn, mean.execute_rows, 1, a, [y.data_ptr()])
    mean.release()


def test_byte_operators_refuse_float_types(enn, ctx):
    refused(enn, enn.add, ctx, enn.AddDesc(count=4, act_dtype=enn.BF16, in0_scale=1.0, in1_scale=1.0, out_scale=1.0))
    refused(enn, enn.mean, ctx, enn.mean_desc((1, 2, 2, 8), (1, 2), enn.F16))
    refused(enn, enn.softmax, ctx, enn.SoftmaxDesc(outer=1, channels=4, inner=1, beta=1.0, act_dtype=enn.F32, in_scale=1.0, out_scale=1.0))


def test_null_context_and_handles(enn):
    h = C.c_void_p()
    assert enn.lib.enn_b200_log_probs_prepare(None, C.byref(enn.LogProbsDesc(m=1, vocab=8, in_dtype=enn.F32, scale=1.0)), C.byref(h)) == enn.INVALID_PARAMS
