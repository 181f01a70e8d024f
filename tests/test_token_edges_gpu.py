"""Token operators: calls that earlier tests do not make.  Tolerances count roundings, u = 2^-24."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import cases
from test_token_ops_gpu import (TYPES, U, check_bytes, check_close, check_log_probs, code, execute, fc_check, fc_inputs, guarded, norm_case, norm_reference,
                                rand, refused, run_log_probs)

pytestmark = pytest.mark.gpu


def kept(buf, rows, offset=0):
    """Everything in a guarded() buffer outside its first `rows` rows is the pattern, what lies before them too."""
    flat = torch.empty(0, dtype=buf.dtype, device="cuda").set_(buf.untyped_storage())
    want = (torch.arange(flat.numel(), device="cuda") % 97).to(buf.dtype)
    end = offset + rows * buf.shape[1]
    return torch.equal(flat[:offset], want[:offset]) and torch.equal(flat[end:], want[end:])


# ---- addresses --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m", [1, 20, 150, 700])
@pytest.mark.parametrize("q_offset,pitch,out_offset", [(0, 101, 0), (1, 112, 0), (0, 208, 1), (3, 150, 3), (16, 112, 8), (0, 112, 4)])
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_token_fc_writes_its_rows_alone(enn, ctx, m, q_offset, pitch, out_offset, out):
    k, n = 100, 9001 if m == 700 else 72
    q, w, s, sw, _ = fc_inputs(9, m, k, n, pitch)
    flat = torch.zeros(q.numel() + 64, dtype=torch.int8, device="cuda")
    moved = flat[q_offset:q_offset + q.numel()].view(q.shape)
    moved.copy_(q)
    torch.cuda.synchronize()
    op = enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=k, n=n, out_dtype=code(enn, out), in_pitch=pitch), w.data_ptr(), sw.data_ptr())
    for rows in (m, max(1, m - 3)):
        y = guarded(m, n, TYPES[out], out_offset)
        execute(op, rows, [moved, s], [y])
        fc_check(y[:rows], q[:rows], w, s[:rows], sw, None, out, k)
        assert kept(y, rows, out_offset)
    op.release()


@pytest.mark.parametrize("out_off,y_off", [(0, 0), (1, 3), (4, 1), (7, 5)])
@pytest.mark.parametrize("m,c,io,out", [(400, 515, "bf16", "bf16"), (30, 1024, "f16", "s8"), (310, 4097, "bf16", "s8"), (5, 1001, "f32", "f16"), (700, 67, "f16", "f32"),
                                        (3, 32767, "bf16", "s8"), (1, 7, "bf16", "bf16")])
def test_token_norm_writes_its_rows_alone(enn, ctx, m, c, io, out, out_off, y_off):
    """What lies before the first row and behind the last, in both results and in the scales, stays as it was."""
    x, r = rand(1, m, c).to(TYPES[io]), rand(2, m, c).to(TYPES[io])
    op = enn.token_norm(ctx, enn.TokenNormDesc(m=m, c=c, norm=enn.NORM_RMS, residual=1, io_dtype=code(enn, io), out_dtype=code(enn, out), eps=1e-6, residual_scale=0.5))
    for rows in {m, max(1, m - 2)}:
        h, y, s = guarded(m, c, TYPES[io], out_off), guarded(m, enn.token_pitch(c) if out == "s8" else c, TYPES.get(out, torch.int8), y_off), guarded(m, 1, torch.float32, 1)
        execute(op, rows, [x, r], [h, y] + ([s] if out == "s8" else []))
        stream, (want, err) = norm_reference(norm_case(m, c, io, out), x[:rows], r[:rows], None, (None,) * 4, 0.5, float(np.float32(1e-6)))
        check_close(h[:rows], *stream, io)
        if out == "s8":
            check_bytes(y[:rows], s[:rows, 0], want, err, c)
        else:
            check_close(y[:rows], want, err, out)
        assert kept(h, rows, out_off) and kept(y, rows, y_off) and kept(s, rows if out == "s8" else 0, 1)
    op.release()


@pytest.mark.parametrize("io,out", [("bf16", "bf16"), ("f16", "s8"), ("f32", "s8"), ("bf16", "f32")])
@pytest.mark.parametrize("m,c", [(3000, 67), (2000, 1001), (1500, 4097), (400, 12301), (900, 264), (5000, 9), (2, 32765)])
@pytest.mark.parametrize("x_off,r_off", [(0, 0), (3, 0), (0, 5), (1, 1)])
def test_token_norm_stream_in_place_between_lines(enn, ctx, m, c, io, out, x_off, r_off):
    """Rows that share lines with their neighbours, written over the stream they were read from: the bits of a run into memory of its own."""
    def place(t, off):
        flat = torch.zeros(t.numel() + 16, dtype=t.dtype, device="cuda")
        return flat[off:off + t.numel()].view(t.shape).copy_(t)
    e = TYPES[io]
    x, r, gate = place(rand(1, m, c).to(e), x_off), place(rand(2, m, c).to(e), r_off), rand(3, -(-m // 50), c).to(e)
    weight = 1 + 0.3 * rand(4, c)
    torch.cuda.synchronize()
    op = enn.token_norm(ctx, enn.TokenNormDesc(m=m, c=c, norm=enn.NORM_RMS, post_norm=enn.NORM_LAYER, residual=1, gate_tokens=50, io_dtype=code(enn, io), out_dtype=code(enn, out),
                                               eps=1e-6, post_eps=1e-6, residual_scale=0.7), weight.data_ptr())
    results = []
    for in_place in (False, True, True):
        stream = place(r, r_off)
        h = stream if in_place else torch.zeros_like(r)
        y = torch.zeros(m, enn.token_pitch(c) if out == "s8" else c, dtype=TYPES.get(out, torch.int8), device="cuda")
        s = torch.zeros(m, device="cuda")
        execute(op, m, [x, stream, gate], [h, y] + ([s] if out == "s8" else []))
        results.append((h.clone(), y, s))
    for again in results[1:]:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(results[0], again))
    op.release()


# ---- log_probs --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m,v,io,early,late", [(200, 8000, "f32", 0, 4096), (500, 8000, "f16", 0, 4096), (230, 20000, "bf16", 3, 16387), (230, 50000, "f32", 1, 32769),
                                               (1, 131072, "f32", 0, 8192), (200, 8000, "f32", 4096, 0)])
def test_log_probs_of_rows_that_are_all_but_certain(enn, ctx, m, v, io, early, late):
    """Two logits l <= l' = l + d in chunks that the same thread sees one after the other, the others far below.  log p' = -log1p(e^-d) and the
    entropy log1p(e^-d) + d / (1 + e^d) are small: they must not be what is left of two numbers of the size of d.
    With a sum of exponentials that counts l' as exactly 1 and l as r = e^-d, off by (4 d + 6) u r <= 6 u from its argument and its own roundings, and two
    roundings of the sum (4 u), log p' is off by 10 u and the logarithm: 12 u.  The sum of d e^-d is off by (4 d + 6) u d e^-d <= 6 u, its quotient by half of the
    sum's error (5 u), and the logarithm by 12 u: 24 u."""
    gaps = torch.linspace(0, 16, m, dtype=torch.float64).to(TYPES[io]) if m > 1 else torch.tensor([2.5], dtype=TYPES[io])
    logits = torch.full((m, v), -math.inf, dtype=TYPES[io], device="cuda")
    logits[:, 7::1000] = -60.0
    logits[:, early] = 0
    logits[:, late] = gaps.cuda()
    ids = torch.tensor([[early, late]] * m, dtype=torch.int32, device="cuda")
    given, entropy, top_ids, top = run_log_probs(enn, ctx, logits, ids, 2)
    d = gaps.cuda().double()
    want = -torch.log1p(torch.exp(-d))
    want_entropy = -want + d / (1 + torch.exp(d))
    assert bool((top <= 0).all()) and bool((given <= 0).all()) and bool((entropy >= 0).all())
    assert torch.equal(top[:, 0], given[:, 1])
    assert bool(((top[:, 0].double() - want).abs() <= 12 * U).all()), float((top[:, 0].double() - want).abs().max() / U)
    assert bool(((given[:, 0].double() - (want - d)).abs() <= (12 + 2 * d) * U).all())
    assert bool(((entropy.double() - want_entropy).abs() <= 24 * U).all()), float((entropy.double() - want_entropy).abs().max() / U)
    assert torch.equal(top_ids[d > 0][:, 0], torch.full_like(top_ids[d > 0][:, 0], late))


@pytest.mark.parametrize("m,v,io,top", [(600, 3000, "bf16", 20), (500, 1001, "f16", 5), (700, 37, "f32", 32), (3000, 500, "f32", 1), (230, 49500, "f32", 20), (500, 20000, "f16", 0)])
def test_log_probs_of_rows_without_a_distribution_among_others(enn, ctx, m, v, io, top):
    """A CTA that takes several rows meets rows of -inf, NaN and +inf between ordinary ones, and rows with little left: each keeps to itself."""
    logits = (rand(m + v, m, v) * 3).to(TYPES[io])
    bad = torch.zeros(m, dtype=torch.bool, device="cuda")
    logits[0::7] = -math.inf
    logits[2::7, v // 2] = math.nan
    logits[4::7, v - 1] = math.inf
    bad[0::7], bad[2::7], bad[4::7] = True, True, True
    logits[1::7, v // 3:] = -math.inf
    logits[3::7, :] = logits[3::7, :].clamp(max=-1)
    logits[3::7, v - 1] = 5
    ids = torch.randint(0, v, (m, 1), device="cuda", dtype=torch.int32)
    given, entropy, top_ids, top_lp = run_log_probs(enn, ctx, logits, ids, top)
    assert bool(torch.isnan(given[bad]).all()) and bool(torch.isnan(entropy[bad]).all()) and (not top or bool(torch.isnan(top_lp[bad]).all()))
    if top:
        assert torch.equal(top_ids[0].long(), torch.arange(top, device="cuda")) and bool((top_ids[2::7, 0] == v // 2).all()) and bool((top_ids[4::7, 0] == v - 1).all())
    ok = ~bad
    check_log_probs(logits[ok], ids[ok], top, (given[ok], entropy[ok], top_ids[ok] if top else None, top_lp[ok] if top else None))


@pytest.mark.parametrize("scale", [2.0 ** 127, 2.0 ** 64, 2.0 ** -126, 1e-45])
def test_log_probs_with_scales_at_the_limits(enn, ctx, scale):
    """A temperature of nearly nothing leaves the largest logits alone, one beyond all logits leaves equal shares: exact but for
    the logarithm: an ulp and a rounding of ln 3 (3 u), of ln 8192 (16 u and 8 u)."""
    v = 8192
    logits = torch.arange(v, dtype=torch.float32, device="cuda").flip(0).repeat(3, 1)
    logits[1, 100:103] = 1e6
    logits[2, 50:] = torch.finfo(torch.float32).min
    ids = torch.tensor([[0, 1], [101, 0], [0, 60]], dtype=torch.int32, device="cuda")
    given, entropy, top_ids, top = run_log_probs(enn, ctx, logits, ids, 2, scale=scale)
    assert top_ids.tolist() == [[0, 1], [100, 101], [0, 1]]
    if scale > 1:
        ln = torch.tensor([0.0, math.log(3), 0.0], device="cuda")
        assert bool(((entropy - ln).abs() <= 3 * U).all()) and bool(((given[:, 0] + ln).abs() <= 3 * U).all())
        far = given[:, 1] if scale > 2.0 ** 100 else given[2:, 1]
        assert bool((far < -1e18).all()) and not bool(torch.isnan(given).any()) and not bool(torch.isnan(top).any())
    else:      # z differs by 2^-126 * 1e6 at most, but for the lowest value: z = -4 there with the scale 2^-126
        shares = torch.tensor([v, v], dtype=torch.float64, device="cuda")
        assert bool(((entropy[:2].double() - torch.log(shares)).abs() <= 24 * U).all()) and bool(((given[:2].double() + torch.log(shares)[:, None]).abs() <= 24 * U).all())


# ---- calls ------------------------------------------------------------------------------------------------------------

def test_outputs_that_share_memory_are_refused(enn, ctx):
    """A stream that is shifted against itself, results inside an input or another result; next to each other they pass."""
    m, c = 16, 40
    flat = torch.zeros(8, m * c + 64, dtype=torch.bfloat16, device="cuda")
    x, r, h, y = (flat[i].data_ptr() for i in range(4))
    size = m * c * 2
    op = enn.token_norm(ctx, enn.TokenNormDesc(m=m, c=c, norm=enn.NORM_RMS, residual=1, io_dtype=enn.BF16, out_dtype=enn.BF16, eps=1e-6, residual_scale=1.0))
    torch.cuda.synchronize()
    for outs in ([r + 2, y], [r + size - 2, y], [r - 2, y], [x + 16, y], [h, r + 80], [h, h + 16], [r, r + 16]):
        refused(enn, op.execute_rows, m, [x, r], outs)
    op.execute_rows(m, [x, r], [r, y])
    op.execute_rows(m // 2, [x, r], [r, r + size // 2])
    ctx.sync()
    op.release()


# ---- kernels that give up on a wait -----------------------------------------------------------------------------------

def gave_up(enn, f, *args):
    with pytest.raises(enn.EnnError) as e:
        f(*args)
    assert e.value.status == enn.CUDA_FAILURE and "gave up" in str(e.value)


@pytest.mark.parametrize("m,k,n", [(3, 1024, 512), (2000, 512, 4096)])
def test_a_replayed_product_that_gives_up_is_known_to_a_call_of_no_rows(enn, m, k, n):
    ctx = enn.Context(0)
    q, w, s, sw, _ = fc_inputs(21, m, k, n)
    torch.cuda.synchronize()
    op = enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=k, n=n, out_dtype=enn.F32), w.data_ptr(), sw.data_ptr())
    y = guarded(m, n, torch.float32)
    stream = torch.cuda.ExternalStream(ctx.stream)
    graphs = []
    for starve in (True, False):
        if starve:
            op.test_starve_next()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            op.execute_rows(m, [q.data_ptr(), s.data_ptr()], [y.data_ptr()])
        graphs.append(graph)
    op.execute_rows(0, [None, None], [None])
    for graph, works in zip(graphs, (False, True)):
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.sync()
        if works:
            op.execute_rows(0, [None, None], [None])
        else:
            gave_up(enn, op.execute_rows, 0, [None, None], [None])
            gave_up(enn, op.execute_rows, m, [q.data_ptr(), s.data_ptr()], [y.data_ptr()])
            op.clear_error()
    fc_check(y[:m], q, w, s, sw, None, "f32", k)
    del graph, graphs
    op.release()
    ctx.close()


@pytest.mark.parametrize("kind", ["token_fc", "conv"])
def test_lists_report_kernels_that_gave_up(enn, ctx, kind):
    """The word that a kernel left is seen by every way of running the list, and nothing else of it changes."""
    ol = enn.OpList(ctx)
    if kind == "token_fc":
        m, k, n = 16, 512, 256
        rng = np.random.default_rng(5)
        host = [rng.integers(-100, 100, (m, k), dtype=np.int8), np.linspace(0.01, 0.02, m, dtype=np.float32)]
        op = enn.token_fc(ctx, enn.TokenFcDesc(m=m, k=k, n=n, out_dtype=enn.F32), rng.integers(-100, 100, (n, k), dtype=np.int8), np.full(n, 0.01, np.float32))
    else:
        d, x, w, b, sc = cases.conv_case(seed=5, n=2, h=16, w=16, cin=64, cout=64, k=1, per_channel=True, out_scale=0.3)
        op = enn.conv2d(ctx, d, w, b, sc)
        host = [np.ascontiguousarray(x)]
    assert op.info.impl == enn.IMPL_TCGEN05
    size = op.info.out_bytes
    ids = [ol.tensor(a.nbytes) for a in host]
    out = ol.tensor(size)
    handle = C.c_void_p(op.h.value)
    if kind == "token_fc":
        ol.add_n(op, ids, [out])
    else:
        ol.add(op, ids, out)
    ol.set_io(ids, [out], [size])
    ol.finalize()
    ins = [a.ctypes.data for a in host]

    def run(how):
        got = np.zeros(size, np.uint8)
        if how == "execute":
            ol.execute_host_ptrs(ins, [got.ctypes.data])
        else:
            ol.submit_host_ptrs(ins, [got.ctypes.data])
            ol.wait()
        return got

    want = run("execute")
    assert want.any() and np.array_equal(want, run("submit"))
    devs = [ctx.to_device(a) for a in host] + [ctx.malloc(size)]
    ctx.check(enn.lib.enn_b200_op_test_starve_next(handle))
    if kind == "token_fc":
        addresses = (C.c_void_p * 2)(devs[0].value, devs[1].value)
        ctx.check(enn.lib.enn_b200_op_execute_rows(handle, 16, addresses, 2, (C.c_void_p * 1)(devs[2].value), 1))
    else:
        ctx.check(enn.lib.enn_b200_op_execute(handle, devs[0], devs[1]))
    ctx.sync()
    gave_up(enn, run, "execute")
    gave_up(enn, run, "submit")
    gave_up(enn, ol.wait)
    gave_up(enn, ol.profile, 1)
    gave_up(enn, ol.execute_device)
    ctx.check(enn.lib.enn_b200_op_clear_error(handle))
    for how in ("execute", "submit", "submit", "execute"):
        assert np.array_equal(want, run(how))
    ol.destroy()
    for d in devs:
        ctx.free(d)


# ---- byte operators and float types -----------------------------------------------------------------------------------

def byte_operators(enn):
    """Each operator that takes a type for its bytes: how it is prepared, a descriptor, and its inputs."""
    rng = np.random.default_rng(9)
    x = rng.integers(0, 256, (1, 6, 6, 8), dtype=np.uint8)
    pool = dict(n=1, h=6, w=6, c=8, kh=2, kw=2, stride_h=2, stride_w=2, out_h=3, out_w=3, out_scale=0.1, out_zp=3)
    q = dict(in_scale=0.1, in_zp=3, out_scale=1 / 256)
    concat = enn.ConcatDesc(n_inputs=2, outer=36, out_scale=0.2, out_zp=4)
    for i in range(2):
        concat.inner[i], concat.in_scale[i], concat.in_zp[i] = 8, 0.1 + 0.1 * i, 3
    return [(enn.add, enn.AddDesc(count=288, in0_scale=0.1, in0_zp=3, in1_scale=0.2, in1_zp=5, out_scale=0.3, out_zp=7), [x, x[:, ::-1]], 288),
            (enn.avgpool, enn.PoolDesc(**pool), [x], 72), (enn.maxpool, enn.PoolDesc(**pool), [x], 72), (enn.mean, enn.mean_desc((1, 6, 6, 8), (1, 2)), [x], 8),
            (enn.concat, concat, [x, x[:, ::-1]], 576), (enn.softmax, enn.SoftmaxDesc(outer=36, channels=8, inner=1, beta=1.0, **q), [x], 288),
            (enn.resize_bilinear, enn.ResizeDesc(n=1, h=6, w=6, c=8, out_h=9, out_w=5), [x], 360)]


@pytest.mark.parametrize("which", range(7))
def test_byte_operators_refuse_the_float_types_and_no_other_value(enn, ctx, which):
    prepare, desc, ins, size = byte_operators(enn)[which]
    devs = [ctx.to_device(a) for a in ins]
    out = ctx.malloc(size)

    def run():
        op = prepare(ctx, desc)
        op.execute_n(devs, out)
        got = ctx.download(out, (size,))
        op.release()
        return got

    desc.act_dtype = enn.U8
    want = run()
    for other in (2, 15, 19, 64, 1 << 20, -1, -16):
        desc.act_dtype = other
        assert np.array_equal(run(), want), other
    for floating in (enn.F32, enn.F16, enn.BF16):
        desc.act_dtype = floating
        refused(enn, prepare, ctx, desc)
    for d in devs + [out]:
        ctx.free(d)
