"""Token operators: calls that earlier tests do not make.  Tolerances count roundings, u = 2^-24."""
import math

import pytest
import torch

from test_token_ops_gpu import TYPES, U, execute, refused, run_log_probs

pytestmark = pytest.mark.gpu


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
