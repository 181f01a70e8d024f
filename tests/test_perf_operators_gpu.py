"""The performance cases of the token operators as a program runs them."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def cases():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), os.pardir, "perf", "operators.py")
    spec = importlib.util.spec_from_file_location("perf_operators_under_test", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.own = True
    stream = torch.cuda.current_stream()
    yield mod
    torch.cuda.synchronize()
    torch.cuda.set_stream(stream)
    mod._library()[1].close()


def test_results_are_read_without_a_wait(cases):
    """What torch reads right after a call is what the call computes, not what lay there before."""
    for case in (cases._fc(None, 16, 8192, 16384, "bf16", False), cases._norm(None, 2048, 4097, "bf16", "rms", "none", True, 256, n=6144),
                 cases._gate(None, 8192, 12288, "bf16", "silu", True), cases._log_probs(None, 2048, 65536, "f32", 1, 1, False)):
        state = cases.prepare(case, 3)
        tensors = lambda r: [r] if isinstance(r, torch.Tensor) else [r[k] for k in sorted(r)]      # noqa: E731
        want = [t.clone() for t in tensors(cases.run(state))]
        torch.cuda.synchronize()
        for _ in range(3):
            for t in tensors(state.out):
                t.zero_()
            got = [t.clone() for t in tensors(cases.run(state))]
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        del state
