"""Arguments of masked steps that do not fit their types, from host and device tensors."""
import pytest
import torch

from tests import masked_harness as H

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("host", [False, True])
def test_windows_and_sinks_that_are_no_32_bit_numbers_are_refused(host):
    step = H.Step([30], [4], window=8, seed=1)
    op = step.operator()
    good = step.inputs(step.packed["key"].clone(), step.packed["value"].clone())
    out = torch.zeros((4, step.hq * step.d), dtype=torch.float16, device=step.dev)
    if host:
        good, out = {k: v.cpu() if isinstance(v, torch.Tensor) and "cache" not in k else v for k, v in good.items()}, out.cpu()
    for name in ("sliding_window", "sink_tokens"):
        for value in (1 << 31, 1 << 32, (1 << 32) + 8, -1, -(1 << 32), 7.5, "8"):
            with pytest.raises(H.pkg.GenaiB200Error, match=name):
                op.evaluate({**good, name: value}, {"output": out})
    torch.cuda.synchronize()
    assert bool((out == 0).all())
    op.evaluate(good, {"output": out})
    torch.cuda.synchronize()
    step.check(out.to(step.dev))
