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


def test_parents_on_the_host_that_are_not_contiguous_are_refused():
    step = H.Step([30], [4], trees=[[-1, 0, 0, 1]], seed=2)
    op = step.operator()
    dev = step.inputs(step.packed["key"].clone(), step.packed["value"].clone())
    host = {k: v.cpu() if isinstance(v, torch.Tensor) and "cache" not in k else v for k, v in dev.items()}
    out = torch.zeros((4, step.hq * step.d), dtype=torch.float16)
    wide = torch.zeros(8, dtype=torch.int32)
    wide[::2] = host["tree_parents"]
    for parents in (wide[::2], wide[::2].numpy()):
        with pytest.raises(H.pkg.GenaiB200Error, match="tree_parents"):
            op.evaluate({**host, "tree_parents": parents}, {"output": out})
    assert bool((out == 0).all())
    for parents in (host["tree_parents"], host["tree_parents"].numpy()):
        op.evaluate({**host, "tree_parents": parents}, {"output": out})
        step.check(out.to(step.dev))
