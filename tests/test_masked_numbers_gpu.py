"""Masked attention on the GPU over numbers that leave the range of the tensor-core kernel's operands."""
import numpy as np
import pytest
import torch

from tests import masked_harness as H

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_keys_of_a_wide_range_in_the_u8_cache(act):
    """Outlier channels: a step of the quantiser that takes (byte - 128) * step out of the f16 range.  Small steps of the softmax keep the logits moderate."""
    for trees in (None, [H.tree(np.random.default_rng(2), 40), None]):
        step = H.Step([90, 200], [40, 1], act=act, cache="u8", scale=2e-5, trees=trees, poison=False, seed=11)
        g = torch.Generator(device=step.dev)
        g.manual_seed(3)
        def widen(x):       # [..., d]: two channels far out, by a different amount for every token
            far = torch.rand(x.shape[:-1], generator=g, device=step.dev) * 9e4 + 1e4
            x = x.clone()
            x[..., 3], x[..., 7] = -far, far
            return x
        step.packed["key"] = step.pack(widen(step.values["key"]), False)
        step.key = widen(step.key.float().view(step.T, step.hkv, step.d)).view(step.T, -1).to(step.key.dtype)
        out, _, _, status = step.run()
        assert status == 0
        step.check(out)
