"""Masked attention on the GPU: how many bits of its numbers survive, where a looser tolerance would not tell."""
import numpy as np
import pytest
import torch

from tests import masked_harness as H

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,bs", [(64, 16), (128, 32)])
def test_bf16_chunks_are_as_exact_as_a_causal_step(d, bs):
    """The operator's tolerance for 16-bit caches, 2e-3 of the result as a whole.  The output's own rounding takes 1.7e-3 of it (a relative error that is spread
    evenly over half a step of 2^-8 .. 2^-9 has a root mean square of 1.66e-3), so probabilities of 8 bits, another 1.6e-3 of the same kind, do not fit."""
    rng = np.random.default_rng(1)
    for past, new, trees, window in (([700, 90], [200, 64], None, 300), ([3000], [100], [H.tree(rng, 100)], 0), ([2, 40], [300, 77], None, 20)):
        step = H.Step(past, new, d=d, bs=bs, act="bf16", cache="bf16", window=window, trees=trees, seed=window)
        out, _, _, status = step.run()
        ref, _ = step.reference()
        err = ((out.double() - ref).norm() / ref.norm()).item()
        assert status == 0 and err <= 2e-3, err


@pytest.mark.parametrize("hq,hkv", [(8, 2), (24, 2)])
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 32)])
def test_single_tokens_over_a_bf16_cache(d, bs, hq, hkv):
    """The same tolerance, with a plan and without one, eight heads a kv head and more."""
    for past, window in (([700, 1500, 90, 300] * 8, 1000), ([4000, 3000, 100, 7] * 8, 3500)):
        step = H.Step(past, [1] * len(past), hq=hq, hkv=hkv, d=d, bs=bs, act="bf16", cache="bf16", window=window, sinks=4, seed=window)
        out, _, _, status = step.run()
        ref, _ = step.reference()
        err = ((out.double() - ref).norm() / ref.norm()).item()
        assert status == 0 and err <= 2e-3, err


@pytest.mark.parametrize("d,bs", [(64, 16), (128, 32)])
def test_u8_chunks_are_rounded_four_times(d, bs):
    """Keys, values, probabilities and the output, each to f16 once: a relative error spread evenly over half a step of 2^-11 .. 2^-12 has a root mean square of 2.1e-4, four
    independent ones 4.2e-4.  Scales rounded on top of that (two more a token) do not fit under 5e-4."""
    rng = np.random.default_rng(2)
    for past, new, trees, window in (([700, 90], [200, 64], None, 300), ([3000], [100], [H.tree(rng, 100)], 0), ([2, 400], [300, 77], None, 100)):
        step = H.Step(past, new, d=d, bs=bs, act="f16", cache="u8", window=window, trees=trees, seed=window)
        out, _, _, status = step.run()
        ref, _ = step.reference()
        err = ((out.double() - ref).norm() / ref.norm()).item()
        assert status == 0 and err <= 5e-4, err
