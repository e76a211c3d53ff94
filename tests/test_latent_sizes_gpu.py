"""Latent attention at every combination of its sizes: each is an instance of the kernels of its own."""
import itertools

import numpy as np
import pytest
import torch

from tests import latent_harness as LH

pytestmark = pytest.mark.gpu

SIZES = list(itertools.product((256, 512), (32, 64), (64, 128), (64, 128)))


@pytest.mark.parametrize("dtype,bs", [("bf16", 32), ("f16", 64), ("bf16", 16)])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "/".join(map(str, s)))
def test_every_size(pkg, sizes, dtype, bs):
    st = LH.Step([0, 333, 64, 1500, 0, 40], [1, 3, 70, 1, 290, 17], heads=9, sizes=sizes, bs=bs, dtype=dtype, seed=sum(sizes) + bs)
    op = st.operator(pkg)
    x, want = st.device_inputs(), st.expected()
    for form in ("absorbed", "expanded", "auto"):
        st.check(st.attend(op, form, x), want)
    assert op.device_status() == 0


@pytest.mark.parametrize("seed", range(24))
def test_steps_drawn_at_random(pkg, seed):
    """Sizes, heads, lengths and forms as they come, two steps of other shapes in turn on one operator."""
    rng = np.random.default_rng(1000 + seed)
    sizes, dtype, bs = SIZES[rng.integers(16)], rng.choice(["bf16", "f16"]), int(rng.choice([16, 32, 64]))
    heads = int(np.exp(rng.uniform(0, np.log(160))))
    length = lambda n, top: np.floor(np.exp(rng.uniform(0, np.log(top), n))).astype(np.int64)
    op = None
    for turn in range(3):
        n = int(length(1, 40)[0])
        new = length(n, rng.choice([2, 6, 100, 400])) - (rng.random(n) < 0.1)
        past = length(n, rng.choice([2, 100, 4000])) - 1
        while int((new * (past + new)).sum()) * heads > 4e7:
            new, past = (new + 1) // 2, past // 2
        st = LH.Step(past, new, heads=heads, sizes=sizes, bs=bs, dtype=dtype, seed=seed * 10 + turn)
        op = op or st.operator(pkg)
        if not st.tokens:
            continue
        x, want = st.device_inputs(), st.expected()
        for form in rng.permutation(["absorbed", "expanded", "auto"]):
            out = st.attend(op, str(form), x)
            st.check(out, want)
            assert torch.equal(out, st.attend(op, str(form), x)), "the same inputs gave other bits"
        assert op.device_status() == 0
