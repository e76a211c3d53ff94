"""Steps of latent attention beside the ordinary: tokens that no sequence owns, more query tiles than the plan lists, contexts that need several passes."""
import math

import numpy as np
import pytest
import torch

from tests import latent_harness as LH

pytestmark = pytest.mark.gpu

BAD_BEGINS = 2


@pytest.mark.parametrize("form", ["absorbed", "expanded", "auto", "append"])
@pytest.mark.parametrize("new", [[3, 2, 1], [90, 2, 70], [5, 300, 18]])
@pytest.mark.parametrize("where", ["in front", "behind"])
def test_tokens_that_no_sequence_owns_are_reported(pkg, form, new, where):
    """subsequence_begins that start behind the first token, or end before the last: these tokens have no output, and the status says so."""
    st = LH.Step([40, 90, 10], new, heads=6, bs=16, seed=17)
    op = st.operator(pkg)
    x = st.append_inputs()
    x["subsequence_begins"][0 if where == "in front" else 3] += 1 if where == "in front" else -1
    if form == "append":
        op.append(x, {"query_rope": torch.empty_like(x["query_rope"].contiguous())})
        assert op.device_status() == BAD_BEGINS
        return
    out = st.attend(op, form, x)
    assert op.device_status() == BAD_BEGINS
    left = slice(0, 1) if where == "in front" else slice(st.tokens - 1, st.tokens)
    assert bool(torch.isnan(out[left]).all())                 # (as they were)
    st.check(out, rows=[1, 2] if where == "in front" else [0, 1])


@pytest.mark.parametrize("form", ["expanded", "auto"])
@pytest.mark.parametrize("long_at", [3, 1023, 1090])
def test_more_query_tiles_than_the_plan_lists(pkg, form, long_at):
    """The plan lists 1024 query tiles in shared memory and searches for later ones: short sequences, some of them empty, with a long one on either side."""
    rng = np.random.default_rng(41)
    new = rng.integers(1, 21, 1300)
    new[rng.choice(1300, 120, replace=False)] = 0
    new[[1, 1022, 1024, 1299]] = [0, 0, 0, 5]
    past = rng.integers(0, 40, 1300)
    new[long_at], past[long_at] = 600, 300
    assert int(((new + 255) // 256).sum()) > 1024
    st = LH.Step(past, new, heads=2, sizes=LH.SMALL, bs=16, dtype="f16", seed=42)
    op = st.operator(pkg)
    x = st.device_inputs()
    out = st.attend(op, form, x)
    st.check(out)
    assert torch.equal(out, st.attend(op, form, x)) and op.device_status() == 0


def _definition(st):
    """The output in 64 bits [T, H, Dv], on the GPU, a head at a time."""
    R, P, Dn, Dv = st.sizes
    up, q = st.up.cuda(), st.query.cuda()
    out = torch.empty((st.tokens, st.heads, Dv), dtype=torch.float64)
    t = 0
    for s, rows in enumerate(st.context):
        n, p = int(st.new[s]), int(st.past[s])
        if n == 0:
            continue
        c = rows.cuda().double()
        hidden = torch.arange(p + n, device="cuda")[None] > p + torch.arange(n, device="cuda")[:, None]
        for h in range(st.heads):
            qh, uh = q[t:t + n, h].double(), up[h].double()
            a = (qh[:, :Dn] @ (c[:, :R] @ uh[:Dn].T).T + qh[:, Dn:] @ c[:, R:].T) / math.sqrt(Dn + P)
            a = torch.softmax(a.masked_fill(hidden, -math.inf), -1)
            out[t:t + n, h] = (a @ (c[:, :R] @ uh[Dn:].T)).cpu()
        t += n
    return out


@pytest.mark.parametrize("form,heads,past,new", [
    ("expanded", 32, [120000], [200]),                                 # two passes, the context cut
    ("expanded", 24, [90000, 40000, 3], [300, 5, 40]),
    ("auto", 128, [90000, 70000, 50000, 900], [1, 1, 3, 100]),         # the passes go by the whole step's contexts, the work by the last one's
])
def test_several_passes_against_the_definition(pkg, form, heads, past, new):
    st = LH.Step(past, new, heads=heads, bs=64, seed=43)
    op = st.operator(pkg)
    x = st.device_inputs()
    before = op.launch_count()
    out = st.attend(op, form, x)
    assert op.launch_count() - before > 3 + 3 * (form == "auto")
    st.check(out, _definition(st))
    assert op.device_status() == 0
