"""Steps of latent attention beside the ordinary: tokens that no sequence owns."""
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
