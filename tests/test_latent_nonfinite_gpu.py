"""Latent attention over not-a-number and infinities that a row sees: they are no answer, in either form and however the context is cut."""
import math

import pytest
import torch

from tests import latent_harness as LH

pytestmark = pytest.mark.gpu

# contexts of one tile, of several and of several pieces, each beside a sequence that is left alone
LENGTHS = {"short": ([40, 70], [2, 1]), "long": ([9000, 300], [1, 2]), "prompt": ([600, 5], [90, 3]), "cut": ([5000, 100], [40, 1])}


def _finite_as(st, got, want, tokens):
    """Outputs of `tokens` are finite where the definition's are, and right there."""
    a, b = got.double().reshape(want.shape)[tokens], want[tokens]
    ok = torch.isfinite(b)
    assert torch.equal(torch.isfinite(a), ok), f"{int((torch.isfinite(a) & ~ok).sum())} elements have a value that the definition does not give"
    if bool(ok.any()):
        assert float((a[ok] - b[ok]).norm() / b[ok].norm()) <= 2 * LH.UNIT[st.dtype]


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("form", ["absorbed", "expanded", "auto"])
@pytest.mark.parametrize("dtype,sizes", [("bf16", LH.WIDE), ("f16", LH.SMALL)])
def test_a_cached_row_that_is_not_finite(pkg, dtype, sizes, form, lengths, value):
    past, new = LENGTHS[lengths]
    st = LH.Step(past, new, heads=8, sizes=sizes, dtype=dtype, seed=13)
    op = st.operator(pkg)
    x = st.device_inputs()
    clean = st.attend(op, form, x)
    R, table = sizes[0], st.meta["block_indices"].tolist()
    mine = slice(0, new[0])
    for at in (0, past[0] // 2, past[0]):
        for element in (5, R + 3):      # of the latent, of the rotated part
            page, slot = table[at // st.bs], at % st.bs
            kept = x["cache"][page, slot, element].clone()
            x["cache"][page, slot, element] = value
            row = st.context[0][at, element].clone()
            st.context[0][at, element] = value
            out = st.attend(op, form, x)
            assert torch.equal(out[new[0]:], clean[new[0]:]), "another sequence's outputs"
            _finite_as(st, out, st.expected(), mine)
            x["cache"][page, slot, element] = kept
            st.context[0][at, element] = row
    assert torch.equal(st.attend(op, form, x), clean) and op.device_status() == 0


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("form", ["absorbed", "expanded", "auto"])
def test_a_query_that_is_not_finite(pkg, form, lengths, value):
    """Only that row of that head is lost."""
    past, new = LENGTHS[lengths]
    st = LH.Step(past, new, heads=8, seed=14)
    op = st.operator(pkg)
    x = st.device_inputs()
    clean = st.attend(op, form, x).reshape(st.tokens, 8, -1)
    for part, element in (("query_nope", 17), ("query_rope", 2)):
        kept = x[part][0, 3, element].clone()
        x[part][0, 3, element] = value
        out = st.attend(op, form, x).reshape(st.tokens, 8, -1)
        x[part][0, 3, element] = kept
        assert not torch.isfinite(out[0, 3]).any(), "a value for a row whose logits have none"
        out[0, 3] = clean[0, 3]
        assert torch.equal(out, clean)
    assert op.device_status() == 0


@pytest.mark.parametrize("lengths", ["short", "long"])
def test_logits_that_are_all_minus_infinity(pkg, lengths):
    """A softmax of nothing but minus infinity has no value either."""
    past, new = LENGTHS[lengths]
    st = LH.Step(past, new, heads=4, seed=15)
    st.query[..., -64:] = -1.0
    for s, rows in enumerate(st.context):
        if s == 0:
            rows[:, -64:] = math.inf
            pos, table = torch.arange(len(rows)), st.meta["block_indices"].long()
            st.cache[table[pos // st.bs], pos % st.bs] = rows
    op = st.operator(pkg)
    for form in ("absorbed", "expanded"):
        _finite_as(st, st.attend(op, form), st.expected(), slice(0, st.tokens))


@pytest.mark.parametrize("past", [30, 6000])
def test_queries_whose_absorbed_row_leaves_the_f16_range(pkg, past):
    """key_up^T q is an operand of the absorbed products and has their type: where it overflows, the row is lost, not made up."""
    st = LH.Step([past], [1], heads=4, dtype="f16", seed=16)
    Dn = st.sizes[2]
    st.query[0, 1, :Dn] = 3e4 * torch.sign(st.up[1, :Dn, 7].float()).half()
    assert float((st.up[1, :Dn, 7].double() * st.query[0, 1, :Dn].double()).sum()) > 65520
    want, op = st.expected(), st.operator(pkg)
    out = st.attend(op, "absorbed").reshape(4, -1)
    assert not torch.isfinite(out[1]).any()
    rest = [0, 2, 3]
    assert float((out[rest].double() - want[0, rest]).norm() / want[0, rest].norm()) <= 2 * LH.UNIT["f16"]
    # the expanded form has no such product
    assert float((st.attend(op, "expanded").reshape(4, -1)[1].double() - want[0, 1]).norm() / want[0, 1].norm()) <= 2 * LH.UNIT["f16"]
