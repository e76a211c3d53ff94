"""Waits of latent attention's kernels that run out: the call returns with its status bit, and nothing of it is left in the calls behind it.

PA_B200_LATENT_TEST_WAIT_POLLS, read when a handle is made, is how often a wait looks at its barrier before it gives up.  With 0 every wait gives up at
once, whatever is under way; with a few, some do and some do not.  No kernel is broken by it: each ends, after what it had asked for has arrived."""
import pytest
import torch

from tests import latent_harness as LH

pytestmark = pytest.mark.gpu

STEPS = {
    "rows": dict(past=[700, 0, 3000, 63], new=[1, 4, 2, 1], heads=10),
    "wide rows": dict(past=[260, 5000], new=[2, 1], heads=96, bs=64),
    "prompts": dict(past=[0, 37, 2500, 5], new=[300, 5, 90, 1], heads=12, bs=16),
    "small prompts": dict(past=[300, 1, 2000], new=[257, 130, 20], heads=6, sizes=LH.SMALL, dtype="f16"),
}


@pytest.mark.parametrize("polls", [0, 1, 8, 64, 512])
@pytest.mark.parametrize("form", ["absorbed", "expanded", "auto"])
def test_the_call_returns_with_its_status_bit(pkg, monkeypatch, form, polls):
    from openvino_genai_b200 import _latent_abi as A
    for name, kw in STEPS.items():
        st = LH.Step(seed=11, **kw)
        x = st.device_inputs()
        monkeypatch.setenv("PA_B200_LATENT_TEST_WAIT_POLLS", str(polls))
        short = st.operator(pkg)
        monkeypatch.delenv("PA_B200_LATENT_TEST_WAIT_POLLS")
        want = st.expected()
        for _ in range(2):      # (the second call finds the first one's bytes in the scratch)
            out = st.attend(short, form, x)
            status = short.device_status()
            assert status in (0, A.PA_DEV_WAIT_TIMEOUT_LATENT), f"{name}: {status:#x}"
            assert status or polls > 0, f"{name}: no wait ran out"
            if status == 0:
                st.check(out, want)
        # another handle on the same device, directly behind it
        whole = st.operator(pkg)
        st.check(st.attend(whole, form, x), want)
        assert whole.device_status() == 0


def test_scratch_of_other_forms_and_steps_leads_nowhere(pkg, monkeypatch):
    """Handles with every wait cut short, over steps whose scratch is laid out in other ways: what an earlier call left is all that the join finds."""
    from openvino_genai_b200 import _latent_abi as A
    steps = [LH.Step(seed=5, **kw) for kw in (dict(past=[4000, 100], new=[1, 300], heads=8), dict(past=[3], new=[1], heads=8), dict(past=[900] * 40, new=[2] * 40, heads=8))]
    monkeypatch.setenv("PA_B200_LATENT_TEST_WAIT_POLLS", "0")
    op = steps[0].operator(pkg)
    for form in ("expanded", "absorbed", "auto", "absorbed"):
        for st in steps:
            st.attend(op, form)
            assert op.device_status() == A.PA_DEV_WAIT_TIMEOUT_LATENT
