"""The kernels of latent attention, read from their sources (comments apart): what a CTA does when one of its bounded waits has run out."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "openvino.genai_b200" / "csrc"
SOURCES = {p.name: re.sub(r"//[^\n]*", "", p.read_text()) for p in sorted(CSRC.glob("latent_*.cu"))}


def _kernels(text):
    """name -> body of every __global__ function."""
    out = {}
    for m in re.finditer(r"__global__ void (?:__launch_bounds__\([^{;]*?\)\s+)?(\w+)\((?:[^()]|\([^()]*\))*\)\s*\{", text):
        depth, i = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        out[m.group(1)] = text[m.end():i]
    return out


KERNELS = {name: body for text in SOURCES.values() for name, body in _kernels(text).items()}


def test_all_kernels_are_found():
    assert set(KERNELS) == {"append_kernel", "project_query_kernel", "attend_kernel", "project_value_kernel", "expanded_plan_kernel", "expand_kernel",
                            "expanded_attend_kernel"}


def test_a_cta_gives_its_memory_back_when_what_it_asked_for_is_there():
    """Behind the barrier at which all roles have ended, and only there, is the abort flag final: copies and products under way are waited for
    behind it, and the tensor memory is freed after that."""
    waiting = {n: b for n, b in KERNELS.items() if "Waiter" in b}
    assert len(waiting) == 5
    for name, body in waiting.items():
        freed = body.rindex("tc05::tmem_dealloc")
        at = body.rindex("abort_flag) drain" if "abort_flag) drain" in body else "(volatile int*)&", 0, freed)
        assert "__syncthreads();" in body[:at], name
        assert "drain_products(" in body[at:freed], f"{name}: products may be under way"
        if "expect_tx" in body:
            assert len(re.findall(r"\bdrain\(", body)) >= 1, f"{name}: copies may be under way"
        # every wait is bounded
        assert re.search(r"Waiter wt\{&(sm\.)?abort_flag, m\.status, m\.wait_polls\};", body), name
        assert not re.search(r"while\s*\(!\s*pa::mbar", body) and "mbar_try_wait" not in body, f"{name}: a wait without a limit"
