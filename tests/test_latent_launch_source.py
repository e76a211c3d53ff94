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


# ---- programmatic dependents: every kernel waits for the one before it, on every path --------------------------------------
# The kernels that read, before they wait, what an earlier kernel than the one before them has written (the plan, in both cases)
EARLY_READERS = {"project_value_kernel": "attend_kernel", "expanded_attend_kernel": "expand_kernel"}


def test_every_kernel_is_a_dependent_and_waits():
    launched = "".join(re.findall(r"launch_dependent\([^;]*;", "".join(SOURCES.values())))
    for name, body in KERNELS.items():
        assert re.search(r"\b%s\b" % name, launched), f"{name} is not launched as a dependent"
        assert "grid_wait()" in body, f"{name} does not wait"
        # the kernel's own returns (a lambda's give a value): none in front of the first wait, but for a branch that waits itself
        ahead = body[:body.rindex("grid_wait()")] if name == "project_value_kernel" else body[:body.index("grid_wait()")]
        for m in re.finditer(r"\breturn;", ahead):
            assert re.search(r"grid_wait\(\);\s*$", ahead[:m.start()]), f"{name} may leave before it has waited"
    assert "<<<" not in "".join(SOURCES.values())


def test_a_kernel_lets_the_next_one_come_only_behind_its_own_wait():
    """So that a kernel that has come early finds what the kernel before the one before it wrote."""
    for name, body in KERNELS.items():
        releases = [m.start() for m in re.finditer(r"grid_release\(\)", body)]
        for at in releases:
            assert re.search(r"grid_wait\(\);\s*pa::$", body[:at]), f"{name}: released at {at} without a wait directly in front"
    for before in EARLY_READERS.values():
        assert "grid_release()" in KERNELS[before]
    assert not any("grid_release()" in KERNELS[n] for n in EARLY_READERS), "what follows them may read what they read early"


def test_early_readers_touch_nothing_of_the_kernel_before_them_ahead_of_their_wait():
    value, attend = KERNELS["project_value_kernel"], KERNELS["expanded_attend_kernel"]
    ahead = value[:value.rindex("grid_wait()")]
    assert "a.token_prefix[B]" in ahead and not re.search(r"a\.(row_part|part_ml|part_o|output)\b", ahead)
    # the two warps that bring in what the expansion made; the others hear of it from them
    loader, values = attend.index("a.order["), attend.index("&a.map_v,")
    for use in ("&a.map_k,", "&a.map_k_rope,", "&a.map_qn,", "atomicAdd(a.arrived"):
        assert attend.index("if (ni == 0) pa::grid_wait();") < attend.index(use), use
    assert loader < attend.index("if (ni == 0) pa::grid_wait();")
    branch = attend.rindex("warp == 10", 0, values)
    assert "pa::grid_wait();" in attend[branch:values]
