"""Masked attention without a GPU: what a row sees as tiles and words of bits (tests/cpp/masked_words_test.cu, host code), the argument structs as
Python lays them out, and the refusals that need no device."""
import ctypes as C
import re
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "openvino.genai_b200" / "csrc"


def test_tiles_and_words_of_bits(pkg, tmp_path):
    from openvino_genai_b200 import build
    exe = tmp_path / "masked_words_test"
    cmd = [build._nvcc(), "-std=c++17", "-O2", "-I", str(CSRC), "-I", str(ROOT / "include"), str(ROOT / "tests" / "cpp" / "masked_words_test.cu"), "-o", str(exe)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


def test_structs_lie_as_the_header_says(pkg, tmp_path):
    from openvino_genai_b200 import _masked_abi as M
    structs = (M.pa_mask_args, M.pa_tree_accept_args)
    lines = []
    for s in structs:
        lines.append(f'printf("%zu\\n", sizeof({s.__name__}));')
        lines += [f'printf("%zu\\n", offsetof({s.__name__}, {name}));' for name, _ in s._fields_]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "masked_b200.h"\nint main(void) {\n' + "\n".join(lines) +
                   '\nprintf("%d\\n%d\\n%d\\n", PA_TREE_MAX_TOKENS, PA_TREE_NONE, (int)PA_DEV_BAD_TREE);\nreturn 0; }\n')
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()]
    want = [v for s in structs for v in [C.sizeof(s)] + [getattr(s, name).offset for name, _ in s._fields_]]
    assert got == want + [M.PA_TREE_MAX_TOKENS, M.PA_TREE_NONE, M.PA_DEV_BAD_TREE]


def test_refusals_without_a_handle(pkg):
    lib = pkg.load_library()
    from openvino_genai_b200 import _abi, _masked_abi as M
    mask, accept, args = M.pa_mask_args(), M.pa_tree_accept_args(), _abi.pa_forward_args()
    assert lib.pa_b200_forward_masked(None, C.byref(args), C.byref(mask)) == _abi.PA_ERR_INVALID_ARG
    assert lib.pa_b200_forward_masked_host(None, C.byref(args), C.byref(mask)) == _abi.PA_ERR_INVALID_ARG
    assert lib.pa_b200_tree_accept(None, C.byref(accept)) == _abi.PA_ERR_INVALID_ARG
    assert lib.pa_b200_masked_reserve(None, 1, 1, 1) == _abi.PA_ERR_INVALID_ARG
    assert b"handle" in lib.pa_b200_last_error()


def test_kernels_behind_the_masks_are_dependents_and_wait():
    """As those of a causal step: launched as programmatic dependents, waiting for the kernel before them on every path."""
    for name in ("masked_rows.cu", "masked_join.cu", "tree_accept.cu"):
        text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
        launched = "".join(re.findall(r"launch_dependent\([^;]*;|launch\([^;]*;", text))
        kernels = re.findall(r"__global__ void (?:__launch_bounds__\([^{;]*?\)\s+)?(\w+)\([^{]*\{(.*?)\n\}", text, flags=re.S)
        assert kernels and "<<<" not in text
        for kernel, body in kernels:
            assert re.search(r"\b%s\b" % kernel, launched), kernel
            assert "grid_wait()" in body and "return" not in body[:body.index("grid_wait()")], kernel
