"""The row-by-row path of masked attention without a GPU: tiles and words of bits of single rows (tests/cpp/masked_rows_test.cu, host code)."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "openvino.genai_b200" / "csrc"


def test_a_row_goes_through_all_that_it_sees_and_nothing_else(pkg, tmp_path):
    from openvino_genai_b200 import build
    exe = tmp_path / "masked_rows_test"
    cmd = [build._nvcc(), "-std=c++17", "-O2", "-I", str(CSRC), "-I", str(ROOT / "include"), str(ROOT / "tests" / "cpp" / "masked_rows_test.cu"), "-o", str(exe)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout
