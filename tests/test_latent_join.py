"""Builds and runs tests/cpp/latent_join_test.cu (host code only): the join of latent attention follows no record out of the scratch.  And the
kernel, read from its source, takes its records through that check only."""
import re
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "openvino.genai_b200" / "csrc"


def test_records_lead_nowhere_outside_the_scratch(pkg, tmp_path):
    from openvino_genai_b200 import build
    exe = tmp_path / "latent_join_test"
    cmd = [build._nvcc(), "-std=c++17", "-I", str(CSRC), "-I", str(ROOT / "include"), str(ROOT / "tests" / "cpp" / "latent_join_test.cu"), "-o", str(exe)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


def test_the_join_reads_its_records_through_the_check():
    text = re.sub(r"//[^\n]*", "", (CSRC / "latent_absorbed.cu").read_text())
    reads = re.findall(r"[^\n]*\ba\.row_part\[[^\n]*", text)
    writes = [line for line in reads if re.search(r"a\.row_part\[[^=]*\] = ", line)]
    assert len(writes) == 1
    assert [line for line in reads if line not in writes and "checked_part(a.row_part[" not in line] == [] and len(reads) == 2
    assert "k.part_rows = s.part_rows;" in (CSRC / "latent_api.cu").read_text()
