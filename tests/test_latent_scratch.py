"""Builds and runs tests/cpp/latent_scratch_test.cu: what a reserve makes room for, over all sizes and forms, without a GPU."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_a_reserve_holds_every_smaller_step(pkg, tmp_path):
    from openvino_genai_b200 import build
    pkg.build_all()
    exe = tmp_path / "latent_scratch_test"
    cmd = [build._nvcc(), "-std=c++17", "-O1", "-I", str(build.CSRC), "-I", str(ROOT / "include"), str(ROOT / "tests" / "cpp" / "latent_scratch_test.cu"),
           "-L", str(build.LIB_DIR), "-lgenai_b200", "-Xlinker", "-rpath", "-Xlinker", str(build.LIB_DIR), "-o", str(exe)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout
