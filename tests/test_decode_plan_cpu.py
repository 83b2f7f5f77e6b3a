"""The plan of the even-split decode (mllm_b200/csrc/decode_stream.cuh), compiled for the host: where the joining kernel
looks for the parts of a pair.  CPU only."""
import os
import subprocess

from mllm_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_parts_of_a_pair(tmp_path):
    """Also where the pair's place was never written (a CTA gave up a wait) and the workspace holds anything there."""
    out = str(tmp_path / "own_parts_check")
    subprocess.run([build.nvcc(), *build.ARCH, "-std=c++17", "-O1", "--expt-relaxed-constexpr",
                    "-I", build.CSRC, "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "native", "own_parts_check.cu"), "-o", out], check=True)
    r = subprocess.run([out], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.split() == ["all_places", "no_tiles", "any_bytes"]
