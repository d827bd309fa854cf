"""Which rows and positions a sequence has for the extremes of what the device arrays may hold: the kernels' own arithmetic, compiled for
the host (tests/kv4_sequence_test.cpp)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rows_and_positions_of_a_sequence(tmp_path):
    exe = str(tmp_path / "kv4_sequence_test")
    subprocess.check_call(["hipcc", "--offload-host-only", "-std=c++17", "-O2", "-x", "hip", os.path.join(ROOT, "tests", "kv4_sequence_test.cpp"), "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "sequences ok" in out.stdout
