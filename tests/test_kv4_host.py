"""Host checks of what the attention over the 4-bit cache takes from the caller's data, and of its refusals (no GPU)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rows_and_positions_of_any_starts(tmp_path):
    """Starts that descend, lie out of range or are as far apart as 32 bits allow."""
    exe = tmp_path / "kv4_rows_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "ternary-llm_amd", "csrc"), os.path.join(ROOT, "tests", "kv4_rows_check.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and "bad=0" in out.stdout, out.stdout + out.stderr
