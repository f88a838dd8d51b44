"""The page plan's counts on the CPU: the arithmetic that the kernel uses (csrc/q36_plan.h) at the borders of an int."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_pages_of_any_two_counts(tmp_path):
    exe = str(tmp_path / "plan_check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-I",
                    os.path.join(HERE, "..", "bundles_amd", "csrc"), "-o", exe, os.path.join(HERE, "plan_check.cpp")], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
