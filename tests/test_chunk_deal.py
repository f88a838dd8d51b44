"""The dealing of the chunk attention's tiles to workgroups, on the CPU: the arithmetic that the kernel uses
(csrc/q36_chunk.h) walked by tests/chunk_check.cpp over single requests at every border and over ragged batches.
Every step of every tile lies in exactly one run, every tile is written once, and the combine reads exactly the
partials that the same call's workgroups write."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("deal") / "chunk_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-I", os.path.join(HERE, "..", "bundles_amd", "csrc"), "-o", out,
                    os.path.join(HERE, "chunk_check.cpp")], check=True)
    return out


@pytest.mark.parametrize("seed", [1, 2])
def test_every_step_once_and_every_partial_read_was_written(exe, seed):
    r = subprocess.run([exe, str(seed), "4000"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
