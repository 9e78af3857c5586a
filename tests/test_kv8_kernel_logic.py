"""CPU tests of device code of the 8-bit cache's attention that runs on the host as well: the headers
are compiled into small programs, which check themselves (tests/kv8_host)."""

import os
import subprocess

import pytest

import build

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "kv8_host")


@pytest.fixture(scope="session")
def run_program(tmp_path_factory):
    def run(name, *args):
        exe = str(tmp_path_factory.mktemp("kv8_host") / name)
        subprocess.run([build.nvcc_path(), "-gencode", "arch=compute_100a,code=sm_100a", "-O1", "-std=c++17", "-I", build.INCLUDE,
                        "-I", build.CSRC, "-o", exe, os.path.join(HERE, name + ".cu"), "-Xcompiler", "-pthread"], check=True)
        res = subprocess.run([exe, *args], capture_output=True, text=True, timeout=300)
        assert res.returncode == 0, res.stdout + res.stderr

    return run


def test_converting_warps_leave_together(run_program):
    """A warp that gives up at the wait for a piece or inside one leaves no other at their barrier."""
    run_program("pieces_together")


def test_line_of_work(run_program):
    """Shares of valid calls cover every tile once, cuts are where the merge looks; sums of query lengths that
    go back and forth, up to sums past 32 bits, lead nowhere outside the tensors."""
    run_program("line")
