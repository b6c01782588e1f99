"""The checkpoint tables of the generator streams (mpc_amd/csrc/prg.hip: the host's walk, the background thread, the device
copy), built for the CPU with a stand-in for the HIP runtime (table_check/) and the thread sanitizer."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def table_check(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("table_check") / "table_check")
    src = os.path.join(HERE, "table_check")
    for sanitize in (["-fsanitize=thread"], []):  # without it where the sanitizer cannot map its memory
        subprocess.run(["g++", "-std=c++17", "-O2", "-g", "-pthread", "-w", *sanitize, "-I", src,
                        "-I", os.path.join(HERE, "..", "mpc_amd", "csrc"), os.path.join(src, "table_check.cpp"), "-o", exe, "-ldl"], check=True)
        if subprocess.run([exe, "nothing"], capture_output=True).returncode == 2:
            break
    return exe


@pytest.mark.parametrize("what", ["short", "long", "sources", "threads"])
def test_tables(table_check, what):
    env = dict(os.environ, MPCX_CKPT_CACHE="", MPCX_PRG_MARKS="", TSAN_OPTIONS="halt_on_error=1")
    r = subprocess.run([table_check, what], env=env, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stderr[-4000:]
