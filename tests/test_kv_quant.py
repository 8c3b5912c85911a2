"""CPU checks of the quantised KV cache and the token log probabilities: the
tile layout, and what the C entry points refuse before they touch a device."""
import os
import subprocess

import pytest

from conftest import PKG, ROOT

CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    lib = os.path.join(PKG, "libuocr_q8.so")
    if not os.path.exists(lib):
        subprocess.run(["make", "-s", "-C", PKG], check=True)
    exe = str(tmp_path_factory.mktemp("kvq") / "kvq_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", f"{CUDA}/include", "-o", exe,
                    os.path.join(ROOT, "tests", "kvq_check.cpp"), lib, f"-Wl,-rpath,{PKG}"],
                   check=True)
    return exe


@pytest.mark.parametrize("part", ["layout", "refusals"])
def test_kvq_check(check, part):
    r = subprocess.run([check, part], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
