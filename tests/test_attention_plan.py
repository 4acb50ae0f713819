"""The attention calls' host-side plans, workspace queries and argument checks
at zero, the smallest and the largest sizes, under AddressSanitizer and
UndefinedBehaviorSanitizer (tests/host/attention_plan_check.cpp, CPU only), and
the same queries of the shipped library; the kernels' index arithmetic with
whatever the device arrays may hold, likewise
(tests/host/attention_index_check.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "distributed_gptq_amd", "csrc")


@pytest.fixture(scope="module")
def checked(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path_factory.mktemp("attention_plan") / "attention_plan_check")
    subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I",
                    os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "host", "attention_plan_check.cpp"),
                    os.path.join(CSRC, "plan.cpp"), os.path.join(CSRC, "status.cpp"), "-o", exe], check=True)
    return subprocess.run([exe], capture_output=True, text=True, timeout=300)


def test_plans(checked):
    assert checked.returncode == 0 and "0 check(s) failed" in checked.stderr, checked.stderr[-2000:]
    assert len(checked.stdout.splitlines()) > 10000


def test_the_shipped_library_agrees(checked):
    from distributed_gptq_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    assert checked.returncode == 0, checked.stderr[-2000:]
    lib = _lib.load()
    for line in checked.stdout.splitlines():
        call, value = line.split(" = ")
        name, *args = call.split()
        assert getattr(lib, name)(*[int(a) for a in args]) == int(value), line


def test_index_arithmetic(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "attention_index_check")
    subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    os.path.join(ROOT, "tests", "host", "attention_index_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and " 0 check(s) failed" in r.stderr, r.stderr[-2000:]
