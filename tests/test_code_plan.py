"""The plan of attention over a quantised cache: rows of a workgroup, parts and
workspace at zero, the smallest and the largest sizes, under AddressSanitizer and
UndefinedBehaviorSanitizer (tests/host/code_plan_check.cpp, CPU only), and the
same queries of the shipped library."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "distributed_gptq_amd", "csrc")


def test_plans(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "code_plan_check")
    subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I",
                    os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "host", "code_plan_check.cpp"),
                    os.path.join(CSRC, "plan.cpp"), os.path.join(CSRC, "status.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and " 0 check(s) failed" in r.stderr, r.stderr[-2000:]
    lines = r.stdout.splitlines()
    assert len(lines) > 10000
    from distributed_gptq_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    size = _lib.load().gptq_code_attention_workspace_size
    for line in lines[::7]:
        *args, want = map(int, line.split())
        assert size(*args) == want, line


def test_kinds_of_calls():
    """What is cut and what is not: one token over many, a batch, a chunk."""
    from distributed_gptq_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    size = _lib.load().gptq_code_attention_workspace_size

    def splits(B, T, H, Hk, D, n):
        b = size(B, T, H, Hk, D, n)
        assert b % (4 * T * H * (D + 2)) == 0
        return max(b // (4 * T * H * (D + 2)), 1)
    assert splits(1, 1, 32, 8, 128, 8192) == 64                       # 512 workgroups of 128 keys or more
    assert splits(1, 1, 32, 8, 128, 128) == 1 and splits(1, 1, 32, 8, 128, 129) == 2
    assert splits(8, 8, 32, 8, 128, 8192) == 8 and splits(9, 9, 32, 8, 128, 8192) == 15  # 1024 for many sequences
    assert splits(1, 64, 32, 8, 128, 16384) == 32                     # 256 rows: two workgroups of 128 a part
    assert splits(1, 65, 32, 8, 128, 16384) == 16                     # 260 rows: two of 256, one to a CU
    assert splits(1, 65, 32, 8, 64, 16384) == 22                      # (heads of up to 64: three of 128)
    assert splits(1, 4096, 32, 8, 128, 16384) == 1
