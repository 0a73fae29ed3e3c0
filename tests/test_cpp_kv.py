"""The paged key-value cache through the C++ host side: tests/cpp/kv_check.cpp, built by __graft_entry__.build()."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXE = os.path.join(ROOT, "tests", "cpp", "_build", "kv_check")


def built():
    if not os.path.exists(EXE):
        import sys
        sys.path.insert(0, ROOT)
        import __graft_entry__ as entry
        entry.build_cpp_kv_check()
    return EXE


def test_errors_arrive_as_exceptions_without_a_device():
    if os.path.exists("/dev/kfd"):
        pytest.skip("a GPU is present")
    out = subprocess.run([built(), "--no-device"], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.count(" ok") == 4, out.stdout + out.stderr


@pytest.mark.gpu
def test_cpp_steps_through_the_cache():
    print("[gpu-case] C++ paged cache", flush=True)
    out = subprocess.run([built()], capture_output=True, text=True, timeout=120)
    print(out.stdout)
    assert out.returncode == 0 and "[cpp-kv] all ok" in out.stdout, out.stdout + out.stderr[-2000:]
