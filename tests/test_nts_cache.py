"""The cache on pages through the nts:: host layer (tests/cpp/nts_cache_tests.cpp): its refusals on the CPU, its results on the GPU."""
import os
import signal
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TESTS = os.path.join(ROOT, "tests", "cpp", "build", "nts_cache_tests")


@pytest.mark.parametrize("case,message", [
    ("type", "Input tensors should have the same data type!"),
    ("hidden", "The hidden size must be a multiple of the size of a head!"),
    ("shape", "Unmatched tensors in a cache!"),
    ("empty", "Empty input tensors!"),
    ("starts", "Unmatched tensors in a cache!"),
    ("integers", "Lengths, starts and page numbers must be integers!"),
    ("prefix", "A negative prefix!"),
    ("abi", "Empty"),
])
def test_refusals(case, message):
    assert os.path.exists(TESTS), "build tests/cpp first (__graft_entry__.build())"
    p = subprocess.run([TESTS, "--abort", case], capture_output=True, text=True, timeout=60)
    assert p.returncode == -signal.SIGABRT, (p.returncode, p.stderr)
    assert p.stderr.startswith("[ERROR]") and message in p.stderr, p.stderr


@pytest.mark.gpu
def test_nts_cache_layer():
    assert os.path.exists(TESTS), "build tests/cpp first (__graft_entry__.build())"
    print("\n[gpu-case] nts_cache_tests", flush=True)
    p = subprocess.run([TESTS], capture_output=True, text=True, timeout=120)
    print(p.stdout, p.stderr)
    assert p.returncode == 0 and "OK! Everything is good!" in p.stdout, p.stdout + p.stderr
