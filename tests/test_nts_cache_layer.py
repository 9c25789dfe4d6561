"""More of the cache on pages through the nts:: host layer (tests/cpp/nts_cache_layer_tests.cpp): tensors without memory are refused on the
CPU; both types, prefixes and rows without a causal limit on the GPU."""
import os
import signal
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TESTS = os.path.join(ROOT, "tests", "cpp", "build", "nts_cache_layer_tests")


@pytest.mark.parametrize("case", ["starts", "rotation", "queries"])
def test_a_tensor_without_memory_is_refused(case):
    """It must not be taken for one that was not given."""
    assert os.path.exists(TESTS), "build tests/cpp first (__graft_entry__.build())"
    p = subprocess.run([TESTS, "--abort", case], capture_output=True, text=True, timeout=60)
    assert p.returncode == -signal.SIGABRT, (p.returncode, p.stderr)
    assert p.stderr.startswith("[ERROR]") and "Empty input tensors!" in p.stderr, p.stderr


@pytest.mark.gpu
def test_cache_layer():
    assert os.path.exists(TESTS), "build tests/cpp first (__graft_entry__.build())"
    print("\n[gpu-case] nts_cache_layer_tests", flush=True)
    p = subprocess.run([TESTS], capture_output=True, text=True, timeout=120)
    print(p.stdout, p.stderr)
    assert p.returncode == 0 and "OK! Everything is good!" in p.stdout, p.stdout + p.stderr
