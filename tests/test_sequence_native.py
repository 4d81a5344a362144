"""Runs the native caller of the sequence operators (tests/native/seq_driver.cpp), built like abi_driver.cpp with the host
code, the library's included, under AddressSanitizer + UBSan."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu
BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native", "_build", "seq_driver")


def test_native_sequence_driver_under_host_sanitizers():
    if not os.path.exists(BIN):
        pytest.skip(f"{BIN} is missing: `make -C tests/native` builds it")
    env = dict(os.environ)
    env["ASAN_OPTIONS"] = "detect_leaks=0:abort_on_error=0:halt_on_error=1"      # the HIP runtime's own allocations
    env["UBSAN_OPTIONS"] = "print_stacktrace=1:halt_on_error=1"
    r = subprocess.run([BIN], env=env, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, f"rc={r.returncode}\nstdout:\n{r.stdout[-2000:]}\nstderr:\n{r.stderr[-4000:]}"
    assert "seq_driver OK" in r.stdout
    assert "ERROR: AddressSanitizer" not in r.stderr and "runtime error:" not in r.stderr, r.stderr[-4000:]
