"""What the tensor-core matrix products leave after a wait that ran out: an error for
the caller to read, and no result stored (tests/cpp/gemm_expired.cu)."""
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
pytestmark = pytest.mark.gpu


def test_nothing_is_stored_after_an_expired_wait():
    subprocess.check_call(["make", "-s", "-C", CPP, "gemm_expired"])
    r = subprocess.run([os.path.join(CPP, "gemm_expired")], capture_output=True, text=True, timeout=300)
    print(r.stdout[-2000:], r.stderr[-2000:])
    assert r.returncode == 0 and "PASS" in r.stdout
