"""Encrypted linear attention with decay and rotary positions on two axes, composed
from the language-model operators, against float64: token by token over kept keys
and values, and as a whole layer over a prompt (both pairings of features). The bars
are derived in tests/cpp/decoder_test.cpp. Parity unpinned by the reference, which
has no transformer code."""
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", [["tokens"], ["layer"], ["layer", "halves"]], ids=" ".join)
def test_decoder(pkg, mode):
    if not os.path.exists(pkg.LIB_PATH):
        pkg.build()
    subprocess.check_call(["make", "-s", "-C", CPP, "decoder_test"])
    cmd = [os.path.join(CPP, "decoder_test"), os.path.join(pkg.PARAM_DIR, "bootparam_40.json")] + mode
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=1500)
    print(r.stdout[-3000:])
    print(r.stderr[-3000:])
    assert r.returncode == 0 and "PASS" in r.stdout
