"""Forms of the encrypted transformer layer that have to leave the same words: attention's
products in blocks of any size, one rank or two, softmax or linear attention, called again; and softmax
attention with rotary positions against float64 (tests/cpp/layer_forms_test.cpp). Parity
unpinned by the reference, which has no transformer code."""
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["blocks softmax", "blocks linear", "ranks softmax", "ranks linear", "again", "rotary"])
def test_layer_forms(pkg, mode):
    if not os.path.exists(pkg.LIB_PATH):
        pkg.build()
    subprocess.check_call(["make", "-s", "-C", CPP, "layer_forms_test"])
    cmd = [os.path.join(CPP, "layer_forms_test"), os.path.join(pkg.PARAM_DIR, "bootparam_40.json")] + mode.split()
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=900)
    print(r.stdout[-3000:])
    print(r.stderr[-3000:])
    assert r.returncode == 0 and "PASS" in r.stdout
