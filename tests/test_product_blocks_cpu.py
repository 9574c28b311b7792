"""Blocks in which attention makes its products of ciphertexts (tests/cpp/product_blocks.cpp), without a GPU."""
import os
import subprocess

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


def test_blocks_cover_a_product(pkg):
    if not os.path.exists(pkg.LIB_PATH):
        pkg.build()
    subprocess.check_call(["make", "-s", "-C", CPP, "product_blocks"])
    r = subprocess.run([os.path.join(CPP, "product_blocks")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "blocks ok" in r.stdout
