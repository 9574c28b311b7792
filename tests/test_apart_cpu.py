"""Which outputs the language-model operators refuse (csrc/apart.h), without a GPU: the
header compiled by itself, against every pair of ranges compared with every other."""
import ctypes as C
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WRAPPER = r"""
#include "apart.h"
typedef const char *const *P;
// 1: refused
extern "C" int refused(size_t bytes, P y, int ny, P x, int nx, P own, size_t w, size_t w_bytes) {
  cfhe::Outputs o(bytes);
  o.add({y, y + ny / 2}, ny / 2);
  o.add({y + ny / 2 * 2}, ny % 2);
  return !o.apart() || o.meet(x, nx, own) || (w_bytes && o.meet((const void *)w, w_bytes));
}
"""


@pytest.fixture(scope="module")
def refused(tmp_path_factory):
    folder = tmp_path_factory.mktemp("apart")
    src, lib = str(folder / "apart.cpp"), str(folder / "apart.so")
    with open(src, "w") as f:
        f.write(WRAPPER)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC",
                           "-I" + os.path.join(ROOT, "cheddar-fhe_b200", "csrc"), src, "-o", lib])
    f = C.CDLL(lib).refused

    def call(size, y, x=(), own=None, w=0, w_size=0):
        def table(t):
            return (C.c_size_t * max(1, len(t)))(*t)
        return bool(f(C.c_size_t(size), table(y), len(y), table(x), len(x), table(own) if own else None,
                      C.c_size_t(w), C.c_size_t(w_size)))
    return call


def test_outputs_that_meet_one_another(refused):
    assert not refused(64, [1000, 1064, 2000, 936])  # one after the other, in any order
    assert refused(64, [1000, 1063]) and refused(64, [1063, 1000]) and refused(64, [1000, 5000, 1000])
    # leading shape [2, 2] with both strides one polynomial: (0, 1) is (1, 0)
    assert refused(64, [1000 + 64 * (i + j) for i in range(2) for j in range(2)])
    assert not refused(64, [1000 + 64 * (2 * i + j) for i in range(2) for j in range(2)])


def test_outputs_that_meet_an_operand(refused):
    y = [1000 + 128 * i for i in range(4)]
    for x in (1000, 1063, 937, 1128, 1383 + 64, 1384 + 0):
        assert refused(64, y, [4000, x]) == any(abs(x - o) < 64 for o in y), x
    assert not refused(64, y, [936, 1064, 1448, 5000])
    assert not refused(64, y, [0, 0])  # an operand that is not there
    # in place, entry by entry; another entry's output is none of its own
    assert not refused(64, y, y, y)
    assert refused(64, y, [y[1], y[0], y[2], y[3]], y)
    assert refused(64, y, [y[0] + 4, y[1], y[2], y[3]], y)
    assert not refused(64, y, [0, y[1], 0, 9000], y)
    # a larger operand, the packed weights
    assert refused(64, y, w=0x10, w_size=1000 - 0x10 + 1) and not refused(64, y, w=0x10, w_size=1000 - 0x10)
    assert refused(64, y, w=1100, w_size=500) and not refused(64, y, w=1064, w_size=64)


def test_against_every_pair(refused):
    rng = random.Random(7)
    seen = set()
    for _ in range(3000):
        size = rng.choice([16, 64, 100])
        y = [4 * rng.randrange(1, 400) for _ in range(rng.randrange(1, 5))]
        x = [4 * rng.randrange(0, 400) for _ in range(rng.randrange(0, 5))]
        own = [rng.choice(y) for _ in x]
        x = [rng.choice([v, v, o]) for v, o in zip(x, own)]
        w, w_size = 4 * rng.randrange(1, 400), rng.choice([0, 4, 300])
        want = any(abs(a - b) < size for i, a in enumerate(y) for b in y[:i])
        want = want or any(v and v != o and abs(v - a) < size for v, o in zip(x, own) for a in y)
        want = want or any(w_size and w < a + size and a < w + w_size for a in y)
        assert refused(size, y, x, own, w, w_size) == want, (size, y, x, own, w, w_size)
        seen.add(want)
    assert seen == {False, True}
