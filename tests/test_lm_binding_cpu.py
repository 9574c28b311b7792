"""Argument handling of the Python calls of the language-model operators
(host/py_calls.c), without a GPU: the module is compiled against a stand-in for the
library that records what an entry point is given. What cannot be passed on safely
has to be an exception, with the entry point not called."""
import ctypes as C
import importlib.util
import os
import subprocess
import sysconfig

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
N = 65536
OTHERS = ["ntt", "intt", "binary", "const_op", "elementwise_multi", "tensor", "permute", "moddown", "keyswitch",
          "hmult", "hoisted_rotations", "linear_transform", "ctpt_gemm", "sample_uniform", "sample_error", "encrypt",
          "encode_coeffs", "beta"]

STAND_IN = r"""
#include <string.h>
#include <stdint.h>
typedef const uint32_t *const *T;
typedef uint32_t *const *W;
int calls = 0, shape[8];
const void *table[8][64];
uint32_t words[3][64];
static void keep(int t, const void *p, int n) { memset(table[t], 0, sizeof(table[t])); if (p) memcpy(table[t], p, n * sizeof(void *)); }
static void copy(int t, const uint32_t *p, int n) { memset(words[t], 0, sizeof(words[t])); if (p) memcpy(words[t], p, n * 4); }
int cfhe_degree(const void *h) { return 65536; }
int cfhe_ctpt_project(void *h, W yb, W ya, T xb, T xa, const void *p, int ni, int no, const uint32_t *b, T rb, T ra,
                      const uint32_t *s, const int *g, int n) {
  keep(0, yb, no); keep(1, ya, no); keep(2, xb, ni); keep(3, xa, ni); keep(4, rb, no); keep(5, ra, no);
  copy(0, b, n * no); copy(1, s, n); shape[0] = ni; shape[1] = no; shape[2] = n; calls++; return 0; }
int cfhe_rotary(void *h, W y, T x, int rows, int pairs, int halves, T c, T s, const int *g, int n) {
  keep(0, y, rows * 2 * pairs); keep(1, x, rows * 2 * pairs); keep(2, c, pairs); keep(3, s, pairs);
  shape[0] = rows; shape[1] = pairs; shape[2] = halves; calls++; return 0; }
int cfhe_rotary_token(void *h, W y, T x, int rows, int pairs, int halves, const uint32_t *c, const uint32_t *s,
                      const int *g, int n) {
  keep(1, x, rows * 2 * pairs); copy(0, c, pairs * n); copy(1, s, pairs * n);
  shape[0] = rows; shape[1] = pairs; shape[2] = halves; calls++; return 0; }
int cfhe_ctct_gemm(void *h, W d0, W d1, W d2, T lb, T la, T rb, T ra, int m, int k, int n, T w, const uint32_t *c,
                   const int *g, int nl) {
  keep(0, d0, m * n); keep(1, d1, m * n); keep(2, d2, m * n); keep(3, lb, m * k); keep(4, la, m * k);
  keep(5, rb, k * n); keep(6, ra, k * n); keep(7, w, w ? m * n : 0); copy(0, c, m * n * nl);
  shape[0] = m; shape[1] = k; shape[2] = n; calls++; return 0; }
"""


class Tensor:
    """What the binding asks of a device tensor: words at addr, any strides."""

    def __init__(self, addr, *shape, stride=None, size=4, device=0):
        self.addr, self.shape, self.size_, self.device_ = addr, tuple(shape), size, device
        if stride is None:
            stride, s = [], 1
            for d in reversed(shape):
                stride.insert(0, s)
                s *= d
        self.stride_ = tuple(stride)

    def data_ptr(self):
        return self.addr

    def stride(self):
        return self.stride_

    def element_size(self):
        return self.size_

    def get_device(self):
        return self.device_


class Binding:
    def __init__(self, folder):
        src, path = os.path.join(folder, "stand_in.c"), os.path.join(folder, "cheddar_b200_calls.so")
        with open(src, "w") as f:
            f.write(STAND_IN + "".join(f"int cfhe_{n}() {{ return -1; }}\n" for n in OTHERS))
        subprocess.check_call(["gcc", "-O1", "-w", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "include"),
                               "-I" + sysconfig.get_paths()["include"], src,
                               os.path.join(ROOT, "cheddar-fhe_b200", "host", "py_calls.c"), "-o", path])
        spec = importlib.util.spec_from_file_location("cheddar_b200_calls", path)
        self.k = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(self.k)
        self.k.set_converters(lambda a: np.ascontiguousarray(a, dtype=np.int32),
                              lambda a: np.ascontiguousarray(a, dtype=np.uint32))
        self.lib = C.CDLL(path)

    def value(self, name):
        return C.c_int.in_dll(self.lib, name).value

    def table(self, t, n):
        return list(((C.c_size_t * 64) * 8).in_dll(self.lib, "table")[t][:n])

    def words(self, t, n):
        return list(((C.c_uint32 * 64) * 3).in_dll(self.lib, "words")[t][:n])

    def shape(self):
        return list((C.c_int * 8).in_dll(self.lib, "shape")[:3])

    def refused(self, error, call, *args):
        before = self.value("calls")
        with pytest.raises(error):
            call(*args)
        assert self.value("calls") == before


@pytest.fixture(scope="module")
def b(tmp_path_factory):
    return Binding(str(tmp_path_factory.mktemp("calls")))


G = [3, 4]  # two limbs
POLY = 2 * N * 4  # bytes


def test_projection_operands(b):
    y, x = Tensor(0x1000, 3, 2, 2, N), [Tensor(0x100 * (k + 1), 2, 2, N) for k in range(2)]
    res = [Tensor(0x40, 2, 2, N), None, Tensor(0x80, 2, 2, N, stride=(8 * N, N, 1))]
    bias, scale = np.arange(6, dtype=np.uint32).reshape(2, 3), np.array([7, 8], dtype=np.uint32)
    assert b.k.ctpt_project(0, 0, y, x, Tensor(16, 4), G, bias, res, scale) == 0
    assert b.shape() == [2, 3, 2]
    assert b.table(0, 3) == [0x1000 + 2 * j * POLY for j in range(3)]
    assert b.table(1, 3) == [0x1000 + (2 * j + 1) * POLY for j in range(3)]
    assert b.table(3, 2) == [0x100 + POLY, 0x200 + POLY]
    assert b.table(4, 3) == [0x40, 0, 0x80] and b.table(5, 3) == [0x40 + POLY, 0, 0x80 + 32 * N]
    assert b.words(0, 6) == list(range(6)) and b.words(1, 2) == [7, 8]
    assert b.k.ctpt_project(0, 0, y, x, Tensor(16, 4), G, None, None, None) == 0
    assert b.table(4, 3) == [0, 0, 0]


def test_rotary_operands(b):
    x = Tensor(0x1000, 2, 4, 2, 2, N)
    assert b.k.rotary(0, 0, x, x, Tensor(0x10, 2, 2, N), [Tensor(0x20, 2, N), Tensor(0x30, 2, N)], G, True) == 0
    assert b.shape() == [4, 2, 1]  # two heads, both polynomials
    assert b.table(1, 16) == [0x1000 + (2 * i + p) * POLY for p in range(2) for i in range(8)]
    assert b.table(2, 2) == [0x10, 0x10 + POLY] and b.table(3, 2) == [0x20, 0x30]
    w = np.arange(4, dtype=np.uint32).reshape(2, 2)
    assert b.k.rotary(0, 0, x, x, w, w + 10, G, False) == 0
    assert b.words(0, 4) == [0, 1, 2, 3] and b.words(1, 4) == [10, 11, 12, 13] and b.shape()[2] == 0


def test_product_operands(b):
    # kept keys [token][feature] read as [feature][token]
    kept = Tensor(0x1000, 2, 3, 2, 2, N, stride=(2 * 2 * N, 2 * 2 * 2 * N, 2 * N, N, 1))
    q, d = Tensor(0x10, 1, 2, 2, 2, N), Tensor(0x20, 1, 3, 3, 2, N)
    assert b.k.ctct_gemm(0, 0, d, q, kept, G, None) == 0
    assert b.shape() == [1, 2, 3]
    assert b.table(5, 6) == [0x1000 + 2 * (j * 2 + t) * POLY for t in range(2) for j in range(3)]
    assert b.table(6, 1) == [0x1000 + POLY]
    assert b.table(2, 3) == [0x20 + (3 * j + 2) * POLY for j in range(3)]
    assert b.k.ctct_gemm(0, 0, [[Tensor(1, 3, 2, N)] * 3], q, kept, G, Tensor(0x40, 1, 3, 2, N)) == 0
    assert b.table(7, 3) == [0x40, 0x40 + POLY, 0x40 + 2 * POLY]
    assert b.k.ctct_gemm(0, 0, d, q, kept, G, np.arange(6, dtype=np.uint32).reshape(1, 3, 2)) == 0
    assert b.words(0, 6) == list(range(6)) and b.table(7, 1) == [0]


def test_refusals(b):
    k, y, x, w = b.k, Tensor(1, 3, 2, 2, N), Tensor(1, 2, 2, 2, N), Tensor(16, 4)
    words = np.zeros(6, dtype=np.uint32)
    for bad in (Tensor(1, 2, 2, 2, N, device=-1), Tensor(1, 2, 2, 2, N, device=1), Tensor(1, 2, 2, 2, N, size=8),
                Tensor(1, 2, 2, 3, N), Tensor(1, 2, 3, 2, N), Tensor(1, 2, 2, 2, N // 2), Tensor(1, 2, 2, N),
                Tensor(1, 2, 2, 2, N, stride=(4 * N, 2 * N, N + 4, 1)),
                Tensor(1, 2, 2, 2, N, stride=(4 * N, 2 * N, N, 2)), [x], [None, None]):
        b.refused((ValueError, AttributeError), k.ctpt_project, 0, 0, y, bad, w, G, None, None, None)
    b.refused(ValueError, k.ctpt_project, 0, 0, y, x, w, G, words[:5], None, None)
    b.refused(ValueError, k.ctpt_project, 0, 0, y, x, w, G, None, [None] * 2, None)
    b.refused(ValueError, k.ctpt_project, 0, 0, y, x, w, G, None, y, words[:3])
    b.refused(TypeError, k.ctpt_project, 0, 0, y, x, w, G, None)
    r = Tensor(1, 1, 4, 2, 2, N)
    b.refused(ValueError, k.rotary, 0, 0, r, Tensor(1, 1, 3, 2, 2, N), words, words, G, False)
    b.refused(ValueError, k.rotary, 0, 0, Tensor(1, 1, 3, 2, 2, N), Tensor(1, 1, 3, 2, 2, N), words, words, G, False)
    b.refused(ValueError, k.rotary, 0, 0, r, r, words[:4], words[:3], G, False)
    b.refused(ValueError, k.rotary, 0, 0, r, r, Tensor(1, 3, 2, N), Tensor(1, 2, 2, N), G, False)
    left, right, d = Tensor(1, 1, 2, 2, 2, N), Tensor(1, 2, 3, 2, 2, N), Tensor(1, 1, 3, 3, 2, N)
    b.refused(ValueError, k.ctct_gemm, 0, 0, d, right, left, G, None)
    b.refused(ValueError, k.ctct_gemm, 0, 0, Tensor(1, 1, 3, 2, 2, N), left, right, G, None)
    b.refused(ValueError, k.ctct_gemm, 0, 0, d, left, right, G, words[:5])
    b.refused(ValueError, k.ctct_gemm, 0, 0, d, left, right, G, Tensor(1, 1, 2, 2, N))
    b.refused(ValueError, k.ctct_gemm, 0, 0, d, [[Tensor(1, 2, 2, N)] * 2, [Tensor(1, 2, 2, N)]], right, G, None)
    b.refused(TypeError, k.ctct_gemm, 0, 0, d, [Tensor(1, 2, 2, N)] * 2, right, G, None)


def test_outputs_that_overlap_are_refused(b):
    """An expanded tensor as output has one polynomial in several places; inputs may."""
    k, w, x = b.k, Tensor(16, 4), Tensor(1, 3, 2, 2, N, stride=(0, 2 * N, N, 1))
    assert k.ctpt_project(0, 0, Tensor(1, 3, 2, 2, N), x, w, G, None, x, None) == 0
    b.refused(ValueError, k.ctpt_project, 0, 0, x, x, w, G, None, None, None)
    b.refused(ValueError, k.ctpt_project, 0, 0, Tensor(1, 3, 2, 2, N, stride=(4 * N, 0, N, 1)), x, w, G, None, None, None)
    words = np.zeros(4, dtype=np.uint32)
    y = Tensor(1, 2, 4, 2, 2, N, stride=(4 * N, 0, 2 * N, N, 1))
    b.refused(ValueError, k.rotary, 0, 0, y, Tensor(1, 2, 4, 2, 2, N), words, words, G, False)
    left, right = Tensor(1, 2, 2, 2, 2, N, stride=(0, 4 * N, 2 * N, N, 1)), Tensor(1, 2, 3, 2, 2, N)
    assert k.ctct_gemm(0, 0, Tensor(1, 2, 3, 3, 2, N), left, right, G, None) == 0
    b.refused(ValueError, k.ctct_gemm, 0, 0, Tensor(1, 2, 3, 3, 2, N, stride=(N, 6 * N, 2 * N, N, 1)), left, right, G, None)
    one = Tensor(1, 1, 3, 2, 2, N, stride=(0, 4 * N, 2 * N, N, 1))  # a single row's stride means nothing
    assert k.rotary(0, 0, Tensor(1, 1, 4, 2, 2, N, stride=(0, 4 * N, 2 * N, N, 1)), Tensor(1, 1, 4, 2, 2, N), words, words,
                    G, False) == 0
    b.refused(ValueError, k.ctct_gemm, 0, 0, one, left, right, G, None)


def test_packed_weights_of_another_device_are_refused(b):
    y, x = Tensor(1, 3, 2, 2, N), Tensor(1, 2, 2, 2, N)
    for device in (-1, 1):
        b.refused(ValueError, b.k.ctpt_project, 0, 0, y, x, Tensor(16, 4, device=device), G, None, None, None)
