"""Host words of the language-model operators' Python calls, without a GPU: words in
another order than the call reads them are refused, not read in the wrong order."""
import numpy as np

from test_lm_binding_cpu import G, N, Tensor, b  # noqa: F401  (b: the binding beside a stand-in of the library)


def words(*shape):
    return np.arange(int(np.prod(shape)), dtype=np.uint32).reshape(shape)


def test_words_of_a_projection(b):  # noqa: F811
    y, x, w = Tensor(0x1000, 3, 2, 2, N), Tensor(0x10, 2, 2, 2, N), Tensor(16, 4)
    for bias in (words(2, 3), words(6), words(2, 3, 1), words(3, 2).T, words(2, 3).tolist()):
        assert b.k.ctpt_project(0, 0, y, x, w, G, bias, None, None) == 0
        assert b.words(0, 6) == list(np.asarray(bias).reshape(-1))
    for bias in (words(3, 2), words(2, 3).T, words(3, 2).tolist(), words(3, 1, 2), words(6, 1, 1, 2)[:3]):
        b.refused(ValueError, b.k.ctpt_project, 0, 0, y, x, w, G, bias, None, None)
    for scale in (words(2), words(2, 1), words(1, 2)):
        assert b.k.ctpt_project(0, 0, y, x, w, G, None, y, scale) == 0
    b.refused(ValueError, b.k.ctpt_project, 0, 0, y, x, w, G, None, y, words(2, 2))


def test_words_of_rotary_positions(b):  # noqa: F811
    x = Tensor(0x1000, 1, 6, 2, 2, N)
    assert b.k.rotary(0, 0, x, x, words(3, 2), words(6), G, False) == 0
    assert b.k.rotary(0, 0, x, x, words(2, 3).T, words(3, 2), G, False) == 0
    assert b.words(0, 6) == [0, 3, 1, 4, 2, 5]
    b.refused(ValueError, b.k.rotary, 0, 0, x, x, words(2, 3), words(2, 3), G, False)
    b.refused(ValueError, b.k.rotary, 0, 0, x, x, words(3, 2), words(2, 3), G, False)


def test_words_of_a_product(b):  # noqa: F811
    left, right, d = Tensor(1, 3, 2, 2, 2, N), Tensor(1, 2, 4, 2, 2, N), Tensor(1, 3, 4, 3, 2, N)
    for decay in (words(3, 4, 2), words(24), words(4, 3, 2).transpose(1, 0, 2)):
        assert b.k.ctct_gemm(0, 0, d, left, right, G, decay) == 0
        assert b.words(0, 24) == list(decay.reshape(-1))
    for decay in (words(4, 3, 2), words(2, 3, 4), words(12, 2), words(3, 8)):
        b.refused(ValueError, b.k.ctct_gemm, 0, 0, d, left, right, G, decay)
    one = Tensor(1, 1, 4, 3, 2, N)  # one row: its dimension says nothing
    assert b.k.ctct_gemm(0, 0, one, Tensor(1, 1, 2, 2, 2, N), right, G, words(4, 2)) == 0
    b.refused(ValueError, b.k.ctct_gemm, 0, 0, one, Tensor(1, 1, 2, 2, 2, N), right, G, words(1, 2, 4))
