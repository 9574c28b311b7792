"""Variants of the language-model operators' kernels where they are delicate, against
plain 64-bit integer arithmetic: every word has to be equal. Parity unpinned by the
reference, which has no such operators."""
import numpy as np
import pytest

from test_lm_ops_gpu import constants, draw, primes_below, want_ctct, want_project

pytestmark = pytest.mark.gpu


def engine_at(pkg, bound):
    return pkg.Engine({"log_degree": 16, "main_primes": primes_below(bound, 2), "terminal_primes": [],
                       "auxiliary_primes": primes_below(1 << 29, 2), "level_config": [[1, 0], [2, 0]],
                       "additional_base": [0, 0]})


@pytest.mark.parametrize("bound", [1270000000, 1 << 31])
@pytest.mark.parametrize("m,n", [(2, 3), (2, 4), (4, 2), (3, 4), (1, 2)])
def test_narrow_products_at_the_largest_primes(pkg, bound, m, n):
    """No more than four results along the longer side: sums of the largest words around
    every stage's end, then more terms than a sum takes before it is brought back."""
    e, g = engine_at(pkg, bound), [0, 1]
    x, y = draw(e, 300, g, 1, 1, 2), draw(e, 301, g, 1, 1, 2)
    for l in range(2):
        x[..., l, :128] = int(e.primes[l]) - 1
        y[..., l, :128] = int(e.primes[l]) - 1
    one = want_ctct(e, x, y, g, None).long()
    for k in (1, 2, 3, 4, 5, 7, 8, 9, 16, 33, 255, 256, 257, 511, 513, 1030):
        d = e.empty(m, n, 3, 2, e.n).fill_(-1)
        e.ctct_gemm_(d, x.expand(m, k, 2, 2, e.n), y.expand(k, n, 2, 2, e.n), g)
        for l in range(2):
            want = one[:, :, :, l] * k % int(e.primes[l])
            assert e.torch.equal(d[:, :, :, l].long(), want.expand(m, n, 3, e.n)), (k, l)
    left, right = draw(e, 302, g, m, 261, 2), draw(e, 303, g, 261, n, 2)
    for w in (None, constants(e, 304, g, m, n), draw(e, 305, g, m, n)):
        d = e.empty(m, n, 3, 2, e.n).fill_(-1)
        e.ctct_gemm_(d, left, right, g, decay=w)
        assert e.torch.equal(d, want_ctct(e, left, right, g, w))
    e.close()


@pytest.mark.parametrize("n_in,n_out,limbs", [(60, 5, 4), (60, 70, 4), (16, 3, 9), (5, 65, 9), (100, 33, 5), (1, 1, 1)])
def test_projection_groups_that_do_not_divide(engine40, n_in, n_out, limbs):
    """Limbs and polynomials of a call in groups whose last is smaller (6 + 2, 16 + 2, 3 of
    4 and so on), bias and residual on all of them."""
    e = engine40
    g = [0, 10, 30, 52, 1, 20, 11, 31, 53][:limbs]
    x, r = draw(e, 310 + n_in, g, n_in, 2), draw(e, 311, g, n_out, 2)
    w = np.ascontiguousarray(np.moveaxis(constants(e, 312, g, n_in, n_out), -1, 0))
    b, s = np.ascontiguousarray(constants(e, 313, g, n_out).T), constants(e, 314, g)
    y = e.empty(n_out, 2, len(g), e.n).fill_(-1)
    e.ctpt_project_(y, x, e.gemm_pack_weights(w, g), g, bias=b, residual=r, res_scale=s)
    for j in range(n_out):
        for l in range(len(g)):
            assert e.torch.equal(y[j, :, l], want_project(e, x, w, g, l, j, b, r, s)), (j, l)
