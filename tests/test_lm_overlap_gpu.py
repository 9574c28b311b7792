"""Outputs of the language-model operators that overlap one another or an operand are
refused, in whatever way the call names them; what the header allows in place is not."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
G = [0, 10]


def residues(e, *lead):
    out = e.empty(*lead, len(G), e.n)
    for l, gi in enumerate(G):
        out[..., l, :] = e.torch.randint(0, int(e.primes[gi]), (*lead, e.n), dtype=e.torch.int32, device="cuda:0")
    return out


def test_outputs_that_overlap_are_refused(engine40, pkg):
    e = engine40
    P = len(G) * e.n  # words of a polynomial
    left, right = residues(e, 2, 3, 2), residues(e, 3, 2, 2)
    pool = e.empty(16, len(G), e.n)
    before = pool.zero_().clone()

    def refused(call, *args, **kw):
        with pytest.raises(pkg.CfheError, match="overlaps"):
            call(*args, **kw)
        e.synchronize()
        assert e.torch.equal(pool, before)

    strides = (3 * P, 3 * P, P, e.n, 1)  # leading strides of one result in both dimensions
    refused(e.ctct_gemm_, pool.as_strided((2, 2, 3, len(G), e.n), strides), left, right, G)
    d = pool[:12].view(4, 3, len(G), e.n)
    refused(e.ctct_gemm_, [[d[0], d[1]], [d[2], d[0]]], left, right, G)
    one = pool[0].expand(3, len(G), e.n)  # the three parts of a result in one place
    refused(e.ctct_gemm_, [[one, d[1]], [d[2], d[3]]], left, right, G)
    refused(e.ctct_gemm_, d[:1, None], pool[:6].view(1, 3, 2, len(G), e.n), right[:, :1], G)
    refused(e.ctct_gemm_, d[:1, None], left[:1], right[:, :1], G, decay=pool[2].view(1, 1, len(G), e.n))
    e.ctct_gemm_(d.view(2, 2, 3, len(G), e.n), left, right, G)
    assert int(d.abs().max()) > 0
    before = pool.zero_().clone()

    w = np.zeros((len(G), 3, 4), dtype=np.uint32)
    packed, x = e.gemm_pack_weights(w, G), residues(e, 3, 2)
    y = pool[:8].view(4, 2, len(G), e.n)
    refused(e.ctpt_project_, [y[0], y[1], y[2], y[1]], x, packed, G)
    refused(e.ctpt_project_, y, [x[0], x[1], y[3]], packed, G)
    refused(e.ctpt_project_, y, x, packed, G, residual=[None, y[2], None, None])  # another output than its own
    refused(e.ctpt_project_, y, x, packed, G, residual=pool[1:9].view(4, 2, len(G), e.n))
    e.ctpt_project_(y, [x[0], x[0], x[1]], packed, G, residual=y)  # its own, and inputs may repeat

    v = pool[:8].view(1, 4, 2, len(G), e.n)
    words = np.zeros((2, len(G)), dtype=np.uint32)
    wide = pool[:10].view(1, 5, 2, len(G), e.n)
    refused(e.rotary_, wide[:, :4], wide[:, 1:], words, words, G)
    refused(e.rotary_, [[v[0, 0], v[0, 1], v[0, 2], v[0, 0]]], residues(e, 1, 4, 2), words, words, G)
    refused(e.rotary_, v, residues(e, 1, 4, 2), pool[7:9], residues(e, 2), G)
    refused(e.rotary_, v, residues(e, 1, 4, 2), residues(e, 2), [pool[9], pool[0]], G)
    e.rotary_(v, v, words, words, G)  # in place
    e.synchronize()
