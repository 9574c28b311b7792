"""The language-model operators on ciphertexts (cfhe_ctpt_project, cfhe_rotary,
cfhe_rotary_token, cfhe_ctct_gemm) against plain 64-bit integer arithmetic.
Every word is a residue, so every word has to be equal: there is no tolerance.
Parity unpinned by the reference, which has no such operators."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
PRIMES = [0, 10, 30, 52]  # a terminal prime, main primes on both sides of 2^30, an auxiliary prime


def draw(e, seed, g, *lead):
    """Uniform residues [*lead, limbs, N] with the extreme ones among them."""
    gen = e.torch.Generator(device="cuda:0").manual_seed(seed)
    out = e.empty(*lead, len(g), e.n)
    for l, gi in enumerate(g):
        q = int(e.primes[gi])
        w = e.torch.randint(0, q, (*lead, e.n), dtype=e.torch.int32, device="cuda:0", generator=gen)
        w[..., :4] = e.torch.tensor([q - 1, 0, 1, q - 1], dtype=e.torch.int32, device="cuda:0")
        out[..., l, :] = w
    return out


def host(t):
    return t.cpu().numpy().view(np.uint32)


def mul(a, b, q):
    """a b 2^-32 mod q for int64 tensors of residues or integers."""
    return a * b % q * pow(1 << 32, -1, q) % q


def constants(e, seed, g, *lead):
    rng = np.random.default_rng(seed)
    k = np.stack([rng.integers(0, int(e.primes[gi]), lead, dtype=np.uint32) for gi in g], axis=-1)
    k.reshape(-1, len(g))[0] = [int(e.primes[gi]) - 1 for gi in g]
    return np.ascontiguousarray(k)


# ---- projection ------------------------------------------------------------
def want_project(e, x, w, g, l, j, bias, residual, scale):
    q = int(e.primes[g[l]])
    out = []
    for p in range(2):
        acc = e.torch.zeros(e.n, dtype=e.torch.int64, device="cuda:0")
        for k in range(len(x)):
            acc += x[k][p, l].long() * int(w[l, k, j]) % q
        y = acc % q * pow(1 << 32, -1, q) % q
        if residual is not None and residual[j] is not None:
            s = int(scale[l]) if scale is not None else (1 << 32) % q
            y += mul(residual[j][p, l].long(), s, q)
        if p == 0 and bias is not None:
            y += int(bias[l, j])
        out.append((y % q).int())
    return e.torch.stack(out)


@pytest.mark.parametrize("n_in,n_out,bias,residual,scaled", [
    (1, 1, True, True, True), (5, 3, False, False, False), (16, 64, True, False, False),
    (33, 129, True, True, False), (130, 77, False, True, True), (40, 65, True, True, True),
    (272, 200, True, True, True), (515, 8, True, True, True)])
def test_project(engine40, n_in, n_out, bias, residual, scaled):
    e, g = engine40, PRIMES
    x = draw(e, 1 + n_in, g, n_in, 2)
    w = np.ascontiguousarray(np.moveaxis(constants(e, 2 + n_in, g, n_in, n_out), -1, 0))
    b = np.ascontiguousarray(constants(e, 3, g, n_out).T) if bias else None
    r = draw(e, 4, g, n_out, 2) if residual else None
    s = constants(e, 5, g) if scaled else None
    y = e.empty(n_out, 2, len(g), e.n).fill_(-1)
    e.ctpt_project_(y, x, e.gemm_pack_weights(w, g), g, bias=b, residual=r, res_scale=s)
    for j in sorted({0, n_out - 1, n_out // 2, min(63, n_out - 1), min(64, n_out - 1)}):
        for l in range(len(g)):
            assert e.torch.equal(y[j, :, l], want_project(e, x, w, g, l, j, b, r, s)), (j, l)


def test_project_equals_its_parts(engine40):
    """Every word of the product, then of the multiplication, sums and bias as single calls."""
    e = engine40
    g = list(e.level_limbs(4))
    n_in, n_out = 21, 150
    x, r = draw(e, 10, g, n_in, 2), draw(e, 11, g, n_out, 2)
    w = np.ascontiguousarray(np.moveaxis(constants(e, 12, g, n_in, n_out), -1, 0))
    b, s = np.ascontiguousarray(constants(e, 13, g, n_out).T), constants(e, 14, g)
    packed = e.gemm_pack_weights(w, g)
    y = e.empty(n_out, 2, len(g), e.n)
    e.ctpt_project_(y, x, packed, g, bias=b, residual=r, res_scale=s)
    z = e.torch.empty_like(y)
    for p in range(2):
        e.ctpt_gemm_([z[j, p] for j in range(n_out)], [x[k, p] for k in range(n_in)], packed, g)
        for j in range(n_out):
            e.const_op_(4, z[j, p], r[j, p], z[j, p], s, g)
            if p == 0:
                e.const_op_(0, z[j, p], z[j, p], None, np.ascontiguousarray(b[:, j]), g)
    e.synchronize()
    assert e.torch.equal(y, z)


def test_project_lists_missing_residuals_and_in_place(engine40):
    e, g = engine40, PRIMES
    n_in, n_out = 7, 70
    x = [draw(e, 20 + k, g, 2) for k in range(n_in)]
    w = np.ascontiguousarray(np.moveaxis(constants(e, 21, g, n_in, n_out), -1, 0))
    packed = e.gemm_pack_weights(w, g)
    r = draw(e, 22, g, n_out, 2)
    some = [r[j] if j % 3 else None for j in range(n_out)]
    y = e.empty(n_out, 2, len(g), e.n)
    e.ctpt_project_([y[j] for j in range(n_out)], x, packed, g, residual=some)
    for j in (0, 1, 3, 68, 69):
        assert e.torch.equal(y[j, :, 2], want_project(e, x, w, g, 2, j, None, some, None)), j
    z = r.clone()
    e.ctpt_project_(z, x, packed, g, residual=z)  # the residual is its own output
    for j in (0, 63, 64, 69):
        assert e.torch.equal(z[j, :, 3], want_project(e, x, w, g, 3, j, None, r, None)), j


# ---- rotary positions --------------------------------------------------------
def want_rotary(e, x, cos, sin, g, halves):
    pairs = x.shape[1] // 2
    pick = (lambda t: (t[:, :pairs], t[:, pairs:])) if halves else (lambda t: (t[:, 0::2], t[:, 1::2]))
    y = e.torch.empty_like(x)
    (u, v), (yu, yv) = pick(x), pick(y)
    for l, gi in enumerate(g):
        q = int(e.primes[gi])
        if isinstance(cos, np.ndarray):
            c, s = (e.torch.from_numpy(t[:, l].astype(np.int64)).cuda()[:, None, None] for t in (cos, sin))
        else:
            c, s = cos[:, None, l].long(), sin[:, None, l].long()
        a, b = u[:, :, :, l].long(), v[:, :, :, l].long()
        yu[:, :, :, l] = ((mul(c, a, q) - mul(s, b, q)) % q).int()
        yv[:, :, :, l] = ((mul(s, a, q) + mul(c, b, q)) % q).int()
    return y


@pytest.mark.parametrize("rows,dim,token,halves", [
    (1, 2, False, False), (1, 2, True, True), (3, 10, False, True), (3, 10, True, False), (5, 26, False, False),
    (16, 64, False, False), (1, 256, True, False), (140, 8, False, True), (300, 2, True, False)])
def test_rotary(engine40, rows, dim, token, halves):
    """From one pair to tables that take several launches (512 pairs x rows, 512 constants)."""
    e, g = engine40, PRIMES[:3]
    x = draw(e, 30 + rows, g, rows, dim, 2)
    if token:
        cos, sin = constants(e, 31, g, dim // 2), constants(e, 32, g, dim // 2)
        sin[0] = 0
    else:
        cos, sin = draw(e, 31, g, dim // 2), draw(e, 32, g, dim // 2)
    want = want_rotary(e, x, cos, sin, g, halves)
    y = e.torch.empty_like(x)
    e.rotary_(y, x, cos, sin, g, halves=halves)
    assert e.torch.equal(y, want)
    e.rotary_(x, x, cos, sin, g, halves=halves)  # in place
    assert e.torch.equal(x, want)


def test_rotary_strides(engine40):
    """Features before rows in memory, every second ciphertext, limbs of a larger ciphertext."""
    e, g = engine40, PRIMES[:2]
    full = draw(e, 40, g, 12, 6, 2)
    x = full.transpose(0, 1)[:, ::2]
    cos, sin = draw(e, 41, g, 3), draw(e, 42, g, 3)
    y = e.empty(6, 6, 2, 2, e.n)
    e.rotary_(y, x, cos, sin, g)
    assert e.torch.equal(y, want_rotary(e, x, cos, sin, g, False))
    wide = draw(e, 43, PRIMES, 2, 2, 2)  # the first two limbs of four
    y = e.empty(2, 2, 2, 2, e.n)
    e.rotary_(y, wide[..., :2, :], cos[:1], sin[:1], g)
    assert e.torch.equal(y, want_rotary(e, wide[..., :2, :], cos[:1], sin[:1], g, False))


# ---- products of ciphertexts ---------------------------------------------------
def want_ctct(e, left, right, g, decay):
    m, k, n = left.shape[0], left.shape[1], right.shape[1]
    d = e.empty(m, n, 3, len(g), e.n)
    for l, gi in enumerate(g):
        q = int(e.primes[gi])
        sums = [e.torch.zeros(m, n, e.n, dtype=e.torch.int64, device="cuda:0") for _ in range(3)]
        for t in range(k):
            lb, la = left[:, t, 0, l].long()[:, None], left[:, t, 1, l].long()[:, None]
            rb, ra = right[t, :, 0, l].long()[None], right[t, :, 1, l].long()[None]
            sums[0] += lb * rb % q
            sums[1] += lb * ra % q + la * rb % q
            sums[2] += la * ra % q
        for p in range(3):
            y = sums[p] % q * pow(1 << 32, -1, q) % q
            if isinstance(decay, np.ndarray):
                y = mul(y, e.torch.from_numpy(decay[:, :, l].astype(np.int64)).cuda()[..., None], q)
            elif decay is not None:
                y = mul(y, decay[:, :, l].long(), q)
            d[:, :, p, l] = y.int()
    return d


SHAPES = [(1, 1, 1), (1, 7, 5), (2, 5, 3), (3, 5, 7), (4, 16, 4), (8, 64, 16), (8, 16, 33), (5, 33, 9), (17, 3, 2),
          (1, 130, 17), (1, 3, 70), (9, 1, 13), (2, 2, 130), (16, 9, 1)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("decay", ["none", "prompt", "token"])
def test_ctct_gemm(engine40, m, k, n, decay):
    e, g = engine40, PRIMES[:2]
    left, right = draw(e, 50 + m, g, m, k, 2), draw(e, 60 + n, g, k, n, 2)
    w = {"none": None, "prompt": draw(e, 70, g, m, n), "token": constants(e, 71, g, m, n)}[decay]
    if decay == "token":
        w[-1, -1] = 0  # a masked place
    if decay == "prompt":
        w[0, 0] = 0
    d = e.empty(m, n, 3, len(g), e.n).fill_(-1)
    e.ctct_gemm_(d, left, right, g, decay=w)
    assert e.torch.equal(d, want_ctct(e, left, right, g, w))


def test_ctct_gemm_largest_residues(engine40):
    """Sums of the largest products: every word q - 1, for lengths around every place
    where a sum is brought back below its bound."""
    e, g = engine40, PRIMES
    for k in list(range(1, 20)) + [31, 32, 33, 100]:
        left, right = e.empty(4, k, 2, len(g), e.n), e.empty(k, 4, 2, len(g), e.n)
        for l, gi in enumerate(g):
            left[..., l, :] = int(e.primes[gi]) - 1
            right[..., l, :] = int(e.primes[gi]) - 1
            right[..., l, 1::2] = 1
        d = e.empty(4, 4, 3, len(g), e.n)
        e.ctct_gemm_(d, left, right, g)
        for l, gi in enumerate(g):
            q = int(e.primes[gi])
            inv = pow(1 << 32, -1, q)
            even, odd = k * inv % q, -k * inv % q
            for p, f in enumerate((1, 2, 1)):
                assert e.torch.all(d[:, :, p, l, 0::2] == f * even % q), (k, l, p)
                assert e.torch.all(d[:, :, p, l, 1::2] == f * odd % q), (k, l, p)


def primes_below(bound, count):
    """Primes of the ring (1 mod 2^17) below `bound`, largest first."""
    out, q = [], (bound - 2) // (1 << 17) * (1 << 17) + 1
    while len(out) < count:
        if all(pow(a, q - 1, q) == 1 for a in (2, 3, 5, 7)) and all(q % d for d in range(3, 1 << 16, 2)):
            out.append(q)
        q -= 1 << 17
    return out


@pytest.mark.parametrize("bound", [1270000000, 1 << 31])
def test_operators_at_the_largest_primes(pkg, bound):
    """Primes of the shipped size and the largest there are: largest words, then random
    ones, in every kernel."""
    main = primes_below(bound, 4)
    aux = primes_below(1 << 29, 2)
    e = pkg.Engine({"log_degree": 16, "main_primes": main, "terminal_primes": [], "auxiliary_primes": aux,
                    "level_config": [[1, 0], [2, 0], [3, 0], [4, 0]], "additional_base": [0, 0]})
    g = [0, 1]
    q0 = int(e.primes[0])
    assert bound - q0 < 1 << 24
    for m, n in ((1, 3), (1, 20), (2, 7), (2, 33), (3, 5), (4, 17), (8, 9), (9, 6)):
        for k in (1, 2, 7, 8, 9, 16, 17, 33):
            left, right = e.empty(m, k, 2, 2, e.n), e.empty(k, n, 2, 2, e.n)
            for l in range(2):
                left[..., l, :] = int(e.primes[l]) - 1
                right[..., l, :] = int(e.primes[l]) - 1
            d = e.empty(m, n, 3, 2, e.n)
            e.ctct_gemm_(d, left, right, g)
            for l in range(2):
                q = int(e.primes[l])
                for p, f in enumerate((1, 2, 1)):
                    assert e.torch.all(d[:, :, p, l] == f * k * pow(1 << 32, -1, q) % q), (m, n, k, l, p)
        left, right = draw(e, m, g, m, 19, 2), draw(e, n, g, 19, n, 2)
        w = constants(e, 3, g, m, n)
        d = e.empty(m, n, 3, 2, e.n)
        e.ctct_gemm_(d, left, right, g, decay=w)
        assert e.torch.equal(d, want_ctct(e, left, right, g, w)), (m, n)
    x = draw(e, 1, g, 2, 6, 2)
    cos, sin = draw(e, 2, g, 3), draw(e, 3, g, 3)
    y = e.torch.empty_like(x)
    e.rotary_(y, x, cos, sin, g)
    assert e.torch.equal(y, want_rotary(e, x, cos, sin, g, False))
    w = np.ascontiguousarray(np.moveaxis(constants(e, 4, g, 6, 5), -1, 0))
    w[:, 1:] = (np.array([int(e.primes[l]) - 1 for l in g], dtype=np.uint32))[:, None, None]
    b, s = np.ascontiguousarray(constants(e, 5, g, 5).T), constants(e, 6, g)
    r = draw(e, 7, g, 5, 2)
    y = e.empty(5, 2, 2, e.n)
    e.ctpt_project_(y, x[0], e.gemm_pack_weights(w, g), g, bias=b, residual=r, res_scale=s)
    for j in range(5):
        for l in range(2):
            assert e.torch.equal(y[j, :, l], want_project(e, x[0], w, g, l, j, b, r, s)), (j, l)
    e.close()


@pytest.mark.parametrize("m,n", [(1, 3), (1, 10), (2, 5), (2, 9), (4, 4), (3, 11), (6, 7)])
def test_ctct_gemm_long_sums(pkg, m, n):
    """More terms than a sum takes before it is brought back below its bound, at the
    largest primes: one ciphertext in all places of a matrix, so that a result is k
    times their product."""
    bound = 1 << 31
    e = pkg.Engine({"log_degree": 16, "main_primes": primes_below(bound, 2), "terminal_primes": [],
                    "auxiliary_primes": primes_below(1 << 29, 2), "level_config": [[1, 0], [2, 0]],
                    "additional_base": [0, 0]})
    g = [0, 1]
    x, y = draw(e, 220, g, 1, 1, 2), draw(e, 221, g, 1, 1, 2)
    for l in range(2):
        x[..., l, :128] = int(e.primes[l]) - 1
        y[..., l, :128] = int(e.primes[l]) - 1
    one = want_ctct(e, x, y, g, None).long()
    for k in (255, 256, 257, 511, 513, 1030):
        d = e.empty(m, n, 3, 2, e.n).fill_(-1)
        e.ctct_gemm_(d, x.expand(m, k, 2, 2, e.n), y.expand(k, n, 2, 2, e.n), g)
        for l in range(2):
            want = one[:, :, :, l] * k % int(e.primes[l])
            assert e.torch.equal(d[:, :, :, l].long(), want.expand(m, n, 3, e.n)), (k, l)
    e.close()


def test_ctct_gemm_equals_tensor_accum(engine40):
    e = engine40
    g = list(e.level_limbs(3))
    m, k, n = 3, 6, 5
    left, right = draw(e, 80, g, m, k, 2), draw(e, 81, g, k, n, 2)
    d, r = e.empty(m, n, 3, len(g), e.n), e.empty(3, len(g), e.n)
    e.ctct_gemm_(d, left, right, g)
    for i in range(m):
        for j in range(n):
            e.tensor_accum_(r[0], r[1], r[2], [left[i, t, 0] for t in range(k)], [left[i, t, 1] for t in range(k)],
                            [right[t, j, 0] for t in range(k)], [right[t, j, 1] for t in range(k)], g)
            e.synchronize()
            assert e.torch.equal(d[i, j], r), (i, j)


def test_ctct_gemm_strides_and_lists(engine40):
    """Kept keys [token][feature] read as [feature][token]; the same as nested lists."""
    e, g = engine40, PRIMES[:2]
    kept = draw(e, 90, g, 9, 4, 2)  # tokens, features
    q = draw(e, 91, g, 1, 4, 2)
    w = constants(e, 92, g, 1, 9)
    d = e.empty(1, 9, 3, len(g), e.n)
    e.ctct_gemm_(d, q, kept.transpose(0, 1), g, decay=w)
    want = want_ctct(e, q, kept.transpose(0, 1), g, w)
    assert e.torch.equal(d, want)
    d.fill_(0)
    e.ctct_gemm_([[d[0, j] for j in range(9)]], [[q[0, t] for t in range(4)]],
                 [[kept[j, t] for j in range(9)] for t in range(4)], g, decay=w)
    assert e.torch.equal(d, want)


# ---- refusals ------------------------------------------------------------------
def test_refusals(engine40, pkg):
    e, g = engine40, [0, 1]
    ct = draw(e, 100, g, 4, 2)
    y = e.torch.empty_like(ct)
    packed = e.gemm_pack_weights(np.zeros((2, 4, 4), dtype=np.uint32), g)
    words = np.zeros((2, 2), dtype=np.uint32)
    with pytest.raises(pkg.CfheError, match="prime index"):
        e.ctpt_project_(y, ct, packed, [0, 999])
    with pytest.raises(pkg.CfheError, match="residual scale"):
        e.ctpt_project_(y, ct, packed, g, res_scale=np.zeros(2, dtype=np.uint32))
    with pytest.raises(ValueError, match="smaller matrix"):
        e.ctpt_project_(draw(e, 1, g, 70, 2), ct, packed, g)
    with pytest.raises(ValueError, match="constants"):
        e.ctpt_project_(y, ct, packed, g, bias=words)
    with pytest.raises(ValueError, match="per output"):
        e.ctpt_project_(y, ct, packed, g, residual=ct[:2])
    with pytest.raises(ValueError, match="device"):
        e.ctpt_project_(y, ct.cpu(), packed, g)
    with pytest.raises(ValueError, match="32-bit"):
        e.ctpt_project_(y, ct.long(), packed, g)
    with pytest.raises(ValueError, match="limbs"):
        e.ctpt_project_(y, ct, packed, [0])
    x = ct[None].clone()
    with pytest.raises(pkg.CfheError, match="prime index"):
        e.rotary_(x, x, words, words, [-1, 0])
    with pytest.raises(ValueError, match="even number"):
        e.rotary_(x[:, :3], x[:, :3], words, words, g)
    with pytest.raises(ValueError, match="cosine"):
        e.rotary_(x, x, ct[:1, 0], ct[:1, 1], g)
    with pytest.raises(ValueError, match="constants"):
        e.rotary_(x, x, words[:1], words[:1], g)
    odd = e.empty(2 * 2 * 2 * e.n + 1)[1:].view(1, 2, 2, 2, e.n)
    with pytest.raises(pkg.CfheError, match="16-byte"):
        e.rotary_(odd, odd, words[:1], words[:1], g)
    d = e.empty(1, 4, 3, 2, e.n)
    with pytest.raises(ValueError, match="do not fit"):
        e.ctct_gemm_(d, x, x, g)
    with pytest.raises(ValueError, match="constants"):
        e.ctct_gemm_(d, x[:, :1], x, g, decay=words)
    with pytest.raises(pkg.CfheError, match="prime index"):
        e.ctct_gemm_(d, x[:, :1], x, [0, 999])
    with pytest.raises(ValueError, match="one after the other"):
        e.ctct_gemm_(d, x[:, :1].transpose(-1, -2).contiguous().transpose(-1, -2), x, g)
    e.synchronize()


# ---- streams and graphs ----------------------------------------------------------
def test_captured_and_replayed(pkg, params40):
    """The three calls captured into one graph; a replay reads the buffers' new contents."""
    e = pkg.Engine(params40)
    torch, g = e.torch, PRIMES[:2]
    x = draw(e, 110, g, 1, 4, 2)
    w = np.ascontiguousarray(np.moveaxis(constants(e, 111, g, 4, 4), -1, 0))
    packed = e.gemm_pack_weights(w, g)
    bias = np.ascontiguousarray(constants(e, 112, g, 4).T)
    cos, sin = constants(e, 113, g, 2), constants(e, 114, g, 2)
    decay = constants(e, 115, g, 1, 1)
    p, r = e.empty(1, 4, 2, 2, e.n), e.empty(1, 4, 2, 2, e.n)
    d = e.empty(1, 1, 3, 2, e.n)

    def calls():
        e.ctpt_project_(p[0], x[0], packed, g, bias=bias, residual=x[0])
        e.rotary_(r, p, cos, sin, g)
        e.ctct_gemm_(d, r, x.transpose(0, 1), g, decay=decay)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        e.use_torch_stream()
        calls()  # the workspace exists from here on
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            calls()
        for seed in (120, 121):
            x.copy_(draw(e, seed, g, 1, 4, 2))
            d.zero_()
            graph.replay()
            stream.synchronize()
            got = d.clone()
            d.zero_()
            calls()
            stream.synchronize()
            assert torch.equal(got, d) and int(d.abs().max()) > 0
    del graph
    e.close()


def test_graphs_share_no_memory(pkg, params40):
    """Two graphs captured from one fresh context, the second one's calls larger; an
    eager call that needs more than either (and regrows the workspace) between the
    captures and the replays; replays of both at once on two streams."""
    e = pkg.Engine(params40)
    torch, g = e.torch, PRIMES[:2]
    streams = [torch.cuda.Stream() for _ in range(3)]
    jobs = []
    for i, (m, k, n) in enumerate([(1, 5, 3), (3, 9, 40)]):
        left, right = draw(e, 160 + i, g, m, k, 2), draw(e, 170 + i, g, k, n, 2)
        x, w = draw(e, 180 + i, g, 3 + i, 2), constants(e, 190 + i, g, 3 + i, 4)
        packed = e.gemm_pack_weights(np.ascontiguousarray(np.moveaxis(w, -1, 0)), g)
        jobs.append((left, right, constants(e, 200 + i, g, m, n), e.empty(m, n, 3, 2, e.n), x, packed,
                     np.moveaxis(w, -1, 0), e.empty(4, 2, 2, e.n)))
    torch.cuda.synchronize()
    graphs = []
    with torch.cuda.stream(streams[2]):
        e.use_torch_stream()
        for left, right, c, d, x, packed, w, y in jobs:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=streams[2]):
                e.ctct_gemm_(d, left, right, g, decay=c)
                e.ctpt_project_(y, x, packed, g, residual=[x[0], x[1], x[2], x[0]])
            graphs.append(graph)
        big = draw(e, 210, g, 260, 2)
        wide = np.zeros((2, 260, 200), dtype=np.uint32)
        e.ctpt_project_(e.empty(200, 2, 2, e.n), big, e.gemm_pack_weights(wide, g), g)
        e.synchronize()
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for left, right, c, d, x, packed, w, y in jobs:
        assert torch.equal(d, want_ctct(e, left, right, g, c))
        for j in range(4):
            want = want_project(e, x, w, g, 1, j, None, [x[0], x[1], x[2], x[0]], None)
            assert torch.equal(y[j, :, 1], want), j
    del graphs
    e.close()


def test_two_engines_on_two_streams(pkg, params40):
    """Calls of two contexts at once, each with its own tables and workspace."""
    import torch
    g = PRIMES[:2]
    jobs = []
    for k in range(2):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            e = pkg.Engine(params40)
            left, right = draw(e, 130 + k, g, 2, 9 + k, 2), draw(e, 140 + k, g, 9 + k, 5, 2)
            jobs.append((e, stream, left, right, e.empty(2, 5, 3, 2, e.n), constants(e, 150 + k, g, 2, 5)))
    torch.cuda.synchronize()
    for _ in range(5):
        for e, stream, left, right, d, w in jobs:
            e.ctct_gemm_(d, left, right, g, decay=w)
    torch.cuda.synchronize()
    for e, stream, left, right, d, w in jobs:
        assert torch.equal(d, want_ctct(e, left, right, g, w))
        e.close()
