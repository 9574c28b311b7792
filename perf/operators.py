"""Measured cases of the language-model operators on ciphertexts: a projection
with bias and residual, rotary positions, and the products of decayed linear
attention.

A ciphertext is a pair (b, a) of polynomials, a polynomial L limbs of N words, a
word a residue x * 2^32 mod q of its limb's prime q < 2^31; a product of words is
x * y * 2^-32 mod q. All results are residues: whole numbers, the same from
every way of computing them. Ciphertexts and encoded plaintexts are uniform
residues, which is what encryption and encoding make of any values.
"""
import functools
import importlib
import json
import math
import os

import torch

own = False

N = 1 << 16  # ring degree of every parameter set
LIMB = 4 * N
MAX_LEVEL = 11


def listed():
    return [
        # Feed-forward projection of the small encoder (hidden 32 to 64) on nearly
        # exhausted ciphertexts, bias only: launches count.
        {"name": "project_32x64_level1", "kind": "project", "params": "bootparam_40", "level": 1,
         "n_in": 32, "n_out": 64, "residual": False},
        # A projection whose sizes fill no tile, residual of another scale.
        {"name": "project_130x77_level5", "kind": "project", "params": "bootparam_35", "level": 5,
         "n_in": 130, "n_out": 77, "residual": True},
        # Output projection of an encrypted BERT-base layer with its residual.
        {"name": "project_768x768_level7", "kind": "project", "params": "bootparam_40", "level": 7,
         "n_in": 768, "n_out": 768, "residual": True},
        # One new token of one small head, nearly exhausted: all latency.
        {"name": "rotary_token_1x16_level1", "kind": "rotary", "params": "bootparam_40", "level": 1,
         "rows": 1, "dim": 16, "token": True, "halves": False},
        # Queries and keys of six heads of 64 features, all tokens of a prompt.
        {"name": "rotary_12x64_level8", "kind": "rotary", "params": "bootparam_40", "level": 8,
         "rows": 12, "dim": 64, "token": False, "halves": False},
        # A head with an odd number of pairs, first half against second half.
        {"name": "rotary_5x26_level4_30", "kind": "rotary", "params": "bootparam_30", "level": 4,
         "rows": 5, "dim": 26, "token": False, "halves": True},
        # Two new tokens against three kept ones, five features: small, latency.
        {"name": "attend_2x5x3_level2", "kind": "attend", "params": "bootparam_40", "level": 2,
         "m": 2, "k": 5, "n": 3, "decay": "token"},
        # Scores of one head over a prompt of 128 tokens: 8 giant steps of the queries
        # by 16 baby steps of the keys over 64 features, decay and causal mask per offset.
        {"name": "attend_8x64x16_level9", "kind": "attend", "params": "bootparam_40", "level": 9,
         "m": 8, "k": 64, "n": 16, "decay": "prompt"},
        # The weighted values of that head: 16 offsets summed into 64 features.
        {"name": "attend_8x16x64_level7", "kind": "attend", "params": "bootparam_40", "level": 7,
         "m": 8, "k": 16, "n": 64, "decay": "none"},
        # One new token against 60 kept keys of 64 features ...
        {"name": "attend_1x64x60_level4", "kind": "attend", "params": "bootparam_40", "level": 4,
         "m": 1, "k": 64, "n": 60, "decay": "token"},
        # ... and the weighted sum of as many kept values.
        {"name": "attend_1x60x64_level2", "kind": "attend", "params": "bootparam_40", "level": 2,
         "m": 1, "k": 60, "n": 64, "decay": "none"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    params = rng.choice(["bootparam_40", "bootparam_40", "bootparam_35", "bootparam_30"])
    kind = rng.choice(["project", "rotary", "attend", "attend"])
    case = {"kind": kind, "params": params, "level": rng.randint(1, MAX_LEVEL)}
    if kind == "project":
        case.update(n_in=_log_int(rng, 1, 768), n_out=_log_int(rng, 1, 768), residual=rng.random() < 0.6)
    elif kind == "rotary":
        case.update(rows=_log_int(rng, 1, 24), dim=2 * _log_int(rng, 1, 32), token=rng.random() < 0.4,
                    halves=rng.random() < 0.5)
    else:
        if rng.random() < 0.4:  # one token, kept keys or kept values
            m, k, n = 1, _log_int(rng, 1, 128), _log_int(rng, 1, 128)
        else:
            m, k, n = _log_int(rng, 1, 16), _log_int(rng, 1, 64), _log_int(rng, 1, 32)
        case.update(m=m, k=k, n=n, decay=rng.choice(["none", "prompt", "token"]))
    # no more than the largest listed case of its kind
    while _weight(case) > {"project": 768 * 768 * 11, "rotary": 12 * 64 * 13, "attend": 8 * 64 * 16 * 14}[kind]:
        case["level"] -= 1
        if case["level"] < 1:
            case["level"] = 1
            big = max(("n_in", "n_out") if kind == "project" else ("rows", "dim") if kind == "rotary" else ("m", "k", "n"),
                      key=lambda f: case[f])
            case[big] -= 2 if big == "dim" else 1
    return case


def _weight(case):
    limbs = len(_primes(case["params"], case["level"]))
    if case["kind"] == "project":
        return case["n_in"] * case["n_out"] * limbs
    if case["kind"] == "rotary":
        return case["rows"] * case["dim"] * limbs
    # products and ciphertexts held
    m, k, n = case["m"], case["k"], case["n"]
    return max(m * k * n, 5 * (m * k + k * n + 2 * m * n)) * limbs


@functools.lru_cache(maxsize=None)
def _file(params):
    with open(os.path.join("cheddar-fhe_b200", "parameters", params + ".json")) as f:
        return json.load(f)


def _primes(params, level):
    """The primes of a level's limbs: terminal primes from the end, then main primes."""
    p = _file(params)
    main, ter = p["level_config"][level]
    return list(reversed((p.get("terminal_primes") or [])[:ter])) + p["main_primes"][:main]


@functools.lru_cache(maxsize=None)
def _engine(params):
    """One context per parameter set for the life of the program."""
    pkg = importlib.import_module("cheddar-fhe_b200")
    return pkg.Engine(pkg.load_params(params + ".json"))


class _State:
    pass


def _residues(gen, primes, lead, tail=(N,)):
    out = torch.empty(*lead, len(primes), *tail, dtype=torch.int32, device="cuda")
    for l, q in enumerate(primes):
        out.select(len(lead), l).copy_(torch.randint(0, q, (*lead, *tail), dtype=torch.int32, device="cuda",
                                                     generator=gen))
    return out


def _host_words(t):
    return t.cpu().numpy().view("uint32")


def _inputs(case, seed):
    s = _State()
    s.kind = case["kind"]
    s.q = primes = _primes(case["params"], case["level"])
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if s.kind == "project":
        n_in, n_out = case["n_in"], case["n_out"]
        s.x = _residues(gen, primes, (n_in, 2))
        s.w = torch.stack([torch.randint(0, q, (n_in, n_out), dtype=torch.int32, device="cuda", generator=gen)
                           for q in primes])
        s.bias = _host_words(_residues(gen, primes, (), (n_out,)))
        s.res = _residues(gen, primes, (n_out, 2)) if case["residual"] else None
        s.res_scale = _host_words(_residues(gen, primes, (), (1,)))[:, 0].copy() if case["residual"] else None
    elif s.kind == "rotary":
        rows, dim = case["rows"], case["dim"]
        s.halves = case["halves"]
        s.x = _residues(gen, primes, (rows, dim, 2))
        if case["token"]:
            s.cos = _host_words(_residues(gen, primes, (dim // 2,), ()))
            s.sin = _host_words(_residues(gen, primes, (dim // 2,), ()))
        else:
            s.cos, s.sin = _residues(gen, primes, (dim // 2,)), _residues(gen, primes, (dim // 2,))
    else:
        m, k, n = case["m"], case["k"], case["n"]
        s.left, s.right = _residues(gen, primes, (m, k, 2)), _residues(gen, primes, (k, n, 2))
        s.decay = None
        if case["decay"] == "prompt":
            s.decay = _residues(gen, primes, (m, n))
        elif case["decay"] == "token":
            s.decay = _host_words(_residues(gen, primes, (m, n), ()))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    L = len(s.q)
    if s.kind == "project":
        s.out = torch.empty(case["n_out"], 2, L, N, dtype=torch.int32, device="cuda")
    elif s.kind == "rotary":
        s.out = torch.empty_like(s.x)
    else:
        s.out = torch.empty(case["m"], case["n"], 3, L, N, dtype=torch.int32, device="cuda")
    if own:
        s.eng = _engine(case["params"])
        s.g = s.eng.level_limbs(case["level"])
        if s.kind == "project":
            s.packed = s.eng.gemm_pack_weights(_host_words(s.w), s.g)
    return s


def run(s):
    if own:
        if s.kind == "project":
            s.eng.ctpt_project_(s.out, s.x, s.packed, s.g, bias=s.bias, residual=s.res, res_scale=s.res_scale)
        elif s.kind == "rotary":
            s.eng.rotary_(s.out, s.x, s.cos, s.sin, s.g, halves=s.halves)
        else:
            s.eng.ctct_gemm_(s.out, s.left, s.right, s.g, decay=s.decay)
        return s.out
    for l, q in enumerate(s.q):
        if s.kind == "project":
            _project(s, l, q)
        elif s.kind == "rotary":
            _rotary(s, l, q)
        else:
            _attend(s, l, q)
    return s.out


def _unscale(v, q):
    """v * 2^-32 mod q."""
    return v * pow(1 << 32, -1, q) % q


def _project(s, l, q):
    # exact products of 16-bit halves in float64: sums of up to 2^21 of them stay below 2^53
    w = s.w[l].t()
    wh, wl = (w >> 16).double(), (w & 0xffff).double()
    for p in range(2):
        x = s.x[:, p, l]
        xh, xl = (x >> 16).double(), (x & 0xffff).double()
        high = (wh @ xh).long() % q * ((1 << 32) % q) % q
        mid = (wh @ xl + wl @ xh).long() % q * (1 << 16) % q
        y = _unscale((high + mid + (wl @ xl).long()) % q, q)
        if s.res is not None:
            y += _unscale(s.res[:, p, l].long() * int(s.res_scale[l]) % q, q)
        if p == 0:
            y += torch.from_numpy(s.bias[l].astype("int64")).cuda()[:, None]
        s.out[:, p, l] = (y % q).int()


def _pairs(x, halves):
    pairs = x.shape[1] // 2
    return (x[:, :pairs], x[:, pairs:]) if halves else (x[:, 0::2], x[:, 1::2])


def _rotary(s, l, q):
    u, v = _pairs(s.x, s.halves)
    yu, yv = _pairs(s.out, s.halves)
    if isinstance(s.cos, torch.Tensor):
        c, d = s.cos[:, l].long(), s.sin[:, l].long()
    else:
        c, d = (torch.from_numpy(t[:, l].astype("int64")).cuda()[:, None] for t in (s.cos, s.sin))
    for r in range(s.x.shape[0]):
        for p in range(2):
            a, b = u[r, :, p, l].long(), v[r, :, p, l].long()
            yu[r, :, p, l] = _unscale((c * a + (q - d) * b) % q, q).int()
            yv[r, :, p, l] = _unscale((d * a + c * b) % q, q).int()


def _attend(s, l, q):
    m, k, n = s.left.shape[0], s.left.shape[1], s.right.shape[1]
    sums = [torch.zeros(m, n, N, dtype=torch.int64, device="cuda") for _ in range(3)]
    for t in range(k):
        lb, la = (s.left[:, t, p, l].long()[:, None] for p in range(2))
        rb, ra = (s.right[t, :, p, l].long()[None] for p in range(2))
        sums[0] += lb * rb % q
        sums[1] += (lb * ra + la * rb) % q
        sums[2] += la * ra % q
    for p in range(3):
        y = _unscale(sums[p] % q, q)
        if isinstance(s.decay, torch.Tensor):
            y = _unscale(y * s.decay[:, :, l] % q, q)
        elif s.decay is not None:
            y = _unscale(y * torch.from_numpy(s.decay[:, :, l].astype("int64")).cuda()[..., None] % q, q)
        s.out[:, :, p, l] = y.int()


# ---- the definition, by another way: balanced digits of 11 bits in float64,
# recombined with Horner's rule; sums of up to 2^30 of their products are exact
def _digits(x):
    x = x.double()
    out = []
    for _ in range(3):
        d = x - 2048.0 * torch.floor(x / 2048.0)
        out.append(d)
        x = (x - d) / 2048.0
    return out


def _sum_of_products(a, b, q, product):
    """product() of a and b mod q, a and b residues; product: a float64 contraction."""
    da, db = _digits(a), _digits(b)
    acc = None
    for power in range(4, -1, -1):
        part = sum(product(da[i], db[power - i]) for i in range(3) if 0 <= power - i < 3)
        part = part.to(torch.int64).remainder(q)
        acc = part if acc is None else (acc.mul(2048) + part).remainder(q)
    return acc


def exact(case, seed):
    s = _inputs(case, seed)
    outs = []
    for l, q in enumerate(s.q):
        shrink = pow(pow(2, 32, q), q - 2, q)  # 2^-32

        def times(u, v):
            return u.to(torch.int64).mul(v.to(torch.int64)).remainder(q).mul(shrink).remainder(q)

        def words(a, like):  # host words of this limb beside polynomials
            return torch.tensor(a.tolist(), dtype=torch.int64, device=like.device).unsqueeze(-1)

        if s.kind == "project":
            polys = []
            for p in range(2):
                y = _sum_of_products(s.w[l], s.x[:, p, l], q, lambda a, b: torch.einsum("kj,kc->jc", a, b))
                y = y.mul(shrink).remainder(q)
                if s.res is not None:
                    y = y + times(s.res[:, p, l], torch.full((1, 1), int(s.res_scale[l]), device="cuda"))
                if p == 0:
                    y = y + words(s.bias[l], y)
                polys.append(y.remainder(q).to(torch.int32))
            outs.append(torch.stack(polys, 1))
        elif s.kind == "rotary":
            x = s.x[:, :, :, l]
            pairs = x.shape[1] // 2
            x = x.unflatten(1, (2, pairs)) if s.halves else x.unflatten(1, (pairs, 2)).transpose(1, 2)
            if isinstance(s.cos, torch.Tensor):
                c, d = s.cos[:, l].unsqueeze(1), s.sin[:, l].unsqueeze(1)
            else:
                c, d = words(s.cos[:, l], x).unsqueeze(1), words(s.sin[:, l], x).unsqueeze(1)
            y = torch.empty_like(x)
            for r in range(x.shape[0]):
                u, v = x[r, 0], x[r, 1]
                y[r, 0] = (times(c, u) - times(d, v)).remainder(q).to(torch.int32)
                y[r, 1] = (times(c, v) + times(d, u)).remainder(q).to(torch.int32)
            outs.append((y if s.halves else y.transpose(1, 2)).reshape(s.x.shape[0], 2 * pairs, 2, N))
        else:
            out = torch.empty(s.left.shape[0], s.right.shape[1], 3, N, dtype=torch.int32, device="cuda")
            for c in range(0, N, 8192):  # one small matrix product per word position
                lb, la = (s.left[:, :, p, l, c:c + 8192].permute(2, 0, 1) for p in range(2))
                rb, ra = (s.right[:, :, p, l, c:c + 8192].permute(2, 0, 1) for p in range(2))
                d1 = _sum_of_products(lb, ra, q, torch.matmul) + _sum_of_products(la, rb, q, torch.matmul)
                parts = [_sum_of_products(lb, rb, q, torch.matmul), d1.remainder(q),
                         _sum_of_products(la, ra, q, torch.matmul)]
                for p, y in enumerate(parts):
                    y = y.mul(shrink).remainder(q).permute(1, 2, 0)
                    if isinstance(s.decay, torch.Tensor):
                        y = times(y, s.decay[:, :, l, c:c + 8192])
                    elif s.decay is not None:
                        y = times(y, words(s.decay[:, :, l], y))
                    out[:, :, p, c:c + 8192] = y.to(torch.int32)
            outs.append(out)
    return torch.stack(outs, -2)


def work(case):
    """Ciphertexts, plaintexts and results once each (weights as one word each); a
    word product with its sum is two operations; a product of two ciphertexts takes
    three word products."""
    L = len(_primes(case["params"], case["level"]))
    if case["kind"] == "project":
        n_in, n_out = case["n_in"], case["n_out"]
        limbs = 2 * (n_in + n_out * (2 if case["residual"] else 1))
        return {"bytes": limbs * L * LIMB + 4 * n_in * n_out * L, "flops": 4 * n_in * n_out * N * L}
    if case["kind"] == "rotary":
        polys = 2 * case["rows"] * case["dim"]
        limbs = 2 * polys + (0 if case["token"] else case["dim"])
        return {"bytes": limbs * L * LIMB, "flops": 4 * polys * N * L}
    m, k, n = case["m"], case["k"], case["n"]
    limbs = 2 * (m * k + k * n) + 3 * m * n + (m * n if case["decay"] == "prompt" else 0)
    return {"bytes": limbs * L * LIMB, "flops": 6 * m * k * n * N * L}
