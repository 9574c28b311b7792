"""The float64 layer with decayed linear attention and rotary positions that checks
the encrypted one (oracle/decoder_plain.h) against NumPy, written another way:
positions as complex numbers, attention as masked matrix products and, token by
token, as a running state. Host only."""
import os
import struct
import subprocess
from math import erf

import numpy as np
import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


def turned(x, pairs, positions, base, halves):
    """x: [tokens, heads, dim]"""
    T, h, dim = x.shape
    z = x[..., :dim // 2] + 1j * x[..., dim // 2:] if halves else x[..., 0::2] + 1j * x[..., 1::2]
    angle = np.zeros((T, dim // 2))
    at = 0
    for n, pos in zip(pairs, positions):
        angle[:, at:at + n] = np.outer(pos, base ** (-np.arange(n) / n))
        at += n
    z = z * np.exp(1j * angle)[:, None]
    if halves:
        return np.concatenate([z.real, z.imag], axis=-1)
    return np.stack([z.real, z.imag], axis=-1).reshape(x.shape)


def layer(x, w, heads, decay, pairs, positions, base, halves, eps, recurrent):
    T, H = x.shape
    D = H // heads
    q, k, v = ((x @ w["w" + n] + w["b" + n]).reshape(T, heads, D) for n in "qkv")
    q, k = (turned(t, pairs, positions, base, halves) for t in (q, k))
    o = np.zeros((T, heads, D))
    age = np.subtract.outer(np.arange(T), np.arange(T))
    for h in range(heads):
        if recurrent:
            state = np.zeros((D, D))
            for t in range(T):
                state = decay[h] * state + np.outer(k[t, h], v[t, h])
                o[t, h] = q[t, h] @ state / np.sqrt(D)
        else:
            mask = np.where(age >= 0, decay[h] ** np.maximum(age, 0), 0.0)
            o[:, h] = (q[:, h] @ k[:, h].T / np.sqrt(D) * mask) @ v[:, h]

    def norm(y, g, b):
        y = y - y.mean(-1, keepdims=True)
        return y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * g + b

    h1 = norm(x + o.reshape(T, H) @ w["wo"] + w["bo"], w["gamma1"], w["beta1"])
    a = h1 @ w["w1"] + w["b1"]
    a = 0.5 * a * (1.0 + np.vectorize(erf)(a / np.sqrt(2.0)))
    return norm(h1 + a @ w["w2"] + w["b2"], w["gamma2"], w["beta2"])


@pytest.mark.parametrize("pairs,halves,T,recurrent", [
    ([8], False, 9, False), ([3, 2], True, 16, True), ([2, 3, 3], False, 12, True), ([], False, 1, False)])
def test_plain_decoder_matches_numpy(tmp_path, pairs, halves, T, recurrent):
    subprocess.check_call(["make", "-s", "-C", CPP, "plain_decoder"])
    rng = np.random.default_rng(7 + T)
    H, heads, F, eps, base = 32, 2, 64, 1e-5, 100.0
    decay = np.array([0.9, 1.0])
    positions = [rng.integers(0, 50, T).astype(float) for _ in pairs]
    shapes = [("wq", (H, H)), ("wk", (H, H)), ("wv", (H, H)), ("wo", (H, H)), ("w1", (H, F)), ("w2", (F, H)),
              ("bq", (H,)), ("bk", (H,)), ("bv", (H,)), ("bo", (H,)), ("b1", (F,)), ("b2", (H,)),
              ("gamma1", (H,)), ("beta1", (H,)), ("gamma2", (H,)), ("beta2", (H,))]
    w = {n: (1.0 if n.startswith("gamma") else 0.0) + 0.08 * rng.standard_normal(s) for n, s in shapes}
    x = rng.standard_normal((T, H))
    blob = struct.pack("<6i", T, H, heads, F, len(pairs), int(halves)) + struct.pack(f"<{len(pairs)}i", *pairs)
    blob += np.array([eps, base]).tobytes() + decay.tobytes()
    for p in positions:
        blob += p.tobytes()
    for n, _ in shapes:
        blob += np.ascontiguousarray(w[n]).tobytes()
    fin, fout = tmp_path / "in.bin", tmp_path / "out.bin"
    fin.write_bytes(blob + np.ascontiguousarray(x).tobytes())
    subprocess.check_call([os.path.join(CPP, "plain_decoder"), str(fin), str(fout)])
    got = np.frombuffer(fout.read_bytes(), dtype="<f8").reshape(T, H)
    want = layer(x, w, heads, decay, pairs, positions, base, halves, eps, recurrent)
    # sums of up to 64 products of order 1 in double precision, divided by a deviation
    # above 0.3: below 64 * 2^-52 / 0.3^2 * a few
    assert np.abs(got - want).max() < 1e-12
