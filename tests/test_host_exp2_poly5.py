"""The degree-5 polynomial that the E4M3-cache kernels use for 2^f on the FMA
pipe (kv8_tc.cuh, KTC_C0..C5; f in [-0.5, 0.5]): the smallest largest relative
error that a polynomial of that degree reaches is found here again by the Remez
exchange, and the committed fp32 coefficients stay under 2^-22,
so that with the fp32 evaluation the exponential is within the 2^-21 that the
documentation of the results counts."""
import re
from pathlib import Path

import numpy as np

SRC = Path(__file__).resolve().parents[1] / "wam-egale_b200" / "csrc" / "kv8_tc.cuh"


def committed():
    text = SRC.read_text()
    return np.array([float(re.search(rf"KTC_C{i} = ([0-9.]+)f;", text).group(1)) for i in range(6)], dtype=np.float32)


def remez(d=5):
    x = np.sort(np.cos(np.pi * np.arange(d + 2) / (d + 1)) * 0.5)
    g = np.linspace(-0.5, 0.5, 200001)
    for _ in range(20):
        a = np.zeros((d + 2, d + 2))
        for i in range(d + 2):
            a[i, :d + 1] = x[i] ** np.arange(d + 1) / np.exp2(x[i])
            a[i, d + 1] = (-1) ** i
        c = np.linalg.solve(a, np.ones(d + 2))[:d + 1]
        e = np.polyval(c[::-1], g) / np.exp2(g) - 1
        ext = [0] + [i for i in range(1, len(g) - 1) if (e[i] - e[i - 1]) * (e[i + 1] - e[i]) <= 0] + [len(g) - 1]
        pts = []
        for i in ext:
            if not pts or np.sign(e[i]) != np.sign(e[pts[-1]]):
                pts.append(i)
            elif abs(e[i]) > abs(e[pts[-1]]):
                pts[-1] = i
        if len(pts) != d + 2:
            break
        x = g[pts]
    return c


def test_coefficients_are_the_remez_fit():
    assert np.allclose(committed(), remez().astype(np.float32), rtol=2e-5)


def test_error_in_fp32():
    c = committed()
    f = np.linspace(-0.5, 0.5, 400001).astype(np.float32)
    p = np.full_like(f, c[5])
    for k in range(4, -1, -1):                 # fused: one rounding a step
        p = (p.astype(np.float64) * f + np.float64(c[k])).astype(np.float32)
    assert np.abs(p / np.exp2(f.astype(np.float64)) - 1).max() < 2.0 ** -21
