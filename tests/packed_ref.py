"""Plain 64-bit forms of the operators on packed weights, and the bounds of
their rounding errors (test infrastructure)."""

from __future__ import annotations

import numpy as np

from dequant import BLOCK, dequantize

U = 2.0 ** -24          # half an ulp of f32, relative
BYTES = {"q4_0": 18, "q4_1": 20, "q5_0": 22, "q5_1": 24, "q8_0": 34, "iq4_nl": 18, "q2_k": 84, "q3_k": 110,
         "q4_k": 144, "q5_k": 176, "q6_k": 210, "iq4_xs": 136, "iq2_xxs": 66, "iq2_xs": 74, "iq2_s": 82,
         "iq3_xxs": 98, "iq3_s": 110}
# byte ranges of the f16 fields of a block, and of the codes (formats with a minimum)
HALVES = {"q4_1": (0, 2), "q5_1": (0, 2), "q2_k": (80, 82), "q3_k": (108,), "q4_k": (0, 2), "q5_k": (0, 2),
          "q6_k": (208,)}
CODES = {"q4_1": (4, 20), "q5_1": (4, 24), "q2_k": (16, 80), "q4_k": (16, 144), "q5_k": (16, 176)}
ROUND = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}    # of a result stored in that type


def random_packed(qtype: str, n: int, k: int, seed: int) -> np.ndarray:
    """(n, row bytes): every code, sign and index bit random, the f16 scales
    around 0.001 (and both signs of Q3_K's and the symmetric types')."""
    rng = np.random.default_rng(seed)
    nb = n * (k // BLOCK[qtype])
    b = rng.integers(0, 256, (nb, BYTES[qtype]), dtype=np.uint8)
    for i, at in enumerate(HALVES.get(qtype, (0,))):
        d = np.exp(rng.normal(-7.0, 0.5, nb)) * (1.0 if i else np.where(rng.random(nb) < 0.1, -1, 1))
        b[:, at:at + 2] = d.astype(np.float16)[:, None].view(np.uint8)
    return b.reshape(n, -1)


def weight64(qtype: str, packed: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(values, |d c| + |m| of each value) of a packed weight: w = d c - m is
    evaluated with roundings of its two parts, not of their difference."""
    w = dequantize(qtype, packed, packed.shape[0])
    if qtype not in CODES:
        return w, np.abs(w)
    z = packed.reshape(-1, BYTES[qtype]).copy()
    z[:, slice(*CODES[qtype])] = 0          # codes of 0 leave -m
    m = np.abs(dequantize(qtype, z, packed.shape[0]))
    return w, np.abs(w) + 2 * m


def random_rows(t: int, k: int, seed: int) -> tuple[np.ndarray, np.ndarray]:
    """Codes over the whole of int8 and scales over three decades."""
    rng = np.random.default_rng(seed)
    q = np.clip(np.rint(rng.normal(0, 45, (t, k))), -128, 127).astype(np.int8)
    s = np.exp(rng.normal(-3, 1, (t, k // 32))).astype(np.float32)
    return q, s


def rows64(q: np.ndarray, s: np.ndarray) -> np.ndarray:
    return q.astype(np.float64) * np.repeat(s.astype(np.float64), 32, 1)


def linear64(qtype, packed, q, s, dtype: str):
    """(y, bound): the product in 64 bits, and how far a result of dtype may be
    off: every group's term has at most 6 f32 roundings on its way (the scale
    of the group, its product with the integer sum, the row's scale) and the
    sum of G terms at most G + 8 more (join of lanes and waves included), each
    relative to a partial sum no larger than the sum of the absolute terms."""
    w, wa = weight64(qtype, packed)
    x = rows64(q, s)
    y = x @ w.T
    groups = q.shape[1] // 32
    return y, (groups + 14) * U * (np.abs(x) @ wa.T) * 1.01 + ROUND[dtype] * np.abs(y) + 1e-30


def adapters64(x: np.ndarray, adapters, ids: np.ndarray, n: int):
    """(delta, bound) of scale * B (A x): the sums of k and r f32 terms, and the
    products A x held to 16 bits at least (2^-16)."""
    t, k = x.shape
    delta, bound = np.zeros((t, n)), np.zeros((t, n))
    for i, (a, b, scale) in enumerate(adapters):
        m = ids == i
        if not m.any():
            continue
        v = x[m] @ a.T
        va = np.abs(x[m]) @ np.abs(a).T
        delta[m] = scale * (v @ b.T)
        bound[m] = abs(scale) * (((k + a.shape[0] + 16) * U * va + 2.0 ** -16 * np.abs(v)) @ np.abs(b).T)
    return delta, bound
