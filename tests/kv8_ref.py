"""The 8-bit page operators in plain 64-bit numpy: codes, scales, the quantising write, attention, rotary positions."""
from __future__ import annotations

import math

import numpy as np

TOP = {"e4m3": 448.0, "int8": 127.0}


def exponent(amax: float, code: str) -> int:
    """Least e in -120 .. 120 with amax <= top * 2^e."""
    if amax <= math.ldexp(TOP[code], -120):
        return -120
    e = math.frexp(amax / TOP[code])[1] - 1
    while e < 120 and amax > math.ldexp(TOP[code], e):
        e += 1
    while e > -120 and amax <= math.ldexp(TOP[code], e - 1):
        e -= 1
    return e


def step_of(x: np.ndarray, code: str) -> np.ndarray:
    """Distance between neighbouring codes around x (x already divided by the scale)."""
    if code == "int8":
        return np.ones_like(x)
    a = np.clip(np.abs(x), 2.0 ** -6, 448.0)
    return np.exp2(np.frexp(a)[1] - 1 - 3)


def encode(x: np.ndarray, code: str) -> np.ndarray:
    """The nearest code's value, ties to even, saturating; NaN -> 0."""
    x = np.where(np.isnan(x), 0.0, np.clip(x, -TOP[code], TOP[code]))
    step = step_of(x, code)
    return np.rint(x / step) * step   # a carry into the next binade lands on its first code


class Page:
    """One page of one kv head and side: 16 rows of code values and the exponent."""

    def __init__(self, hd: int):
        self.c, self.e = np.zeros((16, hd)), None

    def write(self, first: int, x: np.ndarray, code: str) -> None:
        fin = np.abs(x[np.isfinite(x)])
        e = exponent(float(fin.max()) if fin.size else 0.0, code)
        if first and self.e is not None:
            e = max(e, self.e)
            if e > self.e:
                self.c[:first] = encode(self.c[:first] * 2.0 ** (self.e - e), code)
        self.c[first:first + len(x)] = encode(x * 2.0 ** -e, code)
        self.e = e

    def values(self) -> np.ndarray:
        return self.c * 2.0 ** (self.e if self.e is not None else 0)


class Cache:
    """A dense pool: pages[id][head][side]."""

    def __init__(self, n_pages: int, n_kv: int, hd: int, code: str):
        self.p = [[[Page(hd) for _ in range(2)] for _ in range(n_kv)] for _ in range(n_pages)]
        self.n_kv, self.hd, self.code = n_kv, hd, code

    def append(self, table, pos0: int, k: np.ndarray, v: np.ndarray) -> None:
        """k, v [T][n_kv][hd]."""
        t = 0
        while t < len(k):
            cell = pos0 + t
            n = min(16 - cell % 16, len(k) - t)
            for h in range(self.n_kv):
                for side, x in enumerate((k, v)):
                    self.p[table[cell // 16]][h][side].write(cell % 16, x[t:t + n, h].astype(np.float64), self.code)
            t += n

    def values(self, table, n: int, side: int) -> np.ndarray:
        """[n][n_kv][hd]"""
        pages = [np.stack([self.p[i][h][side].values() for h in range(self.n_kv)], 1) for i in table[: -(-n // 16)]]
        return np.concatenate(pages)[:n] if pages else np.zeros((0, self.n_kv, self.hd))


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, n_cells: int, scale: float):
    """One token: q [n_head][hd] over the first n_cells of k, v [cells][n_kv][hd] -> (out, sum p |v|, largest sum |scale q k| seen)."""
    n_head, hd = q.shape
    out, mag, dot = np.zeros((n_head, hd)), np.zeros((n_head, hd)), np.zeros(n_head)
    if n_cells <= 0:
        return out, mag, dot
    group = n_head // k.shape[1]
    for h in range(n_head):
        kk, vv = k[:n_cells, h // group], v[:n_cells, h // group]
        s = kk @ q[h] * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h], mag[h] = p @ vv, p @ np.abs(vv)
        dot[h] = (np.abs(kk) @ np.abs(q[h])).max() * abs(scale)
    return out, mag, dot


def rope_freqs(n_rot, theta, scaling="none", factor=1.0, orig_ctx=0, low=1.0, high=None):
    high = (32.0 if scaling == "yarn" else 4.0) if high is None else high
    if scaling == "ntk" and n_rot > 2:
        theta = theta * factor ** (n_rot / (n_rot - 2))
    f = theta ** (-np.arange(0, n_rot, 2, dtype=np.float64) / n_rot)
    if scaling == "linear":
        return f / factor
    if scaling == "yarn":
        at = lambda turns: n_rot * math.log(orig_ctx / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(at(high)), 0), min(math.ceil(at(low)), n_rot - 1)
        r = np.clip((np.arange(n_rot // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        return f / factor * r + f * (1 - r)
    if scaling == "bands":
        keep = np.clip((orig_ctx * f / (2 * math.pi) - low) / (high - low), 0, 1)
        return f / factor * (1 - keep) + f * keep
    return f


def rotate(x: np.ndarray, positions: np.ndarray, freqs: np.ndarray, layout: str, m: float = 1.0) -> np.ndarray:
    """x [tokens][heads][hd]; the angle by whole turns taken off in extended precision."""
    n, half = 2 * len(freqs), len(freqs)
    turns = np.asarray(positions, np.longdouble)[:, None] * (np.asarray(freqs, np.longdouble) / (2 * np.pi if np.longdouble is np.float64 else np.longdouble("6.283185307179586476925286766559")))
    a = ((turns - np.rint(turns)).astype(np.float64) * 2 * math.pi)[:, None, :]
    c, s = np.cos(a) * m, np.sin(a) * m
    out = x.astype(np.float64).copy()
    i, j = (slice(0, half), slice(half, n)) if layout == "half" else (slice(0, n, 2), slice(1, n, 2))
    p, q = out[..., i].copy(), out[..., j].copy()
    out[..., i], out[..., j] = p * c - q * s, p * s + q * c
    return out
