"""Plain references in 64 bits for the attention path's operators: the 4-bit cache's codes and layout, attention over
it, and the per-head norm with rotation and its gradients.  Definitions: include/kore_hip.h."""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24  # half a step of f32, relative
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def blocks(d: int) -> int:
    return (d + 31) // 32


def quantise(x: np.ndarray):
    """x [..., D] -> codes [..., 32 nb] (0..15) and scale bytes [..., nb], by trying every scale and every code."""
    d, nb = x.shape[-1], blocks(x.shape[-1])
    w = np.zeros(x.shape[:-1] + (nb * 32,), np.float32)
    w[..., :d] = x
    w = w.reshape(x.shape[:-1] + (nb, 32))
    finite = np.isfinite(w).all(-1)
    v = np.where(finite[..., None], w, 0.0).astype(np.float64)
    amax = np.abs(v).max(-1)
    e = np.full(amax.shape, 126)
    for t in range(125, -101, -1):
        e = np.where(amax <= 7.0 * 2.0 ** t, t, e)
    y = np.abs(v) / 2.0 ** e[..., None].astype(np.float64)
    y = np.where(e[..., None] == 126, np.minimum(y, 3.0), y)
    dist = np.abs(y[..., None] - MAGNITUDES)
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])  # of two equally near, the even code
    code = order[np.argmin(dist[..., order], -1)]
    code = code + 8 * np.signbit(np.where(finite[..., None], w, 0.0))
    scale = np.where(finite, e + 127, 255)
    return code.reshape(x.shape[:-1] + (nb * 32,)).astype(np.uint8), scale.astype(np.uint8)


def values(codes: np.ndarray, scales: np.ndarray, d: int) -> np.ndarray:
    """What codes [..., 32 nb] and scale bytes [..., nb] stand for, in 64 bits."""
    m = MAGNITUDES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127.0))
    return (m.reshape(scales.shape + (32,)) * s[..., None]).reshape(codes.shape)[..., :d]


def places(page: int, d: int, t: int, value: bool):
    """Byte offsets, in one page of one key head, of token t's code bytes [16 nb] and scale bytes [nb]."""
    nb = blocks(d)
    j, b = np.arange(16 * nb), np.arange(nb)
    if not value:
        return t * 16 * nb + j, page * nb * 32 + t * nb + b
    tile, g, i = t // 16, t % 16 // 4, t % 4
    return (page * nb * 16 + tile * 256 * nb + ((g * 4 * nb + j // 4) * 4 + i) * 4 + j % 4,
            page * nb * 33 + (tile * nb + b) * 16 + t % 16)


class Cache:
    """A cache on the host: bytes [pages, heads, page * nb * 34]."""

    def __init__(self, pages: int, page: int, heads: int, d: int, fill=None, seed: int = 0):
        self.page, self.d = page, d
        shape = (pages, heads, page * blocks(d) * 34)
        if fill is None:  # what nobody wrote: any bytes at all
            self.bytes = np.random.default_rng(seed).integers(0, 256, shape).astype(np.uint8)
        else:
            self.bytes = np.full(shape, fill, np.uint8)

    def write(self, slots, k, v):
        for t, slot in enumerate(np.asarray(slots, np.uint32)):
            p, at = int(slot) // self.page, int(slot) % self.page
            if p >= self.bytes.shape[0]:
                continue
            for value, x in ((False, k[t]), (True, v[t])):
                codes, scales = quantise(x)
                c, s = places(self.page, self.d, at, value)
                self.bytes[p][:, c] = codes[:, 0::2] | codes[:, 1::2] << 4
                self.bytes[p][:, s] = scales

    def read(self, slots):
        """k, v [T, heads, D] in 64 bits; zeros past the last page."""
        heads, out = self.bytes.shape[1], []
        for value in (False, True):
            x = np.zeros((len(slots), heads, self.d))
            for t, slot in enumerate(np.asarray(slots, np.uint32)):
                p, at = int(slot) // self.page, int(slot) % self.page
                if p < self.bytes.shape[0]:
                    c, s = places(self.page, self.d, at, value)
                    b = self.bytes[p][:, c]
                    codes = np.stack([b & 15, b >> 4], -1).reshape(heads, -1)
                    x[t] = values(codes, self.bytes[p][:, s], self.d)
            out.append(x)
        return out


def attention(q, cache: Cache, table, lens, starts, scale, causal, out):
    """Rows of every sequence into a copy of `out` [tokens, q_heads, D]; returns it and what a result may be off by.

    Off by: a score's error is `u` for q's rounding, and for the sum of 3 nb products of 32 terms at most 3 * 8 + 8 roundings,
    all relative to scale * sum |q k|; the subtraction of the maximum and the exponential 2 u of the score's size and 2 u.
    A probability's three bf16 terms are all of its bits; the row's sums add three roundings for each step of 32 keys
    (a product for each term), 64 for joining what was split, and the division."""
    tokens, q_heads, d = q.shape
    heads = cache.bytes.shape[1]
    group = q_heads // heads
    o, tol = out.astype(np.float64).copy(), np.zeros(out.shape)
    cap = table.shape[1] * cache.page
    for s in range(len(lens)):
        q0, q1 = min(int(starts[s]), tokens), min(int(starts[s + 1]), tokens)
        if q1 <= q0:
            continue
        n = min(int(lens[s]), cap)
        at = np.arange(n)
        pages = table[s][at // cache.page].astype(np.int64) if n else at
        there = pages < cache.bytes.shape[0]
        k, v = cache.read(np.where(there, pages * cache.page + at % cache.page, 0)) if n else (np.zeros((0, heads, d)),) * 2
        for i in range(q0, q1):
            lim = n - (q1 - 1 - i) if causal else n
            seen = np.flatnonzero(there & (at < lim))
            for h in range(q_heads):
                if len(seen) == 0:
                    o[i, h], tol[i, h] = 0.0, 0.0
                    continue
                kk, vv, qq = k[seen, h // group], v[seen, h // group], q[i, h].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    x = kk @ qq * scale
                    p = np.exp(x - x.max())
                    p = p / p.sum()
                    o[i, h] = p @ vv
                    size = np.abs(kk) @ np.abs(qq) * abs(scale)
                    delta = 33 * U * size.max() + 2 * U * np.abs(x).max() + 2 * U
                    tol[i, h] = p @ np.abs(vv) * (2 * delta + (3 * len(seen) / 32 + 64) * U)
    return o, tol


def turn(x, pos, inv_freq, interleaved, back=False):
    """x [T, H, D] rotated by pos [T] * inv_freq, in 64 bits."""
    a = pos.astype(np.float64)[:, None, None] * inv_freq.astype(np.float64)
    c, s = np.cos(a), np.sin(a) * (-1.0 if back else 1.0)
    half = x.shape[-1] // 2
    o = np.empty(x.shape)
    lo, hi = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, half), slice(half, None))
    o[..., lo] = x[..., lo] * c - x[..., hi] * s
    o[..., hi] = x[..., lo] * s + x[..., hi] * c
    return o


def _both(x, interleaved):
    """|a| + |b| of each value's pair, at both places."""
    return turn(np.abs(x), np.zeros(x.shape[0]), np.zeros(x.shape[-1] // 2), interleaved) + _partner(np.abs(x), interleaved)


def _partner(x, interleaved):
    half = x.shape[-1] // 2
    if interleaved:
        return x.reshape(x.shape[:-1] + (half, 2))[..., ::-1].reshape(x.shape)
    return np.concatenate([x[..., half:], x[..., :half]], -1)


def angle_error(pos, inv_freq, interleaved):
    """What the 64-bit angle is off by: three roundings of 2^-53 of it, [T, 1, D]."""
    e = 3 * 2.0 ** -53 * pos.astype(np.float64)[:, None] * inv_freq.astype(np.float64)
    return (np.repeat(e, 2, -1) if interleaved else np.concatenate([e, e], -1))[:, None, :]


def qk_norm_rope(x, w, pos, inv_freq, eps, interleaved):
    """x [T, H, D] -> result and what it may be off by: 12 roundings of the norm (its sum of squares has at most 22, which
    the root halves), 2 of the rotation, 4 of sine and cosine and pi of their argument: 32 of the pair's size hold them."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    tol = _both(y, interleaved) * (32 * U + angle_error(pos, inv_freq, interleaved))
    return turn(y, pos, inv_freq, interleaved), tol


def qk_norm_rope_backward(dy, x, w, pos, inv_freq, eps, interleaved):
    """(dx, dw, tolerances of both): dx is a difference of two terms whose parts have the forward's roundings each; dw's
    sum of T H terms adds at most 192 (rows of a lane, lanes, workgroups) to a term's own 64."""
    x, w, dy = x.astype(np.float64), w.astype(np.float64), dy.astype(np.float64)
    g = turn(dy, pos, inv_freq, interleaved, back=True)
    inv = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n, u = x * inv, g * w
    dx = inv * (u - n * (u * n).mean(-1, keepdims=True))
    size = _both(dy, interleaved)  # what g's two products add up to
    off = 64 * U + angle_error(pos, inv_freq, interleaved)
    dx_tol = off * inv * (size * np.abs(w) + np.abs(n) * (size * np.abs(w * n)).mean(-1, keepdims=True))
    dw_tol = ((192 * U + off) * size * np.abs(n)).sum((0, 1))
    return dx, (g * n).sum((0, 1)), dx_tol, dw_tol


def assert_within(got, want, tol, what=""):
    """|got - want| <= tol per element (plus the smallest normal f32); NaN meets NaN."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (got.shape, want.shape)
    with np.errstate(invalid="ignore"):
        ok = np.abs(got - want) <= np.asarray(tol) + 2.0 ** -126
    ok |= np.isnan(got) & np.isnan(want)
    if not ok.all():
        i = tuple(np.argwhere(~ok)[0])
        raise AssertionError(f"{what}: {np.count_nonzero(~ok)} of {ok.size} outside; first at {i}: got {got[i]!r}, "
                             f"want {want[i]!r}, tolerance {np.broadcast_to(tol, got.shape)[i]!r}")
