"""Plain forms of the paged 4-bit cache's definitions (include/moe_b200.h) for
the tests: the quantizer and the page layout value by value, rotary positions
and attention in 64 bits.  numpy and torch on the CPU."""
import math

import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rope_kind(moe, t):
    return {torch.float32: moe.F32, torch.float16: moe.F16, torch.bfloat16: moe.BF16}[t.dtype]


def rows(moe, x):
    """moe.Rows of a [token, head, value] tensor"""
    assert x.stride(2) == 1 or x.shape[2] == 1
    return moe.Rows(x.data_ptr(), rope_kind(moe, x), x.shape[1], x.stride(0), x.stride(1))


# ------------------------------------------------------------------ rotation
def frequencies(rot, theta, scaling="none", factor=1.0, orig=0.0, fast=32.0, slow=1.0, low=1.0,
                high=4.0, divisors=None):
    out = []
    for i in range(rot // 2):
        f = theta ** (-2.0 * i / rot)
        if divisors is not None:
            f /= float(np.float32(divisors[i]))
        if scaling == "linear":
            f /= factor
        elif scaling == "parts":
            at = lambda n: rot * math.log(orig / (n * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
            a, b = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rot - 1)
            r = min(max((i - a) / max(b - a, 0.001), 0.0), 1.0)
            f = f / factor * r + f * (1 - r)
        elif scaling == "bands":
            s = min(max((orig * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
            f = (1 - s) * f / factor + s * f
        out.append(f)
    return np.array(out)


def rotate(x, pos, freq, layout, magnitude=1.0):
    """float64 rows [token, head, value] turned, and each value's |a| + |b| (for error bounds)"""
    x = np.asarray(x, np.float64)
    y, size = x.copy(), np.abs(x)
    half = len(freq)
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if layout == "pairs" else (i, i + half)
        ang = np.asarray(pos, np.float64) * freq[i]
        c, s = (np.cos(ang) * magnitude)[:, None], (np.sin(ang) * magnitude)[:, None]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., a] * s + x[..., b] * c
        size[..., a] = size[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * magnitude
    return y, size


# ------------------------------------------------------------------ the cache
def quantize(x):
    """codes and fp16 scales of fp32 rows [..., head_len]"""
    x = np.asarray(x, np.float32)
    b = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        hi, lo = b.max(-1), b.min(-1)
        m = np.where(hi >= -lo, hi, lo)
        scale = np.clip(m * np.float32(-0.125), -65504, 65504).astype(np.float16)
        scale = np.where(scale == 0, np.float16(0), scale)   # +0 for either zero
        d = scale.astype(np.float32)
        inv = np.where(d == 0, np.float32(0), np.float32(1) / d)
        codes = np.clip(np.rint(b * inv[..., None]) + 8, 0, 15)
    ok = np.isfinite(b).all(-1)
    codes = np.where(ok[..., None], codes, 8).astype(np.uint8)
    return codes, np.where(ok, scale, np.float16(np.nan))


def values(codes, scale):
    v = (codes.astype(np.float32) - np.float32(8)) * scale.astype(np.float32)[..., None]
    return v.reshape(*codes.shape[:-2], -1)


def places(nb, width):
    """byte of a row that holds value e of the head, and whether in the high nibble"""
    e = np.arange(32 * nb)
    b, k = e // 32, e % 16
    return (k // width) * width * nb + width * b + k % width, e % 32 >= 16


class Pool:
    """Pages in host memory, written and read row by row."""

    def __init__(self, n_pages, P, KVH, D, fill=None, seed=0):
        self.P, self.KVH, self.D, self.nb = P, KVH, D, D // 32
        self.rec = P * (D // 2 + D // 16)
        rng = np.random.default_rng(seed)
        self.data = rng.integers(0, 256, (n_pages, KVH, 2, self.rec), dtype=np.uint8)
        if fill == "nan":   # every scale a NaN: what no result may depend on
            self.scales()[...] = 0x7fff
        else:
            self.scales()[...] = np.float16(0.25).view(np.uint16)

    def scales(self):
        return self.data[..., self.P * self.D // 2:].view(np.uint16).reshape(
            *self.data.shape[:3], self.P, self.nb)

    def put(self, page, at, which, x):
        """fp32 [KVH, D] into a row"""
        codes, scale = quantize(x)
        place, high = places(self.nb, (4, 2)[which])
        row = np.zeros((self.KVH, self.D // 2), np.uint8)
        c = codes.reshape(self.KVH, -1)
        row[:, place[~high]] |= c[:, ~high]
        row[:, place[high]] |= c[:, high] << 4
        a = at * self.D // 2
        self.data[page, :, which, a:a + self.D // 2] = row
        self.scales()[page, :, which, at] = scale.view(np.uint16)

    def get(self, page, at, which):
        """the row's values, fp32 [KVH, D]"""
        place, high = places(self.nb, (4, 2)[which])
        a = at * self.D // 2
        by = self.data[page, :, which, a:a + self.D // 2][:, place]
        code = np.where(high, by >> 4, by & 15).reshape(self.KVH, self.nb, 32)
        return values(code, self.scales()[page, :, which, at].view(np.float16))

    def sequence(self, table, n, which):
        if n == 0:
            return np.zeros((0, self.KVH, self.D), np.float32)
        return np.stack([self.get(table[r // self.P], r % self.P, which) for r in range(n)])


# ------------------------------------------------------------------ attention
def attention(q, k, v, scale, causal=True, window=0):
    """float64 out [n, H, D], lse [n, H], and per row the largest scale * sum |q k| of
    a seen row; query i stands at row len(k) - n + i"""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    n, H, D = q.shape
    S, KVH = k.shape[:2]
    G = H // KVH
    out, lse, size = np.zeros((n, H, D)), np.full((n, H), -np.inf), np.zeros((n, H))
    j = np.arange(S)
    for i in range(n):
        row = S - n + i
        seen = np.ones(S, bool)
        if causal:
            seen &= j <= row
        if window:
            seen &= j > row - window
        if not seen.any():
            continue
        for h in range(H):
            kk, vv = k[seen, h // G], v[seen, h // G]
            s = kk @ q[i, h] * scale
            size[i, h] = np.abs(scale) * (np.abs(kk) @ np.abs(q[i, h])).max()
            m = s.max()
            p = np.exp(s - m)
            out[i, h] = p @ vv / p.sum()
            lse[i, h] = m + np.log(p.sum())
    return out, lse, size


def attention_bounds(dtype, size, vmax, n_rows, out, lse):
    """Largest errors of out [n, H, D] and lse that the kernel's roundings allow.
    A score: products of exact codes with q in fp16 (fp32 rows: two halves, 2^-22),
    summed 16 at a time in fp32 (two sums of a block, each up to 2^-22 of its
    terms), scaled and added over at most 8 blocks (2^-24 each): 2^-20 of sum |q k|.
    A weight: exp of that, of an argument rounded to 2^-23 of its size, and of the
    2-ulp exponential: 2^-20 size + 2^-20; it moves numerator and denominator.
    Weighted sums: a chain of n / 16 products of 16 rows each, every sum cut to 24
    bits (2^-24 of sums that grow evenly, half the last on average: n / 64 * 2^-23),
    joined over the runs.  16-bit rows: a weight is rounded to fp16, and once more
    with its row's scale or its value is (2^-11 each), the result to its type (half
    of eps)."""
    e = 2.0 ** -20 * size[..., None] + 2.0 ** -20
    tol = vmax * (2 * e + (n_rows / 64 + 16) * 2.0 ** -23)
    if dtype != torch.float32:
        tol = tol + vmax * 2 * 2.0 ** -11
    tol = tol + np.abs(out) * torch.finfo(dtype).eps / 2 + float(torch.finfo(dtype).tiny)
    tol_lse = 2.0 ** -20 * size + 2.0 ** -20 * (1 + np.abs(np.where(np.isfinite(lse), lse, 0)))
    return tol, tol_lse
