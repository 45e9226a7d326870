"""Plain numpy statements of the 4-bit KV cache and of the residual RMS norm with 8-bit output (tests only)."""
import numpy as np

F32 = np.float32


def bf16_round(x):
    """fp32 rounded to 8 significand bits, nearest even."""
    u = np.asarray(x, F32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(F32)


def scale16(d):
    return bf16_round(np.clip(np.asarray(d, F32), F32(-8160), F32(8160))).astype(np.float16)


def quantise(x):
    """fp32 [..., D] -> codes uint8 [..., D], fp32 d [..., D / 32] before rounding."""
    b = np.asarray(x, F32).reshape(*x.shape[:-1], -1, 32)
    top, low = b.max(-1), b.min(-1)
    m = np.where(top >= -low, top, low).astype(F32)
    with np.errstate(divide="ignore"):
        inv = np.where(np.abs(m) < F32(2.0 ** -100), F32(0), F32(-8) / m).astype(F32)
    c = np.floor((b * inv[..., None]).astype(F32) + F32(8.5))
    return np.clip(c, 0, 15).astype(np.uint8).reshape(x.shape), (m * F32(-0.125)).astype(F32)


def rotate(x, rope, pos):
    """NEOX rotation of [n, h, D] in fp32, each product and sum rounded; rope [P, D / 2, 2]."""
    D = x.shape[-1]
    c, s = rope[pos][:, None, :, 0].astype(F32), rope[pos][:, None, :, 1].astype(F32)
    a, b = x[..., : D // 2], x[..., D // 2:]
    return np.concatenate([(a * c).astype(F32) - (b * s).astype(F32), (b * c).astype(F32) + (a * s).astype(F32)], -1).astype(F32)


class Pages:
    """A pool in the library's layout, addressed one nibble and one scale at a time."""

    def __init__(self, n_pages, page, kv, D, fill=0):
        self.page, self.kv, self.D, self.NB, self.r = page, kv, D, D // 32, 2 if D == 128 else 4
        self.raw = np.full((n_pages, kv, page // 16, 18 * D), fill, np.uint8)

    def _k_nibble(self, s, dim):
        return s * self.D + ((dim % 32) // 8 * self.NB + dim // 32) * 8 + dim % 8

    def _v_nibble(self, s, dim):
        g, e, m, t = dim // (self.D // 8), dim % (self.D // 8), s // 4, s % 4
        return 16 * self.D + (((m // self.r * 8 + g) * 4 + t) * self.r + m % self.r) * (self.D // 8) + e

    def _scale(self, is_v, s, b):
        return 17 * self.D + 2 * ((b * 4 + s % 4) * 4 + s // 4) if is_v else 16 * self.D + 2 * (s * self.NB + b)

    def put(self, page, pos, h, is_v, codes, scales):
        tile, s = self.raw[page, h, pos % self.page // 16], pos % 16
        for dim in range(self.D):
            n = (self._v_nibble if is_v else self._k_nibble)(s, dim)
            sh = 4 * (n % 2)
            tile[n // 2] = (int(tile[n // 2]) & (0xF0 >> sh)) | (int(codes[dim]) << sh)
        for b in range(self.NB):
            at = self._scale(is_v, s, b)
            tile[at:at + 2] = np.frombuffer(np.float16(scales[b]).tobytes(), np.uint8)

    def values(self, table_row, n, is_v):
        """float64 [n, kv, D] of positions 0 .. n - 1."""
        pos = np.arange(n)
        tiles = self.raw[table_row[pos // self.page], :, pos % self.page // 16]          # [n, kv, bytes]
        dim, s = np.arange(self.D)[None], (pos % 16)[:, None]
        nib = (self._v_nibble if is_v else self._k_nibble)(s, dim)
        byte = np.take_along_axis(tiles, (nib // 2)[:, None, :].repeat(self.kv, 1), 2)
        code = (byte >> (4 * (nib % 2))[:, None, :].astype(np.uint8)) & 15
        at = self._scale(is_v, s, dim // 32)
        lo = np.take_along_axis(tiles, at[:, None, :].repeat(self.kv, 1), 2).astype(np.uint16)
        hi = np.take_along_axis(tiles, (at + 1)[:, None, :].repeat(self.kv, 1), 2).astype(np.uint16)
        return (lo | hi << 8).astype(np.uint16).view(np.float16).astype(np.float64) * (code.astype(np.float64) - 8)


def random_pool(rng, n_pages, page, kv, D):
    """Every nibble random, every scale a positive or negative 8-bit-significand fp16 around 0.1."""
    p = Pages(n_pages, page, kv, D)
    p.raw[...] = rng.integers(0, 256, p.raw.shape, np.uint8)
    sc = scale16(rng.uniform(0.03, 0.2, p.raw.shape[:-1] + (D,)) * rng.choice([-1, 1], p.raw.shape[:-1] + (D,)))
    p.raw[..., 16 * D:] = sc.view(np.uint8)
    return p


def attention(q, k, v, first, scale):
    """float64: rows q [T, heads, D] at positions first + i over k, v [n, kv, D]; rows that see nothing are zero."""
    T, H, D = q.shape
    kv, n = k.shape[1], k.shape[0]
    out = np.zeros((T, H, D))
    for h in range(H):
        z = scale * q[:, h].astype(np.float64) @ k[:, h * kv // H].T
        z = np.where(np.arange(n)[None] <= first + np.arange(T)[:, None], z, -np.inf)
        live = np.isfinite(z).any(1) if n else np.zeros(T, bool)
        if live.any():
            p = np.exp(z[live] - z[live].max(1, keepdims=True))
            out[live, h] = p / p.sum(1, keepdims=True) @ v[:, h * kv // H]
    return out


def attention_bound(q, k, v, scale, n, half):
    """Largest absolute error the kernel's arithmetic allows.

    A score sums D products q k: q is held to 2^-22 (hi + lo halves), the tensor core keeps a sum to 2^-23 of its running
    size at each of its 2 D / 16 steps and D / 32 fp32 updates follow: with A = scale * max sum |q k| at most
    A * (2^-22 + (D / 8 + D / 32) * 2^-23). exp2 of it (and its argument's rounding, A * 2^-23 again) moves p by that
    relatively, 2^-21 more for exp2 itself and p's split into halves. Numerator and sum both carry it (factor 2).
    The sum over positions takes a step for 16 positions of a warp (two, and an fp32 addition, for fp32 q), at most n / 128 * 2 + 2
    of them, and 2^-23 each; joining 8 warps and up to 320 runs adds 2^-24 each. All relative to sum p |v| <= max |v|. fp16 q: p of the numerator is
    rounded to fp16, 2^-11, or 2^-25 where it is subnormal (the sum below is at least 1, of the position that set the maximum), and
    the output adds half a step."""
    D = q.shape[-1]
    A = scale * max(float(np.abs(q).reshape(-1, D).max(0) @ np.abs(k).reshape(-1, D).max(0)), 1e-30) if k.size else 0.0
    top = float(np.abs(v).max()) if v.size else 0.0
    rel = 2 * (A * (2.0 ** -22 + (D / 8 + D / 32 + 1) * 2.0 ** -23) + 2.0 ** -21) + (n / 64 + 2) * 2.0 ** -23 + 330 * 2.0 ** -24
    return top * (rel + (2 * 2.0 ** -11 + n * 2.0 ** -25 if half else 0.0)) + 1e-12


def norm_q8(x, res, w, eps, group):
    """h (as stored), int8 codes, float64 scales [rows, groups]; codes in the formula's fp32 steps."""
    h = x if res is None else (x.astype(F32) + res.astype(F32)).astype(x.dtype)
    f = h.astype(F32)
    d = x.shape[1]
    t = (f * w[None]).astype(F32).reshape(x.shape[0], -1, group or d)
    top = np.abs(t).max(-1)
    tiny = top < F32(2.0 ** -110)
    with np.errstate(divide="ignore", over="ignore"):
        inv = np.where(tiny, F32(0), F32(127) / top).astype(F32)
    q = np.clip(np.rint((t * inv[..., None]).astype(F32)), -127, 127).astype(np.int8).reshape(x.shape)
    rms = np.sqrt((h.astype(np.float64) ** 2).mean(1) + eps)
    return h, q, np.where(tiny, 0.0, top.astype(np.float64) / 127 / rms[:, None])


def prompt_bound(q, k, v, scale, n, half):
    """The same for calls of 256 rows and more, whose products are tcgen05's (128 positions a tile, 8 steps of 16).

    Scores as in attention_bound. fp16 q: p is rounded to fp16 in the numerator alone, half a step of p, 2^-11, or 2^-25 where it
    is subnormal (the sum below it is at least 1, of the position that set the maximum); its sums take n / 16 steps of 2^-23.
    fp32 q: p in halves as there; a tile's sum takes 16 steps, and the tiles are added in fp32, 2^-24 each and as much
    again for the factor of a tile's max."""
    D = q.shape[-1]
    A = scale * max(float(np.abs(q).reshape(-1, D).max(0) @ np.abs(k).reshape(-1, D).max(0)), 1e-30) if k.size else 0.0
    top = float(np.abs(v).max()) if v.size else 0.0
    rel = 2 * (A * (2.0 ** -22 + (D / 8 + D / 32 + 1) * 2.0 ** -23) + 2.0 ** -21) + 330 * 2.0 ** -24
    if half:
        rel += 2 * 2.0 ** -11 + n * 2.0 ** -25 + (n / 16 + 8) * 2.0 ** -23
    else:
        rel += 16 * 2.0 ** -23 + (n / 128 + 1) * 2.0 ** -23
    return top * rel + 1e-12
