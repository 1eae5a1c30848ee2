"""Plain 64-bit forms of rows in 4 bits and of heads' norms and rotation, for small inputs, and the bounds that follow from the roundings the kernels make."""
import numpy as np

from tests import cache_cases as K

F = np.float32
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
E4M3 = np.array([m / 512 if e == 0 else 2.0 ** (e - 7) * (1 + m / 8) for e in range(16) for m in range(8)][:127], np.float64)


def nearest(x, values):
    """Place of the nearest of `values` (rising) for each x >= 0; ties to the even place, beyond the last the last."""
    mid = (values[1:] + values[:-1]) / 2
    low, high = np.searchsorted(mid, x, "left"), np.searchsorted(mid, x, "right")
    return np.where(low % 2 == 0, low, high)


def quantise(x, exponent):
    """Codes [..., d] and scales [..., d / 16] of rows x."""
    y = x.astype(np.float64) * 2.0 ** -exponent
    y = y.reshape(*y.shape[:-1], -1, 16)
    nan = np.isnan(y).any(-1)
    size = np.where(np.isnan(y), 0.0, np.abs(y))
    size = np.minimum(size, 1e300)
    scale = nearest(size.max(-1) / 6, E4M3)
    s = E4M3[scale][..., None]
    code = np.where(s > 0, nearest(size / np.where(s > 0, s, 1.0), E2M1), 0)
    code = code + 8 * np.signbit(y)
    code = np.where(nan[..., None], 0, code)
    return code.reshape(x.shape).astype(np.uint8), np.where(nan, 127, scale).astype(np.uint8)


def values(codes, scales, exponent):
    """What codes and scales stand for (exact in float32); a scale's highest bit says nothing."""
    table = np.concatenate([E2M1, -E2M1])
    s = np.concatenate([E4M3, [np.nan]])[scales & 127]
    v = table[codes].reshape(*codes.shape[:-1], -1, 16) * s[..., None] * 2.0 ** exponent
    return v.reshape(codes.shape).astype(F)


def scale_bytes(d):
    return 4 if d <= 64 else 8 if d <= 128 else 16


def laid_out(codes, scales, fill=0):
    """Bytes as they lie by default: [row][head][d / 2, to a multiple of 16] and [row][head][d / 16, to 4, 8 or 16]; `fill` in the gaps."""
    d = codes.shape[-1]
    a = np.full((*codes.shape[:-1], -(-d // 32) * 16), fill, np.uint8)
    a[..., :d // 2] = codes[..., 0::2] | codes[..., 1::2] << 4
    b = np.full((*scales.shape[:-1], scale_bytes(d)), fill, np.uint8)
    b[..., :d // 16] = scales
    return a, b


def taken_up(a, b, d):
    """laid_out's inverse."""
    codes = np.empty((*a.shape[:-1], d), np.uint8)
    codes[..., 0::2], codes[..., 1::2] = a[..., :d // 2] & 15, a[..., :d // 2] >> 4
    return codes, np.ascontiguousarray(b[..., :d // 16])


class Call4(K.Call):
    """A call over rows in 4 bits: keys and values are what the codes stand for."""

    def attend(self, bf16):
        out, lse, out_tol, lse_tol = super().attend(bf16)
        # weights that meet the values as float16 numbers of which the largest is 2^8: each off by 2^-25 at most beside its half step
        for i, (b, _, q0, t, _) in enumerate(self.segs):
            for h in range(self.kv if t else 0):
                n, ok, _ = self.seen(i, h)
                v = self.values[b:b + n, h].astype(np.float64)
                off = 2.0 ** -33 * ok.astype(np.float64) @ np.where(np.isfinite(v), np.abs(v), 0.0)
                out_tol[q0:q0 + t, h * self.group:(h + 1) * self.group] += off[:, None, :]
        return out, lse, out_tol, lse_tol


def rotate(x, norm, weight, eps, freq, pos, axes, rotary, interleaved, magnitude, bf16):
    """Heads x [token][head][d] (float32 values) -> what they become and how far that may be off."""
    y = x.astype(np.float64)
    size = np.abs(y)
    d = y.shape[-1]
    rel = 0.0
    if norm:
        factor = 1 / np.sqrt((y ** 2).mean(-1, keepdims=True) + float(F(eps)))
        w = 1.0 if weight is None else weight.astype(np.float64)
        y, size = y * factor * w, size * np.abs(factor * w)
        rel = (d / 2 + 8) * K.EPS_F32  # the sum (half of it in each term's error, through the root), the root, its place, two products
    if rotary:
        at = np.zeros(rotary // 2, int) if axes is None else axes.astype(int)
        angle = pos[at].astype(np.float64).T * freq.astype(np.float64)  # [token][pair]
        c, s = (f(angle)[:, None] * magnitude for f in (np.cos, np.sin))
        i = 2 * np.arange(rotary // 2) if interleaved else np.arange(rotary // 2)
        j = i + 1 if interleaved else i + rotary // 2
        a, b = y[..., i].copy(), y[..., j].copy()
        ma, mb = size[..., i].copy(), size[..., j].copy()
        y[..., i], y[..., j] = a * c - b * s, a * s + b * c
        both = (ma + mb) * abs(magnitude)
        # cosine and sine: the angle's 2^-24 of a turn's part (2 pi of it in the value) and the function's 2 units, its scaling, two products and a sum; far positions: 64 bits' 2^-52 of the turns
        off = 2 * np.pi * (2.0 ** -24 + np.abs(angle)[:, None] * 2.0 ** -52) + 8 * K.EPS_F32
        tol = np.zeros_like(y)
        tol[..., i] = tol[..., j] = both * (rel + off)
        tol[..., rotary:] = size[..., rotary:] * rel
    else:
        tol = size * rel
    if bf16:
        tol = tol + 2.0 ** -8 * (np.abs(y) + tol)
    return y, tol + 1e-37
