"""CPU oracle of the 8-bit linears and the norm before them (include/w8_api.h), numpy only, written from the formulas.

Codes are defined exactly (the nearest whole number, the even one of two) and compared for equality; 127 t and the comparison with
the middle of two codes are exact in float64, t having at most 24 bits."""
import numpy as np

F = np.float32
SMALLEST = 2.0 ** -100


def to64(x, bf16):
    """Bits uint16 -> float64."""
    if bf16:
        return (x.astype(np.uint32) << 16).view(F).astype(np.float64)
    return x.view(np.float16).astype(np.float64)


def round16(x, bf16):
    """float64 -> the nearest 16-bit value, as float64."""
    with np.errstate(all="ignore"):
        if not bf16:
            return np.asarray(x, np.float64).astype(np.float16).astype(np.float64)
        # two roundings to float32 and bf16 would differ from one: what float32 cannot hold goes into its lowest bit (round to odd)
        x = np.asarray(x, np.float64)
        f = x.astype(F)
        bits = f.view(np.uint32).copy()
        off = (f.astype(np.float64) != x) & np.isfinite(x) & np.isfinite(f)
        away = off & (np.abs(f.astype(np.float64)) > np.abs(x))
        bits = np.where(away, bits - 1, bits)
        bits = np.where(off, bits | 1, bits).astype(np.uint32)
        nan = np.isnan(x)
        r = ((bits.astype(np.uint64) + 0x7FFF + ((bits >> 16) & 1)) >> 16).astype(np.uint32) << 16
        return np.where(nan, np.nan, r.view(F).astype(np.float64))


def encode(t):
    """float32 rows [N][K] -> codes int8, largest magnitudes float32 (NaN for a row with an infinity or a NaN)."""
    t = np.asarray(t, F)
    with np.errstate(all="ignore"):
        bad = ~np.isfinite(t).all(-1)
        m = np.where(bad, F(0), np.abs(t).max(-1)).astype(F)
        none = m.astype(np.float64) < SMALLEST
        safe = np.where(none, 1.0, m.astype(np.float64))
        codes = np.rint(127.0 * np.where(bad[:, None], F(0), t).astype(np.float64) / safe[:, None])
        codes = np.where((bad | none)[:, None], 0, codes).astype(np.int8)
        return codes, np.where(bad, F(np.nan), np.where(none, F(0), m)).astype(F)


def norm(x, weight, eps, residual, bf16):
    """Bits -> (h as float64 of 16 bits, y float64, t float32, 1 / rms)."""
    h = to64(x, bf16)
    with np.errstate(all="ignore"):
        if residual is not None:
            h = round16(h + to64(residual, bf16), bf16)
        w = to64(weight, bf16)
        inverse = 1 / np.sqrt((h ** 2).mean(-1) + eps)
        return h, h * inverse[:, None] * w, (h.astype(F) * w.astype(F)).astype(F), inverse


def activate(y, act):
    with np.errstate(all="ignore"):
        if act == 1:
            return np.where(y < 0, 0, y)
        if act == 2:
            return 0.5 * y * (1 + np.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3)))
        if act == 3:
            return y / (1 + np.exp(-y))
        return y


def product(codes, scales, w, sw, bias=None):
    """float64 sums [N][M] and the scale of their rounding errors."""
    with np.errstate(all="ignore"):
        s = (codes.astype(np.float64) @ w.astype(np.float64).T) * sw.astype(np.float64) * scales.astype(np.float64)[:, None]
        return (s, np.abs(s)) if bias is None else (s + bias, np.abs(s) + np.abs(bias))


def linear(codes, scales, w, sw, bias=None, act=0):
    """float64 y and its bound of float32 errors (2^-22 of the sum's terms, 2^-16 of an activation's value)."""
    s, mag = product(codes, scales, w, sw, bias)
    y = activate(s, act)
    return y, 1.13 * 2.0 ** -22 * mag + (2.0 ** -16 * np.abs(y) if act > 1 else 0)


def gated(codes, scales, g, sg, u, su, bg=None, bu=None, act=3):
    a, ea = linear(codes, scales, g, sg, bg, act)
    b, eb = linear(codes, scales, u, su, bu, 0)
    return a * b, ea * np.abs(b) + eb * np.abs(a) + 2.0 ** -23 * np.abs(a * b)
