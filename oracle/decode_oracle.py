"""CPU oracle of the decode operators (include/decode_api.h), numpy only, written from the formulas.

The cache's encoding is float32 arithmetic rounded operation by operation, so codes and words are compared for equality;
attention and linears are computed in float64."""
import numpy as np

F = np.float32


def encode(x):
    """float32 [..., D] -> codes uint8 [..., D], words uint32 [...]."""
    x = np.asarray(x, F)
    with np.errstate(all="ignore"):
        hi = np.maximum(np.max(x, -1), F(0))
        lo = np.minimum(np.min(x, -1), F(0))
        fifteenth = F(1.0 / 15.0)
        s = (hi * fifteenth).astype(F) - (lo * fifteenth).astype(F)
        bad = ~np.isfinite(x).all(-1)
        s = np.where(bad, F(1), s).astype(F)
        word = (s.view(np.uint32) + np.uint32(8)) & np.uint32(0xFFFFFFF0)
        word = np.where(s < F(2.0 ** -100), np.uint32(0x3F800000), word)
        z = np.clip(np.rint(np.where(bad, F(0), -lo) * (F(1) / word.view(F))), F(0), F(15))
        word = word | z.astype(np.uint32)
        inv = F(1) / word.view(F)
        codes = np.clip(np.rint(np.where(bad[..., None], F(0), x) * inv[..., None]) + z[..., None], F(0), F(15))
    codes = np.where(bad[..., None], 0, codes).astype(np.uint8)
    return codes, np.where(bad, np.uint32(0x7FC00000), word).astype(np.uint32)


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    return np.stack((packed & 15, packed >> 4), -1).reshape(packed.shape[:-1] + (-1,))


def decode32(packed, words):
    """The values of the cache as float32 products."""
    z = (words & np.uint32(15)).astype(F)
    with np.errstate(all="ignore"):
        return words.view(F)[..., None] * (unpack(packed).astype(F) - z[..., None])


def decode64(packed, words):
    z = (words & np.uint32(15)).astype(np.float64)
    with np.errstate(all="ignore"):
        return words.view(F).astype(np.float64)[..., None] * (unpack(packed).astype(np.float64) - z[..., None])


def rotate(x, table, rows, interleaved):
    """float32 [T][H][D] by table[rows] (cosines, sines), operation by operation in float32; a row outside gives NaN."""
    x, half = np.array(x, F), table.shape[1] // 2
    inside = (rows >= 0) & (rows < table.shape[0])
    t = np.where(inside[:, None], table[np.where(inside, rows, 0)], F(np.nan)).astype(F)
    cos, sin = t[:, None, :half], t[:, None, half:]
    one = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    two = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., one].copy(), x[..., two].copy()
    x[..., one] = (a * cos).astype(F) - (b * sin).astype(F)
    x[..., two] = (b * cos).astype(F) + (a * sin).astype(F)
    return x


def places(lens, cu, tokens):
    """(sequence or -1, place) of every row."""
    seq, place = np.full(tokens, -1), np.full(tokens, -1)
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        for i in range(n):
            seq[cu[b] + i], place[cu[b] + i] = b, lens[b] - n + i
    return seq, place


def attention(q, k_codes, k_words, v_codes, v_words, table, lens, cu, scale, window=0):
    """float64 attention: outputs, sums of p |v| (the scale of rounding errors), log-sum-exp."""
    T, H, D = q.shape
    pages, heads, P = k_words.shape
    share = H // heads
    out, mag = np.zeros((T, H, D)), np.zeros((T, H, D))
    lse = np.full((T, H), -np.inf)
    seq, place = places(lens, cu, T)
    for t in range(T):
        b, p = seq[t], place[t]
        if b < 0 or p < 0 or p >= table.shape[1] * P:
            continue
        first = max(0, p - window + 1) if window else 0
        keys = [j for j in range(first, p + 1) if 0 <= table[b, j // P] < pages]
        if not keys:
            continue
        pg, sl = table[b, np.array(keys) // P], np.array(keys) % P
        for h in range(H):
            k = decode64(k_codes[pg, h // share, sl], k_words[pg, h // share, sl])
            v = decode64(v_codes[pg, h // share, sl], v_words[pg, h // share, sl])
            with np.errstate(all="ignore"):
                x = k @ q[t, h].astype(np.float64) * scale
                m = x.max()
                e = np.exp(x - m)
                out[t, h] = e @ v / e.sum()
                mag[t, h] = e @ np.abs(v) / e.sum()
                lse[t, h] = m + np.log(e.sum())
    return out, mag, lse


def linear(x, codes, scales, zeros, bias=None, act=0):
    """float64 y [N][M], sums of |x s (w - z)| and of |x| s (w + z): the scales of rounding errors."""
    M, K = codes.shape
    G = K // scales.shape[1]
    s = np.repeat(scales.astype(np.float64), G, 1)
    z = np.repeat(zeros.astype(np.float64), G, 1)
    w, x = s * (codes.astype(np.float64) - z), x.astype(np.float64)
    y = x @ w.T
    if bias is not None:
        y = y + bias.astype(np.float64)
    if act == 1:
        y = np.maximum(y, 0)
    elif act == 2:
        y = 0.5 * y * (1 + np.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3)))
    return y, np.abs(x) @ np.abs(w).T, np.abs(x) @ (np.abs(s) * (codes.astype(np.float64) + z)).T
