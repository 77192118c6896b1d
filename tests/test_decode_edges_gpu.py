"""Decode operators at the edges of their number ranges, on the GPU against the float64 oracle.

Tolerances are those of test_decode_gpu.py; where a test adds to one, it says what for."""
import ctypes as C
import os

import numpy as np
import pytest

import spmspm_amd as S
from oracle import decode_oracle as D
from spmspm_amd import api as A
from spmspm_amd import decode as M
from test_decode_gpu import SMALLEST, UNIT, Case, assert_attention, host, to16, torch  # noqa: F401

pytestmark = pytest.mark.gpu


# Sequences of one row each, and of more than 64 rows, run on different kernels; both have the same formula.
FEW, MANY = [(1, 300), (1, 77), (2, 230)], [(100, 300), (80, 80), (90, 230)]


def put_words(c, torch):
    """The case's words, changed by a test, onto the GPU."""
    c.cache.k_words.copy_(torch.from_numpy(c.kw.view(np.int32)))
    c.cache.v_words.copy_(torch.from_numpy(c.vw.view(np.int32)))


def put_values(c, torch):
    put_words(c, torch)
    c.cache.k_codes.copy_(torch.from_numpy(c.kc))
    c.cache.v_codes.copy_(torch.from_numpy(c.vc))


# ---- words of the cache ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("stale", [0x00000001, 0x00007FFF, 0x007FFFFF, 0x00000000, 0x80000001])
@pytest.mark.parametrize("seqs,d", [(FEW, 128), (MANY, 64), (MANY, 96), (MANY, 128)])
def test_attention_does_not_see_small_words_in_hidden_places(torch, seqs, d, stale):
    """Small integers, as reused memory holds them, are subnormal scales: behind the ends of sequences, in absent pages and
    outside a window they change nothing."""
    c = Case(torch, seqs, 4, 2, d, 16, "fp16", seed=d, stale=stale)
    c.table[0, 2], c.table[2, 5] = -1, c.pages + 9
    c.gt = torch.from_numpy(c.table).cuda()
    q, qh = c.queries()
    for window in (0, 40):
        want, mag, lse = c.want(qh, window)
        assert np.isfinite(want).all()
        got, gl = c.attend(q, window=window, return_lse=True)
        assert_attention(got, want, mag, "fp16")
        assert np.allclose(host(gl), lse, rtol=1e-5, atol=2e-4)
    # every place before a window, with the words of places that are seen kept
    written = np.zeros((c.pages, 16), bool)
    for b, (n, L) in enumerate(seqs):
        for p in range(max(0, L - n - 15), L):
            if 0 <= c.table[b, p // 16] < c.pages:
                written[c.table[b, p // 16], p % 16] = True
    for w in (c.kw, c.vw):
        w[~np.broadcast_to(written[:, None, :], w.shape)] = np.uint32(stale)
    put_words(c, torch)
    want, mag, _ = c.want(qh, 16)
    assert_attention(c.attend(q, window=16), want, mag, "fp16")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("seqs", [FEW, MANY])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_attention_over_scales_of_zero_and_below_the_normal_numbers(torch, d, seqs, dtype):
    """A word of 0, which a new cache holds, is a vector of zeros for one row and for many; scales below 2^-126 count as 0 in
    the values, at most 15 2^-126 away."""
    c = Case(torch, seqs, 4, 2, d, 16, dtype, seed=d)
    some = c.rng.random(c.vw.shape) < 0.3
    c.vw[some] = c.rng.choice(np.array([0, 0, 1, 0x7FFF, 0x12345, 0x7FFFFF], np.uint32), int(some.sum()))
    some = c.rng.random(c.kw.shape) < 0.1
    c.kw[some] = c.rng.choice(np.array([0, 0x12345], np.uint32), int(some.sum()))
    put_words(c, torch)
    q, qh = c.queries()
    want, mag, lse = c.want(qh)
    got, gl = c.attend(q, return_lse=True)
    bound = (2.0 ** -11 + 2.0 ** -13) * mag + 1.01 * UNIT[dtype] * np.abs(want) + max(SMALLEST[dtype], 15 * 2.0 ** -126)
    assert (np.abs(host(got) - want) <= bound).all()
    assert np.allclose(host(gl), lse, rtol=1e-5, atol=2e-4)
    c.vw[:], c.kw[:] = 0, 0
    put_words(c, torch)
    _, _, lse = c.want(qh)
    got, gl = c.attend(q, return_lse=True)
    assert (host(got) == 0).all()
    assert np.allclose(host(gl), lse, rtol=1e-5, atol=2e-4)
    # the read-back of the same places
    k, v = S.kv4_gather(c.cache, c.gt, c.gl, cu_tokens=c.gcu, total_tokens=c.tokens, dtype=q.dtype)
    assert (host(k) == 0).all() and (host(v) == 0).all()


# ---- scores ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("many", [False, True])
def test_attention_of_scores_whose_float32_neighbours_are_far_apart(torch, many):
    """Scores of 2^24 to 2^29, a few units of float32's last place apart, the larger one later: the reference of the
    exponentials is a rounded number there, and a probability relative to it must still fit 16 bits.  Key/value heads differ in
    the values' scale, which moves the rounding."""
    hkv, d, page = 32, 64, 16
    seqs, page2 = ([(70, 120)], 4) if many else ([(1, 140)], 8)  # within one split, and one wave
    for top in (2.0 ** 14, 2.0 ** 15, 1.25 * 2.0 ** 13, 1.75 * 2.0 ** 14):
        for word in (64.0, 128.0, 200.0, 512.0):
            c = Case(torch, seqs, hkv, hkv, d, page, "bf16")
            c.kc[:], c.kw[:] = 0, np.float32(1).view(np.uint32)  # a score of 0
            first, later = (c.table[0, 0], slice(None), 0), (c.table[0, page2], slice(None), 2)  # places 0, and 66 or 130
            c.kc[first][:, 0] = 14  # element 0
            c.kw[first] = np.float32(word).view(np.uint32)
            c.kc[later][:] = 0x11
            c.kc[later][:, 0] = 0x1F  # 15 - 1, the others 1 - 1
            c.kw[later] = np.float32(word).view(np.uint32) + np.uint32(1)
            for h in range(hkv):  # values' scales just below powers of two
                c.vw[:, h] = np.float32(2.0 ** (h - 16)).view(np.uint32) - np.uint32(16)
            put_values(c, torch)
            q = np.zeros((c.tokens, hkv, d))
            q[..., 0] = top
            q, qh = to16(torch, q, "bf16")
            scale = float(np.log(2.0))
            _, mag, _ = c.want(qh, scale=scale)
            got = host(c.attend(q, scale=scale))
            # between the two values, whichever way the scores were rounded
            v = D.decode64(c.vc, c.vw)
            a, b = v[first], v[later]
            lo, hi = np.minimum(np.minimum(a, b), 0), np.maximum(np.maximum(a, b), 0)
            room = 1.02 * 2.0 ** -8 * np.maximum(np.abs(lo), np.abs(hi))
            assert np.isfinite(got).all(), (top, word)
            assert ((got >= lo - room) & (got <= hi + room)).all(), (top, word)


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_scores_far_below_zero(torch, d, many):
    """The only key that a row sees has a score of -2^100: its probability is 1 all the same."""
    c = Case(torch, [(80, 80)] if many else [(1, 1), (1, 1)], 2, 2, d, 16, "bf16", seed=d)
    q = np.zeros((c.tokens, 2, d))
    rows = [0] if many else [0, 1]
    for i, t in enumerate(rows):
        k = D.decode64(c.kc, c.kw)[c.table[i, 0], :, 0]
        q[t] = -k * 2.0 ** 105
    q, _ = to16(torch, q, "bf16")
    got, lse = c.attend(q, return_lse=True)
    for i, t in enumerate(rows):
        v = D.decode64(c.vc, c.vw)[c.table[i, 0], :, 0]
        assert (np.abs(host(got)[t] - v) <= (2.0 ** -8 + 2.0 ** -10) * np.abs(v) + 2.0 ** -10 * np.abs(v).max()).all()
        assert np.isfinite(host(lse)[t]).all() and (host(lse)[t] < -2.0 ** 100).all()


@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("top", [2.0 ** 104, 2.0 ** 118, 3.3895e38])
def test_attention_of_chunks_with_the_largest_queries(torch, d, top):
    """One element of a row up to the largest finite bf16: the rows beside it are what they would be without it."""
    c = Case(torch, [(100, 300), (96, 97)], 4, 2, d, 32, "bf16", seed=d)
    x = c.rng.standard_normal((c.tokens, c.hq, d))
    x[150, 0] *= 2.0 ** -40
    x[151, 0] *= 2.0 ** -100
    big = np.zeros((c.tokens, c.hq), bool)
    for t, h, e in ((3, 0, 7), (60, 3, d - 1), (140, 1, 0)):
        x[t, h, e], big[t, h] = top, True
    q, qh = to16(torch, x, "bf16")
    assert np.isfinite(qh).all()
    want, mag, lse = c.want(np.where(big[..., None], 0, qh))
    got, gl = c.attend(q, return_lse=True)
    got, gl = host(got), host(gl)
    bound = (2.0 ** -11 + 2.0 ** -13) * mag + 1.01 * UNIT["bf16"] * np.abs(want)
    assert (np.abs(got - want)[~big] <= bound[~big]).all()
    assert np.allclose(gl[~big], lse[~big], rtol=1e-5, atol=2e-4)
    if top < 2.0 ** 120:  # the row itself looks at one key alone: its scores fit float32
        clean = np.where(big[..., None], np.where(np.abs(qh) > 1e9, 2.0 ** 20, 0), 0)
        one, _, _ = c.want(clean)
        assert (np.abs(got - one)[big] <= 2.0 ** -7 * np.abs(one[big]) + 2.0 ** -9 * np.abs(one).max()).all()


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("top", [2.0 ** 90, 2.0 ** 104, 2.0 ** 118])
def test_attention_of_single_tokens_with_the_largest_queries(torch, d, top):
    """Rows whose scores fit float32 look at one key alone; small rows in the same block stay as they are."""
    c = Case(torch, [(1, 300), (3, 77), (1, 1)], 4, 2, d, 16, "bf16", seed=d)
    x = c.rng.standard_normal((c.tokens, c.hq, d))
    size = np.ones((c.tokens, c.hq, 1))
    size[0, 1], size[2, 0], size[3, 3], size[4] = top, top, 2.0 ** -60, top
    q, qh = to16(torch, x * size, "bf16")
    big = (size > 1)[..., 0]
    want, mag, lse = c.want(np.where(big[..., None], 0, qh))
    got, gl = c.attend(q, return_lse=True)
    got, gl = host(got), host(gl)
    bound = (2.0 ** -11 + 2.0 ** -13) * mag + 1.01 * UNIT["bf16"] * np.abs(want)
    assert (np.abs(got - want)[~big] <= bound[~big]).all()
    assert np.allclose(gl[~big], lse[~big], rtol=1e-5, atol=2e-4)
    one = c.want(np.where(size > 1, qh / top * 2.0 ** 20, 0))[0]
    assert (np.abs(got - one)[big] <= 2.0 ** -7 * np.abs(one[big]) + 2.0 ** -9 * np.abs(one).max()).all()
    assert np.isfinite(gl[big]).all()


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_attention_scores_have_the_bits_of_float32(torch, d, many):
    """Rows that see one key and whose queries have one element: the log of the sum is the score.  Roundings: three of the score's
    2^-24, below 1; the score with the values' exponent, below 4; the reference 7 below it, below 8; two of the logarithm's sum."""
    c = Case(torch, [(70, 70)] * 3 if many else [(1, 5)] * 200, 8, 4, d, 16, "bf16", seed=d)
    c.vc, c.vw = D.encode((c.rng.uniform(0.5, 1.9, c.vw.shape + (1,)) * c.rng.choice((-7.5, 0, 7.5), c.vw.shape + (d,))).astype(np.float32))
    c.vc = D.pack(c.vc)
    put_values(c, torch)
    q = np.zeros((c.tokens, 8, d))
    at = c.rng.integers(0, d, (c.tokens, 8, 1))
    np.put_along_axis(q, at, c.rng.uniform(-0.5, 0.5, at.shape), 2)
    q, qh = to16(torch, q, "bf16")
    _, lse = c.attend(q, window=1, return_lse=True)
    _, _, want = c.want(qh, 1)
    assert np.abs(want).max() < 0.7
    assert np.abs(host(lse) - want).max() <= 1.5 * 2.0 ** -20


# ---- linears ---------------------------------------------------------------------------------------------------------------

def linear_case(torch, M, K, N, G, dtype, seed=0):
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16, (M, K)).astype(np.uint8)
    zeros = rng.integers(0, 16, (M, K // G)).astype(np.uint8)
    scales, sh = to16(torch, rng.uniform(0.001, 0.01, (M, K // G)) * np.where(rng.random((M, K // G)) < 0.2, -1, 1), dtype)
    g = lambda a: torch.from_numpy(a).cuda()
    return rng, codes, sh, zeros, S.W4Linear(g(codes), scales, g(zeros))


LINEARS = [(40, 256, 6, 32), (40, 384, 6, 64), (40, 384, 16, 128), (40, 8320, 50, 32), (640, 8192, 64, 64), (33, 16512, 20, 128)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,K,N,G", LINEARS)
def test_linear_with_infinities_in_x(torch, M, K, N, G, dtype):
    """An infinity times a weight is one of the weight's sign, and NaN for a weight of zero; a NaN spoils its row.  The rows
    beside them do not change by a bit."""
    rng, codes, sh, zeros, layer = linear_case(torch, M, K, N, G, dtype, M + K)
    x, xh = to16(torch, rng.standard_normal((N, K)), dtype)
    ref = layer(x)
    bad = sorted({0, N // 2, N - 1})
    xh[bad[0], K // 3], xh[bad[1], K - 1] = np.inf, -np.inf
    xh[bad[2], 5] = np.nan
    x, xh = to16(torch, xh, dtype)
    got = layer(x)
    fine = [n for n in range(N) if n not in bad]
    assert torch.equal(got[fine], ref[fine])
    w = np.repeat(sh.astype(np.float64), G, 1) * (codes.astype(np.float64) - np.repeat(zeros, G, 1))
    with np.errstate(all="ignore"):
        want = np.stack([(w * xh[n].astype(np.float64)).sum(1) for n in bad])
    got = host(got[bad])
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isinf(want).any()
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])


@pytest.mark.parametrize("M,K,N,G", LINEARS)
def test_linear_with_the_largest_activations(torch, M, K, N, G):
    """bf16 rows whose results are finite and whose sums with the codes as they stand are not."""
    rng, codes, sh, zeros, layer = linear_case(torch, M, K, N, G, "bf16", M + K + 1)
    x = rng.standard_normal((N, K))
    x[N - 1] *= 2e37 / np.sqrt(K / 256)
    x[0] *= 3e36
    x, xh = to16(torch, x, "bf16")
    y, small, _ = D.linear(xh, codes, sh, zeros)
    assert (np.abs(y) < 3.3e38).all()
    got = host(layer(x))
    # rounded sums of the products themselves, and of x (16 + w) where those fit: 32 / |w - z| times as large at most
    big = np.abs(xh.astype(np.float64)) @ (32 * np.repeat(np.abs(sh.astype(np.float64)), G, 1)).T
    bound = (48 + K // G) * 2.0 ** -24 * big + 1.01 * UNIT["bf16"] * np.abs(y)
    assert (np.abs(got - y) <= bound).all()


# Every kernel of the linears at small sizes: the tests' build of the library takes a plan.

@pytest.fixture
def set_plan(monkeypatch):
    lib = C.CDLL(os.path.join(os.path.dirname(S.library_path()), "libSpMM_API_variants.so"))
    monkeypatch.setattr(A, "library", lambda: lib)
    monkeypatch.setattr(M, "_lib", None)
    yield lib.W4_Debug_SetPlan
    lib.W4_Debug_SetPlan(0, 0, 0)


def check_linear(torch, M_, N, K, G, dtype, act, splits):
    """Against float64, an infinity in a row of X and the call's repetition among it."""
    rng, codes, sh, zeros, _ = linear_case(torch, M_, K, N, G, dtype, K + splits)
    g = lambda a: torch.from_numpy(a).cuda()
    bias, bh = to16(torch, rng.standard_normal(M_), dtype)
    scales, _ = to16(torch, sh, dtype)
    layer = S.W4Linear(g(codes), scales, g(zeros), bias=bias, activation=act)
    need = M._library().W4_WorkspaceBytes(M_, N, K, G)
    assert need == (4 * splits * N * (-(-M_ // 16) * 16) if splits > 1 else 0)
    x, xh = to16(torch, rng.standard_normal((N, K)), dtype)
    y, _, big = D.linear(xh, codes, sh, zeros, bh, act)
    got = layer(x)
    # sums of x (16 + w) and, taken off, x (16 + z): 36 rounded additions a group at most in the matrix cores and 12 beside them,
    # one for each group, and the shares' and waves' sums
    s = np.repeat(np.abs(sh.astype(np.float64)), G, 1)
    big = big + np.abs(xh.astype(np.float64)) @ (32 * s).T + np.abs(bh)
    slope = 1.13 if act == 2 else 1.0
    bound = slope * (48 + K // G + splits) * 2.0 ** -24 * big + (1.01 * UNIT[dtype] + (1e-5 if act == 2 else 0)) * np.abs(y) \
        + SMALLEST[dtype] + (1e-6 if act == 2 else 0)
    d = np.abs(host(got) - y)
    assert (d <= bound).all(), (np.max(d / bound), np.argwhere(d > bound)[:4].tolist())
    assert torch.equal(got, layer(x))
    xh[N - 1, K // 2] = np.inf
    x, xh = to16(torch, xh, dtype)
    again = layer(x)
    assert torch.equal(again[:N - 1], got[:N - 1])
    with np.errstate(all="ignore"):
        w = np.repeat(sh.astype(np.float64), G, 1) * (codes.astype(np.float64) - np.repeat(zeros, G, 1))
        y = (w * xh[N - 1].astype(np.float64)).sum(1)
    want = np.where(np.isnan(y), np.nan, np.where(y > 0, np.inf, 0 if act == 1 else np.nan if act == 2 else -np.inf))
    assert np.array_equal(host(again[N - 1]), want, equal_nan=True)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("G,tiles", [(32, 1), (32, 2), (32, 3), (32, 4), (64, 1), (64, 2), (64, 3), (64, 4), (64, 5), (128, 1), (128, 2),
                                     (128, 3), (128, 4), (128, 5), (128, 6), (128, 7)])
def test_linear_of_few_columns_with_every_number_of_row_tiles(torch, set_plan, G, tiles, dtype):
    """Rows that end inside a tile and inside a workgroup's tiles, blocks of K that end a wave's turn at either set of registers, the
    last one not whole, and shares of which one is shorter or empty."""
    for N, blocks, splits, act in ((3, 5, 1, 0), (18, 19, 1, 2), (16, 19, 3, 1), (1, 36, 7, 0), (20, 2, 4, 0)):
        assert set_plan(tiles, 0, splits) == 0
        check_linear(torch, 16 * (2 * tiles - 1) - 5, N, 128 * blocks - (G if G < 128 else 0), G, dtype, act, splits)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("tiles", [2, 4])
def test_linear_of_many_columns_with_every_number_of_column_tiles(torch, set_plan, tiles, G, dtype):
    """One to eight blocks of K for a workgroup, so that a span of two blocks ends at either; shares of odd numbers of blocks; columns
    that end inside a workgroup's."""
    rows = 300
    for N, blocks, splits, act in ((16 * tiles, 1, 1, 0), (16 * tiles + 5, 2, 1, 1), (17, 7, 1, 2), (16 * tiles - 1, 8, 1, 0),
                                   (16 * tiles, 9, 3, 0), (16 * tiles + 1, 10, 4, 2), (33, 5, 2, 1), (20, 3, 5, 0)):
        assert set_plan(0, tiles, splits) == 0
        check_linear(torch, rows, N, 128 * blocks - (G if G < 128 else 0), G, dtype, act, splits)


@pytest.mark.parametrize("M_,N,K,G,dtype", [(512, 16, 32768, 64, "fp16"), (528, 5, 32768, 128, "bf16"), (640, 64, 8192, 64, "bf16"),
                                            (1024, 33, 8192, 64, "fp16"), (529, 50, 25184, 32, "bf16")])
def test_linear_with_a_k_that_the_library_splits(torch, M_, N, K, G, dtype):
    need = M._library().W4_WorkspaceBytes(M_, N, K, G)
    assert need > 0
    check_linear(torch, M_, N, K, G, dtype, 1, need // (4 * N * (-(-M_ // 16) * 16)))


# ---- calls -----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("seqs", [[(5, 3), (40, 33), (1, 20)], [(120, 60), (90, 33), (97, 128)]])
def test_attention_with_the_widest_window(torch, seqs, d):
    """The largest int as a window, over tokens that lie before their sequence's start: it hides nothing."""
    c = Case(torch, seqs, 4, 2, d, 16, "fp16", seed=d)
    q, qh = c.queries()
    want, mag, lse = c.want(qh)
    for window in (2 ** 31 - 1, 2 ** 31 - 60, 1 << 30):
        got, gl = c.attend(q, window=window, return_lse=True)
        assert_attention(got, want, mag, "fp16")
        assert np.array_equal(np.isneginf(host(gl)), np.isneginf(lse))


def test_strides_of_dimensions_of_one_do_not_matter(torch):
    """One token, one head, one page: views whose stride there is any number."""
    c = Case(torch, [(1, 20)], 4, 2, 64, 32, "fp16")
    q, _ = c.queries()
    ref = c.attend(q)
    buf = torch.zeros(600, dtype=torch.float16, device="cuda")
    odd = buf.as_strided((1, 4, 64), (333, 64, 1))
    odd.copy_(q)
    assert torch.equal(c.attend(odd), ref)
    table = torch.as_strided(c.gt, (1, 1), (1, 7))
    assert torch.equal(S.kv4_attention(odd, c.cache, table, c.gl), ref)
    k, v = S.kv4_gather(c.cache, table, c.gl)
    c1 = Case(torch, [(1, 20), (1, 9), (1, 32)], 1, 1, 64, 32, "fp16")
    q, _ = c1.queries()
    ref = c1.attend(q)
    one = torch.empty(3 * 64, dtype=torch.float16, device="cuda").as_strided((3, 1, 64), (64, 13, 1))
    one.copy_(q)
    assert torch.equal(S.kv4_attention(one, c1.cache, c1.gt.t().contiguous().t(), c1.gl), ref)
    S.kv4_append(c.cache, odd[:, :2], odd[:, 2:], table, c.gl)
    back = S.kv4_gather(c.cache, table, c.gl)
    want = S.kv4_gather(c.cache, c.gt, c.gl)
    assert torch.equal(back[0], want[0]) and torch.equal(back[1], want[1]) and not torch.equal(back[0], k)


def test_attention_takes_any_int_as_a_window_and_a_bound(torch):
    """Numbers past 32 bits hide nothing and bound nothing; they are not cut off to their lowest bits."""
    c = Case(torch, [(1, 77), (2, 30)], 4, 2, 64, 16, "fp16")
    q, _ = c.queries()
    ref = c.attend(q)
    for many in (2 ** 31, 2 ** 32 + 5, 2 ** 40 + 1, 2 ** 63 - 1):
        assert torch.equal(c.attend(q, window=many), ref)
        assert torch.equal(c.attend(q, max_len=many), ref)
    with pytest.raises(ValueError):
        S.kv4_gather(c.cache, c.gt, c.gl, cu_tokens=c.gcu, total_tokens=2 ** 32 + 3)


# ---- work that is dealt in other ways at larger sizes ----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("hq,hkv,seqs,window", [(8, 2, [(1, 2100), (1, 700), (1, 1)], 0), (8, 1, [(3, 1500), (1, 40)], 0),
                                                (6, 2, [(9, 1300), (6, 33), (3, 2)], 1100), (8, 2, [(11, 1800), (13, 64)], 0),
                                                (4, 2, [(60, 1500), (20, 20)], 0), (4, 1, [(30, 1200), (5, 9)], 1100)])
def test_attention_with_keys_split_among_workgroups(torch, hq, hkv, seqs, window, d, dtype):
    """Every kernel with more than one share of the keys, some of them empty; rows of no sequence at the end."""
    tail = 2 if sum(n for n, _ in seqs) > len(seqs) else 0
    c = Case(torch, seqs, hq, hkv, d, 16, dtype, seed=d + hq, tail=tail, width=1300)
    need = M._library().KV4_AttentionWorkspaceBytes(c.cache._desc, M._batch(c.cache, c.gt, c.gl, c.gcu, c.tokens), hq, window, 0)
    splits = need // (4 * c.tokens * hq * (d + 2))
    assert splits > 1 and need == 4 * c.tokens * hq * (d + 2) * splits
    q, qh = c.queries(1.5)
    want, mag, lse = c.want(qh, window)
    got, gl = c.attend(q, window=window, return_lse=True)
    assert_attention(got, want, mag, dtype)
    live = np.isfinite(lse)
    assert np.array_equal(np.isneginf(host(gl)), ~live) and np.allclose(host(gl)[live], lse[live], rtol=1e-5, atol=2e-4)
    assert torch.equal(got, c.attend(q, window=window))


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("d,rot,interleaved", [(64, 64, False), (64, 20, False), (96, 96, True), (128, 64, False), (128, 10, True),
                                               (256, 256, False), (128, 0, False)])
def test_append_and_gather_of_long_prompts(torch, d, rot, interleaved, odd):
    """So many tokens that a group of lanes takes several of a token's vectors, the next one's loads ahead of the present one's work;
    rows at odd addresses are read element by element."""
    hq, hkv, page, dtype = (24 if rot else 0), 8, 32, "bf16" if odd else "fp16"
    lens, rng = [5003, 2999], np.random.default_rng(d + rot)
    T, heads = sum(lens), hq + 2 * hkv
    groups = {64: 32, 96: 16, 128: 16, 256: 8}[d]
    assert heads * -(-T // groups) // 2048 >= 2 and 2 * hkv * -(-T // groups) // 2048 >= 1
    flat, fh = to16(torch, rng.standard_normal(T * heads * d + 1), dtype)
    rows, h = flat[odd:T * heads * d + odd].view(T, heads, d), fh[odd:T * heads * d + odd].reshape(T, heads, d)
    counts = [-(-n // page) for n in lens]
    order = rng.permutation(sum(counts) + 2).astype(np.int32)
    table = np.full((2, max(counts)), -1, np.int32)
    table[0, :counts[0]], table[1, :counts[1]] = order[:counts[0]], order[counts[0]:sum(counts)]
    g = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    cache = S.KV4Cache(len(order), page, hkv, d)
    batch = (g(table), g(np.array(lens, np.int32)), g(np.array([0, lens[0], T], np.int32)))
    turn = rng.uniform(-1, 1, (max(lens), rot)).astype(np.float32)
    q = S.kv4_append(cache, rows[:, hq:hq + hkv], rows[:, hq + hkv:], *batch, q=rows[:, :hq] if rot else None,
                     rotation=g(turn) if rot else None, interleaved=interleaved)
    place = np.concatenate([np.arange(n) for n in lens])
    pages, slot = table[np.repeat([0, 1], lens), place // page], place % page
    k = h[:, hq:hq + hkv]
    if rot:
        k = D.rotate(k, turn, place, interleaved)
        want = D.rotate(h[:, :hq], turn, place, interleaved)
        assert torch.equal(q.cpu(), torch.from_numpy(want).to(q.dtype))
    back = S.kv4_gather(cache, *batch, total_tokens=T, dtype=rows.dtype)
    for x, codes, words, read in ((k, cache.k_codes, cache.k_words, back[0]), (h[:, hq + hkv:], cache.v_codes, cache.v_words, back[1])):
        wc, ww = D.encode(x)
        wc = D.pack(wc)
        assert np.array_equal(codes.cpu().numpy()[pages, :, slot], wc)
        assert np.array_equal(words.cpu().numpy().view(np.uint32)[pages, :, slot], ww)
        assert torch.equal(read.cpu(), torch.from_numpy(D.decode32(wc, ww)).to(read.dtype))
