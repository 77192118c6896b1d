"""Decode operators on the GPU against the CPU oracle: the 4-bit cache, its attention, 4-bit linears.

Tolerances.  The cache's codes and words, and the rotated queries, are float32 arithmetic rounded operation by operation: equal.
Attention: every probability is rounded once to 11 bits before the product with the values, 2^-11 of sum p |v| at most; its
exponent carries an error of a few units in the last place of a float32 of magnitude up to 2^8, below 2^-13 of the probability;
the output is rounded once.  Linears: sums of at most 36 rounded additions per group in the matrix cores, one per group and
sixteen when the waves are joined, 2^-24 each, and a scale changed by less than 2^-19; the output is rounded once."""
import numpy as np
import pytest

import spmspm_amd as S
from oracle import decode_oracle as D

pytestmark = pytest.mark.gpu

UNIT = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
SMALLEST = {"fp16": 2.0 ** -25, "bf16": 0.0}


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def ttype(torch, name):
    return torch.float16 if name == "fp16" else torch.bfloat16


def to16(torch, x, name):
    """numpy float -> tensor on the GPU, and its values as float32."""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(ttype(torch, name))
    return t.cuda(), t.float().numpy()


def host(t):
    return t.detach().cpu().double().numpy()


class Case:
    """Sequences of given (new, length) over a cache whose pages are in random order, filled by the oracle's encoding."""

    def __init__(self, torch, seqs, hq, hkv, d, page, dtype, seed=0, spread=1.0, stale="random", width=None, tail=0):
        rng = self.rng = np.random.default_rng(seed)
        self.torch, self.hq, self.hkv, self.d, self.page, self.dtype, self.seqs = torch, hq, hkv, d, page, dtype, seqs
        counts = [max(1, -(-max(L, 0) // page)) for _, L in seqs]
        self.pages = sum(counts) + 2
        order = rng.permutation(self.pages)
        self.table = np.full((len(seqs), width or max(counts)), -1, np.int32)
        at = 0
        for b, c in enumerate(counts):
            c = min(c, self.table.shape[1])
            self.table[b, :c] = order[at:at + c]
            at += c
        shape = (self.pages, hkv, page, d)
        # distinct scales per vector, over a few powers of two
        size = np.exp2(rng.uniform(-3, 2, shape[:3] + (1,)))
        self.kc, self.kw = D.encode((rng.standard_normal(shape) * spread).astype(np.float32))
        self.vc, self.vw = D.encode((rng.standard_normal(shape) * size + 0.3).astype(np.float32))
        self.kc, self.vc = D.pack(self.kc), D.pack(self.vc)
        if stale != "random":  # whatever no sequence's token wrote
            written = np.zeros((self.pages, page), bool)
            for b, (_, L) in enumerate(seqs):
                for p in range(max(min(L, self.table.shape[1] * page), 0)):
                    written[self.table[b, p // page], p % page] = True
            for w, value in ((self.kw, stale), (self.vw, stale)):
                w[~np.broadcast_to(written[:, None, :], w.shape)] = np.uint32(value)
        self.lens = np.array([L for _, L in seqs], np.int32)
        self.cu = np.concatenate(([0], np.cumsum([n for n, _ in seqs]))).astype(np.int32)
        self.tokens = int(self.cu[-1]) + tail
        g = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        self.cache = S.KV4Cache.from_tensors(g(self.kc), g(self.kw.view(np.int32)), g(self.vc), g(self.vw.view(np.int32)))
        self.gt, self.gl = g(self.table), g(self.lens)
        self.gcu = None if all(n == 1 for n, _ in seqs) and not tail else g(self.cu)

    def queries(self, scale=1.0):
        return to16(self.torch, self.rng.standard_normal((self.tokens, self.hq, self.d)) * scale, self.dtype)

    def want(self, q, window=0, scale=None):
        return D.attention(q, self.kc, self.kw, self.vc, self.vw, self.table, self.lens, self.cu,
                           self.d ** -0.5 if scale is None else scale, window)

    def attend(self, q, **kw):
        return S.kv4_attention(q, self.cache, self.gt, self.gl, cu_tokens=self.gcu, **kw)


def assert_attention(got, want, mag, dtype, what=""):
    got = host(got)
    bound = (2.0 ** -11 + 2.0 ** -13) * mag + 1.01 * UNIT[dtype] * np.abs(want) + SMALLEST[dtype]
    bad = np.abs(got - want) > bound
    same_nan = np.isnan(got) == np.isnan(want)
    assert same_nan.all(), f"{what}: NaN in other places"
    assert not bad.any(), f"{what}: worst {np.nanmax(np.abs(got - want) / bound)} of the bound at {np.argwhere(bad)[:4].tolist()}"


# ---- append and gather -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("rot,interleaved", [(0, False), (32, True), (64, False), (20, False), (10, True), (-1, False)])
def test_append_encodes_rotates_and_reads_back(torch, d, rot, interleaved):
    rot = d if rot < 0 else rot
    dtype = "fp16" if (d + rot) % 64 else "bf16"
    c = Case(torch, [(3, 40), (1, 1), (17, 17), (2, 130), (0, 9)], 6, 2, d, 16, dtype, seed=d + rot, tail=2)
    T = c.tokens
    qkv, qkv_h = to16(torch, c.rng.standard_normal((T, 10, d)) * 3, dtype)
    q, k, v = qkv[:, :6], qkv[:, 6:8], qkv[:, 8:]
    table = c.rng.uniform(-1, 1, (140, rot)).astype(np.float32) if rot else None
    out = S.kv4_append(c.cache, k, v, c.gt, c.gl, cu_tokens=c.gcu, q=q if rot else None,
                       rotation=None if not rot else torch.from_numpy(table).cuda(), interleaved=interleaved)
    gk, gv = S.kv4_gather(c.cache, c.gt, c.gl, cu_tokens=c.gcu, total_tokens=T, dtype=ttype(torch, dtype))
    torch.cuda.synchronize()
    seq, place = D.places(c.lens, c.cu, T)
    live = seq >= 0
    want_k, want_q = qkv_h[:, 6:8].copy(), qkv_h[:, :6].copy()
    if rot:
        want_k[live] = D.rotate(want_k[live], table, place[live], interleaved)
        want_q[live] = D.rotate(want_q[live], table, place[live], interleaved)
        assert torch.equal(out.cpu(), torch.from_numpy(want_q).to(ttype(torch, dtype)))
    kc, kw, vc, vw = c.kc.copy(), c.kw.copy(), c.vc.copy(), c.vw.copy()
    for t in np.flatnonzero(live):
        page, slot = c.table[seq[t], place[t] // 16], place[t] % 16
        codes, kw[page, :, slot] = D.encode(want_k[t])
        kc[page, :, slot] = D.pack(codes)
        codes, vw[page, :, slot] = D.encode(qkv_h[t, 8:])
        vc[page, :, slot] = D.pack(codes)
    # the whole cache: the tokens' slots as encoded, everything else untouched
    assert np.array_equal(c.cache.k_codes.cpu().numpy(), kc) and np.array_equal(c.cache.v_codes.cpu().numpy(), vc)
    assert np.array_equal(c.cache.k_words.cpu().numpy().view(np.uint32), kw)
    assert np.array_equal(c.cache.v_words.cpu().numpy().view(np.uint32), vw)
    for got, codes, words in ((gk, kc, kw), (gv, vc, vw)):
        want = np.zeros((T, 2, d), np.float32)
        for t in np.flatnonzero(live):
            page, slot = c.table[seq[t], place[t] // 16], place[t] % 16
            want[t] = D.decode32(codes[page, :, slot], words[page, :, slot])
        assert torch.equal(got.cpu(), torch.from_numpy(want).to(ttype(torch, dtype)))


def test_gather_rounds_the_float32_product(torch):
    """Enough values that one lies where rounding once and rounding twice differ (one in a million does)."""
    rng = np.random.default_rng(3)
    for dtype in ("fp16", "bf16"):
        pages, hkv, P, d = 64, 8, 64, 128
        kc = rng.integers(0, 256, (pages, hkv, P, d // 2)).astype(np.uint8)
        kw = (rng.uniform(0.01, 1, (pages, hkv, P)).astype(np.float32).view(np.uint32))
        g = lambda a: torch.from_numpy(a).cuda()
        cache = S.KV4Cache.from_tensors(g(kc), g(kw.view(np.int32)), g(kc), g(kw.view(np.int32)))
        table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
        T = pages * P
        n = torch.tensor([T], dtype=torch.int32, device="cuda")
        k, v = S.kv4_gather(cache, table, n, cu_tokens=torch.tensor([0, T], dtype=torch.int32, device="cuda"),
                            total_tokens=T, dtype=ttype(torch, dtype))
        want = torch.from_numpy(D.decode32(kc, kw).transpose(0, 2, 1, 3).reshape(T, hkv, d)).to(ttype(torch, dtype))
        assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)


def test_append_special_values(torch):
    """Zeros, one sign, tiny and huge vectors, infinities and NaN: each stays within its own token and head."""
    for dtype in ("fp16", "bf16"):
        x = np.random.default_rng(1).standard_normal((16, 2, 64)).astype(np.float32)
        x[0], x[1, 0], x[2], x[3] = 0, np.abs(x[1, 0]), -np.abs(x[2]), x[3] * 1e-6
        x[4] *= 6e4 / np.abs(x[4]).max() if dtype == "fp16" else 3e38 / np.abs(x[4]).max()
        x[5, 0, 7], x[6, 1, 63], x[7, 0, 0], x[8] = np.inf, -np.inf, np.nan, -0.0
        x[9] = x[9] * 1e-38 if dtype == "bf16" else 6e-8
        x[10] = 5.0
        c = Case(torch, [(16, 16)], 2, 2, 64, 16, dtype)
        t, h = to16(torch, x, dtype)
        S.kv4_append(c.cache, t, t, c.gt, c.gl, cu_tokens=c.gcu)
        codes, words = D.encode(h)
        page = c.table[0, 0]
        assert np.array_equal(c.cache.v_words[page].cpu().numpy().view(np.uint32), words.T)
        assert np.array_equal(c.cache.v_codes[page].cpu().numpy(), D.pack(codes).transpose(1, 0, 2))
        assert np.array_equal(c.cache.k_words[page].cpu().numpy().view(np.uint32), words.T)
        k, _ = S.kv4_gather(c.cache, c.gt, c.gl, cu_tokens=c.gcu, total_tokens=16, dtype=ttype(torch, dtype))
        nan = torch.isnan(k).cpu().numpy()
        want = np.zeros_like(nan)
        want[5, 0] = want[6, 1] = want[7, 0] = True
        assert np.array_equal(nan, want)


def test_append_ignores_tokens_without_a_place(torch):
    c = Case(torch, [(3, 2), (2, 0), (2, 40), (1, 5)], 2, 2, 64, 16, "fp16", width=2)  # places -1, -2.., past the table
    c.table[3, 0] = c.pages  # a page outside the cache
    c.gt = torch.from_numpy(c.table).cuda()
    t, h = to16(torch, c.rng.standard_normal((8, 2, 64)), "fp16")
    before = [x.clone() for x in (c.cache.k_codes, c.cache.k_words, c.cache.v_codes, c.cache.v_words)]
    rot = torch.rand(64, 16, device="cuda")
    q = S.kv4_append(c.cache, t, t, c.gt, c.gl, cu_tokens=c.gcu, q=t, rotation=rot)
    k, v = S.kv4_gather(c.cache, c.gt, c.gl, cu_tokens=c.gcu, total_tokens=8)
    after = [x.cpu().numpy() for x in (c.cache.k_codes, c.cache.k_words, c.cache.v_codes, c.cache.v_words)]
    page = c.table[0, 0]
    for a, b in zip(after, before):
        b = b.cpu().numpy()
        changed = a != b
        changed[page, :, 0:2] = False  # sequence 0's places 0 and 1
        assert not changed.any()
    zero = np.ones(8, bool)
    zero[1:3] = False
    assert (k.cpu().numpy()[zero] == 0).all() and (v.cpu().numpy()[zero] == 0).all()
    assert (v.cpu().numpy()[1:3] != 0).any()
    assert torch.equal(q[0], t[0]) and torch.equal(q[3:5], t[3:5])  # no place: unrotated
    # explicit positions rotate them all the same, one outside the rotation's rows gives NaN
    pos = torch.tensor([0, 1, 2, 63, 64, -1, 5, 6], dtype=torch.int32, device="cuda")
    q = S.kv4_append(c.cache, t, t, c.gt, c.gl, cu_tokens=c.gcu, q=t, rotation=rot, positions=pos)
    want = D.rotate(h, rot.cpu().numpy(), pos.cpu().numpy(), False)
    assert np.array_equal(q.cpu().numpy(), want.astype(np.float16), equal_nan=True)
    assert np.isnan(want[4, 0, 0]) and np.isnan(want[5, 0, 0]) and not np.isnan(want[4, 0, 16])


def test_append_unaligned_rows_in_place_and_another_stream(torch):
    c = Case(torch, [(2, 20), (3, 33)], 3, 2, 128, 32, "bf16")
    T, rot = c.tokens, torch.rand(64, 128, device="cuda") * 2 - 1
    flat, _ = to16(torch, c.rng.standard_normal(T * 7 * 131 + 1), "bf16")
    odd = flat[1:].view(T, 7, 131)[:, :, :128]  # rows at odd addresses
    whole = odd.contiguous()
    a = S.kv4_append(c.cache, odd[:, 3:5], odd[:, 5:], c.gt, c.gl, cu_tokens=c.gcu, q=odd[:, :3], rotation=rot)
    first = [x.clone() for x in (c.cache.k_codes, c.cache.k_words, c.cache.v_codes, c.cache.v_words)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    b = S.kv4_append(c.cache, whole[:, 3:5], whole[:, 5:], c.gt, c.gl, cu_tokens=c.gcu, q=whole[:, :3], rotation=rot,
                     stream=side)
    side.synchronize()
    q = whole[:, :3].contiguous()
    S.kv4_append(c.cache, whole[:, 3:5], whole[:, 5:], c.gt, c.gl, cu_tokens=c.gcu, q=q, rotation=rot, q_out=q)
    assert torch.equal(a, b) and torch.equal(a, q)
    for x, y in zip(first, (c.cache.k_codes, c.cache.k_words, c.cache.v_codes, c.cache.v_words)):
        assert torch.equal(x, y)


# ---- attention -------------------------------------------------------------------------------------------------------------

LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200]


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attention_single_tokens_of_every_length(torch, d, page, dtype):
    c = Case(torch, [(1, L) for L in LENGTHS], 6, 2, d, page, dtype, seed=d + page)
    q, qh = c.queries()
    want, mag, lse = c.want(qh)
    got, gl = c.attend(q, return_lse=True)
    assert_attention(got, want, mag, dtype)
    assert np.allclose(host(gl), lse, rtol=1e-5, atol=2e-4)
    # a bound that splits the work differently defines the same result
    assert_attention(c.attend(q, max_len=200), want, mag, dtype)


@pytest.mark.parametrize("share", [1, 2, 7, 8, 16, 17, 32, 33, 71])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_shared_heads(torch, share, d):
    c = Case(torch, [(1, 70), (1, 3), (1, 161)], 2 * share, 2, d, 16, "fp16", seed=share)
    q, qh = c.queries(2.0)
    want, mag, _ = c.want(qh)
    assert_attention(c.attend(q), want, mag, "fp16")


@pytest.mark.parametrize("window", [0, 1, 5, 32, 33, 100])
@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 4), (96, 2, 1), (128, 8, 2), (256, 3, 1)])
def test_attention_several_new_tokens_and_windows(torch, window, d, hq, hkv):
    seqs = [(5, 5), (1, 40), (33, 100), (16, 64), (0, 7), (2, 129), (70, 70)]
    c = Case(torch, seqs, hq, hkv, d, 32, "bf16" if window % 2 else "fp16", seed=window, tail=3)
    q, qh = c.queries(1.5)
    want, mag, lse = c.want(qh, window)
    got, gl = c.attend(q, window=window, return_lse=True)
    assert_attention(got, want, mag, c.dtype)
    assert (host(got)[-3:] == 0).all() and np.isneginf(host(gl)[-3:]).all()
    assert np.allclose(host(gl)[:-3], lse[:-3], rtol=1e-5, atol=2e-4)


@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_a_chunk_with_many_rows(torch, d):
    c = Case(torch, [(150, 400), (97, 97)], 4, 2, d, 64, "bf16", seed=5)
    q, qh = c.queries()
    want, mag, _ = c.want(qh)
    assert_attention(c.attend(q), want, mag, "bf16")
    assert_attention(c.attend(q, max_len=400), want, mag, "bf16")


@pytest.mark.parametrize("splits", [False, True])
def test_attention_rows_that_see_nothing(torch, splits):
    """Empty sequences, more new tokens than the sequence has, a page outside the cache, places past the table."""
    c = Case(torch, [(2, 0), (4, 2), (1, 30), (1, 50), (3, 70)], 4, 2, 64, 16, "fp16", width=4)
    c.table[3, 1], c.table[3, 2] = -1, c.pages + 5
    c.table[2] = -7
    if splits:  # a wide table: the library splits what may be a long cache
        c.table = np.concatenate((c.table, np.full((5, 1200), -1, np.int32)), 1)
        c.table[4, 4] = c.table[0, 0]
    c.gt = torch.from_numpy(c.table).cuda()
    q, qh = c.queries()
    want, mag, lse = c.want(qh)
    got, gl = c.attend(q, return_lse=True)
    assert_attention(got, want, mag, "fp16")
    none = np.isneginf(lse)
    assert none[:2].all() and none[2:4].all() and none[6].all() and not none[7].any()
    assert np.array_equal(np.isneginf(host(gl)), none) and (host(got)[none] == 0).all()


@pytest.mark.parametrize("stale", [0x7FC00000, 0xFFFFFFFF, 0x7F800000, 0xFF800000, 0x80000001, 0x7F7FFFFF, 0])
def test_attention_does_not_see_what_lies_in_hidden_places(torch, stale):
    c = Case(torch, [(1, 1), (1, 30), (20, 61), (1, 45)], 4, 2, 128, 16, "fp16", stale=stale)
    q, qh = c.queries()
    want, mag, _ = c.want(qh)
    assert np.isfinite(want).all()
    assert_attention(c.attend(q), want, mag, "fp16")


@pytest.mark.parametrize("side", ["k", "v"])
def test_attention_nan_token_shows_where_it_is_seen(torch, side):
    """A token held as NaN: rows before it, and rows whose window has left it behind, stay as they are."""
    c = Case(torch, [(64, 64)], 2, 1, 64, 16, "fp16")
    words = (c.kw if side == "k" else c.vw)
    words[c.table[0, 1], 0, 4] = 0x7FC00000  # place 20
    (c.cache.k_words if side == "k" else c.cache.v_words).copy_(torch.from_numpy(words.view(np.int32)))
    (c.kc if side == "k" else c.vc)[c.table[0, 1], 0, 4] = 0
    q, qh = c.queries()
    got = host(c.attend(q, window=10))
    seen = np.zeros(64, bool)
    seen[20:30] = True
    assert np.array_equal(np.isnan(got).all((1, 2)), seen) and np.array_equal(np.isnan(got).any((1, 2)), seen)
    words[c.table[0, 1], 0, 4] = 0x3F800000
    want, mag, _ = c.want(qh, 10)
    keep = ~seen
    assert (np.abs(got - want)[keep] <= ((2.0 ** -11 + 2.0 ** -13) * mag + 2.0 ** -11 * 1.01 * np.abs(want) + 2.0 ** -25)[keep]).all()


def test_attention_infinite_query_spoils_its_own_row_only(torch):
    c = Case(torch, [(6, 50)], 4, 2, 128, 16, "fp16")
    q, _ = c.queries()
    q[1, 0, 5], q[2, 3, 100] = float("inf"), float("nan")
    qh = q.float().cpu().numpy()
    got = host(c.attend(q))
    clean = qh.copy()
    clean[1, 0], clean[2, 3] = 0, 0
    want, mag, _ = c.want(clean)
    bad = np.zeros((6, 4), bool)
    bad[1, 0] = bad[2, 3] = True
    assert np.isnan(got[bad]).all()
    bound = (2.0 ** -11 + 2.0 ** -13) * mag + 2.0 ** -11 * 1.01 * np.abs(want) + 2.0 ** -25
    assert (np.abs(got - want)[~bad] <= bound[~bad]).all()


@pytest.mark.parametrize("qs,ks", [(1e-4, 1.0), (30.0, 1.0), (300.0, 100.0), (1e-3, 1e3)])
def test_attention_magnitudes(torch, qs, ks):
    """Flat and one-hot softmaxes.  Scores of up to thousands carry float32 errors of their own: 2^-20 of their size."""
    c = Case(torch, [(1, 300), (3, 77)], 4, 2, 64, 16, "fp16", spread=ks)
    q, qh = c.queries(qs)
    want, mag, _ = c.want(qh)
    got = host(c.attend(q))
    top = np.abs(qh).max() * 64 * ks * 5 / 8
    bound = (2.0 ** -11 + 2.0 ** -13 + top * 2.0 ** -20) * mag + 2.0 ** -11 * 1.01 * np.abs(want) + 2.0 ** -25
    assert (np.abs(got - want) <= bound).all()


def test_attention_values_of_very_different_sizes(torch):
    """A probable token with tiny values beside an improbable one with huge values."""
    c = Case(torch, [(1, 64)], 1, 1, 64, 16, "bf16")
    rng = c.rng
    size = np.exp2(rng.integers(-20, 20, (c.pages, 1, 16, 1)).astype(np.float32))
    codes, words = D.encode((rng.standard_normal((c.pages, 1, 16, 64)) * size).astype(np.float32))
    c.vc, c.vw = D.pack(codes), words
    c.cache.v_codes.copy_(torch.from_numpy(c.vc)), c.cache.v_words.copy_(torch.from_numpy(c.vw.view(np.int32)))
    q, qh = c.queries()
    want, mag, _ = c.want(qh)
    assert_attention(c.attend(q), want, mag, "bf16")


def test_attention_strided_queries_scale_and_output(torch):
    c = Case(torch, [(2, 20), (3, 33)], 4, 2, 128, 32, "bf16")
    big, _ = to16(torch, c.rng.standard_normal((c.tokens, 9, 128)), "bf16")
    q = big[:, 1:9:2]
    qh = q.float().cpu().numpy()
    want, mag, _ = c.want(qh, scale=0.3)
    out = torch.full((c.tokens, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    assert c.attend(q, scale=0.3, out=out) is out
    assert_attention(out, want, mag, "bf16")


def test_attention_repeats_exactly_on_streams_and_in_graphs(torch):
    c = Case(torch, [(1, 3000), (1, 1711), (1, 64)], 8, 2, 128, 16, "fp16", seed=3)
    q, qh = c.queries()
    ref = c.attend(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = c.attend(q, stream=side)
    side.synchronize()
    assert torch.equal(ref, other)
    graph = torch.cuda.CUDAGraph()
    qq, out = q.clone(), torch.zeros_like(ref)
    with torch.cuda.graph(graph):
        c.attend(qq, out=out)
    for i in range(4):
        qq.copy_(q * (1 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, c.attend(q * (1 + i)))


def test_attention_long_cache_and_offsets_past_32_bits(torch):
    """A sequence in the last pages of a cache whose codes take more than 4 GiB."""
    pages, hkv, page, d = 35000, 4, 512, 128
    free, _ = torch.cuda.mem_get_info()
    assert free > 12 << 30
    cache = S.KV4Cache(pages, page, hkv, d)
    assert cache.k_codes.numel() > 1 << 32
    rng = np.random.default_rng(0)
    n, L = 3, 5000
    ids = np.array([pages - 1 - 2 * i for i in range(-(-L // page))], np.int32)
    table = torch.from_numpy(ids[None]).cuda()
    k, kh = to16(torch, rng.standard_normal((L, hkv, d)), "bf16")
    lens = torch.tensor([L], dtype=torch.int32, device="cuda")
    S.kv4_append(cache, k, k, table, lens, cu_tokens=torch.tensor([0, L], dtype=torch.int32, device="cuda"))
    codes, words = D.encode(kh)
    got = cache.k_words[ids.astype(np.int64)].transpose(1, 2).reshape(-1, hkv)[:L].cpu().numpy().view(np.uint32)
    assert np.array_equal(got, words)
    q, qh = to16(torch, rng.standard_normal((n, 8, d)), "bf16")
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    out = S.kv4_attention(q, cache, table, lens, cu_tokens=cu)
    pc = D.pack(codes).transpose(1, 0, 2)[None]
    pw = words.T[None].copy()
    want, mag, _ = D.attention(qh, pc, pw, pc, pw, np.array([[0]]), np.array([L]), np.array([0, n]), d ** -0.5)
    # the oracle's one page of L tokens stands for the pages
    assert want.any()
    assert_attention(out, want, mag, "bf16")
    back, _ = S.kv4_gather(cache, table, lens, cu_tokens=torch.tensor([0, L], dtype=torch.int32, device="cuda"),
                           total_tokens=L, dtype=torch.bfloat16)
    assert torch.equal(back.cpu(), torch.from_numpy(D.decode32(D.pack(codes), words)).to(torch.bfloat16))


def test_cache_operators_refuse_bad_arguments(torch):
    c = Case(torch, [(1, 20), (1, 33)], 4, 2, 64, 16, "fp16")
    q, _ = c.queries()
    k = q[:, :2]
    bad = [
        lambda: S.KV4Cache(4, 24, 2, 64), lambda: S.KV4Cache(4, 16, 2, 80), lambda: S.KV4Cache(0, 16, 2, 64),
        lambda: S.KV4Cache.from_tensors(c.cache.k_codes, c.cache.k_words.long(), c.cache.v_codes, c.cache.v_words),
        lambda: S.KV4Cache.from_tensors(c.cache.k_codes, c.cache.k_words[:1], c.cache.v_codes, c.cache.v_words),
        lambda: S.KV4Cache.from_tensors(c.cache.k_codes.cpu(), c.cache.k_words, c.cache.v_codes, c.cache.v_words),
        lambda: S.kv4_attention(q.float(), c.cache, c.gt, c.gl), lambda: S.kv4_attention(q[:, :3], c.cache, c.gt, c.gl),
        lambda: S.kv4_attention(q[:1], c.cache, c.gt, c.gl), lambda: S.kv4_attention(q, c.cache, c.gt.long(), c.gl),
        lambda: S.kv4_attention(q, c.cache, c.gt, c.gl[:1]), lambda: S.kv4_attention(q, c.cache, c.gt.cpu(), c.gl),
        lambda: S.kv4_attention(q[..., :32], c.cache, c.gt, c.gl), lambda: S.kv4_attention(q, c.cache, c.gt, c.gl, window=-1),
        lambda: S.kv4_attention(q, c.cache, c.gt, c.gl, cu_tokens=c.gl),
        lambda: S.kv4_attention(q, c.cache, c.gt, c.gl, out=q.float()),
        lambda: S.kv4_attention(q.transpose(1, 2).contiguous().transpose(1, 2), c.cache, c.gt, c.gl),
        lambda: S.kv4_append(c.cache, k, q, c.gt, c.gl), lambda: S.kv4_append(c.cache, k, k.bfloat16(), c.gt, c.gl),
        lambda: S.kv4_append(c.cache, k, k, c.gt, c.gl, q=q),
        lambda: S.kv4_append(c.cache, k, k, c.gt, c.gl, positions=c.gl),
        lambda: S.kv4_append(c.cache, k, k, c.gt, c.gl, rotation=torch.rand(8, 33, device="cuda")),
        lambda: S.kv4_append(c.cache, k, k, c.gt, c.gl, rotation=torch.rand(8, 66, device="cuda")),
        lambda: S.kv4_append(c.cache, k, k, c.gt, c.gl, rotation=torch.rand(8, 32, device="cuda"), positions=c.gl[:1]),
        lambda: S.kv4_gather(c.cache, c.gt, c.gl, dtype=torch.float32),
        lambda: S.kv4_gather(c.cache, c.gt, c.gl, cu_tokens=torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was accepted")
    # nothing to do
    none = torch.empty((0, 4, 64), dtype=torch.float16, device="cuda")
    e2, e1 = torch.empty((0, 3), dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    assert S.kv4_attention(none, c.cache, e2, e1).shape == (0, 4, 64)
    assert S.kv4_append(c.cache, none[:, :2], none[:, :2], e2, e1) is None
    assert S.kv4_gather(c.cache, e2, e1)[0].shape == (0, 2, 64)


# Chunks with more than 64 rows for a key/value head in the average sequence run on blocks of 128 rows.

CHUNKS = [(60, 60), (130, 230), (0, 7), (0, 0), (90, 33), (97, 128), (1, 161)]


@pytest.mark.parametrize("window", [0, 1, 33, 100])
@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 1), (96, 6, 2), (128, 8, 2), (256, 4, 1)])
def test_attention_of_chunks_with_windows_and_empty_rows(torch, window, d, hq, hkv):
    """Sequences that are empty, shorter than their new tokens, or have none; tokens of no sequence at the end."""
    c = Case(torch, CHUNKS, hq, hkv, d, 16, "fp16" if window % 2 else "bf16", seed=window + d, tail=3)
    q, qh = c.queries(1.5)
    want, mag, lse = c.want(qh, window)
    got, gl = c.attend(q, window=window, return_lse=True)
    assert_attention(got, want, mag, c.dtype)
    assert (host(got)[-3:] == 0).all() and np.isneginf(host(gl)[-3:]).all()
    assert np.array_equal(np.isneginf(host(gl)[:-3]), np.isneginf(lse[:-3]))
    live = ~np.isneginf(lse[:-3])
    assert np.allclose(host(gl)[:-3][live], lse[:-3][live], rtol=1e-5, atol=2e-4)
    assert_attention(c.attend(q, window=window, max_len=230), want, mag, c.dtype)


@pytest.mark.parametrize("stale", [0x7FC00000, 0xFFFFFFFF, 0x7F800000, 0xFF800000, 0x7F7FFFFF])
def test_attention_of_chunks_does_not_see_hidden_places(torch, stale):
    """Stale words behind the ends of sequences and in absent pages: a page number outside the cache in the middle, and one past it."""
    c = Case(torch, [(100, 150), (80, 80), (90, 300)], 4, 2, 128, 16, "fp16", stale=stale)
    c.table[0, 2], c.table[2, 5], c.table[2, 18] = -1, c.pages + 9, -1
    c.gt = torch.from_numpy(c.table).cuda()
    q, qh = c.queries()
    want, mag, _ = c.want(qh)
    assert np.isfinite(want).all()
    assert_attention(c.attend(q), want, mag, "fp16")


@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_chunks_with_queries_of_every_size(torch, d):
    """Rows of a block from 2^-14 to 2^6 times the usual, an infinity and a NaN among them."""
    c = Case(torch, [(100, 300), (96, 97)], 4, 2, d, 32, "bf16", seed=d)
    size = np.exp2(c.rng.integers(-14, 7, (c.tokens, c.hq, 1)))
    q, qh = to16(torch, c.rng.standard_normal((c.tokens, c.hq, d)) * size, "bf16")
    bad = np.zeros((c.tokens, c.hq), bool)
    bad[5, 1] = bad[150, 2] = True
    q[5, 1, 7], q[150, 2, d - 1] = float("inf"), float("nan")
    clean = np.where(bad[..., None], 0, qh)
    want, mag, _ = c.want(clean)
    got = host(c.attend(q))
    assert np.isnan(got[bad]).all()
    # scores carry float32 errors of their own, 2^-20 of their size, as above
    top = np.abs(clean).max(-1, keepdims=True) * d ** 0.5 * 5
    bound = (2.0 ** -11 + 2.0 ** -13 + top * 2.0 ** -20) * mag + 2.0 ** -8 * 1.01 * np.abs(want) + 2.0 ** -25
    assert (np.abs(got - want)[~bad] <= bound[~bad]).all()


@pytest.mark.parametrize("d", [64, 96, 128])
def test_attention_of_chunks_with_a_query_out_of_all_proportion(torch, d):
    """Finite queries far above their neighbours in a block of rows: the neighbours' results do not change with them."""
    c = Case(torch, [(100, 300), (96, 97)], 4, 2, d, 32, "bf16", seed=d)
    size = np.ones((c.tokens, c.hq, 1))
    size[3, 0], size[60, 3], size[140, 1], size[150, 0] = 2.0 ** 30, 2.0 ** 100, 2.0 ** 60, 2.0 ** -40
    q, qh = to16(torch, c.rng.standard_normal((c.tokens, c.hq, d)) * size, "bf16")
    want, mag, _ = c.want(np.where(size > 1, 0, qh))
    got = host(c.attend(q))
    keep = (size <= 1)[..., 0]
    bound = (2.0 ** -11 + 2.0 ** -13) * mag + 1.01 * UNIT["bf16"] * np.abs(want)
    assert (np.abs(got - want)[keep] <= bound[keep]).all()
    # a query that large looks at one key alone
    top = c.want(np.where(size > 1, qh / size * 2.0 ** 20, 0))[0]
    assert np.isfinite(got[~keep]).all() and (np.abs(got - top)[~keep] <= (2.0 ** -7 * np.abs(top) + 2.0 ** -9 * np.abs(got).max())[~keep]).all()


# ---- linears ---------------------------------------------------------------------------------------------------------------

def weights(rng, M, K, G, dtype, torch):
    codes = rng.integers(0, 16, (M, K)).astype(np.uint8)
    zeros = rng.integers(0, 16, (M, K // G)).astype(np.uint8)
    scales, sh = to16(torch, rng.uniform(0.001, 0.01, (M, K // G)) * np.where(rng.random((M, K // G)) < 0.2, -1, 1), dtype)
    return codes, scales, sh, zeros


def assert_linear(got, y, small, big, dtype, K, G, act=0):
    slope = 1.13 if act == 2 else 1.0  # GELU's largest derivative
    err = (48 + K // G) * 2.0 ** -24 * big + 2.0 ** -19 * small
    bound = slope * err + (1.01 * UNIT[dtype] + (1e-5 if act == 2 else 0)) * np.abs(y) + SMALLEST[dtype] + (1e-6 if act == 2 else 0)
    d = np.abs(host(got) - y)
    assert (d <= bound).all(), (np.max(d / bound), np.argwhere(d > bound)[:4].tolist())


@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,K,N", [(16, 128, 1), (1, 128, 2), (50, 640, 3), (64, 1280, 16), (33, 384, 17), (129, 256, 32),
                                   (80, 2048, 33), (17, 896, 64), (100, 128, 65), (48, 1152, 130)])
def test_linear_matches_the_oracle(torch, M, K, N, G, dtype):
    K = -(-K // G) * G
    rng = np.random.default_rng(M + K + N)
    codes, scales, sh, zeros = weights(rng, M, K, G, dtype, torch)
    x, xh = to16(torch, rng.standard_normal((N, K)), dtype)
    g = lambda a: torch.from_numpy(a).cuda()
    y, small, big = D.linear(xh, codes, sh, zeros)
    if dtype == "bf16":  # the kernel's sums hold 128 + code
        big = big + np.abs(xh.astype(np.float64)) @ (256 * np.repeat(np.abs(sh.astype(np.float64)), G, 1)).T
    got = S.W4Linear(g(codes), scales, g(zeros))(x)
    assert_linear(got, y, small, big, dtype, K, G)


@pytest.mark.parametrize("M,K,N,G", [(2213, 3744, 36, 32), (3000, 4096, 33, 64), (4100, 2048, 64, 128), (1025, 8192, 100, 32),
                                     (5000, 1024, 20, 32), (4096, 6144, 32, 128)])
def test_linear_with_a_split_of_k(torch, M, K, N, G):
    """Sizes whose K the library may divide among workgroups, groups of every size."""
    rng = np.random.default_rng(M)
    codes, scales, sh, zeros = weights(rng, M, K, G, "fp16", torch)
    x, xh = to16(torch, rng.standard_normal((N, K)), "fp16")
    g = lambda a: torch.from_numpy(a).cuda()
    y, small, big = D.linear(xh, codes, sh, zeros)
    assert_linear(S.W4Linear(g(codes), scales, g(zeros))(x), y, small, big, "fp16", K, G)


@pytest.mark.parametrize("M,K,N,G", [(40, 8320, 50, 32), (33, 16512, 20, 128), (530, 6080, 64, 64), (700, 9024, 17, 32)])
def test_linear_with_many_shares_of_a_long_k(torch, M, K, N, G):
    """Few rows and a long K: dozens of shares, whose last may be shorter, and a sum of them over several waves."""
    rng = np.random.default_rng(M)
    codes, scales, sh, zeros = weights(rng, M, K, G, "fp16", torch)
    x, xh = to16(torch, rng.standard_normal((N, K)), "fp16")
    bias, bh = to16(torch, rng.standard_normal(M), "fp16")
    g = lambda a: torch.from_numpy(a).cuda()
    y, small, big = D.linear(xh, codes, sh, zeros, bh)
    layer = S.W4Linear(g(codes), scales, g(zeros), bias=bias)
    got = layer(x)
    assert_linear(got, y, small, big + np.abs(bh), "fp16", K, G)
    assert torch.equal(got, layer(x))


@pytest.mark.parametrize("K", [32, 96, 160, 224])
def test_linear_ends_inside_a_block_and_reads_nothing_past_a_row(torch, K):
    """K that is no multiple of 128: the columns behind a row's end belong to somebody else and may be NaN."""
    rng = np.random.default_rng(K)
    codes, scales, sh, zeros = weights(rng, 40, K, 32, "fp16", torch)
    xh = rng.standard_normal((5, K)).astype(np.float16)
    wide = torch.full((5, K + 128), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, :K] = torch.from_numpy(xh)
    g = lambda a: torch.from_numpy(a).cuda()
    y, small, big = D.linear(xh, codes, sh, zeros)
    assert_linear(S.W4Linear(g(codes), scales, g(zeros))(wide[:, :K]), y, small, big, "fp16", K, 32)


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_linear_bias_activation_stream_and_graph(torch, act, dtype):
    M, K, N, G = 72, 512, 9, 64
    rng = np.random.default_rng(act)
    codes, scales, sh, zeros = weights(rng, M, K, G, dtype, torch)
    x, xh = to16(torch, rng.standard_normal((N, K)) * 3, dtype)
    bias, bh = to16(torch, rng.standard_normal(M), dtype)
    g = lambda a: torch.from_numpy(a).cuda()
    layer = S.W4Linear(g(codes), scales, g(zeros), bias=bias, activation=act)
    y, small, big = D.linear(xh, codes, sh, zeros, bh, act)
    if dtype == "bf16":
        big = big + np.abs(xh.astype(np.float64)) @ (256 * np.repeat(np.abs(sh.astype(np.float64)), G, 1)).T
    ref = layer(x)
    assert_linear(ref, y, small, big + np.abs(bh), dtype, K, G, act)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.zeros_like(ref)
    assert layer(x, out=out, stream=side) is out
    side.synchronize()
    assert torch.equal(out, ref)
    graph, xx = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        layer(xx, out=out)
    for i in range(3):
        xx.copy_(x * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer(x * (i + 1)))


def test_linear_special_values(torch):
    """Values at fp16's ends, an infinity in one column of X, large activations through GELU."""
    M, K, G = 32, 256, 64
    rng = np.random.default_rng(0)
    codes, scales, sh, zeros = weights(rng, M, K, G, "fp16", torch)
    xh = rng.standard_normal((6, K)).astype(np.float16)
    xh[0] = 6e-8            # subnormal
    xh[1] *= np.float16(2e-5)
    xh[2] *= np.float16(100)
    xh[3, 7] = np.inf
    xh[4] = 0
    g = lambda a: torch.from_numpy(a).cuda()
    got = S.W4Linear(g(codes), scales, g(zeros))(g(xh))
    fine = [0, 1, 2, 4, 5]
    y, small, big = D.linear(xh[fine], codes, sh, zeros)
    assert_linear(got[fine], y, small, big, "fp16", K, G)
    assert not np.isfinite(host(got)[3]).any() and (host(got)[4] == 0).all()
    bias = torch.linspace(-6e4, 6e4, M, device="cuda").half()
    y = host(S.W4Linear(g(codes), scales, g(zeros), bias=bias, activation=S.ACT_GELU)(g(xh[4:5])))[0]
    b = bias.double().cpu().numpy()
    assert (y[b > 10] == b[b > 10]).all() and (y[b < -10] == 0).all()


def test_linear_refuses_bad_arguments(torch):
    rng = np.random.default_rng(0)
    codes, scales, _, zeros = weights(rng, 32, 256, 64, "fp16", torch)
    g = lambda a: torch.from_numpy(a).cuda()
    gc, gz = g(codes), g(zeros)
    layer = S.W4Linear(gc, scales, gz)
    x = torch.zeros((3, 256), dtype=torch.float16, device="cuda")
    bad = [lambda: S.W4Linear(gc, scales.float(), gz), lambda: S.W4Linear(gc, scales[:, :1], gz),
           lambda: S.W4Linear(gc, scales, gz[:, :1]), lambda: S.W4Linear(gc.cpu(), scales, gz),
           lambda: S.W4Linear(gc, scales, gz, bias=torch.zeros(31, dtype=torch.float16, device="cuda")),
           lambda: S.W4Linear(gc, scales, gz, activation=3), lambda: S.W4Linear(gc.t(), scales, gz),
           lambda: layer(x.bfloat16()), lambda: layer(x[:, :128]), lambda: layer(x.cpu()), lambda: layer(x[0]),
           lambda: layer(torch.zeros((256, 3), dtype=torch.float16, device="cuda").t()),
           lambda: layer(torch.zeros((3, 260), dtype=torch.float16, device="cuda")[:, 2:258]),
           lambda: layer(x, out=torch.zeros((3, 31), dtype=torch.float16, device="cuda"))]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was accepted")
    assert layer(x[:0]).shape == (0, 32)
