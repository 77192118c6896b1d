"""The 8-bit linears' kernels one by one (the tests' build of the library takes a plan), and calls that are easily got wrong:
broadcast and interlaced rows, in-place outputs, refusals of the host layer, graphs that share nothing."""
import ctypes as C
import os

import numpy as np
import pytest

import spmspm_amd as S
from oracle import w8_oracle as O
from spmspm_amd import api as A
from spmspm_amd import w8 as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture
def set_plan(monkeypatch):
    lib = C.CDLL(os.path.join(os.path.dirname(S.library_path()), "libSpMM_API_variants.so"))
    monkeypatch.setattr(A, "library", lambda: lib)
    monkeypatch.setattr(M, "_lib", None)
    yield lib.W8_Debug_SetPlan
    lib.W8_Debug_SetPlan(0, 0, 0, 0)


def weights(torch, M_, K, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-127, 128, (M_, K), generator=gen, dtype=torch.int8, device="cuda")
    return codes, (0.5 + torch.rand(M_, generator=gen, device="cuda")) * (0.01 / K ** 0.5)


def rows8(torch, N, K, seed):
    x = torch.randn((N, K), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").half()
    return S.quantize_x8(x)


def products(torch, gated, M_, K, N, seed=0, act=A.ACT_SILU):
    """A layer, its input and its outputs in float64 with their bound."""
    pairs = [weights(torch, M_, K, seed + i) for i in range(2 if gated else 1)]
    b = [torch.randn(M_, generator=torch.Generator(device="cuda").manual_seed(seed + 5 + i), device="cuda").half()
         for i in range(len(pairs))]
    codes, scales = rows8(torch, N, K, seed + 9)
    n = lambda t: t.cpu().numpy() if t.dtype != torch.float16 else t.double().cpu().numpy()
    if gated:
        layer = S.W8GatedLinear(*pairs[0], *pairs[1], gate_bias=b[0], up_bias=b[1], activation=act)
        want, bound = O.gated(n(codes), n(scales), *[n(t) for p in pairs for t in p], *[n(t) for t in b], act)
    else:
        layer = S.W8Linear(*pairs[0], bias=b[0], activation=act)
        want, bound = O.linear(n(codes), n(scales), *[n(t) for t in pairs[0]], n(b[0]), act)
    return layer, codes, scales, want, bound


def assert_close(got, want, bound):
    off = np.abs(got.double().cpu().numpy() - want) - (2.0 ** -11 * np.abs(want) + 1.01 * bound + 2.0 ** -25)
    assert (off <= 0).all(), off.max()


# rows past and below a tile's end, one block of K and many, fewer columns than a tile and several tiles, an odd M
SIZES = [(33, 100, 5), (300, 1100, 70), (129, 4100, 300), (520, 640, 17)]


@pytest.mark.parametrize("gated,rows", [(False, 1), (False, 2), (False, 4), (True, 2), (True, 4)])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("cols", [1, 2, 3, 4])
@pytest.mark.parametrize("shares", [1, 3])
def test_narrow_kernels(torch, set_plan, gated, size, rows, cols, shares):
    assert set_plan(0, rows, cols, shares) == 0
    layer, codes, scales, want, bound = products(torch, gated, *size)
    got = layer(codes, scales)
    assert_close(got, want, bound)
    assert torch.equal(got, layer(codes, scales))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("size", SIZES + [(1000, 257, 513)])
@pytest.mark.parametrize("kind", [1, 2, 3, 4, 5, 6])
@pytest.mark.parametrize("shares", [1, 2, 7])
def test_tile_kernels(torch, set_plan, gated, size, kind, shares):
    assert set_plan(kind, 0, 0, shares) == 0
    layer, codes, scales, want, bound = products(torch, gated, *size)
    got = layer(codes, scales)
    assert_close(got, want, bound)
    assert torch.equal(got, layer(codes, scales))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kind,shares", [(1, 1), (2, 1), (3, 1), (4, 1), (5, 1), (6, 1), (6, 3)])
def test_many_tiles_of_a_workgroup(torch, set_plan, gated, kind, shares):
    """More tiles than workgroups run at once, of one block of K and of three: loads that are ahead of the products by whole tiles,
    stores that the next tile does not wait for."""
    for K in (40, 380):
        size = (2100, K, 4100) if kind < 4 else (2100, K, 2100)
        assert set_plan(0, 2, 4, 1) == 0
        layer, codes, scales, want, bound = products(torch, gated, *size, act=A.ACT_NONE)
        first = layer(codes, scales)
        assert_close(first[:, :70], want[:, :70], bound[:, :70])
        assert set_plan(kind, 0, 0, shares) == 0
        layer._need.clear()  # the workspace of another plan
        for _ in range(3):
            assert torch.equal(first, layer(codes, scales))


def test_a_rows_result_does_not_depend_on_the_batch(torch):
    """Sums are whole numbers: whatever kernel a batch takes, a row has the same bits."""
    w, g, u = weights(torch, 700, 1000, 1), weights(torch, 700, 1000, 2), weights(torch, 700, 1000, 3)
    codes, scales = rows8(torch, 700, 1000, 4)
    for layer in (S.W8Linear(*w, activation=A.ACT_GELU), S.W8GatedLinear(*g, *u)):
        whole = layer(codes, scales)
        for n in (1, 2, 16, 17, 40, 64, 100, 256, 300):
            assert torch.equal(layer(codes[:n], scales[:n]), whole[:n])
            assert torch.equal(layer(codes[700 - n:], scales[700 - n:].contiguous()), whole[700 - n:])


@pytest.mark.parametrize("K", [48, 777, 1024, 5000])
def test_rows_that_are_one_row(torch, K):
    """Inputs of stride 0: every row the same memory."""
    one = torch.randn((1, K), device="cuda").half()
    x, w = one.expand(5, K), torch.rand(K, device="cuda").half()
    codes, scales = S.quantize_x8(x)
    assert torch.equal(codes, S.quantize_x8(x.contiguous())[0]) and (scales == scales[0]).all()
    y, h = S.rms_norm(x, w, residual=x)
    y2, h2 = S.rms_norm(x.contiguous(), w, residual=x.contiguous())
    assert torch.equal(y, y2) and torch.equal(h, h2)


def test_interlaced_rows_of_one_buffer(torch):
    """x, the residual and both outputs as slices of wider rows, in types of two bytes at odd places."""
    wide = torch.randn((6, 4 * 333 + 1), device="cuda").bfloat16()
    x, r, a, b = (wide[:, 1 + 333 * i:1 + 333 * (i + 1)] for i in range(4))
    w = torch.rand(333, device="cuda").bfloat16()
    want = S.rms_norm(x.contiguous(), w, residual=r.contiguous())
    before = wide.clone()
    room = torch.zeros((6, 2 * 333 + 7), device="cuda").bfloat16()
    y, h = S.rms_norm(x, w, residual=r, out=room[:, 3:336], residual_out=torch.empty((6, 333), device="cuda").bfloat16())
    assert torch.equal(y, want[0]) and torch.equal(h, want[1]) and torch.equal(wide, before)
    assert (room[:, :3] == 0).all() and (room[:, 336:] == 0).all()
    S.rms_norm(x, w, residual=r, out=a, residual_out=b)  # side by side in the rows that x and the residual lie in
    assert torch.equal(a, want[0]) and torch.equal(b, want[1]) and torch.equal(wide[:, :667], before[:, :667])
    with pytest.raises(ValueError):
        S.rms_norm(x, w, residual=r, out=wide[:, 300:633], residual_out=b)


def test_more_rows_than_a_launch_has_threads_for(torch):
    """Three million rows of nine numbers, each as it is alone."""
    x = torch.randn((3_000_001, 9), device="cuda").half()
    r, w = x.flip(0), torch.rand(9, device="cuda").half()
    y, h = S.rms_norm(x, w, residual=r)
    codes, scales, h8 = S.rms_norm_x8(x, w, residual=r)
    c, s = S.quantize_x8(x)
    assert torch.equal(h, x + r) and torch.equal(h8, h)
    for part in (slice(0, 5), slice((1 << 21) - 4, (1 << 21) + 5), slice(2_999_990, None)):
        one = S.rms_norm(x[part], w, residual=r[part])
        assert torch.equal(y[part], one[0])
        one = S.rms_norm_x8(x[part], w, residual=r[part])
        assert torch.equal(codes[part], one[0]) and torch.equal(scales[part], one[1])
        one = S.quantize_x8(x[part])
        assert torch.equal(c[part], one[0]) and torch.equal(s[part], one[1])


@pytest.mark.parametrize("M_,K,N", [(1 << 24, 1, 1), (1 << 24, 2, 19), (1, M.MAX_K, 1), (5, M.MAX_K, 300), (1, 1, 16 * 65535), (33, 40, 16 * 65535)])
@pytest.mark.parametrize("gated", [False, True])
def test_the_largest_sizes(torch, M_, K, N, gated):
    """Against sums in float64, which are exact, on the GPU."""
    pairs = [weights(torch, M_, K, i) for i in range(2 if gated else 1)]
    codes, scales = rows8(torch, N, K, 3)
    layer = S.W8GatedLinear(*pairs[0], *pairs[1], activation=A.ACT_NONE) if gated else S.W8Linear(*pairs[0])
    y = layer(codes, scales)
    assert y.shape == (N, M_)
    for n in range(0, N, 1 << 16):
        part = slice(n, min(N, n + (1 << 16)))
        want = 1
        for w, sw in pairs:
            want = want * ((codes[part].double() @ w.double().t()) * sw.double()) * scales[part].double()[:, None]
        # of a sum its conversion and two products, the gate's product, the rounding to 16 bits, there subnormal too
        bound = (2.0 ** -11 + 7 * 2.0 ** -24) * want.abs() * (1 + 2.0 ** -11) + 2.0 ** -25
        assert ((y[part].double() - want).abs() <= bound).all()
    if N == 1:  # the norm's longest row
        x = torch.randn((1, 1 << 24), device="cuda").bfloat16()
        got = S.rms_norm(x, torch.ones_like(x[0]))
        want = x.double() / (x.double().square().mean() + 1e-5).sqrt()
        # 2^24 squares summed by 1024 lanes, 2^14 each: 2^14 + 16 roundings in the worst order, half of that behind the root
        assert ((got.double() - want).abs() <= (2.0 ** -8 + (2 ** 13 + 20) * 2.0 ** -24) * want.abs()).all()


def test_host_layer_refusals(torch):
    x, w = torch.zeros((4, 64), device="cuda").half(), torch.ones(64, device="cuda").half()
    c, s = S.quantize_x8(x)
    big = torch.zeros((8, 64), device="cuda").half()
    layer = S.W8Linear(*S.quantize_w8(torch.ones((32, 64), device="cuda")))
    for call in (lambda: S.rms_norm(x, w[:32]), lambda: S.rms_norm(x, w.bfloat16()), lambda: S.rms_norm(x, w.cpu()),
                 lambda: S.rms_norm(x, w, eps=0), lambda: S.rms_norm(x, w, eps=float("nan")), lambda: S.rms_norm(x[0], w),
                 lambda: S.rms_norm(x, w, residual=x[:2]), lambda: S.rms_norm(x, w, residual=x.bfloat16()),
                 lambda: S.rms_norm(x, w, residual_out=x), lambda: S.rms_norm(x.t().contiguous().t(), w),
                 lambda: S.rms_norm(x, w, out=x[:2]), lambda: S.rms_norm(big[:4], w, out=big[1:5]),
                 lambda: S.rms_norm(x, w, residual=big[:4], residual_out=big[4:], out=big[4:]),
                 lambda: S.rms_norm(x, w, out=torch.empty((1, 64), device="cuda").half().expand(4, 64)),
                 lambda: S.rms_norm(x, x[0], out=x), lambda: S.rms_norm_x8(x, x[0], residual=x, residual_out=x),
                 lambda: S.rms_norm_x8(x, w, residual_out=x), lambda: S.quantize_x8(x.float()), lambda: S.quantize_x8(x[:, ::2]),
                 lambda: S.quantize_x8(torch.zeros((1, M.MAX_K + 1), device="cuda").half()),
                 lambda: layer(c), lambda: layer(c, s[:2]), lambda: layer(c, s.half()), lambda: layer(x, s), lambda: layer(x.bfloat16()),
                 lambda: layer(c[:, :32], s), lambda: layer(c.cpu(), s), lambda: layer(c.t().contiguous().t(), s),
                 lambda: layer(x, out=torch.empty((4, 31), device="cuda").half()), lambda: layer(x[:, :32], out=x[:, :32]),
                 lambda: layer(x, out=x[:, :32]),
                 lambda: S.W8Linear(c, s.half()), lambda: S.W8Linear(c, s[:2]), lambda: S.W8Linear(c.short(), s),
                 lambda: S.W8Linear(c, s, bias=w), lambda: S.W8Linear(c, s, activation=4), lambda: S.W8Linear(c, s, dtype=torch.float32),
                 lambda: S.W8GatedLinear(c, s, c[:2], s[:2]), lambda: S.w8_pack(c[:, :0], s)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("K", [50, 64, 1029])
def test_codes_that_are_not_laid_out_for_the_kernels(torch, K):
    """Rows at odd places, rows all the same, a last row that ends with its codes: copied, with the same result."""
    layer = S.W8Linear(*weights(torch, 96, K, 1))
    codes, scales = rows8(torch, 5, K, 2)
    want = layer(codes, scales)
    end = (K + 15) // 16 * 16
    tight = torch.empty(4 * end + K, dtype=torch.int8, device="cuda").as_strided((5, K), (end, 1))
    for c in (codes.contiguous(), torch.empty((5, K + 3), dtype=torch.int8, device="cuda")[:, 3:], tight):
        c.copy_(codes)
        assert torch.equal(layer(c, scales), want)
    assert torch.equal(layer(codes[1:2].expand(5, K), scales), layer(codes[1:2].repeat(5, 1), scales))
    far = torch.empty(4 * ((1 << 28) + 16) + end, dtype=torch.int8, device="cuda").as_strided((5, K), ((1 << 28) + 16, 1))
    far.copy_(codes)
    assert torch.equal(layer(far, scales), want)


def test_two_graphs_and_an_eager_call_at_once(torch):
    """Two recorded calls of one layer replayed on two streams beside eager calls: each has a workspace of its own."""
    M_, K, N = 300, 8192, 90  # K in shares
    layer = S.W8Linear(*weights(torch, M_, K, 1))
    xs = [torch.randn((N, K), device="cuda").half() for _ in range(3)]
    want = [layer(x) for x in xs]
    graphs, outs = [], []
    for x in xs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(x))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = layer(xs[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])


def test_workspace_is_what_the_call_asks_for(torch):
    """A call with one byte less than W8_WorkspaceBytes is refused before anything is launched, over sizes with and without shares."""
    L, rng, seen = M._library(), np.random.default_rng(0), set()
    for _ in range(200):
        m, k, n = int(np.exp(rng.uniform(4, 9))), int(np.exp(rng.uniform(4, 11))), int(np.exp(rng.uniform(0, 7)))
        gated, x16 = bool(rng.integers(2)), bool(rng.integers(2))
        need = L.W8_WorkspaceBytes(m, n, k, gated, x16)
        seen.add((need > 0, x16))
        if need:
            f, X = L.W8_Gated if gated else L.W8_Linear, 1 << 20
            assert f(None, X, X, X, None if x16 else X, X, m, n, k, *((None, None) if gated else (None,)), 0, X, need - 1, 0) == 1
    assert (True, False) in seen and (False, False) in seen and (True, True) in seen


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("K", [1, 7, 8, 9, 100, 127, 129, 1000, 2048, 5120, 13696])
@pytest.mark.parametrize("N", [1, 2, 3, 8, 9])
def test_16_bit_rows_are_rounded_alike_inside_and_outside(torch, dtype, K, N):
    """Few rows are rounded by the product's own workgroups: the same bits as of codes made before, rows of every kind among them."""
    kind = torch.float16 if dtype == "fp16" else torch.bfloat16
    wide = torch.randn((N, K + 3), generator=torch.Generator(device="cuda").manual_seed(K), device="cuda").to(kind)
    x = wide[:, 1:K + 1]  # rows at odd places
    for turn in range(2):
        if turn:
            x[0, K - 1] = float("inf")
            x[N - 1] = torch.finfo(kind).tiny
            if N > 2:
                x[1, 0], x[2] = float("nan"), 0
        for M_ in (40, 700):
            w, g, u = (weights(torch, M_, K, i) for i in range(3))
            for layer in (S.W8Linear(*w, activation=A.ACT_GELU, dtype=kind), S.W8GatedLinear(*g, *u, dtype=kind)):
                got, want = layer(x), layer(*S.quantize_x8(x))
                assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7), want.nan_to_num(7))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M_,K", [(1, 6208), (256, 7168), (576, 8192)])
def test_one_16_bit_row_with_k_in_shares(torch, dtype, M_, K):
    """Few enough to be rounded by the product's workgroups, but the kernel that adds up the shares reads the scale from memory: rounded
    by a kernel before the product."""
    kind = torch.float16 if dtype == "fp16" else torch.bfloat16
    assert K <= 8192 and M._library().W8_WorkspaceBytes(M_, 1, K, 1, 0) > 0
    g, u = weights(torch, M_, K, 1), weights(torch, M_, K, 2)
    layer, x = S.W8GatedLinear(*g, *u, dtype=kind), torch.randn((1, K), device="cuda").to(kind)
    codes, scales = S.quantize_x8(x)
    got, n = layer(x), lambda t: t.cpu().numpy()
    want, bound = O.gated(n(codes), n(scales), n(g[0]), n(g[1]), n(u[0]), n(u[1]))
    half = 2.0 ** (-11 if dtype == "fp16" else -8)
    assert (np.abs(got.double().cpu().numpy() - want) <= half * np.abs(want) + 1.01 * bound + 2.0 ** -25).all()
    assert torch.equal(got, layer(codes, scales))


@pytest.mark.parametrize("gated,rows", [(False, 1), (False, 2), (False, 4), (True, 2), (True, 4)])
@pytest.mark.parametrize("N", [1, 3, 8])
def test_few_16_bit_rows_with_k_in_shares(torch, set_plan, gated, rows, N):
    """The same of every kernel that rounds rows itself where K is whole."""
    assert set_plan(0, rows, 1, 3) == 0
    M_, K = 150, 650
    pairs = [weights(torch, M_, K, i) for i in range(2 if gated else 1)]
    layer = S.W8GatedLinear(*pairs[0], *pairs[1]) if gated else S.W8Linear(*pairs[0], activation=A.ACT_GELU)
    assert M._library().W8_WorkspaceBytes(M_, N, K, gated, 0) > 0
    x = torch.randn((N, K), device="cuda").half()
    codes, scales = S.quantize_x8(x)
    n = lambda t: t.cpu().numpy()
    want, bound = O.gated(n(codes), n(scales), *[n(t) for p in pairs for t in p]) if gated else \
        O.linear(n(codes), n(scales), *[n(t) for t in pairs[0]], act=A.ACT_GELU)
    assert_close(layer(x), want, bound)
    assert torch.equal(layer(x), layer(codes, scales))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M_,N", [(300, 90), (700, 193), (40, 5)])
def test_shares_of_k_in_two_graphs_and_an_eager_call_at_once(torch, gated, M_, N):
    """Sums that go through memory to a second kernel: recorded calls of one layer, replayed on two streams beside eager calls on a
    third, have a workspace each."""
    K = 36864
    assert M._library().W8_WorkspaceBytes(M_, N, K, gated, 0) > 0
    pairs = [weights(torch, M_, K, i) for i in range(2 if gated else 1)]
    layer = S.W8GatedLinear(*pairs[0], *pairs[1]) if gated else S.W8Linear(*pairs[0])
    xs = [rows8(torch, N, K, 10 + i) for i in range(3)]
    want = [layer(*x) for x in xs]
    assert not torch.equal(want[0], want[1])
    n = lambda t: t.cpu().numpy()
    exact, bound = (O.gated if gated else O.linear)(n(xs[0][0]), n(xs[0][1]), *[n(t) for p in pairs for t in p])
    assert_close(want[0], exact, bound)
    graphs, outs = [], []
    for x in xs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(*x))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
            with torch.cuda.stream(streams[2]):
                eager = layer(*xs[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])


@pytest.mark.parametrize("K", [1, 7, 8, 9, 100, 520, 1027, 5121, 9210, 33001, 70001])
@pytest.mark.parametrize("N", [1, 5, 300])
@pytest.mark.parametrize("dtype", [0, 1])
def test_bytes_behind_a_rows_codes_stay(torch, K, N, dtype):
    """What a caller keeps between K and the stride, behind the last row too, is there afterwards."""
    if N * K > 1 << 21:
        N = 2
    kind, L = (torch.float16, torch.bfloat16)[dtype], M._library()
    x, w = torch.randn((N, K), device="cuda").to(kind), torch.rand(K, device="cuda").to(kind)
    stride = (K + 15) // 16 * 16 + 16
    scales, stream = torch.empty(N, device="cuda"), torch.cuda.current_stream().cuda_stream
    for norm in (False, True):
        room = torch.full((N + 1, stride), 77, dtype=torch.int8, device="cuda")
        if norm:
            err = L.RMS_Norm(stream, x.data_ptr(), K, None, 0, w.data_ptr(), 1e-5, N, K, None, 0, None, 0, room.data_ptr(), stride,
                             scales.data_ptr(), dtype)
        else:
            err = L.W8_Quantize(stream, x.data_ptr(), K, N, K, room.data_ptr(), stride, scales.data_ptr(), dtype)
        assert err == 0
        t = x.double().cpu().numpy().astype(np.float32)
        want, _ = O.encode(t * w.double().cpu().numpy().astype(np.float32) if norm else t)
        assert np.array_equal(room[:N, :K].cpu().numpy(), want)
        assert (room[:, K:] == 77).all() and (room[N] == 77).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("K", [32776, 131071, 1 << 20, 1 << 24])
@pytest.mark.parametrize("factor", [1.0, 2.0 ** 70])
def test_the_sum_of_squares_of_a_long_row(torch, dtype, K, factor):
    """Rows of nearly equal numbers, whose roundings in a sum all go one way: seven of eight are 1.40625, the eighth is any.  Of a row that
    is read twice a lane adds eight squares, 32 such sums and up to 64 of those, and 22 lanes and waves follow: 126 roundings of
    2^-24, half of them behind the root, and six operations, below 2^-17.  2^70: squares that leave float32 and are summed again."""
    if factor > 1 and dtype == "fp16":
        factor = 2.0 ** 4
    kind, half = (torch.float16, 2.0 ** -11) if dtype == "fp16" else (torch.bfloat16, 2.0 ** -8)
    gen = torch.Generator(device="cuda").manual_seed(K)
    x = torch.full((2, K), 1.40625 * factor, device="cuda")
    x[:, ::8] = (1 + torch.rand((2, (K + 7) // 8), generator=gen, device="cuda")) * factor
    x = x.to(kind)
    w = torch.ones(K, device="cuda").to(kind)
    rms = (x.double().square().mean(-1, keepdim=True) + 1e-5).sqrt()
    want = x.double() / rms
    got = S.rms_norm(x, w)
    assert ((got.double() - want).abs() <= (half + 2.0 ** -17) * want).all()
    if K <= M.MAX_K:
        codes, scales = S.rms_norm_x8(x, w)
        want = x.double().amax(-1) / 127 / rms[:, 0]
        assert ((scales.double() - want).abs() <= (2.0 ** -24 + 2.0 ** -17) * want).all()


def test_a_gradient_is_refused_and_not_lost(torch):
    """There is no backward pass: results of tensors that require a gradient raise where one is asked for, as the registered operators'
    do; without gradients, and for tensors that require none, nothing changes."""
    x, r = (torch.randn((3, 64), device="cuda").half() for _ in range(2))
    gain = torch.ones(64, device="cuda").half()
    bias = torch.zeros(40, device="cuda").half()
    w, u = weights(torch, 40, 64, 1), weights(torch, 40, 64, 2)

    def calls(x, r, gain, bias, scale=None):
        codes, scales = S.quantize_x8(x)
        scales = scales if scale is None else scale
        one, two = S.W8Linear(*w, bias=bias), S.W8GatedLinear(*w, *u, up_bias=bias)
        return [(S.rms_norm(x, gain),), S.rms_norm(x, gain, residual=r), S.rms_norm_x8(x, gain)[1:], S.rms_norm_x8(x, gain, residual=r)[1:],
                (scales,), (one(x),), (one(codes, scales),), (two(x),), (two(codes, scales),),
                (S.rms_norm(x, gain, out=torch.empty_like(x)),)]

    plain = calls(x, r, gain, bias)
    assert not any(t.requires_grad for c in plain for t in c)
    leaf = lambda t: t.clone().requires_grad_()
    for args, touched in (((leaf(x), r, gain, bias), range(10)), ((x, leaf(r), gain, bias), (1, 3)), ((x, r, leaf(gain), bias), (0, 1, 2, 3, 9)),
                          ((x, r, gain, leaf(bias)), (5, 6, 7, 8)), ((x, r, gain, bias, leaf(S.quantize_x8(x)[1])), (6, 8))):
        for i, (got, want) in enumerate(zip(calls(*args), plain)):
            for t, p in zip(got, want):
                assert torch.equal(t, p)
                if i in touched:
                    with pytest.raises(RuntimeError, match="no backward"):
                        t.float().sum().backward()
                elif i != 4:  # the scales may be a leaf of the test
                    assert not t.requires_grad
        with torch.no_grad():
            assert not any(t.requires_grad for i, c in enumerate(calls(*args)) for t in c if i != 4)
    h = S.rms_norm(x, leaf(gain), residual=r)[1]
    h += 1  # the stream is worked on in place
    kept = r.clone()
    y, h = S.rms_norm(x, leaf(gain), residual=kept, residual_out=kept)
    assert h.data_ptr() == kept.data_ptr() and torch.equal(kept, plain[1][1]) and not kept.requires_grad


@pytest.mark.parametrize("gated", [False, True])
def test_a_module_takes_rows_of_its_own_length_only(torch, gated):
    """Weights of 100 and of 128 columns are packed to the same size, which is all that the operator sees of them."""
    w, u = weights(torch, 40, 100, 1), weights(torch, 40, 100, 2)
    layer = S.W8GatedLinear(*w, *u) if gated else S.W8Linear(*w)
    module = layer.module()
    x = torch.randn((3, 128), device="cuda").half()
    assert torch.equal(module(x[:, :100]), layer(x[:, :100]))
    for bad in (x, x[:, :90], x[0, :100]):
        for args in ((bad,), S.quantize_x8(bad) if bad.dim() == 2 else (bad, None)):
            with pytest.raises(ValueError):
                module(*args)


@pytest.mark.parametrize("gated,M_,K,N", [(False, 16384, 1000, 8), (False, 32768, 1000, 1), (False, 32768, 1000, 8), (False, 65536, 500, 1),
                                          (True, 8000, 1000, 8), (True, 16384, 1000, 1), (True, 16384, 1000, 2)])
def test_16_bit_rows_of_many_weights(torch, gated, M_, K, N):
    """On both sides of where rows are rounded by the product's workgroups: the same bits as of codes made before."""
    pairs = [weights(torch, M_, K, i) for i in range(2 if gated else 1)]
    layer = S.W8GatedLinear(*pairs[0], *pairs[1]) if gated else S.W8Linear(*pairs[0], activation=A.ACT_GELU)
    x = torch.randn((N, K), device="cuda").half()
    assert torch.equal(layer(x), layer(*S.quantize_x8(x)))
