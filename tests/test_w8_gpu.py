"""The 8-bit linears and the norm before them on the GPU, against the definitions in 64 bits (oracle/w8_oracle.py).

Tolerances.  A rounding to 16 bits is off by half a step: 2^-11 of a value in fp16, 2^-8 in bf16 (and 2^-25 among fp16's subnormal
numbers).  Before it float32 arithmetic is off by what the oracle's bounds say for products; for a norm by the rounding of the
sum of squares, at most 8 n + 22 additions deep where a lane takes n vectors of eight, 2^-24 each, which the square root halves, and
six more operations: below 2^-17 for rows that are held in registers (n <= 4), 2^-16 for longer ones (n <= 16).  Codes are compared for
equality."""
import numpy as np
import pytest

import spmspm_amd as S
from oracle import w8_oracle as O

pytestmark = pytest.mark.gpu
HALF = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def kind(torch, dtype):
    return torch.float16 if dtype == "fp16" else torch.bfloat16


def bits(t):
    return t.contiguous().view(__import__("torch").int16).cpu().numpy().view(np.uint16)


def values(t):
    return t.double().cpu().numpy()


def rows(torch, N, K, dtype, seed=0, gap=0, offset=0):
    """[N][K] rows K + gap elements apart, `offset` elements into their storage, with a few large channels."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((N, K + gap), generator=gen, device="cuda") * (1 + 15 * (torch.rand(K + gap, generator=gen, device="cuda") < 0.01))
    flat = torch.zeros(N * (K + gap) + offset, dtype=kind(torch, dtype), device="cuda")
    flat[offset:] = x.flatten().to(flat.dtype)
    return flat[offset:].view(N, K + gap)[:, :K]


def check_rows8(codes, scales, t32, factor=None, rel=0.0):
    want, m = O.encode(t32)
    got, sc = codes.cpu().numpy(), scales.cpu().numpy()
    assert np.array_equal(got, want)
    s = m.astype(np.float64) / 127 * (1 if factor is None else factor)
    assert np.array_equal(np.isnan(sc), np.isnan(s))
    ok = ~np.isnan(s)
    assert (np.abs(sc[ok] - s[ok]) <= (2.0 ** -24 + rel) * s[ok]).all()


LENGTHS = [1, 7, 8, 9, 100, 511, 512, 513, 2048, 2049, 4096, 4100, 8192, 8193, 20480, 32768, 32769, 131071]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("K", LENGTHS)
@pytest.mark.parametrize("N,gap,offset", [(1, 0, 0), (5, 3, 1)])
def test_quantize_rows(torch, dtype, K, N, gap, offset):
    x = rows(torch, N, K, dtype, K, gap, offset)
    codes, scales = S.quantize_x8(x)
    assert codes.shape == (N, K) and codes.dtype == torch.int8 and scales.dtype == torch.float32
    check_rows8(codes, scales, values(x).astype(np.float32))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_quantize_codes_between_two(torch, dtype):
    """Every magnitude below a power of two, so that many quotients lie exactly half-way; then quotients a hair beside it."""
    step = 2.0 ** (-11 if dtype == "fp16" else -8)
    for top in (1.0, 127.0, 0.996, 1.5, 254.0 / 256):
        m = torch.tensor([top], dtype=kind(torch, dtype), device="cuda").float().item()
        t = (torch.arange(1, 4097, device="cuda").float() * step * m).clamp(max=m).to(kind(torch, dtype))
        x = torch.stack((t, -t))
        codes, scales = S.quantize_x8(x)
        check_rows8(codes, scales, values(x).astype(np.float32))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("K", [40, 3000, 33000])
def test_quantize_rows_of_every_kind(torch, dtype, K):
    """Zeros, one number alone, subnormal ones, the largest, an infinity, a NaN: each row by itself."""
    x = rows(torch, 9, K, dtype, 3)
    info = torch.finfo(x.dtype)
    x[0] = 0
    x[1] = 0
    x[1, K - 1] = -3
    x[2] = x[2] * info.tiny
    x[3, 5] = info.max
    x[4, K // 2] = float("inf")
    x[5, K - 1] = float("-inf")
    x[6, 0] = float("nan")
    x[7] = 2.0 ** -101 if dtype == "bf16" else info.tiny * info.eps
    codes, scales = S.quantize_x8(x)
    check_rows8(codes, scales, values(x).astype(np.float32))
    assert scales[0] == 0 and torch.isnan(scales[4:7]).all() and (codes[4:7] == 0).all()
    assert (scales[7] == 0) == (dtype == "bf16")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("K", LENGTHS)
@pytest.mark.parametrize("residual", [False, True])
def test_norm(torch, dtype, K, residual):
    N, eps = (6 if K < 600 else 2), 1e-5
    x, w = rows(torch, N, K, dtype, K, 2, 1), rows(torch, 1, K, dtype, 7)[0] * 0.1 + 1
    r = rows(torch, N, K, dtype, 9, 5) if residual else None
    h, y, t, inverse = O.norm(bits(x), bits(w), eps, bits(r) if residual else None, dtype == "bf16")
    rel = 2.0 ** -17 if K <= 32768 else 2.0 ** -16
    got = S.rms_norm(x, w, eps, residual=r)
    if residual:
        got, stored = got
        assert np.array_equal(values(stored), h)
    assert (np.abs(values(got) - y) <= (HALF[dtype] + rel) * np.abs(y) + 2.0 ** -25).all()
    codes, scales, *stored = S.rms_norm_x8(x, w, eps, residual=r)
    assert len(stored) == residual and (not residual or np.array_equal(values(stored[0]), h))
    check_rows8(codes, scales, t, inverse, rel)


@pytest.mark.parametrize("K", [77, 5120, 33001])
@pytest.mark.parametrize("place", ["x", "residual"])
def test_norm_in_place(torch, K, place):
    w = rows(torch, 1, K, "bf16", 1)[0]
    x, r = rows(torch, 3, K, "bf16", 2, 8), rows(torch, 3, K, "bf16", 3, 4)
    y, h = S.rms_norm(x, w, 1e-6, residual=r)
    c, s, _ = S.rms_norm_x8(x, w, 1e-6, residual=r)
    a, b = x.clone(), r.clone()
    a2, b2 = x.clone(), r.clone()
    y2, h2 = S.rms_norm(a, w, 1e-6, residual=b, residual_out=a if place == "x" else b, out=b if place == "x" else a)
    assert torch.equal(y2, y) and torch.equal(h2, h) and torch.equal(a if place == "x" else b, h)
    c2, s2, h2 = S.rms_norm_x8(a2, w, 1e-6, residual=b2, residual_out=a2 if place == "x" else b2)
    assert torch.equal(c2, c) and torch.equal(s2, s) and torch.equal(h2, h)
    z = x.clone()
    assert torch.equal(S.rms_norm(z, w, 1e-6, out=z), S.rms_norm(x, w, 1e-6))


@pytest.mark.parametrize("K", [64, 5000, 40000])
def test_norm_of_large_small_and_broken_rows(torch, K):
    """Squares beyond float32, rows that eps decides, an infinity and a NaN: as the formula says, each row by itself."""
    x = rows(torch, 7, K, "bf16", 5)
    x[0] = x[0] * 1e30
    x[1] = x[1] * 1e-30
    x[2] = 0
    x[3, K - 1] = float("inf")
    x[4, 3] = float("nan")
    x[5] = x[5] * 1e19
    w = rows(torch, 1, K, "bf16", 6)[0]
    h, y, t, inverse = O.norm(bits(x), bits(w), 1e-5, None, True)
    got = values(S.rms_norm(x, w))
    want = np.where(np.isnan(y), 0, y)
    assert np.array_equal(np.isnan(got), np.isnan(y)) and np.isnan(got[4]).all() and np.isnan(got[3]).sum() == 1
    # h / 2^96 and 1 / rms of 2^-96 and below: some bits of subnormal numbers are lost, 2^-22 of them
    assert (np.abs(np.where(np.isnan(got), 0, got) - want) <= (HALF["bf16"] + 2.0 ** -15) * np.abs(want)).all()
    codes, scales = S.rms_norm_x8(x, w)
    check_rows8(codes, scales, t, np.where(np.isfinite(inverse), inverse, np.nan), 2.0 ** -15)


def weights(torch, M, K, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-127, 128, (M, K), generator=gen, dtype=torch.int8, device="cuda")
    scales = (0.5 + torch.rand(M, generator=gen, device="cuda")) * (2.0 / 73 / K ** 0.5 / 3)
    return codes, scales


def biases(torch, M, dtype, seed, wanted):
    return torch.randn(M, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(kind(torch, dtype)) if wanted else None


def close(got, want, bound, dtype):
    got = values(got)
    assert got.shape == want.shape and np.isfinite(got).all()
    off = np.abs(got - want) - (HALF[dtype] * np.abs(want) + 1.01 * bound + 2.0 ** -25)
    assert (off <= 0).all(), off.max()


# (M, K, N): one number, below and past every tile's end, long and short sums, odd everything
SHAPES = [(1, 1, 1), (1, 200, 3), (15, 16, 16), (63, 65, 2), (64, 128, 17), (65, 129, 33), (200, 1000, 1), (300, 257, 130),
          (512, 4096, 64), (513, 1025, 48), (1000, 515, 257), (2049, 384, 100), (130, 16385, 40), (768, 896, 600), (640, 130, 1025),
          (40, 131071, 2), (5120, 640, 8)]


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("dtype,bias,act,x16", [("fp16", False, 0, True), ("bf16", True, 2, False), ("fp16", True, 1, False),
                                                ("bf16", True, 3, True)])
def test_linear(torch, M, K, N, dtype, bias, act, x16):
    x, (w, sw), b = rows(torch, N, K, dtype, M), weights(torch, M, K, K), biases(torch, M, dtype, N, bias)
    layer = S.W8Linear(w, sw, bias=b, activation=act, dtype=kind(torch, dtype))
    codes, scales = S.quantize_x8(x)
    y = layer(x) if x16 else layer(codes, scales)
    want, bound = O.linear(codes.cpu().numpy(), scales.cpu().numpy(), w.cpu().numpy(), sw.cpu().numpy(),
                           None if b is None else values(b), act)
    close(y, want, bound, dtype)


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("dtype,bias,act,x16", [("fp16", False, 3, False), ("bf16", True, 2, True), ("bf16", False, 1, False)])
def test_gated(torch, M, K, N, dtype, bias, act, x16):
    x, g, u = rows(torch, N, K, dtype, M), weights(torch, M, K, K), weights(torch, M, K, K + 1)
    bg, bu = biases(torch, M, dtype, N, bias), biases(torch, M, dtype, N + 1, bias)
    layer = S.W8GatedLinear(*g, *u, gate_bias=bg, up_bias=bu, activation=act, dtype=kind(torch, dtype))
    codes, scales = S.quantize_x8(x)
    y = layer(x) if x16 else layer(codes, scales)
    n = lambda t: None if t is None else (values(t) if t.dtype.is_floating_point and t.dtype != torch.float32 else t.cpu().numpy())
    want, bound = O.gated(n(codes), n(scales), n(g[0]), n(g[1]), n(u[0]), n(u[1]), n(bg), n(bu), act)
    close(y, want, bound, dtype)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,K,N", [(96, 64, 1), (130, 131071, 3), (256, 4096, 96), (512, 8192, 320)])
def test_products_at_the_ends_of_their_range(torch, gated, M, K, N):
    """Codes -128 and 127 throughout: the largest sums there are, exact."""
    for a, b in ((127, 127), (-128, -128), (-128, 127)):
        x = torch.full((N, (K + 15) // 16 * 16), a, dtype=torch.int8, device="cuda")[:, :K]
        w = torch.full((M, K), b, dtype=torch.int8, device="cuda")
        ones = torch.full((M,), 2.0 ** -20, device="cuda")
        scales = torch.full((N,), 0.25, device="cuda")
        if gated:
            y = S.W8GatedLinear(w, ones, w, ones, activation=S.ACT_NONE, dtype=torch.bfloat16)(x, scales)
        else:
            y = S.W8Linear(w, ones, dtype=torch.bfloat16)(x, scales)
        s = float(np.float32(a * b * K)) * 2.0 ** -22
        want = torch.full((N, M), s * s if gated else s, dtype=torch.float64).to(torch.bfloat16)
        assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("N", [3, 70, 300])
def test_rows_stay_by_themselves(torch, N):
    """A row with a NaN, stale codes behind K and codes of rows behind the last one: none reaches another row's results; what lies
    behind the last row of an output stays."""
    M, K = 320, 300
    w, sw = weights(torch, M, K, 1)
    x = rows(torch, N + 4, K, "fp16", 2)
    codes, scales = S.quantize_x8(x)
    wide = torch.full((N + 4, 352), -128, dtype=torch.int8, device="cuda")
    wide[:, :K] = codes
    scales[N:] = float("nan")
    layer = S.W8Linear(w, sw)
    room = torch.full((N + 2, M), 7.0, dtype=torch.float16, device="cuda")
    y = layer(wide[:N, :K], scales[:N], out=room[:N])
    assert y.data_ptr() == room.data_ptr() and (room[N:] == 7).all()
    want, bound = O.linear(codes[:N].cpu().numpy(), scales[:N].cpu().numpy(), w.cpu().numpy(), sw.cpu().numpy())
    close(y, want, bound, "fp16")
    x[1, 7] = float("nan")
    z = layer(x[:N])
    assert torch.isnan(z[1]).all() and torch.equal(z[0], y[0]) and torch.equal(z[2:], y[2:])


def test_relu_keeps_a_nan_and_no_rows_are_nothing(torch):
    w, sw = weights(torch, 64, 64, 1)
    x = torch.full((2, 64), float("nan"), dtype=torch.float16, device="cuda")
    assert torch.isnan(S.W8Linear(w, sw, activation=S.ACT_RELU)(x)).all()
    assert S.W8Linear(w, sw)(x[:0]).shape == (0, 64) and S.quantize_x8(x[:0])[0].shape == (0, 64)
    assert S.rms_norm(x[:0], x[0]).shape == (0, 64)


@pytest.mark.parametrize("N", [1, 50, 400])
def test_side_streams_and_replayed_graphs(torch, N):
    """A feed-forward block on a stream of its own, and in a graph that is replayed with changed contents between eager calls."""
    K, F = 512, 900
    w = rows(torch, 1, K, "fp16", 1)[0] * 0.1 + 1
    gates = S.W8GatedLinear(*weights(torch, F, K, 2), *weights(torch, F, K, 3))
    down = S.W8Linear(*weights(torch, K, F, 4))

    def block(x, h):
        codes, scales, h = S.rms_norm_x8(x, w, residual=h)
        return down(gates(codes, scales)), h

    x, h = rows(torch, N, K, "fp16", 5), rows(torch, N, K, "fp16", 6)
    want = block(x, h)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block(x, h)
        graph = torch.cuda.CUDAGraph()
        xs, hs = x.clone(), h.clone()
        block(xs, hs)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = block(xs, hs)
    for turn in range(4):
        xs.copy_(rows(torch, N, K, "fp16", 10 + turn))
        hs.copy_(rows(torch, N, K, "fp16", 20 + turn))
        eager = block(xs, hs)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


def test_given_stream(torch):
    w, sw = weights(torch, 256, 256, 1)
    layer, x = S.W8Linear(w, sw), rows(torch, 20, 256, "fp16", 2)
    want = layer(x)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream):
        got = layer(x, stream=stream)
        side.synchronize()
        assert torch.equal(got, want)


def test_offsets_past_32_bits(torch):
    """Rows whose offsets pass 2^31 elements, read through a stride; and the outputs of many rows."""
    K, stride = 64, (1 << 31) // 8
    big = torch.empty(17 * stride + K, dtype=torch.int8, device="cuda")
    x = rows(torch, 18, K, "fp16", 1)
    codes, scales = S.quantize_x8(x)
    view = big.as_strided((18, K), (stride, 1))
    view.copy_(codes)
    w, sw = weights(torch, 64, K, 2)
    layer = S.W8Linear(w, sw)
    assert torch.equal(layer(view, scales), layer(codes, scales))
    del big, view
    half = torch.empty((1 << 31) // 8 * 9 + K, dtype=torch.float16, device="cuda")
    far = half.as_strided((10, K), ((1 << 31) // 8, 1))
    far.copy_(x[:10])
    c, s = S.quantize_x8(far)
    assert torch.equal(c, codes[:10]) and torch.equal(s, scales[:10])
    gain = torch.ones(K, dtype=torch.float16, device="cuda")
    assert torch.equal(S.rms_norm(far, gain), S.rms_norm(x[:10], gain))
