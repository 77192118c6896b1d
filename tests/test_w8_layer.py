"""The 8-bit linears and the norm together: a decoder layer over a 4-bit cache, the registered operators, the layer in a graph."""
import numpy as np
import pytest

import spmspm_amd as S
from oracle import decode_oracle as D
from oracle import w8_oracle as O

pytestmark = pytest.mark.gpu
HALF = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def torch():
    import torch
    import spmspm_amd.torch_ops  # noqa: F401
    return torch


def setup(torch, dtype, lens=(20, 33, 1), hidden=256, heads=4, kv_heads=2, ffn=700, page=16, width=4):
    from spmspm_amd.decode_layer import GatedLayer
    kind = torch.float16 if dtype == "fp16" else torch.bfloat16
    angle = torch.arange(64, device="cuda")[:, None] * 0.1 ** torch.arange(32, device="cuda")
    layer = GatedLayer.random(hidden, heads, ffn, kv_heads, torch.cat((angle.cos(), angle.sin()), 1).float().contiguous(), kind)
    pages = len(lens) * width
    cache = S.KV4Cache(pages, page, kv_heads, hidden // heads)
    torch.manual_seed(0)
    table = torch.randperm(pages, device="cuda").int().view(len(lens), width)
    x, r = (torch.randn((sum(lens), hidden), device="cuda").to(kind) for _ in range(2))
    cu = torch.tensor(np.concatenate(([0], np.cumsum(lens))), dtype=torch.int32, device="cuda")
    return layer, cache, table, x, r, torch.tensor(lens, dtype=torch.int32, device="cuda"), cu


def values(t):
    return t.double().cpu().numpy()


def bits(torch, t):
    return t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


def check_linear(torch, layer, x, y, weight, dtype):
    """y of 16-bit x, or of codes and scales, against the formula on that very x."""
    if isinstance(x, tuple):
        codes, scales = (t.cpu().numpy() for t in x)
    else:
        codes, m = O.encode(values(x).astype(np.float32))
        scales = (m / np.float32(127)).astype(np.float32)
    pairs = [t.cpu().numpy() for t in weight]
    want, bound = O.gated(codes, scales, *pairs) if len(pairs) == 4 else O.linear(codes, scales, *pairs)
    assert (np.abs(values(y) - want) <= HALF[dtype] * np.abs(want) + 1.01 * bound + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("residual", [False, True])
def test_layer_is_its_operators_and_each_is_right(torch, dtype, residual, monkeypatch):
    """Every operator of the layer on what it was given, against its formula in 64 bits; and the layer's result is theirs."""
    from spmspm_amd import w8
    given = {}
    real = w8.w8_pack

    def pack(*a, **kw):
        p = real(*a, **kw)
        given[p.data_ptr()] = a
        return p

    monkeypatch.setattr(w8, "w8_pack", pack)
    layer, cache, table, x, r, lens, cu = setup(torch, dtype)
    weight = lambda l: given[l.packed.data_ptr()]
    r = r if residual else None
    y, h = layer(x, r, cache, table, lens, cu)

    other = S.KV4Cache.from_tensors(*(torch.zeros_like(t) for t in (cache.k_codes, cache.k_words, cache.v_codes, cache.v_words)))
    codes, scales, *h1 = S.rms_norm_x8(x, layer.norm1, 1e-5, r)
    eh, _, t, inverse = O.norm(bits(torch, x), bits(torch, layer.norm1), 1e-5, bits(torch, r) if residual else None, dtype == "bf16")
    want, m = O.encode(t)
    assert np.array_equal(codes.cpu().numpy(), want)
    assert np.allclose(scales.double().cpu().numpy(), m.astype(np.float64) / 127 * inverse, rtol=2.0 ** -17, atol=0)
    stream = h1[0] if residual else x
    assert np.array_equal(values(stream), eh)
    qkv = layer.qkv(codes, scales)
    check_linear(torch, layer.qkv, (codes, scales), qkv, weight(layer.qkv), dtype)
    q, k, v = qkv.view(-1, 8, 64).split((4, 2, 2), 1)
    q = S.kv4_append(other, k, v, table, lens, cu, q=q, rotation=layer.rotation)
    a = S.kv4_attention(q, other, table, lens, cu).view(-1, 256)
    host = [t.cpu().numpy() for t in (other.k_codes, other.k_words, other.v_codes, other.v_words)]
    ya, mag, _ = D.attention(values(q), host[0], host[1].view(np.uint32), host[2], host[3].view(np.uint32), table.cpu().numpy(),
                             lens.cpu().numpy(), cu.cpu().numpy(), 64 ** -0.5)
    # a probability is rounded to fp16 before it meets its value, the result to its type
    assert (np.abs(values(a).reshape(ya.shape) - ya) <= HALF[dtype] * np.abs(ya) + 1.1 * 2.0 ** -11 * mag + 2.0 ** -25).all()
    o = layer.out(a)
    check_linear(torch, layer.out, a, o, weight(layer.out), dtype)
    codes, scales, h2 = S.rms_norm_x8(o, layer.norm2, 1e-5, stream)
    eh, _, t, inverse = O.norm(bits(torch, o), bits(torch, layer.norm2), 1e-5, bits(torch, stream), dtype == "bf16")
    assert np.array_equal(codes.cpu().numpy(), O.encode(t)[0]) and np.array_equal(values(h2), eh)
    f = layer.gates(codes, scales)
    check_linear(torch, layer.gates, (codes, scales), f, weight(layer.gates), dtype)
    d = layer.down(f)
    check_linear(torch, layer.down, f, d, weight(layer.down), dtype)
    assert torch.equal(d, y) and torch.equal(h2, h) and torch.equal(other.k_codes, cache.k_codes)


def test_prompt_and_single_tokens_fill_the_cache_alike(torch):
    """Whatever kernels a batch takes, a token's keys and values have the same bits."""
    layer, cache, table, x, r, _, _ = setup(torch, "bf16", lens=(30,))
    lens = torch.tensor([30], dtype=torch.int32, device="cuda")
    layer(x, r, cache, table, lens, torch.tensor([0, 30], dtype=torch.int32, device="cuda"))
    single = S.KV4Cache(*cache.k_codes.shape[:1], 16, 2, 64)
    for t in range(30):
        lens.fill_(t + 1)
        layer(x[t:t + 1], r[t:t + 1], single, table, lens)
    for name in ("k_codes", "k_words", "v_codes", "v_words"):
        assert torch.equal(getattr(cache, name), getattr(single, name))


def test_layer_in_a_graph(torch):
    layer, cache, table, x, r, lens, cu = setup(torch, "fp16", lens=(20, 33, 5))
    layer(x, r, cache, table, lens, cu)
    lens += 1
    step, stream = x[:3].clone(), r[:3].clone()
    layer(step, stream, cache, table, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, h = layer(step, stream, cache, table, lens, max_len=64)
    for turn in range(4):
        step.copy_(x[3 + turn:6 + turn])
        stream.copy_(r[6 + turn:9 + turn])
        want = layer(step, stream, cache, table, lens, max_len=64)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(h, want[1])


@pytest.mark.parametrize("K", [64, 77, 1040, 1100])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_operators_pass_opcheck(torch, K, dtype):
    kind = torch.float16 if dtype == "fp16" else torch.bfloat16
    x, r = (torch.randn((5, K), device="cuda").to(kind) for _ in range(2))
    w = torch.rand(K, device="cuda").to(kind)
    ops = torch.ops.spmspm_amd
    for residual in (None, r):
        torch.library.opcheck(ops.rms_norm.default, (x, w, 1e-5, residual))
        torch.library.opcheck(ops.rms_norm_x8.default, (x, w, 1e-5, residual))
    torch.library.opcheck(ops.quantize_x8.default, (x,))
    codes, scales = ops.quantize_x8(x)
    weight = lambda: S.quantize_w8(torch.randn((40, K), device="cuda"))
    b = torch.randn(40, device="cuda").to(kind)
    one = S.W8Linear(*weight(), bias=b, activation=S.ACT_RELU, dtype=kind)
    two = S.W8GatedLinear(*weight(), *weight(), up_bias=b, dtype=kind)
    for args in ((codes, scales), (x, None)):
        torch.library.opcheck(ops.w8_linear.default, (*args, one.packed, b, 40, S.ACT_RELU, kind))
        torch.library.opcheck(ops.w8_gated.default, (*args, two.packed, None, b, 40, S.ACT_SILU, kind))
        assert torch.equal(one.module()(*args), one(*args)) and torch.equal(two.module()(*args), two(*args))


def test_compiled_block(torch):
    """A feed-forward block traced whole, with the modules."""
    K, F = 256, 320
    w = torch.rand(K, device="cuda").half()
    weight = lambda m, k: S.quantize_w8(torch.randn((m, k), device="cuda") * 0.02)
    gates, down = S.W8GatedLinear(*weight(F, K), *weight(F, K)).module(), S.W8Linear(*weight(K, F)).module()

    def block(x, h):
        codes, scales, h = torch.ops.spmspm_amd.rms_norm_x8(x, w, 1e-5, h)
        return down(gates(codes, scales)), h

    x, h = (torch.randn((9, K), device="cuda").half() for _ in range(2))
    eager, traced = block(x, h), torch.compile(block, fullgraph=True, backend="aot_eager")(x, h)
    assert torch.equal(eager[0], traced[0]) and torch.equal(eager[1], traced[1])


def test_command(torch, monkeypatch, capsys):
    """The command's second layer, at a size of its own choice."""
    from spmspm_amd import decode_layer
    monkeypatch.setattr("sys.argv", ["decode_layer", "--gated"])
    decode_layer.main()
    assert "us a step" in capsys.readouterr().out
