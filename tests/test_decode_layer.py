"""The decode operators together: registered operators, a decoder layer over a 4-bit cache, the layer recorded in a graph."""
import numpy as np
import pytest

import spmspm_amd as S
from oracle import decode_oracle as D

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    import spmspm_amd.torch_ops  # noqa: F401
    return torch


def setup(torch, hidden=256, heads=4, page=16, lens=(20, 33, 1), width=4, seed=0):
    from spmspm_amd.decode_layer import DecodeLayer
    layer = DecodeLayer.random(hidden, heads, group=64, seed=seed)
    pages = len(lens) * width
    cache = S.KV4Cache(pages, page, heads, hidden // heads)
    torch.manual_seed(seed)
    table = torch.randperm(pages, device="cuda").int().view(len(lens), width)
    x = torch.randn((sum(lens), hidden), device="cuda").half()
    cu = torch.tensor(np.concatenate(([0], np.cumsum(lens))), dtype=torch.int32, device="cuda")
    return layer, cache, table, x, torch.tensor(lens, dtype=torch.int32, device="cuda"), cu


def plain_layer(torch, layer, x, cache, table, lens, cu):
    """The layer in float64 over dense weights and the values that the cache holds."""
    def dense(m):
        eye = torch.eye(m.K, dtype=torch.float16, device="cuda")
        return torch.cat([m(eye[i:i + 64]) for i in range(0, m.K, 64)]).double().t()

    def norm(n, t):
        return torch.nn.functional.layer_norm(t, (t.shape[1],), n.weight.double(), n.bias.double())

    T, hidden = x.shape
    x64, heads, d = x.double(), layer.heads, cache.head_dim
    qkv = (norm(layer.norm1, x64) @ dense(layer.qkv).t()).view(T, 3 * heads, d)
    n = lambda t: t.detach().cpu().numpy()
    y, _, _ = D.attention(n(qkv[:, :heads]), n(cache.k_codes), n(cache.k_words).view(np.uint32), n(cache.v_codes),
                          n(cache.v_words).view(np.uint32), n(table), n(lens), n(cu), d ** -0.5)
    h = x64 + torch.from_numpy(y).cuda().view(T, hidden) @ dense(layer.out).t()

    def ffn(l, t):
        eye = torch.eye(l.K, dtype=torch.float16, device="cuda")
        return t @ S.W4Linear.__call__(plain[l], eye).double()

    plain = {}
    for l in (layer.ffn1, layer.ffn2):  # the same weights without bias and activation
        p = object.__new__(S.W4Linear)
        p._adopt(l.packed, l.M, l.K, l.group, l.dtype, None, 0)
        plain[l] = p
    return h + ffn(layer.ffn2, torch.relu(ffn(layer.ffn1, norm(layer.norm2, h))))


def assert_layer(got, want):
    """fp16 roundings at every operator's end (a norm, two SpMMs, attention, two linears, two sums), each 2^-11 of values of the
    output's size or below, and the keys that the layer encoded from rounded products: eight roundings of the root mean square."""
    got, want = got.double().cpu().numpy(), want.detach().cpu().numpy()
    assert np.isfinite(got).all()
    assert np.linalg.norm(got - want) <= 8 * 2.0 ** -11 * np.linalg.norm(want)


def test_layer_prompt_then_steps_match_float64(torch):
    layer, cache, table, x, lens, cu = setup(torch)
    y = layer(x, cache, table, lens, cu)
    assert_layer(y, plain_layer(torch, layer, x, cache, table, lens, cu))
    last = (cu[1:] - 1).long()
    step = y[last].contiguous()
    one = torch.arange(4, dtype=torch.int32, device="cuda")
    for _ in range(3):
        lens = lens + 1
        new = layer(step, cache, table, lens)
        assert_layer(new, plain_layer(torch, layer, step, cache, table, lens, one))
        step = new


def test_layer_step_records_into_a_graph(torch):
    layer, cache, table, x, lens, cu = setup(torch, seed=1)
    y = layer(x, cache, table, lens, cu)
    step = y[(cu[1:] - 1).long()].contiguous()
    layer(step, cache, table, lens)  # lengths as they are: writes the last token's place again
    keep = [t.clone() for t in (cache.k_codes, cache.k_words, cache.v_codes, cache.v_words)]
    static, static_lens = step.clone(), lens.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(static, cache, table, static_lens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(static, cache, table, static_lens)

    def restore():
        for t, k in zip((cache.k_codes, cache.k_words, cache.v_codes, cache.v_words), keep):
            t.copy_(k)

    eager, replayed = [], []
    for run in (lambda a, l: layer(a, cache, table, l).clone(), None):
        restore()
        a, l = step.clone(), lens.clone()
        for i in range(4):
            l = l + 1
            if run:
                a = run(a, l)
                eager.append(a)
            else:
                static.copy_(a)
                static_lens.copy_(l)
                graph.replay()
                torch.cuda.synchronize()
                a = out.clone()
                replayed.append(a)
    for a, b in zip(eager, replayed):
        assert torch.equal(a, b)


def test_registered_operators_match_the_direct_calls_and_compile(torch):
    layer, cache, table, x, lens, cu = setup(torch, seed=2)
    ops, T = torch.ops.spmspm_amd, x.shape[0]
    rows = torch.randn((T, 12, 64), device="cuda").half()
    rotation = torch.rand((64, 32), device="cuda")
    arrays = (cache.k_codes, cache.k_words, cache.v_codes, cache.v_words)
    other = S.KV4Cache.from_tensors(*(t.clone() for t in arrays))
    a = S.kv4_append(cache, rows[:, 4:8], rows[:, 8:], table, lens, cu, q=rows[:, :4], rotation=rotation)
    b = ops.kv4_append(other.k_codes, other.k_words, other.v_codes, other.v_words, rows[:, 4:8], rows[:, 8:], table, lens, cu,
                       rows[:, :4], rotation, False, None)
    assert torch.equal(a, b)
    held = (other.k_codes, other.k_words, other.v_codes, other.v_words)
    assert all(torch.equal(s, t) for s, t in zip(arrays, held))
    y = S.kv4_attention(a, cache, table, lens, cu)
    assert torch.equal(y, ops.kv4_attention(a, *held, table, lens, cu, None, 0, 0))
    for s, t in zip(S.kv4_gather(cache, table, lens, cu, T), ops.kv4_gather(*held, table, lens, cu, T, torch.float16)):
        assert torch.equal(s, t)
    w = layer.ffn1
    z = w(x)
    assert torch.equal(z, w.module()(x))
    with pytest.raises(ValueError):
        ops.w4_linear(x, w.packed[:-16], None, w.M, w.group, 0)
    for op, args in ((ops.w4_linear, (x, w.packed, w.bias, w.M, w.group, 1)),
                     (ops.kv4_attention, (a, *held, table, lens, cu, None, 0, 0))):
        torch.library.opcheck(op.default, args)
    ffn = torch.nn.Sequential(layer.ffn1.module(), layer.ffn2.module())
    assert torch.equal(torch.compile(ffn, fullgraph=True, backend="aot_eager")(x), layer.ffn2(z))
