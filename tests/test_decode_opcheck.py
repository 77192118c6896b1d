"""The registered decode operators under torch's own checks of a registration: schema, fake implementation, tracing."""
import pytest

import spmspm_amd as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    import spmspm_amd.torch_ops  # noqa: F401
    return torch


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("with_q", [False, True])
def test_cache_operators_pass_opcheck(torch, dtype, with_q):
    kind = torch.float16 if dtype == "fp16" else torch.bfloat16
    torch.manual_seed(0)
    cache = S.KV4Cache(8, 16, 2, 64)
    held = (cache.k_codes, cache.k_words, cache.v_codes, cache.v_words)
    table = torch.randperm(8, device="cuda").int().view(2, 4)
    lens = torch.tensor([20, 33], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 20, 53], dtype=torch.int32, device="cuda")
    rows = torch.randn((53, 8, 64), device="cuda").to(kind)
    rotation = torch.rand((64, 32), device="cuda") if with_q else None
    positions = torch.arange(53, dtype=torch.int32, device="cuda") if with_q else None
    ops = torch.ops.spmspm_amd
    # k and v are slices of one product's output, q strided too
    args = (*held, rows[:, 4:6], rows[:, 6:], table, lens, cu, rows[:, :4] if with_q else None, rotation, with_q, positions)
    torch.library.opcheck(ops.kv4_append.default, args)
    q = ops.kv4_append(*args)
    assert q.shape == ((53, 4, 64) if with_q else (0,)) and q.dtype == kind
    torch.library.opcheck(ops.kv4_gather.default, (*held, table, lens, cu, 53, kind))
    torch.library.opcheck(ops.kv4_attention.default, (rows[:, :4].contiguous(), *held, table, lens, cu, 0.2, 7, 64))
    # one token of every sequence
    step = rows[:2]
    args = (*held, step[:, 4:6], step[:, 6:], table, lens, None, step[:, :4] if with_q else None, rotation, with_q, None)
    torch.library.opcheck(ops.kv4_append.default, args)
    torch.library.opcheck(ops.kv4_gather.default, (*held, table, lens, None, 2, kind))


def test_append_is_traced_as_a_change_of_the_cache(torch):
    """A compiled step appends and then reads what it wrote, as the eager one does."""
    cache = [S.KV4Cache(4, 16, 2, 64) for _ in range(2)]
    table, lens = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda"), torch.tensor([17], dtype=torch.int32, device="cuda")
    torch.manual_seed(1)
    rows = torch.randn((1, 8, 64), device="cuda").half()
    ops = torch.ops.spmspm_amd

    def step(rows, kc, kw, vc, vw):
        ops.kv4_append(kc, kw, vc, vw, rows[:, 4:6], rows[:, 6:], table, lens, None, None, None, False, None)
        k, v = ops.kv4_gather(kc, kw, vc, vw, table, lens, None, 1, torch.float16)
        return ops.kv4_attention(rows[:, :4].contiguous(), kc, kw, vc, vw, table, lens, None, None, 0, 0) + k.sum() + v.sum()

    arrays = [(c.k_codes, c.k_words, c.v_codes, c.v_words) for c in cache]
    eager = step(rows, *arrays[0])
    traced = torch.compile(step, fullgraph=True, backend="aot_eager")(rows, *arrays[1])
    assert torch.equal(eager, traced)
    assert all(torch.equal(a, b) for a, b in zip(*arrays)) and arrays[0][1].any()
