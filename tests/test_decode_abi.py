"""The decode operators' C ABI on a machine without a GPU: exported symbols and refusals, which come before any launch."""
import ctypes as C
import os
import re

import numpy as np
import pytest

import spmspm_amd as S
from oracle import decode_oracle as D
from spmspm_amd import build
from spmspm_amd import decode as M

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _declared():
    text = open(os.path.join(ROOT, "include", "decode_api.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b((?:KV4|W4)_[A-Za-z0-9_]*)\s*\([^;{]*\)\s*;", text)))


def test_every_declared_function_is_exported():
    names = _declared()
    assert names == ["KV4_Append", "KV4_Attention", "KV4_AttentionWorkspaceBytes", "KV4_Gather", "W4_Linear", "W4_Pack",
                     "W4_PackedBytes", "W4_WorkspaceBytes"]
    for n in names:
        assert hasattr(S.library(), n)
    for n in M.__all__:
        assert getattr(S, n) is getattr(M, n)
    with pytest.raises(AttributeError):
        S.no_such_operator


@pytest.mark.parametrize("source", ["kv4_cache.hip", "kv4_attention.hip", "w4_linear.hip"])
def test_no_kernel_spills(source):
    res = build.kernel_resources(source)
    assert res
    for name, r in res.items():
        assert r["vgpr_spill"] == 0 and r["sgpr_spill"] == 0 and r["scratch_bytes"] == 0, (name, r)


X = 1 << 20  # an address that is aligned and never read: every call below is refused on the host


def cache(**kw):
    d = dict(k_codes=X, k_words=X, v_codes=X, v_words=X, num_pages=4, page_size=16, kv_heads=2, head_dim=64)
    d.update(kw)
    return M._Cache(**d)


def batch(**kw):
    d = dict(block_table=X, seq_lens=X, cu_tokens=None, batch=3, table_width=4, table_stride=4, total_tokens=3)
    d.update(kw)
    return M._Batch(**d)


def rows(data=X, token=128, head=64):
    return M._Rows(data, token, head)


NONE = M._Rows(None, 0, 0)


def append(c=None, b=None, k=None, v=None, q=NONE, heads=0, out=None, rot=None, dtype=0):
    return M._library().KV4_Append(None, c or cache(), b or batch(), k or rows(), v or rows(), q, heads, out, rot, dtype)


def gather(c=None, b=None, k=X, v=X, dtype=0):
    return M._library().KV4_Gather(None, c or cache(), b or batch(), k, v, dtype)


def attend(c=None, b=None, q=None, heads=4, out=X, lse=None, scale=0.125, window=0, max_len=0, ws=None, ws_bytes=0, dtype=0):
    return M._library().KV4_Attention(None, c or cache(), b or batch(), q or rows(token=256), heads, out, lse, scale, window,
                                      max_len, ws, ws_bytes, dtype)


BAD_CACHES = [dict(head_dim=80), dict(head_dim=32), dict(head_dim=0), dict(page_size=8), dict(page_size=48),
              dict(page_size=2048), dict(page_size=0), dict(num_pages=0), dict(kv_heads=0), dict(kv_heads=-1),
              dict(k_codes=None), dict(v_codes=X + 8), dict(k_words=X + 4), dict(v_words=None)]
BAD_BATCHES = [dict(batch=-1), dict(total_tokens=-1), dict(total_tokens=4), dict(table_width=0), dict(table_stride=3),
               dict(block_table=None), dict(seq_lens=None), dict(seq_lens=X + 1), dict(cu_tokens=X + 2),
               dict(batch=0, cu_tokens=X), dict(table_width=1 << 28, table_stride=1 << 28)]


@pytest.mark.parametrize("call", [append, gather, attend])
def test_bad_caches_and_batches_are_refused(call, capfd):
    for kw in BAD_CACHES:
        assert call(c=cache(**kw)) == 1, kw
    for kw in BAD_BATCHES:
        assert call(b=batch(**kw)) == 1, kw
    assert call(dtype=2) == 1 and call(dtype=-1) == 1
    out = capfd.readouterr().out
    assert out.count("MM_Sparse_API Error") == len(BAD_CACHES) + len(BAD_BATCHES) + 2
    # nothing to do is no error
    assert call(b=batch(batch=0, total_tokens=0)) == 0


def test_append_refusals(capfd):
    rot = M._Rotary(X, None, 100, 32, 0)
    for kw in (dict(k=rows(None)), dict(v=rows(X + 1)), dict(rot=M._Rotary(None, None, 100, 32, 0)),
               dict(rot=M._Rotary(X, None, 100, 33, 0)), dict(rot=M._Rotary(X, None, 100, 66, 0)),
               dict(rot=M._Rotary(X, None, 0, 32, 0)), dict(rot=M._Rotary(X, X + 2, 10, 32, 0)),
               dict(q=rows(), heads=4, out=X), dict(rot=rot, q=rows(), heads=0, out=X),
               dict(rot=rot, q=rows(), heads=4, out=None), dict(rot=rot, q=rows(), heads=4, out=X + 8)):
        assert append(**kw) == 1, kw


def test_attention_refusals(capfd):
    for kw in (dict(heads=3), dict(heads=0), dict(q=rows(None)), dict(q=rows(X + 8)), dict(q=rows(token=129)),
               dict(q=rows(head=65)), dict(out=None), dict(out=X + 4), dict(lse=X + 2), dict(window=-1), dict(max_len=-1),
               dict(scale=float("nan"))):
        assert attend(**kw) == 1, kw
    # a long cache is split: the workspace is needed, and is sized by the same arguments
    c, b = cache(num_pages=5000), batch(batch=1, total_tokens=1, table_width=4096, table_stride=4096)
    need = M._library().KV4_AttentionWorkspaceBytes(c, b, 4, 0, 0)
    assert need > 0 and need % (4 * 4 * 66) == 0
    assert attend(c=c, b=b) == 1 and attend(c=c, b=b, ws=X, ws_bytes=need - 1) == 1
    assert attend(c=c, b=b, ws=X + 4, ws_bytes=need) == 1
    # a short one, by its bound or its window, is not
    assert M._library().KV4_AttentionWorkspaceBytes(c, b, 4, 0, 100) == 0
    assert M._library().KV4_AttentionWorkspaceBytes(c, b, 4, 64, 0) == 0


def test_linear_sizes_and_refusals(capfd):
    L = M._library()
    # codes of 16 rows x 128 columns are 1024 bytes, scales of 16 rows 32 bytes a group, zero points 16 for each of
    # the blocks' groups; a multiple of 16
    assert L.W4_PackedBytes(16, 128, 128) == 1024 + 32 + 16
    assert L.W4_PackedBytes(17, 160, 32) == 2 * 2 * 1024 + 2 * 5 * 32 + 2 * 8 * 16
    assert L.W4_PackedBytes(1048560, 65536, 64) == 65535 * (512 * 1024 + 1024 * 48)
    for bad in ((0, 128, 64), (16, 0, 64), (16, 100, 32), (16, 128, 16), (16, 128, 256), (16 * 65535 + 1, 128, 64)):
        assert L.W4_PackedBytes(*bad) == 0
        assert L.W4_Pack(None, X, X, X, *bad, 0, X) == 1
        assert L.W4_Linear(None, X, X, 4096, X, bad[0], 1, bad[1], bad[2], None, 0, None, 0, 0) == 1
    for codes, scales, zeros, packed in ((None, X, X, X), (X, X + 1, X, X), (X, X, None, X), (X, X, X, X + 8)):
        assert L.W4_Pack(None, codes, scales, zeros, 16, 128, 64, 0, packed) == 1
    ok = dict(packed=X, x=X, stride=128, y=X, M=16, N=4, K=128, G=64, bias=None, act=0, dtype=0)
    for kw in (dict(packed=X + 8), dict(x=X + 2), dict(x=None), dict(y=None), dict(y=X + 1), dict(stride=120),
               dict(stride=129), dict(bias=X + 1), dict(act=3), dict(act=-1), dict(dtype=2), dict(N=-1)):
        a = dict(ok, **kw)
        assert L.W4_Linear(None, a["packed"], a["x"], a["stride"], a["y"], a["M"], a["N"], a["K"], a["G"], a["bias"],
                           a["act"], None, 0, a["dtype"]) == 1, kw
    assert L.W4_Linear(None, X, X, 128, X, 16, 0, 128, 64, None, 0, None, 0, 0) == 0
    # a split K needs its workspace
    need = L.W4_WorkspaceBytes(9216, 64, 36864, 64)
    assert need > 0 and need % (4 * 9216 * 64) == 0 and L.W4_WorkspaceBytes(28672, 16, 7168, 128) == 0
    for ws, size in ((None, need), (X, need - 1), (X + 8, need)):
        assert L.W4_Linear(None, X, X, 36864, X, 9216, 64, 36864, 64, None, 0, ws, size, 0) == 1


def test_linear_workspace_is_what_the_call_asks_for(capfd):
    """Over sizes and groups: a call with one byte less is refused, and one with the workspace is not (without a GPU it goes as
    far as the launch, which fails in another way)."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("would launch")
    L, rng, seen = M._library(), np.random.default_rng(0), set()
    for _ in range(300):
        group = int(rng.choice((32, 64, 128)))
        m, k = int(np.exp(rng.uniform(3, 10.5))), group * max(1, int(np.exp(rng.uniform(5, 10.5))) // group)
        n = int(np.exp(rng.uniform(2.5, 6)))
        need = L.W4_WorkspaceBytes(m, n, k, group)
        seen.add((group, need > 0))
        call = lambda ws, size: L.W4_Linear(None, X, X, k, X, m, n, k, group, None, 0, ws, size, 0)
        assert call(X, need) != 1, (m, n, k, group)
        if need:
            assert call(X, need - 1) == 1 and call(None, need) == 1
    assert len(seen) == 6


def test_attention_workspace_is_what_the_call_asks_for(capfd):
    import torch
    if torch.cuda.is_available():
        pytest.skip("would launch")
    L, rng, seen = M._library(), np.random.default_rng(1), set()
    for _ in range(300):
        heads, share, d = int(rng.choice((1, 2, 8, 40))), int(rng.choice((1, 4, 7, 16, 64))), int(rng.choice((64, 96, 128, 256)))
        b, width = int(np.exp(rng.uniform(0, 4))), int(np.exp(rng.uniform(0, 9)))
        tokens = b if rng.random() < 0.5 else int(np.exp(rng.uniform(0, 8)))
        c = cache(num_pages=9, kv_heads=heads, head_dim=d, page_size=int(rng.choice((16, 64, 256))))
        bt = batch(batch=b, total_tokens=tokens, table_width=width, table_stride=width, cu_tokens=None if tokens == b else X)
        window, most = int(rng.choice((0, 0, 100, 5000))), int(rng.choice((0, 300, 100000)))
        need = L.KV4_AttentionWorkspaceBytes(c, bt, heads * share, window, most)
        seen.add(need > 0)
        call = lambda ws, size: attend(c=c, b=bt, heads=heads * share, q=rows(token=heads * share * d, head=d), window=window,
                                       max_len=most, ws=ws, ws_bytes=size)
        assert call(X, need) != 1
        if need:
            assert call(X, need - 1) == 1 and call(None, need) == 1
    assert len(seen) == 2


def test_cache_encoding_is_within_half_a_step_and_holds_zero_exactly():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((500, 64)).astype(np.float32) * np.exp(rng.uniform(-30, 30, (500, 1))).astype(np.float32)
    x[::7, 3] = 0
    x[1], x[2] = np.abs(x[1]), -np.abs(x[2])
    codes, words = D.encode(x)
    back = D.decode64(D.pack(codes), words)
    scale = words.view(np.float32).astype(np.float64)
    # half a step from rounding the element, half from the zero point's rounding where an end is cut off, and the scale's 2^-20
    assert (np.abs(back - x) <= scale[:, None] * 1.001).all()
    assert (back[::7, 3] == 0).all()
    inner = (codes > 0) & (codes < 15)
    assert (np.abs(back - x)[inner] <= (scale[:, None] * 0.50001 + 0 * x)[inner]).all()


def test_quantize_w4_rounds_to_the_nearest_code():
    import torch
    torch.manual_seed(0)
    w = torch.randn(24, 256) * 0.02
    w[3, :64] = 0
    w[5] = 1e-9
    codes, scales, zeros = S.quantize_w4(w, 64)
    assert codes.dtype == torch.uint8 and int(codes.max()) <= 15 and scales.shape == (24, 4) and scales.dtype == torch.float16
    back = (codes.view(24, 4, 64).double() - zeros.double()[..., None]) * scales.double()[..., None]
    assert ((back - w.view(24, 4, 64).double()).abs() <= 1.01 * scales.double()[..., None]).all()
    assert (back[3, 0] == 0).all()
    with pytest.raises(ValueError):
        S.quantize_w4(w, 96)
