"""C ABI of the 8-bit linears and the norm on a machine without a GPU: exported symbols, sizes, refusals (which come before any launch),
and the oracle against the formulas."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch

import spmspm_amd as S
from oracle import w8_oracle as O
from spmspm_amd import build
from spmspm_amd import w8 as M

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
X = 1 << 20  # an address that is aligned and never read: every call below is refused on the host
BAD = 1      # hipErrorInvalidValue


def test_every_declared_function_is_exported():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "w8_api.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b((?:RMS|W8)_[A-Za-z0-9_]*)\s*\([^;{]*\)\s*;", text)))
    assert names == ["RMS_Norm", "W8_Gated", "W8_Linear", "W8_Pack", "W8_PackedBytes", "W8_Quantize", "W8_WorkspaceBytes"]
    for n in names:
        assert hasattr(S.library(), n)
    for n in M.__all__:
        assert getattr(S, n) is getattr(M, n)
    assert S.ACT_SILU == 3


@pytest.mark.parametrize("source", ["rms_norm.hip", "w8_linear.hip"])
def test_no_kernel_spills(source):
    res = build.kernel_resources(source)
    assert res
    for name, r in res.items():
        assert r["vgpr_spill"] == 0 and r["sgpr_spill"] == 0 and r["scratch_bytes"] == 0, (name, r)


def norm(x=X, x_stride=64, residual=None, r_stride=64, weight=X, eps=1e-5, N=2, K=64, h=None, h_stride=64, y=X, y_stride=64, codes=None,
         c_stride=64, scales=None, dtype=0):
    return M._library().RMS_Norm(None, x, x_stride, residual, r_stride, weight, eps, N, K, h, h_stride, y, y_stride, codes, c_stride,
                                 scales, dtype)


IN8 = dict(y=None, codes=X, scales=X)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(x=X + 1), dict(weight=None), dict(weight=X + 1), dict(residual=X + 1), dict(h=X + 1), dict(y=X + 1),
    dict(h=X, h_stride=63), dict(y_stride=63), dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
    dict(eps=1e-21), dict(N=-1), dict(K=0), dict(K=(1 << 24) + 1), dict(dtype=2), dict(dtype=-1), dict(y=None), dict(codes=X, scales=X),
    dict(IN8, codes=X + 8), dict(IN8, c_stride=72), dict(IN8, c_stride=48), dict(IN8, scales=X + 2), dict(IN8, scales=None),
    dict(IN8, codes=None), dict(IN8, K=131072), dict(IN8, c_stride=(1 << 28) + 16)])
def test_norm_refuses(kw, capfd):
    assert norm(**kw) == BAD
    assert "Error" in capfd.readouterr().out


def test_nothing_to_do_launches_nothing():
    assert norm(N=0) == 0 and norm(N=0, x=None, y=None) == 0
    L = M._library()
    assert L.W8_Quantize(None, None, 64, 0, 64, None, 64, None, 0) == 0
    for f, b in ((L.W8_Linear, (None,)), (L.W8_Gated, (None, None))):
        assert f(None, None, None, 64, None, None, 64, 0, 64, *b, 0, None, 0, 0) == 0


@pytest.mark.parametrize("kw", [dict(x=None), dict(x=X + 1), dict(codes=None), dict(codes=X + 8), dict(c_stride=40), dict(c_stride=32),
                                dict(scales=None), dict(scales=X + 1), dict(N=-1), dict(K=0), dict(K=131072), dict(dtype=7)])
def test_quantize_refuses(kw, capfd):
    a = dict(x=X, N=2, K=64, codes=X, c_stride=64, scales=X, dtype=0)
    a.update(kw)
    assert M._library().W8_Quantize(None, a["x"], 64, a["N"], a["K"], a["codes"], a["c_stride"], a["scales"], a["dtype"]) == BAD
    assert "Error" in capfd.readouterr().out


def test_sizes():
    L = M._library()
    assert L.W8_PackedBytes(64, 128, 0) == 64 * 128 + 256 and L.W8_PackedBytes(32, 128, 1) == 64 * 128 + 256
    assert L.W8_PackedBytes(65, 129, 0) == 128 * 256 + 512 and L.W8_PackedBytes(33, 1, 1) == 128 * 128 + 512
    for m, k in ((0, 64), (64, 0), (-1, 64), ((1 << 24) + 1, 64), (64, 131072)):
        assert L.W8_PackedBytes(m, k, 0) == 0 == L.W8_PackedBytes(m, k, 1)
        assert L.W8_WorkspaceBytes(m, 9, k, 0, 1) == 0
    assert L.W8_PackedBytes(1 << 24, 131071, 0) == (1 << 41) + (1 << 26)  # past 32 bits
    assert L.W8_WorkspaceBytes(64, 9, 100, 0, 1) >= 9 * 112 + 36 and L.W8_WorkspaceBytes(64, 0, 100, 0, 1) == 0
    assert L.W8_WorkspaceBytes(64, 1, 100, 0, 1) == 0  # few rows are rounded where they are read


def product(gated=False, packed=X, x=X, stride=64, scales=X, Y=X, m=64, N=2, K=64, bias=None, act=0, ws=X, room=1 << 40, dtype=0):
    L = M._library()
    f = L.W8_Gated if gated else L.W8_Linear
    return f(None, packed, x, stride, scales, Y, m, N, K, *((bias, None) if gated else (bias,)), act, ws, room, dtype)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kw", [
    dict(packed=None), dict(packed=X + 8), dict(x=None), dict(x=X + 8), dict(stride=40), dict(stride=48), dict(stride=(1 << 28) + 16),
    dict(scales=X + 2), dict(Y=None), dict(Y=X + 1), dict(m=0), dict(m=(1 << 24) + 1), dict(K=0), dict(K=131072), dict(N=-1),
    dict(N=16 * 65535 + 1), dict(bias=X + 1), dict(act=4), dict(act=-1), dict(dtype=2), dict(x=X + 1, scales=None),
    dict(scales=None, K=16384, ws=None), dict(scales=None, K=16384, room=2 * 16384), dict(scales=None, K=16384, ws=X + 8)])
def test_products_refuse(gated, kw, capfd):
    assert product(gated, **kw) == BAD
    assert "Error" in capfd.readouterr().out


@pytest.mark.parametrize("kw", [dict(c=None), dict(s=X + 2), dict(s=None), dict(p=X + 8), dict(p=None), dict(stride=63), dict(m=0), dict(k=0),
                                dict(k=131072), dict(up=(X, 63, X)), dict(up=(X, 64, X + 1)), dict(up=(X, 64, None))])
def test_pack_refuses(kw, capfd):
    a = dict(c=X, s=X, p=X, stride=64, m=2, k=64, up=(None, 0, None))
    a.update(kw)
    assert M._library().W8_Pack(None, a["c"], a["stride"], a["s"], *a["up"], a["m"], a["k"], a["p"]) == BAD
    assert "Error" in capfd.readouterr().out


def test_host_layer_refuses_tensors_that_are_not_on_a_gpu():
    x, w = torch.zeros((2, 64), dtype=torch.float16), torch.ones(64, dtype=torch.float16)
    for call in (lambda: S.rms_norm(x, w), lambda: S.rms_norm_x8(x, w), lambda: S.quantize_x8(x), lambda: S.quantize_x8(x.float()),
                 lambda: S.W8Linear(torch.zeros((4, 64), dtype=torch.int8), torch.ones(4)), lambda: S.rms_norm(x.float(), w)):
        with pytest.raises(ValueError):
            call()


def test_quantize_w8_rounds_to_half_a_step():
    w = torch.randn((40, 300), generator=torch.Generator().manual_seed(0))
    w[3] = 0
    w[4] = 1e-38
    codes8, scales = S.quantize_w8(w)
    assert codes8.dtype == torch.int8 and codes8.abs().max() == 127 and (codes8[3] == 0).all() and (codes8[4] == 0).all()
    off = (w.double() - codes8.double() * scales.double()[:, None]).abs()
    # half a step, and the rounding of a quotient up to 127
    assert (off[:3] <= scales.double()[:3, None] * (0.5 + 127 * 2.0 ** -23)).all() and off[4].max() < 2e-38


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_quantize_w8_keeps_a_broken_row_broken(value, dtype):
    w = torch.randn((4, 70), generator=torch.Generator().manual_seed(1)).to(dtype)
    want, scales = S.quantize_w8(w)
    w[2, 69] = value
    codes8, got = S.quantize_w8(w)
    assert (codes8[2] == 0).all() and got[2].isnan() and got.dtype == torch.float32
    for m in (0, 1, 3):
        assert torch.equal(codes8[m], want[m]) and got[m] == scales[m]


def test_oracle_codes_are_the_nearest():
    rng = np.random.default_rng(0)
    t = rng.standard_normal((50, 400)).astype(np.float32)
    t[0], t[1, 3], t[2, 5], t[3] = 0, np.inf, np.nan, 2.0 ** -101
    t[4] = np.arange(400) / 512.0
    t[4, 0] = 1.0
    c, m = O.encode(t)
    assert np.isnan(m[1]) and np.isnan(m[2]) and (c[:4][[0, 1, 2, 3]] == 0).all() and m[0] == 0 == m[3]
    from fractions import Fraction
    for r in range(4, 50):
        for k in range(0, 400, 7):
            q = 127 * Fraction(float(t[r, k])) / Fraction(float(m[r]))
            assert abs(q - int(c[r, k])) <= Fraction(1, 2) and (abs(q - int(c[r, k])) < Fraction(1, 2) or int(c[r, k]) % 2 == 0)


def test_oracle_rounds_once_to_16_bits():
    rng = np.random.default_rng(1)
    x = rng.standard_normal(20000) * np.exp2(rng.integers(-20, 20, 20000))
    got = O.round16(x, True)
    want = torch.from_numpy(x).to(torch.bfloat16).double().numpy()
    # torch rounds by way of float32: the oracle is at least as near
    assert (np.abs(got - x) <= np.abs(want - x)).all() and (got == want).mean() > 0.999
    assert np.array_equal(O.round16(x, False), x.astype(np.float16).astype(np.float64))
    assert np.isnan(O.round16(np.array([np.nan]), True)[0]) and O.round16(np.array([np.inf]), True)[0] == np.inf


@pytest.mark.parametrize("gated", [0, 1])
def test_room_for_rounded_rows_beside_shares_of_k(gated):
    """The kernel that adds up shares of K reads the rows' scales from memory: 16-bit rows then have codes and scales in the workspace,
    however few they are."""
    L, split = M._library(), 0
    for m in (1, 40, 256, 576, 5120, 20480):
        for n in (1, 2, 5, 8, 40, 193):
            for k in list(range(128, 8193, 128)) + [16384, 36864]:
                part = L.W8_WorkspaceBytes(m, n, k, gated, 0)
                if part:
                    split += n * k <= 8192
                    assert L.W8_WorkspaceBytes(m, n, k, gated, 1) >= part + n * (k + 4)
    assert split > 0 or not gated  # some of them few enough to be rounded where they are read


@pytest.mark.parametrize("m,k,n,gated", [(65536, 512, 8, 0), (32768, 1024, 8, 0), (32768, 1024, 2, 0), (32768, 512, 8, 1), (16384, 1024, 4, 1)])
def test_rows_are_rounded_once_where_workgroups_come_in_rounds(m, k, n, gated):
    """Each workgroup that rounds rows for itself reads all of them: several rows are rounded by a kernel before the product, into the
    workspace, where there are more workgroups than run at once; one row, and the rows of fewer, need none."""
    L = M._library()
    assert L.W8_WorkspaceBytes(m, n, k, gated, 1) >= n * (k + 4)
    assert L.W8_WorkspaceBytes(m // 4, n, k, gated, 1) == 0 == L.W8_WorkspaceBytes(min(m, 16384 if gated else 32768), 1, k, gated, 1)
