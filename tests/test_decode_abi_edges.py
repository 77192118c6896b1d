"""More refusals of the decode operators' C ABI, on a machine without a GPU."""
import pytest

import spmspm_amd as S
from spmspm_amd import decode as M
from test_decode_abi import X, attend, batch, cache


def test_a_window_whose_arithmetic_would_leave_32_bits_is_refused(capfd):
    """Only beside a table of nearly 2^31 places, which such a window does not hold."""
    c = cache(num_pages=9, page_size=1024)
    b = batch(batch=4096, total_tokens=4096, table_width=0x1fffff, table_stride=0x1fffff)
    need = M._library().KV4_AttentionWorkspaceBytes(c, b, 4, 0x7ffffb00, 0)
    assert attend(c=c, b=b, window=0x7ffffb00, ws=X, ws_bytes=need) == 1
    assert "a window of" in capfd.readouterr().out


def test_a_cache_of_sizes_that_are_not_supported_is_refused_before_it_is_allocated():
    """An odd head dimension is not the even one below it."""
    for args in ((4, 16, 2, 65), (4, 16, 2, 97), (4, 16, 2, 129), (4, 16, 2, 257), (4, 16, 2, 80), (4, 24, 2, 64), (4, 8, 2, 64),
                 (4, 2048, 2, 64), (0, 16, 2, 64), (1 << 31, 16, 2, 64), (4, 16, 0, 64), (4, 16, 4097, 64)):
        with pytest.raises(ValueError):
            S.KV4Cache(*args)


def test_a_k_whose_last_block_would_end_past_32_bits_is_refused(capfd):
    L = M._library()
    for K, group in ((2 ** 31 - 32, 32), (2 ** 31 - 64, 64), (2 ** 31 - 128, 128), (2 ** 30 + 128, 128)):
        assert L.W4_PackedBytes(16, K, group) == 0 and L.W4_WorkspaceBytes(16, 1, K, group) == 0
        assert L.W4_Pack(None, X, X, X, 16, K, group, 0, X) == 1
        assert L.W4_Linear(None, X, X, K, X, 16, 1, K, group, None, 0, None, 0, 0) == 1
    assert L.W4_PackedBytes(16, 2 ** 30, 32) == 2 ** 30 * 8 + 2 ** 25 * 32 + 2 ** 23 * 64
    # codes 8 bytes a column, scales 32 and zero points 16 a group


def test_quantize_w4_of_ranges_at_the_ends_of_the_scale_s_type():
    """Scales among fp16's subnormal numbers are rounded up, so that codes reach the group's ends; those past its largest one are it."""
    import torch
    torch.manual_seed(0)
    w = torch.randn(64, 128) * torch.logspace(-9, -3, 64)[:, None]
    codes, scales, zeros = S.quantize_w4(w, 128, torch.float16)
    back = (codes.double() - zeros.double()) * scales.double()
    step = scales.double()
    # half a step, half of one where the zero point's rounding cuts an end off, and the scale's own rounding
    assert ((back - w.double()).abs() <= 1.01 * step).all()
    w = torch.randn(8, 128) * 2e6
    codes, scales, zeros = S.quantize_w4(w, 128, torch.float16)
    assert torch.isfinite(scales).all()
    back = (codes.double() - zeros.double()) * scales.double()
    assert (back.sign() * w.double().sign() >= 0).all() and (back.abs().amax(1) >= 65504).all()
