"""More refusals of the decode operators' C ABI, on a machine without a GPU."""
from spmspm_amd import decode as M
from test_decode_abi import X, attend, batch, cache


def test_a_window_whose_arithmetic_would_leave_32_bits_is_refused(capfd):
    """Only beside a table of nearly 2^31 places, which such a window does not hold."""
    c = cache(num_pages=9, page_size=1024)
    b = batch(batch=4096, total_tokens=4096, table_width=0x1fffff, table_stride=0x1fffff)
    need = M._library().KV4_AttentionWorkspaceBytes(c, b, 4, 0x7ffffb00, 0)
    assert attend(c=c, b=b, window=0x7ffffb00, ws=X, ws_bytes=need) == 1
    assert "a window of" in capfd.readouterr().out
