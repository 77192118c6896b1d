"""MI355X (gfx950) bitmap-compressed SpMM: host layer over libSpMM_API.so.

The functions mirror the reference's public interface for this path
(csrc/SpMM_API.cuh): `InitSparseMatrixA_bitmap` (host encoder) and
`SpMM_SplitK_API` / `SpMM_SplitK_API_bitmap_v3` (device SpMM).
"""
from .api import (  # noqa: F401
    CompressedMatrix,
    InitSparseMatrixA_bitmap,
    InitSparseMatrixA_bitmap_device,
    InitSparseMatrixA_bitmap_device_onepass,
    Our_GenSparseMatrixBinFile,
    SparseLinear,
    ACT_GELU,
    ACT_NONE,
    ACT_RELU,
    ACT_SILU,
    NOALLOC_SCRATCH_BYTES,
    SpMM_SplitK_API,
    SpMM_SplitK_API_NoAlloc,
    SpMM_SplitK_API_Sized,
    SpMM_SplitK_API_BiasAct,
    SpMM_WorkspaceBytesBiasAct,
    SpMM_SplitK_API_bitmap_v3,
    SpMM_ReadWeightFiles,
    SpMM_SplitK_Auto,
    SpMM_SplitK_AutoNoAlloc,
    SpMM_SplitK_CostModel,
    SpMM_SplitK_TableSetMany,
    SpMM_SplitK_TableClear,
    SpMM_SplitK_TableLoad,
    SpMM_SplitK_TableSave,
    SpMM_SplitK_TableSet,
    SpMM_WorkspaceBytes,
    library,
    library_path,
    load_weight_files,
)


def __getattr__(name):
    # the decode operators and the 8-bit linears need torch, which the host encoder and the C ABI do without: imported when first asked for
    if name in ("KV4Cache", "kv4_append", "kv4_gather", "kv4_attention", "W4Linear", "quantize_w4", "w4_pack"):
        from . import decode
        value = globals()[name] = getattr(decode, name)
        return value
    if name in ("rms_norm", "rms_norm_x8", "quantize_x8", "quantize_w8", "w8_pack", "W8Linear", "W8GatedLinear"):
        from . import w8
        value = globals()[name] = getattr(w8, name)
        return value
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
