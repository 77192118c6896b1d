"""Decode operators beside the pruned linears: the 4-bit paged key/value cache with its attention, and 4-bit linears.

Thin host layer over include/decode_api.h: torch supplies device memory and streams, every size, type and stride is checked
here before a kernel sees a pointer (ValueError), and an error of the library raises RuntimeError.  Calls run on torch's
current stream unless `stream` names another; what they allocate then belongs to that stream.  There is no CPU fallback.

    cache = KV4Cache(num_pages=4096, page_size=64, kv_heads=8, head_dim=128)
    q = kv4_append(cache, k, v, block_table, seq_lens, q=q, rotation=table)   # encode k, v; rotate q, k
    y = kv4_attention(q, cache, block_table, seq_lens)                         # [tokens][heads][head_dim]
    layer = W4Linear(*quantize_w4(weight, group=128), bias=b)                  # y = layer(x)

No counterpart in the reference, whose attention and dense linears are those of its FasterTransformer host
(third_party/ft_spinfer.patch:3722-3753 is the one call that its library takes over there).
"""
import contextlib
import ctypes as C

import torch

from . import api as A

__all__ = ["KV4Cache", "kv4_append", "kv4_gather", "kv4_attention", "W4Linear", "quantize_w4", "w4_pack"]

_TYPES = {torch.float16: 0, torch.bfloat16: 1}


class _Cache(C.Structure):
    _fields_ = [("k_codes", C.c_void_p), ("k_words", C.c_void_p), ("v_codes", C.c_void_p), ("v_words", C.c_void_p),
                ("num_pages", C.c_int32), ("page_size", C.c_int32), ("kv_heads", C.c_int32), ("head_dim", C.c_int32)]


class _Batch(C.Structure):
    _fields_ = [("block_table", C.c_void_p), ("seq_lens", C.c_void_p), ("cu_tokens", C.c_void_p), ("batch", C.c_int32),
                ("table_width", C.c_int32), ("table_stride", C.c_int32), ("total_tokens", C.c_int32)]


class _Rows(C.Structure):
    _fields_ = [("data", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64)]


class _Rotary(C.Structure):
    _fields_ = [("table", C.c_void_p), ("positions", C.c_void_p), ("table_rows", C.c_int32), ("dims", C.c_int32),
                ("interleaved", C.c_int32)]


_lib = None


def _library():
    global _lib
    if _lib is None:
        L = A.library()
        cache, batch = C.POINTER(_Cache), C.POINTER(_Batch)
        L.KV4_Append.restype = C.c_int
        L.KV4_Append.argtypes = [C.c_void_p, cache, batch, _Rows, _Rows, _Rows, C.c_int, C.c_void_p, C.POINTER(_Rotary),
                                 C.c_int]
        L.KV4_Gather.restype = C.c_int
        L.KV4_Gather.argtypes = [C.c_void_p, cache, batch, C.c_void_p, C.c_void_p, C.c_int]
        L.KV4_Attention.restype = C.c_int
        L.KV4_Attention.argtypes = [C.c_void_p, cache, batch, _Rows, C.c_int, C.c_void_p, C.c_void_p, C.c_float, C.c_int,
                                    C.c_int, C.c_void_p, C.c_size_t, C.c_int]
        L.KV4_AttentionWorkspaceBytes.restype = C.c_size_t
        L.KV4_AttentionWorkspaceBytes.argtypes = [cache, batch, C.c_int, C.c_int, C.c_int]
        L.W4_PackedBytes.restype = C.c_size_t
        L.W4_PackedBytes.argtypes = [C.c_int] * 3
        L.W4_Pack.restype = C.c_int
        L.W4_Pack.argtypes = [C.c_void_p] * 4 + [C.c_int] * 4 + [C.c_void_p]
        L.W4_Linear.restype = C.c_int
        L.W4_Linear.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p] + [C.c_int] * 4 + [
            C.c_void_p, C.c_int, C.c_void_p, C.c_size_t, C.c_int]
        L.W4_WorkspaceBytes.restype = C.c_size_t
        L.W4_WorkspaceBytes.argtypes = [C.c_int] * 4
        _lib = L
    return _lib


@contextlib.contextmanager
def _context(device, stream):
    with torch.cuda.device(device):
        if stream is None:
            yield torch.cuda.current_stream(device).cuda_stream
            return
        if isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, device=device)
        with torch.cuda.stream(stream):
            yield stream.cuda_stream


def _run(device, stream, call):
    """`call(handle)` with `device` current and torch's allocations on the call's stream."""
    # the two calls behind torch.cuda.current_device() and current_stream(): 2 us less of a call's 10
    if stream is None and torch._C._cuda_getDevice() == device.index:
        return call(torch._C._cuda_getCurrentRawStream(device.index))
    with _context(device, stream) as handle:
        return call(handle)


def _raise(err, what):
    if err == A.HIP_ERROR_INVALID_VALUE:
        raise ValueError(f"{what}: the library refused its arguments (its message is on stdout)")
    if err != A.HIP_SUCCESS:
        raise RuntimeError(f"{what} failed with hipError_t {err}")


def _check(name, t, device, dtype, shape):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the cache or weight on {device}")


def _check_sizes(pages, size, heads, head_dim):
    if head_dim not in (64, 96, 128, 256):
        raise ValueError(f"head_dim {head_dim} is not 64, 96, 128 or 256")
    if size < 16 or size > 1024 or size & (size - 1):
        raise ValueError(f"page_size {size} is not a power of two from 16 to 1024")
    if pages < 1 or pages >= 1 << 31 or heads < 1 or heads > 4096:
        raise ValueError(f"a cache of {pages} pages and {heads} heads (1 to 2^31 - 1, 1 to 4096)")


class KV4Cache:
    """A paged key/value cache of one layer in 4 bits (format: include/decode_api.h): `k_codes`, `v_codes` uint8
    [num_pages][kv_heads][page_size][head_dim/2] and `k_words`, `v_words` int32 [num_pages][kv_heads][page_size], which may
    be copied, saved and moved page by page like any tensors."""

    def __init__(self, num_pages, page_size, kv_heads, head_dim, device="cuda:0"):
        _check_sizes(num_pages, page_size, kv_heads, head_dim)  # before anything is allocated
        device = torch.device(device)
        codes = (num_pages, kv_heads, page_size, head_dim // 2)
        self._adopt(torch.zeros(codes, dtype=torch.uint8, device=device),
                    torch.zeros(codes[:3], dtype=torch.int32, device=device),
                    torch.zeros(codes, dtype=torch.uint8, device=device),
                    torch.zeros(codes[:3], dtype=torch.int32, device=device))

    @classmethod
    def from_tensors(cls, k_codes, k_words, v_codes, v_words):
        """A cache over existing arrays, which it shares.  Words of places that some row sees must be those of kv4_append, or have a
        scale of 0 (a vector of zeros) or a positive normal one; the others may be anything."""
        self = object.__new__(cls)
        self._adopt(k_codes, k_words, v_codes, v_words)
        return self

    def _adopt(self, k_codes, k_words, v_codes, v_words):
        if k_codes.dim() != 4 or k_codes.device.type != "cuda":
            raise ValueError("k_codes must be [num_pages][kv_heads][page_size][head_dim/2] on the GPU")
        pages, heads, size, half = k_codes.shape
        _check_sizes(pages, size, heads, 2 * half)
        device = k_codes.device
        for name, t, dtype, shape in (("k_codes", k_codes, torch.uint8, k_codes.shape),
                                      ("v_codes", v_codes, torch.uint8, k_codes.shape),
                                      ("k_words", k_words, torch.int32, k_codes.shape[:3]),
                                      ("v_words", v_words, torch.int32, k_codes.shape[:3])):
            _check(name, t, device, dtype, shape)
        self.k_codes, self.k_words, self.v_codes, self.v_words = k_codes, k_words, v_codes, v_words
        self.num_pages, self.kv_heads, self.page_size, self.head_dim, self.device = pages, heads, size, 2 * half, device
        self._desc = _Cache(k_codes.data_ptr(), k_words.data_ptr(), v_codes.data_ptr(), v_words.data_ptr(), pages, size,
                            heads, 2 * half)

    def bytes_per_token(self):
        """Bytes one token takes, keys and values of all heads."""
        return 2 * self.kv_heads * (self.head_dim // 2 + 4)


def _batch(cache, block_table, seq_lens, cu_tokens, tokens):
    shape, strides = block_table.shape, block_table.stride()
    if len(shape) != 2 or block_table.dtype != torch.int32 or (shape[1] > 1 and strides[1] != 1) or seq_lens.dtype != torch.int32 \
            or not seq_lens.is_contiguous() or seq_lens.shape != shape[:1]:
        raise ValueError("block_table must be int32 [batch][pages], seq_lens int32 [batch]")
    n, device = seq_lens.shape[0], cache.device
    if block_table.device != device or seq_lens.device != device:
        raise ValueError(f"block_table and seq_lens must be on the cache's device {device}")
    if cu_tokens is None:
        if tokens != n:
            raise ValueError(f"{tokens} tokens of {n} sequences: cu_tokens must say whose they are")
        cu = None
    else:
        if cu_tokens.dtype != torch.int32 or cu_tokens.shape != (n + 1,) or not cu_tokens.is_contiguous() \
                or cu_tokens.device != cache.device:
            raise ValueError("cu_tokens must be int32 [batch + 1] on the cache's device")
        cu = cu_tokens.data_ptr()
    width = shape[1]
    if tokens >= 1 << 31 or (n > 1 and strides[0] >= 1 << 31):
        raise ValueError(f"{tokens} tokens, a block table of stride {strides[0]}: more than 32 bits hold")
    return _Batch(block_table.data_ptr(), seq_lens.data_ptr(), cu, n, width, strides[0] if n > 1 else max(width, 1), tokens)


def _rows(name, t, cache, heads, dtype, tokens):
    shape, strides = t.shape, t.stride()
    if len(shape) != 3 or t.dtype != dtype or shape[0] != tokens or shape[2] != cache.head_dim \
            or (heads is not None and shape[1] != heads) or strides[2] != 1:
        raise ValueError(f"{name} must be {dtype} [{tokens}][{'heads' if heads is None else heads}][{cache.head_dim}] with "
                         "its last dimension contiguous")
    if t.device != cache.device:
        raise ValueError(f"{name} is on {t.device}, the cache on {cache.device}")
    return _Rows(t.data_ptr(), strides[0], strides[1])


def _type(t):
    if t not in _TYPES:
        raise ValueError(f"{t}: activations are float16 or bfloat16")
    return _TYPES[t]


def kv4_append(cache, k, v, block_table, seq_lens, cu_tokens=None, q=None, rotation=None, interleaved=False,
               positions=None, q_out=None, stream=None):
    """Encode the keys and values of the batch's tokens into the cache, keys (and queries) rotated on the way.

    k, v [tokens][kv_heads][head_dim] and q [tokens][heads][head_dim], fp16 or bf16, slices of one product's output or any
    other strided rows.  seq_lens counts the new tokens; cu_tokens [batch + 1] says which rows are whose (None: one token
    per sequence).  rotation: float32 [positions][dims], cosines then sines; None rotates nothing and takes no q.
    positions: int32 [tokens], the rows of `rotation` to use instead of the tokens' places.  Returns the rotated queries
    (`q_out` if given, which may be q itself where that is contiguous) or None."""
    dtype, tokens = _type(k.dtype), k.shape[0]
    batch = _batch(cache, block_table, seq_lens, cu_tokens, tokens)
    kr = _rows("k", k, cache, cache.kv_heads, k.dtype, tokens)
    vr = _rows("v", v, cache, cache.kv_heads, k.dtype, tokens)
    qr, heads, rot = _Rows(None, 0, 0), 0, None
    if rotation is not None:
        if rotation.dim() != 2 or rotation.dtype != torch.float32 or not rotation.is_contiguous() \
                or rotation.shape[1] % 2 or rotation.shape[1] > cache.head_dim or rotation.device != cache.device:
            raise ValueError("rotation must be float32 [positions][dims] on the cache's device, dims even and at most "
                             "head_dim")
        if positions is not None:
            _check("positions", positions, cache.device, torch.int32, (tokens,))
        rot = _Rotary(rotation.data_ptr(), None if positions is None else positions.data_ptr(), rotation.shape[0],
                      rotation.shape[1], bool(interleaved))
    elif positions is not None:
        raise ValueError("positions without a rotation")
    if q is not None:
        if rot is None:
            raise ValueError("q is only rotated: without a rotation there is nothing to do with it")
        qr, heads = _rows("q", q, cache, None, k.dtype, tokens), q.shape[1]
        if q_out is not None:
            _check("q_out", q_out, cache.device, k.dtype, (tokens, heads, cache.head_dim))
    elif q_out is not None:
        raise ValueError("q_out without q")
    if tokens == 0:
        return q_out if q_out is not None or q is None else torch.empty_like(q, memory_format=torch.contiguous_format)
    if q is not None and heads == 0:
        raise ValueError("q has no heads")

    def call(handle):
        out = q_out
        if q is not None and out is None:
            out = k.new_empty((tokens, heads, cache.head_dim))
        err = _library().KV4_Append(handle, cache._desc, batch, kr, vr, qr, heads, None if out is None else out.data_ptr(),
                                    rot, dtype)
        _raise(err, "kv4_append")
        return out

    return _run(cache.device, stream, call)


def kv4_gather(cache, block_table, seq_lens, cu_tokens=None, total_tokens=None, dtype=torch.float16, stream=None):
    """The last tokens of every sequence as the cache holds them: k, v [total_tokens][kv_heads][head_dim].  cu_tokens says
    how many of each (None: one); with whole sequences in it this reads a cache out, to move or reuse a prefix."""
    if total_tokens is None:
        if cu_tokens is not None:
            raise ValueError("total_tokens must be given with cu_tokens (reading it from the device would wait for it)")
        total_tokens = seq_lens.shape[0]
    kind = _type(dtype)
    batch = _batch(cache, block_table, seq_lens, cu_tokens, int(total_tokens))

    def call(handle):
        shape = (int(total_tokens), cache.kv_heads, cache.head_dim)
        k = torch.empty(shape, dtype=dtype, device=cache.device)
        v = torch.empty(shape, dtype=dtype, device=cache.device)
        if shape[0]:
            _raise(_library().KV4_Gather(handle, cache._desc, batch, k.data_ptr(), v.data_ptr(), kind), "kv4_gather")
        return k, v

    return _run(cache.device, stream, call)


def kv4_attention(q, cache, block_table, seq_lens, cu_tokens=None, scale=None, window=0, max_len=0, out=None,
                  return_lse=False, stream=None):
    """Causal attention of the batch's tokens (the last of every sequence) over the cache: [tokens][heads][head_dim].

    q [tokens][heads][head_dim], fp16 or bf16, heads a multiple of kv_heads; strides multiples of 8 elements.  scale:
    head_dim ** -0.5 by default.  window > 0: only the last `window` keys of every query.  max_len: a bound of seq_lens,
    where the caller knows one (the block table's width otherwise); it decides how the work is split, not the result's
    definition.  return_lse: also the logarithms of the sums of exponentials, float32 [tokens][heads]."""
    kind, tokens = _type(q.dtype), q.shape[0]
    batch = _batch(cache, block_table, seq_lens, cu_tokens, tokens)
    rows, heads = _rows("q", q, cache, None, q.dtype, tokens), q.shape[1]
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError(f"{heads} query heads over {cache.kv_heads} key/value heads")
    if window < 0 or max_len < 0:
        raise ValueError("window and max_len must not be negative")
    window, max_len = min(window, 0x7fffffff), min(max_len, 0x7fffffff)  # what a sequence can hold; ctypes would cut the bits off
    if tokens and (rows.data % 16 or (tokens > 1 and rows.token_stride % 8) or (heads > 1 and rows.head_stride % 8)):
        raise ValueError("q's rows must be aligned to 16 bytes")
    if out is not None:
        _check("out", out, cache.device, q.dtype, (tokens, heads, cache.head_dim))

    def call(handle):
        y = q.new_empty((tokens, heads, cache.head_dim)) if out is None else out
        lse = torch.empty((tokens, heads), dtype=torch.float32, device=cache.device) if return_lse else None
        if tokens:
            L = _library()
            need = L.KV4_AttentionWorkspaceBytes(cache._desc, batch, heads, window, max_len)
            ws = cache.k_codes.new_empty(need) if need else None
            err = L.KV4_Attention(handle, cache._desc, batch, rows, heads, y.data_ptr(),
                                  None if lse is None else lse.data_ptr(),
                                  cache.head_dim ** -0.5 if scale is None else float(scale), window, max_len,
                                  None if ws is None else ws.data_ptr(), need, kind)
            _raise(err, "kv4_attention")
        return (y, lse) if return_lse else y

    return _run(cache.device, stream, call)


def quantize_w4(weight, group=128, dtype=None):
    """Round a [M][K] weight to 4 bits: codes uint8 [M][K], scales [M][K/group] (in `dtype`, the weight's own 16-bit type by
    default), zeros uint8 [M][K/group], with weight ~ scale * (code - zero).  Plain torch operations, on any device."""
    dtype = dtype or (weight.dtype if weight.dtype in _TYPES else torch.float16)
    _type(dtype)
    M, K = weight.shape
    if K % group:
        raise ValueError(f"K = {K} is not a multiple of the group {group}")
    w = weight.float().view(M, K // group, group)
    hi, lo = w.amax(-1).clamp_min(0), w.amin(-1).clamp_max(0)
    scales, info = (hi - lo) / 15, torch.finfo(dtype)
    last = info.smallest_normal * info.eps  # subnormal scales have few bits: rounded up, or codes would not reach the group's ends
    scales = torch.where(scales < info.smallest_normal, torch.ceil(scales / last) * last, scales).clamp(max=info.max).to(dtype)
    scales = torch.where(scales > 0, scales, torch.ones_like(scales))  # a group of zeros
    zeros = torch.round(-lo / scales.float()).clamp(0, 15)
    codes = (torch.round(w / scales.float()[..., None]) + zeros[..., None]).clamp(0, 15)
    return codes.to(torch.uint8).view(M, K), scales, zeros.to(torch.uint8)


def w4_pack(codes, scales, zeros, stream=None):
    """The layout that the kernels read, laid out once: an uint8 tensor.  Tensors on the GPU, shapes as quantize_w4's."""
    if codes.dim() != 2 or codes.device.type != "cuda" or scales.dim() != 2 or scales.shape[1] == 0:
        raise ValueError("codes must be [M][K] and scales [M][K/group] on the GPU")
    (M, K), device, kind = codes.shape, codes.device, _type(scales.dtype)
    group = K // scales.shape[1]
    if group not in (32, 64, 128) or K != group * scales.shape[1]:
        raise ValueError(f"{K} columns in {scales.shape[1]} groups: groups are of 32, 64 or 128 columns")
    _check("codes", codes, device, torch.uint8, (M, K))
    _check("scales", scales, device, scales.dtype, (M, K // group))
    _check("zeros", zeros, device, torch.uint8, (M, K // group))

    def call(handle):
        L = _library()
        need = L.W4_PackedBytes(M, K, group)
        if need == 0:
            raise ValueError(f"weights of {M} x {K} in groups of {group} are not supported")
        packed = torch.empty(need, dtype=torch.uint8, device=device)
        _raise(L.W4_Pack(handle, codes.data_ptr(), scales.data_ptr(), zeros.data_ptr(), M, K, group, kind,
                         packed.data_ptr()), "w4_pack")
        return packed

    return _run(device, stream, call)


class W4Linear:
    """One 4-bit weight matrix resident in HBM: y = act(x W^T + bias) for x [N][K], W[m][k] = scale * (code - zero).

    The dense counterpart of SparseLinear, for layers that are not pruned.  codes uint8 [M][K] (0..15), scales [M][K/group]
    in the activations' type (fp16 or bf16), zeros uint8 [M][K/group] (0..15), group 32, 64 or 128: see quantize_w4."""

    def __init__(self, codes, scales, zeros, bias=None, activation=A.ACT_NONE):
        packed = w4_pack(codes, scales, zeros)
        self._adopt(packed, codes.shape[0], codes.shape[1], codes.shape[1] // scales.shape[1], scales.dtype, bias, activation)

    def _adopt(self, packed, M, K, group, dtype, bias, activation):
        """Checks packed weights and takes them over."""
        self.device, self.dtype, self.packed, self.bias = packed.device, dtype, packed, bias
        self.M, self.K, self.group, self.activation = M, K, group, int(activation)
        _type(dtype)
        if packed.dtype != torch.uint8 or not packed.is_contiguous() or packed.device.type != "cuda" \
                or packed.numel() == 0 or packed.numel() != _library().W4_PackedBytes(M, K, group):
            raise ValueError(f"packed weights of another size than {M} x {K} in groups of {group} take")
        if self.activation not in (A.ACT_NONE, A.ACT_RELU, A.ACT_GELU):
            raise ValueError(f"unknown activation {activation}")
        if bias is not None:
            _check("bias", bias, self.device, self.dtype, (M,))

    def module(self):
        """The same resident weights as a `torch.nn.Module` around the registered operator."""
        from .torch_ops import W4LinearModule
        return W4LinearModule(self)

    def bytes_per_call(self, N):
        """Bytes a call with N rows of x must move: codes, scales and zero points, x and y."""
        return self.M * self.K // 2 + 5 * self.M * (self.K // self.group) // 2 + 2 * N * (self.M + self.K)

    def __call__(self, x, out=None, stream=None):
        if x.dim() != 2 or x.shape[1] != self.K or x.dtype != self.dtype or x.device != self.device:
            raise ValueError(f"x must be {self.dtype} [N][{self.K}] on {self.device}")
        N = x.shape[0]
        stride = x.stride(0) if N > 1 else self.K
        if N and (x.stride(1) != 1 or stride % 8 or stride < self.K or x.data_ptr() % 16):
            raise ValueError("x must have contiguous rows aligned to 16 bytes")
        if out is not None:
            _check("out", out, self.device, self.dtype, (N, self.M))

        def call(handle):
            y = x.new_empty((N, self.M)) if out is None else out
            if N:
                L = _library()
                need = L.W4_WorkspaceBytes(self.M, N, self.K, self.group)
                ws = self.packed.new_empty(need) if need else None
                err = L.W4_Linear(handle, self.packed.data_ptr(), x.data_ptr(), stride, y.data_ptr(), self.M, N, self.K,
                                  self.group, None if self.bias is None else self.bias.data_ptr(), self.activation,
                                  None if ws is None else ws.data_ptr(), need, _TYPES[self.dtype])
                _raise(err, "W4Linear")
            return y

        return _run(self.device, stream, call)
