"""8-bit linears and the norm before them: for layers that are neither pruned nor held in 4 bits, above all over prompts.

Thin host layer over include/w8_api.h, in the manner of spmspm_amd/decode.py: every size, type and stride is checked here before a
kernel sees a pointer (ValueError), an error of the library raises RuntimeError, calls run on torch's current stream unless
`stream` names another.  There is no CPU fallback, and no backward pass: asking a result for a gradient raises RuntimeError.

    codes, scales, h = rms_norm_x8(x, norm_weight, residual=h)      # h + x, normed, in 8 bits with a scale per token
    gates = W8GatedLinear(*quantize_w8(w_gate), *quantize_w8(w_up))  # silu(gate) * up in one kernel
    down = W8Linear(*quantize_w8(w_down))
    y = down(gates(codes, scales))                                   # 16-bit rows are rounded to 8 bits within the call

No counterpart in the reference, whose dense linears and norms are those of its FasterTransformer host
(third_party/ft_spinfer.patch:3722-3753 is the one call that its library takes over there).
"""
import ctypes as C

import torch

from . import api as A
from .decode import _TYPES, _check, _raise, _run, _type

__all__ = ["rms_norm", "rms_norm_x8", "quantize_x8", "quantize_w8", "w8_pack", "W8Linear", "W8GatedLinear"]

MAX_K = 131071  # sums of products of codes stay in 32 bits


_lib = None


def _library():
    global _lib
    if _lib is None:
        L = A.library()
        p, n, s = C.c_void_p, C.c_int, C.c_int64
        L.RMS_Norm.argtypes = [p, p, s, p, s, p, C.c_float, n, n, p, s, p, s, p, s, p, n]
        L.W8_Quantize.argtypes = [p, p, s, n, n, p, s, p, n]
        L.W8_Pack.argtypes = [p, p, s, p, p, s, p, n, n, p]
        L.W8_Linear.argtypes = [p, p, p, s, p, p, n, n, n, p, n, p, C.c_size_t, n]
        L.W8_Gated.argtypes = [p, p, p, s, p, p, n, n, n, p, p, n, p, C.c_size_t, n]
        for f in (L.RMS_Norm, L.W8_Quantize, L.W8_Pack, L.W8_Linear, L.W8_Gated):
            f.restype = n
        L.W8_PackedBytes.restype, L.W8_PackedBytes.argtypes = C.c_size_t, [n] * 3
        L.W8_WorkspaceBytes.restype, L.W8_WorkspaceBytes.argtypes = C.c_size_t, [n] * 5
        _lib = L
    return _lib


def _rows(name, t, dtype, shape, device):
    """Stride of 16-bit rows."""
    strides = t.stride()
    if t.dtype != dtype or t.shape != shape or t.device != device or (strides[1] != 1 and shape[1] > 1):
        raise ValueError(f"{name} must be {dtype} {list(shape)} on {device} with contiguous rows")
    return strides[0]


def _out_rows(name, t, like, inputs, outputs=()):
    """Stride of an output's rows; it may be an input itself but not a part of one, nor lap over another output."""
    stride = _rows(name, t, like.dtype, like.shape, like.device)
    if like.shape[0] > 1 and stride < like.shape[1]:
        raise ValueError(f"{name}: rows of an output must not overlap")
    for other in inputs:
        if other is not None and _overlap(t, other) and not (
                t.data_ptr() == other.data_ptr() and (like.shape[0] < 2 or t.stride(0) == other.stride(0)) and t.shape == other.shape):
            raise ValueError(f"{name} overlaps an input without being it")
    for other in outputs:
        if other is not None and _overlap(t, other):
            raise ValueError(f"{name} overlaps another output")
    return stride


def _overlap(a, b):
    """Whether two tensors of rows may share an element: their address ranges meet, and they are not slices side by side of rows of
    one stride."""
    span = lambda t: (t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size())
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    if a0 >= b1 or b0 >= a1:
        return False
    if a.dim() != 2 or b.dim() != 2 or a.dtype != b.dtype or a.stride() != b.stride() or a.stride(1) != 1 or a.stride(0) < 1:
        return True
    stride, apart = a.stride(0), (b0 - a0) // a.element_size()
    return (b0 - a0) % a.element_size() != 0 or apart % stride < a.shape[1] or apart % stride + b.shape[1] > stride


class _NoBackward(torch.autograd.Function):
    """Stands behind a result whose inputs require a gradient."""

    @staticmethod
    def forward(ctx, name, result, *inputs):
        ctx.name = name
        return result.detach()

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name}: no backward pass")


def _without_backward(name, results, *inputs):
    """The results of a call with an input that requires a gradient: asking them for one raises, as it does behind the registered
    operators, where a result without a history would lose it.  Codes, as all whole numbers, carry none."""
    if not isinstance(results, tuple):
        return _NoBackward.apply(name, results, *inputs)
    return tuple(t if t.dtype == torch.int8 else _NoBackward.apply(name, t, *inputs) for t in results)


def _new_codes(x, N, K):
    """Room for N rows of K codes, 16-byte aligned, and their scales.  Long rows lie an odd multiple of 128 bytes apart: rows a power of
    two apart would meet on the same memory channels."""
    width = (K + 15) // 16 * 16 if K < 1024 else ((K + 127) // 128 | 1) * 128
    if K % 16:  # the last row too is readable up to a multiple of 16
        codes = x.new_empty((N, width), dtype=torch.int8)[:, :K]
    else:
        codes = x.new_empty_strided((N, K), (width, 1), dtype=torch.int8)
    return codes, width, x.new_empty(N, dtype=torch.float32)


def _norm(name, x, weight, eps, residual, residual_out, out, codes, stream):
    """Both norms: checks, allocations and the call; `codes` says that the result is in 8 bits."""
    shape, dtype, device = x.shape, x.dtype, x.device
    kind = _type(dtype)
    if len(shape) != 2 or shape[1] == 0 or not x.is_cuda:
        raise ValueError("x must be [tokens][K] on the GPU")
    N, K = shape
    most = MAX_K if codes else 1 << 24
    if N >= 1 << 31 or K > most:
        raise ValueError(f"{N} tokens of {K} numbers: 2^31 - 1 tokens and {most} numbers at most")
    if weight.shape != (K,) or weight.dtype != dtype or weight.device != device or not weight.is_contiguous():
        raise ValueError(f"weight must be {dtype} [{K}], contiguous, on {device}")
    if not 1e-20 <= eps < 3e38:
        raise ValueError(f"eps {eps}: from 1e-20 up")
    x_stride = _rows("x", x, dtype, shape, device)
    added = residual is not None
    r, r_stride = (residual.data_ptr(), _rows("residual", residual, dtype, shape, device)) if added else (None, 0)
    h_stride = y_stride = K
    if residual_out is not None:
        if not added:
            raise ValueError("residual_out without a residual: h is x itself")
        h_stride = _out_rows("residual_out", residual_out, x, (x, residual))
    if out is not None:
        y_stride = _out_rows("out", out, x, (x, residual), (residual_out,))
    if (out is not None and _overlap(out, weight)) or (residual_out is not None and _overlap(residual_out, weight)):
        raise ValueError("an output overlaps the weight")

    def call(handle):
        y, h = out, residual_out
        if codes:
            y, width, scales = _new_codes(x, N, K)
        elif y is None:
            y = x.new_empty((N, K))
        if added and h is None:
            h = x.new_empty((N, K))
        if N:
            at = y.data_ptr()
            err = _library().RMS_Norm(handle, x.data_ptr(), x_stride, r, r_stride, weight.data_ptr(), eps, N, K,
                                      h.data_ptr() if added else None, h_stride, *((None, 0, at, width, scales.data_ptr()) if codes
                                                                                  else (at, y_stride, None, 0, None)), kind)
            if err:
                _raise(err, name)
        if codes:
            return (y, scales, h) if added else (y, scales)
        return (y, h) if added else y

    results = _run(device, stream, call)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (added and residual.requires_grad)):
        return _without_backward(name, results, x, weight, residual)
    return results


def rms_norm(x, weight, eps=1e-5, residual=None, out=None, residual_out=None, stream=None):
    """y = h / sqrt(mean(h^2) + eps) * weight of rows h = x + residual (rounded to their type), or h = x.

    x, residual [tokens][K], fp16 or bf16, contiguous rows of any stride; weight [K] of that type.  Returns y, with a residual
    (y, h).  `out` and `residual_out` take y and h: new tensors by default; either may be x or the residual itself."""
    return _norm("rms_norm", x, weight, eps, residual, residual_out, out, False, stream)


def rms_norm_x8(x, weight, eps=1e-5, residual=None, residual_out=None, stream=None):
    """rms_norm with its result in 8 bits: (codes, scales), with a residual (codes, scales, h).

    codes int8 [tokens][K] (rows 16-byte aligned, in general a slice of wider ones), scales float32 [tokens];
    y ~ codes * scales.  What a W8Linear and a W8GatedLinear take."""
    return _norm("rms_norm_x8", x, weight, eps, residual, residual_out, None, True, stream)


def quantize_x8(x, stream=None):
    """Rows in 8 bits: (codes, scales) with x ~ codes * scales, as rms_norm_x8 returns them.  x [tokens][K], fp16 or bf16, of any stride."""
    kind = _type(x.dtype)
    if x.dim() != 2 or x.shape[1] == 0 or x.shape[1] > MAX_K or x.shape[0] >= 1 << 31 or x.device.type != "cuda":
        raise ValueError(f"x must be [tokens][K] on the GPU, K at most {MAX_K}")
    stride, (N, K) = _rows("x", x, x.dtype, x.shape, x.device), x.shape

    def call(handle):
        codes, width, scales = _new_codes(x, N, K)
        if N:
            err = _library().W8_Quantize(handle, x.data_ptr(), stride, N, K, codes.data_ptr(), width, scales.data_ptr(), kind)
            if err:
                _raise(err, "quantize_x8")
        return codes, scales

    results = _run(x.device, stream, call)
    return _without_backward("quantize_x8", results, x) if x.requires_grad and torch.is_grad_enabled() else results


def quantize_w8(weight):
    """Round a [M][K] weight to 8 bits: codes int8 [M][K] (-127..127), scales float32 [M], weight ~ scale * code.  A row with an
    infinity or a NaN has codes 0 and scale NaN.  Plain torch operations, on any device."""
    w = weight.float()
    scales = w.abs().amax(-1) / 127
    whole = torch.isfinite(scales)
    scales = torch.where(scales > 2.0 ** -100, scales, torch.ones_like(scales))  # a row of zeros
    codes = torch.round(w / scales[:, None]).clamp(-127, 127)
    return (torch.where(whole[:, None], codes, torch.zeros_like(codes)).to(torch.int8),
            torch.where(whole, scales, torch.full_like(scales, float("nan"))))


def w8_pack(codes, scales, up_codes=None, up_scales=None, stream=None):
    """The layout that the kernels read, laid out once: an uint8 tensor.  codes int8 [M][K] and scales float32 [M] on the GPU; with a
    second pair, of the same sizes, the weights of a gated product."""
    if codes.dim() != 2 or codes.device.type != "cuda" or codes.numel() == 0:
        raise ValueError("codes must be [M][K] on the GPU")
    (M, K), device = codes.shape, codes.device
    pairs = [(codes, scales)] + ([] if up_codes is None else [(up_codes, up_scales)])
    for c, s in pairs:
        _check("codes", c, device, torch.int8, (M, K))
        _check("scales", s, device, torch.float32, (M,))
    need = _library().W8_PackedBytes(M, K, len(pairs) == 2) if M < 1 << 31 and K < 1 << 31 else 0
    if need == 0:
        raise ValueError(f"weights of {M} x {K} are not supported")

    def call(handle):
        packed = torch.empty(need, dtype=torch.uint8, device=device)
        w = [v for c, s in pairs for v in (c.data_ptr(), K, s.data_ptr())] + ([None, 0, None] if len(pairs) == 1 else [])
        _raise(_library().W8_Pack(handle, *w, M, K, packed.data_ptr()), "w8_pack")
        return packed

    return _run(device, stream, call)


class _Product:
    """What the two linears share: packed weights and the call."""

    def _adopt(self, packed, M, K, dtype, biases, activation, gated):
        """Checks packed weights and takes them over."""
        _type(dtype)
        self.M, self.K, self.gated, self.dtype, self.activation = M, K, gated, dtype, int(activation)
        self.packed, self.device, self.biases = packed, packed.device, biases
        if packed.dtype != torch.uint8 or not packed.is_contiguous() or packed.device.type != "cuda" or packed.numel() == 0 \
                or packed.numel() != _library().W8_PackedBytes(M, K, gated):
            raise ValueError(f"packed weights of another size than {'two of ' if gated else ''}{M} x {K} take")
        if self.activation not in (A.ACT_NONE, A.ACT_RELU, A.ACT_GELU, A.ACT_SILU):
            raise ValueError(f"unknown activation {activation}")
        for b in biases:
            if b is not None:
                _check("bias", b, self.device, dtype, (M,))
        self._kind, self._need = _TYPES[dtype], {}

    def bytes_per_call(self, N):
        """Bytes a call with N rows of 8-bit x must move: weights and scales, x and y."""
        return (2 if self.gated else 1) * self.M * (self.K + 4) + N * (self.K + 4 + 2 * self.M)

    def __call__(self, x, scales=None, out=None, stream=None):
        """x int8 [N][K] with float32 scales [N] (of rms_norm_x8 or quantize_x8; codes whose rows are not aligned to 16 bytes, and readable
        up to a multiple of 16, are copied first), or 16-bit [N][K] in the layer's type, which is rounded to 8 bits first.  Returns
        [N][M] in the layer's type."""
        shape, K = x.shape, self.K
        if len(shape) != 2 or shape[1] != K or x.device != self.device:
            raise ValueError(f"x must be [N][{K}] on {self.device}")
        N, (stride, inner) = shape[0], x.stride()
        if N > 16 * 65535:
            raise ValueError(f"{N} rows of x: {16 * 65535} at most")
        if inner != 1 and N and K > 1:
            raise ValueError("x must have contiguous rows")
        if scales is None:
            if x.dtype != self.dtype:
                raise ValueError(f"x must be {self.dtype}, or int8 with its scales")
        else:
            if x.dtype != torch.int8:
                raise ValueError("scales belong to int8 codes")
            if scales.shape != (N,) or scales.dtype != torch.float32 or scales.device != self.device or not scales.is_contiguous():
                raise ValueError(f"scales must be float32 [{N}], contiguous, on {self.device}")
            wide = (K + 15) // 16 * 16
            if N and (x.data_ptr() % 16 or (N > 1 and (stride % 16 or stride < wide or stride > 1 << 28))
                      or (wide != K and x.storage_offset() + (N - 1) * stride + wide > x.untyped_storage().nbytes())):
                stride = 0  # not as the kernels read rows: copied
            elif N == 1:
                stride = wide
        if out is not None:
            _check("out", out, self.device, self.dtype, (N, self.M))
            if any(_overlap(out, t) for t in (x, scales, self.packed, *self.biases) if t is not None):
                raise ValueError("out overlaps an input")

        def call(handle):
            y = self.packed.new_empty((N, self.M), dtype=self.dtype) if out is None else out
            if N:
                L, M, gated, codes, width = _library(), self.M, self.gated, x, stride
                if scales is not None and not stride:
                    codes, width, _ = _new_codes(x, N, K)
                    codes.copy_(x)
                need = self._need.get((N, scales is None))
                if need is None:  # of the sizes alone: looked up once for each N that comes
                    if len(self._need) >= 1024:
                        self._need.clear()
                    need = self._need[N, scales is None] = L.W8_WorkspaceBytes(M, N, K, gated, scales is None)
                ws = self.packed.new_empty(need) if need else None
                err = (L.W8_Gated if gated else L.W8_Linear)(
                    handle, self.packed.data_ptr(), codes.data_ptr(), width, None if scales is None else scales.data_ptr(),
                    y.data_ptr(), M, N, K, *[None if b is None else b.data_ptr() for b in self.biases], self.activation,
                    None if ws is None else ws.data_ptr(), need, self._kind)
                if err:
                    _raise(err, type(self).__name__)
            return y

        y = _run(self.device, stream, call)
        if torch.is_grad_enabled() and (x.requires_grad or (scales is not None and scales.requires_grad) or self._learns()):
            return _without_backward(type(self).__name__, y, x, scales, *self.biases)
        return y

    def _learns(self):
        """Whether a bias requires a gradient."""
        for b in self.biases:
            if b is not None and b.requires_grad:
                return True
        return False


class W8Linear(_Product):
    """One 8-bit weight matrix resident in HBM: y = act(x W^T + bias), W[m][k] = scale[m] * code[m][k], x in 8 bits with a scale per row.

    codes int8 [M][K], scales float32 [M] (see quantize_w8); bias [M] and y in `dtype`, fp16 or bf16."""

    def __init__(self, codes, scales, bias=None, activation=A.ACT_NONE, dtype=torch.float16):
        _type(dtype)
        self._adopt(w8_pack(codes, scales), codes.shape[0], codes.shape[1], dtype, (bias,), activation, False)

    def module(self):
        """The same resident weights as a `torch.nn.Module` around the registered operator."""
        from .torch_ops import W8LinearModule
        return W8LinearModule(self)


class W8GatedLinear(_Product):
    """Gate and up of a feed-forward block in one kernel: y = act(x G^T + gate_bias) * (x U^T + up_bias), weights and x in 8 bits as
    W8Linear's, `activation` of the gate (SiLU by default)."""

    def __init__(self, gate_codes, gate_scales, up_codes, up_scales, gate_bias=None, up_bias=None, activation=A.ACT_SILU,
                 dtype=torch.float16):
        _type(dtype)
        self._adopt(w8_pack(gate_codes, gate_scales, up_codes, up_scales), gate_codes.shape[0], gate_codes.shape[1], dtype,
                    (gate_bias, up_bias), activation, True)

    def module(self):
        """The same resident weights as a `torch.nn.Module` around the registered operator."""
        from .torch_ops import W8LinearModule
        return W8LinearModule(self)
