"""Decoder layers on this framework's operators, as a decode step or a prompt runs them.  One of an OPT-shaped model:

    h = x + out(attention(append(qkv(norm(x)))))        qkv and out: pruned weights, bitmap SpMM
    y = h + ffn2(relu(ffn1(norm(h))))                    ffn1 and ffn2: 4-bit weights

Attention reads the layer's 4-bit key/value cache, to which the step's tokens are appended first.  The reference's
counterpart is the patched FasterTransformer decoder layer (third_party/ft_spinfer.patch:2335-2357 its weights,
:3722-3753 its linear calls).

and one of a model with root-mean-square norms and a gated feed-forward block, all of whose linears are held in 8 bits:

    h = x + residual                                     added by the norm that follows
    a = out(attention(append(qkv(norm(h)))))
    y = down(act(gate(norm(h + a))) * up(norm(h + a)))   and h + a, which the next layer's norm adds to y

    python -m spmspm_amd.decode_layer            a prompt and some decode steps with random weights, timed
    python -m spmspm_amd.decode_layer --gated    the same of the second
"""
import sys

import torch

from . import api as A
from . import decode as D
from . import w8 as W
from .torch_ops import SparseLinearModule


def _columns(n):
    """The smallest number of columns the SpMM runs that is not below n."""
    for c in (8, 16, 32, 64):
        if n <= c:
            return c
    return -(-n // 128) * 128


class DecodeLayer:
    """Weights of one layer.  qkv, out: SparseLinearModule (or any callable on [N][K] fp16); ffn1, ffn2: W4Linear.  A pruned
    linear's N is one of the SpMM's widths: rows are padded with zeros up to it."""

    def __init__(self, heads, qkv, out, ffn1, ffn2, norm1, norm2, kv_heads=None, rotation=None, interleaved=False):
        self.heads, self.kv_heads = heads, kv_heads or heads
        self.qkv, self.out, self.ffn1, self.ffn2, self.norm1, self.norm2 = qkv, out, ffn1, ffn2, norm1, norm2
        self.rotation, self.interleaved = rotation, interleaved

    @classmethod
    def random(cls, hidden, heads, sparsity=0.6, group=128, seed=0, device="cuda:0"):
        """An OPT-shaped layer (FFN of 4 hidden) with N(0, 0.02) weights: pruned at random, or rounded to 4 bits."""
        gen = torch.Generator(device=device)
        gen.manual_seed(seed)
        normal = lambda m, k: torch.randn((m, k), generator=gen, device=device) * 0.02

        def pruned(m, k):
            w = normal(m, k)
            w = w.masked_fill_(torch.rand(w.shape, generator=gen, device=device) < sparsity, 0).half()
            values, bitmaps, offsets = A.InitSparseMatrixA_bitmap_device(w)
            return SparseLinearModule(m, k, values, bitmaps, offsets, bias=torch.zeros(m, dtype=torch.float16, device=device))

        def rounded(m, k, activation):
            return D.W4Linear(*D.quantize_w4(normal(m, k).half(), group),
                              bias=torch.zeros(m, dtype=torch.float16, device=device), activation=activation)

        norm = lambda: torch.nn.LayerNorm(hidden, device=device, dtype=torch.float16)
        return cls(heads, pruned(3 * hidden, hidden), pruned(hidden, hidden), rounded(4 * hidden, hidden, A.ACT_RELU),
                   rounded(hidden, 4 * hidden, A.ACT_NONE), norm(), norm())

    def _sparse(self, linear, x):
        n, c = x.shape[0], _columns(x.shape[0])
        return linear(x if n == c else torch.cat((x, x.new_zeros((c - n, x.shape[1])))))[:n]

    @torch.no_grad()
    def __call__(self, x, cache, block_table, seq_lens, cu_tokens=None, max_len=0):
        """x [tokens][hidden] fp16: the tokens of the step, the last of every sequence; seq_lens counts them."""
        tokens, hidden = x.shape
        d, kv = cache.head_dim, self.kv_heads
        rows = self._sparse(self.qkv, self.norm1(x)).view(tokens, self.heads + 2 * kv, d)
        q, k, v = rows.split((self.heads, kv, kv), 1)
        turned = D.kv4_append(cache, k, v, block_table, seq_lens, cu_tokens, q=q if self.rotation is not None else None,
                              rotation=self.rotation, interleaved=self.interleaved)
        y = D.kv4_attention(q if turned is None else turned, cache, block_table, seq_lens, cu_tokens, max_len=max_len)
        h = x + self._sparse(self.out, y.view(tokens, self.heads * d))
        return h + self.ffn2(self.ffn1(self.norm2(h)))


class GatedLayer:
    """Weights of one layer with root-mean-square norms and a gated feed-forward block.  qkv, out, down: W8Linear; gates:
    W8GatedLinear; norm1, norm2: [hidden] in the linears' type.  What a norm writes and a linear reads is 8 bits, what goes
    through the cache 4."""

    def __init__(self, heads, qkv, out, gates, down, norm1, norm2, kv_heads=None, rotation=None, interleaved=False, eps=1e-5):
        self.heads, self.kv_heads, self.eps = heads, kv_heads or heads, eps
        self.qkv, self.out, self.gates, self.down, self.norm1, self.norm2 = qkv, out, gates, down, norm1, norm2
        self.rotation, self.interleaved = rotation, interleaved

    @classmethod
    def random(cls, hidden, heads, ffn, kv_heads=None, rotation=None, dtype=torch.float16, seed=0, device="cuda:0"):
        """N(0, 0.02) weights rounded to 8 bits, SiLU of the gate."""
        gen = torch.Generator(device=device)
        gen.manual_seed(seed)
        weight = lambda m, k: W.quantize_w8(torch.randn((m, k), generator=gen, device=device) * 0.02)
        gain = lambda: (1 + 0.1 * torch.randn(hidden, generator=gen, device=device)).to(dtype)
        size = hidden // heads
        return cls(heads, W.W8Linear(*weight((heads + 2 * (kv_heads or heads)) * size, hidden), dtype=dtype),
                   W.W8Linear(*weight(hidden, hidden), dtype=dtype),
                   W.W8GatedLinear(*weight(ffn, hidden), *weight(ffn, hidden), dtype=dtype),
                   W.W8Linear(*weight(hidden, ffn), dtype=dtype), gain(), gain(), kv_heads, rotation)

    @torch.no_grad()
    def __call__(self, x, residual, cache, block_table, seq_lens, cu_tokens=None, max_len=0):
        """x and residual [tokens][hidden]: what the layer before returned (residual None: x is the stream itself).  Returns (y, h),
        whose sum is the stream behind this layer."""
        tokens, d, kv = x.shape[0], cache.head_dim, self.kv_heads
        codes, scales, *h = W.rms_norm_x8(x, self.norm1, self.eps, residual)
        q, k, v = self.qkv(codes, scales).view(tokens, self.heads + 2 * kv, d).split((self.heads, kv, kv), 1)
        turned = D.kv4_append(cache, k, v, block_table, seq_lens, cu_tokens, q=q if self.rotation is not None else None,
                              rotation=self.rotation, interleaved=self.interleaved)
        a = D.kv4_attention(q if turned is None else turned, cache, block_table, seq_lens, cu_tokens, max_len=max_len)
        a = self.out(a.view(tokens, self.heads * d))
        codes, scales, h = W.rms_norm_x8(a, self.norm2, self.eps, h[0] if h else x)
        return self.down(self.gates(codes, scales)), h


def main():
    gated = "--gated" in sys.argv[1:]
    hidden, heads, batch, prompt, steps, page = 5120, 40, 8, 128, 32, 16
    layer = GatedLayer.random(hidden, heads, 13696) if gated else DecodeLayer.random(hidden, heads)

    def run(x, *batch):
        if not gated:
            return layer(x, *batch)
        y, h = layer(x, None, *batch)
        return y + h

    pages = -(-(prompt + steps) // page)
    cache = D.KV4Cache(batch * pages, page, heads, hidden // heads)
    table = torch.randperm(batch * pages, device="cuda").int().view(batch, pages)
    x = torch.randn((batch * prompt, hidden), device="cuda").half()
    lens = torch.full((batch,), prompt, dtype=torch.int32, device="cuda")
    cu = torch.arange(0, batch * prompt + 1, prompt, dtype=torch.int32, device="cuda")
    y = run(x, cache, table, lens, cu)
    x = y.view(batch, prompt, hidden)[:, -1].contiguous()
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for step in range(steps):
        if step == steps // 2:
            start.record()
        lens += 1
        x = run(x, cache, table, lens)
    stop.record()
    torch.cuda.synchronize()
    us = start.elapsed_time(stop) / (steps - steps // 2) * 1e3
    print(f"{batch} sequences, {prompt} tokens of prompt, {steps} steps through one layer of {hidden}: {us:.1f} us a step, "
          f"{cache.bytes_per_token()} bytes a token in the cache (fp16: {4 * hidden})")


if __name__ == "__main__":
    main()
