"""Performance cases of the 8-bit linears and the norm before them: what a layer runs whose linears are neither pruned nor held
in 4 bits, in a decode step and, above all, over a prompt, where products in 8-bit integers run at twice the rate of 16 bits.

    norm     h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight, as 16-bit numbers or as 8-bit codes with a scale per row
    linear   activations in 8 bits (a scale per token) times weights in 8 bits (a scale per output channel)
    gated    two such products side by side, gate and up, and act(gate) * up of their results
    ffn      a feed-forward block of these: norm, gate and up, product, down

Sizes are those of the OPT-13B / 30B / 66B layers (hidden sizes 5120, 7168, 9216) and generic ones.

8-bit rows.  t = h * weight (or x itself) in float32, m = max |t| of the row,
    code = the whole number nearest to 127 t / m, the even one of two,     value = code * scale,   scale = m / 127 [/ rms]
so that codes depend neither on the order of a sum nor on the rounding of a quotient; a row of zeros has scale 0.  Weights: one
scale per output row.
Sums of products of codes are whole numbers; they are turned into float32, scaled, and rounded once to 16 bits.
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


def norm(name, N, K, residual, out, dtype):
    return dict(name=name, kind="norm", N=N, K=K, residual=residual, out=out, dtype=dtype)


def linear(name, M, K, N, source, dtype, bias, act):
    return dict(name=name, kind="linear", M=M, K=K, N=N, source=source, dtype=dtype, bias=bias, act=act)


def gated(name, F, K, N, source, dtype, bias, act):
    return dict(name=name, kind="gated", M=F, K=K, N=N, source=source, dtype=dtype, bias=bias, act=act)


def ffn(name, F, K, N, dtype, act):
    return dict(name=name, kind="ffn", M=F, K=K, N=N, dtype=dtype, act=act)


def listed():
    return [
        # one token of a 13B layer between two linears: launches and host time
        norm("norm_token_5120", 1, 5120, True, 16, "fp16"),
        # a decode step of a 30B layer, codes for the linears that follow
        norm("norm8_decode_n64_7168", 64, 7168, True, 8, "bf16"),
        # a ragged batch of prompts, rows of an odd length (no vector of loads is aligned), the first norm of a model
        norm("norm_odd_n1777_5121", 1777, 5121, False, 16, "bf16"),
        # a long prompt of a 66B layer
        norm("norm8_prompt_n4099_9216", 4099, 9216, True, 8, "fp16"),
        # output projection of a 13B layer for one token, 16-bit activations rounded to 8 within the call
        linear("w8_5120x5120_n1", 5120, 5120, 1, "x16", "fp16", False, "none"),
        # FFN1 of a 30B layer in a decode step behind its norm, bias and ReLU fused
        linear("w8_28672x7168_n16", 28672, 7168, 16, "norm", "fp16", True, "relu"),
        # FFN2 of a 66B layer, drafted tokens of a large batch: an odd number of columns between weights' and products' bound
        linear("w8_9216x36864_n193", 9216, 36864, 193, "x16", "bf16", True, "none"),
        # FFN1 of a 13B layer over a prompt: the matrix rate decides
        linear("w8_20480x5120_n4096", 20480, 5120, 4096, "norm", "bf16", True, "gelu"),
        # gate and up of one token
        gated("gated_13696x5120_n1", 13696, 5120, 1, "norm", "fp16", False, "silu"),
        # gate and up over a prompt, an odd number of tokens
        gated("gated_20480x5120_n3999", 20480, 5120, 3999, "norm", "bf16", False, "silu"),
        # a feed-forward block in a decode step
        ffn("ffn_13696x5120_n37", 13696, 5120, 37, "fp16", "silu"),
        # a feed-forward block over a prompt, sizes that fill no tile
        ffn("ffn_14333x4100_n2050", 14333, 4100, 2050, "bf16", "gelu"),
    ]


# The most a drawn case may ask for.
MAX_NORM = 4099 * 9216                # elements of the rows
MAX_WEIGHTS = 9216 * 36864            # of one linear; gate and up, or all of a block, count together
MAX_PRODUCTS = 2 * 20480 * 5120 * 3999


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("norm", "linear", "gated", "ffn"), (3, 5, 3, 2))[0]
    dtype = rng.choice(("fp16", "bf16"))
    if kind == "norm":
        K = _log(rng, 64, 20480)
        K = K if rng.random() < 0.4 else max(64, K // 64 * 64)
        return dict(kind=kind, N=_log(rng, 1, min(16384, MAX_NORM // K)), K=K, residual=rng.random() < 0.7,
                    out=rng.choice((8, 16)), dtype=dtype)
    parts = {"linear": 1, "gated": 2, "ffn": 3}[kind]
    while True:
        M, K = _log(rng, 256, 36864), _log(rng, 256, 36864)
        if rng.random() < 0.6:  # as models have them; the others fill no tile
            M, K = max(256, M // 128 * 128), max(256, K // 128 * 128)
        if parts * M * K <= MAX_WEIGHTS:
            break
    N = _log(rng, 1, min(8192, MAX_PRODUCTS // (parts * M * K)))
    case = dict(kind=kind, M=M, K=K, N=N, dtype=dtype)
    if kind == "ffn":
        return dict(case, act=rng.choice(("silu", "gelu")))
    return dict(case, source=rng.choice(("x16", "norm")), bias=rng.random() < 0.5,
                act=rng.choice(("none", "relu", "gelu") if kind == "linear" else ("silu", "gelu", "relu")))


# ---- inputs ----------------------------------------------------------------------------------------------------------------

def _generator(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return gen


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE)


def _stream(gen, N, K, dtype):
    """Rows of a residual stream: a few channels many times as large as the others, as trained models have them."""
    gain = 1 + 19.0 * (torch.rand(K, generator=gen, device=DEVICE) < 0.002).float()
    return (_normal(gen, N, K) * gain).to(dtype)


def _norm_inputs(gen, N, K, residual, dtype):
    s = dict(x=_normal(gen, N, K).to(dtype) if residual else _stream(gen, N, K, dtype),
             residual=_stream(gen, N, K, dtype) if residual else None)
    return dict(s, weight=(1 + 0.1 * _normal(gen, K)).to(dtype))


def _weights(gen, M, K):
    """N(0, 0.02) rounded to codes -127..127, one scale for each row."""
    codes = torch.empty((M, K), dtype=torch.int8, device=DEVICE)
    scales = torch.empty(M, dtype=torch.float32, device=DEVICE)
    rows = max(1, (1 << 25) // K)
    for r in range(0, M, rows):
        w = _normal(gen, min(rows, M - r), K) * 0.02
        s = w.abs().amax(-1) / 127
        codes[r:r + rows], scales[r:r + rows] = torch.round(w / s[:, None]).to(torch.int8), s
    return codes, scales


def _inputs(case, gen):
    N, K, dtype = case["N"], case["K"], TYPES[case["dtype"]]
    if case["kind"] == "norm":
        return _norm_inputs(gen, N, K, case["residual"], dtype)
    if case["kind"] == "ffn":
        s = _norm_inputs(gen, N, K, True, dtype)
        return dict(s, gate=_weights(gen, case["M"], K), up=_weights(gen, case["M"], K), down=_weights(gen, K, case["M"]))
    s = _norm_inputs(gen, N, K, True, dtype) if case["source"] == "norm" else dict(x=_normal(gen, N, K).to(dtype))
    names = ("gate", "up") if case["kind"] == "gated" else ("w",)
    for name in names:
        s[name] = _weights(gen, case["M"], K)
        s[name + "_bias"] = _normal(gen, case["M"]).to(dtype) if case["bias"] else None
    return s


def prepare(case, seed):
    s = dict(_inputs(case, _generator(seed)), case=case)
    if not own or case["kind"] == "norm":
        return s
    import spmspm_amd as S
    act = {"none": S.ACT_NONE, "relu": S.ACT_RELU, "gelu": S.ACT_GELU, "silu": S.ACT_SILU}[case.get("act", "none")]
    dtype = TYPES[case["dtype"]]
    if case["kind"] == "linear":
        s["layer"] = S.W8Linear(*s.pop("w"), bias=s["w_bias"], activation=act, dtype=dtype)
    else:
        s["gates"] = S.W8GatedLinear(*s.pop("gate"), *s.pop("up"), gate_bias=s.get("gate_bias"), up_bias=s.get("up_bias"),
                                     activation=act, dtype=dtype)
    if case["kind"] == "ffn":
        s["lower"] = S.W8Linear(*s.pop("down"), dtype=dtype)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------

def _run_own(s):
    import spmspm_amd as S
    case = s["case"]
    if case["kind"] == "norm":
        if case["out"] == 16:
            y = S.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"])
            return list(y) if case["residual"] else [y]
        codes, scales, *h = S.rms_norm_x8(s["x"], s["weight"], EPS, residual=s["residual"])
        return [codes * scales[:, None], *h]
    if case["kind"] == "ffn":
        codes, scales, h = S.rms_norm_x8(s["x"], s["weight"], EPS, residual=s["residual"])
        return [s["lower"](s["gates"](codes, scales)), h]
    layer = s["layer"] if case["kind"] == "linear" else s["gates"]
    if case["source"] == "x16":
        return [layer(s["x"])]
    codes, scales, h = S.rms_norm_x8(s["x"], s["weight"], EPS, residual=s["residual"])
    return [layer(codes, scales), h]


def _normed(s):
    """The rows that the norm is taken of, in 16 bits, and 1 / rms of each in float32."""
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    f = h.float()
    return h, torch.rsqrt((f * f).mean(-1) + EPS)


def _to8(t):
    """float32 rows -> codes (whole numbers in float32) and the scale of each row.  The quotients are taken in float64: one in
    some hundred thousand lies so near the middle of two codes that float32 would choose the other."""
    m = t.abs().amax(-1)
    none = m < 2.0 ** -100
    codes = torch.round(t.double() * 127 / m.masked_fill(none, math.inf).double()[:, None])
    return codes.float(), m.masked_fill(none, 0) / 127


def _act(y, act):
    if act == "relu":
        return y.clamp_min(0)
    if act == "gelu":
        return 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3)))
    return y / (1 + torch.exp(-y)) if act == "silu" else y


def _product(codes, scales, weight, bias):
    """float32 [N][M] of 8-bit rows and weights."""
    y = (codes @ weight[0].float().t()) * weight[1] * scales[:, None]
    return y if bias is None else y + bias.float()


def _source(s):
    """Codes and scales that a product reads, and what else the call before it returns."""
    if s["case"].get("source") == "x16":
        return *_to8(s["x"].float()), []
    h, r = _normed(s)
    codes, scales = _to8(h.float() * s["weight"].float())
    return codes, scales * r, [h]


def _run_norm(s):
    case = s["case"]
    h, r = _normed(s)
    if case["out"] == 16:
        y = (h.float() * r[:, None] * s["weight"].float()).to(h.dtype)
    else:
        codes, scales = _to8(h.float() * s["weight"].float())
        y = codes * (scales * r)[:, None]
    return [y, h] if case["residual"] else [y]


def _run_linear(s):
    codes, scales, h = _source(s)
    return [_act(_product(codes, scales, s["w"], s["w_bias"]), s["case"]["act"]).to(TYPES[s["case"]["dtype"]])] + h


def _run_gated(s):
    codes, scales, h = _source(s)
    gate = _act(_product(codes, scales, s["gate"], s.get("gate_bias")), s["case"]["act"])
    y = (gate * _product(codes, scales, s["up"], s.get("up_bias"))).to(TYPES[s["case"]["dtype"]])
    if s["case"]["kind"] == "ffn":
        y = _product(*_to8(y.float()), s["down"], None).to(y.dtype)
    return [y] + h


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _run_norm, "linear": _run_linear, "gated": _run_gated, "ffn": _run_gated}[state["case"]["kind"]](state)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------

def _exact_norm(s, K):
    """(rows that are normed, normed rows, 1 / rms) in float64; the rows are held in 16 bits, as the next layer reads them."""
    h = s["x"].double()
    if s["residual"] is not None:
        h = (h + s["residual"].double()).to(s["x"].dtype).double()
    inverse = 1 / torch.sqrt((h ** 2).sum(-1, keepdim=True) / K + EPS)
    return h, h * s["weight"].double() * inverse, inverse


def _exact_held(y):
    """float64 rows as 8-bit codes hold them: whole multiples of a 127th of the row's largest magnitude."""
    top = y.abs().max(-1, keepdim=True).values
    return torch.round(127 * y / torch.where(top > 0, top, torch.ones_like(top))) * (top / 127)


def _exact_product(rows, weight, bias):
    M, K = weight[0].shape
    y = torch.empty((rows.shape[0], M), dtype=torch.float64, device=DEVICE)
    part = max(1, (1 << 26) // K)
    for r in range(0, M, part):
        w = weight[0][r:r + part].double() * weight[1][r:r + part].double()[:, None]
        y[:, r:r + part] = torch.mm(rows, w.t())
    return y if bias is None else y.add_(bias.double())


def _exact_act(y, act):
    if act == "gelu":
        return torch.nn.functional.gelu(y, approximate="tanh")
    return y * torch.sigmoid(y) if act == "silu" else torch.relu(y) if act == "relu" else y


def exact(case, seed):
    s, kind, dtype = _inputs(case, _generator(seed)), case["kind"], TYPES[case["dtype"]]
    h = None
    if kind in ("norm", "ffn") or case["source"] == "norm":
        h, rows, inverse = _exact_norm(s, case["K"])
    else:
        rows = s["x"].double()
    if kind != "norm" or case["out"] == 8:
        if h is not None:  # codes are chosen before the division by the rms, which they do not depend on
            rows = _exact_held(h * s["weight"].double()) * inverse
        else:
            rows = _exact_held(rows)
    if kind == "norm":
        return [rows, h] if case["residual"] else [rows]
    if kind == "linear":
        y = _exact_act(_exact_product(rows, s["w"], s["w_bias"]), case["act"])
    else:
        gate = _exact_act(_exact_product(rows, s["gate"], s.get("gate_bias")), case["act"])
        y = gate.mul_(_exact_product(rows, s["up"], s.get("up_bias")))
        if kind == "ffn":  # the product is handed on in 16 bits
            y = _exact_product(_exact_held(y.to(dtype).double()), s["down"], None)
    return [y] if h is None else [y, h]


def work(case):
    N, K, kind = case["N"], case["K"], case["kind"]
    if kind == "norm":
        # rows (twice with a residual) and weights; h where there is a residual; y in 16 bits, or the values of its codes
        return {"bytes": N * K * (2 + (4 if case["residual"] else 0) + (2 if case["out"] == 16 else 4)) + 2 * K,
                "flops": 4 * N * K}
    M = case["M"]
    parts = {"linear": 1, "gated": 2, "ffn": 3}[kind]
    weights = parts * (M * K + 4 * M) + (2 * parts * M if case.get("bias") else 0)
    source = 6 * N * K + 2 * K if kind == "ffn" or case["source"] == "norm" else 2 * N * K
    return {"bytes": weights + source + 2 * N * (K if kind == "ffn" else M), "flops": 2 * parts * M * K * N}
