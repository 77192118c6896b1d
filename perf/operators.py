"""Performance cases of the decode operators: the 4-bit paged key/value cache and its attention, and linears with 4-bit weights.

    append     keys and values of new tokens go into the cache, rotated and encoded on the way; queries are rotated beside
               them; the new tokens are then read back from the cache as the values that it holds
    attention  the new tokens of every sequence attend to all that the cache holds of it (causal, optionally a window)
    linear     a small batch through weights of 4 bits with a scale and a zero point per group

Sizes are those of the OPT-13B / 30B / 66B layers (heads of 128, 40 heads, sequences up to 2048, the FFN shapes) and generic
ones: shared key/value heads, long caches, small heads.

Cache format.  A page holds P tokens of every key/value head: codes uint8 [page][head][P][D/2], element 2b in the low and
2b+1 in the high half of byte b, and one int32 word per token [page][head][P]: the bits of a float32 scale whose four lowest
mantissa bits are the zero point.  value = float32(word) * (code - (word & 15)).
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def append(name, B, n, ctx, hq, hkv, d, page, rot, interleaved, dtype, spread):
    return dict(name=name, kind="append", B=B, n=n, ctx=ctx, hq=hq, hkv=hkv, d=d, page=page, rot=rot,
                interleaved=interleaved, dtype=dtype, spread=spread)


def attention(name, B, n, length, hq, hkv, d, page, window, dtype, spread):
    return dict(name=name, kind="attention", B=B, n=n, length=length, hq=hq, hkv=hkv, d=d, page=page, window=window,
                dtype=dtype, spread=spread)


def linear(name, M, K, N, group, dtype, bias, act):
    return dict(name=name, kind="linear", M=M, K=K, N=N, group=group, dtype=dtype, bias=bias, act=act)


def listed():
    return [
        # one token of one sequence, small heads, part of each head rotated in neighbouring pairs: launches and host time
        append("append_token_b1_d64", 1, 1, 100, 8, 8, 64, 16, 32, True, "fp16", 0),
        # a decode step of a 13B layer: sixteen sequences of different lengths, learned positions (no rotation)
        append("append_decode_b16_h40", 16, 1, 2046, 40, 40, 128, 16, 0, False, "fp16", 1),
        # prompts of four requests at once, ragged, shared key/value heads, whole heads rotated
        append("append_prompt_b4_gqa", 4, 4093, 0, 32, 8, 128, 64, 128, False, "bf16", 2),
        # one short sequence of a 13B layer: latency
        attention("attend_b1_len77_h40", 1, 1, 77, 40, 40, 128, 16, 0, "fp16", 0),
        # a decode step of a 13B layer, sequences up to the model's 2048 tokens, every head with its own keys
        attention("attend_decode_b16_h40", 16, 1, 2048, 40, 40, 128, 16, 0, "fp16", 1),
        # long contexts in a batch, eight query heads to a key/value head
        attention("attend_decode_b32_gqa8", 32, 1, 16384, 64, 8, 128, 64, 0, "bf16", 2),
        # one long document: few rows, the work lies along the cache
        attention("attend_long_b1_131k", 1, 1, 131071, 32, 8, 128, 128, 0, "fp16", 0),
        # checking drafted tokens, five at a time, small heads, a sliding window
        attention("attend_draft_b8_n5_d64", 8, 5, 4095, 32, 4, 64, 16, 1024, "bf16", 3),
        # a chunk of a long prompt: many rows, matrix products decide
        attention("attend_chunk_b2_n1024", 2, 1024, 8192, 32, 8, 128, 64, 0, "bf16", 4),
        # output projection of a 13B layer for one token
        linear("w4_5120x5120_n1", 5120, 5120, 1, 128, "fp16", False, "none"),
        # FFN1 of a 30B layer in a decode step, bias and ReLU fused
        linear("w4_28672x7168_n16", 28672, 7168, 16, 128, "fp16", True, "relu"),
        # FFN2 of a 66B layer, batched decode, finer groups
        linear("w4_9216x36864_n64", 9216, 36864, 64, 64, "bf16", True, "none"),
    ]


# The most a drawn case may ask for.
MAX_CACHE = 32 * 16384 * 8 * 128      # elements of the keys
MAX_SCORES = 2 * 1024 * 8192 * 32     # query rows times keys
MAX_WEIGHTS = 9216 * 36864
MAX_TOKENS = 4 * 4093


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    hkv = rng.choice((1, 2, 4, 5, 8, 12, 40))
    share = rng.choice((1, 1, 2, 4, 7, 8) if hkv <= 12 else (1,))
    return hkv * share, hkv


def draw(rng):
    kind = rng.choices(("append", "attention", "linear"), (3, 6, 4))[0]
    dtype = rng.choice(("fp16", "bf16"))
    if kind == "linear":
        group = rng.choice((32, 64, 128))
        while True:
            M, K = _log(rng, 512, 36864), group * max(1, _log(rng, 512, 36864) // group)
            if M * K <= MAX_WEIGHTS:
                break
        return dict(kind=kind, M=M, K=K, N=_log(rng, 1, 64), group=group, dtype=dtype, bias=rng.random() < 0.5,
                    act=rng.choice(("none", "relu", "gelu")))
    (hq, hkv), d, page = _heads(rng), rng.choice((64, 96, 128, 128, 256)), rng.choice((16, 32, 64, 128, 256))
    case = dict(kind=kind, hq=hq, hkv=hkv, d=d, page=page, dtype=dtype, spread=rng.randint(0, 1 << 20))
    if kind == "append":
        B = _log(rng, 1, 64)
        n = 1 if rng.random() < 0.5 else _log(rng, 1, max(1, MAX_TOKENS // (B * max(1, hq // 32))))
        case.update(B=B, n=n, ctx=_log(rng, 1, 4096), rot=rng.choice((0, d // 2, d)), interleaved=rng.random() < 0.5)
        return case
    B = _log(rng, 1, 64)
    length = _log(rng, 16, max(16, min(131072, MAX_CACHE // (B * hkv * d))))
    n = 1
    if rng.random() < 0.4:
        n = min(length, _log(rng, 2, max(2, min(1024, MAX_SCORES // (B * length * hq)))))
    case.update(B=B, length=length, n=n, window=0 if rng.random() < 0.75 else _log(rng, 16, 4096))
    return case


def _sequences(case):
    """(new tokens, tokens in the cache with them) of every sequence: the first has the full size, the others lie between
    half of it and all of it (spread 0: all have the full size)."""
    top, new = (case["ctx"] + case["n"], case["n"]) if case["kind"] == "append" else (case["length"], case["n"])
    rng = random.Random(case["spread"])
    out = []
    for b in range(case["B"]):
        full = b == 0 or case["spread"] == 0
        n = new if full else rng.randint((new + 1) // 2, new)
        length = top if full else max(n, rng.randint((top + 1) // 2, top))
        out.append((n, length))
    return out


# ---- the cache format in elementary operations ----------------------------------------------------------------------------

def _encode(x):
    """float32 [..., D] -> codes (int32, 0..15), words (int32): a scale and a zero point for each vector."""
    hi, lo = x.amax(-1).clamp_min(0), x.amin(-1).clamp_max(0)
    fifteenth = 1.0 / 15.0
    scale = hi * fifteenth - lo * fifteenth
    word = (scale.view(torch.int32) + 8) & -16
    word = torch.where(scale < 2.0 ** -100, torch.full_like(word, 0x3F800000), word)
    zero = torch.round(-lo * (1.0 / word.view(torch.float32))).clamp(0, 15)
    word = word | zero.nan_to_num(0).to(torch.int32)
    codes = (torch.round(x * (1.0 / word.view(torch.float32))[..., None]) + zero[..., None]).clamp(0, 15)
    bad = ~torch.isfinite(scale)
    word = torch.where(bad, torch.full_like(word, 0x7FC00000), word)
    return codes.masked_fill(bad[..., None], 0).to(torch.int32), word


def _decode(packed, word):
    """uint8 [..., D/2], int32 [...] -> float32 [..., D]"""
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    return word.view(torch.float32)[..., None] * (codes.to(torch.float32) - (word & 15).to(torch.float32)[..., None])


def _pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def _rotate(x, table, positions, interleaved):
    """float32 [T][H][D], table [positions][rot] = cosines, then sines; elements past `rot` stay."""
    half = table.shape[1] // 2
    rows = table[positions]
    cos, sin = rows[:, None, :half], rows[:, None, half:]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


# ---- inputs ----------------------------------------------------------------------------------------------------------------

def _generator(seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return gen


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE)


def _paged(case, gen, fill):
    """Pages in random order with a few to spare; what lies past a sequence's end is left over from earlier ones."""
    seqs, P, H, D = _sequences(case), case["page"], case["hkv"], case["d"]
    counts = [-(-length // P) for _, length in seqs]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((len(seqs), max(counts)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    new = lambda *shape, dtype: torch.zeros((pages, H, P) + shape, dtype=dtype, device=DEVICE)
    cache = dict(k_codes=new(D // 2, dtype=torch.uint8), k_words=new(dtype=torch.int32),
                 v_codes=new(D // 2, dtype=torch.uint8), v_words=new(dtype=torch.int32))
    if fill:
        # a few channels of the keys are several times as large as the others, as trained models have them
        gain = 0.7 + 3.0 * (torch.rand((H, 1, D), generator=gen, device=DEVICE) < 0.05).float()
        step = max(1, (1 << 25) // (H * P * D))
        for at in range(0, pages, step):
            stop = min(pages, at + step)
            for side in ("k", "v"):
                x = _normal(gen, stop - at, H, P, D)
                codes, words = _encode(x * gain if side == "k" else x * 0.5)
                cache[side + "_codes"][at:stop] = _pack(codes)
                cache[side + "_words"][at:stop] = words
    lens = torch.tensor([length for _, length in seqs], dtype=torch.int32, device=DEVICE)
    cu = [0]
    for n, _ in seqs:
        cu.append(cu[-1] + n)
    return cache, table, lens, cu


def _positions(case, device):
    """Positions of the new tokens in their sequences, and the sequence that each belongs to."""
    where, which = [], []
    for b, (n, length) in enumerate(_sequences(case)):
        where += range(length - n, length)
        which += [b] * n
    return torch.tensor(where, device=device), torch.tensor(which, device=device)


def _rotation_table(rows, rot):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * (10000.0 ** (-torch.arange(rot // 2) / max(1, rot // 2)))
    return torch.cat((angle.cos(), angle.sin()), 1).float().to(DEVICE)


def _append_inputs(case, gen):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    cache, table, lens, cu = _paged(case, gen, False)
    # q, k and v are slices of one product's output
    qkv = _normal(gen, cu[-1], hq + 2 * hkv, d).to(TYPES[case["dtype"]])
    rotation = _rotation_table(case["ctx"] + case["n"], case["rot"]) if case["rot"] else None
    return dict(cache=cache, table=table, lens=lens, cu=cu, q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:],
                rotation=rotation)


def _attention_inputs(case, gen):
    cache, table, lens, cu = _paged(case, gen, True)
    q = _normal(gen, cu[-1], case["hq"], case["d"]).to(TYPES[case["dtype"]])
    return dict(cache=cache, table=table, lens=lens, cu=cu, q=q)


def _linear_inputs(case, gen):
    """Weights N(0, 0.02) rounded to codes 0..15 with one scale and zero point per row and group."""
    M, K, N, G, dtype = case["M"], case["K"], case["N"], case["group"], TYPES[case["dtype"]]
    codes = torch.empty((M, K), dtype=torch.uint8, device=DEVICE)
    scales = torch.empty((M, K // G), dtype=dtype, device=DEVICE)
    zeros = torch.empty((M, K // G), dtype=torch.uint8, device=DEVICE)
    rows = max(1, (1 << 25) // K)
    for r in range(0, M, rows):
        w = (_normal(gen, min(rows, M - r), K) * 0.02).view(-1, K // G, G)
        hi, lo = w.amax(-1), w.amin(-1)
        s = ((hi - lo) / 15).to(dtype)
        z = torch.round(-lo / s.float()).clamp(0, 15)
        codes[r:r + rows] = (torch.round(w / s.float()[..., None]) + z[..., None]).clamp(0, 15).to(torch.uint8).flatten(1)
        scales[r:r + rows], zeros[r:r + rows] = s, z.to(torch.uint8)
    x = _normal(gen, N, K).to(dtype)
    bias = _normal(gen, M).to(dtype) if case["bias"] else None
    return dict(codes=codes, scales=scales, zeros=zeros, x=x, bias=bias)


INPUTS = {"append": _append_inputs, "attention": _attention_inputs, "linear": _linear_inputs}


def prepare(case, seed):
    state = dict(INPUTS[case["kind"]](case, _generator(seed)), case=case)
    if not own:
        if case["kind"] != "linear":
            state["where"], state["which"] = _positions(case, DEVICE)
            state["new"] = torch.tensor([n for n, _ in _sequences(case)], device=DEVICE)
        return state
    import spmspm_amd as S
    if case["kind"] == "linear":
        act = {"none": S.ACT_NONE, "relu": S.ACT_RELU, "gelu": S.ACT_GELU}[case["act"]]
        state["layer"] = S.W4Linear(state.pop("codes"), state.pop("scales"), state.pop("zeros"), bias=state["bias"],
                                    activation=act)
        return state
    c = state["cache"]
    state["cache"] = S.KV4Cache.from_tensors(c["k_codes"], c["k_words"], c["v_codes"], c["v_words"])
    cu = state["cu"]
    # one new token for every sequence needs no list of where each one's tokens begin
    state["cu"] = None if cu[-1] == case["B"] and case["n"] == 1 else torch.tensor(cu, dtype=torch.int32, device=DEVICE)
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------------

def _run_own(s):
    import spmspm_amd as S
    case = s["case"]
    if case["kind"] == "linear":
        return s["layer"](s["x"])
    if case["kind"] == "attention":
        return S.kv4_attention(s["q"], s["cache"], s["table"], s["lens"], cu_tokens=s["cu"], window=case["window"],
                               max_len=case["length"])
    turned = S.kv4_append(s["cache"], s["k"], s["v"], s["table"], s["lens"], cu_tokens=s["cu"],
                          q=s["q"] if case["rot"] else None, rotation=s["rotation"], interleaved=case["interleaved"])
    k, v = S.kv4_gather(s["cache"], s["table"], s["lens"], cu_tokens=s["cu"], total_tokens=s["k"].shape[0],
                        dtype=s["k"].dtype)
    return [k, v] if turned is None else [k, v, turned]


def _run_append(s):
    case, cache = s["case"], s["cache"]
    where, which = s["where"], s["which"]
    dtype, P = s["k"].dtype, case["page"]
    k, v, q = s["k"].float(), s["v"].float(), None
    if case["rot"]:
        k = _rotate(k, s["rotation"], where, case["interleaved"])
        q = _rotate(s["q"].float(), s["rotation"], where, case["interleaved"]).to(dtype)
    page, slot = s["table"][which, where // P].long(), where % P
    out = []
    for side, x in (("k", k), ("v", v)):
        codes, words = _encode(x)
        cache[side + "_codes"][page, :, slot] = _pack(codes)
        cache[side + "_words"][page, :, slot] = words
    for side in ("k", "v"):
        out.append(_decode(cache[side + "_codes"][page, :, slot], cache[side + "_words"][page, :, slot]).to(dtype))
    return out if q is None else out + [q]


def _run_attention(s):
    """All sequences of the batch at once, padded to the longest, in float32."""
    case, cache, table = s["case"], s["cache"], s["table"]
    B, hq, hkv, d, P = case["B"], case["hq"], case["hkv"], case["d"], case["page"]
    share, T = hq // hkv, table.shape[1] * P
    rows = table.clamp_min(0).long()
    # [B][hkv][T][D]
    take = lambda side: _decode(cache[side + "_codes"][rows].transpose(1, 2).reshape(B, hkv, T, d // 2),
                                cache[side + "_words"][rows].transpose(1, 2).reshape(B, hkv, T))
    where, which = s["where"], s["which"]
    slot = where - (s["lens"] - s["new"])[which]
    q = torch.zeros((B, case["n"], hq, d), device=DEVICE)
    q[which, slot] = s["q"].float()
    at = torch.zeros((B, case["n"]), dtype=torch.long, device=DEVICE)
    at[which, slot] = where
    # [B][hkv][n * share][D]: the query heads of one key/value head are rows of one product
    q = q.view(B, case["n"], hkv, share, d).permute(0, 2, 1, 3, 4).reshape(B, hkv, case["n"] * share, d)
    scores = torch.matmul(q, take("k").transpose(2, 3)).view(B, hkv, case["n"], share, T)
    scores *= d ** -0.5
    key = torch.arange(T, device=DEVICE)
    hidden = key > at[..., None]
    if case["window"]:
        hidden |= key <= at[..., None] - case["window"]
    scores.masked_fill_(hidden[:, None, :, None], float("-inf"))
    scores -= scores.amax(-1, keepdim=True)
    p = scores.exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hkv, case["n"] * share, T), take("v")).view(B, hkv, case["n"], share, d) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(B, case["n"], hq, d)
    return o[which, slot].to(s["q"].dtype)


def _run_linear(s):
    case = s["case"]
    M, K, G = case["M"], case["K"], case["group"]
    w = (s["codes"].view(M, K // G, G).float() - s["zeros"].float()[..., None]) * s["scales"].float()[..., None]
    y = s["x"].float() @ w.view(M, K).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if case["act"] == "relu":
        y = y.clamp_min(0)
    elif case["act"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3)))
    return y.to(s["x"].dtype)


def run(state):
    if own:
        return _run_own(state)
    return {"append": _run_append, "attention": _run_attention, "linear": _run_linear}[state["case"]["kind"]](state)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------

def _exact_held(x):
    """float64 [..., D] -> the values that a cache of 4-bit codes holds for it.  A code, and a zero
    point, is a choice between two neighbours: where they are equally near it can fall on the other one than in 32 bits."""
    lo, hi = x.min(-1, keepdim=True).values.clamp(max=0), x.max(-1, keepdim=True).values.clamp(min=0)
    scale = (hi - lo) / 15
    nothing = scale < 2.0 ** -100
    scale = scale.masked_fill(nothing, 1.0)
    # 20 significant bits, the zero point in the four below them
    scale = torch.ldexp(torch.round(torch.ldexp(scale, 20 - torch.frexp(scale).exponent)), torch.frexp(scale).exponent - 20)
    zero = torch.round(-lo / scale).clamp(0, 15)
    scale = scale + torch.ldexp(zero, torch.frexp(scale).exponent - 24)
    return scale * ((torch.round(x / scale) + zero).clamp(0, 15) - zero)


def _exact_append(case, gen):
    s = _append_inputs(case, gen)

    def turned(x):
        if not case["rot"]:
            return x.double()
        half, table, t = case["rot"] // 2, s["rotation"].double(), 0
        out = x.double().clone()
        for n, length in _sequences(case):
            for i in range(half):
                c, z = table[length - n:length, i, None], table[length - n:length, half + i, None]
                one, two = (2 * i, 2 * i + 1) if case["interleaved"] else (i, half + i)
                a, b = x[t:t + n, :, one].double(), x[t:t + n, :, two].double()
                out[t:t + n, :, one] = a * c - b * z
                out[t:t + n, :, two] = a * z + b * c
            t += n
        return out

    held = [_exact_held(turned(s["k"])), _exact_held(s["v"].double())]
    return held + [turned(s["q"])] if case["rot"] else held


def _exact_attention(case, gen):
    s = _attention_inputs(case, gen)
    cache, P, share, W = s["cache"], case["page"], case["hq"] // case["hkv"], case["window"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)

    def side(name, pages, head, length):
        raw = cache[name + "_codes"][pages, head].reshape(-1, case["d"] // 2)[:length].double()
        word = cache[name + "_words"][pages, head].reshape(-1)[:length]
        high = torch.floor(raw / 16)
        both = torch.empty((length, case["d"]), dtype=torch.float64, device=DEVICE)
        both[:, 0::2], both[:, 1::2] = raw - 16 * high, high
        zero = torch.remainder(word, 16).double()
        return (both - zero[:, None]) * word.view(torch.float32).double()[:, None]

    t = 0
    for b, (n, length) in enumerate(_sequences(case)):
        pages = s["table"][b, :-(-length // P)].long()
        age = torch.arange(length - n, length, device=DEVICE)[:, None] - torch.arange(length, device=DEVICE)[None]
        seen = (age >= 0) & (age < W) if W else age >= 0
        for head in range(case["hkv"]):
            k, v = side("k", pages, head, length), side("v", pages, head, length)
            for h in range(head * share, (head + 1) * share):
                x = (s["q"][t:t + n, h].double() @ k.t()) / math.sqrt(case["d"])
                x = torch.softmax(torch.where(seen, x, torch.full_like(x, -math.inf)), -1)
                out[t:t + n, h] = x @ v
        t += n
    return out


def _exact_linear(case, gen):
    s = _linear_inputs(case, gen)
    x, G = s["x"].double(), case["group"]
    y = torch.zeros((case["N"], case["M"]), dtype=torch.float64, device=DEVICE)
    rows = max(1, (1 << 24) // case["K"])
    for r in range(0, case["M"], rows):
        zero = s["zeros"][r:r + rows].double().repeat_interleave(G, 1)
        w = (s["codes"][r:r + rows].double() - zero) * s["scales"][r:r + rows].double().repeat_interleave(G, 1)
        y[:, r:r + rows] = x @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if case["act"] == "relu":
        return torch.relu(y)
    return torch.nn.functional.gelu(y, approximate="tanh") if case["act"] == "gelu" else y


def exact(case, seed):
    gen = _generator(seed)
    return {"append": _exact_append, "attention": _exact_attention, "linear": _exact_linear}[case["kind"]](case, gen)


def _seen(case):
    """Keys that some query of the sequence sees, and query-key pairs, over the batch."""
    keys = pairs = 0
    for n, length in _sequences(case):
        W = case["window"] or length
        keys += min(length, W + n - 1)
        first = length - n + 1  # keys before and at the first new token
        full = max(0, min(n, W - first + 1))  # new tokens that see all before them
        pairs += full * first + full * (full - 1) // 2 + (n - full) * W
    return keys, pairs


def work(case):
    if case["kind"] == "linear":
        M, K, N, G = case["M"], case["K"], case["N"], case["group"]
        # codes; a 16-bit scale and a 4-bit zero point per group; activations and outputs
        return {"bytes": M * K / 2 + 2.5 * M * (K // G) + 2 * N * (K + M) + (2 * M if case["bias"] else 0),
                "flops": 2 * M * K * N}
    hq, hkv, d, seqs = case["hq"], case["hkv"], case["d"], _sequences(case)
    T = sum(n for n, _ in seqs)
    if case["kind"] == "append":
        entry = T * 2 * hkv * (d // 2 + 4)  # written, then read back
        turned = 2 * T * hq * d * 2 if case["rot"] else 0
        return {"bytes": T * 2 * hkv * d * 2 * 2 + 2 * entry + turned, "flops": 0}
    keys, pairs = _seen(case)
    return {"bytes": keys * 2 * hkv * (d // 2 + 4) + 2 * T * hq * d * 2, "flops": 4 * pairs * hq * d}
