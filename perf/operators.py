"""The operators around a cache held in 8 bits, and what they are timed on.

Four kinds of work, each through the package's public entry points:

* ``rotary`` - queries and keys as a fused projection leaves them, (B, L, heads, D) memory, turned to their positions and laid out
  (B, H, L, D) for the cache: ``rope.apply_rotary``;
* ``fetch``  - new tokens written into 8-bit blocks (a scale for each block of tokens and head; the tokens behind the last whole block stay as
  they are in a tail) and the whole cache read back dense, for callers with their own attention: ``blocks.write_blocks``, ``blocks.read_blocks``;
* ``decode`` - one new token per sequence: its rows join the cache and its queries attend over it, over everything or over a sliding
  window and the first tokens (sinks): ``blocks.attend_blocks(..., new=(k, v))``;
* ``attend`` - the last tokens of a cache attend causally, a piece of a prompt or a few drafted tokens: ``blocks.attend_blocks``.

Keys and values are N(0, 1) rows under a LogNormal(0, 0.5) scale per token, queries N(0, 1) (scores are scaled by head_dim^-0.5): the
distributions of this repository's benchmark.
"""

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}

# The largest amount of work of each kind that draw() gives: what the largest listed case of the kind has.
MOST_ROTARY = 8192 * 40 * 128               # tokens x heads x head_dim
MOST_FETCH = 8 * 65536 * 128                # sequences x KV heads x tokens x head_dim
MOST_DECODE = 64 * 8 * 16384 * 128          # sequences x KV heads x context x head_dim
MOST_ATTEND = 32 * 2048 * 16384 * 128       # sequences x query heads x new tokens x context x head_dim


def rotary(name, b, hq, hkv, d, length, offset, dims=None, interleaved=False, scaling="none", base=500000.0, dtype="bf16"):
    return {"name": name, "kind": "rotary", "b": b, "hq": hq, "hkv": hkv, "d": d, "length": length, "offset": offset, "dims": dims or d,
            "interleaved": interleaved, "scaling": scaling, "base": base, "dtype": dtype}


def fetch(name, b, hkv, d, have, new, block=64, codes="int8", dtype="bf16"):
    return {"name": name, "kind": "fetch", "b": b, "hkv": hkv, "d": d, "have": have, "new": new, "block": block, "codes": codes, "dtype": dtype}


def decode(name, b, hq, hkv, d, have, window=0, sinks=0, block=64, codes="int8", dtype="bf16"):
    return {"name": name, "kind": "decode", "b": b, "hq": hq, "hkv": hkv, "d": d, "have": have, "window": window, "sinks": sinks, "block": block,
            "codes": codes, "dtype": dtype}


def attend(name, b, hq, hkv, d, total, queries, window=0, sinks=0, block=64, codes="int8", dtype="bf16"):
    return {"name": name, "kind": "attend", "b": b, "hq": hq, "hkv": hkv, "d": d, "total": total, "queries": queries, "window": window,
            "sinks": sinks, "block": block, "codes": codes, "dtype": dtype}


def listed():
    return [
        # -- rotary positions ----------------------------------------------------------------------------------------------
        # A decode step of four sequences far into a long context: the launch is all there is.
        rotary("rotary_step_b4", 4, 32, 8, 128, 1, 98303),
        # A long piece of a prompt, frequencies scaled for a long context: the largest of its kind.
        rotary("rotary_8k_scaled", 1, 32, 8, 128, 8192, 32768, scaling="llama3"),
        # -- into 8 bits and back ------------------------------------------------------------------------------------------
        # A token that completes a block of a short chat.
        fetch("fetch_token_1k", 1, 8, 128, 1087, 1),
        # A long prompt into a fresh cache, dense keys and values back: the largest of its kind.
        fetch("fetch_64k_prompt", 1, 8, 128, 0, 65519),
        # Prompts of a small batch behind what their caches hold, head_dim 96, 8-bit floats, small blocks.
        fetch("fetch_b4_d96_e4m3", 4, 32, 96, 45, 1500, block=32, codes="e4m3", dtype="fp16"),
        # -- one token per sequence ----------------------------------------------------------------------------------------
        # The start of a chat.
        decode("decode_700_b1", 1, 32, 8, 128, 700),
        # One long-context sequence.
        decode("decode_32k_b1", 1, 32, 8, 128, 32810),
        # Sliding-window layers of a served batch: 4096 tokens and the first four of contexts that have grown past them.
        decode("decode_window_b16_e4m3", 16, 32, 8, 128, 12021, window=4096, sinks=4, codes="e4m3"),
        # A full server. The largest decode step.
        decode("decode_16k_b64", 64, 32, 8, 128, 16383, dtype="fp16"),
        # -- several tokens per sequence -----------------------------------------------------------------------------------
        # Five drafted tokens to be verified, head_dim 64.
        attend("attend_5_draft_d64", 2, 16, 4, 64, 1881, 5, dtype="fp16"),
        # Sliding-window layers under a batch of prompts that come in pieces.
        attend("attend_window_b4_e4m3", 4, 32, 8, 128, 8000, 512, window=1024, sinks=4, codes="e4m3"),
        # A piece of a long prompt: the largest of its kind.
        attend("attend_2k_at_16k", 1, 32, 8, 128, 16384, 2048),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rotary", "fetch", "decode", "attend"])
    d = rng.choice([64, 96, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8, 8, 32])
    hq = min(64, hkv * rng.choice([1, 2, 4, 4, 7, 8]))
    hq -= hq % hkv
    dtype, codes = rng.choice(sorted(DTYPES)), rng.choice(sorted(CODES))
    block = rng.choice([16, 32, 64, 64, 128])
    b = _spread(rng, 1, 32)
    if kind == "rotary":
        length = _spread(rng, 1, 8192)
        b = max(1, min(b, MOST_ROTARY // ((hq + hkv) * d * length)))
        length = max(1, min(length, MOST_ROTARY // ((hq + hkv) * d)))
        return dict(rotary("", b, hq, hkv, d, length, _spread(rng, 1, 1 << 20), rng.choice([d, d, d // 2, d // 4]), rng.random() < 0.5,
                           rng.choice(["none", "linear", "llama3", "yarn"]), rng.choice([10000.0, 500000.0, 1e6]), dtype), name=None)
    if kind == "fetch":
        have, new = rng.choice([0, _spread(rng, 1, 8192)]), _spread(rng, 1, 65536)
        b = max(1, min(b, MOST_FETCH // (hkv * d * (have + new))))
        new = max(1, min(new, MOST_FETCH // (b * hkv * d) - have))
        return dict(fetch("", b, hkv, d, have, new, block, codes, dtype), name=None)
    window = rng.choice([0, 0, _spread(rng, 16, 8192)])
    sinks = rng.choice([0, 4, 64, 100]) if window else 0
    if kind == "decode":
        have = _spread(rng, 1, 131072)
        b = max(1, min(b, MOST_DECODE // (hkv * d * have)))
        have = max(1, min(have, MOST_DECODE // (b * hkv * d)))
        return dict(decode("", b, hq, hkv, d, have, window, sinks, block, codes, dtype), name=None)
    total = _spread(rng, 2, 32768)
    queries = min(total, _spread(rng, 2, 4096))
    b = max(1, min(b, MOST_ATTEND // (hq * d * total * queries)))
    queries = max(1, min(queries, MOST_ATTEND // (b * hq * d * total)))
    return dict(attend("", b, hq, hkv, d, total, queries, window, sinks, block, codes, dtype), name=None)


# ---- what a program has in hand ------------------------------------------------------------------------------------------

def _frequencies(dims, base, scaling):
    """Angle per position of each pair, float64, and the factor on the result, for the four ways that models scale them."""
    f = base ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "llama3":                      # slow pairs by 1 / 8, fast ones as they are, in between a blend by turns per 8192 positions
        turns = 8192.0 * f / (2 * math.pi)
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return f * ((1 - smooth) / 8.0 + smooth), 1.0
    if scaling == "yarn":                        # the blend runs over the pair's index, between 32 turns and 1 turn per 4096 positions
        at = [dims * math.log(4096.0 / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dims - 1)
        ramp = ((torch.arange(dims // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return f * (ramp / 8.0 + (1 - ramp)), 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def _rows(g, shape, dtype):
    scale = torch.exp(0.5 * torch.randn(*shape[:-1], 1, generator=g, device="cuda"))
    return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dtype)


def _encode(x, codes):
    """Rows of whole blocks (..., blocks, block, D), float32: their codes and scales."""
    top = x.abs().amax(dim=(-2, -1))
    largest = torch.full_like(top, TOP[codes])             # (a number over a tensor would be the number times a rounded reciprocal)
    inv = torch.where(top > 0, largest / top, torch.zeros_like(top))
    y = x * inv[..., None, None]
    return (torch.round(y) if codes == "int8" else y).to(CODES[codes]), top / largest


def _cache(g, c, tokens):
    """Storage with room for a few more tokens, ``tokens`` of them written."""
    b, h, d, n = c["b"], c["hkv"], c["d"], c["block"]
    blocks = -(-(tokens + c.get("new", 1)) // n)
    s, whole = {}, tokens // n
    for side in "kv":
        s[side + "_codes"] = torch.zeros(b, h, blocks * n, d, dtype=torch.int8, device="cuda").view(CODES[c["codes"]])
        s[side + "_scales"] = torch.zeros(b, h, blocks, device="cuda")
        s[side + "_tail"] = _rows(g, (b, h, n, d), DTYPES[c["dtype"]])
        if whole:
            x, scales = _encode(_rows(g, (b, h, whole, n, d), DTYPES[c["dtype"]]).float(), c["codes"])
            s[side + "_codes"].view(torch.int8)[:, :, :whole * n] = x.view(torch.int8).reshape(b, h, whole * n, d)
            s[side + "_scales"][:, :, :whole] = scales
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, dt = case, DTYPES[case["dtype"]]
    b, d = c["b"], c["d"]
    if c["kind"] == "rotary":
        f, factor = _frequencies(c["dims"], c["base"], c["scaling"])
        qkv = torch.randn(b, c["length"], c["hq"] + 2 * c["hkv"], d, generator=g, device="cuda").to(dt).transpose(1, 2)
        return {"case": c, "q": qkv[:, :c["hq"]], "k": qkv[:, c["hq"]:c["hq"] + c["hkv"]], "freqs": f.cuda(), "factor": factor}
    if c["kind"] == "fetch":
        s = _cache(g, c, c["have"])
        s["new"] = tuple(_rows(g, (b, c["hkv"], c["new"], d), dt) for _ in "kv")
    elif c["kind"] == "decode":
        s = _cache(g, c, c["have"])
        s["new"] = tuple(_rows(g, (b, c["hkv"], 1, d), dt) for _ in "kv")
        s["q"] = torch.randn(b, c["hq"], 1, d, generator=g, device="cuda").to(dt)
    else:
        s = _cache(g, c, c["total"])
        s["q"] = torch.randn(b, c["hq"], c["queries"], d, generator=g, device="cuda").to(dt)
    return {"case": c, **s}


# ---- the plain form ------------------------------------------------------------------------------------------------------

def _write(s, length):
    """The new tokens behind ``length`` others: whole blocks become codes, the rest joins the tail."""
    c = s["case"]
    n, t = c["block"], s["new"][0].shape[2]
    at, old = length // n, length % n
    whole, rest = (old + t) // n, (old + t) % n
    _write_side(s, "k", s["new"][0], n, at, old, whole, rest)
    _write_side(s, "v", s["new"][1], n, at, old, whole, rest)
    return length + t


def _write_side(s, side, new, n, at, old, whole, rest):
    c, tail = s["case"], s[side + "_tail"]
    b, h, t, d = new.shape
    if whole:
        x = torch.cat([tail[:, :, :old], new], dim=2)
        codes, scales = _encode(x[:, :, :whole * n].float().reshape(b, h, whole, n, d), c["codes"])
        s[side + "_codes"].view(torch.int8)[:, :, at * n:(at + whole) * n] = codes.view(torch.int8).reshape(b, h, whole * n, d)
        s[side + "_scales"][:, :, at:at + whole] = scales
        if rest:
            tail[:, :, :rest] = x[:, :, whole * n:]
    else:
        tail[:, :, old:old + t] = new


def _dense(s, side, length):
    """Float32 rows of all tokens."""
    n = s["case"]["block"]
    whole = length // n
    x = s[side + "_codes"][:, :, :whole * n].float().unflatten(2, (whole, n)) * s[side + "_scales"][:, :, :whole, None, None] if whole else None
    rest = s[side + "_tail"][:, :, :length - whole * n].float()
    return rest if x is None else torch.cat([x.flatten(2, 3), rest], dim=2)


def _attention(s, length):
    c, q = s["case"], s["q"]
    k, v = _dense(s, "k", length), _dense(s, "v", length)
    b, hq, t, d = q.shape
    hkv = k.shape[1]
    scores = q.float().reshape(b, hkv, hq // hkv * t, d) @ k.transpose(-1, -2) * d ** -0.5
    scores = scores.reshape(b, hkv, hq // hkv, t, length)
    behind = torch.arange(length - t, length, device="cuda")[:, None] - torch.arange(length, device="cuda")[None, :]
    hidden = behind < 0
    if c["window"]:
        hidden = hidden | ((behind >= c["window"]) & (torch.arange(length, device="cuda") >= c["sinks"]))
    scores.masked_fill_(hidden, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).reshape(b, hkv, hq // hkv * t, length)
    return (p @ v).reshape(b, hq, t, d).to(q.dtype)


def _turn(x, freqs, offset, interleaved, factor):
    angle = torch.arange(offset, offset + x.shape[2], device="cuda", dtype=torch.float64)[:, None] * freqs
    cos, sin = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    r = 2 * freqs.numel()
    y = x.float()
    if interleaved:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, y[..., r:]], dim=-1).to(x.dtype)


# ---- one pass ------------------------------------------------------------------------------------------------------------

def run(state):
    s, c = state, state["case"]
    if c["kind"] == "rotary":
        if own:
            from mlx_turboquant_b200 import rope
            return rope.apply_rotary(s["q"], s["k"], s["freqs"], c["offset"], interleaved=c["interleaved"], factor=s["factor"])
        return (_turn(s["q"], s["freqs"], c["offset"], c["interleaved"], s["factor"]),
                _turn(s["k"], s["freqs"], c["offset"], c["interleaved"], s["factor"]))
    if own:
        from mlx_turboquant_b200 import blocks
        store = (s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"], s["k_tail"], s["v_tail"])
    if c["kind"] == "fetch":
        if own:
            length = blocks.write_blocks(s["new"][0], s["new"][1], *store, c["have"])
            k, v = blocks.read_blocks(*store, length)
        else:
            length = _write(s, c["have"])
            k, v = _dense(s, "k", length).to(s["k_tail"].dtype), _dense(s, "v", length).to(s["k_tail"].dtype)
        return {"k": k, "v": v, "k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    if c["kind"] == "decode":
        if own:
            out = blocks.attend_blocks(s["q"], *store, c["have"], window=c["window"] or None, sinks=c["sinks"], new=s["new"])
        else:
            out = _attention(s, _write(s, c["have"]))
        return {"out": out, "k_tail": s["k_tail"], "v_tail": s["v_tail"], "k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    if own:
        return blocks.attend_blocks(s["q"], *store, c["total"], window=c["window"] or None, sinks=c["sinks"])
    return _attention(s, c["total"])


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------

def _pairs(total, queries, window, sinks):
    """(query, token) pairs that a head computes, and the tokens that some query sees."""
    first = total - queries
    if not window:
        return queries * first + queries * (queries + 1) // 2, total
    pairs = 0
    for p in range(first, total):
        low = max(0, p - window + 1)
        pairs += p + 1 - low + min(sinks, low)
    low = max(0, first - window + 1)
    return pairs, total - low + min(sinks, low)


def work(case):
    c = case
    b, d = c["b"], c["d"]
    if c["kind"] == "rotary":
        n = b * c["length"] * (c["hq"] + c["hkv"])
        return {"bytes": 2 * 2 * n * d, "flops": 3 * n * c["dims"]}
    lanes, n = b * c["hkv"], c["block"]
    token = 2 * (d + 4 / n)                       # bytes of a token's keys and values in 8 bits, one head
    if c["kind"] == "fetch":
        total = c["have"] + c["new"]
        back = (c["have"] // n * n) * token + (total % n) * 4 * d + total * 4 * d      # what was there is read, everything is written dense
        return {"bytes": lanes * (c["new"] * 4 * d + ((total // n - c["have"] // n) * n) * token + back), "flops": lanes * 2 * total * d * 4}
    total, queries = (c["have"] + 1, 1) if c["kind"] == "decode" else (c["total"], c["queries"])
    pairs, seen = _pairs(total, queries, c["window"], c["sinks"])
    tail = min(total % n, seen)
    return {"bytes": lanes * ((seen - tail) * token + tail * 4 * d) + 4 * b * c["hq"] * queries * d, "flops": 4 * b * c["hq"] * pairs * d}


# ---- 64 bits -------------------------------------------------------------------------------------------------------------

def _exact_codes(x, codes):
    """Whole blocks (b, h, blocks, block, d) in float64 -> the values they stand for, and their scales."""
    s = x.abs().flatten(-2).max(-1).values / TOP[codes]
    y = x / torch.where(s > 0, s, torch.ones_like(s))[..., None, None]
    if codes == "int8":
        y = torch.round(y)
    else:                                         # three bits behind the leading one, 2^-9 the smallest step
        _, e = torch.frexp(y)
        step = torch.exp2((e - 4).clamp(min=-9).double())
        y = torch.round(y / step) * step
    return y * s[..., None, None], s


def _exact_side(s, side, have, new):
    """(values of all tokens in float64, scales, tail) behind the write of ``new`` to ``have`` tokens."""
    n, codes = s["case"]["block"], s["case"]["codes"]
    c, scales, tail = s[side + "_codes"], s[side + "_scales"].double(), s[side + "_tail"].double()
    b, h, _, d = c.shape
    cut = have // n * n
    parts = [c[:, :, :cut].float().double() * scales[:, :, :cut // n].repeat_interleave(n, dim=2)[..., None]]
    fresh = tail[:, :, :have - cut]
    if new is not None:
        fresh = torch.cat([fresh, new.double()], dim=2)
    whole = fresh.shape[2] // n
    if whole:
        x, sc = _exact_codes(fresh[:, :, :whole * n].reshape(b, h, whole, n, d), codes)
        parts.append(x.reshape(b, h, whole * n, d))
        scales = scales.clone()
        scales[:, :, cut // n:cut // n + whole] = sc
    rest = fresh[:, :, whole * n:]
    tail[:, :, :rest.shape[2]] = rest
    return torch.cat(parts + [rest], dim=2), scales, tail


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] == "rotary":
        pos = torch.arange(c["length"], device="cuda", dtype=torch.float64) + c["offset"]
        turn = s["factor"] * torch.polar(torch.ones((), device="cuda", dtype=torch.float64), torch.outer(pos, s["freqs"]))
        r = c["dims"]
        got = []
        for x in (s["q"], s["k"]):
            y = x.double().clone()
            head = y[..., :r].unflatten(-1, (r // 2, 2) if c["interleaved"] else (2, r // 2))
            z = torch.complex(head[..., 0], head[..., 1]) if c["interleaved"] else torch.complex(head[..., 0, :], head[..., 1, :])
            z = torch.view_as_real(z * turn)
            y[..., :r] = (z if c["interleaved"] else z.transpose(-1, -2)).flatten(-2)
            got.append(y)
        return tuple(got)
    have = c.get("have", c.get("total"))
    new = s.get("new", (None, None))
    k, k_scales, k_tail = _exact_side(s, "k", have, new[0])
    v, v_scales, v_tail = _exact_side(s, "v", have, new[1])
    if c["kind"] == "fetch":
        return {"k": k, "v": v, "k_scales": k_scales, "v_scales": v_scales}
    b, hq, t, d = s["q"].shape
    total, group = k.shape[2], hq // c["hkv"]
    out = torch.empty(b, hq, t, d, dtype=torch.float64, device="cuda")
    j = torch.arange(total, device="cuda")
    for i in range(b):
        for first in range(0, t, 256):            # queries first, first + 1, ...: the rest of the scores does not fit
            p = torch.arange(total - t, total, device="cuda")[first:first + 256, None]
            seen = j <= p
            if c["window"]:
                seen &= (j > p - c["window"]) | (j < c["sinks"])
            for h in range(c["hkv"]):
                z = torch.einsum("gtd,nd->gtn", s["q"][i, h * group:(h + 1) * group, first:first + 256].double(), k[i, h]) / math.sqrt(d)
                w = torch.softmax(torch.where(seen, z, -torch.inf), dim=-1)
                out[i, h * group:(h + 1) * group, first:first + 256] = torch.einsum("gtn,nd->gtd", w, v[i, h])
    if c["kind"] == "decode":
        return {"out": out, "k_tail": k_tail, "v_tail": v_tail, "k_scales": k_scales, "v_scales": v_scales}
    return out
