"""Normed heads and an 8-bit cache as cases that can be timed and checked: what
a decoder layer with norms on its queries and keys does before attention, and
what a cache of half the bytes does to writing it, reading it back and
attending over it.

Four operators: the norm of each query and key head with its rotation, and the
gradient; the same with keys and values quantised into a paged cache; the
cache's rows read back; attention of new tokens (one of each sequence, a few
drafted ones, a chunk of a prompt) over the quantised cache.

``listed()`` names the calls, ``draw()`` gives more of the same kinds,
``prepare()`` makes what the program holds before the call, ``run()`` is the
call, ``exact()`` its answer in 64 bits.  With ``own`` false ``run()``
computes the plain form: elementary torch operations in 32 bits, rounded
once.

Heads are those of the 8B-shaped layer (32 over 8, 128 wide), of the
13B-shaped layer (40, 128 wide) and of the 768-wide layer (12, 64 wide) that
this repository's benchmark and tests use, and generic ones around them.
"""
from __future__ import annotations

import itertools
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = {"fp16": 2, "bf16": 2, "fp32": 4}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "fp8": 448.0}
EPS = 1e-6

MAX_NORM = 16384 * 40 * 128          # elements of the longest normed prompt
MAX_TRAIN = 8192 * 40 * 128          # elements of the longest one with a gradient
MAX_APPEND = 4096 * 40 * 128         # elements of the longest stored prompt
MAX_ROWS = 65536 * 8 * 128           # elements read back (keys or values)
MAX_CACHE = 131072 * 8 * 128         # elements of the longest cache (keys or values)
MAX_CHUNK_PAIRS = 512 * 16896 * 32 * 128

HEADS_8B = {"heads": 32, "kv_heads": 8, "dim": 128}
HEADS_13B = {"heads": 40, "kv_heads": 40, "dim": 128}
HEADS_768 = {"heads": 12, "kv_heads": 12, "dim": 64}


def listed():
    return [
        # the queries and keys of a long calibration batch, normed and rotated
        {"name": "norm_16384", "kind": "norm", "tokens": 16384, **HEADS_8B, "rotary": 128, "interleaved": False,
         "train": False, "weight": "bf16", "dtype": "bf16"},
        # a fine-tuning step of the 8B shape: outputs, the heads' gradients and the norms'
        {"name": "norm_train_8192", "kind": "norm", "tokens": 8192, **HEADS_8B, "rotary": 128, "interleaved": False,
         "train": True, "weight": "bf16", "dtype": "bf16"},
        # a small model's step in 32 bits, odd length, half of each head rotated in pairs of neighbours
        {"name": "norm_train_1001_fp32", "kind": "norm", "tokens": 1001, **HEADS_768, "rotary": 32,
         "interleaved": True, "train": True, "weight": "fp32", "dtype": "fp32"},
        # one token of one sequence, normed, rotated, quantised into the cache and read back. The smallest call.
        {"name": "append_1_fp8", "kind": "append", "new": "1", "before": "777", **HEADS_8B, "rotary": 128,
         "interleaved": False, "norm": True, "page": 16, "cache": "fp8", "weight": "bf16", "dtype": "bf16"},
        # a serving step: prompts of two new sequences beside single tokens of others
        {"name": "append_mixed_int8", "kind": "append", "new": "333,1,1,1,1,100,1,1,1", "before": "0,5000,17,64,3001,0,1,815,2048",
         **HEADS_8B, "rotary": 128, "interleaved": False, "norm": True, "page": 16, "cache": "int8",
         "weight": "fp32", "dtype": "bf16"},
        # a prompt of the 13B shape into the cache, no norms
        {"name": "append_2048_13b", "kind": "append", "new": "2048", "before": "0", **HEADS_13B, "rotary": 128,
         "interleaved": False, "norm": False, "page": 16, "cache": "fp8", "weight": "fp16", "dtype": "fp16"},
        # whole sequences read back, for work outside attention
        {"name": "rows_ragged_int8", "kind": "rows", "context": "8192,1,4097,777,16000,64,12001,5000", **HEADS_8B,
         "page": 16, "cache": "int8", "dtype": "bf16"},
        # one new token over 8192 cached ones
        {"name": "decode_1_8k_int8", "kind": "chunk", "new": "1", "context": "8192", **HEADS_8B, "page": 16,
         "cache": "int8", "dtype": "bf16"},
        # one new token for each of 24 sequences of different lengths
        {"name": "decode_24_ragged", "kind": "chunk", "new": ",".join(["1"] * 24),
         "context": "1,17,64,129,500,777,1000,1024,1500,2047,2048,2500,3001,3500,4000,4096,4097,4800,5000,6000,7001,"
                    "7777,8000,8192", **HEADS_8B, "page": 16, "cache": "int8", "dtype": "fp16"},
        # one new token over a very long context: the most bytes
        {"name": "decode_1_128k_fp8", "kind": "chunk", "new": "1", "context": "131072", **HEADS_8B, "page": 64,
         "cache": "fp8", "dtype": "bf16"},
        # five drafted tokens of each of eight sequences
        {"name": "draft_8x5", "kind": "chunk", "new": "5,5,5,5,5,5,5,5", "context": "1029,2048,3333,4096,5000,6144,7005,8197",
         **HEADS_8B, "page": 32, "cache": "fp8", "dtype": "fp16"},
        # a chunk of 512 tokens of a prompt over the 16384 before it
        {"name": "chunk_512_16k", "kind": "chunk", "new": "512", "context": "16896", **HEADS_8B, "page": 16,
         "cache": "fp8", "dtype": "bf16"},
    ]


# ------------------------------------------------------------------ draw --

def _log_int(rng, lo, hi):
    return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def _draw_heads(rng):
    """The repository's own heads half of the time, else generic ones."""
    pick = rng.random()
    if pick < 0.5:
        return dict(rng.choice([HEADS_8B, HEADS_13B, HEADS_768]))
    kv = rng.choice([1, 2, 4, 8, 12])
    return {"heads": kv * rng.choice([1, 2, 3, 4, 7, 8]), "kv_heads": kv, "dim": rng.choice([48, 64, 80, 96, 128])}


def _text(lens):
    return ",".join(str(x) for x in lens)


def draw(rng):
    kind = rng.choice(["norm", "train", "append", "append", "rows", "decode", "decode", "decode", "chunk", "chunk"])
    h = _draw_heads(rng)
    H, Hk, D = h["heads"], h["kv_heads"], h["dim"]
    dtype = rng.choice(["fp16", "bf16"])
    cache = rng.choice(["int8", "fp8"])
    rot = rng.choice([D, D, D // 2])
    page = rng.choice([16, 16, 32, 64, 128, 24])
    if kind in ("norm", "train"):
        dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
        most = (MAX_NORM if kind == "norm" else MAX_TRAIN) // ((H + Hk) * D * SIZES[dtype] // 2)
        return {"kind": "norm", "tokens": _log_int(rng, 1, most), **h, "rotary": rot,
                "interleaved": rng.random() < 0.4, "train": kind == "train",
                "weight": rng.choice([dtype, "fp32"]), "dtype": dtype}
    if kind == "append":
        n = rng.choice([1, 1, 2, 5, 16, 48])
        most = min(8192, MAX_APPEND // (n * H * D))
        new = [_log_int(rng, 1, most) if rng.random() < 0.5 else 1 for _ in range(n)]
        before = [_log_int(rng, 1, 8192) - 1 for _ in range(n)]
        return {"kind": "append", "new": _text(new), "before": _text(before), **h, "rotary": rot,
                "interleaved": rng.random() < 0.3, "norm": rng.random() < 0.6, "page": page, "cache": cache,
                "weight": rng.choice([dtype, "fp32"]), "dtype": dtype}
    if kind == "rows":
        n = _log_int(rng, 1, 24)
        most = min(65536, MAX_ROWS // (n * Hk * D))
        return {"kind": "rows", "context": _text([_log_int(rng, 1, most) for _ in range(n)]), **h, "page": page,
                "cache": cache, "dtype": rng.choice(["fp16", "bf16", "fp32"])}
    if kind == "decode":
        n = _log_int(rng, 1, 48)
        new = [1] * n if rng.random() < 0.75 else [rng.randint(1, 8) for _ in range(n)]
        most = min(131072, MAX_CACHE // (n * Hk * D))
        context = [x + _log_int(rng, max(1, most // 64), most) for x in new]
        return {"kind": "chunk", "new": _text(new), "context": _text(context), **h, "page": page, "cache": cache,
                "dtype": dtype}
    n = rng.choice([1, 1, 2, 3])
    new = [_log_int(rng, 2, 512) for _ in range(n)]
    most = min(32768, MAX_CHUNK_PAIRS // (n * max(new) * H * D), MAX_CACHE // (n * Hk * D))
    context = [x + _log_int(rng, 1, max(1, most - x)) for x in new]
    return {"kind": "chunk", "new": _text(new), "context": _text(context), **h, "page": page, "cache": cache,
            "dtype": dtype}


# ---------------------------------------------------------------- inputs --

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _ints(text):
    return [int(x) for x in str(text).split(",")]


def _prefix(lens):
    return torch.tensor([0, *itertools.accumulate(lens)], dtype=torch.int32, device=DEV)


def _heads(g, tokens, heads, dim, spread):
    """Projected activations: each head of a size of its own, a few wide channels; float."""
    x = torch.randn(tokens, heads, dim, generator=g, device=DEV)
    if spread:
        x *= 0.5 + torch.rand(1, heads, 1, generator=g, device=DEV)
        gain = torch.ones(dim, device=DEV)
        gain[torch.randperm(dim, generator=g, device=DEV)[:max(1, dim // 32)]] = 3.0
        x *= gain
    return x


def _fused(g, tokens, case, dtype):
    """Query, key and value heads as one projection leaves them: parts of its output's rows."""
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    x = torch.cat([_heads(g, tokens, H, D, True).to(dtype), _heads(g, tokens, Hk, D, True).to(dtype),
                   _heads(g, tokens, Hk, D, False).to(dtype)], 1)
    return x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]


def _table(rotary, positions):
    """Cosines and sines (positions, 2, rotary / 2), every frequency divided by four for long contexts."""
    inv = 500000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEV) / rotary) / 4.0
    a = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], 1).float()


def _weight(g, case):
    return (1.0 + 0.3 * torch.randn(case["dim"], generator=g, device=DEV)).to(DTYPES[case["weight"]])


def _cache(g, pages, case, spread):
    """A filled cache: codes (pages, page, heads, dim) and scales (pages, page, heads), each head's rows of
    a page next to each other in memory."""
    Hk, D, page = case["kv_heads"], case["dim"], case["page"]
    codes, scale = _quantised(_heads(g, pages * page, Hk, D, spread).transpose(0, 1), case["cache"])
    codes = codes.view(Hk, pages, page, D).transpose(0, 1).contiguous()
    scale = scale.view(Hk, pages, page).transpose(0, 1).contiguous()
    return codes.transpose(1, 2), scale.transpose(1, 2)


def _places(g, context, page):
    """A block table of shuffled pages for sequences of these lengths, and the pages it takes."""
    counts = [max(1, -(-c // page)) for c in context]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(context), max(counts), dtype=torch.int32, device=DEV)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    return table, pages


def prepare(case, seed):
    g = _gen(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    st = {"case": case}
    if kind == "norm":
        T = case["tokens"]
        st["q"], st["k"], _ = _fused(g, T, case, dt)
        st["wq"], st["wk"] = _weight(g, case), _weight(g, case)
        st["table"] = _table(case["rotary"], 8192)
        st["positions"] = (torch.arange(T, dtype=torch.int32, device=DEV) % 8192).contiguous()
        if case["train"]:
            st["gq"] = (torch.randn(T, H, D, generator=g, device=DEV) * 1e-2).to(dt)
            st["gk"] = (torch.randn(T, Hk, D, generator=g, device=DEV) * 1e-2).to(dt)
            for name in ("q", "k", "wq", "wk"):
                st[name] = st[name].requires_grad_(True)
        return st
    if kind == "append":
        new, before = _ints(case["new"]), _ints(case["before"])
        context, T = [a + b for a, b in zip(new, before)], sum(new)
        st["q"], st["k"], st["v"] = _fused(g, T, case, dt)
        st["wq"], st["wk"] = _weight(g, case), _weight(g, case)
        st["table"] = _table(case["rotary"], 16384)
        at = torch.cat([torch.arange(b, b + n, device=DEV) for n, b in zip(new, before)])
        st["positions"] = at.to(torch.int32)
    else:
        context = _ints(case["context"])
        new = context if kind == "rows" else _ints(case["new"])
        T = sum(new)
    st["block_table"], pages = _places(g, context, case["page"])
    st["cu"] = _prefix(new)
    st["context"] = torch.tensor(context, dtype=torch.int32, device=DEV)
    st["tokens"], st["longest_new"], st["longest"] = T, max(new), max(context)
    st["k_cache"], st["k_scale"] = _cache(g, pages, case, True)
    st["v_cache"], st["v_scale"] = _cache(g, pages, case, False)
    if kind == "append":
        seq = torch.repeat_interleave(torch.arange(len(new), device=DEV), torch.tensor(new, device=DEV))
        place = st["block_table"][seq, at // case["page"]].long() * case["page"] + at % case["page"]
        st["slots"] = place.to(torch.int32)
    elif kind == "chunk":
        st["q"] = _heads(g, T, H, D, True).to(dt)
        st["new"] = torch.tensor(new, dtype=torch.int32, device=DEV)
    return st


# ----------------------------------------------------------- plain forms --

def _quantised(x, kind):
    """Rows of floats as codes of 8 bits and a scale for each row; rows without values to speak of are zeros."""
    x = x.float()
    most = x.abs().amax(-1, keepdim=True)
    top = TOP[kind]
    some = most > 2.0 ** -120
    codes = x * torch.where(some, top / most, torch.zeros_like(most))
    if kind == "int8":
        codes = codes.round().clamp(-top, top).to(torch.int8)
    else:
        codes = codes.clamp(-top, top).to(torch.float8_e4m3fn)
    return codes, torch.where(some, most / top, torch.zeros_like(most)).squeeze(-1)


def _angles(table, positions):
    return table[positions.long()].unsqueeze(2).unbind(1)


def _turned(x, c, s, interleaved):
    """The first channels of each head of floats by their angles."""
    R = 2 * c.shape[-1]
    part, rest = x[..., :R], x[..., R:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = part[..., :R // 2], part[..., R // 2:]
        part = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([part, rest], -1)


def _normed(x):
    """Heads divided by their root mean square, and its reciprocal; float."""
    x = x.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return x * r, r


def _plain_norm(st):
    case = st["case"]
    c, s = _angles(st["table"], st["positions"])
    turn = case["interleaved"]
    out = {}
    for n in "qk":
        x, w, dt = st[n].detach(), st["w" + n].detach(), st[n].dtype
        hat, r = _normed(x)
        out[n] = _turned(hat * w.float(), c, s, turn).to(dt)
        if case["train"]:
            g = _turned(st["g" + n].float(), c, -s, turn)
            out["dw" + n] = (g * hat).sum((0, 1)).to(w.dtype)
            g = g * w.float()
            out["d" + n] = (r * (g - hat * (g * hat).mean(-1, keepdim=True))).to(dt)
    return out


def _at_places(st):
    """Which page and row each of the last cached tokens of a sequence is in, packed."""
    page = st["case"]["page"]
    cu = st["cu"].long()
    i = torch.arange(st["tokens"], device=DEV)
    b = torch.searchsorted(cu, i, right=True) - 1
    key = st["context"].long()[b] - (cu[b + 1] - i)
    return st["block_table"].long()[b, key // page], key % page


def _read(codes, scale, at):
    return codes[at].float() * scale[at].unsqueeze(-1)


def _plain_append(st):
    case, dt = st["case"], st["q"].dtype
    c, s = _angles(st["table"], st["positions"])
    q, k = st["q"].float(), st["k"].float()
    if case["norm"]:
        q, k = _normed(q)[0] * st["wq"].float(), _normed(k)[0] * st["wk"].float()
    q, k = _turned(q, c, s, case["interleaved"]), _turned(k, c, s, case["interleaved"])
    slots = st["slots"].long()
    at = slots // case["page"], slots % case["page"]
    out = {"q": q.to(dt)}
    for n, x in (("k", k), ("v", st["v"])):
        codes, scale = _quantised(x, case["cache"])
        st[n + "_cache"][at], st[n + "_scale"][at] = codes, scale
    at = _at_places(st)
    for n in "kv":
        out[n] = _read(st[n + "_cache"], st[n + "_scale"], at).to(dt)
    return out


def _plain_chunk(st):
    case = st["case"]
    B, N, S, page = st["context"].numel(), st["longest_new"], st["longest"], case["page"]
    at = st["cu"][:-1, None].long() + torch.arange(N, device=DEV)
    inside = at < st["cu"][1:, None]
    q = st["q"].float()[at.clamp(max=st["tokens"] - 1)].transpose(1, 2).contiguous()
    H, D, Hk = q.shape[1], q.shape[3], case["kv_heads"]
    G = H // Hk
    j = torch.arange(S, device=DEV)
    places = st["block_table"].long()[:, j // page], (j % page)[None].expand(B, S)
    k = _read(st["k_cache"], st["k_scale"], places).transpose(1, 2).contiguous().view(B * Hk, S, D)
    v = _read(st["v_cache"], st["v_scale"], places).transpose(1, 2).contiguous().view(B * Hk, S, D)
    last = (st["context"] - st["new"])[:, None] + torch.arange(N, device=DEV)
    seen = (j <= last[..., None]) & (j < st["context"][:, None, None]) & inside[..., None]
    p = torch.bmm(q.reshape(B * Hk, G * N, D), k.transpose(1, 2).contiguous())
    p = p.view(B, Hk, G, N, S).mul_(D ** -0.5)
    p = p.masked_fill_(~seen[:, None, None], float("-inf"))
    p = p.sub_(p.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp(min=1e-37)).view(B * Hk, G * N, S)
    o = torch.bmm(p, v)
    return o.view(B, H, N, D).transpose(1, 2)[inside].to(st["q"].dtype)


# ------------------------------------------------------------------- run --

def run(st):
    case = st["case"]
    if own:
        return _own(st)
    kind = case["kind"]
    if kind == "norm":
        return _plain_norm(st)
    if kind == "append":
        return _plain_append(st)
    if kind == "rows":
        at, dt = _at_places(st), DTYPES[case["dtype"]]
        return {n: _read(st[n + "_cache"], st[n + "_scale"], at).to(dt) for n in "kv"}
    return _plain_chunk(st)


def _own(st):
    from distributed_gptq_amd.models import attention as A
    case, kind = st["case"], st["case"]["kind"]
    if kind == "norm":
        q, k = A.norm_rotary(st["q"], st["k"], st["wq"], st["wk"], st["table"], st["positions"],
                             interleaved=case["interleaved"], eps=EPS)
        if not case["train"]:
            return {"q": q, "k": k}
        dq, dk, dwq, dwk = torch.autograd.grad((q, k), (st["q"], st["k"], st["wq"], st["wk"]), (st["gq"], st["gk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    scales = {"k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    caches = st["k_cache"], st["v_cache"]
    with torch.no_grad():
        if kind == "chunk":
            return A.paged_attention(st["q"], *caches, st["block_table"], st["context"],
                                     st["cu"] if st["longest_new"] > 1 else None, max_context=st["longest"], **scales)
        if kind == "append":
            norm = {"q_weight": st["wq"], "k_weight": st["wk"], "eps": EPS} if case["norm"] else {}
            q = A.rotary_append(st["q"], st["k"], st["v"], st["table"], st["positions"], *caches, st["slots"],
                                interleaved=case["interleaved"], **scales, **norm)
        k, v = A.cached_rows(*caches, st["block_table"], st["context"], st["cu"], st["tokens"],
                             dtype=DTYPES[case["dtype"]], **scales)
    return {"q": q, "k": k, "v": v} if kind == "append" else {"k": k, "v": v}


# ------------------------------------------------------------------ work --

def work(case):
    H, Hk, D, size = case["heads"], case["kv_heads"], case["dim"], SIZES[case["dtype"]]
    kind = case["kind"]
    if kind == "norm":
        T, R = case["tokens"], case["rotary"]
        x = T * (H + Hk) * D
        angles = min(T, 8192) * 4 * R + 4 * T
        if not case["train"]:
            return {"bytes": 2 * x * size + angles, "flops": x * 4 + T * (H + Hk) * 3 * R}
        return {"bytes": 4 * x * size + angles, "flops": x * 14 + 2 * T * (H + Hk) * 3 * R}
    row = D + 4  # codes and scale
    if kind == "append":
        T, R = sum(_ints(case["new"])), case["rotary"]
        written = T * (2 * H * D * size + 2 * Hk * (D * size + row)) + T * (4 * R + 8)
        back = T * 2 * Hk * D * size
        return {"bytes": written + back, "flops": T * (H + Hk) * (3 * R + (4 * D if case["norm"] else 0)) + 6 * T * Hk * D}
    if kind == "rows":
        T = sum(_ints(case["context"]))
        return {"bytes": T * 2 * Hk * (row + D * size), "flops": 2 * T * Hk * D}
    new, context = _ints(case["new"]), _ints(case["context"])
    pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(new, context))
    return {"bytes": 2 * sum(new) * H * D * size + 2 * sum(context) * Hk * row
            + 4 * sum(-(-c // case["page"]) for c in context), "flops": 4 * pairs * H * D}


# ----------------------------------------------------------------- exact --

def _exact_rotate(x, case, positions):
    """Each pair of channels as a complex number, times exp(i angle), in 64 bits."""
    R = case["rotary"]
    inv = torch.tensor([500000.0 ** (-2.0 * i / R) / 4.0 for i in range(R // 2)], dtype=torch.float64, device=DEV)
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV), positions.double()[:, None] * inv[None, :])
    part, rest = x[..., :R], x[..., R:]
    pairs = part.unflatten(-1, (R // 2, 2)) if case["interleaved"] else part.unflatten(-1, (2, R // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None, :])
    part = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
    return torch.cat([part, rest], -1)


def _exact_head_norm(x, w):
    return x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w


def _exact_stored(x, kind):
    """What rows of 64 bits are after quantising: a whole number of steps of their scale, or the nearest float of
    four exponent and three mantissa bits times it; ties to the even one."""
    most = x.abs().max(-1, keepdim=True).values
    step = most / TOP[kind]
    y = x / step.masked_fill(most == 0, 1.0)
    if kind == "int8":
        return y.round() * step
    unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / unit) * unit * step


def _exact_head(q, k, v, first):
    """One head in 64 bits: query i sees the keys up to first + i."""
    s = (q @ k.t()) * q.shape[1] ** -0.5
    at = torch.arange(q.shape[0], device=DEV)[:, None] + first
    s[torch.arange(k.shape[0], device=DEV)[None, :] > at] = -math.inf
    return torch.exp(s - torch.logsumexp(s, 1, keepdim=True)) @ v


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        out = {}
        for n in "qk":
            x = st[n].detach().double().requires_grad_(case["train"])
            w = st["w" + n].detach().double().requires_grad_(case["train"])
            y = _exact_rotate(_exact_head_norm(x, w), case, st["positions"])
            out[n] = y.detach()
            if case["train"]:
                out["d" + n], out["dw" + n] = torch.autograd.grad(y, (x, w), st["g" + n].double())
        return out
    if kind == "append":
        q, k = st["q"].double(), st["k"].double()
        if case["norm"]:
            q, k = _exact_head_norm(q, st["wq"].double()), _exact_head_norm(k, st["wk"].double())
        return {"q": _exact_rotate(q, case, st["positions"]),
                "k": _exact_stored(_exact_rotate(k, case, st["positions"]), case["cache"]),
                "v": _exact_stored(st["v"].double(), case["cache"])}
    page = case["page"]

    def rows(name, b, first, end):
        j = torch.arange(first, end, device=DEV)
        at = st["block_table"][b].long()[torch.div(j, page, rounding_mode="floor")], torch.remainder(j, page)
        return st[name + "_cache"][at].double() * st[name + "_scale"][at].double()[..., None]

    context = _ints(case["context"])
    if kind == "rows":
        return {n: torch.cat([rows(n, b, 0, c) for b, c in enumerate(context)]) for n in "kv"}
    H, G = case["heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    at = 0
    for b, (n, c) in enumerate(zip(_ints(case["new"]), context)):
        k, v = rows("k", b, 0, c), rows("v", b, 0, c)
        q = st["q"][at:at + n].double()
        for h in range(H):
            out[at:at + n, h] = _exact_head(q[:, h], k[:, h // G], v[:, h // G], c - n)
        at += n
    return out
