"""The attention of a decoder layer as cases that can be timed and checked:
what stands between a layer's query/key/value projection and its output
projection, in a prompt, in training and in serving from a paged cache.

Four operators: rotary positions on queries and keys; the same with the
keys and values written into a paged cache; attention of packed sequences,
causal, with grouped heads, and its gradient; attention of new tokens (a
chunk of a prompt, or one token of each sequence) over the paged cache.

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

MAX_ROTARY = 16384 * 40 * 128        # elements of the longest rotated prompt
MAX_PAIRS = 16 * 2048 * 2048 * 12 * 64    # (query, key, channel) triples of the largest prompt
MAX_TRAIN_PAIRS = 2 * 2048 * 2048 * 32 * 128
MAX_CACHE = 131072 * 8 * 128         # elements of the longest cache (keys or values)
MAX_CHUNK_PAIRS = 512 * 16896 * 32 * 128

HEADS_8B = {"heads": 32, "kv_heads": 8, "dim": 128}
HEADS_13B = {"heads": 40, "kv_heads": 40, "dim": 128}
HEADS_768 = {"heads": 12, "kv_heads": 12, "dim": 64}


def listed():
    return [
        # one token of one sequence: rotated, its key and value stored. The smallest call.
        {"name": "append_1", "kind": "append", "tokens": 1, **HEADS_8B, "rotary": 128, "interleaved": False,
         "page": 16, "pages": 64, "dtype": "bf16"},
        # one prompt of the 13B shape into the cache
        {"name": "append_2048_13b", "kind": "append", "tokens": 2048, **HEADS_13B, "rotary": 128,
         "interleaved": False, "page": 16, "pages": 160, "dtype": "fp16"},
        # the queries and keys of a long calibration batch
        {"name": "rotary_16384", "kind": "rotary", "lens": "2048,2048,2048,2048,2048,2048,2048,2048", **HEADS_8B,
         "rotary": 128, "interleaved": False, "train": False, "dtype": "bf16"},
        # fine-tuning on odd lengths: half of each head rotated in pairs of neighbours, and the gradient
        {"name": "rotary_train_3001", "kind": "rotary", "lens": "1999,1002", **HEADS_8B, "rotary": 64,
         "interleaved": True, "train": True, "dtype": "fp16"},
        # a short prompt of odd length
        {"name": "prompt_37", "kind": "prompt", "lens": "37", **HEADS_768, "train": False, "dtype": "fp16"},
        # four prompts of different lengths in one batch
        {"name": "prompt_packed_8b", "kind": "prompt", "lens": "4096,1777,1500,819", **HEADS_8B, "train": False,
         "dtype": "bf16"},
        # a calibration batch of the 768-wide model
        {"name": "prompt_16x2048_768", "kind": "prompt", "lens": ",".join(["2048"] * 16), **HEADS_768,
         "train": False, "dtype": "fp16"},
        # a fine-tuning step of two sequences: output and gradients
        {"name": "train_2x2048_8b", "kind": "prompt", "lens": "2048,2048", **HEADS_8B, "train": True,
         "dtype": "bf16"},
        # one new token over 8192 cached ones
        {"name": "decode_1_8k", "kind": "chunk", "new": "1", "context": "8192", **HEADS_8B, "page": 16,
         "dtype": "bf16"},
        # one new token for each of 24 sequences of different lengths
        {"name": "decode_24_ragged", "kind": "chunk", "new": ",".join(["1"] * 24),
         "context": "1,17,64,129,500,777,1000,1024,1500,2047,2048,2500,3001,3500,4000,4096,4097,4800,5000,6000,7001,"
                    "7777,8000,8192", **HEADS_8B, "page": 16, "dtype": "fp16"},
        # one new token over a very long context: the most bytes
        {"name": "decode_1_128k", "kind": "chunk", "new": "1", "context": "131072", **HEADS_8B, "page": 64,
         "dtype": "bf16"},
        # a chunk of 512 tokens of a prompt over the 16384 before it
        {"name": "chunk_512_16k", "kind": "chunk", "new": "512", "context": "16896", **HEADS_8B, "page": 16,
         "dtype": "bf16"},
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
    return {"heads": kv * rng.choice([1, 2, 3, 4, 7, 8]), "kv_heads": kv, "dim": rng.choice([40, 64, 80, 96, 128])}


def _draw_lens(rng, most, total):
    """Lengths of one to eight sequences, all at most `most`, `total` together."""
    n = rng.choice([1, 1, 2, 3, 4, 8])
    lens = []
    for _ in range(n):
        room = total - sum(lens)
        if room < 1:
            break
        lens.append(_log_int(rng, 1, min(most, room)))
    return lens


def _text(lens):
    return ",".join(str(x) for x in lens)


def draw(rng):
    kind = rng.choice(["append", "rotary", "prompt", "prompt", "train", "train", "decode", "decode", "decode",
                       "chunk"])
    h = _draw_heads(rng)
    H, Hk, D = h["heads"], h["kv_heads"], h["dim"]
    dtype = rng.choice(["fp16", "bf16"])
    rot = rng.choice([D, D, D // 2])
    page = rng.choice([16, 16, 32, 64, 128, 24])
    if kind == "append":
        T = _log_int(rng, 1, min(4096, MAX_ROTARY // (H * D)))
        return {"kind": "append", "tokens": T, **h, "rotary": rot, "interleaved": rng.random() < 0.3, "page": page,
                "pages": -(-T // page) + rng.randint(1, 32), "dtype": dtype}
    if kind == "rotary":
        most = MAX_ROTARY // ((H + Hk) * D)
        return {"kind": "rotary", "lens": _text(_draw_lens(rng, 8192, most)), **h, "rotary": rot,
                "interleaved": rng.random() < 0.5, "train": rng.random() < 0.5,
                "dtype": rng.choice(["fp16", "bf16", "fp32"])}
    if kind in ("prompt", "train"):
        cap = MAX_PAIRS if kind == "prompt" else MAX_TRAIN_PAIRS
        most = int(math.sqrt(cap / (H * D)))
        lens = _draw_lens(rng, min(most, 4096), 8192)
        while len(lens) * max(lens) ** 2 * H * D > cap:
            lens.remove(max(lens))
        return {"kind": "prompt", "lens": _text(lens), **h, "train": kind == "train", "dtype": dtype}
    if kind == "decode":
        n = _log_int(rng, 1, 48)
        most = min(131072, MAX_CACHE // (n * Hk * D))
        context = [_log_int(rng, max(1, most // 64), most) for _ in range(n)]
        return {"kind": "chunk", "new": _text([1] * n), "context": _text(context), **h, "page": page, "dtype": dtype}
    n = rng.choice([1, 1, 2, 3])
    new = [_log_int(rng, 2, 512) for _ in range(n)]
    most = min(32768, MAX_CHUNK_PAIRS // (n * max(new) * H * D), MAX_CACHE // (n * Hk * D))
    context = [x + _log_int(rng, 1, max(1, most - x)) for x in new]
    return {"kind": "chunk", "new": _text(new), "context": _text(context), **h, "page": page, "dtype": dtype}


# ---------------------------------------------------------------- inputs --

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _ints(text):
    return [int(x) for x in str(text).split(",")]


def _prefix(lens):
    return torch.tensor([0, *itertools.accumulate(lens)], dtype=torch.int32, device=DEV)


def _heads(g, tokens, heads, dim, dtype, spread):
    """Projected activations: each head of a size of its own, a few wide channels."""
    x = torch.randn(tokens, heads, dim, generator=g, device=DEV)
    if spread:
        x *= 0.5 + torch.rand(1, heads, 1, generator=g, device=DEV)
        gain = torch.ones(dim, device=DEV)
        gain[torch.randperm(dim, generator=g, device=DEV)[:max(1, dim // 32)]] = 3.0
        x *= gain
    return x.to(dtype)


def _fused(g, tokens, case, dtype):
    """Query, key and value heads as one projection leaves them: parts of its output's rows."""
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    x = torch.cat([_heads(g, tokens, H, D, dtype, True), _heads(g, tokens, Hk, D, dtype, True),
                   _heads(g, tokens, Hk, D, dtype, False)], 1)
    return x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]


def _table(rotary, positions):
    """Cosines and sines (positions, 2, rotary / 2), every frequency divided by four for long contexts."""
    inv = 500000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEV) / rotary) / 4.0
    a = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], 1).float()


def _positions(lens):
    return torch.cat([torch.arange(n, dtype=torch.int32, device=DEV) for n in lens])


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    dt = DTYPES[case["dtype"]]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    st = {"case": case}
    if kind == "append":
        T, page, pages = case["tokens"], case["page"], case["pages"]
        st["q"], st["k"], st["v"] = _fused(g, T, case, dt)
        st["table"] = _table(case["rotary"], 8192)
        first = int(torch.randint(0, 8192 - T, (1,), generator=g, device=DEV))
        st["positions"] = torch.arange(first, first + T, dtype=torch.int32, device=DEV)
        st["k_cache"] = _heads(g, pages * page, Hk, D, dt, True).view(pages, page, Hk, D)
        st["v_cache"] = _heads(g, pages * page, Hk, D, dt, False).view(pages, page, Hk, D)
        order = torch.randperm(pages, generator=g, device=DEV)
        at = torch.arange(T, device=DEV)
        st["slots"] = (order[at // page] * page + at % page).to(torch.int32)
    elif kind == "rotary":
        lens = _ints(case["lens"])
        T = sum(lens)
        st["q"], st["k"], _ = _fused(g, T, case, dt)
        st["table"] = _table(case["rotary"], 8192)
        st["positions"] = _positions(lens)
        if case["train"]:
            st["gq"] = (torch.randn(T, H, D, generator=g, device=DEV) * 1e-2).to(dt)
            st["gk"] = (torch.randn(T, Hk, D, generator=g, device=DEV) * 1e-2).to(dt)
            st["q"], st["k"] = st["q"].requires_grad_(True), st["k"].requires_grad_(True)
    elif kind == "prompt":
        lens = _ints(case["lens"])
        T = sum(lens)
        st["q"], st["k"], st["v"] = _fused(g, T, case, dt)
        st["cu"], st["longest"] = _prefix(lens), max(lens)
        if case["train"]:
            st["g"] = (torch.randn(T, H, D, generator=g, device=DEV) * 1e-2).to(dt)
            for name in "qkv":
                st[name] = st[name].requires_grad_(True)
    else:
        new, context, page = _ints(case["new"]), _ints(case["context"]), case["page"]
        B, T = len(new), sum(new)
        st["q"] = _heads(g, T, H, D, dt, True)
        st["cu"] = None if max(new) == 1 else _prefix(new)
        st["new"] = torch.tensor(new, dtype=torch.int32, device=DEV)
        st["context"] = torch.tensor(context, dtype=torch.int32, device=DEV)
        st["longest_new"], st["longest"] = max(new), max(context)
        counts = [-(-c // page) for c in context]
        pages = sum(counts) + 3
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        table = torch.zeros(B, max(counts), dtype=torch.int32, device=DEV)
        at = 0
        for b, c in enumerate(counts):
            table[b, :c] = order[at:at + c]
            at += c
        st["block_table"] = table
        st["k_cache"] = _heads(g, pages * page, Hk, D, dt, True).view(pages, page, Hk, D)
        st["v_cache"] = _heads(g, pages * page, Hk, D, dt, False).view(pages, page, Hk, D)
    return st


# ----------------------------------------------------------- plain forms --

def _plain_rotate(x, table, positions, interleaved, back=False):
    """Rotates the first channels of each head by their positions' angles; float."""
    x = x.float()
    c, s = table[positions.long()].unsqueeze(2).unbind(1)
    if back:
        s = -s
    R = 2 * c.shape[-1]
    part, rest = x[..., :R], x[..., R:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = part[..., :R // 2], part[..., R // 2:]
        part = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([part, rest], -1)


def _padded(x, cu, longest):
    """Packed rows (tokens, heads, dim) as (sequences, heads, longest, dim), float, zeros past each end."""
    at = cu[:-1, None].long() + torch.arange(longest, device=DEV)
    inside = at < cu[1:, None]
    rows = x.float()[at.clamp(max=x.shape[0] - 1)] * inside[..., None, None]
    return rows.transpose(1, 2).contiguous(), inside


def _plain_scores(q, k, scale, seen):
    """Softmax weights (sequences, kv heads, group * queries, keys) of padded q and k; zero where not seen."""
    B, H, L, D = q.shape
    Hk, S = k.shape[1], k.shape[2]
    G = H // Hk
    s = torch.bmm(q.reshape(B * Hk, G * L, D), k.reshape(B * Hk, S, D).transpose(1, 2).contiguous())
    s = s.view(B, Hk, G, L, S).mul_(scale)
    s = s.masked_fill_(~seen[:, None, None], float("-inf"))
    s = s.sub_(s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)).exp_()
    return s.div_(s.sum(-1, keepdim=True).clamp(min=1e-37)).view(B * Hk, G * L, S)


def _plain_prompt(st):
    case = st["case"]
    q, inside = _padded(st["q"].detach(), st["cu"], st["longest"])
    k, _ = _padded(st["k"].detach(), st["cu"], st["longest"])
    v, _ = _padded(st["v"].detach(), st["cu"], st["longest"])
    B, H, L, D = q.shape
    Hk = k.shape[1]
    scale = D ** -0.5
    i = torch.arange(L, device=DEV)
    seen = (i[None, :] <= i[:, None]) & inside[:, None, :] & inside[:, :, None]
    p = _plain_scores(q, k, scale, seen)
    o = torch.bmm(p, v.reshape(B * Hk, L, D))

    def packed(x, dt):
        return x.view(B, -1, L, D).transpose(1, 2)[inside].to(dt)

    dt = st["q"].dtype
    if not case["train"]:
        return packed(o, dt)
    g, _ = _padded(st["g"], st["cu"], st["longest"])
    g = g.reshape(B * Hk, -1, D)
    dv = torch.bmm(p.transpose(1, 2).contiguous(), g)
    ds = torch.bmm(g, v.reshape(B * Hk, L, D).transpose(1, 2).contiguous())
    ds = ds.sub_((g * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.bmm(ds, k.reshape(B * Hk, L, D))
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), q.reshape(B * Hk, -1, D))
    return {"out": packed(o, dt), "dq": packed(dq, dt), "dk": packed(dk, dt), "dv": packed(dv, dt)}


def _plain_chunk(st):
    case = st["case"]
    B, N = st["context"].numel(), st["longest_new"]
    cu = st["cu"] if st["cu"] is not None else torch.arange(B + 1, device=DEV, dtype=torch.int32)
    q, inside = _padded(st["q"], cu, N)
    H, D = q.shape[1], q.shape[3]
    Hk = case["kv_heads"]
    pages = st["block_table"].long()

    def rows(cache):
        x = cache[pages].flatten(1, 2)
        return x.float().transpose(1, 2).contiguous()

    k, v = rows(st["k_cache"]), rows(st["v_cache"])
    S = k.shape[2]
    j = torch.arange(S, device=DEV)
    last = (st["context"] - st["new"])[:, None] + torch.arange(N, device=DEV)
    seen = (j <= last[..., None]) & (j < st["context"][:, None, None]) & inside[..., None]
    p = _plain_scores(q, k, D ** -0.5, seen)
    o = torch.bmm(p, v.reshape(B * Hk, S, D))
    return o.view(B, H, N, D).transpose(1, 2)[inside].to(st["q"].dtype)


# ------------------------------------------------------------------- run --

def run(st):
    case = st["case"]
    if own:
        return _own(st)
    kind = case["kind"]
    if kind == "append":
        dt = st["q"].dtype
        turn = (st["table"], st["positions"], case["interleaved"])
        st["k_cache"].flatten(0, 1)[st["slots"].long()] = _plain_rotate(st["k"], *turn).to(dt)
        st["v_cache"].flatten(0, 1)[st["slots"].long()] = st["v"]
        return {"q": _plain_rotate(st["q"], *turn).to(dt), "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    if kind == "rotary":
        dt = st["q"].dtype
        turn = (st["table"], st["positions"], case["interleaved"])
        out = {"q": _plain_rotate(st["q"].detach(), *turn).to(dt), "k": _plain_rotate(st["k"].detach(), *turn).to(dt)}
        if case["train"]:
            out["dq"] = _plain_rotate(st["gq"], *turn, back=True).to(dt)
            out["dk"] = _plain_rotate(st["gk"], *turn, back=True).to(dt)
        return out
    if kind == "prompt":
        return _plain_prompt(st)
    return _plain_chunk(st)


def _own(st):
    from distributed_gptq_amd.models import attention as A
    case = st["case"]
    kind = case["kind"]
    if kind == "append":
        with torch.no_grad():
            q = A.rotary_append(st["q"], st["k"], st["v"], st["table"], st["positions"], st["k_cache"],
                                st["v_cache"], st["slots"], interleaved=case["interleaved"])
        return {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    if kind == "rotary":
        q, k = A.rotary(st["q"], st["k"], st["table"], st["positions"], interleaved=case["interleaved"])
        if not case["train"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    if kind == "prompt":
        o = A.attention(st["q"], st["k"], st["v"], st["cu"])
        if not case["train"]:
            return o
        dq, dk, dv = torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["g"])
        return {"out": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    with torch.no_grad():
        return A.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["block_table"], st["context"], st["cu"],
                                 max_context=st["longest"])


# ------------------------------------------------------------------ work --

def work(case):
    H, Hk, D, size = case["heads"], case["kv_heads"], case["dim"], SIZES[case["dtype"]]
    kind = case["kind"]
    if kind == "append":
        T = case["tokens"]
        return {"bytes": 2 * T * (H + 2 * Hk) * D * size + T * (4 * case["rotary"] + 8),
                "flops": 3 * T * (H + Hk) * case["rotary"]}
    if kind == "rotary":
        T, passes = sum(_ints(case["lens"])), 2 if case["train"] else 1
        return {"bytes": passes * 2 * T * (H + Hk) * D * size + T * (4 * case["rotary"] + 4),
                "flops": passes * 3 * T * (H + Hk) * case["rotary"]}
    if kind == "prompt":
        lens = _ints(case["lens"])
        T, pairs = sum(lens), sum(n * (n + 1) // 2 for n in lens)
        rows = T * (2 * H + 2 * Hk) * D * size
        if case["train"]:  # the gradient's five products, and its reads and writes beside the output's
            return {"bytes": rows + T * (2 * H + 2 * Hk) * D * size, "flops": (4 + 10) * pairs * H * D}
        return {"bytes": rows, "flops": 4 * pairs * H * D}
    new, context = _ints(case["new"]), _ints(case["context"])
    pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(new, context))
    return {"bytes": (2 * sum(new) * H + 2 * sum(context) * Hk) * D * size + 4 * sum(-(-c // case["page"]) for c in context),
            "flops": 4 * pairs * H * D}


# ----------------------------------------------------------------- exact --

def _exact_rotate(x, case, positions, sign=1.0):
    """Each pair of channels as a complex number, times exp(i angle), in 64 bits."""
    R = case["rotary"]
    inv = torch.tensor([500000.0 ** (-2.0 * i / R) / 4.0 for i in range(R // 2)], dtype=torch.float64, device=DEV)
    turn = torch.exp(1j * sign * positions.double()[:, None] * inv[None, :])
    x = x.double().clone()
    even, odd = ((slice(0, R, 2), slice(1, R, 2)) if case["interleaved"]
                 else (slice(0, R // 2), slice(R // 2, R)))
    z = torch.complex(x[..., even].contiguous(), x[..., odd].contiguous()) * turn[:, None, :]
    x[..., even], x[..., odd] = z.real, z.imag
    return x


def _exact_head(q, k, v, first, g=None):
    """One head in 64 bits: query i sees the keys up to first + i."""
    S = k.shape[0]
    scale = q.shape[1] ** -0.5
    at = torch.arange(q.shape[0], device=DEV)[:, None] + first
    s = (q @ k.t()) * scale
    s[torch.arange(S, device=DEV)[None, :] > at] = -math.inf
    p = torch.exp(s - torch.logsumexp(s, 1, keepdim=True))
    o = p @ v
    if g is None:
        return o
    t = g @ v.t()
    ds = p * (t - (p * t).sum(1, keepdim=True)) * scale
    return o, ds @ k, ds.t() @ q, p.t() @ g


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    H, Hk = case["heads"], case["kv_heads"]
    G = H // Hk
    if kind == "append":
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        slots = st["slots"].long()
        kc.view(-1, *kc.shape[2:])[slots] = _exact_rotate(st["k"], case, st["positions"])
        vc.view(-1, *vc.shape[2:])[slots] = st["v"].double()
        return {"q": _exact_rotate(st["q"], case, st["positions"]), "k_cache": kc, "v_cache": vc}
    if kind == "rotary":
        out = {n: _exact_rotate(st[n].detach(), case, st["positions"]) for n in "qk"}
        if case["train"]:
            out["dq"] = _exact_rotate(st["gq"], case, st["positions"], -1.0)
            out["dk"] = _exact_rotate(st["gk"], case, st["positions"], -1.0)
        return out
    if kind == "prompt":
        q, k, v = (st[n].detach().double() for n in "qkv")
        g = st["g"].double() if case["train"] else None
        out, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
        at = st["cu"].tolist()
        for a, b in zip(at[:-1], at[1:]):
            for h in range(H):
                n = h // G
                if g is None:
                    out[a:b, h] = _exact_head(q[a:b, h], k[a:b, n], v[a:b, n], 0)
                    continue
                o, x, y, z = _exact_head(q[a:b, h], k[a:b, n], v[a:b, n], 0, g[a:b, h])
                out[a:b, h], dq[a:b, h] = o, x
                dk[a:b, n] += y
                dv[a:b, n] += z
        return out if g is None else {"out": out, "dq": dq, "dk": dk, "dv": dv}
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    page, at = case["page"], 0
    for b, (n, c) in enumerate(zip(_ints(case["new"]), _ints(case["context"]))):
        j = torch.arange(c, device=DEV)
        places = st["block_table"][b].long()[j // page], j % page
        k, v = st["k_cache"][places].double(), st["v_cache"][places].double()
        q = st["q"][at:at + n].double()
        for h in range(H):
            out[at:at + n, h] = _exact_head(q[:, h], k[:, h // G], v[:, h // G], c - n)
        at += n
    return out
