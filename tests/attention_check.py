"""Per-element error bounds for the attention operators against 64 bits.

With u the type's unit roundoff (2^-8 bf16, 2^-11 fp16):

* A score s = c sum_d q_d k_d (c = scale log2 e) is an fp32 sum of exact
  products, |ds| <= (D + 4) 2^-24 c sum_d |q_d k_d|, and a weight 2^(s - m) /
  sum adds the exponential's and the division's roundings: its relative error
  is at most eps = 2 ((D + 4) 2^-24 c ln 2 max_ij sum_d |q_d k_d| + 2^-21).
* The output rounds each weight (u) and the result (u), in sums of absolute
  value A = sum_j p_j |v_j|: |do| <= (2 u + u^2 + eps + n 2^-24) A, and n
  2^-31 max |v| in fp16, whose weights end at 2^-25 of their unit while the
  largest is at least 2^6 of it.  With a gradient to follow, the weights have
  twice the bits, which the bound does not use.
* ds_ij = p_ij (g_i v_j - delta_i) has an error of at most eta E_ij, E_ij =
  p_ij (|g_i| |v_j| + sum_j' p_ij' |g_i| |v_j'|), eta = eps + 8 u^2 + 2^-20
  (delta is of an output with the weights' and its own rounding error left in
  second order), and is rounded once (u): dq, dk <= scale (u |ds| + (eta +
  n 2^-24) E) times |k|, |q|, plus u of the result.  In fp16 ds is rounded as
  a multiple of 2^-25 / 2^e, with 2^e >= 2^13 / (2 max |g| max |v|).
* dv <= (2 u + eps + n 2^-24) sum_i p_ij |g_i|, and n 2^-38 max |g| in fp16.

fp32 ends at 2^-126 (the exponential gives zero below): n 2^-126 times the
largest value is added to each sum of weights times values.

The rows are few enough that 64-bit products of the absolute values give A and
E themselves.
"""
import math

import torch

UNIT = {dt: torch.finfo(dt).eps / 2 for dt in (torch.bfloat16, torch.float16, torch.float32)}


def heads_of(x, G=1):
    """(tokens, heads, dim) -> (heads G, tokens, dim), float64, contiguous."""
    return x.double().repeat_interleave(G, 1).transpose(0, 1).contiguous()


def t(x):
    return x.transpose(1, 2).contiguous()


def one(q, k, v, g=None, causal=True, scale=None, train=False):
    """One sequence: dict of name -> (value, bound), 64 bits, (tokens, heads, dim)."""
    dt, u = q.dtype, UNIT[q.dtype]
    Lq, H, D = q.shape
    Lk, Hk = k.shape[:2]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    if Lk == 0 or Lq == 0:
        z = {"out": torch.zeros(Lq, H, D, dtype=torch.float64, device=q.device)}
        if g is not None:
            z["dq"] = z["out"].clone()
            z["dk"] = torch.zeros(Lk, Hk, D, dtype=torch.float64, device=q.device)
            z["dv"] = z["dk"].clone()
        return {n: (x, torch.zeros_like(x)) for n, x in z.items()}
    q, k, v = heads_of(q), heads_of(k, G), heads_of(v, G)
    s = (q @ t(k)) * scale
    if causal:
        i = torch.arange(Lq, device=q.device)[:, None] + Lk - Lq
        s = s.masked_fill(torch.arange(Lk, device=q.device)[None] > i, -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    o = p @ v
    n = max(Lq, Lk)
    eps = 2 * ((D + 4) * 2.0 ** -24 * scale * (q.abs() @ t(k.abs())).max() + 2.0 ** -21)
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    low = n * 2.0 ** -126
    A = p @ v.abs()
    got = {"out": (o, (2 * u + u * u + eps + n * 2.0 ** -24) * A + low * v.abs().max() + (n * 2.0 ** -31 * v.abs().max() + tiny if tiny else 0))}
    if g is not None:
        g = heads_of(g)
        delta = (g * o).sum(-1, keepdim=True)
        ds = p * (g @ t(v) - delta)
        E = p * (g.abs() @ t(v.abs()) + (g.abs() * A).sum(-1, keepdim=True))
        eta = eps + 8 * u * u + 2.0 ** -20
        e = u * ds.abs() + (eta + n * 2.0 ** -24) * E + low * 2 * g.norm(dim=-1).max() * v.norm(dim=-1).max()
        if tiny:
            e = e + 2.0 ** -25 * 2 * g.norm(dim=-1).max() * v.norm(dim=-1).max() / 2.0 ** 13
        dq, dk, dv = scale * (ds @ k), scale * (t(ds) @ q), t(p) @ g
        bq = scale * (e @ k.abs()) + u * dq.abs() + tiny
        bk = scale * (t(e) @ q.abs())
        bv = (2 * u + eps + n * 2.0 ** -24) * (t(p) @ g.abs()) + low * g.abs().max()
        if tiny:
            bv = bv + n * 2.0 ** -38 * g.abs().max()

        def join(x):
            return x.view(Hk, G, Lk, D).sum(1)
        dk, dv, bk, bv = join(dk), join(dv), join(bk), join(bv)
        bk = bk + u * dk.abs() + tiny
        bv = bv + u * dv.abs() + tiny
        got.update(dq=(dq, bq), dk=(dk, bk), dv=(dv, bv))
    return {name: (x.transpose(0, 1), b.transpose(0, 1)) for name, (x, b) in got.items()}


def packed(q, k, v, cu_q, cu_k, g=None, causal=True, scale=None):
    """Several: name -> (value, bound) of packed rows; rows past the offsets are zero."""
    names = ["out"] + (["dq", "dk", "dv"] if g is not None else [])
    shape = {"out": q, "dq": q, "dk": k, "dv": v}
    got = {n: (torch.zeros_like(shape[n], dtype=torch.float64), torch.zeros_like(shape[n], dtype=torch.float64))
           for n in names}
    for a, b, c, d in zip(cu_q[:-1], cu_q[1:], cu_k[:-1], cu_k[1:]):
        r = one(q[a:b], k[c:d], v[c:d], g[a:b] if g is not None else None, causal, scale)
        for n in names:
            at = slice(a, b) if n in ("out", "dq") else slice(c, d)
            for x, y in zip(got[n], r[n]):
                x[at] = y
    return got


def check(value, want):
    """Every element of ``value`` within its bound of ``want`` = (value, bound)."""
    ref, bound = want
    assert value.shape == ref.shape, (value.shape, ref.shape)
    err = (value.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside; worst {float((err - bound).nan_to_num(1e30).max()):.3g} over"
