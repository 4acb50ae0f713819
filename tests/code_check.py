"""Error bounds for normed heads and quantised caches against 64 bits.

With u the type's unit roundoff (2^-8 bf16, 2^-11 fp16, 2^-24 fp32) and f = 2^-24:

* Norm: the sum of D squares in fp32 is off by at most (D + 4) f relative, its
  root and reciprocal add 3 f, so r = (mean x^2 + eps)^-1/2 is off by (D / 2 + 6) f
  relative; x r w adds 2 f, a rotation of two terms 2 f of their sizes more: kappa
  = (D / 2 + 12) f of |a cos| + |b sin| in all, then u of the result.
* Its gradient: with G the sizes' sum of the turned-back gradient, |dx| is off by
  (2 D + 40) f r (G w + |xhat| mean(G w |xhat|)) (a mean of D products, each of
  factors off by at most (D / 2 + 12) f) and u of the result; dw by (2 D + 40 + 256)
  f sum(G |xhat|) and u of the weights' type, no chain of additions being longer
  than 256 for the sizes tested: at most 32 rows a thread, 128 threads' sums, 32
  workgroups' and 32 at the end.
* A row quantised from values that are off by e: its scale by e / top and 2 f
  relative (two roundings), a code by half a step (1/2 for whole numbers; e4m3:
  2^-4 of the code, at least 2^-10) and by the rounding of x (top / max), 3 f of
  it: the row read back by half a step times the scale, 2 e and 2^-21 |x|.
* Attention: attention_check.one of the rows that the codes stand for.  Products
  are of whole codes, exact; the scale of a key adds 2 f to a score and that of a
  value 2 f to a weight, which the bound's eps (twice what the sums need, 2^-21 for
  the weight) covers.  fp16 weights are held relative to the largest scale: n 2^-31
  max |code| max scale in place of n 2^-31 max |v|.
"""
import math

import torch

from attention_check import UNIT, one

F = 2.0 ** -24
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -150


def turned(x, table, positions, interleaved, back=False):
    """(value, sum of the terms' sizes) of 64-bit heads."""
    if table is None:
        return x, x.abs()
    R = 2 * table.shape[2]
    c, s = table[positions.clamp(0, table.shape[0] - 1).long()].double()[:, None].unbind(2)
    s = -s if back else s
    y, size = x.clone(), x.abs()
    even, odd = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    a, b = x[..., even], x[..., odd]
    y[..., even], y[..., odd] = a * c - b * s, b * c + a * s
    size[..., even], size[..., odd] = a.abs() * c.abs() + b.abs() * s.abs(), b.abs() * c.abs() + a.abs() * s.abs()
    return y, size


def inverse_rms(x, eps):
    return (x.square().mean(-1, keepdim=True) + eps).rsqrt()


def normed(x, w, table, positions, interleaved=False, eps=1e-6):
    """(value, error before the last rounding) of normed and turned heads."""
    x = x.double()
    z = x if w is None else x * inverse_rms(x, eps) * w.double()
    y, size = turned(z, table, positions, interleaved)
    return y, (x.shape[-1] / 2 + 12) * F * size


def rounded(y, e, dtype):
    return y, e + UNIT[dtype] * (y.abs() + e) + tiny(dtype)


def norm_gradients(x, w, g, table, positions, interleaved=False, eps=1e-6):
    """dx and dw, each (value, bound)."""
    dt, D = x.dtype, x.shape[-1]
    x64, w64 = x.double(), w.double()
    g, size = turned(g.double(), table, positions, interleaved, back=True)
    r = inverse_rms(x64, eps)
    hat = x64 * r
    p, P = g * w64, size * w64.abs()
    dx = r * (p - hat * (p * hat).mean(-1, keepdim=True))
    e = (2 * D + 40) * F * r * (P + hat.abs() * (P * hat.abs()).mean(-1, keepdim=True))
    dw = (g * hat).sum((0, 1))
    ew = (2 * D + 40 + 256) * F * (size * hat.abs()).sum((0, 1))
    return rounded(dx, e, dt), rounded(dw, ew, w.dtype)


def stored(y, e, code):
    """(value, bound) of rows read back in 64 bits after quantising values y that are off by e."""
    top = TOP[code]
    scale = y.abs().amax(-1, keepdim=True) / top
    worst = e.amax(-1, keepdim=True)
    if code == torch.int8:
        half = 0.5 * scale
    else:
        half = torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * scale)
    return y, half * (1 + 2.0 ** -18) + 2 * worst + 2.0 ** -21 * y.abs()


def attended(q, kc, ks, vc, vs, scale=None):
    """One sequence: (value, bound) of q over codes (tokens, heads, dim) and scales (tokens, heads)."""
    k, v = kc.double() * ks.double()[..., None], vc.double() * vs.double()[..., None]
    y, b = one(q, k, v, scale=scale)["out"]
    if q.dtype == torch.float16 and k.shape[0]:
        b = b + k.shape[0] * 2.0 ** -31 * vc.double().abs().max() * vs.double().max()
    return y, b


def quantised(x, code):
    """Codes and scales of fp32 rows by the formula in fp32, operation by operation
    (a quotient with a Python number may be a product with its reciprocal on the
    GPU: both sides are tensors)."""
    x = x.float()
    most = x.abs().amax(-1, keepdim=True)
    top = torch.full_like(most, TOP[code])
    some = most > 2.0 ** -120
    y = x * torch.where(some, top / most, torch.zeros_like(most))
    y = torch.minimum(torch.maximum(y, -top), top)
    codes = y.round().to(torch.int8) if code == torch.int8 else y.to(code)
    scale = most / top
    past = scale.double() * TOP[code] > torch.finfo(torch.float32).max  # (of fp32's largest values)
    scale = torch.where(past, torch.nextafter(scale, torch.zeros_like(scale)), scale)
    return codes, torch.where(some, scale, torch.zeros_like(most)).squeeze(-1)
