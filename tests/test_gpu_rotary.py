"""Rotary positions against 64 bits: both pairings, parts of a head, odd sizes,
strides, the gradient, and the cache's update."""
import math

import pytest
import torch

from attention_check import UNIT, check

pytestmark = pytest.mark.gpu


def A():
    from distributed_gptq_amd.models import attention
    return attention


def turned(x, table, positions, interleaved, sign=1.0):
    """(value, bound): three fp32 roundings and the angles' own, then one to the type."""
    R = 2 * table.shape[2]
    c, s = table[positions.clamp(0, table.shape[0] - 1).long()].double()[:, None].unbind(2)
    s = sign * s
    y = x.double().clone()
    bound = torch.zeros_like(y)
    even, odd = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    a, b = x.double()[..., even], x.double()[..., odd]
    y[..., even], y[..., odd] = a * c - b * s, b * c + a * s
    size = (a.abs() * c.abs() + b.abs() * s.abs(), b.abs() * c.abs() + a.abs() * s.abs())
    for at, z in zip((even, odd), size):
        bound[..., at] = 3 * 2.0 ** -24 * z + UNIT[x.dtype] * (1 + 2.0 ** -20) * y[..., at].abs() + 2.0 ** -25 * (
            x.dtype == torch.float16)
    return y, bound


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,Hk,D,R", [(4, 2, 64, 64), (3, 1, 128, 64), (2, 2, 40, 20), (1, 1, 2, 2), (5, 5, 96, 96),
                                      (2, 1, 6, 4), (32, 8, 128, 128)])
@pytest.mark.parametrize("T", [1, 5, 300])
def test_rotary_and_gradient(T, H, Hk, D, R, interleaved, dtype):
    m = A()
    g = torch.Generator(device="cuda").manual_seed(T + D + R)
    table = m.rotary_table(R, 500, base=500.0)
    pos = torch.randint(0, 500, (T,), generator=g, device="cuda")
    q = torch.randn(T, H, D, generator=g, device="cuda").to(dtype).requires_grad_(True)
    k = torch.randn(T, Hk, D, generator=g, device="cuda").to(dtype).requires_grad_(True)
    gq, gk = (torch.randn(x.shape, generator=g, device="cuda").to(dtype) for x in (q, k))
    qo, ko = m.rotary(q, k, table, pos, interleaved=interleaved)
    for x, y in ((q, qo), (k, ko)):
        check(y.detach(), turned(x.detach(), table, pos, interleaved))
        assert torch.equal(y[..., R:], x[..., R:])
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk))
    check(dq, turned(gq, table, pos, interleaved, -1.0))
    check(dk, turned(gk, table, pos, interleaved, -1.0))
    with torch.no_grad():
        q2, k2 = m.rotary(q, k, table, pos.int(), interleaved=interleaved)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)


def test_gradient_against_differences():
    """In fp32, a linear map: differences at step 1 give the gradient up to the
    rounding of their terms."""
    m = A()
    g = torch.Generator(device="cuda").manual_seed(1)
    table, pos = m.rotary_table(8, 50), torch.arange(3, device="cuda")
    q = torch.randn(3, 2, 12, generator=g, device="cuda").requires_grad_(True)
    gq = torch.randn(3, 2, 12, generator=g, device="cuda")
    for interleaved in (False, True):
        out, _ = m.rotary(q, q, table, pos, interleaved)
        dq, = torch.autograd.grad(out, q, gq)
        for t, h, d in ((0, 0, 0), (1, 1, 3), (2, 0, 5), (2, 1, 11)):
            p = q.detach().clone()
            p[t, h, d] += 1.0
            diff = (m.rotary(p, p, table, pos, interleaved)[0] - out.detach()).double()
            size = 2 * 4 * 2.0 ** -24 * (q.abs().max() + 1.0) * 2 * gq.abs().sum()
            assert abs(float((diff * gq.double()).sum()) - float(dq[t, h, d])) <= size


@pytest.mark.parametrize("dtype", list(UNIT))
def test_strides_and_positions(dtype):
    m = A()
    g = torch.Generator(device="cuda").manual_seed(2)
    T, H, Hk, D = 33, 4, 2, 64
    fused = torch.randn(T, H + 2 * Hk, D, generator=g, device="cuda").to(dtype)
    table, pos = m.rotary_table(D, 40), torch.arange(T, device="cuda")
    q, k = fused[:, :H], fused[:, H:H + Hk]
    want = m.rotary(q.contiguous(), k.contiguous(), table, pos)

    def odd(x):
        return torch.empty(x.numel() + 1, device="cuda", dtype=dtype)[1:].view(x.shape).copy_(x)
    for f in (lambda x: x, odd, lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),
              lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)):
        got = m.rotary(f(q), f(k), table, pos)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # positions outside the table are those of its ends
    far = m.rotary(q, k, table, torch.full((T,), 10 ** 6, device="cuda"))
    end = m.rotary(q, k, table, torch.full((T,), 39, device="cuda"))
    low = m.rotary(q, k, table, torch.full((T,), -3, device="cuda", dtype=torch.int32))
    assert torch.equal(far[0], end[0]) and torch.equal(low[0][..., :], m.rotary(q, k, table, pos * 0)[0])
    check(far[0], turned(q, table, torch.full((T,), 39, device="cuda"), False))


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,Hk,D,R,page", [(1, 8, 2, 128, 128, 16), (77, 3, 3, 40, 20, 24), (9, 2, 1, 64, 0, 1),
                                             (300, 4, 4, 64, 32, 64)])
def test_append(T, H, Hk, D, R, page, interleaved, dtype):
    """The queries and keys of ``rotary`` bit for bit, keys and values in their
    slots, every other place of the cache as it was, padding not stored."""
    m = A()
    g = torch.Generator(device="cuda").manual_seed(T + D)
    pages = -(-T // page) + 2
    fused = torch.randn(T, H + 2 * Hk, D, generator=g, device="cuda").to(dtype)
    q, k, v = fused[:, :H], fused[:, H:H + Hk], fused[:, H + Hk:]
    kc, vc = (torch.randn(pages, page, Hk, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T]
    if T > 5:
        slots[3], slots[5] = -1, pages * page  # padding
    pos = torch.randint(0, 100, (T,), generator=g, device="cuda")
    table = m.rotary_table(R, 100) if R else None
    qr, kr = m.rotary(q, k, table, pos, interleaved) if R else (q, k)
    kw, vw = kc.clone(), vc.clone()
    keep = (slots >= 0) & (slots < pages * page)
    kw.view(-1, Hk, D)[slots[keep]] = kr[keep]
    vw.view(-1, Hk, D)[slots[keep]] = v[keep]
    out = m.rotary_append(q, k, v, table, pos if R else None, kc, vc, slots, interleaved)
    assert torch.equal(out, qr) and torch.equal(kc, kw) and torch.equal(vc, vw)
    # a cache with heads before tokens
    k2, v2 = (x.transpose(1, 2).contiguous().transpose(1, 2).zero_() for x in (kc, vc))
    m.rotary_append(q, k, v, table, pos if R else None, k2, v2, slots.int(), interleaved)
    assert torch.equal(k2.reshape(-1, Hk, D)[slots[keep]], kr[keep]) and torch.equal(
        v2.reshape(-1, Hk, D)[slots[keep]], v[keep])


def test_refusals_and_empty():
    m = A()
    table = m.rotary_table(64, 10)
    x = torch.zeros(4, 2, 64, device="cuda").half()
    pos = torch.arange(4, device="cuda")
    for args in [(x, x[:3], table, pos), (x, x, table, pos[:3]), (x, x, table[:, :1], pos), (x, x, table[0], pos),
                 (x[..., :32], x[..., :32], table, pos), (x, x[..., :32], table, pos)]:
        with pytest.raises(ValueError):
            m.rotary(*args)
    for args in [(x, x, table.double(), pos), (x, x, table, pos.float()), (x, x.float(), table, pos),
                 (x.int(), x.int(), table, pos)]:
        with pytest.raises(TypeError):
            m.rotary(*args)
    y = torch.zeros(4, 2, 63, device="cuda").half()
    with pytest.raises(ValueError):
        m.rotary(y, y, table[..., :20].contiguous(), pos)
    cache = torch.zeros(2, 16, 2, 64, device="cuda").half()
    for args in [(x, x, x, table, None, cache, cache.clone(), pos), (x, x, x, table, pos, cache, cache[:1], pos),
                 (x, x, x, table, pos, cache, cache.clone(), pos[:2]), (x, x[:, :1], x[:, :1], table, pos, cache,
                                                                       cache.clone(), pos)]:
        with pytest.raises(ValueError):
            m.rotary_append(*args)
    with pytest.raises(RuntimeError, match="gradient"):
        m.rotary_append(x.clone().requires_grad_(True), x, x, table, pos, cache, cache.clone(), pos)
    e = m.rotary(x[:0], x[:0], table, pos[:0])
    assert e[0].shape == (0, 2, 64)
    before = cache.clone()
    m.rotary_append(x[:0], x[:0], x[:0], table, pos[:0], cache, cache.clone(), pos[:0])
    assert torch.equal(cache, before)
    assert math.isfinite(float(m.rotary(x, x, table, pos)[0].float().sum()))
