"""Normed and turned heads and their gradients against 64 bits (bounds of
code_check.py): sizes, types, layouts, values of any size, graphs and streams."""
import math

import pytest
import torch

from attention_check import UNIT, check
from code_check import norm_gradients, normed, rounded

pytestmark = pytest.mark.gpu
TYPES = list(UNIT)


def A():
    from distributed_gptq_amd.models import attention
    return attention


def inputs(T, H, Hk, D, dtype, wdtype, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + T + D)
    q, k = ((torch.randn(T, n, D, generator=g, device="cuda") * spread).to(dtype) for n in (H, Hk))
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(wdtype) for _ in "qk")
    gq, gk = (torch.randn(x.shape, generator=g, device="cuda").to(dtype) for x in (q, k))
    return q, k, wq, wk, gq, gk


def both(q, k, wq, wk, gq, gk, *args, **kw):
    x = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    qo, ko = A().norm_rotary(*x, *args, **kw)
    dq, dk, dwq, dwk = torch.autograd.grad((qo, ko), x, (gq, gk))
    return {"q": qo.detach(), "k": ko.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


def against(got, q, k, wq, wk, gq, gk, table=None, positions=None, interleaved=False, eps=1e-6):
    for n, x, w, g in (("q", q, wq, gq), ("k", k, wk, gk)):
        check(got[n], rounded(*normed(x, w, table, positions, interleaved, eps), x.dtype))
        dx, dw = norm_gradients(x, w, g, table, positions, interleaved, eps)
        check(got["d" + n], dx)
        check(got["dw" + n], dw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,Hk,D,R", [(4, 2, 64, 64), (3, 1, 128, 64), (32, 8, 128, 128), (2, 2, 40, 20), (5, 5, 96, 96),
                                      (1, 1, 8, 4), (1, 1, 8, 8), (7, 1, 256, 256), (3, 2, 200, 100), (2, 1, 80, 32)])
@pytest.mark.parametrize("T", [1, 5, 300])
def test_norm_rotary_and_gradients(T, H, Hk, D, R, interleaved, dtype):
    wdtype = TYPES[(T + H + D) % 3]
    x = inputs(T, H, Hk, D, dtype, wdtype)
    table = A().rotary_table(R, 500, base=500.0)
    pos = torch.randint(-3, 503, (T,), device="cuda")
    got = both(*x, table, pos, interleaved=interleaved)
    against(got, *x, table, pos, interleaved)
    with torch.no_grad():
        q2, k2 = A().norm_rotary(*x[:4], table, pos.int(), interleaved)
    assert torch.equal(q2, got["q"]) and torch.equal(k2, got["k"])
    again = both(*x, table, pos, interleaved=interleaved)
    for n in got:  # (the same bits from call to call)
        assert torch.equal(again[n], got[n])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [8, 24, 64, 136, 256])
def test_without_a_table(D, dtype):
    x = inputs(33, 3, 2, D, dtype, torch.float32)
    got = both(*x, eps=1e-3)
    against(got, *x, eps=1e-3)


def test_gradient_against_differences():
    """fp32, central differences at step h: off by h^2 of the third derivative
    and 2^-23 of the outputs over h."""
    m = A()
    q, k, wq, wk, gq, gk = inputs(3, 2, 1, 16, torch.float32, torch.float32)
    table, pos = m.rotary_table(8, 50), torch.arange(3, device="cuda")
    got = both(q, k, wq, wk, gq, gk, table, pos)
    h = 2.0 ** -7

    def loss(*x):
        a, b = m.norm_rotary(*x, table, pos)
        return float((a.double() * gq.double()).sum() + (b.double() * gk.double()).sum())
    size = float((gq.abs().sum() + gk.abs().sum())) * 4
    for i, n in enumerate(("dq", "dk", "dwq", "dwk")):
        for at in (0, 5, 13):
            sides = []
            for s in (h, -h):
                x = [t.clone() for t in (q, k, wq, wk)]
                x[i].view(-1)[at] += s
                sides.append(loss(*x))
            diff = (sides[0] - sides[1]) / (2 * h)
            # third derivatives of x / |x| sqrt(D) are at most 12 |g| / rms^3 here, rms > 1/2
            assert abs(diff - float(got[n].view(-1)[at])) <= h * h / 6 * 12 * 8 * float(gq.abs().max()) * 16 + 2.0 ** -23 * size / h


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    """Parts of a fused projection, transposed, misaligned and broadcast tensors:
    the same bits as contiguous ones."""
    m = A()
    T, H, Hk, D = 33, 4, 2, 64
    q, k, wq, wk, gq, gk = inputs(T, H, Hk, D, dtype, torch.bfloat16)
    table, pos = m.rotary_table(D, 64), torch.arange(T, device="cuda")
    want = both(q, k, wq, wk, gq, gk, table, pos)
    fused = torch.cat([q, k, k], 1)
    room = torch.zeros(T * H * D + 3, dtype=dtype, device="cuda")
    odd = room[3:].view(T, H, D).copy_(q)
    wide = torch.zeros(D, 2, dtype=wq.dtype, device="cuda")
    wide[:, 1] = wq
    big = torch.zeros(T + 1, 2, D // 2, device="cuda")
    for q2, k2, wq2, t2, p2 in (
            (fused[:, :H], fused[:, H:H + Hk], wq, table, pos.int()),
            (q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(1, 2).contiguous().transpose(1, 2), wide[:, 1], table, pos),
            (odd, k, torch.cat([wq[:1], wq])[1:], table.view(-1).repeat(2)[64 * D:].view(64, 2, D // 2), pos)):
        got = both(q2, k2, wq2, wk, gq.transpose(0, 1).contiguous().transpose(0, 1), gk, t2, p2)
        for n in want:
            assert torch.equal(got[n], want[n]), n
    del big
    # a broadcast gradient, and a sum's
    x = q.detach().requires_grad_(True)
    out, _ = m.norm_rotary(x, k, wq, wk, table, pos)
    a, = torch.autograd.grad(out, x, gq[:1, :1].expand_as(out), retain_graph=True)
    b, = torch.autograd.grad(out, x, gq[:1, :1].expand_as(out).contiguous(), retain_graph=True)
    assert torch.equal(a, b)
    a, = torch.autograd.grad(out.sum(), x, retain_graph=True)
    b, = torch.autograd.grad(out, x, torch.ones_like(out))
    assert torch.equal(a, b)
    # the same tensor twice: both parts of its gradient
    x = k.detach().requires_grad_(True)
    d, = torch.autograd.grad(m.norm_rotary(x, x, wq, wk, table, pos), x, (gk, gk))
    parts = [both(k, k, wq, wk, g1, g2, table, pos) for g1, g2 in ((gk, gk),)][0]
    assert torch.equal(d, parts["dq"] + parts["dk"])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_of_any_size(dtype):
    """Heads whose squares leave fp32 on either side, and zeros."""
    D = 64
    q, k, wq, wk, gq, gk = inputs(6, 2, 1, D, dtype, torch.float32)
    q = q.double()
    for t, f in enumerate((1e30, 1e18, 1e-6, 1e-18, 1e-30, 0.0)):
        q[t] *= f
    q = q.to(dtype)
    got = both(q, k, wq, wk, gq, gk)
    check(got["q"], rounded(*normed(q, wq, None, None), dtype))
    dx, _ = norm_gradients(q, wq, gq, None, None)
    check(got["dq"][:5], (dx[0][:5], dx[1][:5]))
    assert bool((got["q"][5] == 0).all()) and bool(torch.isfinite(got["dq"]).all()) and bool(torch.isfinite(got["dwq"]).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite_stay_in_their_heads(dtype):
    x = inputs(9, 3, 2, 96, dtype, dtype)
    want = both(*x)
    for bad in (math.nan, math.inf, -math.inf):
        q = x[0].clone()
        q[4, 1, 7] = bad
        got = both(q, *x[1:])
        others = torch.ones(9, 3, dtype=torch.bool, device="cuda")
        others[4, 1] = False
        for n in ("q", "dq"):
            assert torch.equal(got[n][others], want[n][others])
            assert bool(got[n][4, 1].isnan().any())
        for n in ("k", "dk", "dwk"):
            assert torch.equal(got[n], want[n])
        # the formula: others of the head over an infinite root are 0
        ref = normed(q[4:5, 1:2], x[2], None, None)[0]
        assert torch.equal(ref.isnan(), got["q"][4:5, 1:2].isnan())


def test_no_tokens():
    for wdtype in TYPES:
        got = both(*inputs(0, 2, 1, 64, torch.float16, wdtype))
        assert got["q"].shape == (0, 2, 64) and bool((got["dwq"] == 0).all()) and bool((got["dwk"] == 0).all())


def test_refusals():
    f = A().norm_rotary
    q, k, wq, wk, _, _ = inputs(4, 2, 1, 64, torch.float16, torch.float16)
    table, pos = A().rotary_table(64, 8), torch.arange(4, device="cuda")
    for args in [(q, k[:3], wq, wk), (q, k, wq[:32], wk), (q, k, wq[None], wk), (q[0], k[0], wq, wk),
                 (q, k, wq, wk, table, pos[:3]), (q, k, wq, wk, table), (q, k, wq, wk, table[:, :1], pos),
                 (q[..., :20], k[..., :20], wq[:20], wk[:20]), (q, k, wq, wk, A().rotary_table(62, 8), pos),
                 (q, k, wq, wk, A().rotary_table(128, 8), pos), (q, k, wq.cpu(), wk), (q, k, wq, wk, table.cpu(), pos),
                 (q, k, wq, wk, table, pos.cpu())]:
        with pytest.raises(ValueError):
            f(*args)
    for args in [(q, k.float(), wq, wk), (q, k, wq.float(), wk), (q, k, wq.double(), wk.double()),
                 (q, k, wq, wk, table.half(), pos), (q, k, wq, wk, table, pos.float())]:
        with pytest.raises(TypeError):
            f(*args)
    for eps in (0.0, -1.0, 2.0, math.nan):
        with pytest.raises(ValueError, match="eps"):
            f(q, k, wq, wk, eps=eps)


def test_graph_and_streams():
    """Forward and gradient captured together, replayed with other work between;
    and on another stream than the tensors'."""
    m = A()
    x = inputs(130, 8, 2, 128, torch.bfloat16, torch.float32)
    table, pos = m.rotary_table(128, 256), torch.arange(130, device="cuda")
    buf = [t.clone() for t in x]

    def step():
        return both(*buf, table, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
        graphs = []
        for _ in range(2):  # two graphs, each with a workspace of its own
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                out = step()
            graphs.append((graph, out))
    torch.cuda.synchronize()
    g = torch.Generator(device="cuda").manual_seed(9)
    for r in range(4):
        for b in buf:
            b.copy_(torch.randn(b.shape, generator=g, device="cuda").to(b.dtype))
        torch.cuda.synchronize()
        graphs[r % 2][0].replay()
        graphs[1 - r % 2][0].replay()
        torch.cuda.synchronize()
        kept = [{n: t.clone() for n, t in out.items()} for _, out in graphs]
        want = step()
        for got in kept:
            for n in want:
                assert torch.equal(got[n], want[n]), (r, n)
    with torch.cuda.stream(s):
        other = step()
    torch.cuda.current_stream().wait_stream(s)
    for n in want:
        assert torch.equal(other[n], want[n])
