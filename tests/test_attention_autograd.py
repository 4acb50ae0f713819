"""The attention operators' derivatives: what they do not have raises, and is
never left out silently.  On the CPU with stand-ins for the kernels, which the
operators' own autograd calls."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx

from distributed_gptq_amd import _lib
from distributed_gptq_amd.models import attention as A

T, H, Hk, D = 6, 4, 2, 8


def plain(q, k, v, scale):
    """(out, p) of one causal sequence, fp32."""
    k, v = (x.repeat_interleave(q.shape[1] // x.shape[1], 1) for x in (k, v))
    s = torch.einsum("ihd,jhd->hij", q, k) * scale
    p = s.masked_fill(torch.ones_like(s).triu(1).bool(), -math.inf).softmax(-1)
    return torch.einsum("hij,jhd->ihd", p, v), p


def turn(x, table, positions, inverse):
    c, s = table[positions.long()].unsqueeze(2).unbind(1)
    a, b = x.chunk(2, -1)
    s = -s if inverse else s
    return torch.cat([a * c - b * s, b * c + a * s], -1)


@pytest.fixture
def stand_ins():
    try:
        _lib.load_torch_ops()
    except Exception as e:
        pytest.skip(f"libraries not built: {e}")
    lib = torch.library.Library("gptq", "IMPL")

    def forward(q, k, v, cu_q, cu_k, causal, scale):
        out, _ = plain(q, k, v, scale)
        return out, torch.zeros_like(out), torch.zeros(q.shape[:2])

    def backward(grad, q, k, v, out, rest, lse, cu_q, cu_k, causal, scale):
        G = q.shape[1] // k.shape[1]
        p = plain(q, k, v, scale)[1]
        kk, vv = (x.repeat_interleave(G, 1) for x in (k, v))
        ds = scale * p * (torch.einsum("ihd,jhd->hij", grad, vv) - (grad * out).sum(-1).t()[..., None])

        def shared(x):
            return x.unflatten(1, (-1, G)).sum(2)
        return (torch.einsum("hij,jhd->ihd", ds, kk), shared(torch.einsum("hij,ihd->jhd", ds, q)),
                shared(torch.einsum("hij,ihd->jhd", p, grad)))

    def append(q, k, v, table, positions, k_cache, v_cache, slots, interleaved):
        return q.clone()
    lib.impl("attention", lambda q, k, v, cu_q, cu_k, causal, scale: plain(q, k, v, scale)[0], "CPU")
    lib.impl("attention_forward", forward, "CPU")
    lib.impl("attention_backward", backward, "CPU")
    lib.impl("rotary", lambda q, k, t, p, i, inverse: (turn(q, t, p, inverse), turn(k, t, p, inverse)), "CPU")
    lib.impl("rotary_append", append, "CPU")
    lib.impl("paged_attention", lambda q, *a: q.clone(), "CPU")
    yield
    lib._destroy()


def heads():
    g = torch.Generator().manual_seed(0)
    return [torch.randn(T, n, D, generator=g) for n in (H, Hk, Hk)]


def table_and_positions():
    return A.rotary_table(D, 16, device="cpu"), torch.arange(T)


def calls():
    """name -> a call of the operator with its q."""
    q, k, v = heads()
    table, pos = table_and_positions()
    kc, vc = torch.zeros(2, 4, Hk, D), torch.zeros(2, 4, Hk, D)
    bt, ctx = torch.zeros(T, 2, dtype=torch.int32), torch.ones(T, dtype=torch.int32)
    raw = torch.ops.gptq
    return {
        "attention": lambda q: A.attention(q, k, v),
        "attention of keys": lambda q: A.attention(k, q[:, :Hk], v),
        "attention of values": lambda q: A.attention(k, k, q[:, :Hk]),
        "rotary": lambda q: A.rotary(q, k, table, pos)[0],
        "rotary of keys": lambda q: A.rotary(k, q, table, pos)[1],
        "rotary_append": lambda q: A.rotary_append(q, k, v, table, pos, kc, vc, pos),
        "paged_attention": lambda q: A.paged_attention(q, kc, vc, bt, ctx),
        "attention_forward": lambda q: raw.attention_forward(q, k, v, None, None, True, 0.5)[0],
        "attention_backward": lambda q: raw.attention_backward(q, q, k, v, q, q, q[..., 0], None, None, True, 0.5)[0],
    }


NAMES = ["attention", "attention of keys", "attention of values", "rotary", "rotary of keys", "rotary_append",
         "paged_attention", "attention_forward", "attention_backward"]


def test_the_stand_ins_are_differentiated(stand_ins):
    q, k, v = (x.requires_grad_(True) for x in heads())
    table, pos = table_and_positions()
    qr, kr = A.rotary(q, k, table, pos)
    out = A.attention(qr, kr, v)
    g = torch.ones_like(out)
    got = torch.autograd.grad(out, (q, k, v), g)
    ref = plain(turn(q, table, pos, False), turn(k, table, pos, False), v, D ** -0.5)[0]
    for x, y in zip(got, torch.autograd.grad(ref, (q, k, v), g)):
        assert torch.allclose(x, y, atol=1e-5)


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_raises(stand_ins, name):
    call = calls()[name]
    q, _, _ = heads()
    assert call(q) is not None
    with fw.dual_level():
        call(q)  # a level is open, but nothing has a tangent
        with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            call(fw.make_dual(q, torch.ones_like(q)))
        with pytest.raises((RuntimeError, NotImplementedError), match="forward"), torch.no_grad():
            call(fw.make_dual(q, torch.ones_like(q)))
    with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
        torch.func.jvp(call, (q,), (torch.ones_like(q),))


def test_forward_over_reverse_raises(stand_ins):
    q, k, v = heads()
    table, pos = table_and_positions()
    with fw.dual_level():
        for f in (lambda x: A.attention(x, k, v), lambda x: A.rotary(x, k, table, pos)[0]):
            x = q.clone().requires_grad_(True)
            y = f(x)
            with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
                torch.autograd.grad(y, x, fw.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_a_table_that_requires_a_gradient_raises(stand_ins):
    """It would get none: the tables are constants."""
    q, k, v = heads()
    table, pos = table_and_positions()
    table.requires_grad_(True)
    cache = torch.zeros(2, 4, Hk, D)
    for x in (q, q.clone().requires_grad_(True)):
        with pytest.raises(RuntimeError, match="table"):
            A.rotary(x, k, table, pos)
    with pytest.raises(RuntimeError, match="gradient"):
        A.rotary_append(q, k, v, table, pos, cache, cache.clone(), pos)
    with torch.no_grad():
        want = A.rotary(q, k, table, pos)
        A.rotary_append(q, k, v, table, pos, cache, cache.clone(), pos)
    assert torch.equal(A.rotary(q, k, table.detach(), pos)[0], want[0])


TRACES = {"make_fx": lambda f, x: make_fx(f)(*x), "jit": lambda f, x: torch.jit.trace(f, x, check_trace=False)}


@pytest.mark.parametrize("trace,gradient", [("make_fx", False), ("make_fx", True), ("jit", False)])
def test_traces_hold_the_operators(stand_ins, trace, gradient):
    """A trace of rotary and attention, with the gradient too, computes other
    inputs' results."""
    table, pos = table_and_positions()

    def step(q, k, v, g):
        if not gradient:
            return (A.attention(*A.rotary(q, k, table, pos), v),)
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
        out = A.attention(*A.rotary(q, k, table, pos), v)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), g))
    x = (*heads(), torch.ones(T, H, D))
    other = [torch.flip(y, (0,)) * 0.5 for y in x]
    for got, want in zip(TRACES[trace](step, x)(*other), step(*other)):
        assert torch.equal(got, want)
