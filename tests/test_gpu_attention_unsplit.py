"""The gradient of attention where the query rows of a tile of keys are not cut
into parts (many keys and key heads): the products and what is made again where
they are not finite, which write dk and dv themselves."""
import math

import pytest
import torch

from attention_check import check, packed

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def inputs(lens_q, lens_k, H, Hk, D, dtype):
    g = torch.Generator(device="cuda").manual_seed(sum(lens_q) + D)

    def rand(t, h, scale):
        return (torch.randn(t, h, D, generator=g, device="cuda") * scale).to(dtype)
    T, S = sum(lens_q), sum(lens_k)
    return rand(T, H, 2.0), rand(S, Hk, 1.0), rand(S, Hk, 1.0), rand(T, H, 1e-2)


def run(q, k, v, grad, cq, ck, causal=True):
    from distributed_gptq_amd import _lib
    from distributed_gptq_amd.models import attention as A
    S, Hk, D = k.shape
    T, H = q.shape[:2]
    n = _lib.lib().gptq_attention_backward_workspace_size(len(cq) - 1, T, S, H, Hk, D)
    assert n == 4 * (-(-T * H // 4) * 4 + 2048)  # (no room for parts)
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    cq, ck = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (cq, ck))
    out = A.attention(q, k, v, cq, ck, causal=causal)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), grad)
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens_q,lens_k,H,Hk,D", [
    ((961,), (961,), 64, 64, 8), ((700, 1, 263), (700, 1, 263), 64, 64, 64), ((300, 5), (129, 1000), 128, 64, 40),
    ((200,), (1000,), 128, 64, 128), ((100,), (4001,), 16, 16, 96)])
def test_gradients(lens_q, lens_k, H, Hk, D, causal, dtype):
    x = inputs(lens_q, lens_k, H, Hk, D, dtype)
    cq, ck = offsets(lens_q), offsets(lens_k)
    want = packed(*x[:3], cq, ck, x[3], causal)
    got = run(*x, cq, ck, causal)
    for name in want:
        check(got[name], want[name])


@pytest.mark.parametrize("dtype", TYPES)
def test_not_finite_in_places_that_a_row_does_not_see(dtype):
    lens = (100, 900)
    q, k, v, grad = inputs(lens, lens, 64, 64, 40, dtype)
    cu = offsets(lens)
    want = packed(q, k, v, cu, cu, grad)

    def part(name, at):
        return tuple(x[at] for x in want[name])
    for bad in (math.nan, math.inf):
        for place in (0, 63, 99):
            k2, v2 = k.clone(), v.clone()
            k2[place], v2[place] = bad, bad
            got = run(q, k2, v2, grad, cu, cu)
            check(got["dq"][:place], part("dq", slice(0, place)))
            for name in ("dq", "dk", "dv"):
                check(got[name][100:], part(name, slice(100, None)))
            q2, g2 = q.clone(), grad.clone()
            q2[place], g2[place] = bad, bad
            got = run(q2, k, v, g2, cu, cu)
            for name in ("dq", "dk", "dv"):
                check(got[name][place + 1:], part(name, slice(place + 1, None)))
            check(got["dq"][:place], part("dq", slice(0, place)))


def test_same_bits_from_call_to_call():
    x = inputs((961,), (961,), 128, 64, 64, torch.bfloat16)
    a, b = (run(*x, [0, 961], [0, 961]) for _ in range(2))
    assert all(torch.equal(a[n], b[n]) for n in a)
