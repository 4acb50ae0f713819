"""Attention of bf16 values near the end of their range, and of inputs that are
not finite in whole steps."""
import math

import pytest
import torch

from attention_check import check, one

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def A():
    from distributed_gptq_amd.models import attention
    return attention


def near_the_end(L, H, Hk, D, seed=0):
    """q, k, v, grad: values up to bf16's largest, scores that rise by less than
    the rescaling's slack at a time, equal ones, and ordinary ones."""
    g = torch.Generator(device="cuda").manual_seed(seed + L)
    q, k = torch.randn(L, H, D, generator=g, device="cuda"), torch.randn(L, Hk, D, generator=g, device="cuda")
    k[:, 0] = torch.linspace(0, 30, L, device="cuda")[:, None] / 8
    q[:, 0] = 1.0
    if Hk > 1:
        k[:, 1] = 0.0
    v = torch.randn(L, Hk, D, generator=g, device="cuda").clamp(-1, 1) * torch.finfo(BF16).max
    v[..., 0] = torch.finfo(BF16).max
    v[..., 1] = -torch.finfo(BF16).max
    grad = torch.randn(L, H, D, generator=g, device="cuda") * 1e-8
    return [x.to(BF16) for x in (q, k, v, grad)]


@pytest.mark.parametrize("L", [1, 60, 700])
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (2, 2, 128)])
def test_values_near_the_largest(L, H, Hk, D):
    """A weighted mean of finite values is finite."""
    q, k, v, grad = near_the_end(L, H, Hk, D)
    want = one(q, k, v, grad)
    with torch.no_grad():
        check(A().attention(q, k, v), want["out"])
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    out = A().attention(q, k, v)
    check(out.detach(), want["out"])
    for name, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), grad)):
        check(x, want[name])


@pytest.mark.parametrize("new", [1, 3, 200])
@pytest.mark.parametrize("L", [200, 700, 5000])
def test_values_near_the_largest_over_a_cache(new, L):
    """In one part and in many, both kernels."""
    H, Hk, D, page = 8, 2, 64, 16
    q, k, v, _ = near_the_end(L, H, Hk, D)
    pages = -(-L // page)
    kc, vc = torch.zeros(2, pages * page, Hk, D, device="cuda", dtype=BF16)
    kc[:L], vc[:L] = k, v
    table = torch.arange(pages, device="cuda", dtype=torch.int32)[None]
    cu = torch.tensor([0, new], dtype=torch.int32, device="cuda")
    out = A().paged_attention(q[:new], kc.view(pages, page, Hk, D), vc.view(pages, page, Hk, D), table,
                              torch.tensor([L], device="cuda"), cu)
    check(out, one(q[:new], k, v)["out"])
