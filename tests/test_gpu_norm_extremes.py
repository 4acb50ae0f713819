"""Normed heads whose reciprocal roots and weights are far apart: against 64 bits
(bounds of code_check.py), into outputs and into a cache."""
import pytest
import torch

from attention_check import check
from code_check import normed, rounded, stored
from test_gpu_code_cache import empty_cache, gen

pytestmark = pytest.mark.gpu


def A():
    from distributed_gptq_amd.models import attention
    return attention


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [8, 64, 200])
@pytest.mark.parametrize("size,weight", [(1e34, 1e-6), (1e36, 1e-10), (1e-7, 1e34), (1e30, 1e30), (1e-10, 1e-30)])
def test_weights_far_from_the_roots(size, weight, D, dtype):
    """x r is near 1 (or small beside eps), and x r w a number, where r w leaves
    fp32's normal range on either side."""
    g = gen(D)
    q, k = ((torch.randn(9, n, D, generator=g, device="cuda") * size).to(dtype) for n in (3, 2))
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g, device="cuda")) * weight for _ in "qk")
    table, pos = A().rotary_table(D // 2, 50), torch.arange(9, device="cuda")
    got = A().norm_rotary(q, k, wq, wk, table, pos, eps=1e-12)
    for y, x, w in zip(got, (q, k), (wq, wk)):
        check(y, rounded(*normed(x, w, table, pos, eps=1e-12), dtype))


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
def test_weights_far_from_the_roots_into_a_cache(code):
    D, g = 64, gen(1)
    x = torch.randn(16, 2, D, generator=g, device="cuda") * 1e35
    w = (1 + 0.3 * torch.randn(D, generator=g, device="cuda")) * 1e-8
    (kc, ks), (vc, vs) = (empty_cache(1, 16, 2, D, code) for _ in "kv")
    A().rotary_append(x, x, x, None, None, kc, vc, torch.arange(16, device="cuda"), k_scale=ks, v_scale=vs, q_weight=w, k_weight=w)
    check(kc[0].double() * ks[0].double()[..., None], stored(*normed(x, w, None, None), code))
