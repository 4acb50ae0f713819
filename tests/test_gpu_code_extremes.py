"""Attention over codes of rows whose sums are not finite, or whose scales rise by
more powers of two than one fp32 factor spans: against 64 bits, and the same with
contexts in one part and in many.  And the smallest rows that are quantised."""
import math

import pytest
import torch

from attention_check import check
from code_check import attended
from test_gpu_attention_guards import ints
from test_gpu_code_cache import case, empty_cache, expect, gen
from test_gpu_paged_attention import offsets

pytestmark = pytest.mark.gpu
CODES = [torch.int8, torch.float8_e4m3fn]
TYPES = [torch.bfloat16, torch.float16]
PAGE = 16


def A():
    from distributed_gptq_amd.models import attention
    return attention


def places(table, b, n):
    j = torch.arange(n, device="cuda")
    return table[b].long()[j // PAGE], j % PAGE


# ------------------------------------------------------- sums that are no numbers --
# (one part, 2, up to 8 and more: for few rows a part has at least 128 keys, for
# many 512)

@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,context", [(1, 100), (1, 200), (1, 900), (1, 5000), (12, 200), (12, 5000), (100, 600), (100, 3000),
                                         (100, 9000)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_queries_that_are_not_finite(new, context, bad, dtype, code):
    """One head of one token: its output is NaN, whatever the number of parts,
    and no other one changes."""
    q, kc, vc, table, s, rows = case((new,), (context,), PAGE, 4, 2, 128, dtype, code)
    want = expect(q, rows, (new,))
    q = q.clone()
    t, h = new // 2, 3
    q[t, h, 17] = bad
    for longest in (None, 1, 16 * context):
        got = A().paged_attention(q, kc, vc, table, ints([context]), offsets([new]), max_context=longest, **s)
        assert bool(got[t, h].isnan().all())
        got[t, h] = 0
        y, b = (x.clone() for x in want)
        y[t, h], b[t, h] = 0, 0
        check(got, (y, b))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,context", [(1, 1), (1, 40), (5, 100), (20, 90), (70, 70), (140, 500)])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_a_scale_that_is_nan_in_a_short_sequence(which, new, context, dtype, code):
    """All keys in one part of many: NaN for the rows that see the key, the same
    rows whatever max_context says."""
    q, kc, vc, table, s, rows = case((new, 3), (context, 9), PAGE, 4, 2, 64, dtype, code)
    y, b = expect(q, rows, (new, 3))
    cu, ctx = offsets([new, 3]), ints([context, 9])
    for key in {0, context // 2, context - 1}:
        x = s[which].clone()
        x[table[0].long()[key // PAGE], key % PAGE, 1] = math.nan
        sees = torch.arange(context - new, context, device="cuda") >= key
        sees = torch.cat([sees, torch.zeros(3, dtype=torch.bool, device="cuda")])
        for longest in (1, 300, 1000, 100000):
            got = A().paged_attention(q, kc, vc, table, ctx, cu, max_context=longest, **{**s, which: x})
            assert bool(got[sees][:, 2:].isnan().all())
            got[sees, 2:] = 0
            yy, bb = y.clone(), b.clone()
            yy[sees, 2:], bb[sees, 2:] = 0, 0
            check(got, (yy, bb))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,context,past", [(1, 300, 128), (1, 300, 200), (1, 5000, 1500), (12, 300, 128), (100, 1300, 600),
                                              (100, 5000, 2600)])
def test_scores_of_minus_infinity(new, context, past, dtype, code):
    """The first keys' scores are below fp32's range: their weights are 0, in parts
    that have no other keys too.  Where all are, there is no mean: NaN."""
    q, kc, vc, table, s, rows = case((new,), (context,), PAGE, 4, 2, 64, dtype, code)
    q = q.clone()
    q[:, :, 0] = -60000.0
    k, ks, v, vs = rows[0]
    k, ks = k.view(torch.int8).clone(), ks.clone()
    k[:, :, 0] = 0
    k[:past] = 0
    k[:past, :, 0] = 0x70            # 112, or e4m3's 128
    ks[:past] = 2.0 ** 120           # -60000 * 112 * 2^120 / 8 is past -2^128
    at = places(table, 0, context)
    kc.view(torch.int8)[at], s["k_scale"][at] = k, ks
    want = attended(q, k[past:].view(code), ks[past:], v[past:], vs[past:])
    for longest in (None, 1):
        check(A().paged_attention(q, kc, vc, table, ints([context]), offsets([new]), max_context=longest, **s), want)
    for longest in (None, 1):
        got = A().paged_attention(q, kc, vc, table, ints([past]), offsets([new]), max_context=longest, **s)
        assert bool(got.isnan().all())


# -------------------------------------------------------------- scales that rise --

@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype,low,high", [(torch.bfloat16, -90, 90), (torch.bfloat16, -100, 110), (torch.bfloat16, -60, 70),
                                            (torch.bfloat16, -119, 20), (torch.float16, -90, 3)])
@pytest.mark.parametrize("new", [1, 5, 20, 140])
def test_scales_that_rise_along_the_keys(new, dtype, low, high, code):
    """Values of 2^low, then of 2^high, under equal scores and under ordinary ones:
    the weights of the first ones stay in the sum that divides."""
    q, kc, vc, table, s, rows = case((new,), (2048,), PAGE, 4, 2, 64, dtype, code)
    k, ks, v, vs = rows[0]
    vs = vs / vs.amax()
    vs = torch.cat([vs[:1000] * 2.0 ** low, vs[1000:] * 2.0 ** high])
    s["v_scale"][places(table, 0, 2048)] = vs
    for queries in (torch.zeros_like(q), q):
        want = attended(queries, k, ks, v, vs)
        for longest in (None, 1):
            check(A().paged_attention(queries, kc, vc, table, ints([2048]), offsets([new]), max_context=longest, **s), want)


# ----------------------------------------------------------- the smallest rows --

@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_above_the_smallest_that_are_quantised(dtype, code):
    """Rows whose largest value is a little above 2^-120, beside zeros and values
    below fp32's normal range: the codes of the same rows 2^64 as large, and finite
    rows read back; up to 2^-120 zeros."""
    m, D, n = A(), 32, 40
    g = gen(11)
    x = torch.randn(n, 1, D, generator=g, device="cuda").clamp(-1, 1)
    x[:, 0, 3:9] = 0.0
    x[:, 0, 9] *= 2.0 ** -15
    top = 2.0 ** torch.linspace(0, 4, n, device="cuda").double()
    x[:, 0, 11] = 1.0
    small = (x.double() * top[:, None, None] * 2.0 ** -120).to(dtype)
    small[0] = small[0].sign() * 2.0 ** -120       # not above the border
    big = (small.double() * 2.0 ** 64).to(dtype)
    assert torch.equal(small.double() * 2.0 ** 64, big.double())

    def write(y):
        (kc, ks), (vc, vs) = (empty_cache(1, n, 1, D, code) for _ in "kv")
        m.rotary_append(y, y, y, None, None, kc, vc, torch.arange(n, device="cuda"), k_scale=ks, v_scale=vs)
        table, cu = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), ints([0, n])
        back = m.cached_rows(kc, vc, table, ints([n]), cu, n, torch.float32, k_scale=ks, v_scale=vs)
        assert torch.equal(kc.view(torch.int8), vc.view(torch.int8)) and torch.equal(ks, vs) and torch.equal(*back)
        return kc[0], ks[0], back[0]
    got, want = write(small), write(big)
    assert bool((got[0][0].float() == 0).all()) and float(got[1][0]) == 0.0   # (e4m3 has a -0 too)
    assert torch.equal(got[0][1:].view(torch.int8), want[0][1:].view(torch.int8))
    # (scales and products end at 2^-149; 2^-21 of the largest for the code's product)
    assert bool(((got[1][1:].double() * 2.0 ** 64 - want[1][1:].double()).abs() <= 2.0 ** -85).all())
    err = (got[2][1:].double() - small[1:].double()).abs()
    most = small[1:].double().abs().amax(-1, keepdim=True)
    if code == torch.int8:   # half a step, and what the scale's end leaves of the largest code
        bound = most / 254 * (1 + 2.0 ** -18) + 127 * 2.0 ** -149 + 2.0 ** -21 * most
    else:
        bound = torch.maximum(2.0 ** -4 * small[1:].double().abs(), most / 448 * 2.0 ** -10) * (1 + 2.0 ** -18)
        bound = bound + 449 * 2.0 ** -149 + 2.0 ** -21 * most
    assert bool((err <= bound).all())
