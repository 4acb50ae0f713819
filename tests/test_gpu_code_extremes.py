"""Attention over codes of rows whose sums are not finite, or whose scales rise by
more powers of two than one fp32 factor spans: against 64 bits, and the same with
contexts in one part and in many."""
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
