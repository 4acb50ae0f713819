"""Attention over a quantised cache with many rows of a sequence: workgroups of
256 rows, whose two halves take turns, in pages of whole sixteens and others;
pages that lie more than 32 bits apart."""
import math

import pytest
import torch

from attention_check import check
from code_check import attended
from test_gpu_attention_guards import FAR, Room, ints, ptr, strides
from test_gpu_code_cache import A, CODES, TYPES, case, expect, gen, random_rows
from test_gpu_paged_attention import offsets

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (6, 2, 80), (12, 1, 112)])
@pytest.mark.parametrize("page,new,context", [
    (16, (300,), (300,)),
    (32, (257,), (3000,)),                # parts
    (40, (290,), (1111,)),                # half a sixteen at the end of each page
    (48, (400, 1, 0, 130), (401, 63, 70, 64)),
    (5, (260,), (700,)),
])
def test_many_rows(page, new, context, H, Hk, D, dtype, code):
    q, kc, vc, table, s, rows = case(new, context, page, H, Hk, D, dtype, code)
    want = expect(q, rows, new)
    for longest in (None, 1):
        check(A().paged_attention(q, kc, vc, table, ints(context), offsets(new), max_context=longest, **s), want)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 24])
def test_scales_that_are_not_finite(page, dtype, code):
    q, kc, vc, table, s, rows = case((300,), (500,), page, 4, 2, 128, dtype, code)
    cu, ctx = offsets((300,)), ints((500,))
    want = expect(q, rows, (300,))
    for which in ("k_scale", "v_scale"):
        for key in (0, 63, 64, 199, 255, 256, 498, 499):
            x = s[which].clone()
            x[table[0].long()[key // page], key % page, 1] = math.nan
            got = A().paged_attention(q, kc, vc, table, ctx, cu, **{**s, which: x})
            sees = torch.arange(200, 500, device="cuda") >= key
            assert bool(got[sees][:, 2:].isnan().all())
            clean, ref = got.clone(), [t.clone() for t in want]
            for t in (clean, *ref):
                t[sees, 2:] = 0
            check(clean, tuple(ref))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [60, 300])
def test_values_of_any_size(new, dtype, code):
    """Scales that differ by many orders, growing and falling along the keys."""
    q, kc, vc, table, s, rows = case((new,), (400,), 16, 8, 2, 128, dtype, code)
    j = torch.arange(400, device="cuda")
    for low, high in ((-20, 10), (90, 119), (-119, -90)) if dtype == torch.bfloat16 else ((-20, 10), (-12, 0)):
        for way in (1, -1):
            f = torch.exp2(torch.linspace(low, high, 400, device="cuda"))
            f = f if way == 1 else f.flip(0)
            vs = rows[0][3] / rows[0][3].amax() * f[:, None]
            vs[::7] = 0.0
            x = s["v_scale"].clone()
            x[table[0].long()[j // 16], j % 16] = vs
            got = A().paged_attention(q, kc, vc, table, ints([400]), offsets([new]), k_scale=s["k_scale"], v_scale=x)
            y, b = attended(q, *rows[0][:3], vs)
            # (fp16 ends at 65504: from 65520 on, half a step further, a value rounds to
            # infinity; between the bounds it may)
            if dtype == torch.float16:
                assert bool(got[y.abs() - b >= 65520].isinf().all())
            past = got.isinf() & (got.sign() == y.sign()) & (y.abs() + b >= 65520) & (dtype == torch.float16)
            got, y = got.masked_fill(past, 0.0), y.masked_fill(past, 0.0)
            # results below the type's normal range are off by half its smallest step
            check(got, (y, b + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)))


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_of_any_size(dtype):
    """Maxima that rise from tile to tile, far from zero on either side."""
    q, kc, vc, table, s, rows = case((300,), (700,), 16, 4, 2, 128, dtype, torch.int8)
    j = torch.arange(700, device="cuda")
    for f in (torch.linspace(0.02, 3, 700, device="cuda"), torch.linspace(3, 0.02, 700, device="cuda")):
        ks = rows[0][1] * f[:, None]
        x = s["k_scale"].clone()
        x[table[0].long()[j // 16], j % 16] = ks
        for qq in (q, q.abs()):
            got = A().paged_attention(qq, kc, vc, table, ints([700]), offsets([300]), k_scale=x, v_scale=s["v_scale"])
            check(got, attended(qq, rows[0][0], ks, *rows[0][2:]))


@pytest.mark.parametrize("code", [1, 2])
@pytest.mark.parametrize("page", [7, 16, 24])
def test_nothing_outside_is_touched(page, code):
    from distributed_gptq_amd import _lib
    H, Hk, D, pages, width, T = 4, 2, 112, 9, 70, 600
    g = gen(page)
    odd = [0, 3, pages, -1, FAR, -FAR - 1, pages - 1]
    for new, context, longest in (([0, 600], [600], 1), ([0, 600], [FAR], 5000), ([0, FAR], [1100], 5000), ([5, 300], [300], 1)):
        room = Room()
        q = room.input(torch.randn(T, H, D, generator=g, device="cuda").half())
        kc, vc = (room.empty(pages, page, Hk, D, dtype=torch.int8).fill_(3) for _ in "kv")
        ks, vs = (room.empty(pages, page, Hk, dtype=torch.float32).fill_(0.01) for _ in "kv")
        table = room.input(ints([[odd[i % 7] for i in range(width)]]))
        cu, ctx = room.input(ints(new)), room.input(ints(context))
        out = room.empty(T, H, D, dtype=torch.float16).zero_()
        n = _lib.lib().gptq_code_attention_workspace_size(1, T, H, Hk, D, longest)
        ws = room.empty(max(n, 1), dtype=torch.uint8).zero_()
        _lib.call("gptq_code_attention", ptr(q), 1, *strides(q), code, ptr(kc), *kc.stride()[:3], ptr(vc), *vc.stride()[:3],
                  ptr(ks), *ks.stride(), ptr(vs), *vs.stride(), ptr(table), width, width, page, pages, ptr(ctx), ptr(cu), 1, T,
                  H, Hk, D, 0.1, longest, ptr(out), ptr(ws), n, torch.cuda.current_stream().cuda_stream)
        room.check()
        assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("bits", [31, 32])
@pytest.mark.parametrize("new", [(1, 1), (6, 1), (40, 3), (300, 2)])
def test_pages_far_apart(new, bits):
    """Three pages of 16 tokens 2^bits bytes apart: offsets that pass 32 bits, by
    addresses of whole pages and by those of each row."""
    code, dtype, H, Hk, D, page, pages = torch.int8, torch.bfloat16, 4, 2, 128, 16, 3
    far, context = 2 ** bits, (33, 20)
    raw = torch.empty(2 * far + 2 * page * Hk * D, dtype=torch.int8, device="cuda")
    kc, vc = (raw[i * page * Hk * D:].as_strided((pages, page, Hk, D), (far, D, page * D, 1)) for i in (0, 1))
    ks, vs = (torch.full((pages, Hk, page), math.nan, device="cuda").transpose(1, 2) for _ in "kv")
    table = torch.tensor([[2, 1, 0], [1, 2, -1]], dtype=torch.int32, device="cuda")
    g = gen(bits)
    s = {"k_scale": ks, "v_scale": vs}
    # one sequence at a time: its rows are written through the append, and read back
    for b, (n, c) in enumerate(zip(new, context)):
        k, v = (torch.randn(c, Hk, D, generator=g, device="cuda").to(dtype) for _ in "kv")
        j = torch.arange(c, device="cuda")
        slots = (table[b].long()[j // page] * page + j % page).int()
        A().rotary_append(k, k, v, None, None, kc, vc, slots, **s)
        place = (table[b].long()[j // page], j % page)
        rows = [kc[place], ks[place], vc[place], vs[place]]
        back = A().cached_rows(kc, vc, table[b:b + 1], ints([c]), offsets([c]), c, torch.float32, **s)
        assert torch.equal(back[0], rows[0].float() * rows[1][..., None])
        assert torch.equal(back[1], rows[2].float() * rows[3][..., None])
        q = (torch.randn(n, H, D, generator=g, device="cuda") * 2).to(dtype)
        got = A().paged_attention(q, kc, vc, table[b:b + 1], ints([c]), offsets([n]), **s)
        check(got, attended(q, *rows))


@pytest.mark.parametrize("code", [1, 2])
@pytest.mark.parametrize("used,T", [(2, 40), (0, 7), (300, 700), (40, 41), (90, 130)])
def test_rows_behind_the_last_sequence_are_zeros(used, T, code):
    """A padded batch: whatever the output held."""
    from distributed_gptq_amd import _lib
    H, Hk, D, page, pages = 4, 2, 128, 16, 40
    g = gen(T)
    q = torch.randn(T, H, D, generator=g, device="cuda").half()
    q[used:] = math.nan
    kc, vc = (torch.randint(-5, 6, (pages, page, Hk, D), generator=g, device="cuda").to(torch.int8) for _ in "kv")
    if code == 2:
        kc, vc = (x.float().to(torch.float8_e4m3fn).view(torch.int8) for x in (kc, vc))
    ks, vs = (torch.full((pages, page, Hk), 0.01, device="cuda") for _ in "kv")
    table = torch.randperm(pages, generator=g, device="cuda").int()[None]
    cu, ctx = ints([0, used]), ints([600])
    for longest in (1, 640):
        out = torch.full((T, H, D), math.nan, dtype=torch.float16, device="cuda")
        n = _lib.lib().gptq_code_attention_workspace_size(1, T, H, Hk, D, longest)
        ws = torch.full((max(n, 1),), 0xFF, dtype=torch.uint8, device="cuda")
        _lib.call("gptq_code_attention", ptr(q), 1, *strides(q), code, ptr(kc), *kc.stride()[:3], ptr(vc), *vc.stride()[:3],
                  ptr(ks), *ks.stride(), ptr(vs), *vs.stride(), ptr(table), pages, pages, page, pages, ptr(ctx), ptr(cu), 1, T,
                  H, Hk, D, 0.1, longest, ptr(out), ptr(ws), n, torch.cuda.current_stream().cuda_stream)
        assert bool((out[used:] == 0).all()) and bool(torch.isfinite(out[:used]).all())
        if used:
            assert bool((out[:used] != 0).any(-1).all())


# ------------------------------------------------- more than 2^31 elements --

def test_norms_past_32_bits():
    """The rows of a long call are those of short ones, bit for bit, with gradients."""
    T, H, D = 66000, 256, 128
    g = gen(1)
    q = torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda").uniform_(-2, 2, generator=g)
    k = torch.randn(T, 1, D, generator=g, device="cuda").bfloat16()
    w, w2 = (torch.rand(D, generator=g, device="cuda") + 0.5 for _ in "qk")
    table, pos = A().rotary_table(D, 100), torch.arange(T, device="cuda", dtype=torch.int32) % 100
    qo, ko = A().norm_rotary(q, k, w, w2, table, pos)
    dq, dk, *_ = torch.ops.gptq.norm_rotary_backward(q.flip(0), k, q, k, w, w2, table, pos, False, 1e-6, False)
    for rows in (slice(0, 3), slice(65530, 65542), slice(T - 3, T)):
        one = [x[rows].contiguous() for x in (q, k)]
        want = A().norm_rotary(*one, w, w2, table, pos[rows])
        assert torch.equal(qo[rows], want[0]) and torch.equal(ko[rows], want[1])
        grad = q.flip(0)[rows].contiguous()
        back = torch.ops.gptq.norm_rotary_backward(grad, one[1], *one, w, w2, table, pos[rows], False, 1e-6, False)
        assert torch.equal(dq[rows], back[0]) and torch.equal(dk[rows], back[1])


@pytest.mark.parametrize("code", CODES)
def test_rows_past_32_bits(code):
    T, Hk, D, page, pages = 1_100_000, 16, 128, 16, 64
    g = gen(2)
    kc, vc = (torch.randint(-100, 100, (pages, page, Hk, D), generator=g, device="cuda").to(torch.int8) for _ in "kv")
    if code != torch.int8:
        kc, vc = (x.float().to(code) for x in (kc, vc))
    ks, vs = (torch.rand(pages, page, Hk, generator=g, device="cuda") for _ in "kv")
    width = T // page + 1
    table = torch.randint(0, pages, (1, width), generator=g, device="cuda", dtype=torch.int32)
    k, v = A().cached_rows(kc, vc, table, ints([T]), ints([0, T]), T, k_scale=ks, v_scale=vs)
    for rows in (torch.arange(5), torch.arange(2 ** 20 - 5, 2 ** 20 + 5), torch.arange(T - 5, T)):
        place = (table[0].long().cpu()[rows // page], rows % page)
        rows = rows.cuda()
        for got, c, s in ((k, kc, ks), (v, vc, vs)):
            place = tuple(x.cuda() for x in place)
            assert torch.equal(got[rows], (c.float()[place] * s[place][..., None]).bfloat16())


@pytest.mark.parametrize("code", CODES)
def test_attention_past_32_bits(code):
    """One token for each of very many sequences."""
    B, H, Hk, D, page, pages = 140_000, 128, 16, 128, 16, 64
    g = gen(3)
    rows = [random_rows(g, pages * page, Hk, D, code) for _ in "kv"]
    (kc, ks), (vc, vs) = ((c.view(pages, page, Hk, D), s.view(pages, page, Hk)) for c, s in rows)
    table = torch.randint(0, pages, (B, 2), generator=g, device="cuda", dtype=torch.int32)
    ctx = torch.randint(1, 33, (B,), generator=g, device="cuda", dtype=torch.int32)
    q = torch.empty(B, H, D, dtype=torch.float16, device="cuda").uniform_(-2, 2, generator=g)
    out = A().paged_attention(q, kc, vc, table, ctx, max_context=32, k_scale=ks, v_scale=vs)
    for b in (0, 1, 131071, 131072, B - 1):
        j = torch.arange(int(ctx[b]), device="cuda")
        place = (table[b].long()[j // page], j % page)
        check(out[b:b + 1], attended(q[b:b + 1], kc[place], ks[place], vc[place], vs[place]))
