"""Quantised caches against 64 bits (bounds of code_check.py): what is written,
what is read back, attention over it, and a layer that does all of it."""
import math

import pytest
import torch

from attention_check import check
from code_check import TOP, attended, normed, quantised, rounded, stored
from test_gpu_attention_guards import FAR, Room, ints, ptr, strides
from test_gpu_paged_attention import offsets, quantized

pytestmark = pytest.mark.gpu
CODES = [torch.int8, torch.float8_e4m3fn]
TYPES = [torch.bfloat16, torch.float16]


def A():
    from distributed_gptq_amd.models import attention
    return attention


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def empty_cache(pages, page, Hk, D, code, token_major=False):
    """Codes and scales, NaN wherever nothing is written (0x7F: e4m3's NaN)."""
    shape = (pages, page, Hk, D) if token_major else (pages, Hk, page, D)
    c = torch.full(shape, 127, dtype=torch.int8, device="cuda").view(code)
    s = torch.full(shape[:3], math.nan, device="cuda")
    return (c, s) if token_major else (c.transpose(1, 2), s.transpose(1, 2))


def random_rows(g, n, Hk, D, code):
    x = torch.randn(n, Hk, D, generator=g, device="cuda") * (0.2 + 2 * torch.rand(n, Hk, 1, generator=g, device="cuda"))
    return quantised(x, code)


def case(new, context, page, H, Hk, D, dtype, code, seed=0, token_major=False):
    """q, the caches, block table (any number past the contexts), each sequence's codes and scales."""
    g = gen(seed + sum(context) + D)
    counts = [-(-c // page) for c in context]
    pages = sum(counts) + 2
    kc, ks = empty_cache(pages, page, Hk, D, code, token_major)
    vc, vs = empty_cache(pages, page, Hk, D, code, token_major)
    order = torch.randperm(pages, generator=g, device="cuda")
    table = torch.full((len(new), max(counts + [1])), -1, dtype=torch.int32, device="cuda")
    table[:, 1::2] = FAR
    rows, at = [], 0
    for b, (c, n) in enumerate(zip(context, counts)):
        table[b, :n] = order[at:at + n].int()
        j = torch.arange(c, device="cuda")
        place = (table[b].long()[j // page], j % page)
        r = (*random_rows(g, c, Hk, D, code), *random_rows(g, c, Hk, D, code))
        for to, x in zip((kc.view(torch.int8), ks, vc.view(torch.int8), vs), r):
            to[place] = x.view(torch.int8) if x.dtype == code else x
        rows.append(r)
        at += n
    q = (torch.randn(sum(new), H, D, generator=g, device="cuda") * 2).to(dtype)
    return q, kc, vc, table, {"k_scale": ks, "v_scale": vs}, rows


def expect(q, rows, new, scale=None):
    parts, at = [], 0
    for n, r in zip(new, rows):
        parts.append(attended(q[at:at + n], *r, scale=scale))
        at += n
    return tuple(torch.cat(x) for x in zip(*parts))


# ----------------------------------------------------------------- writing --

@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES + [torch.float32])
@pytest.mark.parametrize("H,Hk,D,R,page,norm", [(4, 2, 64, 64, 16, True), (32, 8, 128, 128, 16, False), (3, 1, 80, 40, 7, True),
                                                (2, 2, 16, 8, 1, True), (5, 5, 48, 48, 24, False), (1, 1, 256, 128, 16, True),
                                                (2, 1, 128, 0, 32, True), (2, 1, 96, 0, 32, False)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(H, Hk, D, R, page, norm, interleaved, dtype, code):
    """Queries, and rows read back from their places; places that no token has
    stay as they are."""
    m, g = A(), gen(H + D)
    T, pages = 37, 64 // page + 40
    q, k, v = (torch.randn(T, n, D, generator=g, device="cuda").to(dtype) * 2 for n in (H, Hk, Hk))
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(torch.float32 if H % 2 else dtype) for _ in "qk")
    table = m.rotary_table(R, 100, base=500.0) if R else None
    pos = torch.randint(-2, 103, (T,), generator=g, device="cuda") if R else None
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T]
    slots[3], slots[11], slots[12] = -1, -7, pages * page
    kc, ks = empty_cache(pages, page, Hk, D, code, token_major=D == 48)
    vc, vs = empty_cache(pages, page, Hk, D, code, token_major=D == 48)
    weights = {"q_weight": wq, "k_weight": wk} if norm else {}
    before = [x.clone() for x in (kc.view(torch.int8), ks, vc.view(torch.int8), vs)]
    got = m.rotary_append(q, k, v, table, pos, kc, vc, slots, interleaved, k_scale=ks, v_scale=vs, **weights)
    w = (wq, wk) if norm else (None, None)
    check(got, rounded(*normed(q, w[0], table, pos, interleaved), dtype))
    kept = (slots >= 0) & (slots < pages * page)
    at = slots[kept] // page, slots[kept] % page
    y, e = normed(k, w[1], table, pos, interleaved)
    check(kc[at].double() * ks[at].double()[..., None], stored(y[kept], e[kept], code))
    check(ks[at], (y[kept].abs().amax(-1) / TOP[code],) + ((e[kept].amax(-1) + 2 ** -22 * y[kept].abs().amax(-1)) / TOP[code],))
    codes, scale = quantised(v[kept], code)   # not turned: the fp32 formula, bit for bit
    assert torch.equal(vc[at].view(torch.int8), codes.view(torch.int8)) and torch.equal(vs[at], scale)
    for x, old in zip((kc.view(torch.int8), ks, vc.view(torch.int8), vs), before):
        x, old = x.clone(), old.clone()
        x[at], old[at] = 0, 0
        assert torch.equal(x.nan_to_num(9.0) if x.is_floating_point() else x, old.nan_to_num(9.0) if x.is_floating_point() else old)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES + [torch.float32])
def test_rows_of_any_values(dtype, code):
    """Zeros, the smallest and largest values, ties, infinities and NaN."""
    m, D = A(), 32
    top = torch.finfo(dtype).max
    rows = torch.zeros(12, 1, D, dtype=torch.float64, device="cuda")
    rows[1, 0, 5] = 1.0
    rows[2, 0] = torch.linspace(-1, 1, D) * top
    rows[3, 0] = top
    rows[4, 0, ::2] = torch.finfo(dtype).tiny
    rows[5, 0] = torch.linspace(-127, 127, D).round() + 0.5   # halves between whole numbers
    rows[5, 0, 0] = 127
    rows[6, 0, 3], rows[6, 0, 4] = math.inf, 1.0
    rows[7, 0, 9] = -math.inf
    rows[8, 0, 31] = math.nan
    rows[9, 0] = torch.randn(D, generator=torch.Generator().manual_seed(0))
    rows[10, 0, 0] = 1e-40 if dtype == torch.bfloat16 else 0.0
    rows[11, 0, 1], rows[11, 0, 2] = 1.0, 1e-7
    x = rows.to(dtype)
    kc, ks = empty_cache(1, 12, 1, D, code)
    vc, vs = empty_cache(1, 12, 1, D, code)
    slots = torch.arange(12, device="cuda")
    m.rotary_append(x, x, x, None, None, kc, vc, slots, k_scale=ks, v_scale=vs)
    good = torch.tensor([0, 1, 2, 3, 4, 5, 9, 10, 11], device="cuda")
    codes, scale = quantised(x[good], code)
    for c, s in ((kc, ks), (vc, vs)):
        assert torch.equal(c[0, good].view(torch.int8), codes.view(torch.int8)) and torch.equal(s[0, good], scale)
        assert bool((c[0, 6:9].view(torch.int8) == 0).all()) and bool(s[0, 6:9].isnan().all())
        assert float(s[0, 0]) == 0.0 and float(s[0, 10]) == 0.0
    k, v = m.cached_rows(kc, vc, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), ints([12]), ints([0, 12]), 12, dtype,
                         k_scale=ks, v_scale=vs)
    assert bool(k[6:9].isnan().all()) and bool(torch.isfinite(k[good]).all()) and torch.equal(k[good], v[good])


@pytest.mark.parametrize("dtype", TYPES + [torch.float32])
def test_norms_into_a_cache_of_values(dtype):
    """The rows that norm_rotary gives, bit for bit, beside the values."""
    m, g = A(), gen(1)
    T, H, Hk, D, page, pages = 50, 8, 2, 128, 16, 6
    q, k, v = (torch.randn(T, n, D, generator=g, device="cuda").to(dtype) for n in (H, Hk, Hk))
    wq, wk = (1 + 0.3 * torch.randn(D, generator=g, device="cuda") for _ in "qk")
    table, pos = m.rotary_table(64, 100), torch.arange(T, device="cuda")
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T]
    kc, vc = (torch.full((pages, page, Hk, D), 9.0, dtype=dtype, device="cuda") for _ in "kv")
    got = m.rotary_append(q, k, v, table, pos, kc, vc, slots, q_weight=wq, k_weight=wk)
    want = m.norm_rotary(q, k, wq, wk, table, pos)
    at = slots // page, slots % page
    assert torch.equal(got, want[0]) and torch.equal(kc[at], want[1]) and torch.equal(vc[at], v)
    left = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    left[at] = False
    assert bool((kc[left] == 9).all()) and bool((vc[left] == 9).all())


# ---------------------------------------------------------------- reading --

@pytest.mark.parametrize("code", CODES + TYPES + [torch.float32])
@pytest.mark.parametrize("Hk,D,page", [(8, 128, 16), (1, 16, 7), (3, 80, 24), (2, 256, 1)])
def test_cached_rows(Hk, D, page, code):
    """Whole sequences, their last tokens, ones with more rows than tokens, none,
    and rows behind the last: the fp32 product rounded once, or a copy."""
    m = A()
    new, context = [5, 0, 40, 9, 33], [5, 30, 40, 4, 100]
    coded = code in CODES
    _, kc, vc, table, scales, rows = case(new, context, page, 1, Hk, D, torch.float16, code if coded else torch.int8)
    if not coded:
        kc, vc = (c.to(code) for c in (kc, vc))
        scales = {}
    cu = offsets(new)
    for dtype in (TYPES + [torch.float32] if coded else [code]):
        for T in (sum(new), sum(new) + 70):
            got = m.cached_rows(kc, vc, table.long(), ints(context), cu, T, dtype, **scales)
            for i, y in enumerate(got):
                assert y.shape == (T, Hk, D) and y.dtype == dtype and bool((y[sum(new):] == 0).all())
                at = 0
                for n, c, r in zip(new, context, rows):
                    x = r[2 * i].float() * (r[2 * i + 1][..., None] if coded else 1.0)
                    have = min(n, c)
                    assert torch.equal(y[at + n - have:at + n], x[c - have:c].to(dtype))
                    assert bool((y[at:at + n - have] == 0).all())
                    at += n
    assert m.cached_rows(kc, vc, table, ints(context), cu, 0, **scales)[0].shape == (0, Hk, D)


def test_cached_rows_refusals():
    m = A()
    _, kc, vc, table, s, _ = case([2, 2], [20, 30], 16, 1, 2, 64, torch.float16, torch.int8)
    ctx, cu = ints([20, 30]), offsets([2, 2])
    odd = torch.zeros(kc.numel() + 8, dtype=torch.int8, device="cuda")[8:].view(kc.shape)
    for args, kw in [((kc, vc, table, ctx, cu, 4), {}), ((kc, vc, table, ctx, cu[:2], 4), s), ((kc, vc, table[0], ctx, cu, 4), s),
                     ((kc, vc[:1], table, ctx, cu, 4), s), ((kc, vc, table, ctx, cu, -1), s),
                     ((kc, vc, table, ctx, cu, 4), {**s, "v_scale": s["v_scale"][:1]}),
                     ((kc, vc, table.cpu(), ctx, cu, 4), s), ((odd, vc, table, ctx, cu, 4), s),
                     ((kc[..., :40], vc[..., :40], table, ctx, cu, 4), s), ((kc.half(), vc.half(), table, ctx, cu, 4), s)]:
        with pytest.raises(ValueError):
            m.cached_rows(*args, **kw)
    for args, kw in [((kc, vc, table, ctx, cu, 4, torch.float64), s), ((kc, vc.half(), table, ctx, cu, 4), s),
                     ((kc, vc, table, ctx, cu, 4), {**s, "k_scale": s["k_scale"].half()}),
                     ((kc.half(), vc.half(), table, ctx, cu, 4, torch.bfloat16), {}), ((kc, vc, table.float(), ctx, cu, 4), s)]:
        with pytest.raises(TypeError):
            m.cached_rows(*args, **kw)


# -------------------------------------------------------------- attention --

@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (7, 1, 64), (4, 4, 80), (3, 3, 16), (40, 1, 48), (24, 2, 96), (2, 2, 112)])
@pytest.mark.parametrize("page,new,context", [
    (16, (1, 1, 1, 1, 1, 1), (1, 17, 32, 33, 300, 1024)),
    (7, (5, 1, 3, 0), (5, 64, 700, 9)),
    (64, (200, 33), (700, 33)),
    (24, (9, 130, 40), (4, 100, 40)),     # fewer cached than new: rows that see nothing
    (1, (2, 150), (0, 150)),
])
def test_attention(page, new, context, H, Hk, D, dtype, code):
    q, kc, vc, table, s, rows = case(new, context, page, H, Hk, D, dtype, code)
    cu = offsets(new) if set(new) != {1} else None
    want = expect(q, rows, new)
    for longest in (None, max(context), 1):
        got = A().paged_attention(q, kc, vc, table, ints(context), cu, max_context=longest, **s)
        assert got.dtype == dtype
        check(got, want)
    empty = want[1].amax((1, 2)) == 0
    assert bool((got[empty] == 0).all())


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,context", [((1,), (20000,)), ((1, 1, 1), (9000, 1, 30000)), ((70,), (9000,)), ((6, 6), (5000, 8191))])
def test_attention_of_long_contexts(new, context, dtype, code):
    """Contexts cut into parts, at a scale other than the default too."""
    q, kc, vc, table, s, rows = case(new, context, 32, 8, 2, 128, dtype, code)
    cu = offsets(new) if set(new) != {1} else None
    for scale in (None, 0.01):
        check(A().paged_attention(q, kc, vc, table, ints(context), cu, scale, **s), expect(q, rows, new, scale))


@pytest.mark.parametrize("code", CODES)
def test_layouts(code):
    """Token-major and head-major caches, fused and misaligned queries, 64-bit
    tables: the same bits.  A stride that vectors can not take is refused."""
    f, new, context = A().paged_attention, (1, 4, 90), (50, 300, 200)
    a = case(new, context, 16, 8, 2, 64, torch.bfloat16, code)
    b = case(new, context, 16, 8, 2, 64, torch.bfloat16, code, token_major=True)
    cu, ctx = offsets(new), ints(context)
    want = f(*a[:4], ctx, cu, **a[4])
    q = a[0]
    fused = torch.cat([q, q], 1)[:, 8:]
    odd = torch.zeros(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape).copy_(q)
    for qq, x, t in ((q, b, b[3]), (fused, a, a[3]), (odd, a, a[3].long()), (q.transpose(0, 1).contiguous().transpose(0, 1), b, b[3])):
        assert torch.equal(f(qq, x[1], x[2], t, ctx.long(), cu.long(), **x[4]), want)
    wide = torch.zeros(*a[1].shape[:3], 72, dtype=torch.int8, device="cuda").view(code)
    with pytest.raises(ValueError, match="aligned"):
        f(q, wide[..., :64], a[2], a[3], ctx, cu, **a[4])


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [100, 6])
def test_scales_that_are_not_finite_reach_the_rows_that_see_them(new, dtype, code):
    q, kc, vc, table, s, rows = case((new, 3), (170, 40), 16, 4, 2, 128, dtype, code)
    cu, ctx = offsets((new, 3)), ints((170, 40))
    want = expect(q, rows, (new, 3))
    for which in ("k_scale", "v_scale"):
        for key in (0, 31, 165, 169, 170 - new // 2):
            x = s[which].clone()
            x[table[0].long()[key // 16], key % 16, 1] = math.nan
            got = A().paged_attention(q, kc, vc, table, ctx, cu, **{**s, which: x})
            sees = torch.arange(170 - new, 170, device="cuda") >= key
            sees = torch.cat([sees, torch.zeros(3, dtype=torch.bool, device="cuda")])
            assert bool(got[sees][:, 2:].isnan().all())
            clean = got.clone()
            clean[sees, 2:] = 0
            ref = [t.clone() for t in want]
            for t in ref:
                t[sees, 2:] = 0
            check(clean, tuple(ref))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 5, 140])
def test_values_of_any_size(new, dtype, code):
    """Scales that differ by many orders, zero rows among them, and bf16's largest
    and smallest values: weighted means stay finite and near."""
    q, kc, vc, table, s, rows = case((new,), (400,), 16, 4, 2, 64, dtype, code)
    g = gen(5)
    for low, high in ((-20, 10), (90, 119), (-119, -90)) if dtype == torch.bfloat16 else ((-20, 10), (-12, 0)):
        f = torch.exp2(torch.randint(low, high, (400, 2), generator=g, device="cuda").float())
        f[::7] = 0.0
        vs = rows[0][3] / rows[0][3].amax() * f
        j = torch.arange(400, device="cuda")
        x = s["v_scale"].clone()
        x[table[0].long()[j // 16], j % 16] = vs
        got = A().paged_attention(q, kc, vc, table, ints([400]), offsets([new]), k_scale=s["k_scale"], v_scale=x)
        y, b = attended(q, *rows[0][:3], vs)
        # results below the type's normal range are off by half its smallest step
        b = b + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)
        check(got, (y, b))


def test_graph():
    """Append and attention captured together: replays follow the places and
    lengths, the program's own eager calls between them."""
    m, g = A(), gen(3)
    B, H, Hk, D, page, pages = 5, 8, 2, 128, 16, 64
    x = torch.randn(B, H + 2 * Hk, D, generator=g, device="cuda").half()
    caches = [empty_cache(pages, page, Hk, D, torch.int8) for _ in "kv"]
    (kc, ks), (vc, vs) = caches
    kc.copy_(torch.randint(-127, 128, kc.shape, generator=g, device="cuda"))
    vc.copy_(torch.randint(-127, 128, vc.shape, generator=g, device="cuda"))
    ks.copy_(torch.rand(ks.shape, generator=g, device="cuda") * 0.02)
    vs.copy_(torch.rand(vs.shape, generator=g, device="cuda") * 0.02)
    w = torch.rand(D, generator=g, device="cuda") + 0.5
    table = torch.randperm(pages, generator=g, device="cuda")[:60].view(B, 12).int()
    ctx = ints([1, 30, 64, 100, 150])
    rot = m.rotary_table(D, 256)

    def places():
        at = (ctx - 1).long()
        return (table.gather(1, (at // page)[:, None])[:, 0] * page + at % page).int(), at.int()
    slots, pos = places()

    def step():
        q = m.rotary_append(x[:, :H], x[:, H:H + Hk], x[:, H + Hk:], rot, pos, kc, vc, slots, k_scale=ks, v_scale=vs,
                            q_weight=w, k_weight=w)
        rows = m.cached_rows(kc, vc, table, ctx, ints_cu, B, torch.float16, k_scale=ks, v_scale=vs)
        return (m.paged_attention(q, kc, vc, table, ctx, k_scale=ks, v_scale=vs, max_context=12 * page), *rows)
    ints_cu = offsets([1] * B)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for r in range(5):
        ctx.add_(7 * r % 11)
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        for buf, val in zip((slots, pos), places()):
            buf.copy_(val)
        for y in out:
            y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        kept = [y.clone() for y in out]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b), r


def test_two_streams():
    """Calls on two streams at once, each with a workspace of its own."""
    f = A().paged_attention
    cases = [case((1, 1), (9000, 5000), 16, 8, 2, 128, torch.bfloat16, c, seed=i) for i, c in enumerate(CODES)]
    ctx = ints([9000, 5000])
    want = [f(*x[:4], ctx, **x[4]) for x in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(4):
        for i, (st, x) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(st):
                got[i].append(f(*x[:4], ctx, **x[4]))
    torch.cuda.synchronize()
    for w, ys in zip(want, got):
        for y in ys:
            assert torch.equal(w, y)


# ------------------------------------------------------------------ guards --

@pytest.mark.parametrize("code", [0, 1, 2])
@pytest.mark.parametrize("H,Hk,D,page", [(8, 2, 128, 16), (7, 1, 48, 7), (4, 4, 64, 32)])
def test_nothing_outside_is_touched(H, Hk, D, page, code):
    """Lengths, offsets, pages and slots of any kind through the C entry points:
    no byte around the tensors changes."""
    from distributed_gptq_amd import _lib
    dt = [torch.float16, torch.int8, torch.float8_e4m3fn][code]
    pages, width, T = 9, 70, 300
    g = gen(D)
    odd = [0, 3, pages, -1, FAR, -FAR - 1, pages - 1]
    stream = torch.cuda.current_stream().cuda_stream
    for new, context, longest in (([0, 1, 300], [1, 600], 1), ([0, 40, 300], [FAR, -FAR], 5000), ([9, -1, 200], [0, 5], 5000),
                                  ([0, 300, FAR], [1100, 1100], 5000), ([0, 2, 5], [1100, 77], 1)):
        room = Room()
        q = room.input(torch.randn(T, H, D, generator=g, device="cuda").half())
        k, v = (room.input(torch.randn(T, Hk, D, generator=g, device="cuda").half()) for _ in "kv")
        kc, vc = (room.empty(pages, page, Hk, D, dtype=torch.float16 if code == 0 else torch.int8) for _ in "kv")
        ks, vs = (room.empty(pages, page, Hk, dtype=torch.float32).fill_(0.01) for _ in "kv")
        kc.zero_(), vc.zero_()
        table = room.input(ints([[odd[(b + i) % 7] for i in range(width)] for b in range(2)]))
        cu, ctx = room.input(ints(new)), room.input(ints(context))
        # (every place at most once, beside places that are none)
        slots = room.input(ints([(i if i < pages * page else [-1, -FAR - 1, FAR, pages * page][i % 4]) for i in range(T)]))
        w = room.input(torch.rand(D, generator=g, device="cuda"))
        rot, pos = room.input(torch.rand(5, 2, D // 2, generator=g, device="cuda")), room.input(ints([odd[i % 7] for i in range(T)]))
        out, ko, vo = (room.empty(T, n, D, dtype=torch.float16).zero_() for n in (H, Hk, Hk))
        cs = (*kc.stride()[:3],)
        ss = ks.stride()
        _lib.call("gptq_norm_rotary_append", ptr(q), ptr(k), ptr(v), 1, *strides(q), *strides(k), *strides(v), ptr(w), ptr(w), 0,
                  1e-6, ptr(rot), 5, D, ptr(pos), 0, ptr(slots), page, pages, T, H, Hk, D, ptr(out), code, ptr(kc), *cs, ptr(vc),
                  *cs, ptr(ks), *ss, ptr(vs), *ss, stream)
        _lib.call("gptq_cached_rows", code, ptr(kc), *cs, ptr(vc), *cs, ptr(ks), *ss, ptr(vs), *ss, ptr(table), width, width,
                  page, pages, ptr(ctx), ptr(cu), 2, T, Hk, D, ptr(ko), ptr(vo), 1, stream)
        if code:
            n = _lib.lib().gptq_code_attention_workspace_size(2, T, H, Hk, D, longest)
            ws = room.empty(max(n, 1), dtype=torch.uint8).zero_()
            _lib.call("gptq_code_attention", ptr(q), 1, *strides(q), code, ptr(kc), *cs, ptr(vc), *cs, ptr(ks), *ss, ptr(vs), *ss,
                      ptr(table), width, width, page, pages, ptr(ctx), ptr(cu), 2, T, H, Hk, D, 0.1, longest, ptr(out),
                      ptr(ws), n, stream)
        room.check()


def test_norm_and_gradient_touch_nothing_outside():
    from distributed_gptq_amd import _lib
    g = gen(2)
    for T, H, Hk, D, R in ((1, 1, 1, 8, 4), (33, 5, 2, 40, 40), (300, 8, 2, 128, 64), (7, 3, 1, 256, 256)):
        room = Room()
        q, k, gq, gk = (room.input(torch.randn(T, n, D, generator=g, device="cuda").bfloat16()) for n in (H, Hk, H, Hk))
        w = room.input(torch.rand(D, generator=g, device="cuda").half())
        rot, pos = room.input(torch.rand(5, 2, R // 2, generator=g, device="cuda")), room.input(ints([FAR, -5, 2, 4, -FAR - 1] * T)[:T])
        qo, dq = (room.empty(T, H, D, dtype=torch.bfloat16) for _ in "ab")
        ko, dk = (room.empty(T, Hk, D, dtype=torch.bfloat16) for _ in "ab")
        dwq, dwk = (room.empty(D, dtype=torch.float16) for _ in "ab")
        n = _lib.lib().gptq_norm_rotary_backward_workspace_size(T, H, Hk, D)
        ws = room.empty(n, dtype=torch.uint8)
        stream = torch.cuda.current_stream().cuda_stream
        _lib.call("gptq_norm_rotary", ptr(q), ptr(k), 2, *strides(q), *strides(k), ptr(w), ptr(w), 1, 1e-6, ptr(rot), 5, R,
                  ptr(pos), 0, T, H, Hk, D, ptr(qo), ptr(ko), stream)
        _lib.call("gptq_norm_rotary_backward", ptr(gq), ptr(gk), ptr(q), ptr(k), 2, *strides(gq), *strides(gk), *strides(q),
                  *strides(k), ptr(w), ptr(w), 1, 1e-6, ptr(rot), 5, R, ptr(pos), 1, T, H, Hk, D, ptr(dq), ptr(dk), ptr(dwq),
                  ptr(dwk), ptr(ws), n, stream)
        room.check()


# ---------------------------------------------------------------- refusals --

@pytest.mark.parametrize("code", CODES)
def test_attention_refusals(code):
    f = A().paged_attention
    q, kc, vc, table, s, _ = case((1, 1), (20, 30), 16, 4, 2, 64, torch.float16, code)
    ctx = ints([20, 30])
    for args, kw in [((q[:1], kc, vc, table, ctx), s), ((q, kc[0], vc[0], table, ctx), s), ((q, kc, vc[:1], table, ctx), s),
                     ((q, kc, vc, table[0], ctx), s), ((q, kc, vc, table, ctx[:1]), s), ((q, kc, vc, table, ctx), {}),
                     ((q, kc[..., :32], vc[..., :32], table, ctx), s), ((q, kc, vc, table, ctx, offsets((1,))), s),
                     ((q, kc, vc, table, ctx), {**s, "k_scale": s["k_scale"][:, :8]}), ((q.cpu(), kc, vc, table, ctx), s),
                     ((q[..., :40], kc[..., :40], vc[..., :40], table, ctx), s)]:
        with pytest.raises((ValueError, RuntimeError)):
            f(*args, **kw)
    other = CODES[1 - CODES.index(code)]
    for args, kw in [((q.float(), kc, vc, table, ctx), s), ((q, kc, vc.view(other), table, ctx), s),
                     ((q, kc, vc, table.float(), ctx), s), ((q, kc, vc, table, ctx), {**s, "v_scale": s["v_scale"].double()})]:
        with pytest.raises(TypeError):
            f(*args, **kw)
    with pytest.raises(RuntimeError, match="gradient"):
        f(q.clone().requires_grad_(True), kc, vc, table, ctx, **s)


@pytest.mark.parametrize("code", CODES)
def test_append_refusals(code):
    f = A().rotary_append
    q, k = torch.zeros(3, 4, 64, device="cuda").half(), torch.zeros(3, 2, 64, device="cuda").half()
    kc, ks = empty_cache(4, 16, 2, 64, code)
    s, slots, w = {"k_scale": ks, "v_scale": ks.clone()}, torch.arange(3, device="cuda"), torch.ones(64, device="cuda")
    c = (kc, kc.clone())
    table, pos = A().rotary_table(60, 8), slots
    for args, kw in [((q, k, k, None, None, *c, slots), {}), ((q, k, k, None, None, *c, slots), {"k_scale": ks}),
                     ((q, k, k, None, None, *c, slots[:2]), s), ((q, k[:2], k, None, None, *c, slots), s),
                     ((q, k[:, :1], k[:, :1], None, None, *c, slots), s), ((q, k, k, None, None, *c, slots), {**s, "q_weight": w}),
                     ((q, k, k, None, None, *c, slots), {**s, "q_weight": w[:32], "k_weight": w[:32]}),
                     ((q, k, k, table, pos, *c, slots), s), ((q, k, k, table, None, *c, slots), s),
                     ((q, k, k, None, None, *c, slots), {**s, "q_weight": w, "k_weight": w, "eps": 0.0}),
                     ((q, k, k, None, None, c[0].half(), c[1].half(), slots), s),
                     ((q, k, k, None, None, c[0][:0], c[1][:0], slots), {n: x[:0] for n, x in s.items()})]:
        with pytest.raises(ValueError):
            f(*args, **kw)
    for args, kw in [((q, k, k, None, None, c[0], c[1].half(), slots), s),
                     ((q, k, k, None, None, *c, slots), {**s, "k_scale": ks.half()}),
                     ((q, k, k, None, None, *c, slots.float()), s),
                     ((q, k, k, None, None, *c, slots), {**s, "q_weight": w, "k_weight": w.half()}),
                     ((q, k, k, None, None, c[0].float(), c[1].float(), slots), {"q_weight": w, "k_weight": w})]:
        with pytest.raises(TypeError):
            f(*args, **kw)
    before = kc.view(torch.int8).clone()
    assert f(q[:0], k[:0], k[:0], None, None, *c, slots[:0], **s).shape == (0, 4, 64) and torch.equal(before, kc.view(torch.int8))


# ------------------------------------------------------------------- layer --

@pytest.mark.parametrize("dtype", CODES + [torch.bfloat16])
@pytest.mark.parametrize("rotary", [True, False])
def test_layer_with_norms(rotary, dtype):
    """A layer of normed heads: its prompt whole, then in steps over a cache (of
    codes, too), which give what the functions give one by one, and the whole
    prompt's rows up to the rounding and the codes; gradients reach the norms."""
    from distributed_gptq_amd.models import FusedQuantizedLinear, PagedKVCache, QuantizedAttention
    m, g = A(), gen(0)
    hidden, H, Hk, D = 256, 4, 2, 64
    wq, wk = (1 + 0.3 * torch.randn(D, generator=g, device="cuda") for _ in "qk")
    layer = QuantizedAttention(FusedQuantizedLinear([quantized(n, hidden, g) for n in (H * D, Hk * D, Hk * D)]),
                               quantized(hidden, H * D, g), H, Hk, D, m.rotary_table(D, 512) if rotary else None,
                               q_norm=wq, k_norm=wk).cuda()
    x = torch.randn(103, hidden, generator=g, device="cuda").bfloat16()
    cu = offsets([70, 33])
    with torch.no_grad():
        whole = layer(x, cu)
    cache = PagedKVCache(16, 16, Hk, D, layers=2, dtype=dtype)
    for c in (cache.k, cache.v):
        c.view(torch.int8).fill_(127) if dtype in CODES else c.fill_(math.nan)
    for c in (cache.k_scale, cache.v_scale):
        if c is not None:
            c.fill_(math.nan)
    other = [t.clone() for t in (cache.k, cache.v)]
    scales = [t.clone() for t in (cache.k_scale, cache.v_scale)] if dtype in CODES else []
    names = dict(zip(("k_scale", "v_scale"), (t[1] for t in scales)))
    seqs, done, rows = [x[:70], x[70:]], [0, 0], [[], []]
    for new in ([50, 1], [1, 30], [1, 1], [18, 1]):
        who = [i for i in (0, 1) if new[i]]
        batch = cache.extend([f"s{i}" for i in who], [new[i] for i in who])
        part = torch.cat([seqs[i][done[i]:done[i] + new[i]] for i in who])
        y = layer.step(part, cache, batch, layer=1)
        with torch.no_grad():
            q, k, v = layer._heads(part)
            q = m.rotary_append(q, k, v, layer.table, batch.positions, other[0][1], other[1][1], batch.slots, q_weight=wq,
                                k_weight=wk, **names)
            z = m.paged_attention(q, other[0][1], other[1][1], batch.block_table, batch.context_lens, batch.cu_seqlens,
                                  max_context=batch.max_context, **names)
            assert torch.equal(y, layer.o(z.flatten(-2)))
        for i, r in zip(who, y.split([new[i] for i in who])):
            rows[i].append(r)
            done[i] += new[i]
    assert done == [70, 33]
    got = torch.cat(rows[0] + rows[1]).float()
    # roundings as for a cache of values (6 of 2^-8), and a code's: 1/254 of a head's
    # largest value for whole numbers, at most 4 times the root mean square of its
    # values here, or 2^-4 of each value for e4m3, of the keys and of the values both
    code = {torch.int8: 2 * 4 / 254, torch.float8_e4m3fn: 2 * 2 ** -4, torch.bfloat16: 0.0}[dtype]
    assert (got - whole.float()).norm() <= (6 * 2 ** -8 + code) * whole.float().norm()
    k, v, at = cache.rows(["s1", "s0"], layer=1)
    assert at.tolist() == [0, 33, 103] and k.shape == v.shape == (103, Hk, D) and k.dtype == torch.bfloat16
    with torch.no_grad():
        q0, k0, v0 = layer._heads(x)
        pos = m.packed_positions(cu, 103)
        want = normed(k0, wk, layer.table, pos if rotary else None)
    order = torch.cat([torch.arange(70, 103), torch.arange(70)]).cuda()
    if dtype in CODES:
        for r, (y, b) in ((k, stored(want[0][order], want[1][order] + 2.0 ** -7 * k0.abs().amax(), dtype)),
                          (v, stored(v0[order].double(), torch.full_like(v0, 2.0 ** -7 * float(v0.abs().amax())).double(), dtype))):
            # (projections of other row counts differ in their last bits, here 2^-7 of the largest)
            check(r, (y, b + 2.0 ** -8 * y.abs()))
    xg = x.clone().requires_grad_(True)
    layer(xg, cu).float().pow(2).sum().backward()
    for t in (xg.grad, layer.q_norm.grad, layer.k_norm.grad):
        assert bool(torch.isfinite(t).all()) and float(t.abs().max()) > 0
