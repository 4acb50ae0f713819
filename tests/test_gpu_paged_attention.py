"""Attention of new tokens over a paged cache against 64 bits (bounds of
attention_check.py), the cache's update, and a quantized layer's attention
that runs a prompt whole and token by token."""
import math

import pytest
import torch

from attention_check import check, one

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def A():
    from distributed_gptq_amd.models import attention
    return attention


def case(new, context, page, H, Hk, D, dtype, seed=0, garbage=math.nan):
    """q, the caches (every place outside the contexts holds ``garbage``), block
    table (-1 past the contexts) and each sequence's own keys and values."""
    g = torch.Generator(device="cuda").manual_seed(seed + sum(context) + D)
    counts = [-(-c // page) for c in context]
    pages = sum(counts) + 2
    kc = torch.full((pages, page, Hk, D), garbage, device="cuda", dtype=dtype)
    vc = kc.clone()
    order = torch.randperm(pages, generator=g, device="cuda")
    table = torch.full((len(new), max(counts + [1])), -1, dtype=torch.int32, device="cuda")
    rows, at = [], 0
    for b, (c, n) in enumerate(zip(context, counts)):
        table[b, :n] = order[at:at + n].int()
        j = torch.arange(c, device="cuda")
        place = (table[b].long()[j // page], j % page)
        k = torch.randn(c, Hk, D, generator=g, device="cuda").to(dtype)
        v = torch.randn(c, Hk, D, generator=g, device="cuda").to(dtype)
        kc[place], vc[place] = k, v
        rows.append((k, v))
        at += n
    q = (torch.randn(sum(new), H, D, generator=g, device="cuda") * 2).to(dtype)
    return q, kc, vc, table, rows


def offsets(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def expect(q, rows, new):
    parts, at = [], 0
    for n, (k, v) in zip(new, rows):
        parts.append(one(q[at:at + n], k, v)["out"])
        at += n
    return tuple(torch.cat(x) for x in zip(*parts))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 128), (4, 4, 64), (7, 1, 40), (24, 2, 96), (40, 1, 64)])
@pytest.mark.parametrize("new,context,page", [
    ((1,), (1,), 16), ((1, 1, 1, 1), (5, 64, 65, 700), 16), ((1, 1), (3000, 0), 24), ((1,), (2500,), 1),
    ((3, 1, 40), (3, 900, 77), 32), ((200,), (513,), 16), ((130, 2), (130, 1200), 128), ((5, 0, 2), (2, 10, 2), 7)])
def test_paged(H, Hk, D, new, context, page, dtype):
    """Contexts of zero and one, pages that end inside a tile, chunks, chunks
    longer than the context (their first tokens see nothing and give zeros)."""
    q, kc, vc, table, rows = case(new, context, page, H, Hk, D, dtype)
    ctx = torch.tensor(context, dtype=torch.int32, device="cuda")
    want = expect(q, rows, new)
    cu = None if set(new) == {1} else offsets(new)
    for longest in (None, max(context), 1, 1 << 20):
        check(A().paged_attention(q, kc, vc, table, ctx, cu, max_context=longest), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_context(dtype):
    """A long context in one sequence and short ones beside it: many splits."""
    new, context = (1, 1, 1), (20011, 3, 515)
    q, kc, vc, table, rows = case(new, context, 16, 8, 2, 128, dtype)
    check(A().paged_attention(q, kc, vc, table, torch.tensor(context, device="cuda")), expect(q, rows, new))


@pytest.mark.parametrize("context", [100, 700, 2500])
@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_values_that_a_row_sees(context, dtype):
    """An infinite value of a key gives that channel its infinity, in however
    many parts the keys are taken; the other channels are as without it."""
    q, kc, vc, table, rows = case((1,), (context,), 16, 8, 2, 128, dtype)
    want = expect(q, rows, (1,))
    for key in (3, context - 1):
        for bad in (math.inf, -math.inf):
            v2 = vc.clone()
            v2[int(table[0, key // 16]), key % 16, 0, 5] = bad
            out = A().paged_attention(q, kc, v2, table, torch.tensor([context], device="cuda"))
            assert bool((out[:, :4, 5] == bad).all())
            out[:, :4, 5] = 0
            ref = want[0].clone()
            ref[:, :4, 5] = 0
            check(out, (ref, want[1]))


def test_strided_cache_and_same_bits():
    """A cache with heads before tokens, and one that is a part of a larger
    tensor, give the same bits as a contiguous one; so do two calls."""
    new, context = (1, 1), (333, 40)
    q, kc, vc, table, rows = case(new, context, 16, 8, 2, 64, torch.float16)
    ctx = torch.tensor(context, device="cuda")
    want = A().paged_attention(q, kc, vc, table, ctx)
    assert torch.equal(want, A().paged_attention(q, kc, vc, table, ctx))

    def heads_first(x):
        return x.transpose(1, 2).contiguous().transpose(1, 2)

    def part(x):
        return torch.stack([x, x], 3)[:, :, :, 1]
    for f in (heads_first, part):
        assert torch.equal(want, A().paged_attention(q, f(kc), f(vc), table, ctx))


def test_cache_past_32_bits():
    """Pages more than 4 GiB from the cache's start."""
    page, Hk, D, dtype = 64, 8, 128, torch.bfloat16
    pages = (5 << 30) // (page * Hk * D * 2)
    kc = torch.empty(pages, page, Hk, D, device="cuda", dtype=dtype)
    vc = torch.empty_like(kc)
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = [pages - 1, 0, pages - 5]
    for p in ids:
        kc[p], vc[p] = torch.randn(2, page, Hk, D, generator=g, device="cuda").to(dtype)
    q = torch.randn(1, 8, D, generator=g, device="cuda").to(dtype)
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    k, v = (torch.cat([c[p] for p in ids])[:150] for c in (kc, vc))
    out = A().paged_attention(q, kc, vc, table, torch.tensor([150], device="cuda"))
    check(out, one(q, k, v)["out"])
    new = torch.randn(3, 1, Hk, D, generator=g, device="cuda").to(dtype)
    slot = torch.tensor([pages * page - 3], device="cuda")
    A().rotary_append(new[0], new[1], new[2], None, None, kc, vc, slot)
    assert torch.equal(kc[pages - 1, page - 3], new[1, 0]) and torch.equal(vc[pages - 1, page - 3], new[2, 0])


@pytest.mark.parametrize("dtype", TYPES)
def test_not_finite_later_in_a_chunk(dtype):
    """An infinity or NaN in a later token's value leaves the chunk's earlier
    tokens as they are, in both kernels and with splits."""
    for new in (6, 100):
        q, kc, vc, table, rows = case((new,), (900,), 16, 8, 2, 128, dtype)
        k, v = rows[0]
        want = one(q, k, v)["out"]
        for place in (899, 895):
            j = 900 - new - 1
            vc2 = vc.clone()
            vc2[table[0, place // 16].long(), place % 16, 1] = math.inf
            out = A().paged_attention(q, kc, vc2, table, torch.tensor([900], device="cuda"), offsets((new,)))
            n = place - j - 1
            check(out[:n], tuple(x[:n] for x in want))
            check(out[:, :4], tuple(x[:, :4] for x in want))
            assert not torch.isfinite(out[n:, 4:]).any()


def test_what_the_device_arrays_may_hold():
    """Page numbers outside the cache and contexts outside the table are
    clamped; the other sequences are as they were."""
    new, context = (1, 1), (100, 60)
    q, kc, vc, table, rows = case(new, context, 16, 4, 2, 64, torch.float16, garbage=0.0)
    want = expect(q, rows, new)
    t2 = table.clone()
    t2[0, :3] = torch.tensor([-7, 2 ** 31 - 1, kc.shape[0]], dtype=torch.int32)
    for ctx in ((100, 60), (2 ** 31 - 1, 60), (-5, 60)):
        out = A().paged_attention(q, kc, vc, t2, torch.tensor(ctx, dtype=torch.int32, device="cuda"), max_context=100)
        check(out[1:], tuple(x[1:] for x in want))
    assert not out[0].any()  # a context of -5 is empty


def test_graph():
    """The cache's update and the attention captured together: replays follow
    the lengths, tables and inputs in their buffers, several times over, with
    other work between."""
    H, Hk, D, page = 8, 2, 128, 16
    m = A()
    table = m.rotary_table(D, 4096)
    q, kc, vc, bt, rows = case((1, 1), (1000, 600), page, H, Hk, D, torch.bfloat16, garbage=0.0)
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(2, H + 2 * Hk, D, generator=g, device="cuda").bfloat16()
    ctx = torch.tensor([500, 300], dtype=torch.int32, device="cuda")
    b = torch.arange(2, device="cuda")

    def places():
        at = (ctx - 1).long()
        return (bt[b, at // page] * page + at % page).int(), (ctx - 1).int()

    def step(x, slots, pos):
        qr = m.rotary_append(x[:, :H], x[:, H:H + Hk], x[:, H + Hk:], table, pos, kc, vc, slots)
        return m.paged_attention(qr, kc, vc, bt, ctx, max_context=1000)
    slots, pos = places()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(x, slots, pos)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            y = step(x, slots, pos)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for r in range(5):
        ctx.add_(7 * r)
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        for buf, val in zip((slots, pos), places()):
            buf.copy_(val)
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        kept = y.clone()
        assert torch.equal(kept, step(x, slots, pos)), r


def quantized(N, K, g):
    from distributed_gptq_amd.models import QuantizedLinear
    q = QuantizedLinear(4, 64, K, N, bias=False, packed=True).cuda()
    q.pack_weights(torch.randint(0, 16, (N, K), generator=g, device="cuda", dtype=torch.uint8),
                   torch.rand(N, K // 64, generator=g, device="cuda") * 0.01 + 0.005,
                   torch.full((N, K // 64), 8.0, device="cuda"))
    return q


@pytest.mark.parametrize("rotary", [True, False])
def test_quantized_attention_prompt_and_steps(rotary):
    """A layer's prompt in one pass, in chunks over the cache, and its last
    tokens one by one: the same rows up to the rounding of the projections'
    kernels; the gradient reaches the input."""
    from distributed_gptq_amd.models import FusedQuantizedLinear, PagedKVCache, QuantizedAttention
    m = A()
    hidden, H, Hk, D = 256, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    layer = QuantizedAttention(FusedQuantizedLinear([quantized(n, hidden, g) for n in (H * D, Hk * D, Hk * D)]),
                               quantized(hidden, H * D, g), H, Hk, D, m.rotary_table(D, 512) if rotary else None)
    lens = [70, 33]
    x = torch.randn(sum(lens), hidden, generator=g, device="cuda").bfloat16()
    cu = offsets(lens)
    with torch.no_grad():
        whole = layer(x, cu)
    cache = PagedKVCache(16, 16, Hk, D, layers=2, dtype=x.dtype)
    cache.k.fill_(math.nan), cache.v.fill_(math.nan)
    seqs = [x[:70], x[70:]]
    done = [0, 0]
    rows = [[], []]
    for new in ([50, 1], [1, 30], [1, 1], [1, 1], [17, 0]):
        who = [i for i in (0, 1) if new[i]]
        batch = cache.extend([f"s{i}" for i in who], [new[i] for i in who])
        y = layer.step(torch.cat([seqs[i][done[i]:done[i] + new[i]] for i in who]), cache, batch, layer=1)
        for i, part in zip(who, y.split([new[i] for i in who])):
            rows[i].append(part)
            done[i] += new[i]
    got = torch.cat(rows[0] + rows[1])
    assert cache.length("s0") == 70 and cache.length("s1") == 33
    # a rounding of bf16 in each of the projections, the rotation, the attention
    # and the output: 6 of 2^-8, which a product of K = 256 terms carries as the
    # root of their squares, at most 8 times over all rows
    assert (got.float() - whole.float()).norm() <= 6 * 2 ** -8 * whole.float().norm()
    assert (got.float() - whole.float()).abs().max() <= 8 * 6 * 2 ** -8 * whole.float().pow(2).mean().sqrt()
    xg = x.clone().requires_grad_(True)
    layer(xg, cu).float().pow(2).sum().backward()
    assert bool(torch.isfinite(xg.grad).all()) and float(xg.grad.abs().max()) > 0
    cache.free("s0")
    assert cache.free_pages == 16 - 3 and "s0" not in cache


def test_refusals():
    f = A().paged_attention
    q, kc, vc, table, _ = case((1, 1), (20, 30), 16, 4, 2, 64, torch.float16)
    ctx = torch.tensor((20, 30), dtype=torch.int32, device="cuda")
    for args in [(q[:1], kc, vc, table, ctx), (q, kc[0], vc[0], table, ctx), (q, kc, vc[:1], table, ctx),
                 (q, kc, vc, table[0], ctx), (q, kc, vc, table, ctx[:1]), (q, kc[..., :32], vc[..., :32], table, ctx),
                 (q, kc, vc, table, ctx, offsets((1,))),
                 (q, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, table, ctx)]:
        with pytest.raises(ValueError):
            f(*args)
    with pytest.raises(TypeError):
        f(q, kc.bfloat16(), vc.bfloat16(), table, ctx)
    with pytest.raises(TypeError):
        f(q, kc, vc, table.float(), ctx)
    with pytest.raises(RuntimeError, match="gradient"):
        f(q.clone().requires_grad_(True), kc, vc, table, ctx)
