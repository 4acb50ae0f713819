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


def microseconds(f):
    f()
    times = []
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        f()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return sorted(times)[2]


def step(L, H, Hk, D, dtype):
    g = torch.Generator(device="cuda").manual_seed(5)
    return [torch.randn(L, h, D, generator=g, device="cuda").to(dtype) for h in (H, Hk, Hk, H)]


def train(q, k, v, grad):
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    return torch.autograd.grad(A().attention(q, k, v), (q, k, v), grad)


def nan(x):
    return torch.full_like(x, math.nan)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_step_of_nan_takes_no_longer(dtype):
    """All NaN, as after an overflow: within 10 times the time of a finite step
    (making every row again, one by one, took 200 to 500 times)."""
    q, k, v, grad = step(2048, 16, 8, 128, dtype)
    usual = microseconds(lambda: train(q, k, v, grad))
    for x in ((nan(q), k, v, grad), (q, nan(k), v, grad), (nan(q), nan(k), nan(v), nan(grad)), (q, k, v, nan(grad))):
        assert microseconds(lambda: train(*x)) <= 10 * usual
        assert all(bool(y.isnan().all()) for y in train(*x)[:2])
    with torch.no_grad():
        usual = microseconds(lambda: A().attention(q, k, v))
        assert microseconds(lambda: A().attention(nan(q), k, v)) <= 10 * usual
        kc, vc = (x.view(128, 16, 8, 128) for x in (k, v))
        args = (kc, vc, torch.arange(128, device="cuda", dtype=torch.int32)[None], torch.tensor([2048], device="cuda"))
        usual = microseconds(lambda: A().paged_attention(q[:1], *args))
        assert microseconds(lambda: A().paged_attention(nan(q[:1]), *args)) <= 10 * usual
        assert bool(A().paged_attention(nan(q[:1]), *args).isnan().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinite_values_take_bounded_time(dtype):
    """Sums with an infinity are made again row by row: within 60 times the time
    of a finite step (one row or key after the other took 500 times)."""
    q, k, v, grad = step(2048, 16, 8, 128, dtype)
    usual = microseconds(lambda: train(q, k, v, grad))
    for i in (2, 3):
        x = [q, k, v, grad]
        x[i] = x[i].clone()
        x[i][0 if i == 2 else 2047, :, 3] = math.inf
        assert microseconds(lambda: train(*x)) <= 60 * usual
    with torch.no_grad():
        usual = microseconds(lambda: A().attention(q, k, v))
        v2 = v.clone()
        v2[0, 0, 3] = math.inf
        assert microseconds(lambda: A().attention(q, k, v2)) <= 60 * usual


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("L,H,Hk,D", [(70, 4, 2, 64), (300, 8, 2, 128), (961, 64, 64, 40)])
def test_gradient_of_an_infinite_gradient(L, H, Hk, D, dtype):
    """One infinity in the last row of dL/do, channel 3 of head 1: infinities of
    the formula's signs where sums have them as terms, NaN where two meet, every
    other sum as without it."""
    q, k, v, grad = step(L, H, Hk, D, dtype)
    clean = one(q, k, v, grad)
    head, kv = 1, 1 // (H // Hk)
    g2 = grad.clone()
    g2[L - 1, head, 3] = math.inf
    dq, dk, dv = train(q, k, v, g2)
    # (delta and g v of that row are infinite)
    o3, v3 = clean["out"][0][L - 1, head, 3], v[:, kv, 3].double()
    ds = torch.where(v3.sign() == o3.sign(), math.nan, v3.sign() * math.inf)
    want = {"dq": (dq, clean["dq"][0].clone()), "dk": (dk, clean["dk"][0].clone()), "dv": (dv, clean["dv"][0].clone())}
    want["dq"][1][L - 1, head] = math.nan
    want["dk"][1][:, kv] = ds[:, None] * q[L - 1, head].double()
    want["dv"][1][:, kv, 3] = math.inf
    for name, (got, ref) in want.items():
        fine = ref.isfinite()
        assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.double()[ref.isinf()], ref[ref.isinf()]), name
        check(got[fine], (ref[fine], clean[name][1][fine]))


def spoil(v, seed, n=6):
    """v with infinities of both signs and NaN in some places, and v with zeros there."""
    g = torch.Generator().manual_seed(seed)
    bad, clean = v.clone(), v.clone()
    for i in range(n):
        at = tuple(int(torch.randint(0, s, (1,), generator=g)) for s in v.shape)
        bad[at] = (math.inf, -math.inf, math.nan)[i % 3]
        clean[at] = 0
    return bad, clean


def follows(out, q, k, bad, clean):
    """out: infinite or NaN where the formula is (of what a row sees), within the
    bounds elsewhere; later queries see all earlier keys and their own."""
    L, S, G = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    ref, bound = one(q, k, clean)["out"]
    sees = (torch.arange(S, device="cuda")[None] <= torch.arange(L, device="cuda")[:, None] + S - L).float()

    def count(x):  # of such values that each row sees: (L, heads, channels)
        return torch.einsum("ls,shd->lhd", sees, x.float()).repeat_interleave(G, 1) > 0
    up, down, nan = count(bad == math.inf), count(bad == -math.inf), count(bad.isnan())
    nan = nan | (up & down)
    assert torch.equal(out.isnan(), nan)
    assert torch.equal(out == math.inf, up & ~nan) and torch.equal(out == -math.inf, down & ~nan)
    fine = ~(up | down | nan)
    check(out[fine], (ref[fine], bound[fine]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("L,H,Hk,D", [(70, 7, 1, 40), (200, 6, 2, 96), (333, 4, 4, 64), (150, 8, 2, 128)])
def test_not_finite_values_as_the_formula(L, H, Hk, D, dtype):
    q, k, v, _ = step(L, H, Hk, D, dtype)
    for seed in range(4):
        bad, clean = spoil(v, seed)
        with torch.no_grad():
            follows(A().attention(q, k, bad), q, k, bad, clean)
        follows(A().attention(q.clone().requires_grad_(True), k, bad).detach(), q, k, bad, clean)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Hk,D,page", [(7, 1, 40, 7), (6, 2, 96, 16), (8, 4, 64, 24), (8, 2, 128, 64)])
@pytest.mark.parametrize("new,S", [(1, 50), (1, 3000), (5, 700), (130, 1300)])
def test_not_finite_cached_values_as_the_formula(new, S, H, Hk, D, page, dtype):
    """Few and many rows, one part and many, pages that end inside a tile."""
    _, k, v, _ = step(S, H, Hk, D, dtype)
    q = step(new, H, Hk, D, dtype)[0]
    pages = -(-S // page)
    table = torch.randperm(pages, device="cuda").int()
    place = table.long()[torch.arange(S, device="cuda") // page] * page + torch.arange(S, device="cuda") % page
    for seed in range(3):
        bad, clean = spoil(v, seed)
        kc, vc = (torch.full((pages * page, Hk, D), math.nan, device="cuda", dtype=dtype) for _ in range(2))
        kc[place], vc[place] = k, bad
        out = A().paged_attention(q, kc.view(pages, page, Hk, D), vc.view(pages, page, Hk, D), table[None],
                                  torch.tensor([S], device="cuda"), torch.tensor([0, new], device="cuda"))
        follows(out, q, k, bad, clean)
