"""What the attention calls do with index tensors and layouts beyond the
ordinary ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu

FAR = 2 ** 32


def A():
    from distributed_gptq_amd.models import attention
    return attention


def rand(*shape, seed=0, dtype=torch.float16):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def long(*values):
    return torch.tensor(values, dtype=torch.int64, device="cuda")


def test_slots_beyond_32_bits_are_not_written():
    m = A()
    q, k, v = rand(5, 4, 64), rand(5, 2, 64, seed=1), rand(5, 2, 64, seed=2)
    kc, vc = rand(3, 16, 2, 64, seed=3), rand(3, 16, 2, 64, seed=4)
    kw, vw = kc.clone(), vc.clone()
    kw[0, 7], vw[0, 7] = k[3], v[3]
    m.rotary_append(q, k, v, None, None, kc, vc, long(FAR, FAR + 5, 3 - FAR, 7, 2 ** 63 - 1))
    assert torch.equal(kc, kw) and torch.equal(vc, vw)


def test_positions_beyond_32_bits_are_those_of_the_tables_ends():
    m = A()
    table = m.rotary_table(64, 40)
    q, k = rand(4, 4, 64), rand(4, 2, 64, seed=1)
    got = m.rotary(q, k, table, long(FAR + 1, 1 - FAR, 5, 2 ** 63 - 1))
    want = m.rotary(q, k, table, long(39, 0, 5, 39))
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_lengths_pages_and_offsets_beyond_32_bits_are_clamped():
    m = A()
    q, kc, vc = rand(2, 4, 64), rand(6, 16, 2, 64, seed=1), rand(6, 16, 2, 64, seed=2)
    got = m.paged_attention(q, kc, vc, long(0, FAR, 2, 4, -FAR, 1).view(2, 3), long(FAR + 5, 20), max_context=48)
    want = m.paged_attention(q, kc, vc, long(0, 5, 2, 4, 0, 1).view(2, 3), long(48, 20), max_context=48)
    assert torch.equal(got, want)
    assert not m.paged_attention(q, kc, vc, long(0, 1, 2, 3, 4, 5).view(2, 3), long(5 - FAR, -FAR)).any()
    q, k, v = rand(20, 4, 64), rand(20, 2, 64, seed=1), rand(20, 2, 64, seed=2)
    assert torch.equal(m.attention(q, k, v, long(0, 9, FAR + 12)), m.attention(q, k, v, long(0, 9, 20)))


def test_a_refused_cache_is_not_copied():
    m = A()
    q = rand(1, 4, 64)
    kc = torch.zeros(512, 64, 64, 2, device="cuda", dtype=torch.float16).transpose(2, 3)  # heads that are not contiguous
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(ValueError, match="cache"):
        m.paged_attention(q, kc, kc, torch.zeros(1, 4, dtype=torch.int32, device="cuda"), long(5))
    assert torch.cuda.max_memory_allocated() - before < kc.numel()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tokens_2_to_the_28_values_apart_are_copied(dtype):
    """As other layouts that the kernels do not read: the same bits as from
    contiguous tensors; a cache is refused."""
    m = A()
    far = 2 ** 28
    room = torch.empty(2 * far + 4096, device="cuda", dtype=dtype)

    def spread(x, at):
        y = room.as_strided(x.shape, (far, x.shape[2], 1), at)
        return y.copy_(x)
    x = [rand(3, n, 64, seed=i, dtype=dtype) for i, n in enumerate((4, 2, 2, 4))]
    far_x = [spread(t, 512 * i) for i, t in enumerate(x)]

    def run(q, k, v, g):
        q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
        out = m.attention(q, k, v)
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), g)]
    want = run(*x)
    assert all(torch.equal(a, b) for a, b in zip(run(*far_x), want))
    for i in range(4):  # each of them alone
        assert all(torch.equal(a, b) for a, b in zip(run(*x[:i], far_x[i], *x[i + 1:]), want))
    kc, vc = x[1][None], x[2][None]
    table, context = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), long(3)
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    assert torch.equal(m.paged_attention(far_x[0], kc, vc, table, context, cu),
                       m.paged_attention(x[0], kc, vc, table, context, cu))
    with pytest.raises(ValueError):
        m.paged_attention(x[0], far_x[1][None], vc, table, context, cu)
