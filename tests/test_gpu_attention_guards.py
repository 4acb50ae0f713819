"""No attention call reads or writes outside its tensors: inputs, outputs and
the workspace lie inside larger buffers whose other bytes are compared bit for
bit, with proper offsets, pages and slots and with ones that no caller should
give.  (What the index arithmetic does with those is checked exhaustively on
the CPU.)"""
import itertools

import pytest
import torch

from attention_check import check, packed

pytestmark = pytest.mark.gpu

TYPES = {torch.float16: 1, torch.bfloat16: 2}
ZONE = 1 << 16
FAR = 2 ** 31 - 1


class Room:
    """Tensors with filled zones before and after each."""

    def __init__(self):
        self.all = []

    def empty(self, *shape, dtype, fill=0x5A):
        size = torch.empty((), dtype=dtype).element_size()
        n = size
        for s in shape:
            n *= s
        raw = torch.full((ZONE + -(-n // 256) * 256 + ZONE,), fill, dtype=torch.uint8, device="cuda")
        self.all.append((raw, n, fill))
        return raw[ZONE:ZONE + n].view(dtype).view(shape)

    def input(self, x):
        # (0xFF: NaN in every type, so that a row read from outside shows)
        return self.empty(*x.shape, dtype=x.dtype, fill=0xFF).copy_(x)

    def check(self):
        torch.cuda.synchronize()
        for raw, n, fill in self.all:
            assert bool((raw[:ZONE] == fill).all()) and bool((raw[ZONE + n:] == fill).all())


def ptr(x):
    return None if x is None else x.data_ptr()


def strides(x):
    return x.stride(0), x.stride(1)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def both(room, q, k, v, g, cq, ck, causal=True):
    """Forward and gradients through the C entry points."""
    from distributed_gptq_amd import _lib
    T, H, D = q.shape
    S, Hk = k.shape[:2]
    dt = TYPES[q.dtype]
    scale = D ** -0.5
    q, k, v, g = (room.input(x) for x in (q, k, v, g))
    cq, ck = room.input(ints(cq)), room.input(ints(ck))
    B = cq.numel() - 1
    out, rest, dq = (room.empty(T, H, D, dtype=q.dtype).zero_() for _ in range(3))
    dk, dv = (room.empty(S, Hk, D, dtype=q.dtype).zero_() for _ in range(2))
    lse = room.empty(T, H, dtype=torch.float32).zero_()
    stream = torch.cuda.current_stream().cuda_stream
    _lib.call("gptq_attention", ptr(q), ptr(k), ptr(v), dt, *strides(q), *strides(k), *strides(v), ptr(cq), ptr(ck), B, T,
              S, H, Hk, D, int(causal), scale, ptr(out), ptr(rest), ptr(lse), stream)
    n = _lib.lib().gptq_attention_backward_workspace_size(B, T, S, H, Hk, D)
    ws = room.empty(n, dtype=torch.uint8).zero_()
    _lib.call("gptq_attention_backward", ptr(g), ptr(q), ptr(k), ptr(v), ptr(out), ptr(rest), ptr(lse), dt, *strides(g),
              *strides(q), *strides(k), *strides(v), ptr(cq), ptr(ck), B, T, S, H, Hk, D, int(causal), scale, ptr(dq),
              ptr(dk), ptr(dv), ptr(ws), n, stream)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def heads(T, S, H, Hk, D, dtype):
    gen = torch.Generator(device="cuda").manual_seed(T + S + D)
    return [(torch.randn(t, h, D, generator=gen, device="cuda") * f).to(dtype)
            for t, h, f in ((T, H, 2.0), (S, Hk, 1.0), (S, Hk, 1.0), (T, H, 1e-2))]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 128), (3, 1, 40), (64, 64, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed(H, Hk, D, causal, dtype):
    """Proper offsets: the values too, so that nothing was read from outside."""
    cq, ck = [0, 70, 70, 101], [0, 3, 80, 193]
    room = Room()
    x = heads(101, 193, H, Hk, D, dtype)
    got = both(room, *x, cq, ck, causal)
    room.check()
    want = packed(*x[:3], cq, ck, x[3], causal)
    for name in want:
        check(got[name], want[name])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 128), (3, 1, 40), (128, 64, 8)])
def test_packed_with_offsets_of_any_kind(H, Hk, D, dtype):
    x = heads(129, 130, H, Hk, D, dtype)
    for offsets in ([0, FAR], [5, 64], [0, 50, 20, 129], [-4, 30, 64], [0, FAR, -FAR - 1], [0, 0, 0], [129, 0, 129],
                    [FAR, 7, 1]):
        for other in (offsets, offsets[::-1]):
            room = Room()
            both(room, *x, offsets, other, offsets is other)
            room.check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk,D,page", [(8, 2, 128, 16), (7, 1, 40, 7), (4, 4, 64, 32)])
def test_paged_with_lengths_and_pages_of_any_kind(H, Hk, D, page, dtype):
    from distributed_gptq_amd import _lib
    pages, width = 9, 70
    for new, context, longest in itertools.product(([0, 1, 2], [0, 40, 300], [0, 300, FAR], [9, -1, 200]),
                                                   ([1, 600], [FAR, -FAR], [0, 5], [1100, 1100]), (1, 5000)):
        T = 300 if max(new) > 2 else 2
        q, kc, vc, _ = heads(T, pages * page, H, Hk, D, dtype)
        room = Room()
        q, kc, vc = (room.input(x) for x in (q, kc.view(pages, page, Hk, D), vc.view(pages, page, Hk, D)))
        odd = [0, 3, pages, -1, FAR, -FAR - 1, pages - 1]
        table = room.input(ints([[odd[(b + i) % 7] for i in range(width)] for b in range(2)]))
        cu, ctx = room.input(ints(new)), room.input(ints(context))
        n = _lib.lib().gptq_paged_attention_workspace_size(2, T, H, Hk, D, longest)
        out, ws = room.empty(T, H, D, dtype=dtype), room.empty(max(n, 1), dtype=torch.uint8).zero_()
        _lib.call("gptq_paged_attention", ptr(q), ptr(kc), ptr(vc), TYPES[dtype], *strides(q), *kc.stride()[:3],
                  *vc.stride()[:3], ptr(table), width, width, page, pages, ptr(ctx), ptr(cu), 2, T, H, Hk, D, D ** -0.5,
                  longest, ptr(out), ptr(ws), n, torch.cuda.current_stream().cuda_stream)
        room.check()
        assert bool(torch.isfinite(out).all())  # nothing was read from outside (the zones of the inputs are NaN)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_with_slots_and_positions_of_any_kind(dtype):
    from distributed_gptq_amd.models import attention as A
    T, H, Hk, D, pages, page = 9, 4, 2, 40, 3, 7
    q, k, v, _ = heads(T, T, H, Hk, D, dtype)
    room = Room()
    q, k, v = (room.input(x) for x in (q, k, v))
    kc, vc = (room.empty(pages, page, Hk, D, dtype=dtype).zero_() for _ in range(2))
    table = room.input(A.rotary_table(D, 11))
    pos = room.input(ints([0, -1, 11, FAR, -FAR - 1, 10, 5, 6, 7]))
    slots = room.input(ints([0, -1, pages * page, FAR, -FAR - 1, pages * page - 1, 8, 15, 3]))
    out = A.rotary_append(q, k, v, table, pos, kc, vc, slots)
    room.check()
    assert bool(torch.isfinite(out).all() & torch.isfinite(kc).all() & torch.isfinite(vc).all())
    kept = {0, pages * page - 1, 8, 15, 3}
    written = vc.view(-1, Hk * D).any(1).nonzero().flatten().tolist()
    assert set(written) == kept
