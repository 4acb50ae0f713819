"""What the attention path decides on the host: rotary frequencies, the paged
cache's book-keeping, the kernel plan and the entry points' refusals.  No GPU."""
import ctypes
import math
import os

import pytest
import torch

from distributed_gptq_amd import _lib
from distributed_gptq_amd.models import attention as A


def test_frequencies():
    inv, f = A.rotary_frequencies(8, 10000.0)
    assert f == 1.0 and torch.allclose(inv, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    lin, _ = A.rotary_frequencies(8, 10000.0, {"type": "linear", "factor": 4.0})
    assert torch.allclose(lin, inv / 4)
    ntk, _ = A.rotary_frequencies(8, 10000.0, {"type": "ntk", "factor": 4.0})
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]), float(inv[-1]) / 4, rel_tol=1e-12)
    n = 8192
    bands, _ = A.rotary_frequencies(128, 500000.0, {"type": "bands", "factor": 8.0, "low": 1.0, "high": 4.0,
                                                   "context": n})
    base, _ = A.rotary_frequencies(128, 500000.0)
    turns = n * base / (2 * math.pi)
    assert torch.equal(bands[turns > 4], base[turns > 4]) and torch.allclose(bands[turns < 1], base[turns < 1] / 8)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and bool((bands[mid] < base[mid]).all()) and bool((bands[mid] > base[mid] / 8).all())
    yarn, m = A.rotary_frequencies(128, 10000.0, {"type": "yarn", "factor": 4.0, "context": 4096})
    base, _ = A.rotary_frequencies(128, 10000.0)
    assert math.isclose(m, 0.1 * math.log(4.0) + 1.0)
    turns = 4096 * base / (2 * math.pi)
    assert torch.equal(yarn[turns > 33], base[turns > 33]) and torch.allclose(yarn[turns < 0.9], base[turns < 0.9] / 4)
    assert bool((yarn[1:] < yarn[:-1]).all())


def test_frequencies_refusals():
    for args in ((7,), (0,), (8, 1e4, {"type": "other", "factor": 2.0}), (8, 1e4, {"type": "linear", "factor": 0.5}),
                 (2, 1e4, {"type": "ntk", "factor": 2.0})):
        with pytest.raises(ValueError):
            A.rotary_frequencies(*args)


def test_table():
    t = A.rotary_table(16, 1000, base=10000.0, device="cpu")
    assert t.shape == (1000, 2, 8) and t.dtype == torch.float32
    a = 999 * 10000.0 ** (-torch.arange(0, 16, 2, dtype=torch.float64) / 16)
    assert torch.equal(t[999], torch.stack([a.cos(), a.sin()]).float())
    y = A.rotary_table(16, 4, scaling={"type": "yarn", "factor": 16.0, "context": 128}, device="cpu")
    assert torch.allclose(y[0, 0], torch.full((8,), 0.1 * math.log(16.0) + 1.0))


def test_cache_book_keeping():
    c = A.PagedKVCache(6, 4, 2, 8, layers=3, device="cpu")
    assert c.k.shape == (3, 6, 4, 2, 8) and c.free_pages == 6
    b = c.extend(["a", "b"], [5, 1])
    assert b.cu_seqlens.tolist() == [0, 5, 6] and b.context_lens.tolist() == [5, 1] and b.max_context == 5
    assert b.positions.tolist() == [0, 1, 2, 3, 4, 0]
    pages = b.block_table.tolist()
    assert b.slots.tolist() == [pages[0][0] * 4 + i for i in range(4)] + [pages[0][1] * 4, pages[1][0] * 4]
    assert c.free_pages == 3 and len({pages[0][0], pages[0][1], pages[1][0]}) == 3
    b = c.extend(["b", "a"], [1, 1])
    assert b.cu_seqlens is None and b.positions.tolist() == [1, 5] and b.context_lens.tolist() == [2, 6]
    assert b.slots.tolist() == [pages[1][0] * 4 + 1, pages[0][1] * 4 + 1] and c.free_pages == 3
    with pytest.raises(MemoryError):
        c.extend(["a", "z"], [15, 1])
    assert c.length("a") == 6 and "z" not in c and c.free_pages == 3  # nothing changed
    c.free("a")
    assert c.free_pages == 5 and "a" not in c
    assert all(0 <= s < 24 for s in c.extend(["n"], [20]).slots.tolist()) and c.free_pages == 0
    for bad in ((["n"], [0]), (["n", "n"], [1, 1]), ([], []), (["n"], [1, 1])):
        with pytest.raises(ValueError):
            c.extend(*bad)
    with pytest.raises(ValueError):
        A.PagedKVCache(0, 4, 2, 8, device="cpu")


def test_packed_positions():
    cu = torch.tensor([0, 3, 3, 7], dtype=torch.int32)
    assert A.packed_positions(cu, 7).tolist() == [0, 1, 2, 0, 1, 2, 3]
    assert A.packed_positions(cu, 9).tolist()[:7] == [0, 1, 2, 0, 1, 2, 3]


def test_no_cpu_path():
    x = torch.zeros(4, 2, 64, dtype=torch.float16)
    with pytest.raises((RuntimeError, ValueError), match="GPU"):
        A.attention(x, x, x)
    with pytest.raises((RuntimeError, ValueError), match="GPU"):
        A.rotary(x, x, torch.zeros(4, 2, 32), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        A.QuantizedAttention(torch.nn.Identity(), torch.nn.Identity(), 6, 4, 64)


@pytest.fixture
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return _lib.load()


def test_workspaces(lib):
    size = lib.gptq_paged_attention_workspace_size
    for B, T, H, Hk, D, n in [(1, 1, 32, 8, 128, 8192), (24, 24, 32, 8, 128, 8192), (1, 512, 32, 8, 128, 16896),
                              (1, 1, 1, 1, 8, 10 ** 9), (4096, 4096, 64, 64, 128, 10 ** 6)]:
        b = size(B, T, H, Hk, D, n)
        assert b % (4 * T * H * (D + 2)) == 0 and b // (4 * T * H * (D + 2)) <= 128
        assert size(B, T, H, Hk, D, 1) == 0  # a short context is never split
    assert size(1, 1, 32, 8, 128, 131072) > 0
    for bad in [(0, 1, 4, 4, 64, 9), (1, -1, 4, 4, 64, 9), (1, 1, 4, 3, 64, 9), (1, 1, 4, 4, 60, 9),
                (1, 1, 4, 4, 136, 9), (1, 2 ** 62, 4, 4, 64, 9), (2 ** 62, 1, 4, 4, 64, 9)]:
        assert size(*bad) == 0
    back = lib.gptq_attention_backward_workspace_size
    assert back(1, 10, 10, 4, 4, 64) == 4 * (40 + 2048 + 2 * 8 * 10 * 4 * 64)  # few keys: 8 parts of the rows
    assert back(2, 4096, 4096, 32, 8, 128) == 4 * (4096 * 32 + 2048 + 2 * 2 * 4096 * 8 * 128)
    assert back(1, 16384, 16384, 32, 8, 128) == 4 * (16384 * 32 + 2048)        # many: whole
    assert back(1, 3, 3, 1, 1, 8) % 16 == 0
    for bad in [(1, -1, 4, 4, 4, 64), (1, 2 ** 62, 4, 4, 4, 64), (1, 4, 2 ** 62, 4, 4, 64), (1, 4, 4, 4, 3, 64)]:
        assert back(*bad) == 0


def test_refusals_before_a_launch(lib):
    P, f = ctypes.c_void_p, ctypes.c_float
    x, null = P(64), P(0)

    def forward(dtype=1, q=x, strides=(128, 64) * 3, cu=null, B=1, T=4, S=4, H=2, Hk=2, D=64, scale=0.1):
        return lib.gptq_attention(q, x, x, dtype, *strides, cu, cu, B, T, S, H, Hk, D, 1, f(scale), x, null, null, null)
    assert forward(dtype=0) == _lib.ERR_DTYPE and b"fp16" in lib.gptq_last_error()
    assert forward(q=null) == _lib.ERR_ARG and forward(q=P(8)) == _lib.ERR_ARG
    assert forward(strides=(128, 60) * 3) == _lib.ERR_SHAPE and forward(strides=(-128, 64) * 3) == _lib.ERR_SHAPE
    assert forward(strides=(2 ** 28, 64) * 3) == _lib.ERR_SHAPE
    assert forward(Hk=3) == _lib.ERR_SHAPE and forward(D=20) == _lib.ERR_SHAPE and forward(D=256) == _lib.ERR_SHAPE
    assert forward(B=2) == _lib.ERR_ARG and forward(B=0) == _lib.ERR_SHAPE and forward(T=-1) == _lib.ERR_SHAPE
    assert forward(T=2 ** 40) == _lib.ERR_SHAPE and forward(scale=0.0) == _lib.ERR_ARG
    assert forward(scale=1e-8) == _lib.ERR_ARG and forward(scale=1e8) == _lib.ERR_ARG
    assert forward(T=0) == _lib.OK

    def paged(ws=0, page=16, pages=4, T=1, B=1, cu=null, n=100000):
        return lib.gptq_paged_attention(x, x, x, 2, 128, 64, 2048, 128, 64, 2048, 128, 64, x, 8, 8, page, pages, x, cu, B,
                                        T, 2, 2, 64, f(0.1), n, x, null, ws, null)
    assert paged() == _lib.ERR_WORKSPACE and b"workspace" in lib.gptq_last_error()
    assert paged(page=0) == _lib.ERR_ARG and paged(pages=0) == _lib.ERR_ARG
    assert paged(T=3, B=2) == _lib.ERR_SHAPE
    rc = lib.gptq_rotary(x, x, 5, 64, 64, 64, 64, x, 4, 64, x, 0, 0, 1, 1, 1, 64, x, x, null)
    assert rc == _lib.ERR_DTYPE
    rc = lib.gptq_rotary(x, x, 1, 64, 64, 64, 64, x, 4, 66, x, 0, 0, 1, 1, 1, 64, x, x, null)
    assert rc == _lib.ERR_SHAPE
    rc = lib.gptq_rotary_append(x, x, x, 1, 64, 64, 64, 64, 64, 64, null, 0, 0, null, 0, x, 0, 4, 1, 1, 1, 64, x, x, 64,
                                64, 64, x, 64, 64, 64, null)
    assert rc == _lib.ERR_ARG
    assert forward(T=0) == _lib.OK and lib.gptq_last_error() == b""  # (a call that succeeds clears the message)
