"""Normed heads and quantised caches on the host: the cache's layout, the
module's arguments, the entry points' refusals before a launch, the operators'
derivatives with stand-ins for the kernels, and which cached token a row reads
back.  No GPU."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch
import torch.autograd.forward_ad as fw
import torch.nn as nn

from distributed_gptq_amd import _lib
from distributed_gptq_amd.models import attention as A

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CODES = [torch.int8, torch.float8_e4m3fn]


def test_index_arithmetic(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "cached_rows_check")
    subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    os.path.join(ROOT, "tests", "host", "cached_rows_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and " 0 check(s) failed" in r.stderr, r.stderr[-2000:]


# ------------------------------------------------------------------- cache --

@pytest.mark.parametrize("dtype", CODES)
def test_quantised_cache(dtype):
    c = A.PagedKVCache(6, 4, 2, 32, layers=3, dtype=dtype, device="cpu")
    assert c.k.shape == c.v.shape == (3, 6, 4, 2, 32) and c.k.dtype == dtype
    assert c.k_scale.shape == c.v_scale.shape == (3, 6, 4, 2) and c.k_scale.dtype == torch.float32
    # a head's rows of a page lie next to each other
    assert c.k.stride()[2:] == (32, 4 * 32, 1) and c.k_scale.stride()[2:] == (1, 4)
    s = c.scales(1)
    assert s["k_scale"].data_ptr() == c.k_scale[1].data_ptr() and s["v_scale"].data_ptr() == c.v_scale[1].data_ptr()
    assert c.extend(["a"], [5]).slots.numel() == 5 and c.length("a") == 5
    with pytest.raises(ValueError, match="16"):
        A.PagedKVCache(6, 4, 2, 40, dtype=dtype, device="cpu")
    with pytest.raises(ValueError):
        c.rows(["b"])
    with pytest.raises(ValueError):
        c.rows([])


def test_a_cache_of_values_has_no_scales():
    c = A.PagedKVCache(6, 4, 2, 40, device="cpu")
    assert c.k_scale is None and c.v_scale is None and c.scales() == {} and c.k.is_contiguous()


@pytest.mark.parametrize("dtype", CODES + [torch.float16])
def test_rows_of_a_cache(monkeypatch, dtype):
    """What ``rows`` asks of the operator."""
    c = A.PagedKVCache(6, 4, 2, 32, layers=2, dtype=dtype, device="cpu")
    c.extend(["a", "b"], [5, 1])
    a, b = (c._pages[x] for x in "ab")
    got = []
    monkeypatch.setattr(A, "_op", lambda name, *args: (got.append((name, *args)), (None, None))[1])
    c.rows(["b", "a"], layer=1)
    name, k, v, table, ctx, cu, tokens, ks, vs, out = got[0]
    assert name == "cached_rows" and tokens == 6 and ctx.tolist() == [1, 5] and cu.tolist() == [0, 1, 6]
    assert table.tolist() == [[b[0], 0], a] and k.data_ptr() == c.k[1].data_ptr()
    assert out == (torch.float16 if dtype == torch.float16 else torch.bfloat16) and (ks is None) == (dtype == torch.float16)


# ------------------------------------------------------------------ module --

def test_module_arguments():
    w = torch.ones(8)
    a = nn.Identity(), nn.Identity(), 4, 2, 8
    with pytest.raises(ValueError, match="norm"):
        A.QuantizedAttention(*a, q_norm=w)
    with pytest.raises(ValueError, match="norm"):
        A.QuantizedAttention(*a, q_norm=w, k_norm=torch.ones(16))
    m = A.QuantizedAttention(*a, q_norm=w, k_norm=2 * w)
    assert {n for n, _ in m.named_parameters()} == {"q_norm", "k_norm"} and m.k_norm.requires_grad
    assert not list(A.QuantizedAttention(*a).parameters())
    again = A.QuantizedAttention(*a, q_norm=w, k_norm=w)
    again.load_state_dict(m.state_dict())
    assert torch.equal(again.k_norm, m.k_norm)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", CODES + [torch.float32])
@pytest.mark.parametrize("rotary", [False, True])
def test_what_the_module_calls(monkeypatch, norm, dtype, rotary):
    called = []

    def op(name, *args):
        called.append((name, args))
        return args[:2] if name in ("rotary", "norm_rotary") else torch.zeros(args[0].shape[0], 4, 16)
    monkeypatch.setattr(A, "_op", op)

    class Heads(nn.Module):
        def forward(self, x):
            return x.new_zeros(len(x), 64), x.new_zeros(len(x), 32), x.new_zeros(len(x), 32)
    w = {"q_norm": torch.ones(16), "k_norm": torch.ones(16)} if norm else {}
    m = A.QuantizedAttention(Heads(), nn.Identity(), 4, 2, 16, A.rotary_table(16, 20, device="cpu") if rotary else None, **w)
    m(torch.zeros(5, 8))
    assert [n for n, _ in called] == (["norm_rotary"] if norm else ["rotary"] if rotary else []) + ["attention"]
    if norm:
        args = called[0][1]
        assert args[2] is m.q_norm and args[3] is m.k_norm and (args[4] is None) == (args[5] is None) == (not rotary)
    cache = A.PagedKVCache(8, 8, 2, 16, dtype=dtype, device="cpu")
    called.clear()
    m.step(torch.zeros(5, 8), cache, cache.extend(["a"], [5]))
    coded = dtype in CODES
    assert [n for n, _ in called] == ["norm_rotary_append" if norm or coded else "rotary_append",
                                      "code_attention" if coded else "paged_attention"]
    if norm or coded:
        args = called[0][1]
        assert (args[3] is m.q_norm and args[4] is m.k_norm) if norm else args[3] is args[4] is None
        assert (args[10] is None) == (not coded)


# -------------------------------------------------------------- refusals --

@pytest.fixture
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return _lib.load()


P, F = ctypes.c_void_p, ctypes.c_float
X, NULL = P(64), P(0)


def test_norm_rotary_refusals(lib):
    def call(dtype=1, q=X, strides=(128, 64) * 2, wq=X, wt=0, eps=1e-6, table=X, rows=4, R=64, pos=X, T=4, H=2, Hk=2,
             D=64, out=X):
        return lib.gptq_norm_rotary(q, X, dtype, *strides, wq, X, wt, F(eps), table, rows, R, pos, 0, T, H, Hk, D, out, X,
                                    NULL)
    assert call(dtype=3) == call(wt=7) == _lib.ERR_DTYPE
    assert call(q=NULL) == call(q=P(8)) == call(wq=NULL) == call(wq=P(72)) == call(pos=NULL) == call(out=NULL) == _lib.ERR_ARG
    assert call(table=P(68)) == call(eps=0.0) == call(eps=-1.0) == call(eps=2.0) == call(eps=float("nan")) == _lib.ERR_ARG
    assert call(strides=(128, 60) * 2) == call(strides=(-128, 64) * 2) == _lib.ERR_SHAPE
    assert call(D=20) == call(D=264) == call(D=0) == call(R=66) == call(R=0) == call(R=62) == call(rows=0) == _lib.ERR_SHAPE
    assert call(T=-1) == call(T=2 ** 31) == call(H=0) == call(Hk=65537) == _lib.ERR_SHAPE
    assert call(T=0, q=NULL) == _lib.OK and lib.gptq_last_error() == b""


def test_norm_rotary_backward_refusals(lib):
    size = lib.gptq_norm_rotary_backward_workspace_size
    assert size(4, 2, 2, 64) == 4 * 2 * 64 and size(0, 2, 2, 64) == 4 * 2 * 64
    assert size(10 ** 6, 32, 8, 128) == 1024 * 4 * 2 * 128 and size(33, 1, 1, 8) == 2 * 4 * 2 * 8
    for bad in ((-1, 2, 2, 64), (2 ** 31, 2, 2, 64), (4, 0, 2, 64), (4, 2, 65537, 64), (4, 2, 2, 4), (4, 2, 2, 512)):
        assert size(*bad) == 0

    def call(ws=X, n=10 ** 6, dwq=X, dwk=X, gq=X, T=4, D=64, R=64):
        return lib.gptq_norm_rotary_backward(gq, X, X, X, 1, *(128, 64) * 4, X, X, 0, F(1e-6), X, 4, R, X, 0, T, 2, 2, D,
                                             X, X, dwq, dwk, ws, n, NULL)
    assert call(ws=NULL) == call(n=100) == _lib.ERR_WORKSPACE and b"workspace" in lib.gptq_last_error()
    assert call(dwq=NULL) == call(dwk=NULL) == call(gq=NULL) == call(gq=P(66)) == call(ws=P(65)) == _lib.ERR_ARG
    assert call(D=12) == call(R=6) == _lib.ERR_SHAPE
    assert call(T=0, dwq=NULL, dwk=NULL) == _lib.OK


def test_append_refusals(lib):
    def call(dtype=1, code=1, q=X, wq=X, wk=X, eps=1e-6, table=X, R=64, page=16, pages=4, D=64, cache=X, scale=X, slots=X,
             strides=(2048, 64, 1024), T=2, heads=(128, 64) * 3):
        return lib.gptq_norm_rotary_append(q, X, X, dtype, *heads, wq, wk, 0, F(eps), table, 8, R, X, 0, slots, page, pages,
                                           T, 2, 2, D, X, code, cache, *strides, X, *strides, scale, 32, 1, 16, X, 32, 1, 16,
                                           NULL)
    assert call(dtype=9) == call(code=3) == call(code=-1) == _lib.ERR_DTYPE
    assert call(wk=NULL) == call(wq=NULL) == call(slots=NULL) == call(cache=NULL) == call(scale=NULL) == _lib.ERR_ARG
    assert call(cache=P(72)) == call(q=P(72)) == call(page=0) == call(pages=-1) == call(eps=0.0) == _lib.ERR_ARG
    assert call(D=40, R=40) == call(D=272) == call(strides=(2048, 40, 1024)) == call(strides=(2048, 64, -16)) == _lib.ERR_SHAPE
    assert call(R=60) == _lib.ERR_SHAPE and b"multiple of 8" in lib.gptq_last_error()
    assert call(heads=(128, 60) * 3) == _lib.ERR_SHAPE
    assert call(T=0) == _lib.OK


def test_rows_and_attention_refusals(lib):
    cache = (X, 2048, 64, 1024, X, 2048, 64, 1024)
    scales = (X, 32, 1, 16, X, 32, 1, 16)

    def rows(code=1, k=cache, s=scales, page=16, pages=4, width=4, table=X, ctx=X, B=1, T=4, Hk=2, D=64, out=X, dtype=1):
        return lib.gptq_cached_rows(code, *k, *s, table, 4, width, page, pages, ctx, X, B, T, Hk, D, out, X, dtype, NULL)
    assert rows(code=5) == rows(dtype=4) == _lib.ERR_DTYPE
    assert rows(ctx=NULL) == rows(table=NULL) == rows(out=NULL) == rows(page=0) == rows(pages=0) == rows(width=-1) == _lib.ERR_ARG
    assert rows(s=(NULL, *scales[1:])) == rows(k=(P(72), *cache[1:])) == rows(out=P(68)) == _lib.ERR_ARG
    assert rows(B=0) == rows(T=-1) == rows(Hk=0) == rows(D=40) == rows(D=0) == rows(D=512) == rows(T=2 ** 31) == _lib.ERR_SHAPE
    assert rows(k=(X, 2048, 72, 1024, *cache[4:])) == rows(code=0, D=4) == _lib.ERR_SHAPE
    assert rows(T=0) == _lib.OK

    def attend(dtype=1, q=X, qs=(128, 64), code=2, k=cache, s=scales, page=16, pages=4, width=4, T=1, B=1, H=2, Hk=2, D=64,
               scale=0.1, n=100, ws=0, cu=NULL):
        return lib.gptq_code_attention(q, dtype, *qs, code, *k, *s, X, 4, width, page, pages, X, cu, B, T, H, Hk, D,
                                       F(scale), n, X, NULL, ws, NULL)
    assert attend(dtype=0) == attend(code=0) == attend(code=3) == _lib.ERR_DTYPE
    assert attend(q=NULL) == attend(q=P(8)) == attend(s=(NULL, *scales[1:])) == attend(page=0) == attend(pages=0) == _lib.ERR_ARG
    assert attend(scale=0.0) == attend(scale=1e9) == attend(k=(P(65), *cache[1:])) == _lib.ERR_ARG
    assert attend(D=40) == attend(D=136) == attend(D=144) == attend(H=3) == attend(T=2) == attend(qs=(120, 60)) == _lib.ERR_SHAPE
    assert attend(k=(X, 2048, 64, 1016, *cache[4:])) == attend(k=(X, -16, 64, 1024, *cache[4:])) == _lib.ERR_SHAPE
    assert attend(n=100000) == _lib.ERR_WORKSPACE
    assert attend(T=0) == _lib.OK and lib.gptq_last_error() == b""


def test_python_refusals():
    q = torch.zeros(2, 2, 16)
    codes, scale = torch.zeros(1, 4, 2, 16, dtype=torch.int8), torch.zeros(1, 4, 2)
    bt, ctx = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for kw in ({}, {"k_scale": scale}, {"v_scale": scale}):
        with pytest.raises(ValueError, match="scales"):
            A.paged_attention(q, codes, codes, bt, ctx, **kw)
    with pytest.raises(ValueError, match="scales"):
        A.paged_attention(q, codes.float(), codes.float(), bt, ctx, k_scale=scale, v_scale=scale)
    for f in (lambda: A.norm_rotary(q, q, q[0, 0], q[0, 0]),
              lambda: A.paged_attention(q, codes, codes, bt, ctx, k_scale=scale, v_scale=scale),
              lambda: A.rotary_append(q, q, q, None, None, codes, codes, ctx, k_scale=scale, v_scale=scale),
              lambda: A.cached_rows(codes, codes, bt, ctx, torch.zeros(3, dtype=torch.int32), 2, k_scale=scale, v_scale=scale)):
        with pytest.raises((RuntimeError, ValueError), match="GPU"):
            f()


# ------------------------------------------------------------- derivatives --

T, H, Hk, D, EPS = 6, 4, 2, 16, 1e-6


def turned(x, table, positions, back=False):
    if table is None:
        return x
    c, s = table[positions.long()].unsqueeze(2).unbind(1)
    s = -s if back else s
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def normed(x, w, table, positions):
    return turned(x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w, table, positions)


@pytest.fixture
def stand_ins():
    try:
        _lib.load_torch_ops()
    except Exception as e:
        pytest.skip(f"libraries not built: {e}")
    lib = torch.library.Library("gptq", "IMPL")
    seen = []

    def back(gq, gk, q, k, wq, wk, table, positions, interleaved, eps, weights):
        seen.append(weights)
        got, dw = [], []
        for g, x, w in ((gq, q, wq), (gk, k, wk)):
            g = turned(g, table, positions, True)
            r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
            hat = x * r
            dw.append((g * hat).sum((0, 1)))
            g = g * w
            got.append(r * (g - hat * (g * hat).mean(-1, keepdim=True)))
        none = torch.Tensor()
        return (*got, *(dw if weights else (none, none)))
    lib.impl("norm_rotary", lambda q, k, wq, wk, t, p, i, eps: (normed(q, wq, t, p), normed(k, wk, t, p)), "CPU")
    lib.impl("norm_rotary_backward", back, "CPU")
    lib.impl("norm_rotary_append", lambda q, *a: q.clone(), "CPU")
    lib.impl("cached_rows", lambda k, v, bt, ctx, cu, n, ks, vs, dt: (torch.zeros(n, Hk, D), torch.zeros(n, Hk, D)), "CPU")
    lib.impl("code_attention", lambda q, *a: q.clone(), "CPU")
    yield seen
    lib._destroy()


def heads():
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(T, n, D, generator=g) for n in (H, Hk))
    wq, wk = (1 + 0.3 * torch.randn(D, generator=g) for _ in "qk")
    return q, k, wq, wk


@pytest.mark.parametrize("table", [True, False])
def test_gradients_reach_heads_and_weights(stand_ins, table):
    x = [t.requires_grad_(True) for t in heads()]
    args = (A.rotary_table(D, 16, device="cpu"), torch.arange(T)) if table else (None, None)
    got = torch.autograd.grad(A.norm_rotary(*x, *args), x, [torch.ones(T, H, D), 2 * torch.ones(T, Hk, D)])
    ref = torch.autograd.grad((normed(x[0], x[2], *args), normed(x[1], x[3], *args)), x,
                              [torch.ones(T, H, D), 2 * torch.ones(T, Hk, D)])
    for a, b in zip(got, ref):
        assert torch.allclose(a, b, atol=1e-5)
    assert stand_ins == [True]


def test_frozen_weights_take_no_sums(stand_ins):
    q, k, wq, wk = heads()
    q.requires_grad_(True)
    A.norm_rotary(q, k, wq, wk)[0].sum().backward()
    assert stand_ins == [False] and q.grad is not None and wq.grad is None
    q, k, wq, wk = heads()
    wk.requires_grad_(True)
    A.norm_rotary(q, k, wq, wk)[1].sum().backward()
    assert stand_ins == [False, True] and wk.grad is not None and wq.grad is None


def test_second_derivatives_raise(stand_ins):
    q, k, wq, wk = heads()
    q.requires_grad_(True)
    g, = torch.autograd.grad(A.norm_rotary(q, k, wq, wk)[0].square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()


def test_forward_mode_and_serving_calls_raise(stand_ins):
    q, k, wq, wk = heads()
    table, pos = A.rotary_table(D, 16, device="cpu"), torch.arange(T)
    codes, scale = torch.zeros(2, 4, Hk, D, dtype=torch.int8), torch.zeros(2, 4, Hk)
    s = {"k_scale": scale, "v_scale": scale.clone()}
    bt, ctx = torch.zeros(T, 2, dtype=torch.int32), torch.ones(T, dtype=torch.int32)
    calls = [lambda x: A.norm_rotary(x, k, wq, wk, table, pos)[0], lambda x: A.norm_rotary(k, x, wq, wk)[1],
             lambda x: A.rotary_append(x, k, k, table, pos, codes, codes.clone(), pos, **s),
             lambda x: A.paged_attention(x, codes, codes, bt, ctx, **s)]
    for f in calls:
        assert f(q) is not None
        with fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            f(fw.make_dual(q, torch.ones_like(q)))
    with fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError), match="forward"):
        A.norm_rotary(q, k, fw.make_dual(wq, wk), wk)
    for f in calls[2:]:
        with pytest.raises(RuntimeError, match="gradient"):
            f(q.clone().requires_grad_(True))
        with torch.no_grad():
            f(q.clone().requires_grad_(True))
    weights = {"q_weight": wq.requires_grad_(True), "k_weight": wk}
    with pytest.raises(RuntimeError, match="gradient"):
        A.rotary_append(q, k, k, table, pos, codes, codes.clone(), pos, **s, **weights)
    for f in (lambda t: A.norm_rotary(q, k, wq, wk, t, pos), lambda t: A.norm_rotary(q, k, wq.detach(), wk, t, pos)):
        with pytest.raises(RuntimeError, match="table"):
            f(table.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="gradient"):
        A.cached_rows(codes, codes, bt, ctx, torch.zeros(T + 1, dtype=torch.int32), 2, k_scale=scale.clone().requires_grad_(True),
                      v_scale=scale)
