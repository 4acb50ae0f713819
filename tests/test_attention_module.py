"""QuantizedAttention and its cache: what they do on the host.  No GPU."""
import copy

import pytest
import torch
import torch.nn as nn

from distributed_gptq_amd.models import attention as A


def module(table=None):
    return A.QuantizedAttention(nn.Linear(8, 8), nn.Linear(8, 8), 4, 2, 8, table)


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to(torch.bfloat16),
                                  lambda m: m.double(), lambda m: m.half().float()])
def test_casts_leave_the_table(cast):
    """The rotary table stays float32, bit for bit, when the module or one that
    holds it is cast; it is found among the module's buffers and follows its
    device."""
    table = A.rotary_table(8, 100, device="cpu")
    for wrap in (lambda m: m, lambda m: nn.Sequential(nn.Linear(8, 8), m)):
        m = wrap(module(table.clone()))
        m = copy.deepcopy(cast(m))
        inner = m if isinstance(m, A.QuantizedAttention) else m[1]
        assert inner.table.dtype == torch.float32 and torch.equal(inner.table, table)
        assert any(b is inner.table for b in m.buffers())
    assert cast(module()).table is None
    assert cast(module(table)).qkv.weight.dtype == cast(nn.Linear(8, 8)).weight.dtype


def test_device_moves_take_the_table():
    m = module(A.rotary_table(8, 100, device="cpu")).to("meta", torch.float16)
    assert m.table.is_meta and m.table.dtype == torch.float32 and m.qkv.weight.dtype == torch.float16


@pytest.mark.parametrize("scaling", [{"factor": 4.0}, {"rope_type": "linear", "factor": 4.0},
                                     {"type": None, "factor": 4.0}])
def test_scaling_without_a_type_raises(scaling):
    """It was taken for no scaling at all."""
    with pytest.raises(ValueError, match="scaling"):
        A.rotary_frequencies(8, 1e4, scaling)
    with pytest.raises(ValueError, match="scaling"):
        A.rotary_table(8, 4, scaling=scaling, device="cpu")


def test_no_scaling():
    want = A.rotary_frequencies(8, 1e4)[0]
    for scaling in (None, {}):
        assert torch.equal(A.rotary_frequencies(8, 1e4, scaling)[0], want)


def test_positions_past_the_table_raise(monkeypatch):
    """Where the host knows them: a step's longest context, one sequence's
    length.  (They would all be turned by the table's last angles.)"""
    called = []

    def op(name, *args):
        called.append(name)
        return torch.zeros(args[0].shape[0], 4, 8) if name != "rotary" else args[:2]
    monkeypatch.setattr(A, "_op", op)

    class Heads(nn.Module):
        def forward(self, x):
            return x.new_zeros(len(x), 32), x.new_zeros(len(x), 16), x.new_zeros(len(x), 16)
    for table, most in ((A.rotary_table(8, 20, device="cpu"), 20), (None, 1 << 30)):
        m = A.QuantizedAttention(Heads(), nn.Identity(), 4, 2, 8, table)
        cache = A.PagedKVCache(8, 8, 2, 8, device="cpu")
        for new, total in ((15, 15), (5, 20), (1, 21)):
            batch = cache.extend(["a"], [new])
            if total > most:
                called.clear()
                with pytest.raises(ValueError, match="20"):
                    m.step(torch.zeros(new, 8), cache, batch)
                assert not called
            else:
                assert m.step(torch.zeros(new, 8), cache, batch).shape == (new, 32)
        assert m(torch.zeros(20, 8)).shape == (20, 32)
        if table is not None:
            with pytest.raises(ValueError, match="20"):
                m(torch.zeros(21, 8))
        # offsets or positions of the caller's are on the GPU: the operator clamps
        assert m(torch.zeros(21, 8), positions=torch.zeros(21, dtype=torch.int32)).shape == (21, 32)
        assert m(torch.zeros(21, 8), torch.tensor([0, 11, 21])).shape == (21, 32)


def test_a_cache_of_more_places_than_slots_count_raises():
    """Slots are 32-bit: places from 2^31 on could not be named (extend failed
    there, after it had given the pages away)."""
    A.PagedKVCache(1024, 2 ** 21, 1, 8, device="meta")
    with pytest.raises(ValueError, match="2\\^31"):
        A.PagedKVCache(1025, 2 ** 21, 1, 8, device="meta")
