"""Calls of the serving-step operators and modules at the edges of what their documentation allows, on the CPU (nothing is launched)."""
import ctypes

import pytest
import torch

from test_serving_step_host import _rotary

from mindformers_amd.modules import AdapterBank, RotaryPositions

BF, FP, I32, F32, F64 = torch.bfloat16, torch.float16, torch.int32, torch.float32, torch.float64


def _bank(dtype=BF):
    return AdapterBank(2, 16, (8, 24), 8, dtype, device="cpu").load(1, [torch.ones(4, 16), None], [torch.ones(8, 4), None], scale=0.3)


@pytest.mark.parametrize("convert", [lambda m: m.half(), lambda m: m.to(FP), lambda m: m.to("cpu", FP), lambda m: torch.nn.Sequential(m).half()[0]])
def test_a_bank_changes_its_matrices_type(convert):
    """The scales stay float32, as the products take them, and not by way of 16 bits; the ranks whole numbers."""
    bank = convert(_bank())
    assert bank.dtype == bank.lora_a.dtype == bank.lora_b.dtype == FP
    assert bank.scales.dtype == F32 and bank.scales[1] == torch.tensor(0.3) and bank.ranks.dtype == I32 and bank.ranks.tolist() == [0, 4]
    assert dict(bank.named_buffers())["scales"] is bank.scales
    bank.load(0, [torch.ones(4, 16), None], [torch.ones(8, 4), None], scale=0.7)
    assert bank.scales[0] == torch.tensor(0.7) and bank.bfloat16().dtype == BF and bank.scales[0] == torch.tensor(0.7)


@pytest.mark.parametrize("convert", [lambda m: m.float(), lambda m: m.double(), lambda m: m.to(F64)])
def test_a_bank_refuses_other_types_and_stays_as_it_was(convert):
    bank = _bank()
    before = {name: t.clone() for name, t in bank.named_buffers()}
    with pytest.raises(TypeError):
        convert(bank)
    assert bank.dtype == BF and all(t.dtype == before[n].dtype and torch.equal(t, before[n]) for n, t in bank.named_buffers())
    assert bank.to("cpu") is bank and bank.dtype == BF


def test_a_slot_takes_its_own_matrices_again():
    """With another scale, or its slices in another order."""
    bank = AdapterBank(2, 16, (8, 8), 8, device="cpu")
    gen = torch.Generator().manual_seed(1)
    a, b = [torch.randn(r, 16, generator=gen).to(BF) for r in (4, 6)], [torch.randn(8, r, generator=gen).to(BF) for r in (4, 6)]
    bank.load(1, a, b)
    own = [bank.lora_a[1, 0, :4], bank.lora_a[1, 1, :6]], [bank.lora_b[1, :8, :4], bank.lora_b[1, 8:, :6]]
    bank.load(1, *own, scale=0.5)
    assert all(torch.equal(x, y) for x, y in zip(own[0] + own[1], a + b)) and bank.scales[1] == 0.5
    bank.load(1, own[0][::-1], own[1][::-1])
    assert torch.equal(bank.lora_a[1, 0, :6], a[1]) and torch.equal(bank.lora_a[1, 1, :4], a[0]) and (bank.lora_a[1, 1, 4:] == 0).all()
    assert torch.equal(bank.lora_b[1, :8, :6], b[1]) and torch.equal(bank.lora_b[1, 8:, :4], b[0]) and (bank.lora_b[1, 8:, 4:] == 0).all()


@pytest.mark.parametrize("convert", [lambda m: m.half(), lambda m: m.float(), lambda m: m.to("cpu", BF)])
def test_rotary_positions_refuse_other_types_and_stay_as_they_were(convert):
    rot = RotaryPositions(32, base=5e5, device="cpu")
    before = rot.inv_freq.clone()
    with pytest.raises(TypeError):
        convert(rot)
    assert rot.inv_freq.dtype == F64 and torch.equal(rot.inv_freq, before)
    assert rot.to("cpu") is rot and rot.double() is rot and torch.equal(rot.inv_freq, before)


def _at(i):
    """Addresses that no check reads through."""
    return ctypes.c_void_p(0x10000 * (i + 1))


@pytest.mark.parametrize("over", [dict(k=_at(0), k_out=_at(0)), dict(k=_at(0), k_out=None, **{n: _at(4 + i) for i, n in enumerate(("kc", "vc", "v", "slots"))}),
                                  dict(v=_at(1), kc=_at(5), vc=_at(6), slots=_at(7), num=64), dict(v=_at(0), kc=_at(5), vc=_at(6), slots=_at(7), num=64),
                                  dict(q_out=_at(1), k_out=_at(4)), dict(q_out=_at(4), k_out=_at(0)), dict(q_out=_at(4), k_out=_at(4)), dict(qs=128, qos=192),
                                  dict(ks=64, kos=128)])
def test_rotary_positions_refuse_shared_memory_that_is_written(over):
    """In place the query, the key and the value are read while the others are written; an output with its input's address has its rows."""
    rc, msg = _rotary(**{**dict(q_out=_at(0), q=_at(0), k_out=_at(1), k=_at(1), pos=_at(2), inv=_at(3), num=64), **over})
    assert rc == 1 and msg.startswith("rotary_embedding") and ("share" in msg or "distance" in msg), msg
