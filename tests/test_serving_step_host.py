"""Refusals of the serving-step operators, by the wrappers and by the library (host checks: nothing is launched)."""
import ctypes

import pytest
import torch

from mindformers_amd import _lib, ops

BF, FP, I32, F32, F64 = torch.bfloat16, torch.float16, torch.int32, torch.float32, torch.float64


def _refused(call, *args, **kw):
    with pytest.raises(ValueError):
        call(*args, **kw)


def test_tensors_that_are_not_on_the_gpu_are_refused():
    z = torch.zeros
    _refused(ops.rotary_embedding, z(2, 64, dtype=BF), None, z(2, dtype=I32), z(32, dtype=F64), 64)
    _refused(ops.token_logprobs, z(2, 64), z(2, dtype=I32))
    _refused(ops.adapter_rows, z(2, dtype=I32), 2)
    rows = ops.AdapterRows(z(16, dtype=I32), 2, 1, 16)
    _refused(ops.adapter_linear, z(2, 8, dtype=BF), z(1, 8, 8, dtype=BF), z(1, 8, 8, dtype=BF), rows, z(2, 8, dtype=BF))


def _rc(name, *args):
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    return rc, lib.mf_last_error().decode() if rc else ""


#: an address that no check reads through
P = ctypes.c_void_p(0x1000)


def _rotary(**over):
    a = dict(q_out=P, k_out=P, q=P, k=P, v=None, kc=None, vc=None, pos=P, inv=P, slots=None, t=4, h=2, kv=1, d=64, pairs=32, offset=0,
             near=0, scale=1.0, num=0, qs=0, ks=0, vs=0, qos=0, kos=0, dtype=0, stream=None)
    a.update(over)
    return _rc("mf_rotary_embedding", *a.values())


@pytest.mark.parametrize("over", [dict(dtype=2), dict(t=-1), dict(t=1 << 24), dict(h=0), dict(pairs=0), dict(pairs=33), dict(offset=-1),
                                  dict(offset=2), dict(d=2048, pairs=1024), dict(q=None), dict(q_out=None), dict(pos=None), dict(inv=None),
                                  dict(k=None), dict(kv=0), dict(kc=P), dict(kc=P, vc=P, v=P, slots=P), dict(qs=127), dict(kos=3),
                                  dict(inv=ctypes.c_void_p(0x1004)), dict(q=ctypes.c_void_p(0x1001))])
def test_the_library_refuses_rotary(over):
    rc, msg = _rotary(**over)
    assert rc == 1 and msg.startswith("rotary_embedding")


def _logprobs(**over):
    a = dict(lp=P, ranks=P, entropy=P, top=P, top_lp=P, logits=P, stride=0, tokens=P, rows=4, vocab=100, n=3, dtype=0, ws=None, bytes=0,
             stream=None)
    a.update(over)
    return _rc("mf_token_logprobs", *a.values())


@pytest.mark.parametrize("over", [dict(dtype=3), dict(rows=-1), dict(rows=1 << 24), dict(vocab=0), dict(vocab=0x7c000001), dict(n=-1),
                                  dict(n=65), dict(n=5, vocab=4), dict(stride=99), dict(lp=None), dict(tokens=None), dict(top=None),
                                  dict(logits=ctypes.c_void_p(0x1001)), dict(logits=ctypes.c_void_p(0x1002), dtype=2),
                                  dict(vocab=100000), dict(vocab=100000, ws=P, bytes=16)])
def test_the_library_refuses_logprobs(over):
    rc, msg = _logprobs(**over)
    assert rc == 1 and msg.startswith("token_logprobs")


@pytest.mark.parametrize("args", [(P, P, 4, 1025, 16), (P, P, -1, 4, 16), (P, P, (1 << 20) + 1, 4, 16), (P, P, 4, 4, 32), (None, P, 4, 4, 16),
                                  (P, None, 4, 4, 16), (ctypes.c_void_p(0x1008), P, 4, 4, 16)])
def test_the_library_refuses_rows_by_adapter(args):
    rc, msg = _rc("mf_adapter_rows", *args, None)
    assert rc == 1 and msg.startswith("adapter_rows")


def _adapter(widths=(64,), **over):
    a = dict(out=P, x=P, a=P, b=P, base=P, plan=P, ranks=None, scales=None, widths=(ctypes.c_int32 * len(widths))(*widths),
             slices=len(widths), t=4, n=2, tile=16, k=64, r=16, xs=0, bs=0, os=0, dtype=0, ws=P, bytes=1 << 30, stream=None)
    a.update(over)
    return _rc("mf_adapter_linear", *a.values())


@pytest.mark.parametrize("over", [dict(dtype=2), dict(t=-1), dict(n=0), dict(n=1025), dict(tile=8), dict(k=12), dict(k=0), dict(r=12),
                                  dict(r=136), dict(widths=(0,)), dict(widths=(8,) * 9), dict(widths=(1 << 24, 1)), dict(xs=63), dict(xs=68),
                                  dict(bs=63), dict(os=128), dict(out=None), dict(x=None), dict(a=None), dict(base=None), dict(plan=None),
                                  dict(x=ctypes.c_void_p(0x1008)), dict(a=ctypes.c_void_p(0x1002)), dict(base=ctypes.c_void_p(0x1001)),
                                  dict(ws=None), dict(bytes=64), dict(ws=ctypes.c_void_p(0x1008))])
def test_the_library_refuses_adapters(over):
    rc, msg = _adapter(**over)
    assert rc == 1 and msg.startswith("adapter_linear")


def test_sizes_of_plans_and_workspaces():
    lib = _lib.load()
    assert lib.mf_adapter_rows_ints(0, 4, 16) == 0 and lib.mf_adapter_rows_ints(4, 4, 8) == 0
    assert lib.mf_adapter_rows_ints(5, 3, 16) == 8 + 4 * 4                # at most a tile a group of rows
    assert lib.mf_adapter_workspace_bytes(4, 2, 16, 64, 1, 136) == 0
    assert lib.mf_token_logprobs_workspace_bytes(5000, 1000, 64, 0) == 0  # a workgroup a row
    assert lib.mf_token_logprobs_workspace_bytes(1, 152064, 65, 0) == 0


# ------------------------------------------------------------------------------------------------ modules, on the CPU
def test_a_bank_takes_and_refuses_adapters():
    from mindformers_amd.modules import AdapterBank
    bank = AdapterBank(3, 16, (8, 24), 8, device="cpu")
    a, b = [torch.ones(4, 16), torch.full((2, 16), 2.0)], [torch.ones(8, 4), torch.full((24, 2), 3.0)]
    bank.load(1, a, b, scale=0.5)
    assert bank.ranks.tolist() == [0, 4, 0] and bank.scales[1] == 0.5
    assert (bank.lora_a[1, 0, :4] == 1).all() and (bank.lora_a[1, 1, :2] == 2).all() and (bank.lora_a[1, 1, 2:] == 0).all()
    assert (bank.lora_b[1, :8, :4] == 1).all() and (bank.lora_b[1, 8:, :2] == 3).all() and (bank.lora_b[1, 8:, 2:] == 0).all()
    bank.load(1, [None, a[1]], [None, b[1]])                  # what was there before leaves
    assert (bank.lora_a[1, 0] == 0).all() and (bank.lora_b[1, :8] == 0).all() and bank.ranks[1] == 2
    for slot, x, y in ((3, a, b), (-1, a, b), (0, a[:1], b[:1]), (0, [a[0], None], b), (0, [torch.ones(9, 16), a[1]], [torch.ones(8, 9), b[1]]),
                       (0, [torch.ones(4, 15), a[1]], b), (0, a, [torch.ones(8, 3), b[1]])):
        with pytest.raises(ValueError):
            bank.load(slot, x, y)
    assert bank.unload(1).ranks.tolist() == [0, 0, 0]
    for args in ((0, 16, 8, 8), (1025, 16, 8, 8), (2, 12, 8, 8), (2, 16, 8, 12), (2, 16, 8, 136), (2, 16, (), 8), (2, 16, (8, 0), 8), (2, 16, (8,) * 9, 8)):
        with pytest.raises(ValueError):
            AdapterBank(*args, device="cpu")
    with pytest.raises(TypeError):
        AdapterBank(2, 16, 8, 8, dtype=torch.float32, device="cpu")


def test_a_layer_and_a_cell_refuse_banks_that_do_not_fit():
    from mindformers_amd.decode_layer import QuantDecodeLayer
    from mindformers_amd.modules import AdapterBank, AdapterLinear, Linear
    layer = QuantDecodeLayer(64, 4, 2, 16, 128, device="cpu")
    fits = AdapterBank(2, 64, (64, 32, 32), 8, device="cpu")
    layer.set_adapters({"qkv": fits})
    assert layer.banks["qkv"] is fits and any(k.startswith("banks.qkv") for k in layer.state_dict())
    for banks in ({"gate": fits}, {"wo": fits}, {"qkv": AdapterBank(2, 64, 128, 8, FP, device="cpu")},
                  {"qkv": fits, "wo": AdapterBank(3, 64, 64, 8, device="cpu")}):
        with pytest.raises(ValueError):
            layer.set_adapters(banks)
    layer.set_adapters({})
    assert not layer.banks
    with pytest.raises(ValueError):
        AdapterLinear(Linear(64, 128, device="cpu"), AdapterBank(2, 64, 64, 8, device="cpu"))
    with pytest.raises(NotImplementedError):
        AdapterLinear(Linear(64, 64, activation="silu", device="cpu"), AdapterBank(2, 64, 64, 8, device="cpu"))


def test_rotary_positions_have_the_frequencies_of_the_tables():
    """Against the tables of the float32 classes: the same formulas, so cosines at the first positions agree to float32."""
    import numpy as np
    from mindformers_amd.modules import FreqsMgr, Llama3RotaryEmbedding, RotaryEmbedding, RotaryPositions, YaRNScalingRotaryEmbedding
    d, pos = 32, np.arange(40)

    def near(rot, cos):
        got = np.cos(pos[:, None] * rot.inv_freq.numpy()) * rot.scale
        assert np.abs(got - cos[:40, :d // 2].numpy()).max() < 2e-5

    common = dict(rotary_cos_format=2, rotary_dtype=F32, device="cpu")
    near(RotaryPositions(d, device="cpu"), RotaryEmbedding(d, max_position_embeddings=64, **common).cos_cache)
    near(RotaryPositions(d, base=5e5, device="cpu"), RotaryEmbedding(d, rotary_base=500000, max_position_embeddings=64, **common).cos_cache)
    llama3 = dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=64)
    near(RotaryPositions(d, scaling="llama3", scaling_config=llama3, device="cpu"),
         Llama3RotaryEmbedding(d, max_position_embeddings=64, scaling_factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, orig_max_position=64,
                               **common).cos_cache)
    yarn = dict(factor=4.0, original_max_position_embeddings=64, beta_fast=32, beta_slow=1, mscale=1.0, mscale_all_dim=0.5)
    near(RotaryPositions(d, scaling="YARN", scaling_config=yarn, device="cpu"),
         YaRNScalingRotaryEmbedding(d, scaling_factor=4.0, original_max_position_embeddings=64, mscale=1.0, mscale_all_dim=0.5, **common).cos_cache)
    near(RotaryPositions(d, scaling="linear", scaling_config=dict(factor=2.0), device="cpu"),
         FreqsMgr(d, max_position_embedding=64, rotary_dtype=F32, extend_method="LINEAR", scaling_factor=dict(factor=2.0), device="cpu").freqs_cos)
    near(RotaryPositions(d, scaling="ntk", scaling_config=dict(factor=2.0), device="cpu"),
         FreqsMgr(d, max_position_embedding=64, rotary_dtype=F32, extend_method="NTK", scaling_factor=2.0, device="cpu").freqs_cos)
    part = RotaryPositions(128, rotary_percent=0.25, interleaved=True, offset=96, device="cpu")
    assert part.inv_freq.shape == (16,) and part.inv_freq.dtype == F64 and not part.state_dict()
    for args, kw in (((32,), dict(rotary_percent=0.1)), ((32,), dict(offset=2)), ((32,), dict(scaling="su")), ((32,), dict(scaling="linear")),
                     ((32,), dict(scaling="linear", scaling_config=dict(factor=2, beta_fast=1))), ((32,), dict(scaling_config=dict(factor=2.0)))):
        with pytest.raises(ValueError):
            RotaryPositions(*args, device="cpu", **kw)
    with pytest.raises(TypeError):
        RotaryPositions(32, device="cpu").half()
