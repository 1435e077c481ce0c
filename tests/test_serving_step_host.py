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
