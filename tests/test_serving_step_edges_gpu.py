"""Calls of the serving-step operators at the edges of what their documentation allows."""
import numpy as np
import pytest
import torch

from helpers import EPS, dev, to_np
from oracle import serving as S
from test_serving_step_gpu import BF, F32, FP, _check_logprobs, _i32, _logits
from test_serving_step_modules_gpu import BS, D, HIDDEN, NKV, _layers

from mindformers_amd import ops
from mindformers_amd.modules import AdapterBank, AdapterLinear, ColumnParallelLinear, Linear, RotaryPositions, WeightQuantLinearCell
from mindformers_amd.runner import DecodeStackRunner

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ log probabilities
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("v", [1501, 5003, 32003, 70003])
def test_logprobs_of_many_infinite_logits(dtype, v):
    """+inf counts as the largest float32, which is no value of the 16-bit types and lies above all of theirs: rows of it alone, more of it
    than a workgroup ranks at a time, a few beside as many of the type's own largest value, one row a workgroup and in pieces."""
    inf, most = float("inf"), torch.finfo(dtype).max
    gen = torch.Generator().manual_seed(v)
    x = torch.randn(13, v, generator=gen)
    some = torch.randperm(v, generator=gen)
    x[0] = inf
    x[1, some[:513]] = inf
    x[2, some[:min(3000, v - 1)]] = inf
    x[3, ::2] = inf
    x[4, some[:512]] = inf
    x[5, some[:1000]] = most
    x[5, some[1000:1007]] = inf
    x[6, :1000] = most                                        # the infinite ones behind all of them
    x[6, -3:] = inf
    x[7] = most
    x[7, 1::2] = inf
    x[8] = most
    x[9] = -inf
    x[9, 1:v - 1] = inf
    x[10, some[:700]] = inf
    x[10, some[700:1400]] = float("nan")
    x[11, :600] = -inf
    x[11, 600:601] = inf
    x[12, -600:] = inf
    x = x.to(dtype).cuda()
    for n in (1, 20, 64):
        for tokens in (np.arange(13) * (v // 13), np.r_[v - 1, some[:12].numpy()], np.r_[1, some[990:1002].numpy()]):
            _check_logprobs(x, tokens, n)
    wide = torch.full((3, v + 3), inf, dtype=dtype, device="cuda")
    wide[1, 2::2] = most
    wide[2, :700] = most
    for first in (1, 3):
        _check_logprobs(wide[:, first:first + v - 1], np.array([0, 5, v - 2]), 20)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("v", [65536, 98304, 131072])
def test_logprobs_of_rows_that_end_where_a_piece_begins(dtype, v):
    """The last workgroup of an aligned row has no column then, of others a few."""
    wide = _logits(3, v + 8, dtype, v)
    for first in (0, 1, 8):
        x = wide[:, first:first + v]
        for n in (0, 5, 64):
            _check_logprobs(x, np.array([0, v - 1, v // 2]), n)
    x[0] = float("-inf")
    x[1, :-3] = float("nan")
    x[2, -1] = float("inf")
    _check_logprobs(x, np.array([0, v - 2, v - 1]), 5)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("t,v", [(40, 32000), (31, 47603), (400, 151643)])
def test_sums_of_many_equal_small_terms_beside_a_large_one(dtype, t, v):
    """Each lane begins at 0, goes on with logits of one low value, and one meets a peak: thousands of like terms of a rounding's size beside a
    sum, whose errors all go one way.  Against the sums over the three values in float64; the tolerance is that of the other rows."""
    low = torch.linspace(-10.0, -5.0, t).to(dtype)
    peak = torch.linspace(7.9, 4.0, t).to(dtype)
    x = low[:, None].repeat(1, v)
    x[:, :4096:4] = 0.0
    x[:, 7003] = peak
    counts, values = np.array([[v - 1025, 1024, 1]]), np.stack([to_np(low), np.zeros(t), to_np(peak)], 1).astype(np.float64)
    mass = counts * np.exp(values)
    lp = values - np.log(mass.sum(axis=1, keepdims=True))
    entropy = -(mass / mass.sum(axis=1, keepdims=True) * lp).sum(axis=1)
    got = ops.token_logprobs(x.cuda(), _i32([7003] * t), n_top=1)
    for a, b in ((got.logprobs, lp[:, 2]), (got.top_logprobs[:, 0], lp[:, 2]), (got.entropy, entropy)):
        err = np.abs(to_np(a) - b)
        assert (err <= 4e-6 + 4 * 2.0 ** -24 * np.abs(b)).all(), err.max()


# ------------------------------------------------------------------------------------------------ the cells
@pytest.mark.parametrize("kind,dtype,x_dtype", [("float", FP, F32), ("float", BF, F32), ("parallel", BF, F32), ("parallel", FP, BF), ("w8", FP, BF),
                                                ("w8", BF, F32)])
def test_adapters_beside_a_cell_whose_rows_are_of_another_type(kind, dtype, x_dtype):
    """The cell's own output, to the bit where a row has no adapter, plus the adapters' part, rounded to the bank's type (the cell's, where the
    output is of it) and once more to the output's."""
    rng = np.random.default_rng(2)
    k, n = 128, 96
    if kind == "float":
        layer = Linear(k, n, has_bias=True, compute_dtype=dtype)
    elif kind == "parallel":
        layer = ColumnParallelLinear(k, n, compute_dtype=dtype)
    else:
        layer = WeightQuantLinearCell(k, n, compute_dtype=dtype).quantize_from_float(torch.randn(n, k))
    bank = AdapterBank(3, k, n, 8, dtype)
    bank.load(2, torch.from_numpy(rng.normal(size=(5, k)) / 16).cuda(), torch.from_numpy(rng.normal(size=(n, 5))).cuda(), scale=1.5)
    x, ids = dev(rng.normal(size=(4, 5, k)), x_dtype), rng.integers(-1, 3, 20)
    plain = layer(x)
    got = AdapterLinear(layer, bank)(x, ops.adapter_rows(_i32(ids), 3))
    assert got.dtype == plain.dtype and got.shape == plain.shape
    bare = torch.from_numpy(ids != 2).cuda().view(4, 5)
    assert torch.equal(got[bare], plain[bare])
    delta, mag = S.adapter_linear(to_np(x.to(dtype)).reshape(20, k), to_np(bank.lora_a), to_np(bank.lora_b), ids, np.zeros((20, n)), (n,),
                                  to_np(bank.ranks), to_np(bank.scales))
    want = to_np(plain).reshape(20, n) + delta
    # half a step of the adapters' part and of the output; the second product's operand and the float32 sums as in the product's own test
    tol = EPS[dtype] * np.abs(delta) + EPS.get(plain.dtype, 2.0 ** -24) * np.abs(want) + 2.0 ** -14 * mag + 2.0 ** -25
    assert (np.abs(to_np(got).reshape(20, n) - want) <= tol).all()


# ------------------------------------------------------------------------------------------------ the layer and the runner
@pytest.mark.parametrize("banks", [(), ("wo", "fc2")])
def test_a_w8a8_layer_takes_the_quantised_norm_it_is_handed(banks):
    """The norm of other rows than x, so that it shows: as a tensor and quantised, the same bits."""
    layer, = _layers(1, banks, act_quant=True)
    x, y = (torch.randn(4, HIDDEN, device="cuda").to(BF) for _ in range(2))
    kc, vc = (torch.randn(4, BS, NKV, D, device="cuda").to(BF) for _ in range(2))
    args = (_i32([[0], [1], [2], [3]]), _i32([3, 16, 1, 9]), _i32([2, 31, 32, 56]), None, None)
    view = dict(rotary=(_i32([2, 15, 0, 8]), RotaryPositions(D, interleaved=True)))
    if banks:
        view["adapters"] = ops.adapter_rows(_i32([0, 1, -1, 3]), 5)

    def step(normed):
        return layer(x, kc.clone(), vc.clone(), *args, normed=normed, **view)

    whole = step(ops.rms_norm(y, layer.attn_norm, layer.eps))
    assert torch.equal(step(ops.rms_norm_dynamic_quant(y, layer.attn_norm, layer.eps, layer.qkv_smooth, tiled=True)), whole)
    assert torch.equal(step(ops.rms_norm(x, layer.attn_norm, layer.eps)), step(None)) and not torch.equal(step(None), whole)


@pytest.mark.parametrize("banks,norms", [((), 2), (("wo",), 2), (("qkv", "fc1"), 0)])
def test_a_runner_of_w8a8_layers_makes_each_norm_once(banks, norms, monkeypatch):
    """Quantised where the layer takes it so, one a layer; none where adapters beside its first projection read the norm itself."""
    layers = _layers(2, banks, act_quant=True)
    rot = RotaryPositions(D, rotary_percent=0.5)
    run = DecodeStackRunner(layers, npu_mem_size=0.002, cpu_mem_size=0, block_size=BS, rotary=rot)
    x = torch.randn(3, HIDDEN, device="cuda").to(BF)
    lens, tables, slots = _i32([1, 1, 1]), _i32([[0], [1], [2]]), _i32([0, BS, 2 * BS])
    ids = _i32([0, -1, 3]) if banks else None
    calls, real = {}, {n: getattr(ops, n) for n in ("rms_norm", "rms_norm_dynamic_quant")}
    for name, fn in real.items():
        monkeypatch.setattr(ops, name, lambda *a, _n=name, _f=fn, **kw: (calls.__setitem__(_n, calls.get(_n, 0) + 1), _f(*a, **kw))[1])
    got = run.decode(x, lens, tables, slots, adapter_ids=ids)
    assert calls.get("rms_norm_dynamic_quant", 0) == norms and calls["rms_norm"] == 4 - norms      # the second norm of each layer with them
    rows = None if ids is None else ops.adapter_rows(ids, 5)
    h = x
    for i, layer in enumerate(layers):
        caches = [torch.zeros_like(run.key_cache[i]) for _ in range(2)]
        h = layer(h, *caches, tables, lens, slots, None, None, adapters=rows, rotary=(lens - 1, rot))
    assert torch.equal(got, h)
