"""Adapters and rotary positions in the cells, the layer and the runner, and a run of the serving step's operators together."""
import numpy as np
import pytest
import torch

import oracle as O
import oracle.layer as OL
from helpers import EPS, dev, rounded, to_np
from oracle import serving as S

from mindformers_amd import ops
from mindformers_amd.decode_layer import QuantDecodeLayer
from mindformers_amd.modules import (AdapterBank, AdapterLinear, AllQuantLinearInferCell, BlockTables, Linear, RotaryPositions,
                                     WeightQuantLinearCell)
from mindformers_amd.runner import DecodeStackRunner

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16
HIDDEN, NH, NKV, D, FFN, BS = 512, 8, 2, 64, 1024, 16
SHAPES = {"qkv": (HIDDEN, (NH * D, NKV * D, NKV * D)), "wo": (NH * D, (HIDDEN,)), "fc1": (HIDDEN, (FFN, FFN)), "fc2": (FFN, (HIDDEN,))}


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


def _bank(rng, name, n=5, rank=16, std=1.0, dtype=BF):
    """A bank with adapters of ranks 16, 3, 8 in slots 0, 1 and 3 (slot 1: first slice only), and its arrays."""
    k, widths = SHAPES[name]
    bank = AdapterBank(n, k, widths, rank, dtype)
    for slot, r in ((0, 16), (1, 3), (3, 8)):
        a = [torch.from_numpy(rng.normal(size=(r, k)) * std / np.sqrt(k)).cuda() for _ in widths]
        b = [torch.from_numpy(rng.normal(size=(w, r)) / np.sqrt(r)).cuda() for w in widths]
        if slot == 1:
            a[1:], b[1:] = [None] * (len(a) - 1), [None] * (len(b) - 1)
        bank.load(slot, a, b, scale=0.5 + slot / 4)
    return bank


def _delta(bank, x, ids):
    out, _ = S.adapter_linear(x, to_np(bank.lora_a), to_np(bank.lora_b), ids, np.zeros((len(ids), bank.out_features)), bank.widths,
                              to_np(bank.ranks), to_np(bank.scales))
    return out


def _layers(n, banks=(), act_quant=False, seed=7):
    from mindformers_amd import synthetic
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    got = [synthetic.fill_layer(QuantDecodeLayer(HIDDEN, NH, NKV, D, FFN, 1e-5, BF, act_quant), gen) for _ in range(n)]
    for layer in got:
        layer.set_adapters({name: _bank(rng, name) for name in banks})
    return got


# ------------------------------------------------------------------------------------------------ cells
@pytest.mark.parametrize("cell", ["float", "w8", "w4", "a8"])
def test_adapters_beside_a_linear_cell(cell):
    """The cell's own output plus the adapters', rounded once more."""
    rng = np.random.default_rng(1)
    k, n, dtype = 256, 192, FP
    if cell == "float":
        layer = Linear(k, n, has_bias=True, compute_dtype=dtype, param_init_type=dtype)
    elif cell == "a8":
        layer = AllQuantLinearInferCell(k, n, compute_dtype=dtype).quantize_from_float(torch.randn(n, k)).prepare()
    else:
        layer = WeightQuantLinearCell(k, n, compute_dtype=dtype, weight_bits=8 if cell == "w8" else 4).quantize_from_float(torch.randn(n, k))
    bank = AdapterBank(3, k, n, 8, dtype)
    bank.load(2, torch.from_numpy(rng.normal(size=(5, k)) / 16).cuda(), torch.from_numpy(rng.normal(size=(n, 5))).cuda(), scale=1.5)
    both = AdapterLinear(layer, bank)
    x = dev(rounded(rng.normal(size=(20, k)), dtype), dtype)
    ids = rng.integers(-1, 3, 20)
    plain = layer(x)
    got = both(x, ops.adapter_rows(_i32(ids), 3))
    want = to_np(plain) + _delta(bank, to_np(x), ids)
    assert (np.abs(to_np(got) - want) <= EPS[dtype] * np.abs(want) + 2e-5 * np.abs(want).max()).all()
    assert torch.equal(got[torch.from_numpy(ids != 2).cuda()], plain[torch.from_numpy(ids != 2).cuda()])
    assert torch.equal(both(x), plain)
    bank.unload(2)
    assert torch.equal(both(x, ops.adapter_rows(_i32(ids), 3)), plain)


# ------------------------------------------------------------------------------------------------ the layer
@pytest.mark.parametrize("act_quant", [False, True])
@pytest.mark.parametrize("banks", [("qkv",), ("wo", "fc2"), ("fc1",), ("qkv", "wo", "fc1", "fc2")])
@pytest.mark.parametrize("prefill", [False, True])
def test_a_layer_whose_rows_have_no_adapter_is_the_layer(act_quant, banks, prefill):
    """Rows without an adapter, steps without any, and the layer before it had banks: the same bits."""
    rng = np.random.default_rng(3)
    layer, = _layers(1, act_quant=act_quant)
    t = 24 if prefill else 5
    kc, vc = (torch.randn(8, BS, NKV, D, device="cuda").to(BF) for _ in range(2))
    x = torch.randn(t, HIDDEN, device="cuda").to(BF)
    ang = torch.randn(t, D // 2, device="cuda")
    cos, sin = (torch.cat([f(ang)] * 2, 1).to(BF) for f in (torch.cos, torch.sin))
    if prefill:
        args = (_i32([[0, 1], [2, -1]]), _i32([17, 7]), _i32(list(range(17)) + list(range(32, 39))), cos, sin, _i32([0, 17, 24]))
    else:
        args = (_i32([[i, -1] for i in range(5)]), _i32([3, 9, 16, 1, 12]), _i32([i * BS + n - 1 for i, n in enumerate((3, 9, 16, 1, 12))]), cos, sin)
    want = layer(x, kc.clone(), vc.clone(), *args)
    layer.set_adapters({name: _bank(rng, name) for name in banks})
    empty = ops.adapter_rows(_i32([-1, 2] * (t // 2) + [4] * (t % 2)), 5)     # slots 2 and 4 are empty
    k2, v2 = kc.clone(), vc.clone()
    assert torch.equal(layer(x, k2, v2, *args, adapters=empty), want)
    assert torch.equal(layer(x, k2, v2, *args), want)
    some = layer(x, k2, v2, *args, adapters=ops.adapter_rows(_i32([0] * t), 5))
    assert not torch.equal(some, want) and torch.isfinite(some.float()).all()
    gamma = torch.rand(HIDDEN, device="cuda") + 0.5
    chain = (gamma, 1e-5, torch.rand(HIDDEN, device="cuda") + 0.5) if act_quant else (gamma, 1e-5)
    out, normed = layer(x, k2, v2, *args, adapters=ops.adapter_rows(_i32([0] * t), 5), next_norm=chain)
    assert torch.equal(out, some)
    if not act_quant:
        assert torch.equal(normed, ops.rms_norm(out, gamma, 1e-5))
    layer.set_adapters({})
    assert torch.equal(layer(x, k2, v2, *args), want)


def test_int8_caches_of_a_layer_with_adapters_and_rotary_positions():
    """The quantised cache of rotated keys: against the same layer on 16-bit caches, within the quantisation's step."""
    layer, = _layers(1, ("qkv",))
    scale = torch.full((2, NKV * D), 1 / 16, device="cuda")
    layer.set_kv_quant(scale)
    rot = RotaryPositions(D, rotary_percent=0.5, interleaved=True)
    x = torch.randn(4, HIDDEN, device="cuda").to(BF)
    pos, slots = _i32([5, 6, 0, 100]), _i32([3, 4, 40, 17])
    args = (_i32([[0], [0], [2], [1]]), _i32([1, 1, 1, 1]), slots, None, None)
    kc, vc = (torch.zeros(3, BS, NKV, D, dtype=torch.int8, device="cuda") for _ in range(2))
    k16, v16 = (torch.zeros(3, BS, NKV, D, dtype=BF, device="cuda") for _ in range(2))
    rows = ops.adapter_rows(_i32([0, 1, -1, 3]), 5)
    layer(x, kc, vc, *args, adapters=rows, rotary=(pos, rot))
    layer(x, k16, v16, *args, adapters=rows, rotary=(pos, rot))
    for q, full in ((kc, k16), (vc, v16)):
        want = torch.clamp(torch.round(full.double() * 16), -128, 127)
        assert torch.equal(q.double(), want)


# ------------------------------------------------------------------------------------------------ together
def _rope(pos):
    ang = np.asarray(pos, np.float64)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    emb = np.concatenate([ang, ang], -1).astype(np.float32)
    return rounded(np.cos(emb), BF), rounded(np.sin(emb), BF)


@pytest.mark.parametrize("layout", ["rows", "interleaved part", "yarn"])
def test_a_run_of_prompts_and_steps_with_adapters_and_log_probabilities(layout, monkeypatch):
    """Three requests, two with adapters: prompts, then four decode steps through a runner of two layers, against the oracle's layer with
    the adapters' products in its projections and rotary positions in the place of its own; then the log probabilities of the
    tokens a head picks.

    Tolerance of the hidden rows.  Between its input and its output a value of a layer is rounded 14 times on the device (norms 2,
    projections 4 and 4 more behind the adapters, rotation, probabilities, attention, activation 2) and 10 times by the oracle; a
    projection or a norm spreads the error of a rounding over the row, so that it comes in relative to the row's root mean square, not to
    the element.  A rounding of half a step (2^-8 of the value at most) is off by 2^-8 / sqrt(3) in the square mean at most, 48 of them
    in two layers by sqrt(48 / 3) 2^-8 = 4 x 2^-8: four of these deviations are 16 x 2^-8 of the row's root mean square, and five would be
    met once in 10^6 elements if every rounding were as far off as it can be (they are off by half of that on average)."""
    banks = ("qkv", "wo", "fc1", "fc2")
    layers = _layers(2, banks)
    rot = {"rows": None, "interleaved part": RotaryPositions(D, rotary_percent=0.5, interleaved=True, base=5e5),
           "yarn": RotaryPositions(D, scaling="yarn", scaling_config=dict(factor=8.0, original_max_position_embeddings=64))}[layout]
    run = DecodeStackRunner(layers, npu_mem_size=0.004, cpu_mem_size=0, block_size=BS, rotary=rot)
    rng = np.random.default_rng(5)
    prompt, ids, steps = np.array([37, 21, 5]), np.array([0, -1, 3]), 4
    total = prompt + steps
    xs = [rounded(rng.normal(size=(int(t), HIDDEN)), BF) for t in total]
    mgr = BlockTables(run.npu_num_blocks, BS, 128)
    mgr.init_cache_engine(3)
    tables, slots = mgr.assemble_pa_full_inputs(int(prompt.max()), prompt, [False] * 3)
    slots = slots.reshape(3, -1)
    slots = np.concatenate([slots[i, :n] for i, n in enumerate(prompt)])
    kcs = [np.zeros((run.npu_num_blocks, BS, NKV, D), np.float32) for _ in layers]
    vcs = [np.zeros_like(kcs[0]) for _ in layers]
    cfg = dict(n_head=NH, n_kv_head=NKV, head_dim=D, eps=1e-5)

    def want(x, lens, tb, sl, pos, row_ids, q_lens):
        cos, sin = _rope(pos)
        if rot is not None:
            monkeypatch.setattr(OL, "apply_rotary_half", lambda v, c, s, h: S.rotary(v, pos, to_np(rot.inv_freq), D, rot.interleaved, rot.scale))
        for i, layer in enumerate(layers):
            def lin(a, name):
                y = O.w8a16_linear(a, to_np(getattr(layer, name + "_w")), to_np(getattr(layer, name + "_s")))
                return y + _delta(layer.banks[name], a, row_ids)
            p = {"attn_norm": to_np(layer.attn_norm), "ffn_norm": to_np(layer.ffn_norm)}
            x = OL._decode_layer(x, p, cfg, kcs[i], vcs[i], tb, lens, sl, cos, sin, "bf16", lin, q_lens)
        return x

    def close(got, ref):
        tol = 16 * EPS[BF] * np.maximum(np.abs(ref), np.sqrt((ref ** 2).mean(axis=1, keepdims=True)))
        assert np.all(np.abs(to_np(got) - ref) <= tol), (np.abs(to_np(got) - ref) / tol).max()

    x0 = np.concatenate([x[:n] for x, n in zip(xs, prompt)])
    pos0, ids0 = np.concatenate([np.arange(n) for n in prompt]), np.repeat(ids, prompt)
    close(run.forward(dev(x0, BF), prompt, tables, slots, prefill=True, adapter_ids=ids), want(x0, prompt, tables, slots, pos0, ids0, prompt))
    head = torch.randn(HIDDEN, 3001, device="cuda") / 16
    lens = prompt.copy()
    for _ in range(steps):
        lens = lens + 1
        tables, slots = mgr.assemble_pa_inc_inputs(lens, [False] * 3)
        x = np.stack([xs[i][lens[i] - 1] for i in range(3)])
        hidden = run.forward(dev(x, BF), lens, tables, slots, prefill=False, adapter_ids=_i32(ids) if lens[0] % 2 else ids)
        close(hidden, want(x, lens, tables, slots, lens - 1, ids, None))
        logits = hidden.float() @ head
        got = ops.token_logprobs(logits, logits.argmax(1).int(), n_top=5)
        lp, rank, entropy, top, top_lp = S.token_logprobs(to_np(logits), to_np(logits).argmax(1), 5)
        assert np.array_equal(to_np(got.ranks), rank) and np.array_equal(to_np(got.top_tokens), top) and not rank.any()
        for a, b in ((got.logprobs, lp), (got.entropy, entropy), (got.top_logprobs, top_lp)):
            assert np.abs(to_np(a) - b).max() <= 4e-6
    again = run.decode(dev(x, BF), _i32(lens), _i32(tables), _i32(slots), adapter_ids=_i32(ids))
    assert torch.equal(again, hidden)
    with pytest.raises(ValueError):
        run.forward(dev(x, BF), lens, tables, slots, prefill=False, adapter_ids=[0, 1])
    with pytest.raises(ValueError):
        DecodeStackRunner(_layers(1), npu_mem_size=0.001, cpu_mem_size=0, block_size=BS).decode(
            dev(x, BF), _i32(lens), _i32(np.zeros((3, 1))), _i32(slots), adapter_ids=_i32(ids))


def test_chunked_prompts_with_adapters_are_the_whole_prompts():
    layers = _layers(2, ("qkv", "fc1"))
    rng = np.random.default_rng(8)
    total, ids = np.array([41, 30]), np.array([3, 0])
    x = dev(rounded(rng.normal(size=(71, HIDDEN)), BF), BF)
    rot = RotaryPositions(D, interleaved=True)
    whole, parts = (DecodeStackRunner(layers, npu_mem_size=0.002, cpu_mem_size=0, block_size=BS, rotary=rot) for _ in range(2))
    mgr = BlockTables(whole.npu_num_blocks, BS, 64)
    mgr.init_cache_engine(2)
    tables, slots = mgr.assemble_pa_full_inputs(41, total, [False] * 2)
    slots = slots.reshape(2, -1)
    slots = np.concatenate([slots[i, :n] for i, n in enumerate(total)])
    want = to_np(whole.forward(x, total, tables, slots, prefill=True, adapter_ids=ids))
    got, done, starts = np.zeros_like(want), np.zeros(2, np.int64), np.array([0, 41])
    while (done < total).any():
        step = np.minimum(16, total - done)
        rows = np.concatenate([np.arange(starts[i] + done[i], starts[i] + done[i] + step[i]) for i in range(2)])
        done = done + step
        got[rows] = to_np(parts.forward(x[torch.from_numpy(rows).cuda()], done, tables, slots[rows], prefill=False, q_seq_lens=step,
                                        adapter_ids=_i32(ids)))
    # both sides' roundings, of the same number (see the run above, 14 on each)
    tol = 16 * EPS[BF] * np.maximum(np.abs(want), np.sqrt((want ** 2).mean(axis=1, keepdims=True)))
    assert np.all(np.abs(got - want) <= tol)


def test_a_captured_step_with_adapters_follows_its_ids_and_lengths():
    layers = _layers(2, ("qkv", "wo", "fc1", "fc2"))
    rot = RotaryPositions(D, rotary_percent=0.5, interleaved=True)
    run = DecodeStackRunner(layers, npu_mem_size=0.004, cpu_mem_size=0, block_size=BS, rotary=rot)
    rng = np.random.default_rng(9)
    b = 6
    x = torch.randn(b, HIDDEN, device="cuda").to(BF)
    tables, lens = _i32(np.arange(b * 4).reshape(b, 4)), _i32([1] * b)
    slots, ids = _i32([i * 4 * BS for i in range(b)]), _i32([0, 1, -1, 3, 2, 0])
    head = torch.randn(HIDDEN, 900, device="cuda") / 16

    def step():
        h = run.decode(x, lens, tables, slots, adapter_ids=ids)
        return [h, *ops.token_logprobs(h.float() @ head, ids, n_top=4)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        n = rng.integers(1, 4 * BS, b)
        lens.copy_(_i32(n))
        slots.copy_(_i32(np.arange(b) * 4 * BS + n - 1))
        ids.copy_(_i32(rng.integers(-1, 5, b)))
        x.copy_(torch.randn(b, HIDDEN, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, w in zip(got, step()):
            assert torch.equal(a, w)


def test_ids_past_32_bits_and_a_runner_with_its_own_layer_loop():
    layers = _layers(1, ("wo",))
    x = torch.randn(3, HIDDEN, device="cuda").to(BF)
    lens, tables, slots = np.array([1, 1, 1]), np.arange(3, dtype=np.int32).reshape(3, 1), np.arange(3, dtype=np.int32) * BS
    plain = DecodeStackRunner(layers, npu_mem_size=0.002, cpu_mem_size=0, block_size=BS)
    none = plain.forward(x, lens, tables, slots, prefill=False)
    some = plain.forward(x, lens, tables, slots, prefill=False, adapter_ids=[1, -1, 2])
    assert not torch.equal(some, none) and torch.equal(some[1], none[1])
    wide = torch.tensor([1, 2 ** 32, -2 ** 32 + 2], device="cuda")           # the slots 0 and 2 in their lowest 32 bits
    for ids in (wide, wide.cpu().numpy()):
        got = plain.forward(x, lens, tables, slots, prefill=False, adapter_ids=ids)
        assert torch.equal(got[0], some[0]) and torch.equal(got[1:], none[1:])

    class Own(DecodeStackRunner):
        def _run_layers(self, h, tables, lens_t, slots, cos, sin, q_starts):
            return super()._run_layers(h, tables, lens_t, slots, cos, sin, q_starts)

    own = Own(layers, npu_mem_size=0.002, cpu_mem_size=0, block_size=BS)
    assert torch.equal(own.forward(x, lens, tables, slots, prefill=False), none)
    assert torch.equal(own.decode(x, _i32(lens), _i32(tables), _i32(slots)), none)
