"""Calls of the generation-side operators at the edges of what their documentation allows."""
import numpy as np
import pytest
import torch

from test_generation_gpu import ACT, _beams, _hold, _np, _paged, _select, _stack

pytestmark = pytest.mark.gpu


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


# --------------------------------------------------------------------------------------------- lists of copies
def _copy(entries, blocks, block=8, row=(2, 32), dtype=torch.float16):
    """Runs a device list and holds it to the list taken entry by entry up to the first negative source."""
    from mindformers_amd import ops
    caches = [torch.randint(-100, 100, (blocks, block) + row, device="cuda").to(dtype) for _ in range(3)]
    want = [c.clone() for c in caches]
    for s, d, r in np.asarray(entries).tolist():
        if s < 0:
            break
        if s < blocks and 0 <= d < blocks:
            for c in want:
                c[d, :max(0, min(r, block))] = c[s, :max(0, min(r, block))]
    ops.copy_blocks(caches, _i32(entries))
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


@pytest.mark.parametrize("entries", [
    [[5, 6, 8], [-1, 3, 8], [7, 9, 8]], [[5, 6, 8], [-1, -1, 0], [7, 9, 8], [8, 10, 8]], [[-1, 5, 8], [0, 1, 8]], [[-7, 5, 8]],
    [[0, 1, 8], [2, 3, 8], [-1, 4, 8], [5, 6, 8]], [[0, 1, 8], [99, 3, 8], [4, 99, 8], [5, 6, 8], [-1, 7, 8]], [[0, 1, 8]] + [[-1, 2, 8], [3, 4, 8]] * 9])
def test_a_list_of_copies_ends_at_its_first_negative_source(entries):
    """Whatever lies behind it, a valid destination of its own included."""
    _copy(entries, 12)
    _copy(entries, 12, block=8, row=(3,), dtype=torch.int8)   # rows that are no multiple of 16 bytes


@pytest.mark.parametrize("n", [64, 65, 200, 513, 2049, 4096, 5000, 9000])
def test_long_lists_of_copies_with_holes(n):
    """Several lists one behind the other, and single negative sources anywhere in a full one: at the ends of what a lane, a wave and a
    workgroup read at a time, where 16384 workgroups take the entries and where 2048 do."""
    rng = np.random.default_rng(n)
    perm = rng.permutation(2 * n)
    full = np.stack([perm[:n], perm[n:], rng.integers(1, 3, n)], axis=1)
    _copy(full, 2 * n, block=2, row=(16,))
    for hole in sorted({0, 1, 63, 64, 65, 255, 256, 511, 512, 513, 2047, 2048, 4095, n - 2, n - 1, int(rng.integers(n))}):
        if hole < n:
            entries = full.copy()
            entries[hole, 0] = -1 - hole % 2                  # its destination stays
            _copy(entries, 2 * n, block=2, row=(16,))
    parts = full.copy()
    parts[n // 3:n // 2] = (-1, -1, 0)
    parts[2 * n // 3:] = (-1, -1, 0)
    _copy(parts, 2 * n, block=2, row=(16,))


# --------------------------------------------------------------------------------------------- beam search
@pytest.mark.parametrize("vocab,beams,eos", [(2, 2, 1), (3, 4, -1), (4, 4, 2), (5, 4, 0), (2, 3, -1), (33, 32, 4)])
def test_beams_of_a_small_vocabulary_share_no_open_block(vocab, beams, eos):
    """No more words than beams: the first step goes on from beams that are out too.  Every row's cache holds the tokens of its own
    line of beams, whatever the others write."""
    from mindformers_amd.modules import BeamSearch
    rng = np.random.default_rng(vocab)
    lens, bs, width = [5, 8, 1], 4, 8
    blocks = 3 * beams * width + 10
    caches = [torch.zeros(blocks, bs, 1, 8, dtype=torch.int32, device="cuda") for _ in range(2)]
    tables = np.full((3, width), -1)
    perm = iter(rng.permutation(blocks).tolist())
    hist = []
    for g, n in enumerate(lens):
        for j in range(-(-n // bs)):
            tables[g, j] = next(perm)
        for t in range(n):
            for c in caches:
                c[int(tables[g, t // bs]), t % bs] = -1 - 100 * g - t
        hist += [[-1 - 100 * g - t for t in range(n)]] * beams
    logits = lambda rows: torch.from_numpy(rng.normal(0, 1, (rows, vocab)).astype(np.float32)).cuda()  # noqa: E731
    search = BeamSearch(caches, beams, eos_token_id=eos)
    search.start(tables, np.array(lens), logits(3))
    for step in range(6):
        if step:
            search.step(logits(3 * beams))
            hist = [hist[p] for p in search._steps[-1].next_rows.view(-1).tolist()]
        slots = search.slot_mapping.tolist()
        assert min(slots) >= 0 and len(set(slots)) == len(slots), f"step {step}"
        for r, s in enumerate(slots):
            for c in caches:
                c.view(-1, 8)[s] = 1000 * step + r + 1
            hist[r] = hist[r] + [1000 * step + r + 1]
        t, n = search.block_tables.tolist(), search.context_lens.tolist()
        held = [c.view(-1, 8).cpu().numpy() for c in caches]
        for r in range(3 * beams):
            assert n[r] == len(hist[r])
            for h in held:
                got = h[[t[r][p // bs] * bs + p % bs for p in range(n[r])]]
                assert (got == np.array(hist[r])[:, None]).all(), f"step {step}, row {r}"


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [24, 30, 32, 33, 34, 36, 60, 127])
def test_selection_of_logits_whose_neighbours_are_far_apart(sign, power):
    """Float32 logits a few of their steps apart, the larger one in a later step of the same lane: what lies between is more than
    the reference's reach, less than it, or just at it."""
    v, n = 70001, 8                                           # a wave walks 2048 columns, 1024 at a time
    ulp = 2.0 ** (power - 23)
    logits = torch.full((6, v), -3.0e38 if sign < 0 else 0.0, device="cuda")
    base = sign * 2.0 ** power - (16 * ulp if sign < 0 else 0)
    for r, k in enumerate((1, 2, 3)):
        logits[r, 5] = base
        logits[r, 1024 + 5] = base + k * ulp
        logits[r, 2048 + 9] = base - 5 * ulp
    logits[3:] = torch.randn(3, v, device="cuda") * 2.5
    _select(logits, torch.tensor([[-1.0, -1.5], [-2.0, -1.0], [-0.5, -20.0]], device="cuda"), n=n, eos=5)
    _select(logits[[0, 3, 1, 4, 2, 5]].contiguous(), torch.full((3, 2), -1.0, device="cuda"), n=n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,k,v,n", [(2, 1, 16, 8), (1, 1, 25, 25), (3, 2, 39, 24), (2, 2, 5003, 20), (1, 1, 70001, 64), (1, 2, 70001, 64), (2, 40, 3001, 64)])
def test_tokens_of_one_beam_whose_scores_are_one_number_go_by_their_logits(b, k, v, n, dtype):
    """Beside +inf, and logits that vanish beside the largest one: equal scores in float64, up to more of them than the join's list
    holds.  Order: score, beam, logit, token."""
    from mindformers_amd import ops
    logits, scores = _beams(b, k, v, dtype, seed=v)
    if dtype == torch.float32:
        logits[::2] *= 1e-25                                  # beside their largest, 3: one number
        logits[::2, v // 2] = 3.0
    else:
        logits[0, v // 3] = float("inf")
    logits[-1, v - 2] = float("inf")
    logits[:, 3] = logits[:, 1]                               # equal logits too
    got = ops.beam_search_select(logits, scores, n_candidates=n)
    x = np.minimum(_np(logits).astype(np.float64), np.finfo(np.float32).max).reshape(b, k, v)
    d = x - x.max(-1, keepdims=True)
    total = _np(scores)[..., None] + (d - np.log(np.exp(d).sum(-1, keepdims=True)))
    beam, token = (a.reshape(-1) for a in np.meshgrid(np.arange(k), np.arange(v), indexing="ij"))
    for g in range(b):
        order = np.lexsort((token, -x[g].reshape(-1), beam, -total[g].reshape(-1)))[:n]
        np.testing.assert_array_equal(_np(got.beams[g]), beam[order])
        np.testing.assert_array_equal(_np(got.tokens[g]), token[order])
        want = total[g].reshape(-1)[order]
        assert (np.abs(_np(got.scores[g]) - want) <= 2.0 ** -24 * np.abs(want) + 1.4e-10).all()


def test_an_end_token_outside_the_vocabulary_ends_nothing():
    from mindformers_amd import ops
    logits, scores = _beams(2, 3, 50, torch.float32, seed=2)
    want = ops.beam_search_select(logits, scores)
    for eos in (50, 2 ** 31 - 1, 2 ** 31 + 5, 2 ** 32 + int(want.tokens[0, 0]), -1, -2 ** 32 + int(want.tokens[0, 0]), -2 ** 40):
        for have, w in zip(ops.beam_search_select(logits, scores, eos_token_id=eos), want):
            assert torch.equal(have, w), eos


def test_selection_from_the_longest_row():
    """0x7c000000 logits of one beam: columns next to 2^31.  Zeros but for a few, so that the sum is a whole number of ones and these:
    2^-24 for the result's rounding, 5.6e-11 of the exponential and 2^-53 an addition of a lane's 508000."""
    from mindformers_amd import ops
    v = 0x7c000000
    logits = torch.zeros(1, v, dtype=torch.bfloat16, device="cuda")
    places, values = [v - 1, 5, v - 70001, v // 2 + 1], [9.0, 8.0, 7.5, 7.0]
    logits[0, torch.tensor(places, device="cuda")] = torch.tensor(values, device="cuda").bfloat16()
    got = ops.beam_search_select(logits, torch.zeros(1, 1, device="cuda"), n_candidates=6)
    assert got.tokens[0].tolist() == places + [0, 1]
    want = np.array(values + [0.0, 0.0]) - np.log((v - 4) + np.exp(values).sum())
    assert (np.abs(got.scores[0].cpu().numpy() - want) <= 2.0 ** -24 * np.abs(want) + 5.6e-11 + 508000 * 2.0 ** -53).all()
    with pytest.raises(ValueError):
        ops.beam_search_select(torch.empty(1, device="cuda").expand(1, v + 1), torch.zeros(1, 1, device="cuda"))


def test_sizes_that_pass_32_bits_are_refused():
    from mindformers_amd import ops
    t, n = _i32(np.zeros((2, 3))), _i32([4, 5])
    for call in (lambda: ops.fork_blocks(t, n, 8, 2 ** 32 + 16), lambda: ops.fork_blocks(t, n, 8, 16, new_tokens=2 ** 32 + 1),
                 lambda: ops.compact_blocks(t, 8, 2 ** 32 + 16), lambda: ops.fork_blocks(t, n, 2 ** 32 + 8, 16)):
        with pytest.raises(ValueError):
            call()


def test_copies_within_blocks_of_2_gib_and_more_are_refused():
    from mindformers_amd import ops
    small = torch.zeros(2, 1, 8, dtype=torch.int8, device="cuda")
    for row in (2 ** 31, 2 ** 32 + 8):                        # the latter is 8 bytes in 32 bits
        big = torch.empty(2, 1, row, dtype=torch.int8, device="cuda")
        for caches in ([big], [small, big]):
            with pytest.raises(ValueError, match="2 GiB"):
                ops.copy_blocks(caches, [[0, 1]])

# --------------------------------------------------------------------------------------------- captures
def test_a_capture_takes_workspaces_of_its_own():
    from mindformers_amd import ops
    dev = torch.device("cuda", torch.cuda.current_device())
    eager = ops.workspace(1 << 20, dev, "gemm")
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            got.append([ops.workspace(1 << 20, dev, tag).fill_(1) for tag in ("gemm", "pa")])
    places = [eager.data_ptr()] + [w.data_ptr() for ws in got for w in ws]
    assert all(abs(a - b) >= 1 << 20 for i, a in enumerate(places) for b in places[:i])
    assert ops.workspace(1 << 20, dev, "gemm") is eager


@pytest.mark.parametrize("act_quant", [False, True])
@pytest.mark.parametrize("window,sinks", [(None, 0), (900, 4)])
def test_steps_of_a_stack_replayed_at_once_share_no_workspace(window, sinks, act_quant):
    """Two captured decode steps of the serving runner, whose attention and products are cut, replayed together on two streams."""
    from mindformers_amd.runner import DecodeStackRunner
    layers, bs, rows, width = _stack(window, sinks, act_quant), 16, 5, 100
    runs = [DecodeStackRunner(layers, npu_mem_size=0.05, cpu_mem_size=0, block_size=bs) for _ in range(2)]
    assert runs[0].npu_num_blocks >= rows * width
    gen = torch.Generator(device="cuda")
    steps = []
    for i, run in enumerate(runs):
        gen.manual_seed(i)
        for c in run.caches():
            c.normal_(generator=gen)
        n = torch.randint(1000, width * bs, (rows,), generator=gen, device="cuda").int()
        tables = torch.randperm(rows * width, generator=gen, device="cuda").int().view(rows, width)
        slots = (torch.gather(tables, 1, ((n - 1) // bs)[:, None].long())[:, 0] * bs + (n - 1) % bs).int()
        steps.append((torch.randn(rows, 512, generator=gen, device="cuda").bfloat16(), n, tables, slots))
    want = [run.decode(*s).clone() for run, s in zip(runs, steps)]
    torch.cuda.synchronize()
    graphs, got = [], []
    for run, s in zip(runs, steps):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            for _ in range(4):                                # the same step again: the token's row is written anew each time
                out = run.decode(*s)
        got.append(out)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(30):
        for out in got:
            out.zero_()
        for g, st in zip(graphs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# --------------------------------------------------------------------------------------------- windowed attention
def test_windows_over_the_widest_tables():
    """Tables that name 2^30 tokens, walks of 40000, cut in other places than behind tables that end with the context: every query
    finds its one key, whose probability is 1 in either."""
    from mindformers_amd import ops
    bs, b, nh, d = 16384, 32, 8, 32
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    kc, vc = (torch.randn(3, bs, nh, d, generator=gen, device="cuda").bfloat16() for _ in range(2))
    narrow = torch.arange(3, dtype=torch.int32, device="cuda").repeat(b, 1)
    wide = torch.full((b, (1 << 30) // bs), -1, dtype=torch.int32, device="cuda")
    wide[:, :3] = narrow
    n, starts = torch.randint(33000, 40001, (b,), generator=gen, device="cuda").int(), torch.arange(b + 1, device="cuda").int()
    q = torch.randn(4 * b, nh, d, generator=gen, device="cuda").bfloat16()
    kc.mul_(0.01)

    def plant(row, token):                                    # a score of about 0.2 * 32 * 32, the others' are below 2
        kc.view(-1, nh, d)[token] = 32 * q[row]
        return vc.view(-1, nh, d)[token].reshape(-1).clone()

    for window, sinks in ((2 ** 31 - 1, 0), (1 << 30, 3), (35000, 5100)):
        keep = kc.clone()
        want = torch.stack([plant(i, int(n[i]) - 1 - 1031 * i) for i in range(b)])
        for t in (wide, narrow):
            assert torch.equal(ops.paged_attention(q[:b].reshape(b, -1), kc, vc, t, n, nh, nh, 0.2, window=window, sinks=sinks), want)
        kc.copy_(keep)
    n = torch.arange(33000, 33000 + 220 * b, 220, device="cuda").int()
    want = torch.stack([plant(4 * i + j, int(n[i]) - 4 + j - 50 * j) for i in range(b) for j in range(4)])
    for t in (wide, narrow):
        assert torch.equal(ops.paged_attention_prefill(q.reshape(4 * b, -1), kc, vc, t, n, 4 * starts, nh, nh, 0.2, window=200, sinks=3), want)


@pytest.mark.parametrize("dtype", ACT)
@pytest.mark.parametrize("b,nh,nkv,hi,window", [(3, 8, 2, 40, 20), (5, 8, 2, 1500, 900), (70, 8, 2, 200, 64), (80, 4, 1, 1900, 1500), (131, 2, 1, 1900, 1500),
                                                (16, 8, 2, 700, 513)])
def test_tiled_codes_of_windowed_decode_equal_two_calls(dtype, b, nh, nkv, hi, window):
    """The layout that the W8A8 layers take, of walks in one partition and in several, with whole 64 rows and without."""
    from helpers import untile_int8
    from mindformers_amd import ops
    rng = np.random.default_rng(b)
    lens = rng.integers(0, hi + 1, b)
    q, cache, _, tables, _, _ = _paged(rng, dtype, lens, [1] * b, nh, nkv, 64, 16, window, 5)
    dq, kc, vc = (torch.from_numpy(x).to(dtype).cuda() for x in (q, *cache))
    k = nh * 64
    for smooth in (None, torch.rand(k, device="cuda") + 0.5):
        args = (dq, kc, vc, _i32(tables), _i32(lens), nh, nkv, 0.1)
        want = ops.paged_attention(*args, window=window, sinks=5)
        assert (want[torch.from_numpy(lens == 0).cuda()] == 0).all()
        rows, scales = ops.dynamic_quant(want, smooth)
        for tiled in (False, True):
            out, xq, xs = ops.paged_attention(*args, quant=(smooth, tiled), window=window, sinks=5)
            codes = untile_int8(xq.data.cpu().numpy(), b, k) if tiled else xq.cpu().numpy()
            assert torch.equal(out, want) and torch.equal(xs, scales)
            np.testing.assert_array_equal(codes, rows.cpu().numpy())


@pytest.mark.parametrize("rows", [2, 5, 70])
def test_a_w8a8_layer_behind_a_long_window_is_its_separate_operators(rows, monkeypatch):
    """The walk is cut: the attention's partitions are joined by the kernel that quantises the row too."""
    from mindformers_amd import ops
    from mindformers_amd.decode_layer import QuantDecodeLayer
    layer, = _stack(1500, 7, act_quant=True, n=1)
    bs, width = 32, 60
    kc, vc = (torch.randn(rows * width, bs, 2, 64, device="cuda").bfloat16() for _ in range(2))
    tables = torch.randperm(rows * width, device="cuda").int().view(rows, width)
    n = torch.randint(1, width * bs + 1, (rows,), device="cuda").int()
    slots = (torch.gather(tables, 1, ((n - 1) // bs)[:, None].long())[:, 0] * bs + (n - 1) % bs).int()
    x = torch.randn(rows, 512, device="cuda").bfloat16()
    cos, sin = torch.ones(rows, 64, device="cuda").bfloat16(), torch.zeros(rows, 64, device="cuda").bfloat16()
    got = layer(x, kc.clone(), vc.clone(), tables, n, slots, cos, sin)
    calls, whole = [], ops.paged_attention

    def in_two(*args, quant=None, **kw):
        out = whole(*args, **kw)
        calls.append(kw)
        return out if quant is None else (out, *ops.dynamic_quant(out, quant[0], tiled=quant[1]))

    monkeypatch.setattr(ops, "paged_attention", in_two)
    want = QuantDecodeLayer.forward(layer, x, kc.clone(), vc.clone(), tables, n, slots, cos, sin)
    assert calls == [dict(window=1500, sinks=7)]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 2.0 ** 40), (torch.bfloat16, 2.0 ** -50), (torch.bfloat16, 2.0 ** 25), (torch.float16, 2.0 ** 15),
                                        (torch.float16, 2.0 ** -24), (torch.bfloat16, 0.0), (torch.bfloat16, 2.0 ** -110)])
@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("window,sinks", [(40, 0), (70, 1), (230, 3)])
def test_int8_windows_with_large_and_small_queries_at_a_channels_own_tolerance(dtype, size, rows, window, sinks):
    """One row a sequence in the decode form, more of them as chunks; the largest key of the queries' channel is the first token, which
    the window leaves."""
    from mindformers_amd import ops
    rng = np.random.default_rng(rows)
    lens, nh, nkv, d, block = [255, 254, 0, 255], 8, 2, 64, 16
    q_lens = [rows, 1, rows if rows == 1 else 0, rows]
    q = np.zeros((sum(q_lens), nh, d))
    q[:, :, 5] = size
    cache = rng.integers(-127, 128, (2, 64, block, nkv, d))
    cache[0].reshape(4, 256, nkv, d)[..., 5] = 127 - np.minimum(np.arange(256), 254)[None, :, None]
    keys, values = ([c.reshape(4, 256, nkv, d)[b, :n] / 128.0 for b, n in enumerate(lens)] for c in cache)
    dq = torch.from_numpy(q.reshape(-1, nh * d)).to(dtype).cuda()
    kc, vc = (torch.from_numpy(c).to(torch.int8).cuda() for c in cache)
    starts = None if rows == 1 else _i32(np.concatenate([[0], np.cumsum(q_lens)]))
    got = ops.paged_attention_int8kv(dq, kc, vc, _i32(np.arange(64).reshape(4, 16)), _i32(lens), torch.full((2, nkv * d), 1 / 128.0, device="cuda"),
                                     None, nh, nkv, 0.125, q_starts=starts, window=window, sinks=sinks)
    _hold(_np(got), (q.reshape(-1, nh * d), keys, values, lens, q_lens, nh, nkv, 0.125, window, sinks), dtype, f"size {size}", "channel")


# Tolerance: as in the form without offsets, of the int8 values and of the offset, which is taken off their sum.
@pytest.mark.parametrize("dtype", ACT)
@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1, 1], [1, 40, 7, 0, 200]])
@pytest.mark.parametrize("nh,nkv,d,block", [(8, 2, 64, 16), (7, 1, 128, 128), (4, 4, 32, 12)])
@pytest.mark.parametrize("window,sinks", [(5, 3), (300, 20)])
def test_windows_over_int8_caches_with_offsets(dtype, q_lens, nh, nkv, d, block, window, sinks):
    from helpers import assert_within
    from mindformers_amd import ops
    from oracle import generation as G
    rng = np.random.default_rng(d)
    lens = [1, 97, 300, 0, 1100]
    q, cache, scales, tables, _, _ = _paged(rng, dtype, lens, q_lens, nh, nkv, d, block, window, sinks, "channel")
    offset = rng.integers(-30, 31, (2, nkv * d)).astype(np.float32)
    need = [-(-n // block) for n in lens]
    raw, keys, values = [], [], []
    for b, n in enumerate(lens):
        k8, v8 = (c[np.maximum(tables[b, :need[b]], 0)].astype(np.float64).reshape(-1, nkv, d)[:n] for c in cache)
        s, o = scales.reshape(2, nkv, d), offset.reshape(2, nkv, d)
        keys.append((k8 - o[0]) * s[0])
        values.append((v8 - o[1]) * s[1])
        raw.append((np.abs(v8) + np.abs(o[1])) * s[1])
    s, o = torch.from_numpy(scales).float().cuda(), torch.from_numpy(offset).cuda()
    starts = None if max(q_lens) == 1 else _i32(np.concatenate([[0], np.cumsum(q_lens)]))
    dq, (kc, vc) = torch.from_numpy(q).to(dtype).cuda(), (torch.from_numpy(c).to(torch.int8).cuda() for c in cache)
    got = ops.paged_attention_int8kv(dq, kc, vc, _i32(tables), _i32(lens), s, o, nh, nkv, 1 / np.sqrt(d), q_starts=starts, window=window, sinks=sinks)
    rest = (lens, q_lens, nh, nkv, 1 / np.sqrt(d), window, sinks)
    extra = 2.0 ** -25 * G.window_attention(q, keys, raw, *rest, of="sum") + (2.0 ** -25 if dtype == torch.float16 else 0)
    want = G.window_attention(q, keys, values, *rest)
    assert_within(_np(got), want, G.window_attention(q, keys, raw, *rest, of="magnitude"), dtype, ulps=3.0, extra=extra, what="offsets")
    if max(q_lens) == 1:
        assert (got[3] == 0).all()


@pytest.mark.parametrize("kind", ["16", "channel", "token"])
def test_windowed_attention_repeats_itself_bit_for_bit(kind):
    """Walks in one and in several partitions: the order in which waves arrive changes no sum."""
    from mindformers_amd import ops
    rng = np.random.default_rng(2)
    lens = rng.integers(1, 2600, 20)
    q, cache, scales, tables, _, _ = _paged(rng, torch.bfloat16, lens, [1] * 20, 8, 2, 128, 32, 1200, 4, kind, poison=False)
    dq, (kc, vc) = torch.from_numpy(q).bfloat16().cuda(), (torch.from_numpy(c).to(torch.bfloat16 if kind == "16" else torch.int8).cuda() for c in cache)
    t = _i32(tables)
    few = torch.randn(int(min(lens[0], 9)) + 30, 1024, device="cuda").bfloat16()
    lens[1] = max(lens[1], 30)
    n, starts = _i32(lens), _i32(np.concatenate([[0, few.shape[0] - 30], np.full(19, few.shape[0])]))
    s = None if scales is None else torch.from_numpy(scales).float().cuda()
    par = dict(token_scales=(s[0].contiguous(), s[1].contiguous())) if kind == "token" else {}
    view = dict(window=1200, sinks=4)

    def calls():
        if kind == "16":
            return [ops.paged_attention(dq, kc, vc, t, n, 8, 2, 0.1, **view), ops.paged_attention_prefill(few, kc, vc, t, n, starts, 8, 2, 0.1, **view)]
        return [ops.paged_attention_int8kv(x, kc, vc, t, n, None if par else s, None, 8, 2, 0.1, q_starts=st, **par, **view)
                for x, st in ((dq, None), (few, starts))]

    want = calls()
    for _ in range(20):
        for have, w in zip(calls(), want):
            assert torch.equal(have, w)


@pytest.mark.parametrize("blocks,rows", [(1 << 19, 3), ((1 << 19) - 128, 3), ((1 << 19) - 128 * 8, 248), ((1 << 19) + 1, 5)])
def test_pools_whose_bitmap_is_64_kb(blocks, rows):
    from mindformers_amd import ops
    from oracle import generation as G
    rng = np.random.default_rng(rows)
    tables = rng.choice(blocks, (rows, 40), replace=False)
    tables[0, :3] = (blocks - 1, 0, blocks - 2)
    lens = rng.integers(1, 161, rows)
    got = ops.fork_blocks(_i32(tables), _i32(lens), blocks, 4, new_tokens=3)
    for have, w in zip(got, G.fork_blocks(tables, lens, blocks, 4, new_tokens=3)):
        np.testing.assert_array_equal(have.cpu().numpy().reshape(np.shape(w)), w)
    named = np.sort(np.unique(tables))
    to = dict(zip(named[named >= len(named)].tolist(), np.setdiff1d(np.arange(len(named)), named).tolist()))
    out, copies, live = ops.compact_blocks(_i32(tables), blocks, 4)
    assert int(live) == len(named)
    np.testing.assert_array_equal(out.cpu().numpy(), np.vectorize(lambda p: to.get(p, p))(tables))
    np.testing.assert_array_equal(copies[:len(to)].cpu().numpy(), [(a, b, 4) for a, b in to.items()])
    assert (copies[len(to):] == torch.tensor([-1, -1, 0], device="cuda")).all()


@pytest.mark.parametrize("kind", ["16", "channel", "token"])
@pytest.mark.parametrize("lens,window,sinks", [([9000, 7, 0, 2049] + [40] * 30, 8192, 5), ([6200, 6143, 6300], 6100, 40), ([9000] + [300] * 9, 2 ** 31 - 1, 0)])
def test_long_windows_over_ragged_contexts_match_the_oracle(kind, lens, window, sinks):
    """Walks that are cut however many sequences there are, and walks next to that length."""
    from test_generation_gpu import _windowed
    _windowed(torch.bfloat16, lens, [1] * len(lens), 8, 8, 32, 32, window, sinks, kind)


@pytest.mark.parametrize("longest", [9000, 36000])
def test_long_windows_with_quantised_output_equal_two_calls(longest):
    """Five partitions, joined by the kernel that quantises, and eighteen, which it does not take; a workspace smaller than they need is
    refused."""
    from mindformers_amd import _lib, ops
    bs, b, nh, nkv, d = 128, 40, 8, 8, 32
    width = -(-longest // bs)
    kc, vc = (torch.randn(width, bs, nkv, d, device="cuda").bfloat16() for _ in range(2))
    tables = torch.stack([torch.randperm(width, device="cuda").int() for _ in range(b)])
    n = torch.randint(1, 1000, (b,), device="cuda").int()
    n[7] = longest
    q = torch.randn(b, nh * d, device="cuda").bfloat16()
    want = ops.paged_attention(q, kc, vc, tables, n, nh, nkv, 0.2, window=longest)
    full = ops.paged_attention(q, kc, vc, tables, n, nh, nkv, 0.2)
    assert (want.float() - full.float()).abs().max() <= 2 * 2.0 ** -8 * vc.float().abs().max()
    for tiled in (False, True):
        out, xq, xs = ops.paged_attention(q, kc, vc, tables, n, nh, nkv, 0.2, quant=(None, tiled), window=longest)
        wq, ws = ops.dynamic_quant(want, None, tiled=tiled)
        assert torch.equal(out, want) and torch.equal(xs, ws)
        from helpers import untile_int8
        codes = [untile_int8(x.data.cpu().numpy(), b, nh * d) if tiled else x.cpu().numpy() for x in (xq, wq)]
        np.testing.assert_array_equal(*codes)
    lib = _lib.load()
    need = lib.mf_window_attention_workspace_bytes(b, nh, d, width * bs, longest, 0)
    parts = -(-(width * bs) // 2048)
    assert need >= b * nh * parts * (d + 2) * 4
