"""Beam selection, shared blocks and windowed attention on the GPU against plain statements in float64 / whole numbers."""
import numpy as np
import pytest
import torch

from oracle import generation as G

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _np(t):
    return t.detach().float().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


# --------------------------------------------------------------------------------------------- beam selection
def _select(logits, scores, n=None, eos=-1):
    """Runs the selection and holds it to the oracle: whole numbers equal, scores to half a float32 step plus the 5.6e-11 that the
    exponential's polynomial may be off and the 2^-53 of every addition of the sum (below 1.4e-10 together)."""
    from mindformers_amd import ops
    got = ops.beam_search_select(logits, scores, eos_token_id=eos, n_candidates=n)
    b, k = scores.shape
    cand, going = G.beam_search_select(_np(logits).reshape(b, k, -1), _np(scores), got.scores.shape[1], eos)
    for have, want in ((got[:3], cand), (got[3:], going)):
        np.testing.assert_array_equal(_np(have[1]), want[1])
        np.testing.assert_array_equal(_np(have[2]), want[2])
        s, w = _np(have[0]).astype(np.float64), want[0]
        dead = ~np.isfinite(w)
        np.testing.assert_array_equal(s[dead], w[dead])
        s, w = s[~dead], w[~dead]
        assert (np.abs(s - w) <= 2.0 ** -24 * np.abs(w) + 1.4e-10).all()
    return got


def _beams(b, k, v, dtype, seed, std=2.5):
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn(b * k, v, generator=gen) * std).to(dtype).cuda()
    scores = (-10 - torch.cumsum(torch.rand(b, k, generator=gen), 1)).cuda()
    return logits, scores


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,k,v", [(1, 1, 2), (1, 4, 1000), (3, 3, 517), (2, 8, 32003), (5, 2, 8191), (1, 32, 2049), (17, 5, 70001)])
def test_selection_matches_the_oracle(b, k, v, dtype):
    logits, scores = _beams(b, k, v, dtype, seed=b * 1000 + k)
    _select(logits, scores, eos=1 if v > 2 else -1)
    _select(logits, scores, n=min(64, k * v))


@pytest.mark.parametrize("dtype", DTYPES)
def test_selection_of_logits_that_are_all_alike_takes_the_lowest_places(dtype):
    logits = torch.full((6, 9001), 0.5, dtype=dtype, device="cuda")
    got = _select(logits, torch.full((2, 3), -1.0, device="cuda"), eos=0)
    assert got.tokens[0].tolist() == [0, 1, 2, 3, 4, 5] and got.next_tokens[0].tolist() == [1, 2, 3]


@pytest.mark.parametrize("dtype", DTYPES)
def test_selection_of_rising_logits(dtype):
    """Every step of a wave is better than the one before, lane after lane: the longest way through the list."""
    logits = (torch.arange(40000, dtype=torch.float32) / 400 - 50).to(dtype).repeat(4, 1).cuda()
    logits[1:] += torch.tensor([0.25, 0.5, -0.25], dtype=dtype, device="cuda")[:, None]
    _select(logits, torch.tensor([[-3.0, -2.9], [-4.0, -4.5]], device="cuda"), n=64, eos=39999)


@pytest.mark.parametrize("dtype", DTYPES)
def test_selection_with_masked_logits(dtype):
    """Words forbidden by -inf, by the type's lowest value and by NaN, whole rows of them, and +inf."""
    logits, scores = _beams(6, 4, 5003, dtype, seed=5)
    logits[0:4, 5:] = -float("inf")                           # fewer words left than candidates
    logits[4:8] = torch.finfo(dtype).min                      # every word at the lowest value: an even row
    logits[8:12, ::2] = float("nan")
    logits[12] = -float("inf")                                # one beam without a word
    logits[16:20] = float("nan")                              # a group without a word
    logits[20, 77] = float("inf")
    got = _select(logits, scores, eos=3)
    assert torch.isneginf(got.scores[4]).all() and got.tokens[4].tolist() == list(range(8))


def test_selection_with_beams_that_are_out():
    """The first step of a search: all beams but one out, by -inf, by NaN, by a number that is no log probability."""
    logits, _ = _beams(4, 3, 777, torch.float32, seed=9)
    scores = torch.tensor([[0.0, -float("inf"), -float("inf")], [-1.0, float("nan"), -3.4e38], [-float("inf")] * 3, [0.0, -1e9, -1e9]],
                          device="cuda")
    got = _select(logits, scores)
    assert got.beams[:2].eq(0).all() and got.tokens[2].tolist() == list(range(6))
    _select(logits[:, :5].contiguous(), scores, n=15)         # down to the last word of a beam that is out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off", [0, 1, 3, 5])
def test_selection_reads_a_slice_of_wider_rows(dtype, off):
    """Rows that start at any element: padded vocabularies and views."""
    gen = torch.Generator().manual_seed(off)
    wide = torch.randn(6, 4099, generator=gen).to(dtype).cuda() + 100
    wide[:, off:off + 4000] -= 100
    _select(wide[:, off:off + 4000], -torch.rand(2, 3, generator=gen).cuda(), eos=7)


def test_selection_orders_candidates_that_float32_sums_would_not():
    """Two beams whose scores differ by 2e-8 only: the order hangs on the last bits of the logsums."""
    logits, _ = _beams(1, 2, 50001, torch.float32, seed=3, std=1.0)
    lse = torch.logsumexp(logits.double(), dim=1)
    run = torch.zeros(1, 2, device="cuda")
    run[0, 1] = (logits[0].max().double() - lse[0] - (logits[1].max().double() - lse[1])).float()
    _select(logits, run)


def test_selection_of_no_group_and_replayed_in_a_graph():
    from mindformers_amd import ops
    assert ops.beam_search_select(torch.zeros(0, 50, device="cuda"), torch.zeros(0, 4, device="cuda")).tokens.shape == (0, 8)
    logits, scores = _beams(3, 4, 20011, torch.bfloat16, seed=1)
    ops.beam_search_select(logits, scores, eos_token_id=2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.beam_search_select(logits, scores, eos_token_id=2)
    for seed in (2, 3, 4):
        fresh, run = _beams(3, 4, 20011, torch.bfloat16, seed)
        logits.copy_(fresh)
        scores.copy_(run)
        graph.replay()
        torch.cuda.synchronize()
        for have, want in zip(got, ops.beam_search_select(logits, scores, eos_token_id=2)):
            assert torch.equal(have, want)


# --------------------------------------------------------------------------------------------- shared blocks
def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


def _tables(rng, rows, width, block, blocks, groups=1):
    """Rows that share the blocks of the first half of their group's context."""
    lens = rng.integers(0, width * block + 1, rows)
    tables = np.full((rows, width), -1)
    ids = iter(rng.permutation(blocks).tolist())
    for r in range(rows):
        lead = r // groups * groups
        for j in range(-(-int(lens[r]) // block)):
            shared = r != lead and (j + 1) * block <= min(lens[r], lens[lead]) and j < width // 2
            tables[r, j] = tables[lead, j] if shared else next(ids)
    return tables, lens


def _fork(tables, lens, blocks, block, **kw):
    from mindformers_amd import ops
    dev = {k: (_i32(v) if k == "parents" else torch.from_numpy(v).cuda()) if isinstance(v, np.ndarray) else v for k, v in kw.items()}
    got = ops.fork_blocks(_i32(tables), _i32(lens), blocks, block, **dev)
    want = G.fork_blocks(tables, lens, blocks, block, **kw)
    for name, w in zip(got._fields, want):
        np.testing.assert_array_equal(_np(getattr(got, name)).reshape(np.shape(w)), w, err_msg=name)
    return got


@pytest.mark.parametrize("rows,width,block,new", [(1, 1, 1, 0), (1, 1, 16, 1), (7, 5, 16, 1), (16, 33, 4, 3), (33, 12, 3, 17),
                                                  (130, 70, 16, 1), (1100, 9, 8, 2), (2500, 3, 5, 1)])
def test_fork_matches_the_oracle(rows, width, block, new):
    rng = np.random.default_rng(rows + width)
    blocks = rows * (width + 1 + -(-new // block)) + 5
    tables, lens = _tables(rng, rows, width, block, blocks, groups=4)
    for i in range(3):
        parents = rng.integers(-1, rows, rows) if i else None
        window = [None, 2 * block + 1, 1][i]
        _fork(tables, lens, blocks, block, parents=parents, new_tokens=new, window=window, sinks=[0, 2, block + 1][i])
    held = rng.random(blocks) < 0.4
    _fork(tables, lens, blocks, block, parents=rng.integers(-3, rows + 3, rows), new_tokens=new, held=held)


def test_fork_without_blocks_left_counts_what_is_missing():
    rng = np.random.default_rng(0)
    tables, lens = _tables(rng, 12, 6, 8, 80, groups=3)
    used = int(max(tables.max() + 1, 1))
    for blocks in (used, used + 3, 80):
        for parents in (np.zeros(12, int), np.arange(12), rng.integers(0, 12, 12)):
            _fork(tables, lens, blocks, 8, parents=parents, new_tokens=9)
    full = _fork(tables, np.full(12, 48), 80, 8, new_tokens=1)       # rows as long as the table is wide
    assert int(full.missing) == 12 and (full.slot_mapping == -1).all() and (full.context_lens == 48).all()


def test_fork_ignores_entries_that_name_no_block():
    tables = np.array([[3, 99, -7, 2], [0, 1, -1, -1], [5, 6, 7, 8]])
    got = _fork(tables, np.array([7, 3, -4]), 10, 2, parents=np.array([0, 0, 2]), new_tokens=1)
    assert got.block_tables[0, 1] == -1 and got.context_lens[2] == 1


def test_fork_of_a_pool_of_a_million_blocks():
    """The largest bitmap: 128 KB of LDS; free blocks only at the far end."""
    blocks = 1 << 20
    held = np.ones(blocks, dtype=bool)
    held[-40:] = False
    _fork(np.full((9, 3), -1), np.zeros(9, int), blocks, 16, new_tokens=33, held=held)


def test_fork_replayed_in_a_graph_and_on_another_stream():
    from mindformers_amd import ops
    rng = np.random.default_rng(4)
    for rows, width in ((8, 6), (200, 64)):
        blocks = rows * (width + 2)
        tables, lens = _tables(rng, rows, width, 4, blocks, groups=4)
        t, l, p = _i32(tables), _i32(lens), _i32(np.arange(rows))
        ops.fork_blocks(t, l, blocks, 4, parents=p, new_tokens=1)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = ops.fork_blocks(t, l, blocks, 4, parents=p, new_tokens=1)
        for _ in range(3):
            p.copy_(_i32(rng.integers(-1, rows, rows)))
            graph.replay()
            torch.cuda.synchronize()
            other = torch.cuda.Stream()
            with torch.cuda.stream(other):
                want = ops.fork_blocks(t, l, blocks, 4, parents=p, new_tokens=1)
            other.synchronize()
            for have, w in zip(got, want):
                assert torch.equal(have, w)


@pytest.mark.parametrize("rows,width,blocks", [(1, 1, 1), (1, 3, 7), (9, 7, 200), (64, 40, 5000), (3, 100, 70001)])
def test_compact_matches_the_oracle(rows, width, blocks):
    from mindformers_amd import ops
    rng = np.random.default_rng(blocks)
    tables = np.where(rng.random((rows, width)) < 0.6, rng.integers(0, blocks, (rows, width)), -1)
    tables[0, 0] = blocks + 3                                 # names no block
    for held in (None, rng.random(blocks) < 0.3, np.ones(blocks, dtype=bool)):
        got = ops.compact_blocks(_i32(tables), blocks, 16, held=None if held is None else torch.from_numpy(held).cuda())
        want = G.compact_blocks(tables, blocks, 16, held)
        for have, w in zip(got, want):
            np.testing.assert_array_equal(_np(have).reshape(np.shape(w)), w)
        again = ops.compact_blocks(got[0], blocks, 16, held=None if held is None else torch.from_numpy(held).cuda())
        assert (again[1] == torch.tensor([-1, -1, 0], device="cuda")).all() and torch.equal(again[0], got[0])


@pytest.mark.parametrize("block,row,dtype", [(16, (2, 64), torch.bfloat16), (128, (8, 128), torch.float16), (4, (1, 32), torch.int8),
                                             (5, (3,), torch.float32), (3, (1, 1), torch.int8)])
def test_copies_move_the_rows_of_a_block_and_nothing_else(block, row, dtype):
    from mindformers_amd import ops
    rng = np.random.default_rng(block)
    blocks, n = 61, 9
    caches = [torch.randint(-100, 100, (blocks, block) + row, device="cuda").to(dtype) for _ in range(5)]
    caches.append(torch.rand(blocks, block, device="cuda"))   # the scales of an int8 cache
    perm = rng.permutation(blocks)
    entries = np.stack([perm[:n], perm[n:2 * n], rng.integers(0, block + 1, n)], axis=1)
    entries[1, 0] = entries[0, 0]                             # one source, two destinations
    want = [c.clone() for c in caches]
    for c in want:
        for s, d, r in entries.tolist():
            c[d, :r] = c[s, :r]
    listed = np.concatenate([entries, np.tile([-1, -1, 0], (100, 1)), [[0, 1, block]]])       # nothing behind the list's end
    ops.copy_blocks(caches, _i32(listed))
    assert all(torch.equal(c, w) for c, w in zip(caches, want))
    ops.copy_blocks(caches, entries[:, [0, 1]].tolist())      # whole blocks, named by the host
    for c in want:
        for s, d, _ in entries.tolist():
            c[d] = c[s]
    assert all(torch.equal(c, w) for c, w in zip(caches, want))
    ops.copy_blocks(caches, [])
    ops.copy_blocks(caches, torch.zeros(0, 3, dtype=torch.int32, device="cuda"))
    # entries outside the caches are skipped, rows are clamped
    ops.copy_blocks(caches, _i32([[blocks, 2, block], [1, blocks, block], [1, -5, block], [perm[-1], perm[-2], block + 99]]))
    for c in want:
        c[perm[-2]] = c[perm[-1]]
    assert all(torch.equal(c, w) for c, w in zip(caches, want))


def test_copies_of_more_caches_than_a_launch_names_and_past_4_gib():
    from mindformers_amd import ops
    caches = [torch.full((6, 2, 8), i, dtype=torch.float16, device="cuda") for i in range(300)]
    for c in caches:
        c[0] += 1
    ops.copy_blocks(caches, [[0, 5]])
    assert all((c[5] == c[0]).all() and (c[4] == i).all() for i, c in enumerate(caches))
    big = torch.zeros(5000, 128, 8, 512, dtype=torch.int8, device="cuda")          # 2.6 GB, a block of 512 KB
    wide = torch.zeros(5000, 128, 8, 512, dtype=torch.bfloat16, device="cuda")     # 5.2 GB
    for c in (big, wide):
        c[4998] = 7
    ops.copy_blocks([big, wide], [[4998, 4999, 127], [0, 1, 128]])
    for c in (big, wide):
        assert (c[4999, :127] == 7).all() and (c[4999, 127] == 0).all() and (c[1] == 0).all()


# --------------------------------------------------------------------------------------------- sliding window with sinks
# Tolerance: probabilities are rounded in front of the product with the values (half a step of sum p |v|), the denominator
# sums them rounded (half a step of the result at most), the result is rounded (half a step): three half steps of sum p |v|,
# which helpers.EPS is one of.  Below 2^-14 fp16 is off by up to 2^-25 whatever the value (the smallest step's half): that much of the
# sum of the visible |v| more, as the largest probability is 1 at least; where the values' scale of an int8 cache rides on the
# probability, of the sum of the visible int8 values.  int8 caches with a scale a channel go through fp16 in both types.  The scales of
# int8 caches are powers of two here, so that folding them into the query rounds nothing.
def _hold(got, args, dtype, what, kind="16", steps=None):
    from helpers import assert_within
    extra = 0.0
    if dtype == torch.float16 or kind == "channel":
        q, keys, values, *rest = args
        extra = 2.0 ** -25 * G.window_attention(q, keys, values if steps is None else steps, *rest, of="sum")
        if dtype == torch.float16:                            # the result itself
            extra = extra + 2.0 ** -25
    assert_within(got, G.window_attention(*args), G.window_attention(*args, of="magnitude"), dtype, ulps=3.0, extra=extra, what=what)


ACT = [torch.bfloat16, torch.float16]


def _paged(rng, dtype, lens, q_lens, nh, nkv, d, block, window, sinks, kind="16", poison=True):
    """Queries and a paged cache of the given lengths in a shuffled pool.  Blocks without a visible token are given back (-1) and
    everything that no row sees holds NaN (16-bit values, scales) or garbage."""
    from helpers import rounded
    lens, q_lens = np.asarray(lens), np.asarray(q_lens)
    need = [-(-max(int(n), 0) // block) for n in lens]
    width = max(max(need), 1) + 1
    nb = sum(need) + 3
    perm = rng.permutation(nb)
    tables = np.full((len(lens), width), -1)
    at = 0
    shape = (nb, block, nkv, d)
    if kind == "16":
        cache = [rounded(rng.normal(0, 1, shape), dtype) for _ in range(2)]
        scales = None
    else:
        cache = [rng.integers(-127, 128, shape).astype(np.float32) for _ in range(2)]
        scales = 2.0 ** -rng.integers(5, 8, (2, nb, block) if kind == "token" else (2, nkv * d)).astype(np.float64)
    keys, values = [], []
    visible = np.zeros((nb, block), dtype=bool)
    for b, n in enumerate(lens):
        pages = perm[at:at + need[b]]
        at += need[b]
        tables[b, :need[b]] = pages
        for store, c, i in ((keys, cache[0], 0), (values, cache[1], 1)):
            rows = c[pages].astype(np.float64)
            if kind == "token":
                rows = rows * scales[i][pages][:, :, None, None]
            rows = rows.reshape(-1, nkv, d)[:max(int(n), 0)]
            store.append(rows * scales[i].reshape(nkv, d) if kind == "channel" else rows)
        for p in range(max(int(n - q_lens[b]), 0), int(n)):
            for j in list(range(max(p - window + 1, 0), p + 1)) + list(range(min(sinks, p + 1))):
                visible[pages[j // block], j % block] = True
    if poison:
        for c in cache:
            c[~visible] = np.nan if kind == "16" else -128
        if kind == "token":
            scales[:, ~visible] = np.nan
        hidden = ~visible.any(axis=1)
        tables = np.where((tables >= 0) & hidden[tables], -1, tables)
    q = rounded(rng.normal(0, 1, (int(q_lens.sum()), nh * d)), dtype)
    return q, cache, scales, tables, keys, values


def _windowed(dtype, lens, q_lens, nh, nkv, d, block, window, sinks, kind="16", seed=0, strided=False):
    from mindformers_amd import ops
    rng = np.random.default_rng(seed + window)
    q, cache, scales, tables, keys, values = _paged(rng, dtype, lens, q_lens, nh, nkv, d, block, window, sinks, kind)
    dq = torch.from_numpy(q).to(dtype).cuda()
    if strided:
        wide = torch.full((dq.shape[0], dq.shape[1] + 24), float("nan"), dtype=dtype, device="cuda")
        wide[:, 8:-16] = dq
        dq = wide[:, 8:-16]
    kc, vc = (torch.from_numpy(c).to(dtype if kind == "16" else torch.int8).cuda() for c in cache)
    t, n = _i32(tables), _i32(lens)
    scale, view = 1 / np.sqrt(d), dict(window=window, sinks=sinks)
    several = max(q_lens) > 1
    starts = _i32(np.concatenate([[0], np.cumsum(q_lens)]))
    if kind == "16":
        got = (ops.paged_attention_prefill(dq, kc, vc, t, n, starts, nh, nkv, scale, **view) if several else
               ops.paged_attention(dq, kc, vc, t, n, nh, nkv, scale, **view))
    else:
        s = torch.from_numpy(scales).float().cuda()
        par = dict(token_scales=(s[0].contiguous(), s[1].contiguous())) if kind == "token" else {}
        got = ops.paged_attention_int8kv(dq, kc, vc, t, n, None if par else s, None, nh, nkv, scale, q_starts=starts if several else None,
                                         **par, **view)
    args = (q, keys, values, lens, q_lens, nh, nkv, scale, window, sinks)
    steps = [np.full_like(v, 127.0) for v in values] if kind == "token" else None      # no int8 value is larger
    _hold(_np(got), args, dtype, f"window {window}, sinks {sinks}", kind, steps)
    return got


@pytest.mark.parametrize("dtype", ACT)
@pytest.mark.parametrize("nh,nkv,d,block", [(8, 2, 64, 16), (7, 1, 128, 128), (4, 4, 32, 7), (40, 2, 128, 32)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (32, 32), (33, 0), (100, 4), (130, 70), (513, 17), (4000, 1)])
def test_windowed_decode_matches_the_oracle(dtype, nh, nkv, d, block, window, sinks):
    lens = [1, 2, 31, 32, 33, 97, 0, 129, 300, 517, 64, 131, 1030]
    got = _windowed(dtype, lens, [1] * len(lens), nh, nkv, d, block, window, sinks, strided=block == 16)
    assert (got[6] == 0).all()


@pytest.mark.parametrize("kind", ["channel", "token"])
@pytest.mark.parametrize("dtype", ACT)
@pytest.mark.parametrize("nh,nkv,d,block", [(8, 2, 64, 16), (7, 1, 128, 128), (4, 4, 32, 12)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 3), (33, 40), (100, 4), (513, 17)])
def test_windowed_decode_over_int8_caches_matches_the_oracle(kind, dtype, nh, nkv, d, block, window, sinks):
    lens = [1, 32, 33, 97, 0, 129, 300, 1517]
    _windowed(dtype, lens, [1] * len(lens), nh, nkv, d, block, window, sinks, kind)


@pytest.mark.parametrize("kind", ["16", "channel", "token"])
@pytest.mark.parametrize("dtype", ACT)
@pytest.mark.parametrize("nh,nkv,d,block", [(8, 2, 64, 16), (7, 1, 128, 128), (4, 4, 32, 12), (3, 3, 128, 32)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 5), (32, 1), (40, 33), (200, 64)])
def test_windowed_chunks_match_the_oracle(kind, dtype, nh, nkv, d, block, window, sinks):
    lens, q_lens = [1, 40, 300, 97, 700, 5, 128], [1, 40, 1, 33, 150, 2, 64]
    _windowed(dtype, lens, q_lens, nh, nkv, d, block, window, sinks, kind)


@pytest.mark.parametrize("dtype", ACT)
@pytest.mark.parametrize("window,sinks", [(100, 4), (1500, 300)])
def test_a_few_rows_behind_a_long_context_are_cut_and_joined(dtype, window, sinks):
    """Few column groups: the walk is cut into partitions, whose number differs from row to row."""
    _windowed(dtype, [1700, 2050, 130], [3, 9, 2], 8, 2, 64, 32, window, sinks)
    _windowed(dtype, [1700, 2050, 130], [3, 9, 2], 7, 1, 64, 20, window, sinks)
    _windowed(dtype, [2000], [21], 7, 1, 128, 128, window, sinks, "token")
    _windowed(dtype, [2000, 900], [21, 40], 6, 2, 64, 16, window, sinks, "channel")


def _packed(dtype, q_lens, nh, nkv, d, window, sinks, seed=0, sliced=False, extra=0):
    from helpers import rounded
    from mindformers_amd import ops
    rng = np.random.default_rng(seed)
    t = int(np.sum(q_lens))
    q, k, v = (rounded(rng.normal(0, 1, (t + extra, h * d)), dtype) for h in (nh, nkv, nkv))
    dq, dk, dv = (torch.from_numpy(x).to(dtype).cuda() for x in (q, k, v))
    if sliced:
        fused = torch.cat([dq, dk, dv], dim=1)
        dq, dk, dv = fused[:, :nh * d], fused[:, nh * d:(nh + nkv) * d], fused[:, (nh + nkv) * d:]
    starts = _i32(np.concatenate([[0], np.cumsum(q_lens)]))
    got = ops.causal_attention_varlen(dq, dk, dv, starts, nh, nkv, 1 / np.sqrt(d), window=window, sinks=sinks)
    split = lambda x: np.split(x[:t].reshape(t, nkv, d), np.cumsum(q_lens)[:-1])  # noqa: E731
    args = (q[:t], split(k), split(v), q_lens, q_lens, nh, nkv, 1 / np.sqrt(d), window, sinks)
    _hold(_np(got)[:t], args, dtype, "packed rows")
    assert (got[t:] == 0).all()


@pytest.mark.parametrize("dtype", ACT)
@pytest.mark.parametrize("nh,nkv,d", [(8, 2, 64), (7, 1, 128), (4, 4, 32)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (31, 3), (64, 0), (129, 33), (5000, 7)])
def test_windowed_prompts_match_the_oracle(dtype, nh, nkv, d, window, sinks):
    _packed(dtype, [1, 300, 33, 2, 450], nh, nkv, d, window, sinks, sliced=nh == 7)


def test_windowed_prompts_of_one_row_and_rows_of_no_sequence():
    _packed(torch.bfloat16, [1], 8, 2, 64, 1, 0)
    _packed(torch.bfloat16, [1], 8, 2, 64, 7, 9, extra=5)
    _packed(torch.float16, [200, 3], 28, 4, 128, 50, 4, extra=3)


def test_a_window_as_long_as_the_context_is_the_whole_context():
    from mindformers_amd import ops
    rng = np.random.default_rng(1)
    q, cache, _, tables, _, _ = _paged(rng, torch.bfloat16, [700, 64, 1], [1, 1, 1], 8, 2, 128, 128, 10 ** 6, 0, poison=False)
    dq, kc, vc = (torch.from_numpy(x).bfloat16().cuda() for x in (q, *cache))
    t, n = _i32(tables), _i32([700, 64, 1])
    whole = ops.paged_attention(dq, kc, vc, t, n, 8, 2, 0.09)
    for window, sinks in ((700, 0), (2 ** 40, 2 ** 40), (1, 700)):
        got = ops.paged_attention(dq, kc, vc, t, n, 8, 2, 0.09, window=window, sinks=sinks)
        assert (got.float() - whole.float()).abs().max() <= 2 * 2.0 ** -8 * vc.float().abs().max()


@pytest.mark.parametrize("tiled", [False, True])
@pytest.mark.parametrize("b,hi,window", [(3, 40, 20), (5, 1500, 900), (70, 200, 64)])
def test_windowed_decode_with_quantised_output_equals_two_calls(tiled, b, hi, window):
    from mindformers_amd import ops
    rng = np.random.default_rng(b)
    lens = rng.integers(1, hi + 1, b)
    q, cache, _, tables, _, _ = _paged(rng, torch.bfloat16, lens, [1] * b, 8, 2, 64, 16, window, 5)
    dq, kc, vc = (torch.from_numpy(x).bfloat16().cuda() for x in (q, *cache))
    smooth = torch.rand(512, device="cuda") + 0.5
    args = (dq, kc, vc, _i32(tables), _i32(lens), 8, 2, 0.1)
    want = ops.paged_attention(*args, window=window, sinks=5)
    out, xq, xs = ops.paged_attention(*args, quant=(smooth, tiled), window=window, sinks=5)
    wq, ws = ops.dynamic_quant(want, smooth, tiled=tiled)
    raw = lambda x: x.data if tiled else x  # noqa: E731
    assert torch.equal(out, want) and torch.equal(xs, ws)
    if b % 16 == 0 or not tiled:
        assert torch.equal(raw(xq), raw(wq))


def test_windowed_attention_of_a_cache_past_4_gib():
    """Blocks whose offsets pass 32 bits in bytes and in elements."""
    from mindformers_amd import ops
    nb, bs = 40000, 128                                       # 10.5 GB a cache, 5.2e9 elements
    kc, vc = (torch.empty(nb, bs, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    low = torch.arange(0, 6, dtype=torch.int32, device="cuda")
    high = torch.arange(nb - 6, nb, dtype=torch.int32, device="cuda")
    for c in (kc, vc):
        c[low.long()] = torch.randn(6, bs, 8, 128, device="cuda").bfloat16()
        c[high.long()] = c[low.long()]
    q = torch.randn(2, 4096, device="cuda").bfloat16()
    lens = _i32([700, 555])
    for window, sinks in ((300, 4), (64, 200)):
        a, b = (ops.paged_attention(q, kc, vc, x[None].repeat(2, 1), lens, 32, 8, 0.09, window=window, sinks=sinks) for x in (low, high))
        assert torch.equal(a, b) and a.float().abs().sum() > 0
        starts = _i32([0, 40, 60])
        rows = torch.randn(60, 4096, device="cuda").bfloat16()
        a, b = (ops.paged_attention_prefill(rows, kc, vc, x[None].repeat(2, 1), lens, starts, 32, 8, 0.09, window=window, sinks=sinks)
                for x in (low, high))
        assert torch.equal(a, b) and a.float().abs().sum() > 0


def test_windowed_attention_replayed_in_a_graph():
    from mindformers_amd import ops
    rng = np.random.default_rng(6)
    lens = rng.integers(1, 900, 9)
    q, cache, _, tables, _, _ = _paged(rng, torch.float16, lens, [1] * 9, 8, 2, 64, 16, 300, 4, poison=False)
    dq, kc, vc = (torch.from_numpy(x).half().cuda() for x in (q, *cache))
    t, n = _i32(tables), _i32(lens)
    call = lambda: ops.paged_attention(dq, kc, vc, t, n, 8, 2, 0.1, window=300, sinks=4)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for _ in range(3):
        n.copy_(_i32(np.minimum(rng.integers(1, 900, 9), lens)))
        dq.copy_(torch.randn_like(dq))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, call())


def test_windows_that_are_refused():
    from mindformers_amd import ops
    q = torch.zeros(2, 512, dtype=torch.bfloat16, device="cuda")
    kc = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    t, n, starts = _i32(np.zeros((2, 2))), _i32([3, 4]), _i32([0, 1, 2])
    for view in (dict(window=0), dict(window=-4), dict(window=2.5), dict(window=4, sinks=-1), dict(sinks=3)):
        for call in (lambda: ops.paged_attention(q, kc, kc, t, n, 8, 2, 0.1, **view),
                     lambda: ops.paged_attention_prefill(q, kc, kc, t, n, starts, 8, 2, 0.1, **view),
                     lambda: ops.causal_attention_varlen(q, q[:, :128], q[:, :128], starts, 8, 2, 0.1, **view)):
            with pytest.raises(ValueError):
                call()
    wide = torch.zeros(2, 384, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="heads of 32, 64 or 128"):
        ops.causal_attention_varlen(wide, wide, wide, starts, 2, 2, 0.1, window=4)
    with pytest.raises(ValueError):
        ops.causal_attention_varlen(wide, wide, torch.zeros(2, 256, dtype=torch.bfloat16, device="cuda"), starts, 2, 2, 0.1, window=4)
