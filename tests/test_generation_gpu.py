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


def test_selection_of_the_last_rows_of_sequences():
    """Logits [groups, beams, vocab] that are slices: one beam a group with the rows of a longer step between, and beams of one group."""
    wide = torch.randn(5, 7, 301, device="cuda")
    scores = torch.randn(5, 1, device="cuda")
    from mindformers_amd import ops
    for got, want in zip(ops.beam_search_select(wide[:, -1:], scores), ops.beam_search_select(wide[:, -1].contiguous(), scores)):
        assert torch.equal(got, want)
    for got, want in zip(ops.beam_search_select(wide[2:3, ::2], scores[:4].view(1, 4)), ops.beam_search_select(wide[2, ::2].contiguous(), scores[:4].view(1, 4))):
        assert torch.equal(got, want)
    for bad in (wide[:, ::3], wide.transpose(1, 2)[:, :1], wide[:1, :1].expand(5, 1, 301)):
        with pytest.raises(ValueError):
            ops.beam_search_select(bad, torch.zeros(5, bad.shape[1], device="cuda"))


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


@pytest.mark.parametrize("new", [5, 40])
def test_a_row_as_long_as_its_table_takes_no_block_from_another(new):
    tables = np.full((3, 8), -1)
    tables[0], tables[1, 0], tables[2] = np.arange(8), 8, np.arange(9, 17)
    need = -(-new // 8)
    got = _fork(tables, np.array([64, 8, 64]), 17 + need, 8, new_tokens=new)       # the pool holds what row 1 needs
    assert int(got.missing) == 2 * need and (_np(got.slot_mapping).reshape(3, new)[1] >= 0).all()


def test_fork_ignores_entries_that_name_no_block():
    tables = np.array([[3, 99, -7, 2], [0, 1, -1, -1], [5, 6, 7, 8]])
    got = _fork(tables, np.array([7, 3, -4]), 10, 2, parents=np.array([0, 0, 2]), new_tokens=1)
    assert got.block_tables[0, 1] == -1 and got.context_lens[2] == 1


@pytest.mark.parametrize("rows,width,block,new,blocks", [(64, 257, 3, 1, 16500), (64, 256, 1, 2, 40001), (300, 100, 2, 20, 33001), (1030, 33, 2, 1, 70000),
                                                         (70, 300, 2, 1, 1 << 20), (9, 16000, 1, 1, 150001)])
def test_fork_of_large_tables_matches_the_oracle(rows, width, block, new, blocks):
    rng = np.random.default_rng(width)
    used = rows * width
    tables, lens = _tables(rng, rows, width, block, min(blocks, used + 9) if blocks < (1 << 20) else used, groups=7) if blocks > used else (
        rng.integers(-1, blocks + 2, (rows, width)), rng.integers(0, width * block + 1, rows))
    if blocks == 1 << 20:
        tables = np.where(tables >= 0, (1 << 20) - 1 - 37 * tables, -1)   # the upper end of the pool too
    held = rng.random(blocks) < 0.5
    for kw in (dict(), dict(parents=rng.integers(-1, rows, rows), held=held), dict(parents=rng.integers(0, rows, rows), window=width // 2, sinks=1)):
        _fork(tables, lens, blocks, block, new_tokens=new, **kw)


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


# The largest key of the queries' channel is the first token that the window leaves, which takes the whole probability where the
# scores are 2^31 apart; where they are 2^-40 the probabilities are equal.
@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 2.0 ** 40), (torch.bfloat16, 2.0 ** -50), (torch.bfloat16, 2.0 ** 25), (torch.float16, 2.0 ** 15),
                                        (torch.float16, 2.0 ** -24), (torch.bfloat16, 0.0), (torch.bfloat16, 2.0 ** -110)])
@pytest.mark.parametrize("rows", [1, 20, 200])
@pytest.mark.parametrize("window,sinks", [(40, 0), (70, 1)])
def test_windows_over_int8_caches_with_large_and_small_queries(dtype, size, rows, window, sinks):
    from mindformers_amd import ops
    rng = np.random.default_rng(rows)
    lens, nh, nkv, d, block = [255, 254, 0, 255], 8, 2, 64, 16
    q_lens = [rows, 1, 0, rows]
    q = np.zeros((sum(q_lens), nh, d))
    q[:, :, 5] = size
    cache = rng.integers(-127, 128, (2, 64, block, nkv, d))
    cache[0].reshape(4, 256, nkv, d)[..., 5] = 127 - np.minimum(np.arange(256), 254)[None, :, None]
    tables = np.arange(64).reshape(4, 16)
    keys, values = ([c.reshape(4, 256, nkv, d)[b, :n] / 128.0 for b, n in enumerate(lens)] for c in cache)
    dq = torch.from_numpy(q.reshape(-1, nh * d)).to(dtype).cuda()
    assert (_np(dq) == q.reshape(-1, nh * d)).all()
    kc, vc = (torch.from_numpy(c).to(torch.int8).cuda() for c in cache)
    got = ops.paged_attention_int8kv(dq, kc, vc, _i32(tables), _i32(lens), torch.full((2, nkv * d), 1 / 128.0, device="cuda"), None, nh, nkv,
                                     0.125, q_starts=_i32(np.concatenate([[0], np.cumsum(q_lens)])), window=window, sinks=sinks)
    _hold(_np(got), (q.reshape(-1, nh * d), keys, values, lens, q_lens, nh, nkv, 0.125, window, sinks), dtype, f"size {size}", "channel",
          [np.full_like(v, 127.0) for v in values])


@pytest.mark.parametrize("kind", ["16", "channel", "token"])
@pytest.mark.parametrize("dtype", ACT)
@pytest.mark.parametrize("window,sinks", [(2000, 3), (40, 2 ** 31 - 1), (2 ** 31 - 1, 0), (20, 0)])
def test_rows_of_no_sequence_are_zero_and_their_queries_unread(kind, dtype, window, sinks):
    from mindformers_amd import ops
    rng = np.random.default_rng(11)
    lens, q_lens, nh, nkv, d, block = np.array([3000, 0, 700, 9]), np.array([4, 0, 5, 9]), 4, 2, 64, 16
    q, cache, scales, tables, keys, values = _paged(rng, dtype, lens, q_lens, nh, nkv, d, block, window, sinks, kind)
    wide = torch.full((27, nh * d), float("nan"), dtype=dtype, device="cuda")
    wide[3:21] = torch.from_numpy(q).to(dtype)
    out = torch.full_like(wide, float("nan"))
    kc, vc = (torch.from_numpy(c).to(dtype if kind == "16" else torch.int8).cuda() for c in cache)
    t, n, starts, scale = _i32(tables), _i32(lens), _i32([3, 7, 7, 12, 21]), 1 / np.sqrt(d)
    view = dict(window=window, sinks=sinks, out=out)
    if kind == "16":
        ops.paged_attention_prefill(wide, kc, vc, t, n, starts, nh, nkv, scale, **view)
    else:
        s = torch.from_numpy(scales).float().cuda()
        par = dict(token_scales=(s[0].contiguous(), s[1].contiguous())) if kind == "token" else {}
        ops.paged_attention_int8kv(wide, kc, vc, t, n, None if par else s, None, nh, nkv, scale, q_starts=starts, **par, **view)
    assert (out[:3] == 0).all() and (out[21:] == 0).all()
    _hold(_np(out[3:21]), (q, keys, values, lens, q_lens, nh, nkv, scale, window, sinks), dtype, f"window {window}, sinks {sinks}", kind,
          [np.full_like(v, 127.0) for v in values] if kind == "token" else None)


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


# --------------------------------------------------------------------------------------------- the operators together
def _stack(window, sinks, act_quant=False, dtype=torch.bfloat16, seed=3, n=2):
    from mindformers_amd import synthetic
    from mindformers_amd.decode_layer import QuantDecodeLayer
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return [synthetic.fill_layer(QuantDecodeLayer(512, 8, 2, 64, 1024, 1e-5, dtype, act_quant, window=window, sinks=sinks), gen)
            for _ in range(n)]


@pytest.mark.parametrize("window,sinks", [(None, 0), (24, 3)])
def test_a_beam_search_over_shared_blocks_is_one_over_private_ones(window, sinks):
    """Beam search of three prompts through a two-layer stack whose beams share blocks, against the same search with every beam's
    cache copied as a whole to blocks of its own: the same tokens, and the layers' outputs bit for bit."""
    from mindformers_amd import ops
    from mindformers_amd.modules import BeamSearch, BlockTables
    from mindformers_amd.runner import DecodeStackRunner
    bs, width, k, vocab, steps = 8, 9, 3, 211, 30
    layers = _stack(window, sinks)
    shared, private = (DecodeStackRunner(layers, npu_mem_size=0.004, cpu_mem_size=0, block_size=bs) for _ in range(2))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(11)
    embed = torch.randn(vocab, 512, generator=gen, device="cuda").bfloat16()
    head = torch.randn(512, vocab, generator=gen, device="cuda") / 16
    lens = np.array([13, 1, 32])
    blocks = BlockTables(shared.npu_num_blocks, bs, width * bs)
    blocks.init_cache_engine(3)
    tables, slots = blocks.assemble_pa_full_inputs(32, lens, [False] * 3)
    slots = slots.reshape(3, -1)
    words = [torch.randint(0, vocab, (int(n),), generator=gen, device="cuda") for n in lens]
    x = embed[torch.cat(words)]
    hidden = shared.forward(x, lens, tables, np.concatenate([slots[i, :n] for i, n in enumerate(lens)]), prefill=True)
    first = hidden[torch.tensor(np.cumsum(lens) - 1, device="cuda")].float() @ head

    rows = 3 * k
    own = torch.arange(rows * width, device="cuda", dtype=torch.int32).view(rows, width)
    assert private.npu_num_blocks >= rows * width
    for a, b in zip(shared.caches(), private.caches()):
        for r in range(rows):
            for j in range(-(-int(lens[r // k]) // bs)):
                b[own[r, j].item()] = a[int(tables[r // k, j])]

    search = BeamSearch(shared.caches(), k, eos_token_id=5, window=window, sinks=sinks)
    tokens = search.start(tables, lens, first)
    beams = [[] for _ in range(rows)]                         # the tokens of every row, kept on the host
    scores = torch.full((3, k), -torch.inf, device="cuda")
    scores[:, 0] = 0
    logits, n = first.repeat_interleave(k, 0), torch.from_numpy(lens).cuda().repeat_interleave(k)
    finished = [[] for _ in range(3)]
    for step in range(steps):
        sel = ops.beam_search_select(logits, scores, eos_token_id=5)
        assert torch.equal(sel.next_tokens.view(-1), tokens)
        for g in range(3):
            for s, b, t in zip(sel.scores[g, :k].tolist(), sel.beams[g, :k].tolist(), sel.tokens[g, :k].tolist()):
                if t == 5 and np.isfinite(s):
                    finished[g].append((s / (step + 1), beams[g * k + b] + [5]))
        parents, scores = sel.next_rows.view(-1), sel.next_scores
        beams = [beams[p] + [t] for p, t in zip(parents.tolist(), tokens.tolist())]
        for c in private.caches():
            c[:rows * width] = c[:rows * width].view(rows, width, *c.shape[1:])[parents.long()].view(rows * width, *c.shape[1:])
        n = n + 1
        slot = own[torch.arange(rows, device="cuda"), (n - 1) // bs] * bs + ((n - 1) % bs).int()
        got = shared.decode(embed[tokens.long()], search.context_lens, search.block_tables, search.slot_mapping)
        want = private.decode(embed[tokens.long()], n.int(), own, slot.int())
        assert torch.equal(got, want), f"step {step}"
        if step == 12:
            before = torch.unique(search.block_tables[search.block_tables >= 0]).numel()
            assert int(search.compact()) == before and int(search.block_tables.max()) == before - 1
        logits = got.float() @ head
        if step + 1 < steps:
            tokens = search.step(logits)
    used = torch.unique(search.block_tables[search.block_tables >= 0]).numel()
    assert used < 9 * 6 and (window is None or used <= 9 * 4 + 9)
    live = [[(s / steps, beams[g * k + i]) for i, s in enumerate(scores[g].tolist())] for g in range(3)]
    for g, found in enumerate(search.hypotheses()):
        assert sorted(t for _, t in found) == sorted(t for _, t in finished[g] + live[g])
        assert [s for s, _ in found] == sorted((s for s, _ in found), reverse=True)
        np.testing.assert_allclose(sorted(s for s, _ in found), sorted(s for s, _ in finished[g] + live[g]), rtol=1e-12)
    search.release([1])
    search.step(logits)
    assert (search.block_tables[k:2 * k] == -1).all() and (search.slot_mapping[k:2 * k] == -1).all()
    assert (search.context_lens[k:2 * k] == 0).all() and (search.slot_mapping[:k] >= 0).all()
    again = shared.decode(embed[tokens.long()], search.context_lens, search.block_tables, search.slot_mapping)
    assert torch.isfinite(again.float()).all()


def test_a_beam_search_without_blocks_says_so():
    from mindformers_amd.modules import BeamSearch
    caches = [torch.zeros(4, 4, 1, 32, dtype=torch.float16, device="cuda")]
    search = BeamSearch(caches, 4)
    search.start(np.array([[0, 1, -1, -1]]), np.array([7]), torch.randn(1, 50, device="cuda"))
    with pytest.raises(RuntimeError, match="short"):          # 1 prompt block and 4 open ones do not fit 4 blocks
        search.hypotheses()


@pytest.mark.parametrize("act_quant", [False, True])
@pytest.mark.parametrize("rows", [3, 40])
def test_a_windowed_layer_is_a_full_one_on_the_tokens_that_it_sees(act_quant, rows, dtype=torch.bfloat16):
    """A decode step through a window without sinks against the same layer without a window on a cache that holds the window's
    tokens only: the same operands in another place (the tiles of a walk start at multiples of 32, so do the copies here)."""
    bs, window = 32, 64
    layer, = _stack(window, 0, act_quant, dtype, n=1)
    full, = _stack(None, 0, act_quant, dtype, n=1)
    nb = rows * 8
    kc, vc = (torch.randn(nb, bs, 2, 64, device="cuda").to(dtype) for _ in range(2))
    tables = torch.randperm(nb, device="cuda").int().view(rows, 8)
    n = torch.full((rows,), 160, dtype=torch.int32, device="cuda")       # the window is tokens 96 to 159: blocks 3 and 4
    slots = tables[:, 4] * bs + 31
    x = torch.randn(rows, 512, device="cuda").to(dtype)
    cos, sin = torch.ones(rows, 64, device="cuda").to(dtype), torch.zeros(rows, 64, device="cuda").to(dtype)
    k2, v2 = kc.clone(), vc.clone()
    hidden = tables.clone()
    hidden[:, :3] = -1
    got = layer(x, kc, vc, hidden, n, slots, cos, sin)
    want = full(x, k2, v2, tables[:, 3:].contiguous(), torch.full_like(n, 64), slots, cos, sin)
    assert torch.equal(kc, k2) and torch.equal(vc, v2)
    assert torch.equal(got, want)


def test_a_layer_from_a_checkpoint_has_its_window_over_16_bit_and_int8_caches():
    from mindformers_amd import checkpoint, ops
    rng = np.random.default_rng(5)
    nh, nkv, d, ffn, bs, rows = 8, 2, 64, 512, 32, 5
    cfg = dict(num_heads=nh, n_kv_heads=nkv, hidden_size=nh * d, intermediate_size=ffn, qkv_concat=False)
    hf = {f"model.layers.0.{name}.weight": rng.normal(0, 0.03, shape).astype(np.float32) for name, shape in (
        ("self_attn.q_proj", (512, 512)), ("self_attn.k_proj", (128, 512)), ("self_attn.v_proj", (128, 512)), ("self_attn.o_proj", (512, 512)),
        ("mlp.gate_proj", (ffn, 512)), ("mlp.up_proj", (ffn, 512)), ("mlp.down_proj", (512, ffn)))}
    hf.update({f"model.layers.0.{name}.weight": np.ones(512, np.float32) for name in ("input_layernorm", "post_attention_layernorm")})
    layer, full = (checkpoint.load_decode_layer(hf, 0, cfg, dtype=torch.bfloat16, **view) for view in (dict(window=64, sinks=0), {}))
    assert (layer.window, layer.sinks, full.window) == (64, 0, None)
    tables = torch.randperm(rows * 8, device="cuda").int().view(rows, 8)
    n = torch.full((rows,), 160, dtype=torch.int32, device="cuda")       # the window is tokens 96 to 159: blocks 3 and 4
    x, slots = torch.randn(rows, 512, device="cuda").bfloat16(), tables[:, 4] * bs + 31
    cos, sin = torch.ones(rows, d, device="cuda").bfloat16(), torch.zeros(rows, d, device="cuda").bfloat16()
    caches = [torch.randn(rows * 8, bs, nkv, d, device="cuda").bfloat16() for _ in range(2)]
    hidden = tables.clone()
    hidden[:, :3] = -1
    got = layer(x, *[c.clone() for c in caches], hidden, n, slots, cos, sin)
    assert torch.equal(got, full(x, *[c.clone() for c in caches], tables[:, 3:].contiguous(), torch.full_like(n, 64), slots, cos, sin))
    scale = torch.full((2, nkv * d), 2.0 ** -5, device="cuda")
    layer.set_kv_quant(scale)
    kc, vc = (torch.randint(-127, 128, (rows * 8, bs, nkv, d), device="cuda").to(torch.int8) for _ in range(2))
    want = ops.paged_attention_int8kv(x, kc, vc, hidden, n, scale, None, nh, nkv, layer.scale_value, window=64)
    assert torch.equal(layer.attend(x, kc, vc, hidden, n).view_as(want), want)
    k2, v2 = kc.clone(), vc.clone()
    out = layer(x, k2, v2, hidden, n, slots, cos, sin)
    written = torch.zeros(rows * 8 * bs, dtype=torch.bool, device="cuda")
    written[slots.long()] = True
    assert torch.isfinite(out.float()).all()
    for old, new in ((kc, k2), (vc, v2)):
        assert torch.equal(old.view(-1, nkv * d)[~written], new.view(-1, nkv * d)[~written])


def test_the_modules_pass_their_window_on():
    """InferAttention and FlashAttention in every form of their attention, a manager and its quantised successor."""
    from mindformers_amd import ops
    from mindformers_amd.modules import FlashAttention, InferAttention, PagedAttentionMgr, QuantPagedAttentionMgr
    nh, nkv, d, bs, nb, view = 4, 2, 64, 16, 12, dict(window=20, sinks=2)
    t = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    n = _i32([50, 33])
    mk = lambda r, h: torch.randn(r, h * d, device="cuda").half()  # noqa: E731
    q, k, v = mk(2, nh), mk(2, nkv), mk(2, nkv)
    slots = torch.tensor([3 * 16 + 1, 4 * 16 + 2 * 16], dtype=torch.int32, device="cuda")
    attn = InferAttention(nh, d, nkv, scale_value=0.1, block_size=bs, num_blocks=nb, use_rope_rotary_emb=False, **view)
    mgr = attn.paged_attention_mgr
    mgr.scale_value = 0.1
    mgr.key_cache.normal_()
    mgr.value_cache.normal_()
    attn.is_first_iteration = False
    got = attn(q, k, v, n, t, slots)
    want = ops.paged_attention(q, mgr.key_cache, mgr.value_cache, t, n, nh, nkv, 0.1, **view)
    assert torch.equal(got, want) and not torch.equal(got, ops.paged_attention(q, mgr.key_cache, mgr.value_cache, t, n, nh, nkv, 0.1))
    flash = FlashAttention(nh, d, nkv, scale_value=0.1, **view)
    flash.is_prefill = False
    assert torch.equal(flash(q, k, v, slots, t, n, key_cache=mgr.key_cache, value_cache=mgr.value_cache), want)
    # prompts
    q, k, v = mk(60, nh), mk(60, nkv), mk(60, nkv)
    ends, starts = _i32([37, 60]), _i32([0, 37, 60])
    want = ops.causal_attention_varlen(q, k, v, starts, nh, nkv, 0.1, **view)
    none = torch.full((60,), -1, dtype=torch.int32, device="cuda")
    flash.is_prefill = attn.is_first_iteration = True
    assert torch.equal(flash(q, k, v, none, actual_seq_qlen=ends, key_cache=mgr.key_cache, value_cache=mgr.value_cache), want)
    assert torch.equal(attn(q, k, v, ends, t, none), want)
    # chunks
    q, lens = mk(9, nh), _i32([5, 4])
    chunked = PagedAttentionMgr(nh, d, nkv, (nb, bs, nkv, d), chunk_prefill=True, **view)
    chunked.key_cache.copy_(mgr.key_cache)
    chunked.value_cache.copy_(mgr.value_cache)
    want = ops.paged_attention_prefill(q, mgr.key_cache, mgr.value_cache, t, n, _i32([0, 5, 9]), nh, nkv, chunked.scale_value, **view)
    assert torch.equal(chunked.paged_attn(q, n, t, q_seq_lens=lens), want)
    for gran in ("per_channel", "per_token"):
        quant = QuantPagedAttentionMgr.from_float(chunked, gran)
        assert (quant.window, quant.sinks) == (20, 2)
        quant.key_cache.random_(-100, 100)
        quant.value_cache.random_(-100, 100)
        if gran == "per_token":
            quant.key_scale_cache.fill_(0.01)
            quant.value_scale_cache.fill_(0.01)
        out = quant.paged_attn(q, n, t, q_seq_lens=lens)
        quant.window = None
        assert not torch.equal(out, quant.paged_attn(q, n, t, q_seq_lens=lens))
    with pytest.raises(NotImplementedError):
        FlashAttention(nh, d, nkv, pa_mla_v_dim=512, **view)
    for make in (lambda: InferAttention(nh, d, nkv, window=0), lambda: FlashAttention(nh, d, nkv, sinks=3),
                 lambda: PagedAttentionMgr(nh, d, nkv, (nb, bs, nkv, d), window=-1)):
        with pytest.raises(ValueError):
            make()


@pytest.mark.parametrize("rows,width,block,new", [(3, 40, 16, 500), (70, 30, 8, 17), (5, 6, 4, 40), (1, 1, 1, 300)])
def test_fork_with_the_tokens_of_a_prompt(rows, width, block, new):
    """More new tokens than a thread places by itself, and more than the table or the pool holds."""
    rng = np.random.default_rng(new)
    blocks = rows * (width + 1)
    tables, lens = _tables(rng, rows, width, block, blocks, groups=2)
    lens[0] = 0
    for parents in (None, rng.integers(-1, rows, rows)):
        _fork(tables, lens, blocks, block, parents=parents, new_tokens=new)
        _fork(tables, lens, max(blocks // 3, int(tables.max()) + 1, 1), block, parents=parents, new_tokens=new)


def test_graphs_replayed_at_once_share_no_workspace():
    """Two captures of each operator, replayed together on two streams over and over: the answers of one are never the other's."""
    from mindformers_amd import ops
    rng = np.random.default_rng(3)
    sets = []
    for seed in (1, 2):
        lens = rng.integers(1000, 1500, 8)
        q, cache, _, tables, _, _ = _paged(rng, torch.bfloat16, lens, [1] * 8, 8, 2, 64, 16, 900, 4, poison=False)
        q, kc, vc = (torch.from_numpy(x).bfloat16().cuda() for x in (q, *cache))
        logits, scores = _beams(4, 4, 60000, torch.float32, seed)
        t, l = _tables(rng, 200, 64, 4, 200 * 70, groups=4)
        sets.append((q, kc, vc, _i32(tables), _i32(lens), logits, scores, _i32(t), _i32(l), _i32(rng.integers(-1, 200, 200))))

    def calls(q, kc, vc, tables, lens, logits, scores, t, l, p):
        fork = ops.fork_blocks(t, l, 200 * 70, 4, parents=p, new_tokens=1)
        return [ops.paged_attention(q, kc, vc, tables, lens, 8, 2, 0.1, window=900, sinks=4), *ops.beam_search_select(logits, scores),
                *fork, *ops.compact_blocks(fork.block_tables, 200 * 70, 4)]

    want = [[x.clone() for x in calls(*s)] for s in sets]
    graphs, got = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(calls(*s))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(20):
        for g, st in zip(graphs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for w, h in zip(want, got):
            assert all(torch.equal(a, b) for a, b in zip(w, h))


def test_a_device_side_decode_step_replayed_in_a_graph():
    from mindformers_amd.runner import DecodeStackRunner
    run = DecodeStackRunner(_stack(40, 3), npu_mem_size=0.004, cpu_mem_size=0, block_size=16)
    for c in run.caches():
        c.normal_()
    tables = torch.arange(32, dtype=torch.int32, device="cuda").view(4, 8)
    lens, slots = _i32([5, 0, 128, 77]), _i32([4, -1, 2 * 128 + 127, 3 * 128 + 76])
    x = torch.randn(4, 512, device="cuda").bfloat16()
    run.decode(x, lens, tables, slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run.decode(x, lens, tables, slots)
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        again = got.clone()
        assert torch.equal(again, run.decode(x, lens, tables, slots))
    with pytest.raises(ValueError):
        run.decode(x, lens.long(), tables, slots)
    with pytest.raises(ValueError):
        run.decode(x, lens, tables[:3], slots)
