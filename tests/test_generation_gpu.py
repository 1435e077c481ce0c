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
