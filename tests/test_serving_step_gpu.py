"""Operators of a serving step against their definitions in float64: rotary positions, log probabilities, low-rank adapters."""
import numpy as np
import pytest
import torch

from helpers import EPS, NAME, rounded, to_np
from oracle import serving as S

from mindformers_amd import _lib, ops

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


def _dev(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a)).to(device="cuda", dtype=dtype)


def _inv(pairs, base=10000.0):
    return base ** (-np.arange(pairs) / pairs)


# ------------------------------------------------------------------------------------------------ rotary positions
def _check_rotary(got, x, positions, inv, d, near, scale, offset, dtype, what):
    """Turned columns: the rounding of the result, half a step of it, and in float32 before that: cosines and sines within 2^-21 (turns
    rounded to 2^-25, times 2 pi; the functions' own 2 ulp), three roundings of the products and the sum.  Others: the input's bits."""
    t, p = len(positions), len(inv)
    want = S.rotary(x, positions, inv, d, near, scale, offset).reshape(t, -1, d)
    x, got = x.reshape(t, -1, d), to_np(got).astype(np.float64).reshape(t, -1, d)
    first = offset + (2 * np.arange(p) if near else np.arange(p))
    second = first + (1 if near else p)
    turned = np.zeros(d, bool)
    turned[first] = turned[second] = True
    assert np.array_equal(got[:, :, ~turned], x[:, :, ~turned]), what
    mag = abs(scale) * (np.abs(x[:, :, first]) + np.abs(x[:, :, second]))
    for c in (first, second):
        tol = EPS[dtype] * np.abs(want[:, :, c]) + mag * 2.0 ** -20 + 2.0 ** -25      # the last: fp16 values below its normal ones
        err = np.abs(got[:, :, c] - want[:, :, c])
        assert (err <= tol).all(), f"{what}: {err.max()} over {tol.flat[np.argmax(err - tol)]}"


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("t,heads,kv,d,pairs,offset", [(1, 32, 8, 128, 64, 0), (5, 28, 4, 128, 32, 0), (3, 7, 1, 80, 10, 0), (4, 4, 2, 64, 16, 32),
                                                       (2, 3, 3, 18, 9, 0), (2, 3, 1, 20, 5, 3), (6, 2, 2, 96, 24, 8), (3, 1, 1, 2, 1, 0),
                                                       (2049, 8, 2, 64, 32, 0), (2050, 3, 1, 256, 128, 0), (1, 1, 1, 1024, 512, 0),
                                                       (2051, 2, 1, 640, 300, 40), (4097, 8, 2, 64, 32, 0), (4098, 3, 1, 256, 128, 0),
                                                       (4099, 2, 1, 640, 300, 40), (4100, 1, 1, 16, 8, 0), (4101, 3, 1, 80, 10, 5), (5003, 12, 2, 64, 16, 8)])
def test_rotary_layouts_and_parts(dtype, near, t, heads, kv, d, pairs, offset):
    rng = np.random.default_rng(t * 1000 + d)
    inv = _inv(pairs)
    pos = rng.integers(0, 1 << 20, t)
    q, k = (rounded(rng.normal(size=(t, h * d)) * 2, dtype) for h in (heads, kv))
    qt, kt = _dev(q, dtype), _dev(k, dtype)
    got = ops.rotary_embedding(qt, kt, _i32(pos), torch.from_numpy(inv).cuda(), d, interleaved=near, scale=1.25, offset=offset)
    assert got[0] is qt and got[1] is kt                      # in place
    _check_rotary(qt, q, pos, inv, d, near, 1.25, offset, dtype, "query")
    _check_rotary(kt, k, pos, inv, d, near, 1.25, offset, dtype, "key")


def test_rotary_far_and_negative_positions():
    """Angles of 2^31 radians hang on their last bits: 2^31 2^-52 in float64, where float32 has nothing left."""
    rng = np.random.default_rng(0)
    pos = np.array([2 ** 31 - 1, 2 ** 31 - 2, 1999999999, 123456789, 16777217, -1, -77777, 0])
    inv = np.array([1.0, 0.7310585786300049, 1e-3, 1e-7, 0.0])
    x = rounded(rng.normal(size=(8, 20)), BF)
    xt = _dev(x, BF)
    ops.rotary_embedding(xt, None, _i32(pos), torch.from_numpy(inv).cuda(), 10)
    _check_rotary(xt, x, pos, inv, 10, False, 1.0, 0, BF, "query")


@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,pad", [(37, 0), (37, 1), (37, 2), (37, 4), (37, 8), (4111, 0), (4111, 2), (4111, 8)])
def test_rotary_of_column_slices_into_a_cache(dtype, near, t, pad):
    """query, key and value as slices of a fused projection whose rows are `pad` columns further apart (every width of access), into outputs
    of their own and the cache; rows of slots outside of it leave the cache as it was."""
    rng = np.random.default_rng(pad)
    h, kv, d, pairs, off = 6, 2, 48, 16, 8
    inv = _inv(pairs)
    wide = rounded(rng.normal(size=(t, (h + 2 * kv) * d + pad)), dtype)
    qkv = _dev(wide, dtype)
    q, k, v = qkv[:, :h * d], qkv[:, h * d:(h + kv) * d], qkv[:, (h + kv) * d:(h + 2 * kv) * d]
    pos = rng.integers(0, 5000, t)
    nb, bs = t // 16 + 3, 16
    slots = rng.permutation(nb * bs)[:t]
    slots[[3, 11, 20]] = [-1, nb * bs, 2 ** 31 - 1]
    kc, vc = (rounded(rng.normal(size=(nb, bs, kv, d)), dtype) for _ in range(2))
    kct, vct = _dev(kc, dtype), _dev(vc, dtype)
    q_out = torch.full((t, h * d + pad), 9.0, dtype=dtype, device="cuda")[:, :h * d]
    args = (_i32(pos), torch.from_numpy(inv).cuda(), d)
    more = dict(interleaved=near, offset=off, value=v, key_cache=kct, value_cache=vct, slot_mapping=_i32(slots))
    got = ops.rotary_embedding(q, k, *args, out=(q_out, None), **more)
    assert got[0].data_ptr() == q_out.data_ptr() and got[1] is None
    assert torch.equal(qkv, _dev(wide, dtype))                # inputs as they were
    _check_rotary(q_out, wide[:, :h * d], pos, inv, d, near, 1.0, off, dtype, "query")
    ok = (slots >= 0) & (slots < nb * bs)
    cached = kct.reshape(-1, kv * d)
    _check_rotary(cached[torch.from_numpy(slots[ok]).cuda()], wide[ok, h * d:(h + kv) * d], pos[ok], inv, d, near, 1.0, off, dtype, "key cache")
    vc.reshape(-1, kv * d)[slots[ok]] = wide[ok, (h + kv) * d:(h + 2 * kv) * d]
    assert np.array_equal(to_np(vct), vc)
    rest = np.setdiff1d(np.arange(nb * bs), slots[ok])
    assert np.array_equal(to_np(cached)[rest], kc.reshape(-1, kv * d)[rest])
    # in place, with the caches: the same bits
    first = (q_out.clone(), kct.clone())
    ops.rotary_embedding(q, k, *args, **more)
    assert torch.equal(q, first[0]) and torch.equal(kct, first[1])
    assert torch.equal(k[torch.from_numpy(np.flatnonzero(ok)).cuda()], cached[torch.from_numpy(slots[ok]).cuda()])
    # into a key of its own, without caches
    again = _dev(wide, dtype)
    k_out = torch.empty((t, kv * d), dtype=dtype, device="cuda")
    ops.rotary_embedding(again[:, :h * d], again[:, h * d:(h + kv) * d], *args, interleaved=near, offset=off, out=(q_out, k_out))
    assert torch.equal(q_out, first[0]) and torch.equal(k_out, k)


@pytest.mark.parametrize("dtype,near,d,pairs", [(BF, False, 128, 64), (FP, True, 128, 32), (BF, True, 80, 10)])
def test_rotary_of_long_inputs_is_that_of_their_pieces(dtype, near, d, pairs):
    """Inputs of more than 80 MB, which are read another way, and their thirds: the same bits, into outputs, a cache and in place."""
    t, h, kv = 10007 * 128 // d, 28, 4
    gen = torch.Generator(device="cuda").manual_seed(d)
    qkv = torch.randn(t, (h + 2 * kv) * d, generator=gen, device="cuda").to(dtype)
    pos, slots = torch.arange(t, dtype=torch.int32, device="cuda") * 7, torch.arange(t, dtype=torch.int32, device="cuda")
    inv = torch.from_numpy(_inv(pairs)).cuda()

    def turn(cuts):
        q_out = torch.empty(t, h * d, dtype=dtype, device="cuda")
        kc, vc = (torch.zeros(t // 16 + 1, 16, kv, d, dtype=dtype, device="cuda") for _ in range(2))
        rows = qkv.clone()
        for a, b in zip([0, *cuts], [*cuts, t]):
            x = rows[a:b]
            q, k, v = x[:, :h * d], x[:, h * d:(h + kv) * d], x[:, (h + kv) * d:]
            more = dict(interleaved=near, value=v, key_cache=kc, value_cache=vc, slot_mapping=slots[a:b])
            ops.rotary_embedding(q, k, pos[a:b], inv, d, out=(q_out[a:b], None), **more)
            ops.rotary_embedding(q, k, pos[a:b], inv, d, interleaved=near)
        return q_out, kc, vc, rows

    for whole, thirds in zip(turn([]), turn([t // 3, t // 3 * 2])):
        assert torch.equal(whole, thirds)


def test_rotary_equals_the_cell_of_the_tables_at_near_positions():
    """Against apply_rotary_pos_emb on float32 rows of the same angles: the same formula, within the roundings of both."""
    rng = np.random.default_rng(1)
    t, h, d = 9, 4, 64
    inv = (1.0 / np.float32(10000.0) ** (np.arange(0, d, 2, dtype=np.float32) / np.float32(d))).astype(np.float32)
    x = rounded(rng.normal(size=(t, h * d)), BF)
    ang = np.arange(t)[:, None] * inv[None].astype(np.float64)
    cos, sin = (torch.from_numpy(np.tile(f(ang), 2).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    a, b = _dev(x, BF), _dev(x, BF)
    ops.apply_rotary_pos_emb(a, None, cos, sin, h, 0, d)
    ops.rotary_embedding(b, None, _i32(np.arange(t)), torch.from_numpy(inv.astype(np.float64)).cuda(), d)
    _check_rotary(b, x, np.arange(t), inv, d, False, 1.0, 0, BF, "query")
    assert (a != b).float().mean() < 0.01                     # near-ties of the rounding


def test_rotary_of_infinite_and_nan_values_stays_in_their_pairs():
    x = rounded(np.random.default_rng(2).normal(size=(2, 64)), BF)
    for near in (False, True):
        y = x.copy()
        y[0, 3], y[1, 40], y[1, 63] = np.inf, np.nan, -np.inf
        clean, got = _dev(x, BF), _dev(y, BF)
        args = (_i32([5, 9]), torch.from_numpy(_inv(10)).cuda(), 32)
        ops.rotary_embedding(clean, None, *args, interleaved=near)
        ops.rotary_embedding(got, None, *args, interleaved=near)
        touched = np.zeros((2, 64), bool)
        for r, c in ((0, 3), (1, 40), (1, 63)):
            touched[r, c] = True
            if c % 32 < 20:
                touched[r, (c // 2 * 2 + 1 - c % 2) if near else c // 32 * 32 + (c % 32 + 10) % 20] = True
        same = (clean.view(torch.int16) == got.view(torch.int16)).cpu().numpy()
        assert same[~touched].all() and not np.isfinite(to_np(got)[touched]).any()


def test_rotary_of_no_rows():
    q = torch.empty((0, 64), dtype=BF, device="cuda")
    assert ops.rotary_embedding(q, None, _i32([]), torch.from_numpy(_inv(32)).cuda(), 64)[0] is q


# ------------------------------------------------------------------------------------------------ log probabilities
def _check_logprobs(logits, tokens, n):
    """Whole numbers exactly.  Log probabilities and entropy: float32 sums of v terms, whose errors go the way of sqrt(v) 2^-24 at most
    (each lane adds v / 64 of them or fewer, pairwise behind that), terms within 2^-21 (the exponential's argument rounded at up to
    8 in the terms that count, its own error), and the rounding of a result of this size."""
    got = ops.token_logprobs(logits, _i32(tokens), n_top=n)
    lp, rank, entropy, top, top_lp = S.token_logprobs(to_np(logits), tokens, n)
    assert np.array_equal(to_np(got.ranks), rank), "ranks"
    assert np.array_equal(to_np(got.top_tokens), top), "top tokens"
    for name, a, b in (("logprobs", got.logprobs, lp), ("top_logprobs", got.top_logprobs, top_lp), ("entropy", got.entropy, entropy)):
        a, b = to_np(a).astype(np.float64), b
        with np.errstate(over="ignore"):
            b = np.where(np.isfinite(b), b, -np.inf)
        fine = np.isfinite(b)
        assert np.array_equal(a[~fine], b[~fine]), name
        err = np.abs(a[fine] - b[fine])
        tol = 4e-6 + 4 * 2.0 ** -24 * np.abs(b[fine])
        assert (err <= tol).all(), f"{name}: {err.max()}"
    return got


def _logits(t, v, dtype, seed, std=2.5):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(t, v, generator=gen) * std).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("t,v,n", [(1, 1, 1), (1, 2, 2), (3, 7, 7), (2, 64, 64), (5, 999, 5), (1, 32000, 20), (4, 32001, 0), (7, 4097, 64),
                                   (64, 5000, 1), (300, 2049, 3), (2, 151643, 20), (40, 70001, 33), (2500, 1025, 2)])
def test_logprobs_of_odd_sizes(dtype, t, v, n):
    rng = np.random.default_rng(v)
    x = _logits(t, v, dtype, v + t)
    tokens = rng.integers(0, v, t)
    tokens[::5] = to_np(x).argmax(1)[::5]
    tokens[-1] = v - 1
    tokens[0] = 0
    _check_logprobs(x, tokens, n)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_logprobs_of_masked_infinite_and_equal_logits(dtype):
    v = 5003
    x = _logits(14, v, dtype, 5)
    x[0, 5:] = -float("inf")
    x[1] = torch.finfo(dtype).min                             # every word at the lowest value: an even row
    x[2, ::2] = float("nan")
    x[3] = -float("inf")                                      # no word
    x[4] = float("nan")
    x[5, 77] = float("inf")
    x[6, [9, 4000]] = float("inf")
    x[7] = 0.5
    x[8, 1:] = -float("inf")                                  # one word
    x[9, :3000] = 0.0
    x[9, 1000:2000] = -0.0                                    # zeros of both signs are alike
    x[9, 3000:] = -1.0
    x[10, 4000] = torch.finfo(dtype).max
    x[11, ::3] = torch.finfo(dtype).tiny / 4                  # denormal
    x[12, 100:] = float("nan")
    for tokens in (np.arange(14) * 350, np.array([4, 5002, 2, 9, 8, 77, 4000, 2500, 0, 1500, 4000, 3, 99, 5002]),
                   np.array([5, 0, 3, 5002, 0, 78, 9, 5002, 1, 2999, 0, 4, 100, -1]), np.full(14, 5003)):
        for n in (0, 1, 20, 64):
            _check_logprobs(x, tokens, n)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("v", [20011, 100003])
def test_logprobs_of_many_equal_or_crowded_logits(dtype, v):
    """More equal logits at the n-th place than a workgroup ranks at a time, and the best ones crowded: side by side, in one lane's columns, in
    the last piece, as far apart as the type allows; a row that is masked but for a few."""
    gen = torch.Generator().manual_seed(v)
    x = (torch.rand(9, v, generator=gen) < 0.5).float() * 2 - 1
    x[1] = torch.randint(0, 40, (v,), generator=gen).float() / 8
    x[2] = torch.randn(v, generator=gen)
    x[2, 7000:10000] += 20                                    # side by side
    x[3] = torch.randn(v, generator=gen) / 16
    x[3, 5::4096] = 30                                        # of one lane, all alike
    x[4] = torch.randn(v, generator=gen) / 16
    for i in range(8):
        x[4, 40 + i::1024] = 10 + torch.arange(len(x[4, 40 + i::1024])).float() / 64
    x[5] = torch.linspace(-30, 30, v)
    x[6] = -float("inf")
    x[6, [3, 7777, v - 1]] = torch.tensor([1.0, 2.0, 1.0])
    x[7] = 0.0
    x[7, ::3] = -0.0
    x[8] = torch.randn(v, generator=gen)
    x[8, -700:] = 50
    x = x.to(dtype).cuda()
    for n in (1, 20, 64):
        _check_logprobs(x, np.array([0, 5, 9999, 5 + 4096, v - 1, v // 2, 3, 3, v - 1]), n)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("v", [2011, 20011, 100003])
def test_logprobs_of_equal_logits_below_zero(dtype, v):
    """More equal logits than a workgroup ranks at a time at values below zero, with none, few and many above them, and next to one."""
    eps = torch.finfo(dtype).eps
    x = torch.full((6, v), -1.5)
    x[1, 700::900] = -1.25
    x[2, 100:1700] = -1.5 * (1 + eps)                         # the values next to it
    x[3, ::2] = -1.5 * (1 - eps)
    x[4] = -40000.0
    x[4, -3:] = -0.0
    x[5] = -torch.finfo(dtype).tiny
    x[5, 1::3] = 0.0
    x = x.to(dtype).cuda()
    for n in (1, 20, 64):
        _check_logprobs(x, np.array([0, 700, 100, 2, v - 3, 1]), n)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_logprobs_of_masked_rows_in_pieces(dtype):
    """As the rows above, over several workgroups a row: pieces without a logit, and with fewer than are asked for."""
    v = 70003
    x = _logits(7, v, dtype, 6)
    x[0, 5:] = -float("inf")
    x[1, :69000] = float("nan")
    x[2] = -float("inf")
    x[3] = torch.finfo(dtype).min
    x[4, 20000:] = -float("inf")
    x[5, [9, 40000]] = float("inf")
    x[6, ::2] = float("nan")
    for tokens in (np.arange(7) * 10000, np.array([3, 69500, v - 1, 50000, 20001, 40000, 60001])):
        for n in (0, 5, 64):
            _check_logprobs(x, tokens, n)


def test_logprobs_of_large_logits_of_both_signs():
    """Distances of the logits up to the range of float32 and past it: the smaller ones are out, -(a float) or -inf as the difference is."""
    x = _logits(4, 3000, F32, 3)
    x[0] *= 1e20
    x[1] += 1e6
    x[2, 10], x[2, 11] = 3e38, -3e38
    x[3] *= 60.0
    tokens = np.array([0, 17, 10, 5])
    got = ops.token_logprobs(x, _i32(tokens), n_top=4)
    lp, rank, entropy, top, top_lp = S.token_logprobs(to_np(x), tokens, 4)
    assert np.array_equal(to_np(got.ranks), rank) and np.array_equal(to_np(got.top_tokens), top)
    # a difference of the logits rounded once, a logarithm of the sum beside it
    assert np.allclose(to_np(got.logprobs), lp, rtol=2.0 ** -22, atol=4e-6) and np.allclose(to_np(got.top_logprobs), top_lp, rtol=2.0 ** -22, atol=4e-6)
    assert np.allclose(to_np(got.entropy), entropy, rtol=2.0 ** -20, atol=4e-6)
    assert to_np(ops.token_logprobs(x[2:3], _i32([11])).logprobs)[0] == -np.inf      # -6e38 is no float32


@pytest.mark.parametrize("dtype", [BF, F32])
def test_logprobs_of_slices_at_every_alignment(dtype):
    wide = _logits(6, 9011, dtype, 9)
    for first in range(0, 9):
        x = wide[:, first:first + 9000 - first]
        _check_logprobs(x, np.array([0, 1, 4500, 8990, 8, 77]), 6)
        _check_logprobs(x[:, :5], np.array([0, 1, 4, 3, 2, 1]), 5)
    _check_logprobs(wide[1::2, :8000], np.array([3, 4, 5]), 4)


def test_logprobs_rising_and_falling():
    """The best logits come last in every lane, and first."""
    up = (torch.arange(40000, dtype=F32) / 400 - 50).repeat(3, 1).cuda()
    up[1] = up[1].flip(0)
    up[2, 20000:] = up[2, :20000].flip(0).clone()
    for dtype in (F32, BF):
        _check_logprobs(up.to(dtype), np.array([39999, 20000, 777]), 64)


def test_logprobs_replayed_in_a_graph_beside_eager_calls():
    x, tokens = _logits(9, 40000, BF, 1), _i32(np.arange(9) * 4000)
    ops.token_logprobs(x, tokens, n_top=5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.token_logprobs(x, tokens, n_top=5)
    for seed in range(4):
        x.copy_(_logits(9, 40000, BF, 100 + seed))
        want = ops.token_logprobs(x, tokens, n_top=5)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ adapters
@pytest.mark.parametrize("t,n", [(1, 1), (1, 1024), (64, 5), (1000, 300), (1024, 1024), (1025, 3), (5000, 1000), (70001, 40)])
def test_rows_by_adapter(t, n):
    rng = np.random.default_rng(t + n)
    ids = rng.integers(-2, n + 2, t)
    ids[t // 2:t // 2 + t // 4] = n // 2                      # a prompt
    rows = ops.adapter_rows(_i32(ids), n)
    plan = to_np(rows.plan)
    key = np.where((ids >= 0) & (ids < n), ids, n)
    want = np.argsort(key, kind="stable")
    assert np.array_equal(plan[:t], want)
    tiles = plan[(t + 3) // 4 * 4:].reshape(-1, 4)
    expect = []
    for a in np.unique(key):
        first, count = int((key < a).sum()), int((key == a).sum())
        expect += [(a if a < n else -1, first + i, min(rows.tile, count - i), 0) for i in range(0, count, rows.tile)]
    assert len(tiles) >= len(expect)
    assert np.array_equal(tiles[:len(expect)], np.array(expect)) and (tiles[len(expect):, 2] == 0).all()


def _bank(rng, n, widths, r, k, dtype, ranks):
    a = rounded(rng.normal(size=(n, len(widths), r, k)) / np.sqrt(k), dtype)
    b = rounded(rng.normal(size=(n, sum(widths), r)) / np.sqrt(r), dtype)
    at, bt = _dev(a, dtype), _dev(b, dtype)
    for i, ri in enumerate(ranks):                            # what lies behind a rank is not to be seen
        at[i, :, ri:] = float("nan")
        bt[i, :, ri:] = float("nan")
    return a, b, at, bt


def _check_adapters(got, want, mag, x, k, dtype):
    """Half a step of the result, and the second product's operand within 2^-16 (bf16: two values of 8 bits; fp16 has 22), sums in
    float32 whose order is open: (k / 64 + rank) 2^-24 of the terms, at k = 8192 below 2^-16."""
    got = to_np(got).astype(np.float64)
    tol = EPS[dtype] * np.abs(want) + 2.0 ** -14 * mag + 2.0 ** -25
    err = np.abs(got - want)
    assert (err <= tol).all(), f"{err.max()} over {tol.flat[np.argmax(err - tol)]}"


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("t,n,r,k,widths", [(1, 1, 8, 8, (1,)), (1, 3, 16, 4096, (4096,)), (3, 2, 24, 40, (70, 1, 65)), (17, 4, 8, 72, (64, 64)),
                                            (64, 48, 64, 1000, (512, 128, 128)), (100, 7, 128, 136, (200,)), (33, 5, 40, 4104, (96, 40)),
                                            (256, 200, 32, 512, (328,)), (1030, 6, 16, 264, (256, 64, 64)), (1500, 3, 128, 64, (100, 30)),
                                            (2000, 40, 32, 200, (24, 24, 24, 24, 24, 24, 24, 24))])
def test_adapters_of_many_requests(dtype, t, n, r, k, widths):
    rng = np.random.default_rng(t * 7 + k)
    ranks = rng.integers(0, r + 1, n)
    ranks[0] = r
    scales = rng.uniform(0.25, 2, n).astype(np.float32)
    scales[-1] *= -1
    ids = rng.integers(-1, n, t)
    ids[:1] = 0
    if t > 1024:
        ids = np.sort(ids)
    a, b, at, bt = _bank(rng, n, widths, r, k, dtype, ranks)
    x, base = rounded(rng.normal(size=(t, k)), dtype), rounded(rng.normal(size=(t, sum(widths))), dtype)
    xt, baset = _dev(x, dtype), _dev(base, dtype)
    rows = ops.adapter_rows(_i32(ids), n)
    got = ops.adapter_linear(xt, at, bt, rows, baset, widths=widths, ranks=_i32(ranks), scales=torch.from_numpy(scales).cuda())
    want, mag = S.adapter_linear(x, a, b, ids, base, widths, ranks, scales)
    _check_adapters(got, want, mag, x, k, dtype)
    none = (ids < 0) | (ranks[np.clip(ids, 0, n - 1)] == 0)
    assert np.array_equal(to_np(got)[none], base[none]) and torch.equal(baset, _dev(base, dtype))
    assert ops.adapter_linear(xt, at, bt, rows, baset, widths=widths, ranks=_i32(ranks), scales=torch.from_numpy(scales).cuda(), out=baset) is baset
    assert torch.equal(baset, got)                            # in place



@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n,r,k,widths", [(3, 8, 8, (1, 3)), (3, 32, 4096, (70, 1, 1025)), (2, 24, 4104, (1024, 1024)), (2, 128, 1024, (300,)),
                                          (2, 128, 1032, (300,)), (4, 40, 520, (64, 64)), (2, 16, 8192, (2049,)), (2, 8, 14336, (100,))])
def test_adapters_of_a_single_row(dtype, n, r, k, widths):
    """Both sides of the size up to which one kernel computes a row's products, ranks that end inside the pieces they are taken in."""
    rng = np.random.default_rng(k + r)
    for rank in sorted({1, 5, 8, r // 2 + 3, r - 1, r} - {0}):
        if rank > r:
            continue
        ranks = np.full(n, r)
        ranks[n - 1] = rank
        a, b, at, bt = _bank(rng, n, widths, r, k, dtype, ranks)
        x, base = rounded(rng.normal(size=(1, k)), dtype), rounded(rng.normal(size=(1, sum(widths))), dtype)
        xt, baset, scales = _dev(x, dtype), _dev(base, dtype), torch.full((n,), 0.75, device="cuda")
        rows = ops.adapter_rows(_i32([n - 1]), n)
        got = ops.adapter_linear(xt, at, bt, rows, baset, widths=widths, ranks=_i32(ranks), scales=scales)
        want, mag = S.adapter_linear(x, a, b, [n - 1], base, widths, ranks, np.full(n, 0.75, np.float32))
        _check_adapters(got, want, mag, x, k, dtype)
        ops.adapter_linear(xt, at, bt, rows, baset, widths=widths, ranks=_i32(ranks), scales=scales, out=baset)
        assert torch.equal(baset, got)
        none = ops.adapter_linear(xt, at, bt, ops.adapter_rows(_i32([-1]), n), baset, widths=widths, ranks=_i32(ranks), scales=scales)
        assert torch.equal(none, baset)


@pytest.mark.parametrize("pad", [1, 4, 8])
def test_adapters_of_column_slices(pad):
    """x, base and out as slices of wider rows, at alignments that are copied, moved element by element, and moved whole."""
    rng = np.random.default_rng(pad)
    t, n, r, k, widths = 40, 3, 16, 64, (128, 72)
    a, b, at, bt = _bank(rng, n, widths, r, k, BF, [r] * n)
    wide = rounded(rng.normal(size=(t, k + 200 + 3 * pad)), BF)
    w = _dev(wide, BF)
    x, base = w[:, pad:pad + k], w[:, k + 2 * pad:k + 2 * pad + 200]
    out = torch.full((t, 200 + 2 * pad), 7.0, dtype=BF, device="cuda")
    ids = rng.integers(-1, n, t)
    got = ops.adapter_linear(x, at, bt, ops.adapter_rows(_i32(ids), n), base, widths=widths, out=out[:, pad:pad + 200])
    want, mag = S.adapter_linear(to_np(x), a, b, ids, to_np(base), widths, [r] * n, np.ones(n))
    _check_adapters(got, want, mag, x, k, BF)
    assert (out[:, :pad] == 7).all() and (out[:, pad + 200:] == 7).all() and torch.equal(w, _dev(wide, BF))
    inside = ops.adapter_linear(x, at, bt, ops.adapter_rows(_i32(ids), n), base, widths=widths, out=base)
    assert inside is base and torch.equal(base, got)


def test_adapters_whose_hidden_values_pass_the_range_of_fp16():
    """lora_a x of 10^6 and of 10^-6, which come back into range with lora_b."""
    rng = np.random.default_rng(3)
    t, n, r, k, widths = 20, 2, 16, 512, (96,)
    a, b, at, bt = _bank(rng, n, widths, r, k, FP, [r, r])
    a, b = rounded(a * [[[[3e4]]], [[[2e-6]]]], FP), rounded(b * [[[2e-5]], [[5e3]]], FP)
    at, bt = _dev(a, FP), _dev(b, FP)
    x, base = rounded(rng.normal(size=(t, k)) * 40, FP), np.zeros((t, 96), np.float32)
    x[1::2] = rounded(x[1::2] * 1e-2, FP)
    ids = np.arange(t) % 2
    got = ops.adapter_linear(_dev(x, FP), at, bt, ops.adapter_rows(_i32(ids), n), _dev(base, FP))
    want, mag = S.adapter_linear(x, a, b, ids, base, widths, [r, r], np.ones(n))
    assert np.abs(S.adapter_linear(x, a[:, :, :1], np.ones((n, 1, 1)), ids, base[:, :1], (1,), [1, 1], np.ones(n))[0]).max() > 65504
    _check_adapters(got, want, mag, x, k, FP)


def test_adapters_infinite_and_nan_rows_stay_by_themselves():
    rng = np.random.default_rng(4)
    t, n, r, k, widths = 40, 2, 16, 64, (64,)
    a, b, at, bt = _bank(rng, n, widths, r, k, BF, [r, r])
    x, base = rounded(rng.normal(size=(t, k)), BF), rounded(rng.normal(size=(t, 64)), BF)
    ids = np.arange(t) % 3 - 1
    rows = ops.adapter_rows(_i32(ids), n)
    clean = ops.adapter_linear(_dev(x, BF), at, bt, rows, _dev(base, BF))
    y = x.copy()
    y[4, 3], y[8, 9], y[9, 0] = np.nan, np.inf, np.inf       # row 9 has no adapter
    got = ops.adapter_linear(_dev(y, BF), at, bt, rows, _dev(base, BF))
    hit = np.isin(np.arange(t), [4, 8])
    assert np.array_equal(to_np(got)[~hit], to_np(clean)[~hit])
    assert not np.isfinite(to_np(got)[hit & (ids >= 0)]).any()


def test_adapters_replayed_in_a_graph_with_other_ids():
    rng = np.random.default_rng(5)
    t, n, r, k, widths = 48, 9, 32, 256, (128, 64)
    _, _, at, bt = _bank(rng, n, widths, r, k, BF, [r] * n)
    x, base, ids = _dev(rng.normal(size=(t, k)), BF), _dev(rng.normal(size=(t, 192)), BF), _i32(rng.integers(-1, n, t))

    def step():
        return ops.adapter_linear(x, at, bt, ops.adapter_rows(ids, n), base, widths=widths)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                        # two graphs, replayed at once on streams of their own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out, torch.cuda.Stream()))
    for seed in range(4):
        rng = np.random.default_rng(seed)
        x.copy_(_dev(rng.normal(size=(t, k)), BF))
        ids.copy_(_i32(rng.integers(-1, n, t) if seed < 3 else np.full(t, seed)))
        want = step()
        torch.cuda.synchronize()
        for g, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, out, _ in graphs:
            assert torch.equal(out, want)


def test_operators_on_another_stream():
    rng = np.random.default_rng(6)
    t, n, r, k = 30, 4, 16, 128
    _, _, at, bt = _bank(rng, n, (64,), r, k, BF, [r] * n)
    x, base, ids = _dev(rng.normal(size=(t, k)), BF), _dev(rng.normal(size=(t, 64)), BF), _i32(rng.integers(-1, n, t))
    logits = _logits(t, 9000, F32, 2)

    def step():
        y = ops.adapter_linear(x, at, bt, ops.adapter_rows(ids, n), base)
        ops.rotary_embedding(y, None, ids, torch.from_numpy(_inv(16)).cuda(), 32)
        return [y, *ops.token_logprobs(logits, ids, n_top=3)]

    want = step()
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        got = step()
    other.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_rows_and_cache_rows_past_32_bits():
    """Rows 2^31 elements apart, cache rows behind 2^31 elements: as the same rows side by side."""
    big = torch.empty(2 * 2 ** 31 + 6000, dtype=BF, device="cuda")

    def apart(x):
        y = big.as_strided(x.shape, (2 ** 31, 1))
        return y.copy_(x)

    gen = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randn(3, 5003, generator=gen, device="cuda").to(BF)
    tokens = _i32([7, 5002, -1])
    for a, b in zip(ops.token_logprobs(apart(logits), tokens, n_top=5), ops.token_logprobs(logits, tokens, n_top=5)):
        assert torch.equal(a, b)

    rng = np.random.default_rng(4)
    _, _, at, bt = _bank(rng, 2, (96,), 16, 64, BF, [16, 8])
    ranks, rows = _i32([16, 8]), ops.adapter_rows(_i32([1, -1, 0]), 2)
    x, base = logits[:, :64].contiguous(), logits[:, 64:160].contiguous()
    want = ops.adapter_linear(x, at, bt, rows, base, ranks=ranks)
    assert torch.equal(ops.adapter_linear(apart(x), at, bt, rows, base, ranks=ranks), want)
    far = apart(base)
    assert ops.adapter_linear(x, at, bt, rows, far, ranks=ranks, out=far) is far and torch.equal(far, want)

    block, heads, d = 128, 8, 128
    blocks = 2 ** 31 // (block * heads * d) + 2
    kc, vc = (torch.empty(blocks, block, heads, d, dtype=BF, device="cuda") for _ in range(2))
    slots, pos, inv = _i32([blocks * block - 1, 5, blocks * block - 129]), _i32([3, 1000, 70000]), torch.from_numpy(_inv(64)).cuda()
    qkv = logits[:, :(4 + 2 * heads) * d].contiguous()
    q, k, v = qkv[:, :4 * d], qkv[:, 4 * d:(4 + heads) * d], qkv[:, (4 + heads) * d:]
    q_want, k_want = torch.empty(3, 4 * d, dtype=BF, device="cuda"), torch.empty(3, heads * d, dtype=BF, device="cuda")
    ops.rotary_embedding(q, k, pos, inv, d, out=(q_want, k_want))
    wide = apart(qkv)
    ops.rotary_embedding(wide[:, :4 * d], wide[:, 4 * d:(4 + heads) * d], pos, inv, d, value=wide[:, (4 + heads) * d:], key_cache=kc, value_cache=vc,
                         slot_mapping=slots)
    assert torch.equal(wide[:, :4 * d], q_want) and torch.equal(wide[:, 4 * d:(4 + heads) * d], k_want)
    at = slots.long()
    assert torch.equal(kc.view(-1, heads * d)[at], k_want) and torch.equal(vc.view(-1, heads * d)[at], v)


def _bad_rotary():
    def case(**over):
        z = lambda *shape, dtype=BF: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
        a = dict(query=z(3, 128), key=z(3, 64), positions=z(3, dtype=torch.int32), inv_freq=z(32, dtype=torch.float64), head_dim=64)
        for name, value in over.items():
            a[name] = value(z) if callable(value) else value
        return a
    cache = dict(value=lambda z: z(3, 64), key_cache=lambda z: z(2, 4, 1, 64), value_cache=lambda z: z(2, 4, 1, 64),
                 slot_mapping=lambda z: z(3, dtype=torch.int32))
    return [case(positions=lambda z: z(3, dtype=torch.int64)), case(inv_freq=lambda z: z(32, dtype=F32)), case(query=lambda z: z(3, 100)),
            case(query=lambda z: z(3, 128, dtype=F32)), case(query=lambda z: z(4, 128)), case(query=lambda z: z(1, 128).expand(3, 128)),
            case(query=lambda z: z(128, 3).t()), case(key=lambda z: z(3, 64, dtype=FP)), case(key=lambda z: z(2, 64)),
            case(key=lambda z: z(3, 64, dtype=BF).cpu()), case(positions=lambda z: z(3, dtype=torch.int32).cpu()), case(offset=1), case(offset=-1),
            case(head_dim=0), case(inv_freq=lambda z: z(33, dtype=torch.float64)), case(inv_freq=lambda z: z(64, dtype=torch.float64)[::2]),
            case(value=lambda z: z(3, 64)), case(**{**cache, "slot_mapping": None}), case(**{**cache, "value": lambda z: z(3, 128)}),
            case(**{**cache, "key_cache": lambda z: z(2, 4, 1, 64, dtype=FP)}), case(**{**cache, "value_cache": lambda z: z(2, 5, 1, 64)}),
            case(**{**cache, "slot_mapping": lambda z: z(3, dtype=torch.int64)}), case(**{**cache, "slot_mapping": lambda z: z(4, dtype=torch.int32)}),
            case(**{**cache, "key": None}), case(out=lambda z: (z(3, 128), None)), case(out=lambda z: (z(3, 64), z(3, 64))),
            case(out=lambda z: (z(3, 128), z(3, 128))), case(key=None, out=lambda z: (z(3, 128), z(3, 64)))]


def test_refused_calls_on_the_gpu():
    for a in _bad_rotary():
        with pytest.raises(ValueError):
            ops.rotary_embedding(**a)
    z = lambda *shape, dtype=BF: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
    t3 = z(3, dtype=torch.int32)
    for args in ((z(3, 50), t3.long()), (z(3, 50), z(4, dtype=torch.int32)), (z(50), t3), (z(3, 50, dtype=torch.float64), t3), (z(3, 50), t3, 51),
                 (z(3, 100), t3, 65), (z(3, 50), t3, -1), (z(50, 3).t(), t3), (z(1, 50).expand(3, 50), t3), (z(3, 50), t3.cpu()), (z(3, 0), t3),
                 (z(3, 50), z(6, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError):
            ops.token_logprobs(*args)
    for args in ((t3.long(), 2), (t3, 0), (t3, 1025), (t3.view(1, 3), 2), (z(6, dtype=torch.int32)[::2], 2)):
        with pytest.raises(ValueError):
            ops.adapter_rows(*args)
    rows = ops.adapter_rows(t3, 2)
    good = dict(x=z(3, 64), lora_a=z(2, 16, 64), lora_b=z(2, 96, 16), rows=rows, base=z(3, 96))
    ops.adapter_linear(**good)
    for over in (dict(x=z(4, 64)), dict(x=z(3, 56)), dict(x=z(3, 64, dtype=FP)), dict(x=z(1, 64).expand(3, 64)), dict(base=z(3, 95)),
                 dict(base=z(2, 96)), dict(base=z(3, 96).cpu()), dict(base=z(1, 96).expand(3, 96)), dict(out=z(3, 96, dtype=F32)),
                 dict(out=z(2, 96)), dict(out=z(96, 3).t()), dict(lora_a=z(3, 16, 64)), dict(lora_a=z(2, 12, 64), lora_b=z(2, 96, 12)),
                 dict(lora_a=z(2, 16, 60), x=z(3, 60)), dict(lora_b=z(2, 96, 8)), dict(lora_b=z(2, 16, 96).transpose(1, 2)), dict(widths=(96, 1)),
                 dict(widths=(48, 48)), dict(widths=(96, 0)), dict(ranks=z(2, dtype=torch.int64)), dict(ranks=z(3, dtype=torch.int32)),
                 dict(scales=z(2)), dict(scales=z(1, dtype=F32)), dict(lora_a=z(2, 136, 64), lora_b=z(2, 96, 136))):
        with pytest.raises(ValueError):
            ops.adapter_linear(**{**good, **over})
