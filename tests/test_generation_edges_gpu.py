"""Calls of the generation-side operators at the edges of what their documentation allows."""
import numpy as np
import pytest
import torch

from test_generation_gpu import _beams, _select, _stack

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


def test_an_end_token_outside_the_vocabulary_ends_nothing():
    from mindformers_amd import ops
    logits, scores = _beams(2, 3, 50, torch.float32, seed=2)
    want = ops.beam_search_select(logits, scores)
    for eos in (50, 2 ** 31 - 1, 2 ** 31 + 5, 2 ** 32 + int(want.tokens[0, 0]), -1, -2 ** 32 + int(want.tokens[0, 0]), -2 ** 40):
        for have, w in zip(ops.beam_search_select(logits, scores, eos_token_id=eos), want):
            assert torch.equal(have, w), eos


def test_sizes_that_pass_32_bits_are_refused():
    from mindformers_amd import ops
    t, n = _i32(np.zeros((2, 3))), _i32([4, 5])
    for call in (lambda: ops.fork_blocks(t, n, 8, 2 ** 32 + 16), lambda: ops.fork_blocks(t, n, 8, 16, new_tokens=2 ** 32 + 1),
                 lambda: ops.compact_blocks(t, 8, 2 ** 32 + 16), lambda: ops.fork_blocks(t, n, 2 ** 32 + 8, 16)):
        with pytest.raises(ValueError):
            call()

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
    """Tables that name 2^30 tokens, walks of 40000: the same bits as behind tables that end with the context."""
    from mindformers_amd import ops
    bs, b, nh, nkv, d = 16384, 32, 8, 8, 32
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    kc, vc = (torch.randn(3, bs, nkv, d, generator=gen, device="cuda").bfloat16() for _ in range(2))
    narrow = torch.arange(3, dtype=torch.int32, device="cuda").repeat(b, 1)
    wide = torch.full((b, (1 << 30) // bs), -1, dtype=torch.int32, device="cuda")
    wide[:, :3] = narrow
    n, starts = torch.randint(33000, 40001, (b,), generator=gen, device="cuda").int(), torch.arange(b + 1, device="cuda").int()
    q = torch.randn(b, nh * d, generator=gen, device="cuda").bfloat16()
    for window, sinks in ((2 ** 31 - 1, 0), (1 << 30, 3), (35000, 100)):
        got, want = (ops.paged_attention(q, kc, vc, t, n, nh, nkv, 0.2, window=window, sinks=sinks) for t in (wide, narrow))
        assert torch.equal(got, want) and got.float().abs().amax(1).min() > 0
    rows = torch.randn(4 * b, nh * d, generator=gen, device="cuda").bfloat16()
    got, want = (ops.paged_attention_prefill(rows, kc, vc, t, n, 4 * starts, nh, nkv, 0.2, window=300, sinks=3) for t in (wide, narrow))
    assert torch.equal(got, want) and got.float().abs().amax(1).min() > 0
