"""The generation-side operators that this package is timed on: attention through a sliding window with sinks, the pages of
a cache that is shared between beams, and the selection of a beam-search step.

``run`` computes them either through the package's entry points (``own``) or in their plain form, elementary torch
operations in float32 (float64 where two candidates' order hangs on the last bits of a score).  Lengths are ragged and
fixed by the case, so that its bytes and operations are known; contents and placements come from the seed.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One user far into a conversation: a single new token, the window's pages and four sink tokens.
        dict(name="window_decode_one", path="decode", batch=1, lo=1777, hi=1777, heads=32, kv=8, dim=128, block=128,
             window=1024, sinks=4, cache="bf16"),
        # A serving batch of ragged contexts, some shorter than the window, some four times as long.
        dict(name="window_decode_batch", path="decode", batch=64, lo=512, hi=4096, heads=32, kv=8, dim=128, block=128,
             window=1024, sinks=4, cache="bf16"),
        # Long contexts of a 70B-class layer over an int8 cache with per-channel scales.
        dict(name="window_decode_long_int8", path="decode", batch=16, lo=16384, hi=32768, heads=64, kv=8, dim=128,
             block=128, window=4096, sinks=64, cache="int8"),
        # Three ragged prompts entering a model with a short window.
        dict(name="window_prompts", path="prompt", rows=4137, prompts=3, heads=28, kv=4, dim=128, window=512, sinks=4,
             type="fp16"),
        # One long document.
        dict(name="window_long_prompt", path="prompt", rows=16001, prompts=1, heads=32, kv=8, dim=128, window=2048,
             sinks=4, type="bf16"),
        # A chunked-prefill scheduler's mixed step: two chunks beside 24 decoding sequences, over pages.
        dict(name="window_chunks", path="chunk", decodes=24, chunks=2, chunk=512, lo=512, hi=4096, heads=32, kv=8,
             dim=128, block=128, window=1024, sinks=4, type="bf16"),
        # The page bookkeeping of a small beam search's step: every beam goes on from a parent and gets one more token.
        dict(name="fork_small", path="fork", groups=4, beams=4, width=32, block=16, blocks=1024, window=0, sinks=0, new=1),
        # The same for 512 beams on long tables, pages behind the window given back.
        dict(name="fork_large", path="fork", groups=64, beams=8, width=256, block=128, blocks=131072, window=4096, sinks=4,
             new=1),
        # The open pages that such a step has to copy, in every layer's keys and values.
        dict(name="copy_open_pages", path="copy", layers=32, pairs=24, blocks=128, block=128, kv=8, dim=128, type="bf16"),
        # A pool emptied in places is closed up: the plan and the page moves.
        dict(name="compact_pool", path="compact", layers=8, rows=64, width=32, blocks=1024, block=128, kv=8, dim=128, type="bf16"),
        # Beam search of one request.
        dict(name="beams_one", path="beams", groups=1, beams=4, vocab=32000, type="bf16", eos=2),
        # Beam search of a serving batch on a large vocabulary, logits in float32.
        dict(name="beams_batch", path="beams", groups=64, beams=8, vocab=152064, type="fp32", eos=151645),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], evenly spread over its logarithm."""
    return int(round(float(lo) * (float(hi) / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["decode", "decode", "prompt", "prompt", "chunk", "fork", "copy", "compact", "beams", "beams"])
    heads, kv = rng.choice([(32, 8), (28, 4), (64, 8), (8, 2), (8, 8), (8, 1)])
    window, sinks = _log(rng, 1, 4096), rng.choice([0, 1, 4, 17, 64])
    if kind == "decode":
        batch = _log(rng, 1, 64)
        hi = _log(rng, 2, min(32768, 524288 // batch))
        return dict(path="decode", batch=batch, lo=max(1, hi // rng.randint(1, 8)), hi=hi, heads=heads, kv=kv,
                    dim=rng.choice([64, 128]), block=rng.choice([16, 128]), window=window, sinks=sinks,
                    cache=rng.choice(["bf16", "fp16", "int8", "int8_token"]))
    if kind == "prompt":
        rows = _log(rng, 1, 8192)
        return dict(path="prompt", rows=rows, prompts=min(rows, rng.randint(1, 4)), heads=min(heads, 32), kv=min(kv, 8), dim=rng.choice([64, 128]),
                    window=min(window, 2048), sinks=min(sinks, 17), type=rng.choice(["bf16", "fp16"]))
    if kind == "chunk":
        hi = _log(rng, 128, 4096)
        return dict(path="chunk", decodes=_log(rng, 1, 24), chunks=rng.randint(1, 2), chunk=_log(rng, 2, 512),
                    lo=max(1, hi // rng.randint(1, 8)), hi=hi, heads=min(heads, 32), kv=min(kv, 8), dim=rng.choice([64, 128]),
                    block=rng.choice([16, 128]), window=min(window, 2048), sinks=sinks, type=rng.choice(["bf16", "fp16"]))
    if kind == "fork":
        groups, beams, width = _log(rng, 1, 64), rng.randint(1, 8), _log(rng, 2, 256)
        return dict(path="fork", groups=groups, beams=beams, width=width, block=rng.choice([16, 32, 128]),
                    blocks=groups * beams * (width + 1) + rng.randint(0, 999), window=rng.choice([0, window]), sinks=sinks,
                    new=rng.randint(0, 3))
    if kind == "copy":
        return dict(path="copy", layers=rng.randint(1, 32), pairs=_log(rng, 1, 48), blocks=rng.randint(96, 128),
                    block=rng.choice([16, 128]), kv=rng.choice([1, 4, 8]), dim=rng.choice([64, 128]),
                    type=rng.choice(["bf16", "fp16"]))
    if kind == "compact":
        rows, width = _log(rng, 1, 64), _log(rng, 2, 32)
        return dict(path="compact", layers=rng.randint(1, 8), rows=rows, width=width, blocks=min(1024, rows * width * 2 + rng.randint(1, 64)),
                    block=rng.choice([16, 128]), kv=rng.choice([1, 4, 8]), dim=rng.choice([64, 128]),
                    type=rng.choice(["bf16", "fp16"]))
    groups, beams = _log(rng, 1, 64), rng.randint(1, 8)
    return dict(path="beams", groups=groups, beams=beams, vocab=_log(rng, 1000, 152064), type=rng.choice(["bf16", "fp16", "fp32"]),
                eos=rng.choice([-1, 2, 7]))


# ------------------------------------------------------------------------------------------------ sizes of a case
def _spread(n, lo, hi):
    """n ragged lengths of [lo, hi], the same for every seed (golden-ratio steps)."""
    at = ((np.arange(n) + 1) * 0.6180339887498949) % 1.0
    return (lo + np.floor(at * (hi - lo + 1))).astype(np.int64)


def _split(rows, parts):
    """rows cut into ragged parts of at least one row."""
    cuts = np.unique(np.linspace(0, rows, parts + 1).astype(np.int64))
    if len(cuts) > 2 and rows > 8 * parts:
        cuts[1:-1] += rows // (4 * parts)
    return np.diff(cuts)


def _lengths(case):
    """(new rows per sequence, context length per sequence with the new rows) of an attention case."""
    if case["path"] == "prompt":
        q = _split(case["rows"], case["prompts"])
        return q, q
    if case["path"] == "chunk":
        q = np.concatenate([np.full(case["chunks"], case["chunk"]), np.ones(case["decodes"], np.int64)])
        return q, np.maximum(_spread(len(q), case["lo"], case["hi"]), q)
    lens = _spread(case["batch"], case["lo"], case["hi"])
    return np.ones(len(lens), np.int64), lens


def _visible(q, lens, window, sinks):
    """(keys that some row of a sequence sees, (row, visible key) pairs), summed over the sequences."""
    keys = pairs = 0
    for n, l in zip(q.tolist(), lens.tolist()):
        p = np.arange(l - n, l)
        behind = np.maximum(p - window + 1, 0)                     # tokens in front of a row's window
        pairs += int((np.minimum(p + 1, window) + np.minimum(behind, sinks)).sum())
        first = max(l - n - window + 1, 0)
        keys += l - first + min(first, sinks)
    return keys, pairs


def work(case):
    path = case["path"]
    if path in ("decode", "prompt", "chunk"):
        q, lens = _lengths(case)
        keys, pairs = _visible(q, lens, case["window"], case["sinks"])
        size = 1 if case.get("cache", "").startswith("int8") else 2
        row = 2 * case["kv"] * case["dim"] * size + (8 if case.get("cache") == "int8_token" else 0)
        return dict(bytes=float(keys) * row + 4.0 * int(q.sum()) * case["heads"] * case["dim"],
                    flops=4.0 * pairs * case["heads"] * case["dim"])
    if path == "fork":
        rows = case["groups"] * case["beams"]
        return dict(bytes=8.0 * rows * case["width"] + 4.0 * rows * (6 + case["new"]), flops=0.0)
    row = 2 * 2 * 2.0 * case["layers"] * case.get("kv", 0) * case.get("dim", 0) if path != "beams" else 0   # read + written, K + V
    if path == "copy":
        return dict(bytes=row * int(_spread(case["pairs"], 1, case["block"]).sum()) + 12.0 * case["pairs"], flops=0.0)
    if path == "compact":
        live = _live(case)
        return dict(bytes=row * case["block"] * (live - live * live // case["blocks"]) + 8.0 * case["rows"] * case["width"], flops=0.0)
    rows, size = case["groups"] * case["beams"], 4 if case["type"] == "fp32" else 2
    return dict(bytes=float(size) * rows * case["vocab"] + 48.0 * rows, flops=4.0 * rows * case["vocab"])


def _live(case):
    """Pages that a pool to be closed up holds."""
    return int(min(case["rows"] * case["width"], case["blocks"] * 3 // 4))


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    return {"decode": _attention_inputs, "prompt": _attention_inputs, "chunk": _attention_inputs, "fork": _fork_inputs,
            "copy": _copy_inputs, "compact": _compact_inputs, "beams": _beam_inputs}[case["path"]](case, gen, rng)


def _randn(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dtype)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).to(DEV)


def _attention_inputs(case, gen, rng):
    q, lens = _lengths(case)
    heads, kv, d = case["heads"], case["kv"], case["dim"]
    kind = case.get("cache", case.get("type"))
    dtype = TYPES["bf16" if kind.startswith("int8") else kind]
    s = dict(case=case, scale=1.0 / math.sqrt(d), starts=_i32(np.concatenate([[0], np.cumsum(q)])),
             query=_randn((int(q.sum()), heads * d), gen, dtype), qmax=int(q.max()), lmax=int(lens.max()))
    if case["path"] == "prompt":
        s["key"], s["value"] = (_randn((int(q.sum()), kv * d), gen, dtype) for _ in range(2))
        return s
    bs = case["block"]
    need = -(-lens // bs)
    perm = rng.permutation(int(need.sum()) + 2)
    tables = np.full((len(lens), int(need.max())), -1)
    at = np.concatenate([[0], np.cumsum(need)])
    cols = np.arange(tables.shape[1])
    held = cols[None, :] < need[:, None]
    tables[held] = perm[:at[-1]]
    shape = (len(perm), bs, kv, d)
    s["lens"], s["tables"] = _i32(lens), _i32(tables)
    if not kind.startswith("int8"):
        s["key"], s["value"] = (_randn(shape, gen, dtype) for _ in range(2))
        return s
    s["key"], s["value"] = (torch.clamp(torch.round(32 * _randn(shape, gen, torch.float32)), -128, 127).to(torch.int8) for _ in range(2))
    size = (2, len(perm), bs) if kind == "int8_token" else (2, kv * d)
    s["kv_scale"] = (0.5 + torch.rand(size, generator=gen, device=DEV)) / 32
    return s


def _fork_inputs(case, gen, rng):
    """Beams in the middle of a search: each group shares the pages of its prompt, every beam owns the later ones."""
    g, k, m, bs, nb = case["groups"], case["beams"], case["width"], case["block"], case["blocks"]
    lens = np.repeat(rng.integers(max(1, m * bs // 2), m * bs - 2 * case["new"], g), k)       # the beams of a group are equally long
    used = -(-lens // bs)
    shared = (used // 2)[::k]
    perm = rng.permutation(nb)
    tables = np.full((g * k, m), -1)
    cols = np.arange(m)[None, :]
    mine = (cols >= np.repeat(shared, k)[:, None]) & (cols < used[:, None])
    prompt = cols < shared[:, None]
    n_shared = int(prompt.sum())
    first = np.full((g, m), -1)
    first[prompt] = perm[:n_shared]
    tables[:] = np.repeat(first, k, axis=0)
    tables[mine] = perm[n_shared:n_shared + int(mine.sum())]
    parents = (np.arange(g)[:, None] * k + rng.integers(0, k, (g, k))).reshape(-1)
    if g > 1:
        parents[:k] = -1                                            # a group that has finished gives its pages back
    return dict(case=case, tables=_i32(tables), lens=_i32(lens), parents=_i32(parents))


def _caches(case, gen):
    shape = (case["blocks"], case["block"], case["kv"], case["dim"])
    base = _randn((min(case["blocks"], 64),) + shape[1:], gen, TYPES[case["type"]])            # 64 pages of noise, repeated with a step a tensor
    reps = -(-case["blocks"] // base.shape[0])
    return [(base + i).repeat(reps, 1, 1, 1)[:case["blocks"]].contiguous() for i in range(2 * case["layers"])]


def _copy_inputs(case, gen, rng):
    n = case["pairs"]
    perm = rng.permutation(case["blocks"])
    entries = np.stack([perm[:n], perm[n:2 * n], _spread(n, 1, case["block"])], axis=1)
    unused = np.tile([-1, -1, 0], (n // 3 + 1, 1))                  # rows of the step that need no copy
    return dict(case=case, caches=_caches(case, gen), copies=_i32(np.concatenate([entries, unused])))


def _compact_inputs(case, gen, rng):
    tables = np.full(case["rows"] * case["width"], -1)
    tables[rng.permutation(len(tables))[:_live(case)]] = rng.permutation(case["blocks"])[:_live(case)]
    return dict(case=case, caches=_caches(case, gen), tables=_i32(tables.reshape(case["rows"], case["width"])))


def _beam_inputs(case, gen, rng):
    g, k, v = case["groups"], case["beams"], case["vocab"]
    logits = 2.5 * _randn((g * k, v), gen, torch.float32)
    logits[:, torch.randint(0, v, (16,), generator=gen, device=DEV)] += 8.0    # the few words that fit
    logits[:, torch.randint(0, v, (v // 50 + 1,), generator=gen, device=DEV)] = -math.inf    # words that a grammar forbids
    scores = -torch.cumsum(torch.rand((g, k), generator=gen, device=DEV) * 2, dim=1) - 10
    return dict(case=case, logits=logits.to(TYPES[case["type"]]), scores=scores)


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    path = case["path"]
    if own:
        return _own(s, case, path)
    if path == "decode":
        return _plain_decode(s, case)
    if path == "prompt":
        return _plain_prompt(s, case)
    if path == "chunk":
        return _plain_chunk(s, case)
    if path == "fork":
        return _plain_fork(s, case)
    if path == "copy":
        return _plain_copy(s["caches"], s["copies"])
    if path == "compact":
        tables, copies, live = _plain_compact(s, case)
        return [tables, copies, live] + _plain_copy(s["caches"], copies)
    return _plain_beams(s, case)


def _own(s, case, path):
    from mindformers_amd import ops
    if path in ("decode", "prompt", "chunk"):
        view = dict(window=case["window"], sinks=case["sinks"])
        heads = (case["heads"], case["kv"])
    if path == "decode":
        if case["cache"] == "int8":
            return ops.paged_attention_int8kv(s["query"], s["key"], s["value"], s["tables"], s["lens"], s["kv_scale"], None,
                                              *heads, s["scale"], **view)
        if case["cache"] == "int8_token":
            return ops.paged_attention_int8kv(s["query"], s["key"], s["value"], s["tables"], s["lens"], None, None, *heads,
                                              s["scale"], token_scales=(s["kv_scale"][0], s["kv_scale"][1]), **view)
        return ops.paged_attention(s["query"], s["key"], s["value"], s["tables"], s["lens"], *heads, s["scale"], **view)
    if path == "prompt":
        return ops.causal_attention_varlen(s["query"], s["key"], s["value"], s["starts"], *heads, s["scale"], **view)
    if path == "chunk":
        return ops.paged_attention_prefill(s["query"], s["key"], s["value"], s["tables"], s["lens"], s["starts"], *heads,
                                           s["scale"], **view)
    if path == "fork":
        return ops.fork_blocks(s["tables"], s["lens"], case["blocks"], case["block"], parents=s["parents"],
                               new_tokens=case["new"], window=case["window"] or None, sinks=case["sinks"] if case["window"] else 0)
    if path == "copy":
        ops.copy_blocks(s["caches"], s["copies"])
        return s["caches"]
    if path == "compact":
        tables, copies, live = ops.compact_blocks(s["tables"], case["blocks"], case["block"])
        ops.copy_blocks(s["caches"], copies)
        return [tables, copies, live] + s["caches"]
    return ops.beam_search_select(s["logits"], s["scores"], eos_token_id=case["eos"])


# ------------------------------------------------------------------------------------------------ plain forms
def _softmax_value(scores, seen, value):
    """sum_j softmax_j(scores) value_j over the seen keys; zeros where none is seen."""
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = torch.clamp(scores.amax(dim=-1, keepdim=True), min=-1e30)
    p = torch.exp(scores - top)
    total = p.sum(dim=-1, keepdim=True)
    return torch.matmul(p, value) / torch.where(total > 0, total, torch.ones_like(total))


def _values_of(s, case, slots):
    """Keys and values of cache slots [B, J] as float32 [B, kv, J, D]."""
    kv, d = case["kv"], case["dim"]
    k, v = (c.reshape(-1, kv, d)[slots].to(torch.float32) for c in (s["key"], s["value"]))
    if case.get("cache") == "int8":
        k, v = k * s["kv_scale"][0].reshape(kv, d), v * s["kv_scale"][1].reshape(kv, d)
    if case.get("cache") == "int8_token":
        k, v = (x * s["kv_scale"][i].reshape(-1)[slots][..., None, None] for i, x in enumerate((k, v)))
    return k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()


def _slots(s, case, pos):
    bs = case["block"]
    page = torch.gather(s["tables"].long(), 1, torch.clamp(pos // bs, 0, s["tables"].shape[1] - 1))
    return torch.clamp(page, min=0) * bs + pos % bs


def _plain_decode(s, case):
    b, h, kv, d, w = case["batch"], case["heads"], case["kv"], case["dim"], case["window"]
    lens = s["lens"].long()[:, None]
    w = min(w, s["lmax"])
    first = torch.clamp(lens - w, min=0)                            # first token of the window
    j = torch.arange(case["sinks"] + w, device=DEV)[None, :]
    pos = torch.where(j < case["sinks"], j.expand(b, -1), first + j - case["sinks"])
    seen = torch.where(j < case["sinks"], pos < first, pos < lens)
    k, v = _values_of(s, case, _slots(s, case, torch.where(seen, pos, torch.zeros_like(pos))))
    q = s["query"].reshape(b, kv, h // kv, d).to(torch.float32)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    return _softmax_value(scores, seen[:, None, None, :], v).reshape(b, h * d).to(s["query"].dtype)


def _plain_prompt(s, case):
    """Queries in blocks of 256 rows, each against the rows that its window can reach; the sinks of every row beside them."""
    t, h, kv, d, w, ns = case["rows"], case["heads"], case["kv"], case["dim"], min(case["window"], case["rows"]), case["sinks"]
    c = 256
    n = -(-t // c)
    row = torch.arange(n * c, device=DEV)
    live = row < t
    starts = s["starts"].long()
    seq = torch.clamp(torch.searchsorted(starts, torch.clamp(row, max=t - 1), right=True) - 1, max=starts.numel() - 2)
    begin = starts[seq]                                             # first packed row of the row's sequence
    q = s["query"][torch.clamp(row, max=t - 1)].to(torch.float32).reshape(n, c, kv, h // kv, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, kv, -1, d)              # [blocks, kv, heads a kv head x rows, D]
    key, value = (s[x].reshape(t, kv, d).to(torch.float32) for x in ("key", "value"))
    near = (torch.arange(n, device=DEV) * c - w + 1)[:, None] + torch.arange(w + c - 1, device=DEV)[None, :]
    at = torch.clamp(near, 0, t - 1)
    k, v = (x[at].transpose(1, 2).contiguous() for x in (key, value))
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).reshape(n, kv, h // kv, c, -1) * s["scale"]
    r = row.reshape(n, c, 1)
    seen = (near[:, None, :] <= r) & (near[:, None, :] > r - w) & (near[:, None, :] >= begin.reshape(n, c, 1)) & live.reshape(n, c, 1)
    scores = torch.where(seen[:, None, None], scores, torch.full_like(scores, -math.inf))
    sink = begin[:, None] + torch.arange(ns, device=DEV)[None, :]   # [rows, sinks]
    sink_seen = (sink <= row[:, None] - w) & live[:, None]
    ks, vs = (x[torch.clamp(sink, max=t - 1)].reshape(n, c, ns, kv, d) for x in (key, value))
    qs = q.reshape(n, kv, h // kv, c, d)
    far = (qs[:, :, :, :, None, :] * ks.permute(0, 3, 1, 2, 4)[:, :, None]).sum(-1) * s["scale"]
    far = torch.where(sink_seen.reshape(n, 1, 1, c, ns), far, torch.full_like(far, -math.inf))
    top = torch.clamp(scores.amax(dim=-1, keepdim=True), min=-1e30)
    if ns:
        top = torch.maximum(top, far.amax(dim=-1, keepdim=True))
    p, pf = torch.exp(scores - top), torch.exp(far - top)
    total = p.sum(-1, keepdim=True) + pf.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(n, kv, -1, p.shape[-1]), v).reshape(n, kv, h // kv, c, d)
    out = (out + (pf[..., None] * vs.permute(0, 3, 1, 2, 4)[:, :, None]).sum(-2)) / torch.where(total > 0, total, torch.ones_like(total))
    return out.permute(0, 3, 1, 2, 4).reshape(n * c, h * d)[:t].to(s["query"].dtype)


def _plain_chunk(s, case):
    h, kv, d, w = case["heads"], case["kv"], case["dim"], case["window"]
    starts, lens = s["starts"].long(), s["lens"].long()
    b, n = lens.numel(), s["qmax"]
    rows = starts[1:] - starts[:-1]
    i = torch.arange(n, device=DEV)[None, :]
    live = i < rows[:, None]
    q = s["query"][torch.clamp(starts[:-1, None] + i, max=s["query"].shape[0] - 1)].to(torch.float32)
    q = q.reshape(b, n, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)
    pos = (lens - rows)[:, None] + i                                # [B, rows]
    j = torch.arange(s["lmax"], device=DEV)[None, :].expand(b, -1)
    k, v = _values_of(s, case, _slots(s, case, torch.where(j < lens[:, None], j, torch.zeros_like(j))))
    scores = (torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]).reshape(b, kv, h // kv, n, -1)
    jj, pp = j[:, None, :], pos[:, :, None]
    seen = (jj <= pp) & ((jj > pp - w) | (jj < case["sinks"])) & live[:, :, None]
    out = _softmax_value(scores.reshape(b, kv, -1, scores.shape[-1]),
                         seen[:, None, None].expand(b, kv, h // kv, n, -1).reshape(b, kv, -1, scores.shape[-1]), v)
    out = out.reshape(b, kv, h // kv, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, h * d)
    return out[live].to(s["query"].dtype)


def _plain_fork(s, case):
    tables, lens, parents = s["tables"].long(), s["lens"].long(), s["parents"].long()
    bs, nb, new = case["block"], case["blocks"], case["new"]
    rows, m = tables.shape
    live = (parents >= 0) & (parents < rows)
    p = torch.clamp(parents, 0, rows - 1)
    l = torch.where(live, torch.clamp(lens[p], 0, m * bs), torch.zeros_like(p))
    used = (l + bs - 1) // bs
    me, j = torch.arange(rows, device=DEV), torch.arange(m, device=DEV)[None, :]
    row = tables[p]
    kept = live[:, None] & (j < used[:, None]) & (row >= 0) & (row < nb)
    if case["window"]:
        kept &= ~(((j + 1) * bs <= (l - case["window"] + 1)[:, None]) & (j * bs >= case["sinks"]))
    eldest = torch.full((rows,), rows, device=DEV).scatter_reduce(0, p, torch.where(live, me, torch.full_like(me, rows)), "amin")
    last = torch.clamp(used - 1, min=0)
    split = live & (l % bs != 0) & (eldest[p] != me) & kept[me, last]
    open_page = row[me, last]
    kept &= ~(split[:, None] & (j == last[:, None]))
    out = torch.where(kept, row, torch.full_like(row, -1))
    taken = torch.zeros(nb + 1, dtype=torch.int32, device=DEV)
    taken[torch.where(kept, row, torch.full_like(row, nb)).reshape(-1)] = 1
    order = torch.sort(taken[:nb], stable=True).indices             # the free pages first, ascending
    n_free = nb - taken[:nb].sum()
    after = l + torch.where(live, new, 0)
    wanted = (after + bs - 1) // bs - used                          # fresh pages behind the open one
    asked = wanted + split
    begin = torch.cumsum(asked, 0) - asked
    rank = torch.where(j < used[:, None], begin[:, None], (begin + split)[:, None] + j - used[:, None])
    fresh = (split[:, None] & (j == last[:, None])) | ((j >= used[:, None]) & (j < (used + wanted)[:, None]))
    given = fresh & (rank < n_free)
    out = torch.where(given, order[torch.clamp(rank, 0, nb - 1)], out)
    copied = split & (begin < n_free)
    copies = torch.full((rows + 1, 3), -1, dtype=torch.int64, device=DEV)
    copies[:, 2] = 0
    place = torch.where(copied, torch.cumsum(copied.long(), 0) - 1, torch.full_like(me, rows))
    copies[place] = torch.where(copied[:, None], torch.stack([open_page, order[torch.clamp(begin, 0, nb - 1)], l % bs], 1),
                                torch.tensor([-1, -1, 0], device=DEV))
    at = l[:, None] + torch.arange(new, device=DEV)[None, :]
    page = torch.gather(out, 1, torch.clamp(at // bs, max=m - 1))
    slots = torch.where(live[:, None] & (at < m * bs) & (page >= 0), page * bs + at % bs, torch.full_like(at, -1))
    missing = asked.sum() - given.sum()
    return [x.to(torch.int32) for x in (out, torch.clamp(after, max=m * bs), slots.reshape(-1), copies[:rows], missing.reshape(1))]


def _plain_copy(caches, copies):
    copies = copies[copies[:, 0] >= 0].long()
    row = torch.arange(caches[0].shape[1], device=DEV)[None, :, None, None] < copies[:, 2].reshape(-1, 1, 1, 1)
    for c in caches:
        c[copies[:, 1]] = torch.where(row, c[copies[:, 0]], c[copies[:, 1]])
    return caches


def _plain_compact(s, case):
    tables, nb = s["tables"].long(), case["blocks"]
    named = (tables >= 0) & (tables < nb)
    live = torch.zeros(nb + 1, dtype=torch.bool, device=DEV)
    live[torch.where(named, tables, torch.full_like(tables, nb)).reshape(-1)] = True
    live = live[:nb]
    n = live.sum()
    page = torch.arange(nb, device=DEV)
    target = page < n
    moves, holes = live & ~target, target & ~live
    source = torch.sort((~moves).to(torch.int32), stable=True).indices[:nb // 2]
    hole = torch.sort((~holes).to(torch.int32), stable=True).indices[:nb // 2]
    used = torch.arange(nb // 2, device=DEV) < moves.sum()
    to = page.clone()
    to[source] = torch.where(used, hole, to[source])
    none = torch.full_like(source, -1)
    copies = torch.stack([torch.where(used, source, none), torch.where(used, hole, none),
                          torch.where(used, case["block"], 0)], 1)
    out = torch.where(named, to[torch.clamp(tables, 0, nb - 1)], torch.full_like(tables, -1))
    return out.to(torch.int32), copies.to(torch.int32), n.reshape(1).to(torch.int32)


def _plain_beams(s, case):
    g, k, v = case["groups"], case["beams"], case["vocab"]
    n = 2 * k
    x = s["logits"].to(torch.float64)
    top = torch.clamp(x.amax(dim=-1, keepdim=True), min=-1e300)
    x = x - top
    x = s["scores"].to(torch.float64).reshape(-1, 1) + (x - torch.log(torch.exp(x).sum(dim=-1, keepdim=True)))
    x = x.reshape(g, k * v)
    least = torch.topk(x, n, dim=-1).values[:, -1:]
    above, at = torch.topk(torch.where(x > least, x, torch.full_like(x, -math.inf)), n, dim=-1)
    index = torch.arange(k * v, device=DEV, dtype=torch.float64)[None, :]
    level = -torch.topk(torch.where(x == least, -index, torch.full_like(x, -math.inf)), n, dim=-1).values     # lowest places first
    score = torch.cat([above, torch.where(torch.isinf(level), torch.full_like(level, -math.inf), least.expand_as(level))], 1)
    place = torch.cat([torch.where(above > least, at.to(torch.float64), torch.full_like(above, math.inf)), level], 1)
    by = torch.sort(place, dim=1, stable=True).indices
    score, place = torch.gather(score, 1, by), torch.gather(place, 1, by)
    by = torch.sort(torch.where(torch.isinf(place), torch.full_like(score, -math.inf), score), dim=1, descending=True, stable=True).indices[:, :n]
    score, place = torch.gather(score, 1, by).to(torch.float32), torch.gather(place, 1, by).long()
    beam, token = place // v, place % v
    last = (token == case["eos"]).to(torch.int32)
    by = torch.sort(last, dim=1, stable=True).indices[:, :k]        # the first K that go on
    rows = torch.arange(g, device=DEV)[:, None] * k + beam
    return [score, beam.to(torch.int32), token.to(torch.int32), torch.gather(score, 1, by),
            torch.gather(rows, 1, by).to(torch.int32), torch.gather(token, 1, by).to(torch.int32)]


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["path"] == "beams":
        return _exact_beams(s, case)
    if case["path"] not in ("decode", "prompt", "chunk"):
        return None                                                 # whole numbers and copies
    q, lens = _lengths(case)
    h, kv, d = case["heads"], case["kv"], case["dim"]
    out = torch.zeros((int(q.sum()), h, d), dtype=torch.float64, device=DEV)
    first = 0
    for b, (n, l) in enumerate(zip(q.tolist(), lens.tolist())):
        key, value = _exact_rows(s, case, b, first, l)              # [L, kv, D]
        for r0 in range(0, n, 512):
            r1 = min(n, r0 + 512)
            p = torch.arange(l - n + r0, l - n + r1, device=DEV)
            lo = max(0, l - n + r0 - case["window"] + 1)            # nothing in front of it is seen but the sinks
            j = torch.cat([torch.arange(min(lo, case["sinks"]), device=DEV), torch.arange(lo, l - n + r1, device=DEV)])
            seen = (j[None] <= p[:, None]) & ((j[None] > p[:, None] - case["window"]) | (j[None] < case["sinks"]))
            for head in range(h):
                a = s["query"][first + r0:first + r1].reshape(-1, h, d)[:, head].double() @ key[j, head * kv // h].T.contiguous() * s["scale"]
                a = torch.softmax(a.masked_fill(~seen, -math.inf), dim=1)
                out[first + r0:first + r1, head] = a @ value[j, head * kv // h]
        first += n
    return out.reshape(out.shape[0], h * d)


def _exact_rows(s, case, b, first, l):
    kv, d = case["kv"], case["dim"]
    if case["path"] == "prompt":
        return tuple(s[x][first:first + l].reshape(l, kv, d).double() for x in ("key", "value"))
    bs = case["block"]
    pages = s["tables"][b, :-(-l // bs)].long()
    got = []
    for i, x in enumerate(("key", "value")):
        rows = s[x][pages].reshape(-1, kv, d)[:l].double()
        if case.get("cache") == "int8":
            rows = rows * s["kv_scale"][i].double().reshape(1, kv, d)
        if case.get("cache") == "int8_token":
            rows = rows * s["kv_scale"][i][pages].double().reshape(-1, 1, 1)[:l]
        got.append(rows)
    return tuple(got)


def _exact_beams(s, case):
    g, k, v = case["groups"], case["beams"], case["vocab"]
    best, going = [], []
    for i in range(g):
        total = s["scores"][i].double()[:, None] + torch.log_softmax(s["logits"][i * k:(i + 1) * k].double(), dim=1)
        score, at = torch.sort(total.reshape(-1), descending=True, stable=True)
        score, at = score[:2 * k], at[:2 * k]
        best.append(score)
        going.append(score[at % v != case["eos"]][:k])
    return [torch.stack(best), None, None, torch.stack(going), None, None]
