"""Operators of a serving step that this package is timed on beside those of ``operators.py``: rotary positions of other layouts
and scalings with the cache write behind them, low-rank adapters of many requests beside a layer's shared projections, and log
probabilities of given tokens with entropy and top alternatives.

``run`` computes them either through the package's entry points (``own``) or in their plain form, elementary torch
operations in float32 (the angles of far positions in float64).  Which rows, ranks and lengths there are is fixed by the
case, so that its bytes and operations are known; contents and placements come from the seed.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_LOGITS = 4137 * 152064


def listed():
    return [
        # One user far into a long conversation: a single token's query and key, scaled for long contexts, and the cache row.
        dict(name="rotary_decode_one", path="rotary", rows=1, heads=32, kv=8, dim=128, part=128, interleaved=False,
             scaling="llama3", far=131072, block=128, cache=True, type="bf16"),
        # A decode batch of a model that turns half of every head, neighbours in pairs; some rows are padding.
        dict(name="rotary_decode_batch", path="rotary", rows=64, heads=28, kv=4, dim=128, part=64, interleaved=True,
             scaling="none", far=32768, block=16, cache=True, type="fp16"),
        # Packed prompts entering the cache, yarn scaling.
        dict(name="rotary_prompts", path="rotary", rows=8191, heads=32, kv=8, dim=128, part=128, interleaved=False,
             scaling="yarn", far=40960, block=128, cache=True, type="bf16"),
        # One long document without a cache, a quarter of heads that are 80 wide.
        dict(name="rotary_document", path="rotary", rows=16001, heads=64, kv=8, dim=80, part=20, interleaved=True,
             scaling="linear", far=16001, block=16, cache=False, type="bf16"),
        # One request with an adapter on every projection of an 8B-class layer.
        dict(name="adapters_one", path="adapters", rows=1, hidden=4096, query=4096, kv=1024, ffn=14336, parts="qkv,wo,fc1,fc2",
             adapters=8, used=1, rank=16, ranks="all", spread="random", none=0.0, type="bf16"),
        # A decode batch whose requests have chosen among 48 adapters of several ranks, some none.
        dict(name="adapters_decode", path="adapters", rows=64, hidden=4096, query=4096, kv=1024, ffn=14336, parts="qkv,wo,fc1,fc2",
             adapters=48, used=24, rank=64, ranks="mixed", spread="random", none=0.1, type="bf16"),
        # A large batch of a 70B-class layer, attention projections only, nearly every request its own adapter.
        dict(name="adapters_decode_wide", path="adapters", rows=256, hidden=8192, query=8192, kv=1024, ffn=29568, parts="qkv,wo",
             adapters=128, used=128, rank=32, ranks="mixed", spread="random", none=0.05, type="fp16"),
        # Packed prompts of three requests with adapters of their own, and a fourth without.
        dict(name="adapters_prompts", path="adapters", rows=8191, hidden=4096, query=4096, kv=1024, ffn=14336, parts="qkv,wo",
             adapters=8, used=3, rank=32, ranks="all", spread="runs", none=0.1, type="bf16"),
        # The token that one request has sampled, with five alternatives.
        dict(name="logprobs_one", path="logprobs", rows=1, vocab=32000, top=5, type="fp32"),
        # A decode batch over a large vocabulary, twenty alternatives.
        dict(name="logprobs_decode", path="logprobs", rows=64, vocab=152064, top=20, type="bf16"),
        # The scores of a rollout's tokens: no alternatives asked for.
        dict(name="logprobs_rollout", path="logprobs", rows=1001, vocab=151643, top=0, type="fp32"),
        # Log probabilities of a whole prompt's tokens.
        dict(name="logprobs_prompt", path="logprobs", rows=4137, vocab=152064, top=5, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(min(hi, max(lo, math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["rotary", "adapters", "logprobs"])
    if kind == "rotary":
        heads, kv = rng.choice([(32, 8), (28, 4), (64, 8), (8, 2), (8, 8), (7, 1)])
        dim = rng.choice([64, 80, 96, 128, 256])
        rows = _log(rng, 1, min(16001, 16001 * 64 * 80 // (heads * dim)))
        return dict(path="rotary", rows=rows, heads=heads, kv=kv, dim=dim, part=rng.choice([dim, dim // 2, dim // 4]),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "llama3", "yarn"]),
                    far=max(rows, _log(rng, 64, 1000000)), block=rng.choice([16, 128]), cache=rng.random() < 0.6,
                    type=rng.choice(["bf16", "fp16"]))
    if kind == "adapters":
        hidden, query, kv, ffn = rng.choice([(512, 512, 128, 1376), (3584, 3584, 512, 18944), (4096, 4096, 1024, 14336),
                                             (8192, 8192, 1024, 29568)])
        parts = rng.choice(["qkv,wo,fc1,fc2", "qkv,wo", "qkv", "fc1,fc2", "wo"])
        spread = rng.choice(["random", "random", "runs"])
        rows = _log(rng, 1, 512) if spread == "random" else _log(rng, 8, 8191 * 4096 // max(hidden, 4096) // (4 if "fc" in parts else 1))
        adapters = _log(rng, 1, 128)
        return dict(path="adapters", rows=rows, hidden=hidden, query=query, kv=kv, ffn=ffn, parts=parts, adapters=adapters,
                    used=max(1, min(adapters, rows if spread == "random" else min(8, rows // 4), _log(rng, 1, 128))),
                    rank=rng.choice([8, 16, 32, 64]), ranks=rng.choice(["all", "mixed"]), spread=spread,
                    none=rng.choice([0.0, 0.1, 0.5]), type=rng.choice(["bf16", "fp16"]))
    vocab = _log(rng, 1000, 152064)
    return dict(path="logprobs", rows=_log(rng, 1, min(4137, MOST_LOGITS // vocab)), vocab=vocab, top=rng.choice([0, 1, 5, 20]),
                type=rng.choice(["bf16", "fp16", "fp32"]))


# ------------------------------------------------------------------------------------------------ sizes of a case
def _projections(case):
    """(input width, output widths) of the projections that have adapters."""
    h, q, kv, f = case["hidden"], case["query"], case["kv"], case["ffn"]
    every = {"qkv": (h, (q, kv, kv)), "wo": (q, (h,)), "fc1": (h, (f, f)), "fc2": (f, (h,))}
    return [every[p] for p in case["parts"].split(",")]


def _counts(case):
    """Rows of each adapter that is used, ragged, one at least; what is left of the rows has none."""
    n = case["used"]
    rows = max(n, case["rows"] - int(case["none"] * case["rows"]))
    weight = 1.0 + ((np.arange(n) + 1) * 0.6180339887498949) % 1.0 * 3
    at = np.concatenate([[0.0], np.cumsum(weight)]) / weight.sum() * (rows - n)
    return 1 + np.diff(np.floor(at + 1e-9)).astype(np.int64)


def _ranks(case):
    """Rank of each slot of the bank."""
    most = case["rank"]
    several = [r for r in (8, 16, 32, 64) if r <= most]
    return np.array([several[i % len(several)] if case["ranks"] == "mixed" else most for i in range(case["adapters"])])


def _used(case):
    """Slots of the adapters that are used."""
    return (np.arange(case["used"]) * case["adapters"]) // case["used"]


def work(case):
    if case["path"] == "rotary":
        row = case["dim"] * (2.0 * case["heads"] + 2.0 * case["kv"] + (2.0 * case["kv"] if case["cache"] else 0.0))
        return dict(bytes=2 * row * case["rows"] + 8.0 * case["rows"], flops=3.0 * case["rows"] * (case["heads"] + case["kv"]) * case["part"])
    if case["path"] == "logprobs":
        size = 4 if case["type"] == "fp32" else 2
        return dict(bytes=float(size) * case["rows"] * case["vocab"] + case["rows"] * (16.0 + 8.0 * case["top"]),
                    flops=6.0 * case["rows"] * case["vocab"])
    ranks, counts = _ranks(case)[_used(case)], _counts(case)
    total = dict(bytes=4.0 * case["rows"], flops=0.0)
    for k, widths in _projections(case):
        n, s = sum(widths), len(widths)
        total["bytes"] += 2.0 * (float(ranks.sum()) * (s * k + n) + float(counts.sum()) * k + 2.0 * case["rows"] * n)
        total["flops"] += 2.0 * float((ranks * counts).sum()) * (s * k + n)
    return total


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    return {"rotary": _rotary_inputs, "adapters": _adapter_inputs, "logprobs": _logit_inputs}[case["path"]](case, gen, rng)


def _randn(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dtype)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).to(DEV)


def _inv_freq(case):
    """Radians a position of every pair, float64, and the factor that goes with the scaling."""
    d, base, factor = case["part"], 500000.0, 8.0
    i = np.arange(0, d, 2, dtype=np.float64)
    f = base ** (-i / d)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "llama3":                                 # low frequencies divided, high ones kept, between them mixed
        turns = 8192 * f / (2 * math.pi)
        mix = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        return f * (mix + (1 - mix) / factor), 1.0
    if case["scaling"] == "yarn":
        pair = lambda turns: d * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), d - 1)
        ramp = np.clip((i / 2 - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _rotary_inputs(case, gen, rng):
    t, h, kv, d, bs = case["rows"], case["heads"], case["kv"], case["dim"], case["block"]
    dtype = TYPES[case["type"]]
    qkv = _randn((t, (h + 2 * kv) * d), gen, dtype)                 # a fused projection's rows
    inv, scale = _inv_freq(case)
    s = dict(case=case, query=qkv[:, :h * d], key=qkv[:, h * d:(h + kv) * d], value=qkv[:, (h + kv) * d:], scale=scale,
             inv_freq=torch.from_numpy(inv).to(DEV), q_out=torch.empty((t, h * d), dtype=dtype, device=DEV))
    if not case["cache"]:                                           # one document: its positions in turn
        s["positions"] = _i32(np.arange(t) + rng.integers(0, case["far"] - t + 1))
        s["k_out"] = torch.empty((t, kv * d), dtype=dtype, device=DEV)
        return s
    if t <= 512:                                                    # decode: anywhere, every sixteenth row padding
        s["positions"] = _i32(rng.integers(case["far"] // 2, case["far"], t))
        blocks = 2 * t + 8
        slots = rng.permutation(blocks * bs)[:t]
        slots[15::16] = -1
    else:                                                           # prompts of a few thousand tokens, the later ones chunks
        s["positions"] = _i32(np.concatenate([np.arange(n) + rng.integers(0, case["far"] - n + 1) for n in _prompts(t)]))
        blocks = -(-t // bs) + 8
        page = rng.permutation(blocks)
        slots = page[np.arange(t) // bs] * bs + np.arange(t) % bs
    live = np.flatnonzero(slots >= 0)
    s.update(slots=_i32(slots), live=torch.from_numpy(live).to(DEV), at=torch.from_numpy(slots[live].astype(np.int64)).to(DEV))
    s["key_cache"], s["value_cache"] = (_randn((blocks, bs, kv, d), gen, dtype) for _ in range(2))
    return s


def _prompts(rows):
    n = max(1, rows // 2500)
    return np.diff(np.linspace(0, rows, n + 1).astype(np.int64))


def _adapter_inputs(case, gen, rng):
    dtype, slots, rank = TYPES[case["type"]], case["adapters"], case["rank"]
    t, counts, used, ranks = case["rows"], _counts(case), _used(case), _ranks(case)
    ids = np.full(t, -1, np.int64)
    if case["spread"] == "runs":                                    # prompts one behind the other, those without an adapter last
        ids[:counts.sum()] = np.repeat(rng.permutation(used), counts)
    else:
        ids[rng.permutation(t)[:counts.sum()]] = np.repeat(used, counts)
    rows = [np.flatnonzero(ids == a) for a in used]                 # of each adapter, filled up with its first
    table = np.full((len(used), max(len(r) for r in rows)), 0)
    real = np.zeros(table.shape, bool)
    for i, r in enumerate(rows):
        table[i, :len(r)], real[i, :len(r)] = r, True
    inside = torch.from_numpy(np.arange(rank)[None, :] < ranks[:, None]).to(DEV)
    s = dict(case=case, ids=_i32(ids), ranks=_i32(ranks), scales=0.5 + 1.5 * torch.rand(slots, generator=gen, device=DEV), parts=[],
             used=torch.from_numpy(used).to(DEV), table=torch.from_numpy(table).to(DEV),
             real=torch.from_numpy(np.flatnonzero(real.reshape(-1))).to(DEV), to=torch.from_numpy(table[real]).to(DEV))
    for k, widths in _projections(case):
        a = _randn((slots, len(widths), rank, k), gen, torch.float32) / math.sqrt(k) * inside[:, None, :, None]
        b = _randn((slots, sum(widths), rank), gen, torch.float32) / math.sqrt(rank) * inside[:, None, :]
        s["parts"].append(dict(widths=widths, a=a.to(dtype), b=b.to(dtype), x=_randn((t, k), gen, dtype),
                               base=_randn((t, sum(widths)), gen, dtype)))
    return s


def _logit_inputs(case, gen, rng):
    t, v, dtype = case["rows"], case["vocab"], TYPES[case["type"]]
    logits = torch.empty((t, v), dtype=dtype, device=DEV)
    few = torch.randint(0, v, (16,), generator=gen, device=DEV)     # the few words that fit
    gone = torch.randint(0, v, (v // 50 + 1,), generator=gen, device=DEV)     # words that a grammar forbids
    step = max(1, (1 << 28) // v)
    for r in range(0, t, step):
        x = 2.5 * torch.randn((min(step, t - r), v), generator=gen, device=DEV)
        x[:, few] += 8.0
        x[:, gone] = -math.inf
        logits[r:r + step] = x.to(dtype)
    tokens = torch.where(torch.rand(t, generator=gen, device=DEV) < 0.7, few[torch.randint(0, 16, (t,), generator=gen, device=DEV)],
                         torch.randint(0, v, (t,), generator=gen, device=DEV)).to(torch.int32)
    return dict(case=case, logits=logits, tokens=tokens)


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return {"rotary": _plain_rotary, "adapters": _plain_adapters, "logprobs": _plain_logprobs}[case["path"]](s, case)


def _own(s, case):
    from mindformers_amd import ops
    if case["path"] == "rotary":
        view = dict(interleaved=case["interleaved"], scale=s["scale"])
        if not case["cache"]:
            return ops.rotary_embedding(s["query"], s["key"], s["positions"], s["inv_freq"], case["dim"], out=(s["q_out"], s["k_out"]), **view)
        q, _ = ops.rotary_embedding(s["query"], s["key"], s["positions"], s["inv_freq"], case["dim"], value=s["value"],
                                    key_cache=s["key_cache"], value_cache=s["value_cache"], slot_mapping=s["slots"],
                                    out=(s["q_out"], None), **view)
        return [q, s["key_cache"], s["value_cache"]]
    if case["path"] == "adapters":
        rows = ops.adapter_rows(s["ids"], case["adapters"])
        return [ops.adapter_linear(p["x"], p["a"], p["b"], rows, p["base"], widths=p["widths"], ranks=s["ranks"], scales=s["scales"])
                for p in s["parts"]]
    got = ops.token_logprobs(s["logits"], s["tokens"], n_top=case["top"])
    return list(got) if case["top"] else list(got[:3])


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_rotary(s, case):
    d, p = case["dim"], case["part"]
    angle = s["positions"].to(torch.float64)[:, None] * s["inv_freq"][None, :]
    cos, sin = ((f(angle) * s["scale"]).to(torch.float32)[:, None, :] for f in (torch.cos, torch.sin))

    def turned(x):
        x = x.reshape(x.shape[0], -1, d).to(torch.float32)
        a, b = (x[..., 0:p:2], x[..., 1:p:2]) if case["interleaved"] else (x[..., :p // 2], x[..., p // 2:p])
        a, b = a * cos - b * sin, b * cos + a * sin
        ab = torch.stack([a, b], -1).reshape(x.shape[0], -1, p) if case["interleaved"] else torch.cat([a, b], -1)
        return torch.cat([ab, x[..., p:]], -1).reshape(x.shape[0], -1)

    s["q_out"].copy_(turned(s["query"]))
    key = turned(s["key"]).to(s["key"].dtype)
    if not case["cache"]:
        s["k_out"].copy_(key)
        return [s["q_out"], s["k_out"]]
    s["key_cache"].view(-1, key.shape[1])[s["at"]] = key[s["live"]]
    s["value_cache"].view(-1, key.shape[1])[s["at"]] = s["value"][s["live"]]
    return [s["q_out"], s["key_cache"], s["value_cache"]]


def _plain_adapters(s, case):
    """The rows of each adapter as a batch of products, filled up to the longest."""
    def one(p):
        x = p["x"][s["table"]].to(torch.float32)                    # [adapters used, rows, K]
        a = p["a"][s["used"]].to(torch.float32).flatten(1, 2).transpose(1, 2).contiguous()
        b = p["b"][s["used"]].to(torch.float32).transpose(1, 2).contiguous().split(p["widths"], dim=2)
        h = torch.matmul(x, a).split(case["rank"], dim=2)
        delta = torch.cat([torch.matmul(hi, bi.contiguous()) for hi, bi in zip(h, b)], 2) * s["scales"][s["used"]][:, None, None]
        out = p["base"].to(torch.float32)
        out[s["to"]] += delta.flatten(0, 1)[s["real"]]
        return out.to(p["base"].dtype)

    return [one(p) for p in s["parts"]]


def _order(x):
    """int64 keys whose order is that of float32 values, and of places behind it, the lowest first."""
    u = x.contiguous().view(torch.int32).to(torch.int64)
    u = torch.where(u < 0, -(u & 0x7fffffff), u)
    return u * (1 << 31) - torch.arange(x.shape[1], device=DEV)[None, :]


def _plain_logprobs(s, case):
    tok = s["tokens"].to(torch.int64)[:, None]
    x = s["logits"].to(torch.float32)
    top = x.amax(dim=1, keepdim=True)
    given = torch.gather(x, 1, tok)
    above = (x > given).sum(dim=1) + ((x == given) & (torch.arange(x.shape[1], device=DEV)[None, :] < tok)).sum(dim=1)
    d = x - top
    e = torch.exp(d)
    total = e.sum(dim=1, keepdim=True)
    mean = torch.where(e > 0, d * e, torch.zeros_like(e)).sum(dim=1, keepdim=True) / total
    log = torch.log(total)
    out = [(given - top - log)[:, 0], above.to(torch.int32), (log - mean)[:, 0]]
    if case["top"]:
        best = torch.topk(_order(x), case["top"], dim=1).indices
        out += [best.to(torch.int32), torch.gather(x, 1, best) - top - log]
    return out


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "adapters": _exact_adapters, "logprobs": _exact_logprobs}[case["path"]](s, case)


def _exact_rotary(s, case):
    """Pairs as complex numbers times e^(i angle)."""
    d, p = case["dim"], case["part"]
    turn = torch.polar(torch.full((), s["scale"], dtype=torch.float64, device=DEV), s["positions"].double()[:, None] * s["inv_freq"])
    first = torch.arange(0, p, 2, device=DEV) if case["interleaved"] else torch.arange(p // 2, device=DEV)
    second = first + 1 if case["interleaved"] else first + p // 2

    def turned(x):
        y = x.reshape(x.shape[0], -1, d).double().clone()
        z = torch.complex(y[..., first], y[..., second]) * turn[:, None, :]
        y[..., first], y[..., second] = z.real, z.imag
        return y.reshape(x.shape[0], -1)

    q, k = turned(s["query"]), turned(s["key"])
    if not case["cache"]:
        return [q, k]
    caches = [s["key_cache"].double(), s["value_cache"].double()]
    for c, x in zip(caches, (k, s["value"].double())):
        c.view(-1, x.shape[1]).index_copy_(0, s["at"], x[s["live"]])
    return [q] + caches


def _exact_adapters(s, case):
    """One adapter after the other, its rows found from the ids."""
    outs = []
    for p in s["parts"]:
        out = p["base"].double()
        for a in range(case["adapters"]):
            rows = torch.nonzero(s["ids"] == a)[:, 0]
            at = 0
            for i, n in enumerate(p["widths"] if rows.numel() else ()):
                h = torch.mm(p["x"][rows].double(), p["a"][a, i].double().t())
                out[rows, at:at + n] += s["scales"][a].double() * torch.mm(h, p["b"][a, at:at + n].double().t())
                at += n
        outs.append(out)
    return outs


def _exact_logprobs(s, case):
    t, step = case["rows"], max(1, (1 << 27) // case["vocab"])
    got = [[], [], []]
    for r in range(0, t, step):
        lp = torch.log_softmax(s["logits"][r:r + step].double(), dim=1)
        got[0].append(torch.gather(lp, 1, s["tokens"][r:r + step, None].long())[:, 0])
        got[1].append(torch.special.entr(lp.exp()).sum(dim=1))
        got[2].append(torch.topk(lp, case["top"], dim=1).values if case["top"] else lp[:, :0])
    lp, entropy, best = (torch.cat(x) for x in got)
    return [lp, None, entropy, None, best] if case["top"] else [lp, None, entropy]
