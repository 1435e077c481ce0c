"""Oracle of the operators that a generation loop runs between two model steps: beam selection and the block tables of
sequences that share blocks.  Plain loops over definitions, float64; nothing here is taken from the package.
"""
import numpy as np


def beam_search_select(logits, scores, n, eos=-1):
    """logits [B, K, V], scores [B, K] -> candidates (score float64, beam, token) [B, n] by score, then place, and the first K that
    are not eos (score, row, token) [B, K].  NaN logits are -inf, +inf the largest float32; a beam without a finite running
    score scores -inf."""
    b, k, v = logits.shape
    cand, going = [], []
    for g in range(b):
        x = logits[g].astype(np.float64)
        x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max))
        total = np.full((k, v), -np.inf)
        for i in range(k):
            run, top = float(scores[g, i]), x[i].max()
            if abs(run) < 1e30 and top > -np.inf:
                d = x[i] - top
                total[i] = run + (d - np.log(np.exp(d).sum()))
        flat = total.reshape(-1)
        order = np.lexsort((np.arange(k * v), -flat))[:n]
        cand.append([(flat[o], o // v, o % v) for o in order])
        going.append([(s, g * k + i, t) for s, i, t in cand[-1] if t != eos][:k])
    pick = lambda rows, j, t: np.array([[e[j] for e in r] for r in rows], dtype=t)  # noqa: E731
    return ((pick(cand, 0, np.float64), pick(cand, 1, np.int64), pick(cand, 2, np.int64)),
            (pick(going, 0, np.float64), pick(going, 1, np.int64), pick(going, 2, np.int64)))


def fork_blocks(tables, lens, num_blocks, block_size, parents=None, new_tokens=0, window=None, sinks=0, held=None):
    """(tables, lens, slots, copies, missing) of ``mindformers_amd.ops.fork_blocks``, token by token."""
    s, m = tables.shape
    parents = np.arange(s) if parents is None else parents
    out, olens = np.full((s, m), -1, np.int64), np.zeros(s, np.int64)
    eldest, opens = {}, []
    for r in range(s):
        p = int(parents[r])
        if not 0 <= p < s:
            continue
        n = olens[r] = min(max(int(lens[p]), 0), m * block_size)
        for j in range(m):
            tokens = [t for t in range(j * block_size, (j + 1) * block_size)]
            page = int(tables[p, j])
            seen = window is None or any(t > n - window or t < sinks for t in tokens)
            if tokens[0] < n and 0 <= page < num_blocks and seen:
                out[r, j] = page
        j = n // block_size
        if n % block_size and out[r, j] >= 0:
            if p in eldest:
                opens.append((r, j, int(out[r, j]), n % block_size))
                out[r, j] = -1
            else:
                eldest[p] = r
    named = set(out[out >= 0].tolist())
    free = [i for i in range(num_blocks) if i not in named and not (held is not None and held[i])]
    copies, missing = [], 0
    slots = np.full((s, new_tokens), -1, np.int64)
    for r in range(s):
        if not 0 <= int(parents[r]) < s:
            continue
        want = [(j, src, n) for row, j, src, n in opens if row == r]
        n = int(olens[r])
        want += [(j, -1, 0) for j in range(-(-n // block_size), -(-(n + new_tokens) // block_size))]
        for j, src, rows in want:
            page = free.pop(0) if free and j < m else -1            # no block is taken where the table has no place for it
            if page < 0:
                missing += 1
                continue
            out[r, j] = page
            if src >= 0:
                copies.append((src, page, rows))
        for t in range(new_tokens):
            if n + t < m * block_size and out[r, (n + t) // block_size] >= 0:
                slots[r, t] = out[r, (n + t) // block_size] * block_size + (n + t) % block_size
        olens[r] = min(n + new_tokens, m * block_size)
    copies += [(-1, -1, 0)] * (s - len(copies))
    return out, olens, slots.reshape(-1), np.array(copies), missing


def compact_blocks(tables, num_blocks, block_size, held=None):
    """(tables, copies, n) of ``mindformers_amd.ops.compact_blocks``."""
    mine = [i for i in range(num_blocks) if not (held is not None and held[i])]
    live = [i for i in mine if (tables == i).any()]
    target = mine[:len(live)]
    moves = [i for i in live if i not in target]
    holes = [i for i in target if i not in live]
    to = dict(zip(moves, holes))
    out = np.array([[to.get(int(p), int(p)) if 0 <= p < num_blocks else -1 for p in row] for row in tables])
    copies = [(a, b, block_size) for a, b in zip(moves, holes)]
    copies += [(-1, -1, 0)] * (num_blocks // 2 - len(copies))
    return out, np.array(copies).reshape(-1, 3), len(live)


def window_attention(query, keys, values, lens, q_lens, n_heads, n_kv, scale, window, sinks, of="value"):
    """Attention where the row at position p sees the tokens j <= p with j > p - window or j < sinks, float64.  query [T, H * D], the
    sequences' rows packed; keys / values: per sequence [L, n_kv, D].  ``of``: "value", "magnitude" (the same of |values|) or "sum" (the
    visible |values| added up)."""
    t = query.shape[0]
    d = query.shape[1] // n_heads
    out, row = np.zeros((t, n_heads, d)), 0
    for k, v, n, ql in zip(keys, values, lens, q_lens):
        for i in range(int(ql)):
            p = int(n) - int(ql) + i
            if p >= 0:
                seen = [j for j in range(p + 1) if j > p - window or j < sinks]
                kk, vv = (np.repeat(x[seen].astype(np.float64), n_heads // n_kv, axis=1) for x in (k, v if of == "value" else np.abs(v)))
                s = np.einsum("hd,jhd->hj", query[row].reshape(n_heads, d).astype(np.float64), kk) * scale
                w = np.exp(s - s.max(axis=1, keepdims=True))
                w = w * 0 + 1 if of == "sum" else w / w.sum(axis=1, keepdims=True)
                out[row] = np.einsum("hj,jhd->hd", w, vv)
            row += 1
    return out.reshape(t, -1)
