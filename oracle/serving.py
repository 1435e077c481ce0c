"""Operators of a serving step, in float64: rotary positions of any layout, log probabilities of given tokens, low-rank adapters.
Test infrastructure only."""
import numpy as np


def rotary(x, positions, inv_freq, head_dim, interleaved=False, scale=1.0, offset=0):
    """x [T, heads * head_dim]: the pairs of the 2 * len(inv_freq) columns from ``offset`` on of every head as complex numbers, times
    scale * e^(i position inv_freq)."""
    inv_freq = np.asarray(inv_freq, dtype=np.float64)
    t, p = len(positions), len(inv_freq)
    y = np.array(x, dtype=np.float64).reshape(t, -1, head_dim)
    first = offset + (2 * np.arange(p) if interleaved else np.arange(p))
    second = first + (1 if interleaved else p)
    turn = scale * np.exp(1j * np.asarray(positions, dtype=np.float64)[:, None] * inv_freq)
    z = (y[:, :, first] + 1j * y[:, :, second]) * turn[:, None, :]
    y[:, :, first], y[:, :, second] = z.real, z.imag
    return y.reshape(t, -1)


def token_logprobs(logits, tokens, n):
    """-> (log probabilities, ranks, entropy, top tokens, their log probabilities).  NaN logits are -inf, +inf the largest float32;
    a token outside the vocabulary has -inf and rank -1; ties go to the lowest token."""
    x = np.array(logits, dtype=np.float64)
    x[np.isnan(x)] = -np.inf
    x = np.minimum(x, np.float64(np.finfo(np.float32).max))
    t, v = x.shape
    lp, entropy = np.full_like(x, -np.inf), np.zeros(t)
    for i in range(t):
        if np.isfinite(x[i]).any():
            d = x[i] - x[i].max()
            e = np.exp(d)
            lp[i] = d - np.log(e.sum())
            p = e / e.sum()
            entropy[i] = -(p[p > 0] * lp[i][p > 0]).sum()
    order = np.argsort(-x, axis=1, kind="stable")
    rank = np.empty_like(order)
    np.put_along_axis(rank, order, np.arange(v)[None, :].repeat(t, 0), axis=1)
    tok = np.asarray(tokens, dtype=np.int64)
    ok = (tok >= 0) & (tok < v)
    at = np.where(ok, tok, 0)
    row = np.arange(t)
    top = order[:, :n]
    return (np.where(ok, lp[row, at], -np.inf), np.where(ok, rank[row, at], -1), entropy, top, np.take_along_axis(lp, top, axis=1))


def adapter_linear(x, a, b, ids, base, widths, ranks, scales):
    """x [T, K], a [n, slices, R, K], b [n, N, R], base [T, N].  -> (result, magnitude of its terms), both [T, N]."""
    x, base = np.asarray(x, np.float64), np.asarray(base, np.float64)
    out, mag = base.copy(), np.abs(base)
    for t, i in enumerate(ids):
        if not 0 <= i < len(a):
            continue
        at, r = 0, int(ranks[i])
        for s, n in enumerate(widths):
            ai, bi = np.asarray(a[i, s, :r], np.float64), np.asarray(b[i, at:at + n, :r], np.float64)
            out[t, at:at + n] += scales[i] * (bi @ (ai @ x[t]))
            mag[t, at:at + n] += abs(scales[i]) * (np.abs(bi) @ np.abs(ai @ x[t]))
            at += n
    return out, mag
