"""Plain 64-bit restatements of the serving operators (moonshine_amd/ops.py) for their tests: numpy on the CPU, element by element from
the definitions, without the library's layout or kernels."""
from __future__ import annotations

import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise(x: np.ndarray) -> np.ndarray:
    """The values that stand for x [..., width] in the 4-bit cache."""
    x = np.nan_to_num(np.asarray(x, np.float64), nan=0.0, posinf=float(np.finfo(np.float32).max), neginf=-float(np.finfo(np.float32).max))
    out = np.zeros_like(x)
    for at in range(0, x.shape[-1], 32):
        part = x[..., at:at + 32]
        amax = np.abs(part).max(-1, keepdims=True)
        mantissa, power = np.frexp(amax)                       # amax = mantissa * 2^power, mantissa in [1/2, 1) (0: 0)
        power = np.clip(power - 1 + (mantissa * 2 >= 1.75) - 2, -100, 125)
        power = np.where(amax == 0, -100, power)
        unit = np.ldexp(1.0, power)
        y = np.abs(part) / unit
        d = np.abs(y[..., None] - MAGNITUDES)
        best = d.min(-1, keepdims=True)
        ties = d == best                                       # two neighbours at most: the even code
        code = np.where(ties.sum(-1) > 1, np.where(ties[..., 0::2].any(-1), 2 * ties[..., 0::2].argmax(-1), 0), d.argmin(-1))
        out[..., at:at + 32] = np.sign(part) * MAGNITUDES[code] * unit
    return out


def attention(q, k, v, visible, scale):
    """q [rows, heads, d], k / v [tokens, kv_heads, d], visible [rows, tokens] -> out, lse, and for the error bounds: the largest
    sum |q_i k_i| * scale of a visible token, the largest |score|, and sum p |v|."""
    rows, heads, d = q.shape
    per = heads // k.shape[1]
    out, lse = np.zeros((rows, heads, d)), np.full((rows, heads), -np.inf)
    mass, top, spread = np.zeros((rows, heads)), np.zeros((rows, heads)), np.zeros((rows, heads, d))
    for h in range(heads):
        kk, vv = k[:, h // per], v[:, h // per]
        s = scale * (q[:, h] @ kk.T)
        a = abs(scale) * (np.abs(q[:, h]) @ np.abs(kk).T)
        for r in range(rows):
            see = visible[r]
            if not see.any():
                continue
            x = s[r, see]
            m = x.max()
            e = np.exp(x - m)
            lse[r, h] = m + np.log(e.sum())
            p = e / e.sum()
            out[r, h] = p @ vv[see]
            spread[r, h] = p @ np.abs(vv[see])
            mass[r, h], top[r, h] = a[r, see].max(), np.abs(x).max()
    return out, lse, mass, top, spread


def visible(n_rows, n_tokens, causal, window=0):
    t = np.arange(n_tokens)[None, :]
    place = n_tokens - n_rows + np.arange(n_rows)[:, None]
    if not causal:
        return np.ones((n_rows, n_tokens), bool)
    see = t <= place
    return see & (t > place - window) if window > 0 else see


def beam_select(logits, scores, finished, eos):
    """-> scores, parents, tokens, finished and the candidates' 64-bit scores in order (beams + 1 of them, -inf behind)."""
    batch, beams, vocab = logits.shape
    outs = []
    for b in range(batch):
        cands = []
        for k in range(beams):
            if not scores[b, k] > -np.inf:
                continue
            if finished[b, k]:
                cands.append((-float(scores[b, k]), k * vocab + max(eos, 0), eos))
                continue
            x = np.asarray(logits[b, k], np.float64)
            x = np.where(np.isnan(x), -np.inf, np.minimum(x, float(np.finfo(np.float32).max)))
            m = x.max()
            if m == -np.inf:
                continue
            logp = float(scores[b, k]) - (m + np.log(np.exp(x - m).sum())) + x
            keep = np.lexsort((np.arange(vocab), -x))[:beams + 1]        # by logit, then by id
            cands += [(-float(logp[v]), k * vocab + int(v), int(v)) for v in keep if x[v] > -np.inf]
        cands.sort(key=lambda c: c[:2])
        row = []
        for i in range(beams):
            if i < len(cands):
                s, flat, token = cands[i]
                parent = flat // vocab
                row.append((-s, parent, token, bool(finished[b, parent]) or token == eos))
            else:
                row.append((-np.inf, i, eos, True))
        outs.append((row, [-c[0] for c in cands[:beams + 1]], [c[1] // vocab for c in cands[:beams + 1]]))
    pick = lambda i, t: np.array([[c[i] for c in row] for row, _, _ in outs], t)  # noqa: E731
    return pick(0, np.float64), pick(1, np.int64), pick(2, np.int64), pick(3, bool), [(s, p) for _, s, p in outs]


def reorder(state, parents, lengths):
    """state [outer, batch, beams, inner, rows, ...]"""
    out = state.copy()
    for b in range(parents.shape[0]):
        for k in range(parents.shape[1]):
            p = int(parents[b, k])
            if 0 <= p < parents.shape[1]:
                out[:, b, k, :, :lengths[b]] = state[:, b, p, :, :lengths[b]]
    return out


def page_plan(table, kv_lens, new_lens, row_start, rows, free, page):
    table, slots, used = table.copy(), np.full(rows, -1, np.int64), 0
    width = table.shape[1]
    for b in range(table.shape[0]):
        held = min(max(int(kv_lens[b]), 0), width * page)
        new = min(max(int(new_lens[b]), 0), held)
        kept, need = -(-(held - new) // page), -(-held // page)
        for c in range(kept, width):
            table[b, c] = -1
            if c < need:
                if used < len(free):
                    table[b, c] = free[used]
                used += 1
        for i in range(new):
            at = int(row_start[b]) + i
            if 0 <= at < rows:
                p = held - new + i
                slots[at] = table[b, p // page] * page + p % page if table[b, p // page] >= 0 else -1
    return table, slots, used
