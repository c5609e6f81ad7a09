"""What the operators around the 4-bit cache compute (include/prima_b200.h), in 64 bits and cell by cell: attention behind common prefixes, logarithms of rows' sums, sums of cells' weights, the
choice of cells that stay, verification of drafts."""
import numpy as np

import ref_kv4 as R


def read(pages, ids, length, dim):
    """keys, values [kv_heads, cells, dim] and which cells there are, of the pages `ids` of a layer [pages, kv_heads, bytes]"""
    length = max(int(length), 0)
    n = min(-(-length // R.CELLS), len(ids))
    ids = np.asarray(ids[:n])
    good = (ids >= 0) & (ids < len(pages))
    heads = pages.shape[1]
    with np.errstate(invalid="ignore", over="ignore"):
        kv = R.unpack(pages[np.where(good, ids, 0)], dim) if n else [np.zeros((0, heads, R.CELLS, dim))] * 2
    k, v = (x.transpose(1, 0, 2, 3).reshape(heads, -1, dim) for x in kv)
    here = np.repeat(good, R.CELLS) & (np.arange(n * R.CELLS) < length)
    return np.where(here[None, :, None], k, 0.0), np.where(here[None, :, None], v, 0.0), here


def attend(q, pages, table, q_start, kv_len, n_head_kv, dim, scale, window=0, first=0, group_start=None, prefix_len=None, prefix_table=None):
    """q [tokens, heads, dim] -> out, bound of its error, lse, bound of its error, weights: of each sequence [cells of its own] (added up over queries and heads) and bound of their error.

    The bounds are ref_kv4.attend's: a score is a sum of dim products, each rounded and added with 2^-23 of the sum of magnitudes at most, twice that for operands of 22 bits; a weight is off by its
    score's error, 2^-22 of the exponential and 2^-23 of its argument, |score| times that.  A logarithm: its sum's error, and half a step of itself.  A weight by a logarithm that was rounded: that, too,
    and the logarithm's product with log2 e."""
    group = q.shape[1] // n_head_kv
    out, bound = np.full(q.shape, np.nan), np.zeros(q.shape)
    lse, lse_bound = (np.full(q.shape[:2], x) for x in (np.nan, 0.0))
    sums, sums_bound, fronts = [], [], {}
    for s in range(len(kv_len)):
        n, length = q_start[s + 1] - q_start[s], max(int(kv_len[s]), 0)
        k, v, here = read(pages, table[s], length, dim)
        at = np.arange(k.shape[1])
        if group_start is not None and group_start[0] <= s < group_start[-1]:
            g = int(np.searchsorted(group_start, s, side="right")) - 1
            if g not in fronts:
                fronts[g] = read(pages, prefix_table[g], prefix_len[g], dim)
            pk, pv, ph = fronts[g]
            k, v, here, at = np.concatenate((pk, k), 1), np.concatenate((pv, v), 1), np.concatenate((ph, here)), np.concatenate((np.full(pk.shape[1], -2 ** 40), at))
        worth, worth_bound = np.zeros(length), np.zeros(length)
        for i in range(n):
            p, row = int(kv_len[s]) - n + i, q_start[s] + i
            see = here & (at <= p)
            if window:
                see = see & ((p - at < window) | (at < first))
            out[row], lse[row] = 0.0, -np.inf
            if not see.any():
                continue
            for h in range(n_head_kv):
                mine = slice(h * group, (h + 1) * group)
                kk, vv, qq = k[h][see], v[h][see], q[row, mine]
                z = qq @ kk.T * scale
                top = z.max(-1, keepdims=True)
                w = np.exp(z - top)
                total = w.sum(-1, keepdims=True)
                w /= total
                out[row, mine] = w @ vv
                lse[row, mine] = (top + np.log(total))[:, 0]
                mag = (np.abs(qq) @ np.abs(kk).T).max(-1) * abs(scale)
                rel = 2 * (dim + 8) * 2.0 ** -23 * mag + np.abs(z).max(-1) * 2.0 ** -22 + 2.0 ** -20 + (see.sum() / 16 + 64) * 2.0 ** -23
                bound[row, mine] = (rel * np.abs(vv).max())[:, None]
                lse_bound[row, mine] = rel + np.abs(lse[row, mine]) * 2.0 ** -22
                own = at[see] >= 0
                worth[at[see][own]] += w.sum(0)[own]
                worth_bound[at[see][own]] += ((rel + 3 * np.abs(lse[row, mine]) * 2.0 ** -23)[:, None] * w).sum(0)[own]
        sums.append(worth)
        sums_bound.append(worth_bound + worth * (n * q.shape[1] + 16) * 2.0 ** -24)
    return out, bound, lse, lse_bound, sums, sums_bound


def select(sums, length, budget, first, last):
    """indices of the cells that stay, ascending"""
    x = np.where(np.isnan(sums[:length]), -np.inf, sums[:length]) + 0.0
    count = max(0, min(length, budget))
    last = min(last, count)
    first = min(first, count - last)
    between = sorted(range(first, length - last), key=lambda j: (-x[j], j))[:count - first - last]
    return np.array(sorted([*range(first), *between, *range(length - last, length)]), dtype=np.int64)


def softmax(x, t):
    """[vocab] of logits times t; None: there are no weights"""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf or not t >= 0:
        return None
    if t == np.inf:
        w = np.zeros(len(x))
        w[int(np.argmax(x))] = 1.0
    elif top == np.inf:
        w = (x == np.inf).astype(np.float64)
    else:
        w = np.where(x == -np.inf, 0.0, np.exp((np.where(x == -np.inf, top, x) - top) * t))
    return w / w.sum()


def draw(w, v):
    c = np.cumsum(w)
    above = np.nonzero((c > v * c[-1]) & (w > 0))[0]
    return int(above[0]) if len(above) else int(np.nonzero(w > 0)[0][-1])


def verify(target, draft, tokens, t, u, v):
    """one sequence: target [n + 1, vocab], draft [n, vocab] or None -> (accepted, the token behind them, how near a decision was to the other way)"""
    near = np.inf
    for i, x in enumerate(tokens):
        p = softmax(target[i], t)
        q = softmax(draft[i], t) if draft is not None else np.eye(1, target.shape[1], x if 0 <= x < target.shape[1] else -1)[0]
        inside = p is not None and 0 <= x < len(p)
        px, qx = (p[x], 0.0 if q is None else q[x]) if inside else (0.0, 0.0)
        if inside and px > 0:
            near = min(near, abs(u[i] * qx / px - 1.0))
        if inside and u[i] * qx < px:
            continue
        if p is None:
            return i, -1, near
        if draft is None:
            q = np.zeros(len(p))
            if 0 <= x < len(p):
                q[x] = p[x]
        rest = np.maximum(p - (0.0 if q is None else q), 0.0)
        return i, draw(rest if rest.sum() > 0 else p, v), near
    p = softmax(target[len(tokens)], t)
    return len(tokens), -1 if p is None else draw(p, v), near
