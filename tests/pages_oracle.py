"""Plain 64-bit forms of the paged cache's operators and of sampling, from the
definitions in include/surge.h, on numpy arrays."""
import numpy as np


def where(table, pages, page, s, j):
    """(page, row) of slot j of sequence s, or None where the page is not in the pool."""
    p = int(table[s, j // page])
    return (p, j % page) if 0 <= p < pages else None


def store(k, v, kp, vp, table, span, weight, pos):
    """In place. k, v [n_seq][n][n_kv][hd]; a row is float16(x), which numpy rounds to nearest even."""
    pages, page = kp.shape[:2]
    cap = table.shape[1] * page
    for s in range(len(table)):
        first, rows, at = (int(x) for x in span[s])
        for i in range(min(rows, k.shape[1])):
            if first < 0 or first + i >= cap:
                continue
            c = where(table, pages, page, s, first + i)
            if c is None:
                continue
            with np.errstate(over="ignore"):
                kp[c], vp[c] = k[s, i].astype(np.float16), v[s, i].astype(np.float16)
            if weight is not None:
                weight[s, :, first + i] = 0
            if pos is not None:
                pos[s, :, first + i] = np.uint32((at + i) & 0xFFFFFFFF).astype(np.int32) if at + i >= 2 ** 31 else at + i


def attn(q, kp, vp, table, lens, scale, weight=None):
    """out, weights, and a bound on the error of each in f32 arithmetic.

    With A = the largest sum of |q_d k_d| |scale| of a head's scores, a score that is summed in f32 is off by at most
    A (8 sqrt(hd) + 8) 2^-24 (its roundings, each at most half a step of the sum so far, taken as independent and at
    eight times their deviation), and a weight, exp of a difference of two of them over a sum, by 2 that plus the
    roundings of exp, sum and quotient; the values' sum adds 8 sqrt(len) roundings more."""
    n, nh, hd = q.shape
    pages, page, nkv = kp.shape[:3]
    g, cap, u = nh // nkv, table.shape[1] * page, 2.0 ** -24
    out, ob = np.zeros((n, nh, hd)), np.zeros((n, nh, hd))
    w = np.zeros((n, nkv, cap)) if weight is None else weight.astype(np.float64)
    wb = np.zeros((n, nkv, cap))
    for s in range(n):
        ln = min(max(int(lens[s]), 0), cap)
        cells = [where(table, pages, page, s, j) for j in range(ln)]
        js = np.array([j for j in range(ln) if cells[j] is not None], dtype=int)
        if not len(js):
            continue
        a, b = (np.array([cells[j][i] for j in js]) for i in (0, 1))
        for h in range(nh):
            kd, vd = kp[a, b, h // g].astype(np.float64), vp[a, b, h // g].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                x = (kd @ q[s, h].astype(np.float64)) * float(scale)
                big = (np.abs(kd) @ np.abs(q[s, h].astype(np.float64))).max() * abs(float(scale))
                p = np.exp(x - x.max())
                p /= p.sum()
                e = (2 * big * (8 * np.sqrt(hd) + 8) + 8 * np.sqrt(len(js)) + 16) * u
                out[s, h], ob[s, h] = p @ vd, (p @ np.abs(vd)) * e + 1e-30
            w[s, h // g, js] += p
            wb[s, h // g, js] += p * e
    return out, ob, w, wb + np.abs(w) * 2 * (g + 1) * u + 1e-37


def evict(kp, vp, table, lens, weight, pos, keep, recent):
    """Pools in place; weight_out and pos_out, of which the slots below min(keep, len) count."""
    pages, page, nkv = kp.shape[:3]
    cap = table.shape[1] * page
    wo, po = weight.copy(), pos.copy()
    for s in range(len(table)):
        ln = min(max(int(lens[s]), 0), cap)
        if ln <= keep:
            continue
        for h in range(nkv):
            p = pos[s, h, :ln].astype(np.int64)
            w = weight[s, h, :ln].astype(np.float64)
            new = p > p.max() - recent
            w = np.where(new, np.inf, w)
            nan = np.isnan(w)
            order = np.lexsort((np.arange(ln), -np.where(nan, 0, w), nan, ~new))
            best = order[:keep]
            holes, movers = np.setdiff1d(np.arange(keep), best), np.sort(best[best >= keep])
            assert len(holes) == len(movers)
            wo[s, h, holes], po[s, h, holes] = weight[s, h, movers], pos[s, h, movers]
            for d, f in zip(holes, movers):
                x, y = where(table, pages, page, s, int(f)), where(table, pages, page, s, int(d))
                if x is not None and y is not None:
                    kp[y][h], vp[y][h] = kp[x][h], vp[x][h]
    return wo, po


def sample(x, temperature, top_k, top_p, min_p, u):
    """One row: (token or -1, probabilities, the distance of the nearest border over the sum it is a border of)."""
    temperature, top_p, min_p, u = (float(np.float32(v)) for v in (temperature, top_p, min_p, u))
    probs = np.zeros(len(x))
    x = x.astype(np.float64)
    ids = np.flatnonzero(x > -np.inf)
    if not len(ids):
        return -1, probs, 1.0
    if not temperature > 0:
        temperature, top_k = 1.0, 1
    ids = ids[np.argsort(-x[ids], kind="stable")]
    if 0 < top_k < len(ids):
        ids = ids[:top_k]
    top = x[ids[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x[ids] == top, 1.0, np.exp((x[ids] - top) / temperature) if top < np.inf else 0.0)
    w = w.astype(np.longdouble)
    margin = 1.0
    if top_p < 1:
        before = np.concatenate([[0], np.cumsum(w)[:-1]])
        lim = top_p * w.sum()
        stay = before < lim
        stay[0] = True
        margin = min(margin, float(np.abs(before[1:] - lim).min() / w.sum()) if len(w) > 1 else 1.0)
        ids, w = ids[stay], w[stay]
    if min_p > 0:
        stay = (w >= min_p)
        stay[0] = True
        margin = min(margin, float(np.abs(w[1:] - min_p).min()) if len(w) > 1 else 1.0)
        ids, w = ids[stay], w[stay]
    back = np.argsort(ids)
    ids, w = ids[back], w[back]
    total = w.sum()
    u = 0.0 if not u > 0 else min(u, 1 - 2.0 ** -24)
    cum = np.cumsum(w)
    at = int(np.flatnonzero(cum > u * total)[0])
    if u:
        margin = min(margin, float(np.abs(cum - u * total).min() / total))
    probs[ids] = (w / total).astype(np.float64)
    return int(ids[at]), probs, margin
