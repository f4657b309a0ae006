"""Plain 64-bit forms of the beam-search and paged-cache operators (include/b200_whisper.h), written from their formulas."""
import numpy as np


def beam_select(logits, score, done, banned, eos, n_beam):
    """logits [rows][V] float64, score [rows], done [rows] or None, banned [rows or 1][V] bool or None."""
    rows, V = logits.shape
    out = dict(score=[], token=[], parent=[], done=[])
    for s in range(rows // n_beam):
        cand = []
        for b in range(n_beam):
            r = s * n_beam + b
            if not score[r] > -np.inf:
                continue
            if done is not None and done[r]:
                cand.append((-float(score[r]), b, eos if 0 <= eos < V else 0, eos, True))
                continue
            x = logits[r].astype(np.float64).copy()
            x[np.isnan(x)] = -np.inf
            if banned is not None:
                x[banned[r % len(banned)]] = -np.inf
            m = x.max()
            if m == -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                d = np.where(x == m, 0.0, x - m)
            lp = float(score[r]) + (d - np.log(np.exp(d).sum()))
            best = np.lexsort((np.arange(V), -lp))[:n_beam]
            cand += [(-lp[v], b, int(v), int(v), int(v) == eos) for v in best if lp[v] > -np.inf]
        cand.sort(key=lambda c: c[:3])
        for k in range(n_beam):
            if k < len(cand):
                out["score"].append(-cand[k][0]); out["parent"].append(cand[k][1]); out["token"].append(cand[k][3]); out["done"].append(int(cand[k][4]))
            else:
                out["score"].append(-np.inf); out["parent"].append(-1); out["token"].append(-1); out["done"].append(1)
    return {k: np.array(v) for k, v in out.items()}


def ceil(n, ps):
    return -(-int(n) // ps)


def pages_update(tables, lens, refs, parent, keep, n_new, ps):
    """Returns tables, lens, refs, copies [(src, dst, tokens)], status; status != 0 leaves the state as it was."""
    rows, width = tables.shape
    refs = [int(r) for r in refs]
    for i in range(rows):
        p, k, n = int(parent[i]), int(keep[i]), int(n_new[i])
        if not (0 <= p < rows and k >= 0 and n >= 0 and 0 <= lens[i] <= width * ps and k + n <= width * ps) or k > lens[p]:
            return tables.copy(), lens.copy(), np.array(refs), [], -1
        if any(not 0 <= t < len(refs) for t in tables[i, :ceil(lens[i], ps)]):
            return tables.copy(), lens.copy(), np.array(refs), [], -1
    free = [p for p, r in enumerate(refs) if r == 0]
    new = [[int(t) for t in tables[int(parent[i]), :ceil(keep[i], ps)]] for i in range(rows)]
    held = list(refs)
    for i in range(rows):
        for t in tables[i, :ceil(lens[i], ps)]:
            held[t] -= 1
        for t in new[i]:
            held[t] += 1
    writes = [new[i][-1] if keep[i] % ps and n_new[i] > 0 else None for i in range(rows)]
    copies, wanted = [], 0
    plan = []
    for i in range(rows):
        w = writes[i]
        copy = w is not None and (w in writes[:i] or held[w] > writes.count(w))
        more = ceil(keep[i] + n_new[i], ps) - ceil(keep[i], ps)
        plan.append((copy, more))
        wanted += copy + more
    if wanted > len(free):
        return tables.copy(), lens.copy(), np.array(refs), [], wanted - len(free)
    for i, (copy, more) in enumerate(plan):
        if copy:
            d = free.pop(0)
            copies.append((new[i][-1], d, int(keep[i]) % ps))
            held[new[i][-1]] -= 1
            held[d] = 1
            new[i][-1] = d
        for _ in range(more):
            d = free.pop(0)
            held[d] = 1
            new[i].append(d)
    out = np.full_like(tables, -1)
    for i in range(rows):
        out[i, :len(new[i])] = new[i]
    return out, np.array([int(a) + int(b) for a, b in zip(keep, n_new)]), np.array(held), copies, 0


def pages_compact(tables, lens, refs, ps):
    """Returns tables, lens, refs, remap, moves [(src, dst)]."""
    live = [p for p, r in enumerate(refs) if r != 0]
    n = len(live)
    src, dst = [p for p in live if p >= n], [p for p in range(n) if refs[p] == 0]
    remap = np.full(len(refs), -1)
    for p in live:
        remap[p] = p
    for a, b in zip(src, dst):
        remap[a] = b
    held = np.zeros(len(refs), int)
    for p in live:
        held[remap[p]] = refs[p]
    out = np.full_like(tables, -1)
    for i in range(len(tables)):
        u = ceil(lens[i], ps)
        out[i, :u] = remap[tables[i, :u]]
    return out, lens.copy(), held, remap, list(zip(src, dst))


def attention(q, k, v, n_new, length, scale, causal):
    """q [n_new][H][D], k, v [length][Hkv][D], all float64 -> out, lse, and sum_j w_j |v_j| / sum_j w_j, the size that roundings scale with."""
    H, D = q.shape[1:]
    g = H // k.shape[1] if k.shape[1] else 1
    out, mag, lse = np.zeros(q.shape), np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    reach = np.zeros(q.shape[:2])
    seen = np.array([length - n_new + t + 1 if causal else length for t in range(n_new)])
    hidden = np.arange(length)[None, :] >= seen[:, None]
    rows = seen > 0
    if length == 0 or not rows.any():
        return out, lse, mag, reach
    for h in range(H):
        kh, vh = k[:, h // g], v[:, h // g]
        with np.errstate(invalid="ignore"):
            s = q[:, h] @ kh.T * scale
        s[hidden] = -np.inf
        s, hid = s[rows], hidden[rows]
        m = s.max(1, keepdims=True)
        w = np.exp(s - m)
        w[hid] = 0
        total = w.sum(1)
        lse[rows, h] = m[:, 0] + np.log(total)
        out[rows, h] = w @ vh / total[:, None]
        mag[rows, h] = w @ np.abs(vh) / total[:, None]
        a = np.abs(q[rows, h]) @ np.abs(kh).T                   # largest sum of |products| behind a score
        a[hid] = 0
        reach[rows, h] = a.max(1) * abs(scale)
    return out, lse, mag, reach
