"""Plain implementations of beam selection, in 64 bits, and of forks of paged
requests, in whole numbers, for the tests."""
from __future__ import annotations

import numpy as np

OK, EINVAL, ENOMEM = 0, 1, 3


def select(logits, scores, width, k, done=None, eos=-1):
    """(parent, token, score, done, gap) of every place; `gap`: how far the
    score lies from the next one, in 64 bits.  logits [rows][vocab], scores
    [rows]."""
    logits, scores = np.asarray(logits, np.float64), np.asarray(scores, np.float64)
    out = []
    for g in range(len(scores) // width):
        cand = []
        for r in range(g * width, (g + 1) * width):
            if not np.isfinite(scores[r]):
                continue
            if done is not None and done[r]:
                cand.append((-scores[r], r, eos, 1))
                continue
            x = logits[r]
            if np.isnan(x).any() or (x == np.inf).any() or not np.isfinite(x).any():
                continue
            top = x.max()
            lse = top + np.log(np.exp(x - top).sum())
            best = np.argsort(-x, kind="stable")[:k + 1]
            cand += [(-(scores[r] + (x[t] - lse)), r, int(t), int(t == eos)) for t in best if x[t] > -np.inf]
        cand.sort(key=lambda c: c[:2])  # (equal scores of a beam stand in token order)
        for i in range(k):
            if i < len(cand):
                s, r, t, d = cand[i]
                out.append((r, t, -s, d, cand[i + 1][0] - s if i + 1 < len(cand) else np.inf))
            else:
                out.append((-1, -1, -np.inf, 0, np.inf))
    return out


def fork(lens, parent, table, shared, ring, cursor, pages, ps):
    """One call.  Returns (status, copies [(from, to, rows)]); lens, table,
    shared, ring and cursor, lists, are changed in place."""
    n, width = len(parent), len(table[0])
    head, free = cursor
    status = [EINVAL if not -1 <= parent[i] < n or lens[i] < 0 or -(-lens[i] // ps) > width else OK for i in range(n)]
    if any(status):
        return status, []
    used = [-(-c // ps) for c in lens]
    in_pool = lambda p: 0 <= p < pages  # noqa: E731
    keeps, wants = {}, []
    for j in range(n):
        sons = [i for i in range(n) if parent[i] == j]
        last = table[j][lens[j] // ps] if lens[j] % ps else -1
        if not sons or not in_pool(last):
            continue
        heir = j if j in sons else sons[0]
        keeps[j] = heir if shared[last] <= 0 else -1
        wants += [i for i in sons if i != keeps[j]]
    wants.sort()
    if len(wants) > free:
        return [ENOMEM if i in wants else OK for i in range(n)], []
    fresh = {i: ring[(head + k) % pages] for k, i in enumerate(wants)}
    old, old_len = [list(t) for t in table], list(lens)
    holders = {p: shared[p] + 1 for j in range(n) for p in old[j][:used[j]] if in_pool(p)}
    for j in range(n):
        for p in old[j][:used[j]]:
            if in_pool(p):
                holders[p] -= 1
    copies = []
    for i in range(n):
        j = parent[i]
        lens[i] = old_len[j] if j >= 0 else 0
        if j < 0:
            continue
        row = old[j][:used[j]]
        if i in fresh:
            if in_pool(fresh[i]):
                copies.append((row[-1], fresh[i], old_len[j] % ps))
            row[-1] = fresh[i]
        for p in row if i not in fresh else row[:-1]:
            if in_pool(p):
                holders[p] += 1
        table[i][:used[j]] = row
    gone = []
    for k in range(width):
        for j in range(n):
            p = old[j][k] if k < used[j] else -1
            if in_pool(p) and holders[p] == 0 and p not in gone:
                gone.append(p)
    for p, h in holders.items():
        shared[p] = max(h - 1, 0)
    for k, p in enumerate(gone):
        ring[(head + free + k) % pages] = p
    cursor[:] = [(head + len(wants)) % pages, free - len(wants) + len(gone)]
    return status, copies
