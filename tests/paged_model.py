"""Plain implementations of the paged KV cache's operators, in whole numbers
and in 64 bits, for the tests: the plan request by request in Python, the
attention row by row from its definition, and the error bound of the
attention's arithmetic."""
from __future__ import annotations

import numpy as np

OK, EINVAL, ERANGE, ENOMEM = 0, 1, 2, 3


def plan(lens, rows, table, ring, cursor, pages, ps, max_seq, max_rows):
    """One step.  Returns a dict of the plan's arrays; `table` and `ring` (or
    None) are lists and are changed in place."""
    n, width = len(lens), len(table[0])
    head, free = cursor if ring is not None else (0, 0)
    row_start, status, out_len, need = [0], [], [], []
    taken = asked = 0
    pushed = []
    for i in range(n):
        new = max(rows[i], 0)
        st = OK
        have, full = -(-lens[i] // ps), -(-(lens[i] + new) // ps)
        if lens[i] < 0 or lens[i] > max_seq or rows[i] < -1:
            st = EINVAL
        elif rows[i] and (lens[i] + new > max_seq or max(have, full) > width):
            st = ERANGE
        elif rows[i] > 0 and any(not 0 <= table[i][j] < pages
                                 for j in range(lens[i] // ps, have if ring is not None else full)):
            st = EINVAL
        elif rows[i] > 0 and row_start[i] + new > max_rows:
            st = ERANGE
        row_start.append(row_start[i] + min(new, max_rows + 1))
        want = full - have if st == OK and rows[i] > 0 and ring is not None else 0
        asked += want
        if want and asked > free:
            st = ENOMEM
        placed = st == OK and rows[i] > 0
        if placed:
            for j in range(want):
                table[i][have + j] = ring[(head + taken + j) % pages]
            taken += want
        if st == OK and rows[i] == -1:
            pushed += [p for p in table[i][:have] if 0 <= p < pages]
        status.append(st)
        need.append(want)
        out_len.append(0 if st == OK and rows[i] == -1 else lens[i] + new if placed else lens[i])
    pos, slot = [-1] * max_rows, [-1] * max_rows
    for i in range(n):
        if status[i] == OK and rows[i] > 0:
            for r in range(rows[i]):
                p = lens[i] + r
                pos[row_start[i] + r] = p
                page = table[i][p // ps]
                slot[row_start[i] + r] = page * ps + p % ps if 0 <= page < pages else -1
    if ring is not None:
        for k, p in enumerate(pushed):
            ring[(head + free + k) % pages] = p
    return {"status": status, "lens": out_len, "row_start": row_start, "row_pos": pos,
            "row_slot": slot,
            "cursor": [(head + taken) % pages, free - taken + len(pushed)] if ring is not None
            else None}


def attend(q, k, v, pos, seen):
    """One request and one q head in float64: q [rows][128], k and v
    [keys][128], pos [rows], seen [keys] (key's page is in the pool).  Returns
    (out, bound): the definition, and how far f16 weights, f32 scores and sums
    and one f16 rounding may be from it.

    The kernel's weight of a key is its exact one times (1 + e), |e| <= 2^-11
    (the f16 rounding of p; weights below 2^-14 of the largest, 2^-25 of it
    instead) + d, d the relative error of p itself: its exponent is off by
    128 * 2^-24 * sum |q k| / sqrt(128) (f32 dot of 128 products) and a few
    2^-24 of the exponent and of exp2 (2^-18 covers |exponent| < 16 in
    2^-24 steps, and exp2's own error).  Perturbed weights move a weighted
    mean by at most 2 max|e| * mean |v - out| (numerator and denominator, first
    order; 1.05 covers the rest).  f32 sums of n terms add n * 2^-24 * mean |v|
    twice (numerator, denominator), and the result is rounded to f16 once:
    2^-11 |out| + 2^-25."""
    scale = 128 ** -0.5
    s = q @ k.T * scale
    vis = (np.arange(len(k))[None] <= np.asarray(pos)[:, None]) & seen[None]
    out = np.zeros_like(q)
    bound = np.zeros_like(q)
    for r in range(len(q)):
        if not vis[r].any():
            continue
        x, vv = s[r][vis[r]], v[vis[r]]
        p = np.exp(x - x.max())
        p /= p.sum()
        out[r] = p @ vv
        d = 128 * 2.0 ** -24 * (np.abs(q[r]) @ np.abs(k[vis[r]]).T).max() * scale + 2.0 ** -18
        e = 2.0 ** -11 + d
        tiny = 2.0 ** -25 * len(x) * np.abs(vv).max()  # weights that round as subnormals
        bound[r] = (1.05 * 2 * e * (p @ np.abs(vv - out[r])) + 2 * len(x) * 2.0 ** -24 * (p @ np.abs(vv))
                    + tiny + 2.0 ** -11 * np.abs(out[r]) + 2.0 ** -25)
    return out, bound
