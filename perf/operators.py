"""Timed cases of the operators of a paged KV cache: what a program that serves
many transcriptions from one pool of pages has it do, once a step and once a
layer, through the public entry points of `qasr_attn`.

A case is a dict of plain values.  `op` says which operator it is:

  plan    block tables, row maps and the attention schedule of one step, built
          on the GPU from the requests' lengths (`paged_plan`): once a step
  append  qk-norm + RoPE of new rows, K and V stored through the row map
          (`paged_append`): once a layer
  attn    attention of each request's new rows over its pages
          (`paged_attn`): once a layer

A batch is `singles` requests of one new row (decode) at contexts in
[lo, hi] and `chunks` requests of rows in [rows_lo, rows_hi] at contexts in
[start_lo, start_hi].  Heads, positions and contexts are those of bench.py and
the tests (16 q / 8 kv heads of 128, 420-row prompts, contexts of 400-2400 and
8192 keys, prompts of 150-450 rows).  With `layers` above one the framework's
calls are captured in a HIP graph, as bench.py runs its layers: one layer's
launch is shorter than a Python call, and a serving loop replays its step.
"""
import math
import os
import sys

import torch

own = False

NQH, NKVH, HD = 16, 8, 128
QDIM, KDIM = NQH * HD, NKVH * HD
TOT = QDIM + 2 * KDIM
EPS = 1e-6
THETA = 1e6
MAX_SEQ = 16384


def _case(name, op, layers=1, page=16, singles=0, lo=1, hi=1, chunks=0, rows_lo=1, rows_hi=1,
          start_lo=0, start_hi=0, done=0, short=False):
    return {"name": name, "op": op, "layers": layers, "page": page, "singles": singles, "lo": lo,
            "hi": hi, "chunks": chunks, "rows_lo": rows_lo, "rows_hi": rows_hi,
            "start_lo": start_lo, "start_hi": start_hi, "done": done, "short": short}


def listed():
    return [
        # A small server's token step: every request grows by one row.
        _case("plan 16 singles", "plan", singles=16, lo=400, hi=2400),
        # A busy server's step: decodes, continuations and admissions together,
        # some requests ending, more pages wanted than are free.
        _case("plan 256 mixed", "plan", singles=220, lo=64, hi=4000, chunks=20, rows_lo=5,
              rows_hi=450, start_hi=1500, done=16, short=True),
        # One live transcription's new token, all layers.
        _case("append 1 row", "append", layers=28, singles=1, lo=511, hi=511),
        # A batch job's admission: 16 prompts of 150-450 rows.
        _case("append 16 prompts", "append", page=64, chunks=16, rows_lo=150, rows_hi=450),
        # One live transcription, 512 keys, all layers: latency.
        _case("attn 1 single", "attn", layers=28, singles=1, lo=511, hi=511),
        # The headline decode workload on pages: 16 ragged contexts.
        _case("attn 16 singles ragged", "attn", layers=28, singles=16, lo=400, hi=2400),
        # One long recording.
        _case("attn 1 single long", "attn", layers=28, page=64, singles=1, lo=8192, hi=8192),
        # The prompt of 30 s of audio.
        _case("attn prompt 420", "attn", layers=28, page=32, chunks=1, rows_lo=420, rows_hi=420),
        # Streams that append a second or two of audio each.
        _case("attn 8 continuations", "attn", layers=8, chunks=8, rows_lo=7, rows_hi=45,
              start_lo=200, start_hi=1700),
        # Decodes and admissions of one step together.
        _case("attn mixed", "attn", layers=4, singles=24, lo=100, hi=2400, chunks=4, rows_lo=100,
              rows_hi=450, start_hi=600),
        # The last chunk of a long prompt prefilled in 512-row chunks.
        _case("attn 512 at 7680", "attn", layers=4, page=256, chunks=1, rows_lo=512, rows_hi=512,
              start_lo=7680, start_hi=7680),
        # Two long prompts in large chunks.
        _case("attn 2 x 2048 at 4096", "attn", page=128, chunks=2, rows_lo=2048, rows_hi=2048,
              start_lo=4096, start_hi=4096),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attn", "attn", "attn"])
    page = rng.choice([16, 32, 64, 128, 256])
    lo, rows_lo = _log_int(rng, 1, 1500), _log_int(rng, 1, 200)
    c = {"page": page, "lo": lo, "hi": _log_int(rng, lo, 4000), "rows_lo": rows_lo,
         "rows_hi": _log_int(rng, rows_lo, 450), "start_lo": rng.choice([0, rng.randint(1, 300)]),
         "start_hi": _log_int(rng, 300, 2000)}
    if op == "plan":
        c.update(singles=_log_int(rng, 1, 220), chunks=_log_int(rng, 1, 21) - 1,
                 done=rng.choice([0, rng.randint(1, 16)]), short=rng.random() < 0.3)
    elif op == "append":
        c.update(layers=rng.randint(1, 8), singles=_log_int(rng, 1, 64),
                 chunks=_log_int(rng, 1, 14) - 1)
    else:
        shape = rng.choice(["singles", "long", "chunk", "mixed"])
        if shape == "singles":
            c.update(layers=rng.randint(2, 12), singles=_log_int(rng, 1, 16))
        elif shape == "long":
            n = _log_int(rng, 2000, 15000)
            c.update(layers=rng.randint(1, 8), singles=rng.randint(1, 3), lo=n,
                     hi=min(16000, n + rng.randint(0, 3000)))
        elif shape == "chunk":
            rows, at = _log_int(rng, 2, 1024), rng.choice([0, _log_int(rng, 30, 7680)])
            c.update(layers=rng.randint(1, 2), chunks=1, rows_lo=rows, rows_hi=rows, start_lo=at,
                     start_hi=at)
        else:
            c.update(layers=rng.randint(1, 4), singles=_log_int(rng, 1, 24),
                     chunks=rng.randint(1, 6))
    case = _case("", op, **c)
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------

def _lengths(lo, hi, n, salt):
    """n lengths over [lo, hi], the same for every seed of a case (the work of
    a case is fixed), by a SplitMix64 walk."""
    state, out = (0x51A50000 + salt) & (2 ** 64 - 1), []
    for _ in range(n):
        state = (state + 0x9E3779B97F4A7C15) & (2 ** 64 - 1)
        z = state
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & (2 ** 64 - 1)
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & (2 ** 64 - 1)
        out.append(lo + (z ^ (z >> 31)) % (hi - lo + 1))
    return out


def _batch(case):
    """(rows in the cache, rows to append) of each request: chunks spread
    among the singles, then the requests that end (rows = -1)."""
    s = [(n, 1) for n in _lengths(case["lo"], case["hi"], case["singles"], 3)]
    c = list(zip(_lengths(case["start_lo"], case["start_hi"], case["chunks"], 41),
                 _lengths(case["rows_lo"], case["rows_hi"], case["chunks"], 23)))
    both = sorted([((i + 0.5) / len(s), x) for i, x in enumerate(s)] +
                  [((i + 0.4) / len(c), x) for i, x in enumerate(c)])
    d = [(n, -1) for n in _lengths(case["lo"], case["hi"], case["done"], 5)]
    return [x for _, x in both] + d


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, std=1.0, mean=0.0):
    return (torch.randn(shape, device="cuda", generator=g) * std + mean).half()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    """Everything a case's call takes, from the seed: lengths, a table of
    shuffled pages, the ring of free pages, cache contents and rows."""
    g, ps, layers = _gen(seed), case["page"], case["layers"]
    batch = _batch(case)
    n = len(batch)
    held = [-(-c // ps) for c, _ in batch]
    full = [-(-(c + max(r, 0)) // ps) for c, r in batch]
    grow = sum(full) - sum(held)
    free = grow * 2 // 3 if case["short"] else grow + 7
    pages = sum(held) + free + 5
    ids = torch.randperm(pages, device="cuda", generator=g).int()
    plan = case["op"] == "plan"
    width = max(full) + 3
    col = torch.arange(width, device="cuda")
    have = _i32(held if plan else full).long()
    at = have.cumsum(0) - have
    table = torch.where(col < have[:, None],
                        ids[(at[:, None] + col).clamp(max=pages - 1)], -1).int()
    used = sum(held if plan else full)
    rows = sum(max(r, 0) for _, r in batch)
    x = {"op": case["op"], "ps": ps, "layers": layers, "pages": pages, "table": table,
         "len": _i32([c for c, _ in batch]), "rows": _i32([r for _, r in batch]),
         "total": rows, "most_rows": max(r for _, r in batch),
         "most_keys": max(c + max(r, 0) for c, r in batch)}
    if plan:
        # The free ids stand in the ring from a seeded place on.
        head = int(seed) % pages
        ring = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        ring[(head + torch.arange(free, device="cuda")) % pages] = ids[used:used + free]
        x.update(ring=ring, cursor=_i32([head, free]))
        return x
    if case["op"] == "append":
        pool = torch.zeros((layers, pages, 2, NKVH, ps, HD), dtype=torch.float16, device="cuda")
        inv = THETA ** (-2.0 * torch.arange(HD // 2, dtype=torch.float64) / HD)
        ang = torch.arange(MAX_SEQ, dtype=torch.float64)[:, None] * inv.repeat(2)
        x.update(pool=pool, qkv=_normal(g, (layers, rows, TOT)),
                 gains=_normal(g, (layers, 2, HD), 0.1, 1.0),
                 cos=ang.cos().float().half().cuda(), sin=ang.sin().float().half().cuda())
    else:
        x.update(pool=_normal(g, (layers, pages, 2, NKVH, ps, HD)),
                 q=_normal(g, (layers, rows, QDIM), 1.5))
    return x


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        _bind(st, case)
    return st


# ---- the framework's calls ---------------------------------------------------

def _bind(st, case):
    """What a server keeps: a context, its pool of pages with the cached rows
    in it, a plan for its batch; and the graph that it replays."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                    "qwen3-asr-wgpu_amd"))
    import qasr_attn as q

    ctx = q.Context(NQH, NKVH, HD, st["layers"], EPS, MAX_SEQ, 0)
    pool = q.PagePool(ctx, st["pages"], st["ps"])
    plan = q.PagedPlan(ctx, pool, st["len"].numel(), max(st["total"], 1))
    st.update(q_=q, ctx=ctx, pages_=pool, plan=plan)
    if st["op"] == "plan":
        return
    pool.tensor().copy_(st["pool"])
    st["pool"] = pool.tensor()
    q.paged_plan(ctx, plan, st["len"], st["rows"], st["table"])
    st["out"] = torch.zeros((st["layers"], st["total"], QDIM), dtype=torch.float16, device="cuda")
    if st["op"] == "append":
        ctx.set_rope_tables(st["cos"].cpu().view(torch.uint16).numpy(),
                            st["sin"].cpu().view(torch.uint16).numpy())
    if st["layers"] > 1:
        _layers(st)  # argument checks and code loading, before the capture
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _layers(st)
        st["graph"] = graph


def _layers(st):
    q = st["q_"]
    for l in range(st["layers"]):
        if st["op"] == "append":
            q.paged_append(st["ctx"], st["plan"], l, st["qkv"][l], st["gains"][l, 0],
                           st["gains"][l, 1], st["out"][l])
        else:
            q.paged_attn(st["ctx"], st["plan"], l, st["table"], st["q"][l], st["out"][l])


def _run_own(st):
    if st["op"] == "plan":
        p = st["plan"]
        st["q_"].paged_plan(st["ctx"], p, st["len"], st["rows"], st["table"], st["ring"],
                            st["cursor"])
        n = st["len"].numel()
        return {"table": st["table"], "ring": st["ring"], "cursor": p.cursor,
                "status": p.status[:n], "lens": p.lens[:n], "row_start": p.row_start[:n + 1],
                "row_pos": p.row_pos, "row_slot": p.row_slot}
    if "graph" in st:
        st["graph"].replay()
    else:
        _layers(st)
    return [st["out"], st["pool"]] if st["op"] == "append" else st["out"]


# ---- the plain forms ---------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plain_plan, "append": _plain_append, "attn": _plain_attn}[state["op"]](state)


def _row_maps(st):
    """Per row: its request and position; a plain batch has no refused rows."""
    rows = st["rows"].clamp(min=0).long()
    end = rows.cumsum(0)
    r = torch.arange(st["total"], device="cuda")
    req = torch.searchsorted(end, r, right=True)
    pos = st["len"].long()[req] + r - (end - rows)[req]
    return req, pos, r - (end - rows)[req]


def _plain_plan(st):
    ps, pages, table, ring = st["ps"], st["pages"], st["table"], st["ring"]
    n, width = table.shape
    length, rows = st["len"].long(), st["rows"].long()
    head, free = st["cursor"].long()
    new = rows.clamp(min=0)
    row_end = new.cumsum(0)
    row_start = torch.cat([torch.zeros_like(row_end[:1]), row_end])
    end = length + new
    before, after = (length + ps - 1) // ps, (end + ps - 1) // ps
    status = torch.where((rows >= 0) & ((end > MAX_SEQ) | (after > width)
                                        | (row_end > max(st["total"], 1))), 2, 0)
    last = table.gather(1, (length // ps).clamp(max=width - 1)[:, None])[:, 0]
    torn = (new > 0) & (length % ps != 0) & ((last < 0) | (last >= pages))
    status = torch.where((status == 0) & torn, 1, status)
    need = torch.where((status == 0) & (rows >= 0), after - before, 0)
    total = need.cumsum(0)
    status = torch.where((status == 0) & (need > 0) & (total > free), 3, status)
    placed = (status == 0) & (rows >= 0)
    take = torch.where(placed, need, 0)
    # New pages from the ring, in request order.
    col = torch.arange(width, device="cuda")
    fresh = placed[:, None] & (col >= before[:, None]) & (col < after[:, None])
    k = (total - need)[:, None] + col - before[:, None]
    table.copy_(torch.where(fresh, ring[(head + k) % pages], table))
    # Pages of ended requests to the ring's end, in table order.
    gone = (rows == -1)[:, None] & (col < before[:, None]) & (table >= 0) & (table < pages)
    back = gone.reshape(-1).cumsum(0)
    where = torch.where(gone.reshape(-1), (head + free + back - 1) % pages, pages)
    wide = torch.cat([ring, ring[:1]])
    wide[where] = table.reshape(-1)
    ring.copy_(wide[:pages])
    cursor = torch.stack([(head + take.sum()) % pages, free - take.sum() + back[-1]]).int()
    req, pos, _ = _row_maps(st)
    good = placed[req]
    page = table.long()[req, (pos // ps).clamp(max=width - 1)]
    return {"table": table, "ring": ring, "cursor": cursor, "status": status.int(),
            "lens": torch.where(rows == -1, 0, torch.where(placed, end, length)).int(),
            "row_start": row_start.int(), "row_pos": torch.where(good, pos, -1).int(),
            "row_slot": torch.where(good, page * ps + pos % ps, -1).int()}


def _plain_append(st):
    req, pos, _ = _row_maps(st)
    ps, pool, (layers, rows) = st["ps"], st["pool"], st["qkv"].shape[:2]
    page, off = st["table"].long()[req, pos // ps], pos % ps
    x = st["qkv"].float().view(layers, rows, NQH + 2 * NKVH, HD)
    qk, v = x[:, :, :NQH + NKVH], x[:, :, NQH + NKVH:]
    gain = st["gains"].float().repeat_interleave(torch.tensor([NQH, NKVH], device="cuda"), 1,
                                                 output_size=NQH + NKVH)
    y = qk * (1.0 / torch.sqrt(qk.square().mean(-1, keepdim=True) + EPS)) * gain[:, None]
    c, s = st["cos"][pos].float()[:, None], st["sin"][pos].float()[:, None]
    turned = torch.cat([-y[..., HD // 2:], y[..., :HD // 2]], -1)
    y = (y * c + turned * s).half()
    pool[:, page, 0, :, off] = y[:, :, NQH:].transpose(0, 1)
    pool[:, page, 1, :, off] = v.half().transpose(0, 1)
    return [y[:, :, :NQH].reshape(layers, rows, QDIM), pool]


def _plain_attn(st):
    """The requests padded to the longest, every layer's scores whole."""
    req, pos, at = _row_maps(st)
    ps, n, m = st["ps"], st["len"].numel(), st["most_rows"]
    used = -(-st["most_keys"] // ps)
    table = st["table"][:, :used].long().clamp(min=0)
    last = torch.full((n, m), -1, dtype=torch.long, device="cuda")
    last[req, at] = pos
    hidden = torch.arange(used * ps, device="cuda") > last[:, :, None]
    hidden = hidden.repeat(1, 2, 1)[:, None]  # the two q heads of a kv head, one after the other
    out = []
    for pool, q in zip(st["pool"], st["q"]):
        k, v = (pool[table, i].float().transpose(1, 2).reshape(n, NKVH, used * ps, HD)
                for i in (0, 1))
        x = torch.zeros((n, m, NQH, HD), device="cuda")
        x[req, at] = q.float().view(-1, NQH, HD)
        x = x.view(n, m, NKVH, 2, HD).permute(0, 2, 3, 1, 4).reshape(n, NKVH, 2 * m, HD)
        s = torch.matmul(x, k.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(HD))
        s.masked_fill_(hidden, -math.inf)
        top = s.amax(-1, keepdim=True).clamp(min=-1e30)
        e = s.sub_(top).exp_()
        e = torch.matmul(e, v) / e.sum(-1, keepdim=True)
        e = e.view(n, NKVH, 2, m, HD).permute(0, 3, 1, 2, 4)
        out.append(e[req, at].reshape(-1, QDIM).half())
    return torch.stack(out)


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    batch, ps = _batch(case), case["page"]
    rows = sum(max(r, 0) for _, r in batch)
    if case["op"] == "plan":
        # lengths and rows in; status, lengths and row starts out; two words a
        # row; one ring word and one table word a page that changes hands.
        moved = sum(-(-(c + r) // ps) - -(-c // ps) if r >= 0 else -(-c // ps) for c, r in batch)
        return {"bytes": 4 * (5 * len(batch) + 2 * rows + 2 * moved),
                "flops": 10 * (len(batch) + rows + moved)}
    if case["op"] == "append":
        return {"bytes": case["layers"] * 2 * rows * 2 * TOT,
                "flops": case["layers"] * rows * (NQH + NKVH) * HD * 8}
    b = sum(2 * (2 * KDIM * (c + r) + 2 * r * QDIM) for c, r in batch)
    f = sum(4 * HD * NQH * (r * c + r * (r + 1) // 2) for c, r in batch)
    return {"bytes": case["layers"] * b, "flops": case["layers"] * f}


# ---- the same results in 64 bits ---------------------------------------------

def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "plan":
        return None  # whole numbers alone
    batch, ps = _batch(case), case["page"]
    table = x["table"].tolist()
    if case["op"] == "append":
        pool = x["pool"].double()
        page = _i32([table[i][p // ps] for i, (c, r) in enumerate(batch)
                     for p in range(c, c + r)]).long()
        pos = _i32([p for c, r in batch for p in range(c, c + r)]).long()
        ang = pos.double()[:, None] * THETA ** (
            -torch.arange(0, HD, 2, dtype=torch.float64, device="cuda") / HD)
        c, s = (t.float().half().double() for t in (ang.cos(), ang.sin()))
        out = []
        for l in range(case["layers"]):
            h = x["qkv"][l].double().view(len(pos), -1, HD)
            roped = []
            for a, b, i in ((0, NQH, 0), (NQH, NQH + NKVH, 1)):
                z = h[:, a:b]
                z = z * (z.square().sum(-1, keepdim=True) / HD + EPS) ** -0.5
                z = z * x["gains"][l, i].double()
                u, w = z.split(HD // 2, -1)
                roped.append(torch.cat([u * c[:, None] - w * s[:, None],
                                        w * c[:, None] + u * s[:, None]], -1))
            out.append(roped[0].reshape(len(pos), QDIM))
            pool[l, page, 0, :, pos % ps] = roped[1]
            pool[l, page, 1, :, pos % ps] = h[:, NQH + NKVH:]
        return [torch.stack(out), pool]
    out = torch.empty((case["layers"], x["total"], QDIM), dtype=torch.float64, device="cuda")
    for l in range(case["layers"]):
        r0 = 0
        for i, (c, r) in enumerate(batch):
            ids = torch.tensor(table[i][:-(-(c + r) // ps)], device="cuda")
            kv = x["pool"][l, ids].double().permute(1, 2, 0, 3, 4).reshape(2, NKVH, -1, HD)
            k, v = kv[:, :, :c + r].repeat_interleave(2, 1)
            seen = torch.ones((r, c + r), dtype=torch.bool, device="cuda").tril(c)
            q = x["q"][l, r0:r0 + r].double().view(r, NQH, HD).transpose(0, 1)
            for h in range(0, NQH, 4):
                s = torch.matmul(q[h:h + 4], k[h:h + 4].mT.contiguous()) * HD ** -0.5
                p = torch.softmax(torch.where(seen, s, -math.inf), -1)
                out[l, r0:r0 + r].view(r, NQH, HD)[:, h:h + 4] = torch.matmul(
                    p, v[h:h + 4]).transpose(0, 1)
            r0 += r
    return out
