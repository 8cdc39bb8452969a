"""Timed cases of the operators with which a program that serves transcriptions
from one pool of pages keeps them in 8 bits and searches them with beams,
through the public entry points of `qasr_attn`.

A case is a dict of plain values.  `op` says which operator it is:

  append  qk-norm + RoPE of new rows, K and V stored in e4m3 with one power of
          two for each block of 16 rows and head (`paged_append`): once a layer
  attn    attention of each request's new rows over such pages
          (`paged_attn`): once a layer
  beam    the best continuations of each group of beams: log-softmax over the
          vocabulary, selection over beams and tokens (`beam_select`): once a
          step
  fork    the requests of a step go on as their parents: tables follow, pages
          are shared, the last, unfinished ones copied, those that nobody
          holds any more given back (`paged_fork`): once a step

A batch of append and attn is `singles` requests of one new row (decode) at
contexts in [lo, hi] and `chunks` requests of rows in [rows_lo, rows_hi] at
contexts in [start_lo, start_hi].  beam and fork take `groups` x `width` beams;
fork's hold [lo, hi] rows, of which the last `own` to 2 `own` are no longer
those of the group's other beams.  Heads, contexts and the vocabulary are those
of bench.py and the tests (16 q / 8 kv heads of 128, 420-row prompts, contexts
of 400-2400 and 8192 keys, prompts of 150-450 rows, 151936 tokens).  With
`layers` above one the framework's layer calls are captured in a HIP graph, as
bench.py runs its layers: a serving loop replays its step.
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
BLOCK = 16  # rows of a scale
VOCAB = 151936
EOS = 151645


def _case(name, op, layers=1, page=16, singles=0, lo=1, hi=1, chunks=0, rows_lo=1, rows_hi=1,
          start_lo=0, start_hi=0, groups=0, width=0, k=0, vocab=0, done=0, own=0, f8=True):
    return {"name": name, "op": op, "layers": layers, "page": page, "singles": singles, "lo": lo,
            "hi": hi, "chunks": chunks, "rows_lo": rows_lo, "rows_hi": rows_hi,
            "start_lo": start_lo, "start_hi": start_hi, "groups": groups, "width": width, "k": k,
            "vocab": vocab, "done": done, "own": own, "f8": f8}


def listed():
    return [
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
        # The last chunk of a long prompt prefilled in 512-row chunks.
        _case("attn 512 at 7680", "attn", layers=4, page=256, chunks=1, rows_lo=512, rows_hi=512,
              start_lo=7680, start_hi=7680),
        # One transcription searched with 5 beams.
        _case("beam 1 x 5", "beam", groups=1, width=5, k=5, vocab=VOCAB),
        # 16 of them, twice as many candidates as beams (a caller that puts
        # ended ones aside itself).
        _case("beam 16 x 5 of 10", "beam", groups=16, width=5, k=10, vocab=VOCAB),
        # A large batch in which some beams have ended.
        _case("beam 64 x 4", "beam", groups=64, width=4, k=4, vocab=VOCAB, done=40),
        # The step's reordering of one transcription's beams, f16 pages.
        _case("fork 1 x 5", "fork", layers=28, groups=1, width=5, lo=523, hi=523, own=12, f8=False),
        # Of 16 transcriptions of different lengths.
        _case("fork 16 x 5", "fork", layers=28, groups=16, width=5, lo=400, hi=1500, own=40),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "beam", "beam", "fork"])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "beam":
        groups, width = _log_int(rng, 1, 32), rng.randint(1, 8)
        k = rng.choice([width, 2 * width])
        c = {"groups": groups, "width": width, "k": k,
             "vocab": rng.choice([VOCAB, _log_int(rng, 40, VOCAB)]),
             "done": rng.choice([0, rng.randint(0, groups * width)])}
    elif op == "fork":
        lo = _log_int(rng, 20, 800)
        c = {"layers": rng.randint(1, 28), "page": page, "groups": _log_int(rng, 1, 16),
             "width": rng.randint(2, 5), "lo": lo, "hi": _log_int(rng, lo, 1500),
             "own": _log_int(rng, 1, 40), "f8": rng.random() < 0.7}
    else:
        lo, rows_lo = _log_int(rng, 1, 1500), _log_int(rng, 1, 200)
        c = {"page": page, "lo": lo, "hi": _log_int(rng, lo, 4000), "rows_lo": rows_lo,
             "rows_hi": _log_int(rng, rows_lo, 450), "start_lo": rng.choice([0, rng.randint(1, 300)]),
             "start_hi": _log_int(rng, 300, 2000)}
        if op == "append":
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
                c.update(layers=rng.randint(1, 2), chunks=1, rows_lo=rows, rows_hi=rows,
                         start_lo=at, start_hi=at)
            else:
                c.update(layers=rng.randint(1, 4), singles=_log_int(rng, 1, 24),
                         chunks=rng.randint(1, 6))
    case = _case("", op, **c)
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------

def _walk(n, salt):
    """n numbers of a SplitMix64 walk: what a case's work depends on is the
    same for every seed."""
    state, out = (0x51A50000 + salt) & (2 ** 64 - 1), []
    for _ in range(n):
        state = (state + 0x9E3779B97F4A7C15) & (2 ** 64 - 1)
        z = state
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & (2 ** 64 - 1)
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & (2 ** 64 - 1)
        out.append(z ^ (z >> 31))
    return out


def _lengths(lo, hi, n, salt):
    return [lo + z % (hi - lo + 1) for z in _walk(n, salt)]


def _batch(case):
    """(rows in the cache, rows to append) of each request: chunks spread among
    the singles."""
    s = [(n, 1) for n in _lengths(case["lo"], case["hi"], case["singles"], 3)]
    c = list(zip(_lengths(case["start_lo"], case["start_hi"], case["chunks"], 41),
                 _lengths(case["rows_lo"], case["rows_hi"], case["chunks"], 23)))
    both = sorted([((i + 0.5) / len(s), x) for i, x in enumerate(s)] +
                  [((i + 0.4) / len(c), x) for i, x in enumerate(c)])
    return [x for _, x in both]


def _beams(case):
    """Per beam: (rows in the cache, rows that the group's beams share, beam it
    goes on from).  Every beam of a group goes on from one of its better half
    more often than not; in every seventh group one has no successor at all."""
    g, w = case["groups"], case["width"]
    lens = _lengths(case["lo"], case["hi"], g, 7)
    apart = [min(n, a) for n, a in zip(lens, _lengths(case["own"], 2 * case["own"], g, 11))]
    z = _walk(g * w, 13)
    out = []
    for i in range(g * w):
        a, b = z[i] % w, (z[i] >> 20) % w
        p = -1 if i // w % 7 == 6 and i % w == w - 1 else i // w * w + min(a, b)
        out.append((lens[i // w], lens[i // w] - apart[i // w], p))
    return out


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, std=1.0, mean=0.0):
    return (torch.randn(shape, device="cuda", generator=g) * std + mean).half()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pages(g, layers, pages, ps, f8):
    """Filled pages; with f8 the values of 16-row blocks in e4m3 and their
    scales, of several sizes (a head's keys and values are not all of one)."""
    shape = (layers, pages, 2, NKVH, ps, HD)
    if not f8:
        return _normal(g, shape), None
    e = torch.randint(-10, -6, shape[:4] + (ps // BLOCK,), device="cuda", generator=g)
    x = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    for l in range(layers):
        x[l] = (torch.randn(shape[1:], device="cuda", generator=g) * 100).clamp_(-440, 440)
    return x, _e8m0(e)


def _e8m0(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _inputs(case, seed):
    """Everything a case's call takes, from the seed."""
    make = {"beam": _beam_inputs, "fork": _fork_inputs}.get(case["op"], _step_inputs)
    return {"op": case["op"], **make(case, _gen(seed))}


def _step_inputs(case, g):
    ps, layers = case["page"], case["layers"]
    batch = _batch(case)
    full = [-(-(c + r) // ps) for c, r in batch]
    pages, width = sum(full) + 5, max(full) + 3
    ids = torch.randperm(pages, device="cuda", generator=g).int()
    col, have = torch.arange(width, device="cuda"), _i32(full).long()
    at = have.cumsum(0) - have
    table = torch.where(col < have[:, None], ids[(at[:, None] + col).clamp(max=pages - 1)], -1)
    rows = sum(r for _, r in batch)
    pool, scales = _pages(g, layers, pages, ps, True)
    x = {"ps": ps, "layers": layers, "pages": pages, "table": table.int(), "pool": pool,
         "scales": scales, "len": _i32([c for c, _ in batch]), "rows": _i32([r for _, r in batch]),
         "total": rows, "most_rows": max(r for _, r in batch),
         "most_keys": max(c + r for c, r in batch)}
    if case["op"] == "append":
        inv = THETA ** (-2.0 * torch.arange(HD // 2, dtype=torch.float64) / HD)
        ang = torch.arange(MAX_SEQ, dtype=torch.float64)[:, None] * inv.repeat(2)
        x.update(qkv=_normal(g, (layers, rows, TOT)), gains=_normal(g, (layers, 2, HD), 0.1, 1.0),
                 cos=ang.cos().float().half().cuda(), sin=ang.sin().float().half().cuda())
    else:
        x.update(q=_normal(g, (layers, rows, QDIM), 1.5))
    return x


def _beam_inputs(case, g):
    """Logits whose best few stand out, as a decoder's do, and scores of beams
    some steps on; every fifth group is at its first step, with one beam."""
    groups, w, v = case["groups"], case["width"], case["vocab"]
    logits = torch.randn((groups * w, v), device="cuda", generator=g) * 2.0
    best = torch.randint(0, v, (groups * w, 8), device="cuda", generator=g)
    logits.scatter_add_(1, best, torch.rand((groups * w, 8), device="cuda", generator=g) * 9.0)
    scores = -10.0 * torch.rand((groups, w), device="cuda", generator=g)
    scores[4::5, 1:] = -math.inf
    ended = torch.rand(groups * w, device="cuda", generator=g).argsort()[:case["done"]]
    done = torch.zeros(groups * w, dtype=torch.int32, device="cuda")
    done[ended] = 1
    return {"groups": groups, "width": w, "k": case["k"], "vocab": v, "logits": logits,
            "scores": scores.view(-1), "done": done, "eos": min(EOS, v - 1)}


def _fork_inputs(case, g):
    """Beams whose first pages, whole ones, are the group's; tables of shuffled
    pages, the free ones in a ring."""
    ps, w = case["page"], case["width"]
    beams = _beams(case)
    n, groups = len(beams), case["groups"]
    both = [s // ps for _, s, _ in beams]
    full = [-(-c // ps) for c, _, _ in beams]
    prefix = sum(both[::w])
    used = prefix + sum(f - b for f, b in zip(full, both))
    pages, width = used + n + 3, max(full) + 2
    ids = torch.randperm(pages, device="cuda", generator=g).int()
    col = torch.arange(width, device="cuda")
    b, f = _i32(both).long()[:, None], _i32(full).long()[:, None]
    pre = b[::w].cumsum(0) - b[::w]
    apart = (f - b).cumsum(0) - (f - b) + prefix
    at = torch.where(col < b, pre.repeat_interleave(w, 0) + col, apart + col - b)
    table = torch.where(col < f, ids[at.clamp(max=pages - 1)], -1).int()
    shared = torch.zeros(pages, dtype=torch.int32, device="cuda")
    shared[ids[:prefix].long()] = w - 1
    head = int(ids[0])  # the free ids stand in the ring from a seeded place on
    ring = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    ring[(head + torch.arange(pages - used, device="cuda")) % pages] = ids[used:]
    pool, scales = _pages(g, case["layers"], pages, ps, case["f8"])
    return {"ps": ps, "layers": case["layers"], "pages": pages, "f8": case["f8"], "pool": pool,
            "scales": scales, "table": table, "shared": shared, "ring": ring,
            "cursor": _i32([head, pages - used]), "len": _i32([c for c, _, _ in beams]),
            "parent": _i32([p for _, _, p in beams])}


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        _bind(st)
    return st


# ---- the framework's calls ---------------------------------------------------

def _bind(st):
    """What a server keeps: a context, its pool of pages with the cached rows
    in it, a plan for its batch, a fork's or a selection's workspace; and the
    graph of layers that it replays."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                    "qwen3-asr-wgpu_amd"))
    import qasr_attn as q

    ctx = q.Context(NQH, NKVH, HD, st.get("layers", 1), EPS, MAX_SEQ, 0)
    st.update(q_=q, ctx=ctx)
    if st["op"] == "beam":
        st["sel"] = q.BeamSelect(ctx, st["groups"], st["width"], st["vocab"], st["k"])
        n = st["groups"] * st["k"]
        st.update(parent=torch.empty(n, dtype=torch.int32, device="cuda"),
                  token=torch.empty(n, dtype=torch.int32, device="cuda"),
                  out_done=torch.empty(n, dtype=torch.int32, device="cuda"),
                  out_scores=torch.empty(n, device="cuda"))
        return
    f8 = st["scales"] is not None
    pool = q.PagePool(ctx, st["pages"], st["ps"], "e4m3" if f8 else "f16")
    pool.tensor().copy_(st["pool"])
    st.update(pages_=pool, pool=pool.tensor())
    if f8:
        pool.scales().view(torch.uint8).copy_(st["scales"].view(torch.uint8))
        st["scales"] = pool.scales()
    if st["op"] == "fork":
        st["fork"] = q.PagedFork(ctx, pool, *st["table"].shape)
        return
    plan = q.PagedPlan(ctx, pool, st["len"].numel(), st["total"])
    st["plan"] = plan
    q.paged_plan(ctx, plan, st["len"], st["rows"], st["table"])
    st["out"] = torch.zeros((st["layers"], st["total"], QDIM), dtype=torch.float16, device="cuda")
    if st["op"] == "append":
        ctx.set_rope_tables(st["cos"].cpu().view(torch.uint16).numpy(),
                            st["sin"].cpu().view(torch.uint16).numpy())
    if st["layers"] > 1:
        keep = pool.tensor().clone(), pool.scales().view(torch.uint8).clone()
        _layers(st)  # argument checks and code loading, before the capture
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _layers(st)
        pool.tensor().copy_(keep[0])
        pool.scales().view(torch.uint8).copy_(keep[1])
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
    if st["op"] == "beam":
        st["q_"].beam_select(st["ctx"], st["sel"], st["logits"], st["scores"], st["parent"],
                             st["token"], st["out_scores"], st["done"], st["eos"], st["out_done"])
        return {"parent": st["parent"], "token": st["token"], "scores": st["out_scores"],
                "done": st["out_done"]}
    if st["op"] == "fork":
        st["q_"].paged_fork(st["ctx"], st["fork"], st["len"], st["parent"], st["table"],
                            st["shared"], st["ring"], st["cursor"])
        return _forked(st)
    if "graph" in st:
        st["graph"].replay()
    else:
        _layers(st)
    return [st["out"], st["pool"], st["scales"]] if st["op"] == "append" else st["out"]


def _forked(st):
    return {x: st[x] for x in ("table", "len", "shared", "ring", "cursor", "pool", "scales")}


# ---- the plain forms ---------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attn": _plain_attn, "beam": _plain_beam,
            "fork": _plain_fork}[state["op"]](state)


def _row_maps(st):
    """Per row: its request, its position, its place among the request's."""
    rows = st["rows"].long()
    end = rows.cumsum(0)
    r = torch.arange(st["total"], device="cuda")
    req = torch.searchsorted(end, r, right=True)
    at = r - (end - rows)[req]
    return req, st["len"].long()[req] + at, at


def _scale_of(amax):
    """The smallest power of two, 2^-15 at least, that amax is at most 448 of."""
    m, e = torch.frexp(amax / 448.0)
    return torch.where(m > 0.5, e, e - 1).clamp(min=-15)


def _two(e):
    """2^e, exactly."""
    return ((e + 127) << 23).int().view(torch.float32)


def _to_e4m3(x, e):
    """x / 2^e in e4m3.  At the largest scale what would round past the largest
    f16 stays below it."""
    y = x * _two(-e)
    y = torch.where(e >= 8, y.clamp(-240.0, 240.0), y)
    return torch.where(torch.isfinite(y), y, math.nan).to(torch.float8_e4m3fn)


def _plain_append(st):
    req, pos, _ = _row_maps(st)
    ps, pool, (layers, rows) = st["ps"], st["pool"], st["qkv"].shape[:2]
    x = st["qkv"].float().view(layers, rows, NQH + 2 * NKVH, HD)
    qk, v = x[:, :, :NQH + NKVH], x[:, :, NQH + NKVH:]
    gain = st["gains"].float().repeat_interleave(torch.tensor([NQH, NKVH], device="cuda"), 1,
                                                 output_size=NQH + NKVH)
    y = qk * (1.0 / torch.sqrt(qk.square().mean(-1, keepdim=True) + EPS)) * gain[:, None]
    c, s = st["cos"][pos].float()[:, None], st["sin"][pos].float()[:, None]
    turned = torch.cat([-y[..., HD // 2:], y[..., :HD // 2]], -1)
    y = (y * c + turned * s).half()
    # The 16-row blocks that the rows fall into, with what they hold.
    page, off = st["table"].long()[req, pos // ps], pos % ps
    at, inv = torch.unique(page * (ps // BLOCK) + off // BLOCK, return_inverse=True)
    old = pool.view(layers, -1, 2, NKVH, ps // BLOCK, BLOCK, HD)
    p, b = at // (ps // BLOCK), at % (ps // BLOCK)
    e0 = st["scales"].view(torch.uint8)[:, p, :, :, b].int().permute(1, 0, 2, 3) - 127
    cur = old[:, p, :, :, b].float().permute(1, 0, 2, 3, 4, 5)  # layer, block, kv, head, row, dim
    new = torch.stack([y[:, :, NQH:], v.half()], 2).float()     # layer, row, kv, head, dim
    amax = torch.where(torch.isfinite(new), new.abs(), 0.0).amax(-1)
    most = torch.zeros((layers, len(at), 2, NKVH), device="cuda").index_reduce_(
        1, inv, amax, "amax")
    first = torch.full((len(at),), BLOCK, device="cuda").scatter_reduce_(
        0, inv, off % BLOCK, "amin")[:, None, None]
    e = _scale_of(most)
    e = torch.where(first > 0, torch.maximum(e, e0), e)
    kept = (cur * _two(e0 - e)[..., None, None]).to(torch.float8_e4m3fn)
    row = torch.arange(BLOCK, device="cuda")[:, None]
    kept = torch.where(row < first[..., None, None], kept.float(), cur)
    kept[:, inv, :, :, off % BLOCK] = _to_e4m3(new, e[:, inv][..., None]).float().transpose(0, 1)
    old[:, p, :, :, b] = kept.permute(1, 0, 2, 3, 4, 5).to(torch.float8_e4m3fn)
    st["scales"].view(torch.uint8)[:, p, :, :, b] = (e.permute(1, 0, 2, 3) + 127).to(torch.uint8)
    return [y[:, :, :NQH].reshape(layers, rows, QDIM), pool, st["scales"]]


def _values(pool, scales):
    """What e4m3 pages stand for, in f32."""
    b = pool.float().view(*scales.shape, BLOCK, HD)
    return (b * _two(scales.view(torch.uint8).int() - 127)[..., None, None]).flatten(-3, -2)


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
    for pool, scales, q in zip(st["pool"], st["scales"], st["q"]):
        k, v = (_values(pool[table, i], scales[table, i]).transpose(1, 2).reshape(
            n, NKVH, used * ps, HD) for i in (0, 1))
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


def _plain_beam(st):
    """Scores next to each other decide the order: in 64 bits."""
    g, w, v, k, eos = st["groups"], st["width"], st["vocab"], st["k"], st["eos"]
    x = st["logits"].double()
    top = x.amax(-1, keepdim=True)
    p = x - top - (x - top).exp_().sum(-1, keepdim=True).log_()
    ended = (st["done"] != 0)[:, None]
    at_end = torch.arange(v, device="cuda") == eos
    p = torch.where(ended, torch.where(at_end, 0.0, -math.inf), p)
    p = (p + st["scores"].double()[:, None]).view(g, w * v)
    # (Equal scores, next to none here, go to the lowest place.)
    best, at = torch.sort(p, -1, descending=True, stable=True) if w * v <= 4096 else p.topk(min(k, w * v))
    best, at = best[:, :k], at[:, :k]
    some = best > -math.inf
    row = at // v + torch.arange(0, g * w, w, device="cuda")[:, None]
    token = at % v
    done = some & ((st["done"][row] != 0) | (token == eos))
    res = {"parent": torch.where(some, row, -1).int(), "token": torch.where(some, token, -1).int(),
           "scores": best.float(), "done": done.int()}
    return {name: x.reshape(-1) for name, x in res.items()}


def _plain_fork(st):
    ps, pages, table, ring, shared = st["ps"], st["pages"], st["table"], st["ring"], st["shared"]
    n, width = table.shape
    length, parent = st["len"].long(), st["parent"].long()
    head, free = st["cursor"].long()
    i, col = torch.arange(n, device="cuda"), torch.arange(width, device="cuda")
    live, src = parent >= 0, parent.clamp(min=0)
    dest = torch.where(live, parent, n)
    sons = torch.bincount(dest, minlength=n + 1)[:n]
    # A request's unfinished page stays with itself, or the first that goes on
    # from it, if no other request holds it; the others get copies.
    heir = torch.full((n + 1,), n, device="cuda").scatter_reduce_(
        0, dest, torch.where(parent == i, -1, i), "amin")[:n]
    heir = torch.where(heir < 0, i, heir)
    whole, rest = length // ps, length % ps
    last = table.gather(1, whole.clamp(max=width - 1)[:, None])[:, 0].long()
    alone = (rest > 0) & (shared[last.clamp(min=0)] == 0)
    copy = live & (rest[src] > 0) & ~((heir[src] == i) & alone[src])
    rank = copy.cumsum(0) - copy.long()
    fresh = ring[(head + rank) % pages]
    # How many more requests hold each page.
    more = torch.where(col < whole[:, None], (sons - 1)[:, None],
                       torch.where((col == whole[:, None]) & (rest > 0)[:, None],
                                   ((sons > 0) & alone).long()[:, None] - 1, 0))
    at = table.long().clamp(min=0)
    shared.index_add_(0, at.reshape(-1), more.reshape(-1).int())
    # Those that none holds any more, by their place, then by their request.
    order = (col * n)[None] + i[:, None]
    gone = (more < 0) & (shared[at] < 0)
    first = torch.full((pages,), n * width, device="cuda").scatter_reduce_(
        0, at.reshape(-1), torch.where(gone, order, n * width).reshape(-1), "amin")
    back = (gone & (first[at] == order)).t().reshape(-1)
    k = back.cumsum(0)
    wide = torch.cat([ring, ring[:1]])
    wide[torch.where(back, (head + free + k - 1) % pages, pages)] = table.t().reshape(-1)
    shared.clamp_(min=0)
    # Tables, copies, lengths.
    used = live[:, None] & (col < ((length + ps - 1) // ps)[src][:, None])
    new = torch.where(used, table[src], table)
    new = torch.where(copy[:, None] & (col == whole[src][:, None]), fresh[:, None], new)
    to = copy.nonzero()[:, 0]
    a, b, r = last[src[to]], fresh[to].long(), rest[src[to]]
    row = torch.arange(ps, device="cuda") < r[:, None]
    bits = st["pool"].view(torch.uint8 if st["f8"] else torch.int16)
    bits[:, b] = torch.where(row[:, None, None, :, None], bits[:, a], bits[:, b])
    if st["f8"]:
        held = torch.arange(0, ps, BLOCK, device="cuda") < r[:, None]
        bits = st["scales"].view(torch.uint8)
        bits[:, b] = torch.where(held[:, None, None], bits[:, a], bits[:, b])
    table.copy_(new)
    ring.copy_(wide[:pages])
    st["len"].copy_(torch.where(live, length[src], 0))
    st["cursor"].copy_(torch.stack([(head + copy.sum()) % pages, free - copy.sum() + k[-1]]))
    return _forked(st)


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    ps, layers = case["page"], case["layers"]
    if case["op"] == "beam":
        rows = case["groups"] * case["width"]
        return {"bytes": 4 * rows * case["vocab"] + 8 * rows + 16 * case["groups"] * case["k"],
                "flops": 4 * rows * case["vocab"]}
    if case["op"] == "fork":
        # Table entries in and out; unfinished pages' rows read and written.
        beams = _beams(case)
        taken, copied = set(), 0
        for i, (c, _, p) in sorted(enumerate(beams), key=lambda x: x[0] != x[1][2]):
            if p >= 0:
                copied += (c % ps) * (p in taken)
                taken.add(p)
        item = 2 * KDIM * (1 if case["f8"] else 2)
        entries = sum(-(-c // ps) for c, _, _ in beams)
        return {"bytes": 2 * copied * layers * item + 8 * entries + 12 * len(beams),
                "flops": 2 * entries}
    batch = _batch(case)
    rows = sum(r for _, r in batch)
    if case["op"] == "append":
        return {"bytes": layers * rows * (2 * TOT + 2 * QDIM + 2 * KDIM),
                "flops": layers * rows * (NQH + NKVH) * HD * 8}
    b = sum(2 * KDIM * (c + r) + 4 * r * QDIM for c, r in batch)
    f = sum(4 * HD * NQH * (r * c + r * (r + 1) // 2) for c, r in batch)
    return {"bytes": layers * b, "flops": layers * f}


# ---- the same results in 64 bits ---------------------------------------------

def exact(case, seed):
    if case["op"] == "fork":
        return None  # whole numbers, and values that only move
    return {"append": _exact_append, "attn": _exact_attn, "beam": _exact_beam}[case["op"]](
        case, _inputs(case, seed))


def _exact_append(case, x):
    """Request by request, block by block."""
    batch, ps = _batch(case), case["page"]
    table = x["table"].tolist()
    pool, scales = x["pool"].double(), x["scales"].double()
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
        kv = torch.stack([roped[1].float().half().double(), h[:, NQH + NKVH:]], 1)
        r0 = 0
        for i, (n, r) in enumerate(batch):
            at = n
            while at < n + r:
                to = min(n + r, at // BLOCK * BLOCK + BLOCK)
                page, row, blk = table[i][at // ps], at % ps, at % ps // BLOCK
                new = kv[r0 + at - n:r0 + to - n].permute(1, 2, 0, 3)  # kv, head, row, dim
                top = new.abs().amax((2, 3))
                e = torch.ceil(torch.log2(top.clamp(min=1e-30) / 448.0)).clamp(min=-15.0)
                unit = 2.0 ** e
                if at % BLOCK:
                    unit = torch.maximum(unit, scales[l, page, :, :, blk])
                    z = slice(row // BLOCK * BLOCK, row)
                    pool[l, page, :, :, z] = _nearest(
                        pool[l, page, :, :, z] * (scales[l, page, :, :, blk] / unit)[..., None, None])
                q = _nearest(new / unit[..., None, None])
                top = torch.where(unit >= 256.0, 240.0, 448.0)[..., None, None]
                pool[l, page, :, :, row:row + to - at] = torch.minimum(torch.maximum(q, -top), top)
                scales[l, page, :, :, blk] = unit
                at = to
            r0 += r
    return [torch.stack(out), pool, scales]


def _nearest(x):
    """The nearest of e4m3's numbers, ties to even: 4 significant bits, steps of
    2^-9 at least."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return torch.round(x / step) * step


def _exact_attn(case, x):
    batch, ps = _batch(case), case["page"]
    table = x["table"].tolist()
    out = torch.empty((case["layers"], x["total"], QDIM), dtype=torch.float64, device="cuda")
    for l in range(case["layers"]):
        r0 = 0
        for i, (c, r) in enumerate(batch):
            ids = torch.tensor(table[i][:-(-(c + r) // ps)], device="cuda")
            unit = x["scales"][l, ids].double().repeat_interleave(BLOCK, -1)
            kv = x["pool"][l, ids].double() * unit[..., None]
            kv = kv.permute(1, 2, 0, 3, 4).reshape(2, NKVH, -1, HD)
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


def _exact_beam(case, x):
    """The scores; the beams and tokens that they belong to are whole numbers."""
    g, w, k = case["groups"], case["width"], case["k"]
    p = torch.log_softmax(x["logits"].double(), -1)
    p[x["done"] != 0] = -math.inf
    p[x["done"] != 0, x["eos"]] = 0.0
    p += x["scores"].double()[:, None]
    best = p.view(g, -1).sort(-1, descending=True)[0][:, :k]
    return {"parent": None, "token": None, "scores": best.reshape(-1), "done": None}
