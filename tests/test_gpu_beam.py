"""Beam selection on the GPU against a plain one in 64 bits."""
from __future__ import annotations

import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import beam_model as B  # noqa: E402
import qasr_attn as Q  # noqa: E402
from gpu_helpers import say  # noqa: E402

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


class Sel:
    def __init__(self, groups, width, vocab, k):
        self.ctx = Q.Context(layers=1)
        self.sel = Q.BeamSelect(self.ctx, groups, width, vocab, k)

    def run(self, logits, scores, done=None, eos=-1):
        n = logits.shape[0] // self.sel.width * self.sel.k
        out = [torch.full((n + 1,), 77, dtype=t, device="cuda") for t in (torch.int32, torch.int32, torch.float32, torch.int32)]
        Q.beam_select(self.ctx, self.sel, logits, scores, *out[:3], done, eos, out[3])
        torch.cuda.synchronize()
        assert all(float(t[n]) == 77 for t in out), "places behind the last are left as they were"
        return [t[:n].cpu() for t in out]

    def close(self):
        torch.cuda.synchronize()
        self.sel.close()
        self.ctx.close()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def peaked(seed, rows, vocab, std=2.0):
    g = gen(seed)
    x = torch.randn((rows, vocab), device="cuda", generator=g) * std
    n = min(8, vocab)
    at = torch.randint(0, vocab, (rows, n), device="cuda", generator=g)
    return x.scatter_add_(1, at, torch.rand((rows, n), device="cuda", generator=g) * 9)


def score_bound(vocab, top):
    """How far a score may be from the exact one.  The exponent of a term is
    rounded twice and scaled (3 * 2^-24 of it; terms with exponents past 40
    weigh nothing at this size of vocabulary), exp2 is off by 2^-22, sums of a
    lane's up to 32 terms and of 64 lanes and 8 waves by 2^-24 each addition:
    relative to the sum, so absolute in its logarithm.  Then one rounding of the
    score to f32."""
    terms = 40 * 3 * 2.0 ** -24 + 2.0 ** -22 + (32 + 6 + 8) * 2.0 ** -24
    return terms + 2.0 ** -24 * abs(top)


def check(got, logits, scores, width, k, done=None, eos=-1):
    parent, token, score, ended = (t.numpy() for t in got)
    want = B.select(logits.cpu().numpy(), scores.cpu().numpy(), width, k,
                    None if done is None else done.cpu().numpy(), eos)
    for i, (r, t, s, d, gap) in enumerate(want):
        # Scores nearer to each other than the sums' error have no order.
        if gap <= 4 * score_bound(logits.shape[1], s) and gap > 0:
            continue
        if i % k and want[i - 1][4] <= 4 * score_bound(logits.shape[1], s) and want[i - 1][4] > 0:
            continue
        assert (parent[i], token[i], ended[i]) == (r, t, d), (i, want[i], parent[i], token[i], score[i])
        if r < 0:
            assert score[i] == -INF
        else:
            assert abs(score[i] - s) <= score_bound(logits.shape[1], s), (i, s, score[i])


@pytest.mark.parametrize("groups,width,vocab,k", [
    (1, 1, 1, 1), (2, 1, 3, 4), (1, 5, 151936, 5), (3, 4, 40, 8), (2, 3, 4095, 3), (2, 3, 4096, 16),
    (1, 2, 4097, 2), (5, 2, 151936, 4), (2, 8, 20011, 16), (1, 32, 5000, 32), (40, 4, 1000, 4),
    (1, 2, 262144, 5), (1, 2, 262145, 32), (1, 1, 600001, 32), (1, 2, 1 << 20, 7), (1024, 1, 100, 1)])
def test_select_against_64_bits(gpu, groups, width, vocab, k):
    say(f"beam {groups} x {width} of {vocab}, {k}")
    s = Sel(groups, width, vocab, k)
    logits = peaked(1, groups * width, vocab)
    scores = -10 * torch.rand(groups * width, device="cuda", generator=gen(2))
    check(s.run(logits, scores), logits, scores, width, k)
    s.close()


@pytest.mark.parametrize("vocab", [7, 4096, 151936])
def test_ended_and_dead_beams(gpu, vocab):
    """Groups with every mix of them; a NaN among the logits of ended or dead
    beams is nobody's."""
    groups, width, k = 24, 4, 6
    s = Sel(groups, width, vocab, k)
    rows, rnd = groups * width, random.Random(3)
    logits = peaked(1, rows, vocab)
    scores = -10 * torch.rand(rows, device="cuda", generator=gen(2))
    done = torch.zeros(rows, dtype=torch.int32, device="cuda")
    for r in range(rows):
        kind = rnd.choice(["", "", "ended", "-inf", "nan", "+inf"])
        if kind == "ended":
            done[r] = rnd.choice([1, -5, 1 << 31 - 1])
        elif kind:
            scores[r] = float(kind)
        if kind and rnd.random() < 0.5:
            logits[r, rnd.randrange(vocab)] = NAN
    check(s.run(logits, scores, done, vocab // 2), logits, scores, width, k, done, vocab // 2)
    check(s.run(logits, scores, done), logits, scores, width, k, done)
    s.close()


@pytest.mark.parametrize("vocab", [50, 9000])
def test_masked_tokens(gpu, vocab):
    """Tokens of -inf are none, down to rows with one or none left; a row with a
    NaN or +inf offers nothing."""
    groups, width, k = 6, 3, 7
    s = Sel(groups, width, vocab, k)
    logits = peaked(1, groups * width, vocab)
    scores = -torch.rand(groups * width, device="cuda", generator=gen(2))
    allowed = [vocab, 5, 1, 0, 2, 0, 0, 0, 0, 30, 40, 1]
    for r, n in enumerate(allowed):
        keep = torch.randperm(vocab, device="cuda", generator=gen(10 + r))[:n]
        row = torch.full((vocab,), -INF, device="cuda")
        row[keep] = logits[r, keep]
        logits[r] = row
    logits[12, vocab - 1] = INF
    logits[13, 0] = NAN
    logits[14, vocab // 2] = -NAN
    check(s.run(logits, scores), logits, scores, width, k)
    s.close()


@pytest.mark.parametrize("vocab,k", [(6000, 5), (151936, 16), (300000, 32)])
def test_equal_scores_go_to_the_lowest_place(gpu, vocab, k):
    """Rows of one value; the same row for several beams; ties between the first
    and the last token, and 0 with -0."""
    groups, width = 4, 3
    s = Sel(groups, width, vocab, k)
    logits = torch.zeros((groups * width, vocab), device="cuda")
    logits[1::2] = -0.0
    logits[3:6] = peaked(5, 1, vocab)
    logits[6, :] = -3.0
    logits[6, vocab - 1] = logits[6, 0] = logits[6, vocab // 2] = 2.5
    logits[7] = logits[6]
    logits[8] = logits[6]
    scores = torch.full((groups * width,), -2.0, device="cuda")
    got = s.run(logits, scores)
    want = B.select(logits.cpu().numpy(), scores.cpu().numpy(), width, k)
    assert got[0].tolist() == [w[0] for w in want]
    assert got[1].tolist() == [w[1] for w in want]
    s.close()


@pytest.mark.parametrize("order", ["up", "down", "one lane", "large", "tiny", "far"])
def test_hostile_orders(gpu, order):
    """Sorted rows; the best all with one lane or one thread; values up to f32's
    ends."""
    vocab, width, k = 151936, 2, 32
    s = Sel(1, width, vocab, k)
    x = torch.randn((width, vocab), device="cuda", generator=gen(4)) * 3
    if order == "up":
        x = x.sort(-1)[0]
    elif order == "down":
        x = x.sort(-1, descending=True)[0]
    elif order == "one lane":
        x[:, 12::2048] += 40
        x[:, 13::2048] += 40
    elif order == "large":
        x *= 1e38
        x.clamp_(-3e38, 3e38)
    elif order == "tiny":
        x *= 1e-38
    elif order == "far":
        x -= 3e38
    scores = torch.tensor([-1.0, -1.0001], device="cuda")
    got = s.run(x, scores)
    if order in ("up", "down", "one lane"):
        check(got, x, scores, width, k)
    else:  # differences past what a score in f32 shows: the order alone
        for r in range(width):
            mine = got[1][got[0] == r]
            want = torch.sort(x[r], descending=True, stable=True)[1][:len(mine)].cpu()
            assert torch.equal(x[r][mine.long().cuda()], x[r][want.cuda()])
    s.close()


def test_rows_apart_unaligned_and_in_place(gpu):
    """A view of wider rows from an odd place on; scores and done replaced in
    place; the same bits whatever the batch."""
    groups, width, vocab = 5, 4, 30001
    s = Sel(groups, width, vocab, width)
    wide = peaked(1, groups * width, vocab + 6)
    logits = wide[:, 3:3 + vocab]
    scores = -10 * torch.rand(groups * width, device="cuda", generator=gen(2))
    done = (torch.rand(groups * width, device="cuda", generator=gen(3)) < 0.2).int()
    want = s.run(logits, scores, done, 17)
    check(want, logits.contiguous(), scores, width, width, done, 17)
    assert all(torch.equal(a, b) for a, b in zip(s.run(logits.contiguous(), scores, done, 17), want))
    for g in (0, 3):
        rows = slice(g * width, (g + 1) * width)
        one = s.run(logits[rows], scores[rows], done[rows], 17)
        part = [t[rows] for t in want]
        part[0] = torch.where(part[0] >= 0, part[0] - g * width, -1)
        assert all(torch.equal(a, b) for a, b in zip(one, part))
    parent, token = (torch.empty(groups * width, dtype=torch.int32, device="cuda") for _ in range(2))
    Q.beam_select(s.ctx, s.sel, logits, scores, parent, token, scores, done, 17, done)
    assert all(torch.equal(a.cpu(), b) for a, b in zip((parent, token, scores, done), want))
    s.close()


def test_replayed_on_another_stream(gpu):
    groups, width, vocab, k = 7, 3, 20000, 5
    s = Sel(groups, width, vocab, k)
    logits, scores = torch.zeros((groups * width, vocab), device="cuda"), torch.zeros(groups * width, device="cuda")
    n = groups * k
    out = [torch.zeros(n, dtype=t, device="cuda") for t in (torch.int32, torch.int32, torch.float32)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        Q.beam_select(s.ctx, s.sel, logits, scores, *out)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        Q.beam_select(s.ctx, s.sel, logits, scores, *out)
    for i in range(4):
        logits.copy_(peaked(20 + i, groups * width, vocab))
        scores.copy_(-torch.rand(groups * width, device="cuda", generator=gen(40 + i)))
        graph.replay()
        got = [t.cpu() for t in out]
        want = s.run(logits, scores)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    del graph
    s.close()


def test_the_largest_selection(gpu):
    """1024 groups of 32 beams, 32 candidates each, most of them equal."""
    groups, width, vocab, k = 1024, 32, 33, 32
    s = Sel(groups, width, vocab, k)
    logits = torch.randint(-2, 3, (groups * width, vocab), device="cuda", generator=gen(1)).float()
    scores = -torch.randint(0, 4, (groups * width,), device="cuda", generator=gen(2)).float()
    got = [t.view(groups, k) for t in s.run(logits, scores)]
    x = logits.double()
    p = (x - x.logsumexp(-1, keepdim=True) + scores.double()[:, None]).view(groups, width * vocab).cpu()
    at = (got[0] % width).long() * vocab + got[1]
    bound = score_bound(vocab, 12.0)
    # The k best, whatever stands between equal ones of different rows, whose
    # sums may differ in their last bits; each once, best first.
    assert float((p.gather(1, at) - p.topk(k)[0]).abs().max()) <= 2 * bound
    assert float((p.gather(1, at) - got[2]).abs().max()) <= bound
    assert bool((at.sort(-1)[0].diff() > 0).all()) and bool((got[2].diff() <= 0).all())
    s.close()


def test_two_at_once_and_two_graphs_of_one_workspace(gpu):
    """Selections on two streams, each with its own workspace; then two graphs of
    one workspace, replayed in turn with an eager call between them."""
    vocab, width = 151936, 4
    a, b = Sel(3, width, vocab, 4), Sel(20, width, 5000, 9)
    x = peaked(1, 3 * width, vocab), peaked(2, 20 * width, 5000)
    sc = [-torch.rand(t.shape[0], device="cuda", generator=gen(3)) for t in x]
    want = a.run(x[0], sc[0]), b.run(x[1], sc[1])
    outs = [[torch.zeros(n, dtype=t, device="cuda") for t in (torch.int32, torch.int32, torch.float32)] for n in (12, 180)]
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate((a, b)):
            Q.beam_select(s.ctx, s.sel, x[i], sc[i], *outs[i], stream=streams[i].cuda_stream)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(t.cpu(), u) for t, u in zip(o, w))
    graphs = []
    for rows in (slice(0, 4), slice(0, 12)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            Q.beam_select(a.ctx, a.sel, x[0][rows], sc[0][rows], *outs[0])
        graphs.append(g)
    for _ in range(3):
        graphs[0].replay()
        assert all(torch.equal(t[:4].cpu(), u[:4]) for t, u in zip(outs[0], want[0]))
        a.run(x[0][:8], sc[0][:8])
        graphs[1].replay()
        assert all(torch.equal(t.cpu(), u) for t, u in zip(outs[0], want[0]))
    del g, graphs
    a.close()
    b.close()


def test_logits_past_32_bits(gpu):
    """Rows whose offsets pass 2^32 bytes and 2^31 values."""
    vocab, rows = 1 << 20, 2600
    s = Sel(1, 2, vocab, 3)
    wide = torch.zeros((rows, vocab), device="cuda")
    step = rows - 1
    wide[0], wide[step] = peaked(1, 1, vocab)[0], peaked(2, 1, vocab)[0]
    logits = wide[::step]
    assert logits.stride(0) > 1 << 31
    scores = torch.tensor([-1.0, -1.5], device="cuda")
    check(s.run(logits, scores), logits, scores, 2, 3)
    s.close()


def test_select_refuses(gpu):
    ctx = Q.Context(layers=1)
    for bad in ((0, 1, 10, 1), (1025, 1, 10, 1), (1, 0, 10, 1), (1, 33, 10, 1), (1, 1, 0, 1), (1, 1, (1 << 20) + 1, 1),
                (1, 1, 10, 0), (1, 1, 10, 33)):
        with pytest.raises(Q.QasrError) as e:
            Q.BeamSelect(ctx, *bad)
        assert e.value.code == Q.QASR_EINVAL
    sel = Q.BeamSelect(ctx, 2, 3, 100, 4)
    i = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    f = lambda *n: torch.zeros(n, device="cuda")  # noqa: E731
    good = dict(logits=f(6, 100), scores=f(6), parent=i(8), token=i(8), out_scores=f(8), done=None, eos=-1, out_done=None)

    def refused(code=Q.QASR_EINVAL, **k):
        with pytest.raises(Q.QasrError) as e:
            Q.beam_select(ctx, sel, *{**good, **k}.values())
        assert e.value.code == code

    refused(Q.QASR_ERANGE, logits=f(9, 100), scores=f(9), parent=i(12), token=i(12), out_scores=f(12))
    refused(eos=100)
    refused(eos=-2)
    same = f(16)
    refused(scores=same[:6], out_scores=same[:8])  # in place with k other than width
    refused(scores=same[:6], out_scores=same[4:12])
    both = i(12)
    refused(parent=both[:8], token=both[4:])
    x = f(6, 100)
    refused(logits=x, out_scores=x.view(-1)[50:58])
    for t in (dict(scores=f(6).double()), dict(parent=f(8)), dict(done=f(6)), dict(logits=f(6, 100).half()),
              dict(logits=f(6, 100).cpu())):
        with pytest.raises(ValueError):
            Q.beam_select(ctx, sel, *{**good, **t}.values())
    Q.beam_select(ctx, sel, *good.values())
    other = Q.Context(layers=1)
    with pytest.raises(Q.QasrError):
        Q.beam_select(other, sel, *good.values())
    sel.close()
    with pytest.raises(Q.QasrError):
        Q.beam_select(ctx, sel, *good.values())
    other.close()
    ctx.close()
