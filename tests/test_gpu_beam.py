"""Beams: the best continuations over beams and vocabulary (qwn_hip_ext_beam_select_device), and what
the beams keep following them (qwn_hip_ext_paged_kv_beam_advance_device)."""
import math
import random

import pytest
import torch

import serving as sv
from qwanto_amd import abi

pytestmark = pytest.mark.gpu


# ---- selection ------------------------------------------------------------------


def select(ctx, logits, scores, beams, vocab, count, dtype, ends=(), stride=0, following=True):
    """(values, parents, tokens, next scores, next parents, next tokens) on the host."""
    seqs = scores.numel() // beams
    x, s = logits.to(sv.DEV), scores.to(sv.DEV)
    out = [torch.full((seqs, n), -7, dtype=t, device=sv.DEV) for n in (count, beams) for t in (torch.float32, torch.int32, torch.int32)]
    work = torch.full((ctx.beam_select_workspace_bytes(seqs, beams, vocab, count),), 0xff, dtype=torch.uint8, device=sv.DEV)
    r = ctx.beam_select_request(seqs, beams, vocab, count, dtype, sv.ptr(x), sv.ptr(s), *(sv.ptr(o) for o in out[:3]), sv.ptr(work),
                                in_stride=stride, end_tokens=ends,
                                **(dict(zip(("next_scores_ptr", "next_parents_ptr", "next_tokens_ptr"), map(sv.ptr, out[3:]))) if following else {}))
    ctx.beam_select_device(r, stream=sv.stream())
    torch.cuda.synchronize()
    return [o.cpu() for o in out]


def reference(logits, scores, beams, vocab, count, ends=()):
    """The same in 64 bits, and the 64-bit values of all candidates [seqs][beams * vocab]."""
    seqs = scores.numel() // beams
    x = logits[:, :vocab].double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.amax(1, keepdim=True)
    total = top + torch.where(x > -math.inf, torch.exp(x - top), 0.0).sum(1, keepdim=True).log()
    s = scores.reshape(-1, 1).double()
    live = torch.isfinite(s) & torch.isfinite(top)
    c = torch.where(live & (x > -math.inf), s + (x - torch.where(live, total, 0.0)), -math.inf).reshape(seqs, -1)
    value, at = torch.sort(c, dim=1, descending=True, stable=True)
    value, at = value[:, :count], at[:, :count]
    if value.shape[1] < count:
        value = torch.nn.functional.pad(value, (0, count - value.shape[1]), value=-math.inf)
        at = torch.nn.functional.pad(at, (0, count - at.shape[1]))
    none = value == -math.inf
    parent = torch.where(none, -1, at // vocab + beams * torch.arange(seqs)[:, None])
    token = torch.where(none, -1, at % vocab)
    nxt = [[], [], []]
    for q in range(seqs):
        on = [i for i in range(count) if not none[q, i] and int(token[q, i]) not in ends][:beams]
        fill = beams - len(on)
        nxt[0].append([float(value[q, i]) for i in on] + [-math.inf] * fill)
        nxt[1].append([int(parent[q, i]) for i in on] + [-1] * fill)
        nxt[2].append([int(token[q, i]) for i in on] + [-1] * fill)
    return value, parent, token, *nxt, c


# The kernel's logarithm of a row's sum: each term is off by 2^-23 of itself (the power of 2) and, of
# its exponent of at most 40 / ln 2 where it counts, by three roundings (the difference, log2 e, their
# product), 2^-24 each: 3 * 40 * 2^-24 of the term.  Chains of at most 32 + 8 fp32 sums.
LSE = 2.0 ** -23 + 3 * 40 * 2.0 ** -24 + 40 * 2.0 ** -24


def check(got, want, vocab):
    value, parent, token, ns, np_, nt, c = want
    beams = c.shape[1] // vocab
    # Candidates of one row are in the order of their logits, whatever its sum; of two rows, where they
    # are further apart than the sums may be off.  Else each is as large as the one of its place, none
    # comes twice, and those of a row are in order.
    top, at = (x[:, :value.shape[1] + 1] for x in c.sort(dim=1, descending=True, stable=True))
    gap, row = top[:, :-1] - top[:, 1:], at // vocab
    near = (row[:, :-1] != row[:, 1:]) & (gap < 2 * LSE) & (top[:, 1:] > -math.inf) & (gap > 0)
    for s in range(c.shape[0]):
        if not bool(near[s].any()):
            assert torch.equal(got[1][s].long(), parent[s]) and torch.equal(got[2][s].long(), token[s])
            assert got[4][s].tolist() == np_[s] and got[5][s].tolist() == nt[s]
            continue
        n = int((value[s] > -math.inf).sum())
        places = (got[1][s].long() - s * beams) * vocab + got[2][s].long()
        assert bool(((c[s][places[:n]] - value[s][:n]).abs() <= 2 * LSE).all()) and len(set(places[:n].tolist())) == n
        for b in range(beams):
            mine = places[:n][places[:n] // vocab == b]
            assert torch.equal(mine, at[s][:-1][row[s][:-1] == b][:len(mine)])
    for a, b in ((got[0], value), (got[3], torch.tensor(ns, dtype=torch.float64))):
        inf = b == -math.inf
        assert torch.equal(a == -math.inf, inf)
        assert bool(((a.double() - b).abs()[~inf] <= 2 * LSE + 2.0 ** -24 * b.abs()[~inf]).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("seqs,beams,vocab,count,odd", [(1, 1, 1, 1, 0), (1, 4, 2, 8, 1), (2, 3, 5, 64, 0), (3, 4, 1000, 8, 3), (1, 1, 4096, 1, 0),
                                                        (2, 5, 4097, 16, 0), (1, 2, 8191, 64, 5), (7, 8, 20000, 17, 1), (1, 32, 3001, 64, 0),
                                                        (16, 4, 151936, 8, 0), (1, 4, 151936, 64, 8), (300, 2, 333, 4, 0)])
def test_select(gpu_ctx, dtype, seqs, beams, vocab, count, odd):
    g = sv.gen(vocab + count)
    rows = seqs * beams
    # 16-bit logits lie on a grid: beams' scores that no difference of two logits makes up for
    x = (3 * sv.normal(g, rows, vocab + odd)).to(sv.DTYPES[dtype])
    x[:, vocab:] = float("nan")
    scores = -10 * torch.rand(seqs, beams, generator=g) - 0.37 * torch.arange(beams)
    ends = [int(i) for i in torch.randint(0, vocab, (2,), generator=g)]
    want = reference(x, scores, beams, vocab, count, ends)
    check(select(gpu_ctx, x, scores, beams, vocab, count, dtype, ends, stride=vocab + odd), want, vocab)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_ties(gpu_ctx, dtype):
    """Equal logits: the lower token; beams alike: the lower beam; all logits of a row alike."""
    vocab, beams = 9000, 3
    x = torch.zeros(6, vocab).to(sv.DTYPES[dtype])
    x[3:, ::17] = 2.0
    x[3:, 5000] = 3.0
    scores = torch.tensor([[-1.0, -1.0, -1.0], [-2.0, -2.0, -2.0]])
    got = select(gpu_ctx, x, scores, beams, vocab, 12, dtype)
    assert got[1][0].tolist() == [0] * 12 and got[2][0].tolist() == list(range(12))
    assert got[1][1].tolist() == [3, 4, 5] + [3] * 9
    assert got[2][1].tolist() == [5000] * 3 + [17 * i for i in range(9)]
    got = select(gpu_ctx, torch.full((2, vocab), -0.0).to(sv.DTYPES[dtype]) * torch.tensor([1, -1]).repeat(vocab // 2).to(sv.DTYPES[dtype]),
                 torch.zeros(1, 2), 2, vocab, 5, dtype)
    assert got[2][0].tolist() == list(range(5))                                  # -0 is 0


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_beams_and_logits_that_are_left_out(gpu_ctx, dtype):
    vocab, beams = 5000, 4
    g = sv.gen(1)
    x = (2 * sv.normal(g, 4 * beams, vocab)).to(sv.DTYPES[dtype])
    scores = -torch.rand(4, beams, generator=g) - torch.arange(beams)
    scores[0, 1:] = -math.inf                                                    # a first step
    scores[1] = torch.tensor([math.nan, math.inf, -3.0, -math.inf])
    x[8] = -math.inf                                                             # rows with nothing left, with a logit of +inf, with few
    x[9, 77] = math.inf
    x[10] = math.nan
    x[11, torch.randperm(vocab, generator=g)[3:]] = -math.inf
    x[12:, ::2] = math.nan
    x[13, 1:] = -math.inf
    want = reference(x, scores, beams, vocab, 16, [5])
    got = select(gpu_ctx, x, scores, beams, vocab, 16, dtype, [5])
    check(got, want, vocab)
    assert got[1][2].tolist() == [11] * 3 + [-1] * 13
    assert got[3][2].tolist()[3:] == [-math.inf] and got[4][2].tolist()[3:] == [-1]
    everything = select(gpu_ctx, torch.full_like(x, -math.inf), scores, beams, vocab, 16, dtype)
    assert bool((everything[0] == -math.inf).all()) and all(bool((everything[i] == -1).all()) for i in (1, 2, 4, 5))


def test_all_that_is_best_ends(gpu_ctx):
    x = torch.zeros(2, 100)
    x[:, 10:14] = 9.0
    got = select(gpu_ctx, x, torch.tensor([[0.0, -5.0]]), 2, 100, 4, "f32", [10, 11, 12, 13])
    assert got[2][0].tolist() == [10, 11, 12, 13]
    assert got[3][0].tolist() == [-math.inf] * 2 and got[4][0].tolist() == [-1, -1] and got[5][0].tolist() == [-1, -1]
    got = select(gpu_ctx, x, torch.tensor([[0.0, -5.0]]), 2, 100, 4, "f32", following=False)
    assert bool((got[3] == -7).all()) and bool((got[4] == -7).all()) and bool((got[5] == -7).all())


@pytest.mark.parametrize("size", [1e30, 3e38, 1e-30])
def test_logits_of_any_size(gpu_ctx, size):
    g = sv.gen(4)
    x = (2 * torch.rand(2, 3000, generator=g) - 1) * size
    got = select(gpu_ctx, x, torch.tensor([[-1.0, -2.0]]), 2, 3000, 6, "f32")
    want = reference(x, torch.tensor([[-1.0, -2.0]]), 2, 3000, 6)
    if size > 1:
        assert torch.equal(got[1].long(), want[1]) and torch.equal(got[2].long(), want[2])
    tol = LSE + 2.0 ** -23 * want[0].abs()
    assert bool((((got[0].double() - want[0]).abs() <= tol) | (got[0].double() == want[0].float().double())).all())


def best_by_logit(logits, scores, beams, vocab, count):
    """[seqs][count] rows and tokens by value (a beam's by their logits: its sum and score are the same to all of
    them), the lower beam, the lower token; for beams whose values lie far apart."""
    rows, tokens = [], []
    for s in range(scores.shape[0]):
        order = sorted(((b, t) for b in range(beams) for t in range(vocab) if float(logits[s * beams + b, t]) > -math.inf),
                       key=lambda c: (-float(scores[s, c[0]]), c[0], -float(logits[s * beams + c[0], c[1]]), c[1]))[:count]
        rows.append([s * beams + b for b, _ in order])
        tokens.append([t for _, t in order])
    return rows, tokens


@pytest.mark.parametrize("size,score", [(1e-30, 0.0), (2.0 ** -40, -1.0), (1e-3, -1e9), (0.25, -1e12), (1.0, -3e38)])
def test_logits_apart_by_less_than_their_value_shows(gpu_ctx, size, score):
    """Of one beam the larger logits come first, also where score + logit is one 64-bit number for all of them (a
    score of -1e9 for beams that are not yet in use): over several parts of the vocabulary, in both orders."""
    vocab, count = 9001, 12
    g = sv.gen(int(-score) % 1000)
    up = (torch.arange(vocab) + 1.0) * (size / vocab)
    for x in (up, up.flip(0), up[torch.randperm(vocab, generator=g)]):
        logits = torch.full((2, vocab), -math.inf)
        logits[0, [5, 4097]] = torch.tensor([2.0, 3.0])
        logits[1] = x
        scores = torch.tensor([[score / 2 + 1.0, score]])
        if score == 0.0:
            scores = torch.tensor([[50.0, score]])
        got = select(gpu_ctx, logits, scores, 2, vocab, count, "f32")
        rows, tokens = best_by_logit(logits, scores, 2, vocab, count)
        assert rows[0][:2] == [0, 0] and rows[0][2:] == [1] * (count - 2)
        assert got[1].tolist() == rows and got[2].tolist() == tokens


def test_select_refusals(gpu_ctx):
    seqs, beams, vocab, count = 2, 3, 50, 6
    x = torch.zeros(seqs * beams, 2 * vocab, device=sv.DEV)
    s = torch.zeros(seqs, beams, device=sv.DEV)
    o = [torch.zeros(seqs, 8, dtype=torch.int32, device=sv.DEV) for _ in range(6)]
    work = torch.zeros(gpu_ctx.beam_select_workspace_bytes(seqs, beams, vocab, count) + 64, dtype=torch.uint8, device=sv.DEV)

    def req(**kw):
        base = dict(sequences=seqs, beams=beams, vocab=vocab, count=count, dtype="f32", logits_ptr=sv.ptr(x), scores_ptr=sv.ptr(s),
                    values_ptr=sv.ptr(o[0]), parents_ptr=sv.ptr(o[1]), tokens_ptr=sv.ptr(o[2]), workspace_ptr=sv.ptr(work),
                    in_stride=2 * vocab, end_tokens=[1], next_scores_ptr=sv.ptr(o[3]), next_parents_ptr=sv.ptr(o[4]), next_tokens_ptr=sv.ptr(o[5]))
        base.update(kw)
        return gpu_ctx.beam_select_request(**base)

    def status(r):
        with pytest.raises(abi.AbiError) as e:
            gpu_ctx.beam_select_device(r, stream=sv.stream())
        return e.value.status

    none = dict(next_scores_ptr=None, next_parents_ptr=None, next_tokens_ptr=None)
    for good in (req(), req(next_scores_ptr=sv.ptr(s)), req(**none), req(end_tokens=[1, 2, 3, 4])):
        gpu_ctx.beam_select_device(good, stream=sv.stream())
    for bad in (dict(sequences=0), dict(beams=0), dict(vocab=0), dict(count=0), dict(logits_ptr=None), dict(scores_ptr=None),
                dict(values_ptr=None), dict(parents_ptr=None), dict(tokens_ptr=None), dict(workspace_ptr=None),
                dict(workspace_ptr=sv.ptr(work) + 8), dict(in_stride=vocab - 1), dict(next_scores_ptr=None), dict(next_tokens_ptr=None),
                dict(values_ptr=sv.ptr(s)), dict(values_ptr=sv.ptr(x)), dict(parents_ptr=sv.ptr(o[2])), dict(tokens_ptr=sv.ptr(work) + 4),
                dict(next_parents_ptr=sv.ptr(s)), dict(next_scores_ptr=sv.ptr(s) + 4), dict(next_tokens_ptr=sv.ptr(x) + 4),
                dict(workspace_ptr=sv.ptr(x)), dict(next_tokens_ptr=sv.ptr(o[0]) + 4 * (seqs * count - 1))):
        assert status(req(**bad)) == -1, bad
    for bad in (dict(beams=33, sequences=1), dict(count=65), dict(vocab=2 ** 24 + 1, in_stride=0), dict(sequences=65536, beams=1)):
        assert status(req(**bad)) == -5, bad
    for sizes in ((0, 1, 1, 1), (1, 33, 1, 1), (1, 1, 0, 1), (1, 1, 1, 65), (65536, 1, 5, 5)):
        assert gpu_ctx.beam_select_workspace_bytes(*sizes) == 0
    r = req()
    r.end_count = 5
    assert status(r) == -1
    r = req()
    r.dtype = 3
    assert status(r) == -1
    torch.cuda.synchronize()


def test_select_captured_and_on_two_streams(gpu_ctx):
    """Recorded once, its scores in place, replayed with other logits, eager calls on another stream
    between."""
    seqs, beams, vocab, count = 5, 4, 12345, 8
    x = torch.zeros(seqs * beams, vocab, device=sv.DEV)
    n = gpu_ctx.beam_select_workspace_bytes(seqs, beams, vocab, count)

    def one():
        s = torch.zeros(seqs, beams, device=sv.DEV)
        o = [torch.zeros(seqs, k, dtype=t, device=sv.DEV) for k, t in ((count, torch.float32), (count, torch.int32), (count, torch.int32),
                                                                      (beams, torch.int32), (beams, torch.int32))]
        work = torch.zeros(n, dtype=torch.uint8, device=sv.DEV)
        return s, o, work, gpu_ctx.beam_select_request(seqs, beams, vocab, count, "f32", sv.ptr(x), sv.ptr(s), *(sv.ptr(t) for t in o[:3]),
                                                       sv.ptr(work), end_tokens=[3], next_scores_ptr=sv.ptr(s), next_parents_ptr=sv.ptr(o[3]),
                                                       next_tokens_ptr=sv.ptr(o[4]))

    a, b = one(), one()
    gpu_ctx.beam_select_device(b[3], stream=sv.stream())
    b[0].zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu_ctx.beam_select_device(a[3], stream=sv.stream())
    side = torch.cuda.Stream()
    for i in range(4):
        before = a[0].cpu()
        x.copy_(3 * sv.normal(sv.gen(i), seqs * beams, vocab))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            gpu_ctx.beam_select_device(b[3], stream=sv.stream())
        torch.cuda.synchronize()
        assert torch.equal(a[0], b[0]) and all(torch.equal(p, q) for p, q in zip(a[1], b[1]))
        check([t.cpu() for t in (*a[1][:3], a[0], a[1][3], a[1][4])], reference(x.cpu(), before, beams, vocab, count, [3]), vocab)


# ---- what the beams keep ----------------------------------------------------------


def advance_reference(beams, page, added, parents, past, table, spare, tokens, history):
    """The rows' states after a step, by the operator's description; and (from page, to page, slots) of
    what is copied."""
    rows, stride = table.shape
    out = [past.clone(), table.clone(), spare.clone(), history.clone()]
    copies = []
    for first in range(0, rows, beams):
        group = range(first, first + beams)
        real = {r: first <= int(parents[r]) < first + beams and int(past[parents[r]]) >= 0 for r in group}
        parent = {r: int(parents[r]) if real[r] else r for r in group}
        goes = [r for r in group if int(past[parent[r]]) >= 0]
        childless = [q for q in group if q not in [parent[r] for r in goes]]
        seen, free = set(), iter(childless)
        for r in goes:
            p = parent[r]
            n = min(int(past[p]) + added, 2 ** 31 - 1)
            full, used = n // page, n % page
            later = p in seen
            seen.add(p)
            q = next(free, None) if later else None
            out[0][r] = n
            row = table[p].clone()
            row[full + 1:] = -1
            if used == 0 or later:
                if full < stride:
                    row[full] = spare[r]
                if used and full < stride and 0 <= int(table[p, full]) and int(spare[r]) >= 0 and int(table[p, full]) != int(spare[r]):
                    copies.append((int(table[p, full]), int(spare[r]), used))
            out[1][r] = row
            if used == 0:
                out[2][r] = -1
            elif later:
                out[2][r] = -1
                if q is not None and int(past[q]) >= 0:
                    m = int(past[q]) + added
                    if m % page and m // page < stride:
                        out[2][r] = table[q, m // page]
            out[3][r] = history[p]
            if real[r] and n < history.shape[1]:
                out[3][r, n] = tokens[r]
    return out, copies


class Beams:
    """Caches of a few layers, filled page by page, and rows that own two pages each."""

    def __init__(self, ctx, seqs, beams, page, lengths, layers=2, kv_heads=2, d=64, seed=0, history=40):
        g = sv.gen(seed)
        self.ctx, self.beams, self.page, self.rows, self.hk, self.d = ctx, beams, page, seqs * beams, kv_heads, d
        n = [lengths[r // beams] if isinstance(lengths, list) else lengths for r in range(self.rows)]
        self.stride = max(n) // page + 2
        whole = sum(n[s * beams] // page for s in range(seqs))
        self.pages = whole + 4 * self.rows + 2
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.table = torch.full((self.rows, self.stride), -1, dtype=torch.int32)
        at = 0
        for s in range(seqs):
            full = n[s * beams] // page
            for r in range(s * beams, (s + 1) * beams):
                self.table[r, :full] = order[at:at + full]
                self.table[r, full] = order[whole + r]                           # where the next token goes
            at += full
        self.spare = order[whole + self.rows:whole + 2 * self.rows].clone()
        self.past = torch.tensor(n, dtype=torch.int32)
        self.history = torch.randint(0, 999, (self.rows, history), generator=g, dtype=torch.int32)
        self.caches = [ctx.paged_kv_create(self.pages, page, kv_heads, d) for _ in range(layers)]
        # every slot of every page holds numbers of its own
        self.everything = torch.arange(self.pages, dtype=torch.int32, device=sv.DEV).reshape(1, -1).contiguous()
        slots = self.pages * page
        self.ends = torch.tensor([0, slots], dtype=torch.int32, device=sv.DEV)
        self.zero = torch.zeros(1, dtype=torch.int32, device=sv.DEV)
        self.all = ctx.paged_batch(1, slots, sv.ptr(self.ends), sv.ptr(self.zero), sv.ptr(self.everything), self.pages)
        for c in self.caches:
            k, v = (sv.normal(g, slots, kv_heads * d).to(sv.DEV) for _ in range(2))
            ctx.paged_kv_append_device(c, ctx.paged_append_request(self.all, "f32", sv.ptr(k), sv.ptr(v)), stream=sv.stream())
            torch.cuda.synchronize()

    def contents(self):
        """[layer][keys, values][page][slot][channels] of the whole pools."""
        out = torch.zeros(len(self.caches), 2, self.pages * self.page, self.hk * self.d, device=sv.DEV)
        for c, x in zip(self.caches, out):
            self.ctx.paged_kv_read_device(c, self.all, sv.ptr(x[0]), sv.ptr(x[1]), stream=sv.stream())
        torch.cuda.synchronize()
        return out.cpu().reshape(len(self.caches), 2, self.pages, self.page, -1)

    def run(self, parents, tokens, added=1, in_place=False, state=None):
        """(past, table, spare, history) after a step, on the host."""
        dev = [x.to(sv.DEV).contiguous() for x in (state or (self.past, self.table, self.spare, self.history))]
        out = [torch.full_like(x, -99) for x in dev]
        if in_place:
            out[1], out[3] = dev[1], dev[3]
        p, t = parents.to(sv.DEV), tokens.to(sv.DEV)
        r = self.ctx.beam_advance_request(self.rows // self.beams, self.beams, self.page, self.stride, sv.ptr(p), sv.ptr(dev[0]), sv.ptr(out[0]),
                                          sv.ptr(dev[1]), sv.ptr(out[1]), sv.ptr(dev[2]), sv.ptr(out[2]), added=added, tokens_ptr=sv.ptr(t),
                                          history_ptr=sv.ptr(dev[3]), history_out_ptr=sv.ptr(out[3]), history_length=dev[3].shape[1])
        self.ctx.paged_kv_beam_advance_device(self.caches, r, stream=sv.stream())
        torch.cuda.synchronize()
        return [x.cpu() for x in out]

    def close(self):
        torch.cuda.synchronize()
        for c in self.caches:
            self.ctx.paged_kv_destroy(c)


def check_advance(b, parents, tokens, added=1, in_place=False, state=None):
    state = state or (b.past, b.table, b.spare, b.history)
    before = b.contents()
    got = b.run(parents, tokens, added, in_place, state)
    past, table, spare, history = state
    want, copies = advance_reference(b.beams, b.page, added, parents, past, table, spare, tokens, history)
    for name, x, y in zip(("past", "table", "spare", "history"), got, want):
        assert torch.equal(x, y), name
    after, expect, touched = b.contents(), before.clone(), torch.zeros(b.pages, b.page, dtype=torch.bool)
    for src, dst, used in copies:
        expect[:, :, dst, :used] = before[:, :, src, :used]
        touched[dst, used:-(-used // 16) * 16] = True                           # the rest of the last tile is no slot of the row
    assert torch.equal(after[:, :, ~touched], expect[:, :, ~touched])
    return got


def owned(b, state):
    """The pages in use and the spares of the rows: each has one owner."""
    past, table, spare, _ = state
    mine = [int(table[r, int(past[r]) // b.page]) for r in range(b.rows)] + [int(s) for s in spare if s >= 0]
    return len(mine) == len(set(mine)) and min(mine) >= 0


@pytest.mark.parametrize("seqs,beams,page,length,hk,d", [(1, 1, 16, 5, 1, 64), (1, 4, 16, 20, 2, 64), (3, 4, 32, 30, 2, 128), (2, 8, 64, 130, 1, 80),
                                                         (5, 3, 16, 15, 3, 256), (1, 32, 16, 40, 2, 32), (70, 2, 128, 260, 1, 64), (2, 5, 16, 0, 2, 64)])
@pytest.mark.parametrize("in_place", [False, True])
def test_advance(gpu_ctx, seqs, beams, page, length, hk, d, in_place):
    """Several steps, each from what the one before left; parents at random."""
    rng = random.Random(seqs + 100 * beams + length)
    b = Beams(gpu_ctx, seqs, beams, page, length, kv_heads=hk, d=d, seed=beams)
    try:
        state = (b.past, b.table, b.spare, b.history)
        for step in range(4):
            parents = torch.tensor([r // beams * beams + rng.randrange(beams) if rng.random() < 0.9 else -1 for r in range(b.rows)], dtype=torch.int32)
            tokens = torch.tensor([rng.randrange(999) for _ in range(b.rows)], dtype=torch.int32)
            state = check_advance(b, parents, tokens, in_place=in_place, state=state)
            assert owned(b, state)
            # a page has just become full: the caller hands out others, here pages that are no row's
            gone = set(state[1].flatten().tolist()) | set(state[2].tolist())
            free = [p for p in range(b.pages) if p not in gone]
            for r in range(b.rows):
                if int(state[2][r]) < 0:
                    state[2][r] = free.pop()
    finally:
        b.close()


def test_advance_parents_of_every_kind(gpu_ctx):
    """One parent for all, each its own, the last one's, parents of another sequence and out of range,
    lengths that differ and negative ones, pages and spares that are none, full pages, a full table."""
    b = Beams(gpu_ctx, 2, 4, 16, [21, 31], history=24)
    try:
        t = torch.arange(8, dtype=torch.int32) + 100
        i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
        full = (b.past, b.table, b.spare, b.history)
        for parents in (i(0, 0, 0, 0, 4, 4, 4, 4), i(0, 1, 2, 3, 4, 5, 6, 7), i(3, 2, 1, 0, 7, 7, 6, 6), i(4, 5, 6, 7, 0, 1, 2, 3),
                        i(-1, 99, 2 ** 31 - 1, -2 ** 31, 4, -1, 4, -1), i(1, 1, 3, 3, 5, 4, 5, 4)):
            for added in (0, 1, 3, 11, 2 ** 31 - 1):
                check_advance(b, parents, t, added=added, state=full)
        past = i(21, 5, -1, 16, 31, -7, 0, 2 ** 31 - 1)
        for parents in (i(0, 1, 2, 3, 4, 5, 6, 7), i(2, 2, 0, 1, 5, 4, 4, 6), i(1, 1, 1, 1, 7, 7, 6, 6)):
            check_advance(b, parents, t, state=(past, b.table, b.spare, b.history))
        none = b.table.clone()
        none[0, 1], none[5, 1] = -1, b.pages
        bad = b.spare.clone()
        bad[1], bad[2], bad[6] = -1, b.pages, -2 ** 31
        before = b.contents()
        got = b.run(i(0, 0, 1, 1, 5, 5, 4, 4), t, state=(b.past, none, bad, b.history))
        want, _ = advance_reference(4, 16, 1, i(0, 0, 1, 1, 5, 5, 4, 4), b.past, none, bad, t, b.history)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        after = b.contents()                     # row 3 (from 1) and row 7 (from 4) have pages to copy between
        changed = [p for p in range(b.pages) if not torch.equal(after[:, :, p], before[:, :, p])]
        assert set(changed) <= {int(b.spare[3]), int(b.spare[7])}
    finally:
        b.close()


class Owned:
    """A sequence's rows as a caller keeps them, at lengths of their own: every page in use and every spare has one
    owner, whole pages are shared; rows of a negative length have a spare and nothing else."""

    def __init__(self, b, past, rng):
        page, width = b.page, b.stride
        pages = list(range(b.pages))
        rng.shuffle(pages)
        whole = [pages.pop() for _ in range(3)]
        self.past = torch.tensor(past, dtype=torch.int32)
        self.table = torch.full((len(past), width), -1, dtype=torch.int32)
        for r, n in enumerate(past):
            for c in range(n // page if n >= 0 else 0):
                self.table[r, c] = whole[c]
            if n >= 0 and n // page < width:
                self.table[r, n // page] = pages.pop()
        self.spare = torch.tensor([pages.pop() for _ in past], dtype=torch.int32)
        self.history = torch.zeros(len(past), 4, dtype=torch.int32)

    def state(self):
        return self.past, self.table, self.spare, self.history


def check_ownership(b, parents, before, after):
    """A step of one token by the rule of ownership.  Of the rows' pages, in use before or spare, each is afterwards the
    page in use or the spare of one row, as long as there are rows without a spare to take it; the first row with a
    parent goes on in that one's page in use, further ones and rows that begin a page in their own spare."""
    past, table, spare, _ = before
    past2, table2, spare2, _ = after
    rows, width, page = len(past), table.shape[1], b.page
    real = [0 <= int(p) < rows and int(past[p]) >= 0 for p in parents]
    parent = [int(p) if ok else r for r, (p, ok) in enumerate(zip(parents, real))]
    goes = [int(past[parent[r]]) >= 0 for r in range(rows)]
    cell = lambda t, r, n: int(t[r, n // page]) if n // page < width else -1  # noqa: E731
    gone_on, mine, given = set(), {}, set()
    for r in range(rows):
        if not goes[r]:
            assert int(past2[r]) == int(past[r]) and torch.equal(table2[r], table[r]) and int(spare2[r]) == int(spare[r])
            continue
        p, n = parent[r], int(past[parent[r]]) + 1
        assert int(past2[r]) == n
        if n % page == 0 and n // page == width:                                 # no column for another page: the spare stays
            assert int(spare2[r]) == int(spare[r])
            gone_on.add(p)
            continue
        takes = n % page == 0 or p in gone_on
        gone_on.add(p)
        assert cell(table2, r, n) == (int(spare[r]) if takes else cell(table, p, n))
        mine[r] = cell(table2, r, n)
        if not takes:
            assert int(spare2[r]) == int(spare[r])
        elif int(spare2[r]) >= 0:
            given.add(int(spare2[r]))
    # what rows that nothing goes on from leave: their pages in use
    left = {cell(table, q, int(past[q]) + 1) for q in range(rows) if int(past[q]) >= 0 and q not in gone_on and (int(past[q]) + 1) % page} - {-1}
    assert given <= left
    without = [r for r in range(rows) if goes[r] and int(spare2[r]) < 0]
    assert given == left or not without, (given, left, without)
    owned_now = list(mine.values()) + [int(s) for s in spare2 if s >= 0]
    assert len(owned_now) == len(set(owned_now))
    return left - given


@pytest.mark.parametrize("past,parents", [
    ([-1, 21, 21, 21], [-1, 1, 1, 2]),                                           # a row without a length before one that leaves a page
    ([-1, 5, 5], [-1, 1, 1]),
    ([5, -1, 5, -1, 5, 5], [4, 4, 4, -1, 4, 4]),
    ([21, 31, 21, 21], [2, 1, 2, 2]),                                            # rows that nothing goes on from, one with a page just full
    ([31, 21, 31, 21, 21], [0, 3, 0, 3, 3]),                                     # a row that begins a page among those that copy
    ([21, 15], [1, 1]),                                                          # a page in use is left, and only rows that begin one
    ([46, 46, 46], [1, 1, 1]),
    ([47, 47, 47], [0, 1, 1]),                                                   # the table ends: no column for a next page
    ([47, 30, 47], [2, 2, 2]),
])
def test_advance_loses_no_page(gpu_ctx, past, parents):
    b = Beams(gpu_ctx, 1, len(past), 16, 20, layers=1)                           # tables of 3 pages
    try:
        o = Owned(b, past, random.Random(1))
        contents = b.contents()
        got = b.run(torch.tensor(parents, dtype=torch.int32), torch.arange(len(past), dtype=torch.int32), state=o.state())
        lost = check_ownership(b, parents, o.state(), got)
        assert not lost or all(n < 0 or n // 16 == b.stride for n in got[0].tolist())
        after = b.contents()
        for r, p in enumerate(parents):                                          # every row has its parent's tokens
            p = p if p >= 0 else r
            for t in range(int(o.past[p]) + 1 if int(o.past[p]) >= 0 else 0):
                src, dst = int(o.table[p, t // 16]), int(got[1][r, t // 16])
                assert torch.equal(after[:, :, dst, t % 16], contents[:, :, src, t % 16])
    finally:
        b.close()


def test_advance_owns_pages_at_any_lengths(gpu_ctx):
    rng = random.Random(7)
    b = Beams(gpu_ctx, 1, 8, 16, 20, layers=1)
    try:
        for _ in range(150):
            alike = rng.randrange(1, 46)
            past = [alike if rng.random() < 0.6 else rng.choice([-1, 14, 15, 16, 30, 31, rng.randrange(0, 46)]) for _ in range(8)]
            parents = [rng.choice([-1, *range(8), *[rng.randrange(8)] * 8]) for _ in range(8)]
            o = Owned(b, past, rng)
            got = b.run(torch.tensor(parents, dtype=torch.int32), torch.arange(8, dtype=torch.int32), state=o.state())
            assert not check_ownership(b, parents, o.state(), got), (past, parents)
    finally:
        b.close()


def test_advance_without_caches_tokens_or_histories(gpu_ctx):
    b = Beams(gpu_ctx, 1, 4, 16, 20)
    try:
        p = torch.tensor([0, 0, 2, 2], dtype=torch.int32)
        dev = [x.to(sv.DEV).contiguous() for x in (b.past, b.table, b.spare)]
        out = [torch.full_like(x, -99) for x in dev]
        pd = p.to(sv.DEV)
        before = b.contents()
        r = gpu_ctx.beam_advance_request(1, 4, 16, b.stride, sv.ptr(pd), sv.ptr(dev[0]), sv.ptr(out[0]), sv.ptr(dev[1]), sv.ptr(out[1]),
                                         sv.ptr(dev[2]), sv.ptr(out[2]))
        gpu_ctx.paged_kv_beam_advance_device([], r, stream=sv.stream())
        torch.cuda.synchronize()
        want, _ = advance_reference(4, 16, 1, p, b.past, b.table, b.spare, p, b.history)
        assert all(torch.equal(x.cpu(), y) for x, y in zip(out, want))
        assert torch.equal(b.contents(), before)
    finally:
        b.close()


def test_advance_refusals(gpu_ctx):
    b = Beams(gpu_ctx, 1, 4, 16, 20)
    other = gpu_ctx.paged_kv_create(b.pages, 16, 1, 64)
    wide = gpu_ctx.paged_kv_create(b.pages, 32, 2, 64)
    few = gpu_ctx.paged_kv_create(b.pages - 1, 16, 2, 64)
    try:
        i = {n: torch.zeros(4, b.stride if n.startswith("table") else 40 if n.startswith("history") else 1, dtype=torch.int32, device=sv.DEV)
             for n in ("parents", "past", "past_out", "table", "table_out", "spare", "spare_out", "tokens", "history", "history_out")}
        i["spare"] -= 1

        def req(**kw):
            base = dict(sequences=1, beams=4, page_tokens=16, table_stride=b.stride, history_length=40) | {n + "_ptr": sv.ptr(t) for n, t in i.items()}
            base.update(kw)
            return gpu_ctx.beam_advance_request(**base)

        def status(r, caches=b.caches):
            with pytest.raises(abi.AbiError) as e:
                gpu_ctx.paged_kv_beam_advance_device(caches, r, stream=sv.stream())
            return e.value.status

        for good in (req(), req(table_out_ptr=sv.ptr(i["table"])), req(history_out_ptr=sv.ptr(i["history"])), req(tokens_ptr=None),
                     req(history_ptr=None, history_out_ptr=None)):
            gpu_ctx.paged_kv_beam_advance_device(b.caches, good, stream=sv.stream())
        bad = [{n + "_ptr": None} for n in i if n != "tokens"]
        bad += [{n + "_ptr": sv.ptr(i[m])} for n in ("past_out", "spare_out", "table_out", "history_out") for m in i
                if m != n and (n, m) not in (("table_out", "table"), ("history_out", "history"))]
        bad += [dict(sequences=0), dict(beams=0), dict(table_stride=0), dict(page_tokens=24), dict(page_tokens=8), dict(page_tokens=2048),
                dict(history_length=0), dict(added=2 ** 31), dict(page_tokens=32), dict(table_out_ptr=sv.ptr(i["table"]) + 4)]
        for kw in bad:
            assert status(req(**kw)) == -1, kw
        for kw in (dict(beams=33), dict(sequences=20000)):
            assert status(req(**kw)) == -5, kw
        assert status(req(), b.caches * 129) == -5
        for c in (other, wide, few):
            assert status(req(), [b.caches[0], c]) == -1
        gone = abi.Handle()
        assert status(req(), [gone]) == -1
        torch.cuda.synchronize()
    finally:
        b.close()
        for c in (other, wide, few):
            gpu_ctx.paged_kv_destroy(c)
