"""Prompts taken in and continued by several beams each, the operators in the order in which they are
used: rotary positions, attention over the prompts' own keys and values, the cache, then steps of
rotary positions, append, attention over the cache, selection of the beams, and what they keep.  Every
stage against its definition from what the stage before it left; eager, captured, and two at once.
The projections between the operators are tables by token."""
import math

import pytest
import torch

import serving as sv
from qwanto_amd import abi
from test_gpu_beam import Beams, advance_reference
from test_gpu_beam import check as check_select
from test_gpu_beam import reference as select_reference
from test_gpu_prompt_attention import check as check_prompt
from test_gpu_rotary import check as check_rotary
from test_gpu_rotary import reference as rotary_reference

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, VOCAB, PAGE, BEAMS, COUNT, END, EPS, THETA = 4, 2, 64, 500, 16, 3, 6, 7, 1e-6, 1e6
SECTIONS, SCALE, HISTORY, SLOTS, POOL = [16, 8, 8], DIM ** -0.5, 96, 80, 120


class Generation:
    """Sequences with prompts of the given lengths; every buffer is made once, what changes from step to
    step is on the device."""

    def __init__(self, ctx, lengths, dtype, seed):
        self.ctx, self.dtype, self.lengths, self.seqs, self.rows = ctx, dtype, lengths, len(lengths), len(lengths) * BEAMS
        g, t, dev = sv.gen(seed), sv.DTYPES[dtype], sv.DEV
        f = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
        i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
        x = lambda *s: torch.zeros(*s, dtype=t, device=dev)  # noqa: E731
        # "projections" of a token, and its part of the next one's logits
        self.tables = [sv.normal(g, VOCAB, n * DIM).to(t).to(dev) for n in (HEADS, KV_HEADS, KV_HEADS)]
        self.head = sv.normal(g, VOCAB, VOCAB).to(dev)
        self.mix = torch.randint(0, HEADS * DIM, (VOCAB,), generator=g).to(dev)
        self.norms = [(1 + 0.2 * sv.normal(g, DIM)).to(dev) for _ in range(2)]
        p, n, rows = sv.ptr, sum(lengths), self.rows
        self.prompt = torch.randint(8, VOCAB, (n,), generator=g, dtype=torch.int32)
        # two axes of the prompts differ from the first, as where it has an image
        self.prompt_at = torch.cat([torch.arange(m) for m in lengths]).to(torch.int32).repeat(3, 1).contiguous()
        self.prompt_at[1:, 3:9] = torch.randint(0, 20, (2, 6), generator=g, dtype=torch.int32)

        self.cache = ctx.paged_kv_create(POOL, PAGE, KV_HEADS, DIM)
        order = torch.randperm(POOL, generator=g).to(torch.int32).tolist()
        table = torch.full((rows, SLOTS // PAGE), -1, dtype=torch.int32)
        for s, m in enumerate(lengths):
            for r in range(s * BEAMS, (s + 1) * BEAMS):
                if r == s * BEAMS:
                    for c in range(m // PAGE):
                        table[r, c] = order.pop()
                table[r, m // PAGE] = order.pop()     # the page in use; of the other beams it becomes a spare
        self.free = order
        self.past = torch.tensor([m for m in lengths for _ in range(BEAMS)], dtype=torch.int32, device=dev)
        self.table, self.spare = table.to(dev), torch.tensor([order.pop() for _ in range(rows)], dtype=torch.int32, device=dev)
        self.history = i(rows, HISTORY) - 1
        self.scores = torch.full((rows,), -math.inf, device=dev)
        self.scores[::BEAMS] = 0.0
        self.tokens = i(rows)
        self.out = [torch.empty_like(b) for b in (self.past, self.table, self.spare, self.history)]

        # prompts
        self.starts, self.first = torch.tensor([sum(lengths[:s]) for s in range(self.seqs + 1)], dtype=torch.int32, device=dev), i(self.seqs)
        self.first_table = self.table[::BEAMS].contiguous()
        self.at = self.prompt_at.to(dev)
        self.pq, self.pk, self.pv = (w[self.prompt.long().to(dev)].contiguous() for w in self.tables)
        self.pqr, self.pkr, self.po = torch.empty_like(self.pq), torch.empty_like(self.pk), torch.full_like(self.pq, 5.0)
        rotary = dict(sections=SECTIONS, in_turn=True, q_norm_ptr=p(self.norms[0]), k_norm_ptr=p(self.norms[1]), eps=EPS)
        self.prompt_rotary = ctx.rotary_request(n, dtype, DIM, DIM, THETA, p(self.at), query_heads=HEADS, q_ptr=p(self.pq), q_out_ptr=p(self.pqr),
                                                key_heads=KV_HEADS, k_ptr=p(self.pk), k_out_ptr=p(self.pkr), **rotary)
        self.prompt_attention = ctx.prompt_attention_request(self.seqs, n, p(self.starts), dtype, HEADS, KV_HEADS, DIM, p(self.pqr), p(self.pkr),
                                                             p(self.pv), p(self.po), SCALE)
        self.prompt_batch = ctx.paged_batch(self.seqs, n, p(self.starts), p(self.first), p(self.first_table), SLOTS // PAGE)
        self.prompt_append = ctx.paged_append_request(self.prompt_batch, dtype, p(self.pkr), p(self.pv))

        # steps
        self.q, self.qr, self.o = (x(rows, HEADS * DIM) for _ in range(3))
        self.k, self.kr, self.v = (x(rows, KV_HEADS * DIM) for _ in range(3))
        self.positions, self.logits = i(3, rows), f(rows, VOCAB)
        self.each = torch.arange(rows + 1, dtype=torch.int32, device=dev)
        self.values, self.parents, self.best = f(self.seqs, COUNT), i(self.seqs, COUNT), i(self.seqs, COUNT)
        self.next = [f(rows), i(rows), i(rows)]
        self.rotary = ctx.rotary_request(rows, dtype, DIM, DIM, THETA, p(self.positions), query_heads=HEADS, q_ptr=p(self.q), q_out_ptr=p(self.qr),
                                         key_heads=KV_HEADS, k_ptr=p(self.k), k_out_ptr=p(self.kr), **rotary)
        self.batch = ctx.paged_batch(rows, rows, p(self.each), p(self.past), p(self.table), SLOTS // PAGE)
        self.append = ctx.paged_append_request(self.batch, dtype, p(self.kr), p(self.v))
        self.attention = ctx.paged_attention_request(self.batch, dtype, HEADS, p(self.qr), p(self.o), SCALE)
        self.work = torch.full((ctx.paged_attention_workspace_bytes(self.cache, self.attention),), 0xff, dtype=torch.uint8, device=dev)
        self.attention.workspace = p(self.work)
        self.select_work = torch.full((ctx.beam_select_workspace_bytes(self.seqs, BEAMS, VOCAB, COUNT),), 0xff, dtype=torch.uint8, device=dev)
        self.select = ctx.beam_select_request(self.seqs, BEAMS, VOCAB, COUNT, "f32", p(self.logits), p(self.scores), p(self.values), p(self.parents),
                                              p(self.best), p(self.select_work), end_tokens=[END],
                                              next_scores_ptr=p(self.next[0]), next_parents_ptr=p(self.next[1]), next_tokens_ptr=p(self.next[2]))
        advance = lambda added: ctx.beam_advance_request(  # noqa: E731
            self.seqs, BEAMS, PAGE, SLOTS // PAGE, p(self.next[1]), p(self.past), p(self.out[0]), p(self.table), p(self.out[1]), p(self.spare),
            p(self.out[2]), added=added, tokens_ptr=p(self.next[2]), history_ptr=p(self.history), history_out_ptr=p(self.out[3]),
            history_length=HISTORY)
        self.first_advance, self.advance = advance(0), advance(1)
        for s, m in enumerate(lengths):
            self.history[s * BEAMS, :m] = self.prompt[sum(lengths[:s]):sum(lengths[:s]) + m].to(dev)

    def logits_of(self, tokens, o):
        """Their logits: the token's, and a channel of the attention for each."""
        torch.add(self.head.index_select(0, tokens.clamp(min=0).long()), o.float().index_select(1, self.mix), alpha=3.0, out=self.logits)

    def take_prompts(self):
        st = sv.stream()
        self.ctx.rotary_device(self.prompt_rotary, stream=st)
        self.ctx.prompt_attention_device(self.prompt_attention, stream=st)
        self.ctx.paged_kv_append_device(self.cache, self.prompt_append, stream=st)
        last = (self.starts[1:] - 1).long().repeat_interleave(BEAMS)
        self.logits_of(self.prompt.to(sv.DEV)[last], self.po[last])
        self.ctx.beam_select_device(self.select, stream=st)
        self.ctx.paged_kv_beam_advance_device([self.cache], self.first_advance, stream=st)

    def step(self):
        st = sv.stream()
        at = self.tokens.clamp(min=0).long()
        for w, x in zip(self.tables, (self.q, self.k, self.v)):
            x.copy_(w.index_select(0, at))
        self.positions.copy_(self.past.expand(3, -1))
        self.ctx.rotary_device(self.rotary, stream=st)
        self.ctx.paged_kv_append_device(self.cache, self.append, stream=st)
        self.ctx.paged_kv_attention_device(self.cache, self.attention, stream=st)
        self.logits_of(self.tokens, self.o)
        self.ctx.beam_select_device(self.select, stream=st)
        self.ctx.paged_kv_beam_advance_device([self.cache], self.advance, stream=st)

    def take_over(self):
        """The step's results are the next one's state; rows without a spare page get one."""
        spare = self.out[2].cpu()
        for r in range(self.rows):
            if spare[r] < 0:
                spare[r] = self.free.pop()
        self.out[2].copy_(spare)
        for a, b in zip((self.past, self.table, self.spare, self.history, self.scores, self.tokens), (*self.out, self.next[0], self.next[2])):
            a.copy_(b)
        torch.cuda.synchronize()

    def state(self):
        return [x.cpu() for x in (*self.out, *self.next, self.values, self.parents, self.best, self.o)]

    def rows_in_cache(self, past):
        """[row][keys, values][token][channels] of what each row's table holds."""
        out = []
        for r in range(self.rows):
            n = int(past[r])
            ends, zero = torch.tensor([0, n], dtype=torch.int32, device=sv.DEV), torch.zeros(1, dtype=torch.int32, device=sv.DEV)
            b = self.ctx.paged_batch(1, n, sv.ptr(ends), sv.ptr(zero), sv.ptr(self.table[r]), SLOTS // PAGE)
            kv = torch.zeros(2, n, KV_HEADS * DIM, device=sv.DEV)
            self.ctx.paged_kv_read_device(self.cache, b, sv.ptr(kv[0]), sv.ptr(kv[1]), stream=sv.stream())
            torch.cuda.synchronize()
            out.append(kv.cpu())
        return out

    def close(self):
        torch.cuda.synchronize()
        self.ctx.paged_kv_destroy(self.cache)


def check_selected(gen, scores):
    got = [x.cpu() for x in (gen.values, gen.parents, gen.best, *(y.reshape(gen.seqs, BEAMS) for y in gen.next))]
    check_select(got, select_reference(gen.logits.cpu(), scores.reshape(gen.seqs, BEAMS), BEAMS, VOCAB, COUNT, [END]), VOCAB)


def check_advanced(gen, before, added):
    want, copies = advance_reference(BEAMS, PAGE, added, gen.next[1].cpu(), *before[:3], gen.next[2].cpu(), before[3])
    for name, x, y in zip(("past", "table", "spare", "history"), gen.out, want):
        assert torch.equal(x.cpu(), y), name
    return copies


def heads_close(got, k, v, q, past, dtype):
    want, lim = sv.attention_rows(torch.stack((k, v)), q, [past], [1], KV_HEADS, HEADS, DIM, SCALE, dtype, "decode")
    off = (got.double().reshape(1, HEADS, DIM) - want).square().sum(-1).sqrt()
    return bool((off <= lim).all())


@pytest.mark.parametrize("dtype,lengths", [("f32", [37, 18]), ("bf16", [15, 33, 2]), ("f16", [9])])
def test_prompts_and_beams_together(gpu_ctx, dtype, lengths):
    gen = Generation(gpu_ctx, lengths, dtype, 5)
    n = sum(lengths)
    try:
        before = [x.cpu() for x in (gen.past, gen.table, gen.spare, gen.history)]
        scores = gen.scores.cpu()
        gen.take_prompts()
        torch.cuda.synchronize()
        for x, y, heads, w in ((gen.pq, gen.pqr, HEADS, gen.norms[0]), (gen.pk, gen.pkr, KV_HEADS, gen.norms[1])):
            want, size = rotary_reference(x.cpu(), heads, DIM, DIM, gen.prompt_at, SECTIONS, True, w.cpu(), THETA, EPS)
            check_rotary(y.cpu(), want, size, dtype)
        check_prompt(gen.po, gen.pqr.cpu(), gen.pkr.cpu(), gen.pv.cpu(), lengths, HEADS, KV_HEADS, DIM, SCALE, dtype)
        check_selected(gen, scores)
        check_advanced(gen, before, 0)
        gen.take_over()
        # keys and values that each row's cache was given, token by token
        given = []
        for s, m in enumerate(lengths):
            at = sum(lengths[:s])
            given += [[x[at:at + m].cpu() for x in (gen.pkr, gen.pv)] for _ in range(BEAMS)]
        copied = 0
        for _ in range(20):
            before = [x.cpu() for x in (gen.past, gen.table, gen.spare, gen.history)]
            scores, past = gen.scores.cpu(), gen.past.cpu()
            gen.step()
            torch.cuda.synchronize()
            at = past.repeat(3, 1)
            for x, y, heads, w in ((gen.q, gen.qr, HEADS, gen.norms[0]), (gen.k, gen.kr, KV_HEADS, gen.norms[1])):
                want, size = rotary_reference(x.cpu(), heads, DIM, DIM, at, SECTIONS, True, w.cpu(), THETA, EPS)
                check_rotary(y.cpu(), want, size, dtype)
            given = [[torch.cat((a, b[r:r + 1].cpu())) for a, b in zip(given[r], (gen.kr, gen.v))] for r in range(gen.rows)]
            check_selected(gen, scores)
            copied += len(check_advanced(gen, before, 1))
            o, qr, parents = gen.o.cpu(), gen.qr.cpu(), gen.next[1].cpu().tolist()
            kept = given
            gen.take_over()
            given = [list(given[p if p >= 0 else r]) for r, p in enumerate(parents)]
            held = gen.rows_in_cache(gen.past.cpu())
            for r in range(gen.rows):
                # to the bit what a cache holds to which the row's keys and values are given at once
                fresh = sv.Cache(gpu_ctx, [SLOTS], KV_HEADS, DIM)
                try:
                    m = given[r][0].shape[0]
                    b = fresh.batch([0], [m])
                    fresh.append(b, given[r][0].to(sv.DEV), given[r][1].to(sv.DEV), dtype)
                    kv = fresh.read(b)
                finally:
                    fresh.close()
                assert torch.equal(held[r], kv), r
                if parents[r] >= 0:
                    p = parents[r]
                    assert kept[p][0].shape[0] == m
                    assert heads_close(o[p], kv[0], kv[1], qr[p:p + 1], m - 1, dtype), (r, p)
        assert copied > 0                                        # beams that go on from the same one
    finally:
        gen.close()


def test_captured_steps_replay(gpu_ctx):
    """A step captured once and replayed, its own state carried on between: what eager steps give."""
    gen, eager = (Generation(gpu_ctx, [21, 14], "bf16", 8) for _ in range(2))
    try:
        for x in (gen, eager):
            x.take_prompts()
            x.take_over()
        keep = [x.clone() for x in (gen.past, gen.table, gen.spare, gen.history, gen.scores, gen.tokens)]
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            gen.step()                               # what a first call sets up is set up
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gen.step()
        for x, y in zip((gen.past, gen.table, gen.spare, gen.history, gen.scores, gen.tokens), keep):
            assert torch.equal(x, y)                 # a step leaves its state as it was
        for i in range(20):
            graph.replay()
            eager.step()
            torch.cuda.synchronize()
            for a, b in zip(gen.state(), eager.state()):
                assert torch.equal(a, b), i
            gen.take_over()
            eager.take_over()
        for a, b in zip(gen.rows_in_cache(gen.past.cpu()), eager.rows_in_cache(eager.past.cpu())):
            assert torch.equal(a, b)
    finally:
        gen.close()
        eager.close()


def test_two_at_once(gpu_ctx):
    """Two of them, on streams of their own, as each alone."""
    def alone(lengths, dtype, seed, steps):
        gen = Generation(gpu_ctx, lengths, dtype, seed)
        try:
            gen.take_prompts()
            gen.take_over()
            out = []
            for _ in range(steps):
                gen.step()
                torch.cuda.synchronize()
                out.append(gen.state())
                gen.take_over()
            return out
        finally:
            gen.close()
    cases = [([40, 3], "f32", 1), ([17, 30, 26], "bf16", 2)]
    want = [alone(*c, 8) for c in cases]
    gens, streams = [Generation(gpu_ctx, *c) for c in cases], [torch.cuda.Stream() for _ in cases]
    try:
        torch.cuda.synchronize()
        for g, s in zip(gens, streams):
            with torch.cuda.stream(s):
                g.take_prompts()
        torch.cuda.synchronize()
        for g in gens:
            g.take_over()
        for i in range(8):
            for g, s in zip(gens, streams):
                with torch.cuda.stream(s):
                    g.step()
            torch.cuda.synchronize()
            for g, w in zip(gens, want):
                for a, b in zip(g.state(), w[i]):
                    assert torch.equal(a, b), i
            for g in gens:
                g.take_over()
    finally:
        for g in gens:
            g.close()


def test_more_than_a_launch_counts(gpu_ctx):
    """A launch has less than 2^32 threads: more are refused on the host, before anything is read."""
    far = lambda i: (1 << 44) + (i << 42)  # noqa: E731
    b = Beams(gpu_ctx, 1, 4, 16, 20)
    try:
        calls = [
            (gpu_ctx.rotary_device, (gpu_ctx.rotary_request(2 ** 31 - 1, "f16", DIM, DIM, THETA, far(0), query_heads=2, q_ptr=far(1),
                                                            q_out_ptr=far(2)),)),
            (gpu_ctx.prompt_attention_device, (gpu_ctx.prompt_attention_request(1, 1 << 26, far(0), "bf16", 32, 8, 1, far(1), far(2), far(3), far(4),
                                                                                1.0),)),
            (gpu_ctx.paged_kv_beam_advance_device, (b.caches * 128, gpu_ctx.beam_advance_request(16383, 4, 16, 2, *(far(i) for i in range(7))))),
        ]
        for call, args in calls:
            with pytest.raises(abi.AbiError) as e:
                call(*args, stream=sv.stream())
            assert e.value.status == -5, call
        torch.cuda.synchronize()
    finally:
        b.close()
