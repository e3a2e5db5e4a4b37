"""The operators of a batched serving step together, as a server runs them
around the framework's projections: every stage against its definition, on
streams of the caller's, two at once, and captured and replayed with batches
that change on the device."""
import numpy as np
import pytest
import torch

import serving as sv
from parity import gemv_close
from qwanto_amd import synth
from test_gpu_logits import check as check_logits
from test_gpu_logits import reference as logits_reference
from test_gpu_norm import check as check_norm
from test_gpu_paged import check_cached
from test_gpu_paged import reference as attention_reference

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV_HEADS, DIM, VOCAB, ROWS, EPS = 256, 4, 2, 64, 1000, 16, 1e-6
SCALE = DIM ** -0.5


class Step:
    """One layer's attention half and the head, of a ragged batch of up to ROWS tokens: every buffer
    is made once, what changes from step to step is on the device."""

    def __init__(self, ctx, weights, slots):
        self.ctx, self.w = ctx, weights
        self.cache = sv.Cache(ctx, slots, KV_HEADS, DIM, rope=DIM)
        dev = sv.DEV
        f = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
        i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
        b = lambda n: torch.zeros(n, dtype=torch.uint8, device=dev)  # noqa: E731
        n = len(slots)
        self.starts, self.past = i(n + 1), i(n)
        self.x, self.delta, self.h, self.h2 = (f(ROWS, HIDDEN) for _ in range(4))
        self.q8, self.s = torch.zeros(ROWS, HIDDEN, dtype=torch.int8, device=dev), f(ROWS)
        self.q8b, self.sb = torch.zeros_like(self.q8), f(ROWS)
        self.q8o, self.so = torch.zeros_like(self.q8), f(ROWS)
        self.y, self.yb = f(ROWS, HIDDEN), f(ROWS, HIDDEN)
        self.q, self.qr, self.k, self.v = f(ROWS, HEADS * DIM), f(ROWS, HEADS * DIM), f(ROWS, KV_HEADS * DIM), f(ROWS, KV_HEADS * DIM)
        self.o, self.d, self.raw, self.out = f(ROWS, HEADS * DIM), f(ROWS, HIDDEN), f(ROWS, VOCAB), f(ROWS, VOCAB)
        self.ids = i(ROWS)
        self.history, self.history_starts, self.prompts = i(ROWS * 30), i(ROWS + 1), i(ROWS)
        self.history[:] = -1
        self.rep, self.pres, self.freq = f(ROWS) + 1.3, f(ROWS) + 0.25, f(ROWS) + 0.125
        self.image = b(ctx.mfma_image_bytes(weights["q"]))
        self.image_o = b(ctx.mfma_image_bytes(weights["o"]))
        self.image_head = b(ctx.mfma_image_bytes(weights["head"]))
        p = sv.ptr
        self.batch = ctx.paged_batch(n, ROWS, p(self.starts), p(self.past), p(self.cache.table), self.cache.table.shape[1])
        self.norm1 = ctx.norm_request(ROWS, HIDDEN, "f32", p(self.x), p(weights["norm1"]), EPS, residual_ptr=p(self.delta),
                                      residual_out_ptr=p(self.h), y_ptr=p(self.y), q8_ptr=p(self.q8), scales_ptr=p(self.s))
        self.app = ctx.paged_append_request(self.batch, "f32", p(self.k), p(self.v), q_ptr=p(self.q), q_out_ptr=p(self.qr),
                                            query_heads=HEADS)
        self.att = ctx.paged_attention_request(self.batch, "f32", HEADS, p(self.qr), p(self.o), SCALE)
        self.work = b(ctx.paged_attention_workspace_bytes(self.cache.h, self.att))
        self.att.workspace = p(self.work)
        self.norm2 = ctx.norm_request(ROWS, HIDDEN, "f32", p(self.d), p(weights["norm2"]), EPS, residual_ptr=p(self.h),
                                      residual_out_ptr=p(self.h2), y_ptr=p(self.yb), q8_ptr=p(self.q8b), scales_ptr=p(self.sb))
        self.lwork = b(ctx.logits_workspace_bytes(ROWS, VOCAB))
        self.logits = ctx.logits_request(ROWS, VOCAB, "f32", p(self.raw), p(self.out), history_ptr=p(self.history),
                                         history_starts_ptr=p(self.history_starts), history_capacity=self.history.numel(),
                                         prompt_counts_ptr=p(self.prompts), repetition_ptr=p(self.rep), presence_ptr=p(self.pres),
                                         frequency_ptr=p(self.freq), ids_ptr=p(self.ids), workspace_ptr=p(self.lwork))

    def run(self):
        ctx, w, p, s = self.ctx, self.w, sv.ptr, sv.stream()
        ctx.norm_quantize_device(self.norm1, stream=s)
        ctx.mfma_image_device(w["q"], p(self.q8), ROWS, HIDDEN, p(self.image), stream=s)
        for name, out in (("q", self.q), ("k", self.k), ("v", self.v)):
            ctx.gemm_mfma_device(w[name], p(self.image), p(self.s), p(out), ROWS, stream=s)
        ctx.paged_kv_append_device(self.cache.h, self.app, stream=s)
        ctx.paged_kv_attention_device(self.cache.h, self.att, stream=s)
        ctx.quantize_device(p(self.o), ROWS, HIDDEN, HIDDEN, p(self.q8o), HIDDEN, p(self.so), stream=s)
        ctx.mfma_image_device(w["o"], p(self.q8o), ROWS, HIDDEN, p(self.image_o), stream=s)
        ctx.gemm_mfma_device(w["o"], p(self.image_o), p(self.so), p(self.d), ROWS, stream=s)
        ctx.norm_quantize_device(self.norm2, stream=s)
        ctx.mfma_image_device(w["head"], p(self.q8b), ROWS, HIDDEN, p(self.image_head), stream=s)
        ctx.gemm_mfma_device(w["head"], p(self.image_head), p(self.sb), p(self.raw), ROWS, stream=s)
        ctx.logits_process_device(self.logits, stream=s)

    def set(self, seed, past, new):
        """The next batch, on the device; the same seed, the same step."""
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        assert starts[-1] <= ROWS
        g = sv.gen(seed)
        x, delta = sv.normal(g, ROWS, HIDDEN), 0.3 * sv.normal(g, ROWS, HIDDEN)
        hist = [torch.randint(0, VOCAB, (1 + (7 * r + seed) % 30,), generator=g, dtype=torch.int32) for r in range(ROWS)]
        hs = [0]
        for v in hist:
            hs.append(hs[-1] + len(v))
        flat = torch.cat(hist)
        self.x.copy_(x)
        self.delta.copy_(delta)
        self.starts.copy_(torch.tensor(starts, dtype=torch.int32))
        self.past.copy_(torch.tensor(past, dtype=torch.int32))
        self.history[:len(flat)].copy_(flat)
        self.history_starts.copy_(torch.tensor(hs, dtype=torch.int32))
        self.prompts.copy_(torch.tensor([len(v) // 2 for v in hist], dtype=torch.int32))
        return x, delta, hist

    def results(self):
        names = ("h", "y", "q8", "s", "q", "qr", "k", "v", "o", "d", "h2", "yb", "q8b", "sb", "raw", "out", "ids")
        return {n: getattr(self, n).cpu() for n in names}

    def close(self):
        self.cache.close()


@pytest.fixture(scope="module")
def weights(gpu_ctx):
    rng = np.random.default_rng(5)
    shapes = dict(q=(HEADS * DIM, HIDDEN), k=(KV_HEADS * DIM, HIDDEN), v=(KV_HEADS * DIM, HIDDEN), o=(HIDDEN, HEADS * DIM),
                  head=(VOCAB, HIDDEN))
    w = {n: gpu_ctx.upload(synth.q4_0_weights(rng, *s, std=0.2), "q4_0", *s) for n, s in shapes.items()}
    held = list(w.values())
    g = sv.gen(6)
    w["norm1"], w["norm2"] = ((1 + 0.2 * sv.normal(g, HIDDEN)).to(sv.DEV) for _ in range(2))
    yield w
    torch.cuda.synchronize()
    for h in held:
        gpu_ctx.release(h)


def projected(ctx, w, q8, s, rows):
    return torch.from_numpy(ctx.gemm(w, q8.numpy(), rows, q8.shape[1], scales=s.numpy()))


def same(a, b, rows):
    """The batch's rows of two runs are alike to the bit."""
    return [n for n in a if not torch.equal(a[n][:rows], b[n][:rows])]


def check_step(step, past, new, inputs, cached):
    """Every stage of the step against its definition, from what the stage before it left; `cached`
    holds the keys and values of each sequence so far."""
    ctx, w, r = step.ctx, step.w, step.results()
    x, delta, hist = inputs
    rows = sum(new)
    check_norm(r["h"], r["y"], r["q8"], r["s"], x, delta, w["norm1"].cpu(), "f32", EPS)
    for n in ("q", "k", "v"):
        ok, worst = gemv_close(r[n].numpy(), projected(ctx, w[n], r["q8"], r["s"], r[n].shape[1]).numpy())
        assert ok, (n, worst)
    pos = torch.tensor([p + i for p, n in zip(past, new) for i in range(n)])
    kv = step.cache.read(step.batch)
    kr = sv.rotate(r["k"][:rows].reshape(rows, KV_HEADS, DIM), pos, DIM, step.cache.theta).float()
    check_cached(kv[0, :rows].reshape(rows, KV_HEADS, DIM), kr, True)
    check_cached(kv[1, :rows].reshape(rows, KV_HEADS, DIM), r["v"][:rows].reshape(rows, KV_HEADS, DIM), False)
    qr = sv.rotate(r["q"][:rows].reshape(rows, HEADS, DIM), pos, DIM, step.cache.theta).reshape(rows, -1)
    assert bool(((r["qr"][:rows].double() - qr).abs() <= 2.0 ** -23 * qr.abs() + 2.0 ** -24).all())
    at = 0
    for s, n in enumerate(new):
        cached[s] = torch.cat([cached[s], kv[:, at:at + n]], dim=1)
        at += n
    want, tol = attention_reference(torch.cat(cached, dim=1), r["qr"][:rows], past, new, KV_HEADS, HEADS, DIM, SCALE, "f32")
    assert bool(((r["o"][:rows].double() - want).abs() <= tol).all())
    check_norm(r["h2"], r["yb"], r["q8b"], r["sb"], r["d"], r["h"], w["norm2"].cpu(), "f32", EPS)
    ok, worst = gemv_close(r["raw"].numpy(), projected(ctx, w["head"], r["q8b"], r["sb"], VOCAB).numpy())
    assert ok, worst
    none = [[] for _ in range(ROWS)]
    f32 = lambda t: t.cpu().tolist()  # noqa: E731
    want = logits_reference(r["raw"], [h.tolist() for h in hist], [len(h) // 2 for h in hist], f32(step.rep), f32(step.pres),
                            f32(step.freq), none, [None] * ROWS)
    check_logits((r["out"], r["ids"].tolist()), want, r["raw"])


# prompts, then single tokens, drafted ones, a sequence that pauses and one that comes late
BATCHES = [([0, 0, 0, 0], [9, 4, 3, 0]), ([9, 4, 3, 0], [1, 1, 0, 12]), ([10, 5, 3, 12], [1, 5, 1, 1]), ([11, 10, 4, 13], [1, 1, 1, 1]),
           ([12, 11, 5, 14], [13, 1, 1, 1])]


def test_a_step_together(gpu_ctx, weights):
    step = Step(gpu_ctx, weights, [64] * 4)
    try:
        cached = [torch.zeros(2, 0, KV_HEADS * DIM) for _ in range(4)]
        for i, (past, new) in enumerate(BATCHES):
            inputs = step.set(i, past, new)
            step.run()
            torch.cuda.synchronize()
            check_step(step, past, new, inputs, cached)
    finally:
        step.close()


def test_a_captured_step_replays(gpu_ctx, weights):
    """Captured once, replayed with other batches: each replay equals the eager step, which runs on a
    cache of its own in between."""
    step, eager = Step(gpu_ctx, weights, [64] * 4), Step(gpu_ctx, weights, [64] * 4)
    try:
        step.set(99, [0] * 4, [1] * 4)
        step.run()                                   # what a first call sets up is set up
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step.run()
        for i, (past, new) in enumerate(BATCHES):
            step.set(i, past, new)
            graph.replay()
            eager.set(i, past, new)
            eager.run()
            torch.cuda.synchronize()
            assert not (d := same(step.results(), eager.results(), sum(new))), (i, d)
            graph.replay()                           # the same step again
            torch.cuda.synchronize()
            assert not (d := same(step.results(), eager.results(), sum(new))), (i, d)
    finally:
        step.close()
        eager.close()


def test_two_steps_at_once(gpu_ctx, weights):
    """Two batches on two streams, each with its own cache and workspaces, equal what they are one
    after the other on the default stream."""
    steps = [Step(gpu_ctx, weights, [64] * 4) for _ in range(4)]
    try:
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for i, (past, new) in enumerate(BATCHES):
            for j, s in enumerate(steps):
                s.set(10 * i + j % 2, past, new)
            steps[0].run()
            steps[1].run()
            for st, s in zip(streams, steps[2:]):
                st.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(st):
                    s.run()
            torch.cuda.synchronize()
            for j in range(2):
                assert not (d := same(steps[j].results(), steps[2 + j].results(), sum(new))), (i, j, d)
    finally:
        for s in steps:
            s.close()


@pytest.mark.parametrize("dtype,new,slots", [("f16", 1, 5000), ("bf16", 90, 3000), ("f32", 3, 700)])
def test_readers_of_one_cache_at_once(gpu_ctx, dtype, new, slots):
    """Calls that read one cache on two streams, with workspaces of their own; and one workspace for
    calls that follow each other."""
    c = sv.Cache(gpu_ctx, [slots], 2, 64)
    try:
        g = sv.gen(slots)
        k, v = sv.normal(g, slots, 128).to(sv.DEV), sv.normal(g, slots, 128).to(sv.DEV)
        c.append(c.batch([0], [slots]), k, v, "f32")
        b = c.batch([slots - new], [new])
        qs = [sv.normal(g, new, 8 * 64).to(sv.DTYPES[dtype]).to(sv.DEV) for _ in range(6)]
        outs = [torch.zeros_like(q) for q in qs]
        reqs = [c.request(b, q, o, dtype, 8, 0.125) for q, o in zip(qs, outs)]
        for r in reqs:
            gpu_ctx.paged_kv_attention_device(c.h, r, stream=sv.stream())
        torch.cuda.synchronize()
        want = [o.clone() for o in outs]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for i, r in enumerate(reqs):
            r.workspace = reqs[i % 2].workspace                  # one of each stream's
        for o in outs:
            o.zero_()
        for i, r in enumerate(reqs):
            streams[i % 2].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(streams[i % 2]):
                gpu_ctx.paged_kv_attention_device(c.h, r, stream=sv.stream())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    finally:
        c.close()


def test_a_page_that_comes_twice(gpu_ctx):
    """A table may name a page twice: its tokens are attended to at both places."""
    hk, d, heads = 2, 64, 4
    c = sv.Cache(gpu_ctx, [48], hk, d)
    try:
        g = sv.gen(3)
        k, v = sv.normal(g, 48, hk * d), sv.normal(g, 48, hk * d)
        c.append(c.batch([0], [48]), k.to(sv.DEV), v.to(sv.DEV), "f32")
        order = [0, 1, 1, 2, 0, 1]
        table = c.table[:, order].contiguous()
        slots = 16 * len(order)
        b = c.batch([0], [slots], table=table)
        kv = c.read(b)
        q = sv.normal(g, 2, heads * d)
        out = torch.zeros(2, heads * d, device=sv.DEV)
        c.attend(c.batch([slots - 2], [2], table=table), q.to(sv.DEV), out, "f32", heads, 0.125)
        want, tol = attention_reference(kv, q, [slots - 2], [2], hk, heads, d, 0.125, "f32")
        assert bool(((out.cpu().double() - want).abs() <= tol).all())
    finally:
        c.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prompt_attention_captured(gpu_ctx, dtype):
    """The kernels of many rows, their contexts cut and joined, recorded once and replayed with other
    lengths, rows and pages."""
    slots = [3000, 700, 400]
    c = sv.Cache(gpu_ctx, slots, 2, 128)
    try:
        g = sv.gen(8)
        k, v = sv.normal(g, sum(slots), 256).to(sv.DEV), sv.normal(g, sum(slots), 256).to(sv.DEV)
        c.append(c.batch([0, 0, 0], slots), k, v, "f32")
        rows = 128
        q = sv.normal(g, rows, 8 * 128).to(sv.DTYPES[dtype]).to(sv.DEV)
        out, want = torch.zeros_like(q), torch.zeros_like(q)
        b = c.batch([0, 0, 0], [rows, 0, 0])
        r, e = c.request(b, q, out, dtype, 8, 0.1), c.request(b, q, want, dtype, 8, 0.1)
        starts, past, table = (torch.zeros(4, dtype=torch.int32, device=sv.DEV), torch.zeros(3, dtype=torch.int32, device=sv.DEV),
                               c.table.clone())
        b.starts, b.past, b.page_table = sv.ptr(starts), sv.ptr(past), sv.ptr(table)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gpu_ctx.paged_kv_attention_device(c.h, r, stream=sv.stream())
        for ps, ns, flip in (([2900, 600, 300], [100, 20, 8], False), ([0, 0, 0], [128, 0, 0], False), ([10, 650, 390], [1, 50, 10], True),
                             ([2872, 0, 0], [128, 0, 0], False), ([5, 5, 5], [40, 40, 40], True)):
            starts.copy_(torch.tensor([0, ns[0], ns[0] + ns[1], sum(ns)], dtype=torch.int32))
            past.copy_(torch.tensor(ps, dtype=torch.int32))
            table.copy_(c.table.flip(0) if flip else c.table)
            for o in (out, want):
                o.fill_(2.0)
            graph.replay()
            gpu_ctx.paged_kv_attention_device(c.h, e, stream=sv.stream())
            torch.cuda.synchronize()
            assert torch.equal(out, want), (ps, ns)
            assert bool((out[sum(ns):] == 2.0).all())
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), (ps, ns)
    finally:
        c.close()
