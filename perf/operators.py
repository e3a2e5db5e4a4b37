"""The operators of a batched serving step, as cases that can be timed and checked.

Between the quantized projections of a step over many sequences lie four
operators, each reached through qwanto_amd.abi (device pointers):

op "norm"       the residual's addition, RMSNorm, and the per-token int8
                quantization the projections read.
op "append"     new keys and values into a paged cache held in 4 bits, the
                keys (and the queries) rotated for their positions on the way.
op "attention"  causal attention of each sequence's new tokens over its pages
                of that cache.
op "logits"     penalties for repeated tokens, biases and grammar masks on the
                logits, and the greedy id of each row.

With ``own`` false, run() computes them in elementary torch operations; with
``own`` true, it makes the library's calls.

Batches are ragged: sequence s has past[s] cached tokens and the new rows
starts[s] .. starts[s + 1]; rows behind the last sequence belong to none.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"

# Layer shapes of the two models the repository's benchmark decodes.
QWEN2_1P5B = dict(heads=12, kv_heads=2, head_dim=128)
QWEN3_4B = dict(heads=32, kv_heads=8, head_dim=128)
VOCAB = 151936
ROPE_THETA = 1.0e6
EPS = 1.0e-6
GROUP = 64          # channels of a token and head that share a scale and a minimum
F16_MAX = 65504.0

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ------------------------------------------------------------------


def listed():
    return [
        # one decoded token of a small model: all latency
        dict(name="norm_token_f32", op="norm", dtype="f32", tokens=1, cols=1536, pad=0),
        # a decode batch of sequences, rows strided as in a wider buffer
        dict(name="norm_61_tokens_bf16", op="norm", dtype="bf16", tokens=61, cols=2560, pad=64),
        # a long prompt's rows: bytes
        dict(name="norm_4099_tokens_f32", op="norm", dtype="f32", tokens=4099, cols=2560, pad=0),
        # one token of one short chat
        dict(name="append_token_f32", op="append", dtype="f32", seqs=1, past_max=40, new_max=1, page=16, mix=1, rows_pad=0,
             **QWEN2_1P5B),
        # a decode batch: one token of each sequence, far and near positions
        dict(name="append_61_tokens_bf16", op="append", dtype="bf16", seqs=61, past_max=40000, new_max=1, page=16, mix=2,
             rows_pad=3, **QWEN3_4B),
        # prompts of several users at once
        dict(name="append_prompts_bf16", op="append", dtype="bf16", seqs=5, past_max=333, new_max=4000, page=64, mix=3,
             rows_pad=0, **QWEN3_4B),
        # one token of one short chat
        dict(name="attention_token_f32", op="attention", dtype="f32", seqs=1, past_max=333, new_max=1, page=16, mix=4,
             rows_pad=0, **QWEN2_1P5B),
        # an ordinary decode batch, contexts from a few tokens to thousands
        dict(name="attention_61_tokens_bf16", op="attention", dtype="bf16", seqs=61, past_max=8191, new_max=1, page=16, mix=5,
             rows_pad=3, **QWEN3_4B),
        # few sequences with very long contexts
        dict(name="attention_long_f16", op="attention", dtype="f16", seqs=2, past_max=131000, new_max=1, page=64, mix=6,
             rows_pad=0, **QWEN3_4B),
        # prompts in chunks behind what is cached
        dict(name="attention_prompts_bf16", op="attention", dtype="bf16", seqs=4, past_max=2048, new_max=512, page=32, mix=7,
             rows_pad=0, **QWEN3_4B),
        # one sequence's next token
        dict(name="logits_token_f32", op="logits", dtype="f32", rows=1, vocab=VOCAB, history=500, biases=20, mask=False, mix=8),
        # a batch of sequences, some under a grammar
        dict(name="logits_61_rows_f32", op="logits", dtype="f32", rows=61, vocab=VOCAB, history=4000, biases=300, mask=True,
             mix=9),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges the listed ones stand for: rows of 64 to 9728
    channels, 1 to 4096 tokens, head dims 32 to 256, contexts of 1 to 131072
    tokens, pages of 16 to 128, vocabularies of 1000 to 152000."""
    op = rng.choice(["norm", "append", "attention", "attention", "logits"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "norm":
        cols = _log_int(rng, 64, 9728)
        return dict(op=op, dtype=dtype, tokens=_log_int(rng, 1, max(1, min(4096, 10_400_000 // cols))), cols=cols,
                    pad=rng.choice([0, 0, 1, 8, 64]))
    if op == "logits":
        vocab = _log_int(rng, 1000, VOCAB)
        return dict(op=op, dtype=dtype, rows=_log_int(rng, 1, max(1, min(61, 9_000_000 // vocab))), vocab=vocab,
                    history=_log_int(rng, 1, 4000), biases=rng.choice([0, _log_int(rng, 1, 300)]), mask=rng.random() < 0.5,
                    mix=rng.randrange(1 << 20))
    kv = rng.choice([1, 2, 4, 8])
    case = dict(op=op, dtype=dtype, kv_heads=kv, heads=kv * rng.choice([1, 2, 3, 4, 6, 8]),
                head_dim=rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256]), page=rng.choice([16, 16, 32, 64, 128]),
                rows_pad=rng.choice([0, 0, 1, 7]), mix=rng.randrange(1 << 20))
    if op == "append":
        case.update(seqs=_log_int(rng, 1, 64), past_max=_log_int(rng, 1, 100000))
        case["new_max"] = rng.choice([1, _log_int(rng, 1, 4000 // case["seqs"])])
        return case
    if rng.random() < 0.6:
        # single tokens, or a few drafted ones
        case.update(new_max=rng.choice([1, 1, rng.randint(2, 8)]), past_max=_log_int(rng, 1, 131000))
        case["seqs"] = _log_int(rng, 1, max(1, min(64, 262000 // case["past_max"])))
    else:
        case.update(seqs=rng.randint(1, 4), new_max=_log_int(rng, 9, 512), past_max=_log_int(rng, 1, 2048))
    # no dearer than the largest listed ones
    while work(case)["flops"] > 4.0e10 or work(case)["bytes"] > 2.9e8:
        case["past_max"] = max(1, case["past_max"] // 2)
        case["new_max"] = max(1, case["new_max"] * 3 // 4)
    return case


def _lengths(case):
    """(past, new) tokens of each sequence: the first the longest, the others spread over the range."""
    rng = random.Random(case["mix"])
    past = [case["past_max"]] + [_log_int(rng, 1, case["past_max"]) if rng.random() < 0.9 else 0 for _ in range(case["seqs"] - 1)]
    new = [case["new_max"]] + [_log_int(rng, 1, case["new_max"]) if rng.random() < 0.95 else 0 for _ in range(case["seqs"] - 1)]
    return past, new


def work(case):
    op, size = case["op"], SIZE[case["dtype"]]
    if op == "norm":
        n = case["tokens"] * case["cols"]
        return {"bytes": n * (3 * size + 1) + case["cols"] * 4 + case["tokens"] * 4, "flops": n * 8}
    if op == "logits":
        n = case["rows"] * case["vocab"]
        extra = case["rows"] * (case["history"] * 4 + case["biases"] * 8 + 20)
        return {"bytes": n * 2 * size + (n // 8 if case["mask"] else 0) + extra, "flops": n * 2}
    past, new = _lengths(case)
    groups = -(-case["head_dim"] // GROUP)
    token = case["kv_heads"] * (case["head_dim"] + 8 * groups)     # K and V of one token in 4 bits
    q = sum(new) * case["heads"] * case["head_dim"]
    if op == "append":
        kv = sum(new) * case["kv_heads"] * case["head_dim"]
        # keys, values and queries read; queries and codes written; the codes read back as fp32 values
        return {"bytes": size * (2 * kv + 2 * q) + 2 * sum(new) * token + 8 * kv, "flops": 6 * q + 20 * kv}
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))
    return {"bytes": sum(p + n for p, n in zip(past, new) if n) * token + 2 * size * q,
            "flops": 4 * pairs * case["heads"] * case["head_dim"]}


# ---- inputs ---------------------------------------------------------------------


def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + salt)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _norm_inputs(case, seed):
    g = _gen(seed, 11)
    t, c, stride = case["tokens"], case["cols"], case["cols"] + case["pad"]
    dt = DTYPES[case["dtype"]]
    # a layer's output next to a residual stream with a few large channels
    big = torch.where(torch.rand(stride, generator=g, device=DEV) < 0.005, 12.0, 1.0)
    x = (0.5 * _normal(g, t, stride)).to(dt)[:, :c]
    r = (1.5 * _normal(g, t, stride) * big).to(dt)[:, :c]
    return x, r, 1.0 + 0.2 * _normal(g, c)


def _batch(case):
    past, new = _lengths(case)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    need = [-(-(p + n) // case["page"]) for p, n in zip(past, new)]
    return past, new, starts, need


def _kv_inputs(case, seed, tokens, g=None):
    """Keys with channels of their own scale and offset, values, in the case's type."""
    g = g or _gen(seed, 12)
    c, dt = case["kv_heads"] * case["head_dim"], DTYPES[case["dtype"]]
    scale = 0.3 + 1.2 * torch.rand(c, generator=g, device=DEV)
    offset = torch.where(torch.rand(c, generator=g, device=DEV) < 0.05, 4.0, 0.3) * _normal(g, c)
    k = (_normal(g, tokens, c) * scale + offset).to(dt)
    v = (_normal(g, tokens, c) * scale.flip(0)).to(dt)
    return k, v


def _query(case, seed, tokens):
    return (1.2 * _normal(_gen(seed, 13), tokens, case["heads"] * case["head_dim"])).to(DTYPES[case["dtype"]])


def _table(case, seed, need):
    """A pool a tenth larger than needed, its pages handed out in no order; -1 behind a sequence's last page."""
    pages = sum(need) + max(1, sum(need) // 10)
    order = torch.randperm(pages, generator=_gen(seed, 14), device=DEV).to(torch.int32)
    width = max(need)
    table = torch.full((len(need), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return pages, table


def _logits_inputs(case, seed):
    g = _gen(seed, 15)
    rng = random.Random(case["mix"])
    rows, vocab = case["rows"], case["vocab"]
    x = (2.5 * _normal(g, rows, vocab)).to(DTYPES[case["dtype"]])
    lens = [case["history"]] + [_log_int(rng, 1, case["history"]) for _ in range(rows - 1)]
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    # a few tokens come often, most once; ids of -1 are padding
    u = torch.rand(starts[-1], generator=g, device=DEV)
    history = (u ** 4 * vocab).to(torch.int32).clamp_(0, vocab - 1)
    history = torch.where(torch.rand(starts[-1], generator=g, device=DEV) < 0.01, -1, history).to(torch.int32)
    prompts = torch.tensor([n * rng.randint(0, 4) // 4 for n in lens], dtype=torch.int32, device=DEV)
    per_row = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=g, device=DEV)  # noqa: E731
    blens = [case["biases"]] + [rng.randint(0, case["biases"]) for _ in range(rows - 1)]
    bstarts = [0]
    for n in blens:
        bstarts.append(bstarts[-1] + n)
    btokens = torch.randint(0, vocab, (bstarts[-1],), generator=g, device=DEV, dtype=torch.int32)
    bvalues = 3.0 * _normal(g, bstarts[-1])
    words = -(-vocab // 32)
    mask = index = None
    if case["mask"]:
        # two rows of three under a grammar: from a handful of tokens to most of them
        n = max(1, rows - rows // 3)
        share = 0.001 + 0.95 * torch.rand(n, 1, 1, generator=g, device=DEV) ** 2
        bits = torch.rand(n, words, 32, generator=g, device=DEV) < share
        shift = torch.arange(32, device=DEV, dtype=torch.int64)
        word = (bits.to(torch.int64) << shift).sum(dim=2)
        mask = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)
        index = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
        index[:n] = torch.randperm(n, generator=g, device=DEV).to(torch.int32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(x=x, history=history, starts=i32(starts), prompts=prompts, repetition=per_row(1.0, 1.5), presence=per_row(0.0, 1.0),
                frequency=per_row(0.0, 0.7), btokens=btokens, bvalues=bvalues, bstarts=i32(bstarts), mask=mask, index=index)


class _State:
    """What a program keeps between calls; closes what it opened in the library."""

    def __init__(self, case):
        self.case = case
        self.ctx = None

    def open(self):
        from qwanto_amd import abi
        self.stream = abi.NULL_STREAM
        self.ctx = abi.Context(abi.load(), device=0)
        return self.ctx

    def __del__(self):
        try:
            if self.ctx is not None:
                self.ctx.close()
        except Exception:
            pass


def prepare(case, seed):
    st = _State(case)
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "norm":
        st.x, st.r, st.w = _norm_inputs(case, seed)
        t, c = case["tokens"], case["cols"]
        st.out = torch.empty(t, c, device=DEV, dtype=dt)
        if own:
            st.q8 = torch.empty(t, c, device=DEV, dtype=torch.int8)
            st.scales = torch.empty(t, device=DEV)
            st.req = st.open().norm_request(t, c, case["dtype"], x_ptr=st.x.data_ptr(), x_stride=st.x.stride(0),
                                            residual_ptr=st.r.data_ptr(), residual_stride=st.r.stride(0),
                                            residual_out_ptr=st.out.data_ptr(), norm_ptr=st.w.data_ptr(), eps=EPS,
                                            q8_ptr=st.q8.data_ptr(), scales_ptr=st.scales.data_ptr())
        return st
    if op == "logits":
        st.inp = _logits_inputs(case, seed)
        if own:
            i, ptr = st.inp, lambda t: t.data_ptr() if t is not None else None
            rows, vocab = case["rows"], case["vocab"]
            st.out = torch.empty(rows, vocab, device=DEV, dtype=dt)
            st.ids = torch.empty(rows, device=DEV, dtype=torch.int32)
            ctx = st.open()
            st.work = torch.empty(max(1, ctx.logits_workspace_bytes(rows, vocab)), device=DEV, dtype=torch.uint8)
            st.req = ctx.logits_request(rows, vocab, case["dtype"], logits_ptr=ptr(i["x"]), out_ptr=ptr(st.out),
                                        history_ptr=ptr(i["history"]), history_starts_ptr=ptr(i["starts"]),
                                        history_capacity=i["history"].numel(), prompt_counts_ptr=ptr(i["prompts"]),
                                        repetition_ptr=ptr(i["repetition"]), presence_ptr=ptr(i["presence"]),
                                        frequency_ptr=ptr(i["frequency"]), bias_tokens_ptr=ptr(i["btokens"]),
                                        bias_values_ptr=ptr(i["bvalues"]), bias_starts_ptr=ptr(i["bstarts"]),
                                        bias_capacity=i["btokens"].numel(), mask_ptr=ptr(i["mask"]),
                                        mask_rows=i["mask"].shape[0] if i["mask"] is not None else 0,
                                        mask_index_ptr=ptr(i["index"]), ids_ptr=ptr(st.ids), workspace_ptr=ptr(st.work))
        return st
    past, new, starts, need = _batch(case)
    rows, hd = starts[-1] + case["rows_pad"], case["head_dim"]
    pages, st.table = _table(case, seed, need)
    st.past = torch.tensor(past, dtype=torch.int32, device=DEV)
    st.starts = torch.tensor(starts, dtype=torch.int32, device=DEV)
    st.total, st.new_max, st.rows = starts[-1], max(new), rows
    st.q = _query(case, seed, rows)
    rope = hd if op == "append" else 0
    if own:
        ctx = st.open()
        st.cache = ctx.paged_kv_create(pages, case["page"], case["kv_heads"], hd, rope_dims=rope, rope_theta=ROPE_THETA)
        st.batch = ctx.paged_batch(case["seqs"], rows, st.starts.data_ptr(), st.past.data_ptr(), st.table.data_ptr(),
                                   st.table.shape[1])
    else:
        half = -(-hd // 2)
        groups = -(-hd // GROUP)
        # the pool as [slot][head]: two codes a byte, (step, minimum) pairs
        st.pool = [(torch.zeros(pages * case["page"], case["kv_heads"], half, dtype=torch.uint8, device=DEV),
                    torch.zeros(pages * case["page"], case["kv_heads"], groups, 2, dtype=torch.float16, device=DEV)) for _ in range(2)]
    if op == "append":
        st.k, st.v = _kv_inputs(case, seed, rows)
        if own:
            c = case["kv_heads"] * hd
            st.q_out = torch.zeros_like(st.q)
            st.kv = torch.zeros(2, rows, c, device=DEV)
            st.req = ctx.paged_append_request(st.batch, case["dtype"], k_ptr=st.k.data_ptr(), v_ptr=st.v.data_ptr(),
                                              q_ptr=st.q.data_ptr(), q_out_ptr=st.q_out.data_ptr(), query_heads=case["heads"])
        return st
    # the whole contexts, new tokens among them, are in the cache
    total = [p + n for p, n in zip(past, new)]
    k, v = _kv_inputs(case, seed, sum(total))
    if own:
        at = torch.tensor([0] + total, dtype=torch.int32, device=DEV).cumsum(0).to(torch.int32)
        zero = torch.zeros(case["seqs"], dtype=torch.int32, device=DEV)
        fill = ctx.paged_batch(case["seqs"], sum(total), at.data_ptr(), zero.data_ptr(), st.table.data_ptr(), st.table.shape[1])
        ctx.paged_kv_append_device(st.cache, ctx.paged_append_request(fill, case["dtype"], k_ptr=k.data_ptr(), v_ptr=v.data_ptr()),
                                   stream=st.stream)
        st.out = torch.zeros_like(st.q)
        st.req = ctx.paged_attention_request(st.batch, case["dtype"], case["heads"], q_ptr=st.q.data_ptr(),
                                             out_ptr=st.out.data_ptr(), scale=hd ** -0.5)
        st.work = torch.empty(max(1, ctx.paged_attention_workspace_bytes(st.cache, st.req)), device=DEV, dtype=torch.uint8)
        st.req.workspace = st.work.data_ptr()
        torch.cuda.synchronize()
    else:
        seq, at = _rows_of(torch.tensor(total, device=DEV), sum(total))
        slot = _slots(case, st.table, seq, at)
        for x, (codes, scales) in zip((k, v), st.pool):
            c, s = _quantize4(x.reshape(-1, case["kv_heads"], hd).float())
            codes[slot], scales[slot] = _pack(c), s
    return st


# ---- the plain forms ------------------------------------------------------------


def _rows_of(counts, total):
    """(sequence, index within it) of each of `total` rows laid one sequence after the other."""
    seq = torch.repeat_interleave(torch.arange(counts.numel(), device=DEV), counts.long(), output_size=total)
    first = torch.cumsum(counts.long(), 0) - counts.long()
    return seq, torch.arange(total, device=DEV) - first[seq]


def _slots(case, table, seq, position):
    return table[seq, position // case["page"]].long() * case["page"] + position % case["page"]


def _quantize4(x):
    """fp32 [..., head_dim] as 4-bit codes and (step, minimum) of each group, as the cache defines them."""
    hd = x.shape[-1]
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).clamp(-F16_MAX, F16_MAX)
    parts = [_quantize_group(x[..., i:i + GROUP]) for i in range(0, hd, GROUP)]
    return torch.cat([p[0] for p in parts], dim=-1), torch.stack([p[1] for p in parts], dim=-2)


def _quantize_group(x):
    lo, hi = x.amin(dim=-1, keepdim=True), x.amax(dim=-1, keepdim=True)
    least = lo.half()
    span = hi - lo
    step = (span / torch.full_like(span, 15.0)).half()
    # next to a border between codes the quotient decides: 64 bits
    t = (x.double() - least.double()) / step.double()
    code = torch.where(step > 0, t.round().clamp(0, 15), torch.zeros_like(t)).to(torch.uint8)
    return code, torch.cat([step, least], dim=-1)


def _pack(codes):
    if codes.shape[-1] % 2:
        codes = torch.nn.functional.pad(codes, (0, 1))
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _values(codes, scales, hd):
    """The fp32 values that packed codes and their (step, minimum) pairs stand for."""
    c = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)[..., :hd].float()
    s = scales.float().repeat_interleave(GROUP, dim=-2)[..., :hd, :]
    return s[..., 0] * c + s[..., 1]


def _rotate(x, position):
    """Half-split rotation of [rows][heads][head_dim], in 64 bits."""
    hd = x.shape[-1]
    half = hd // 2
    freq = ROPE_THETA ** (-2.0 * torch.arange(half, device=DEV, dtype=torch.float64) / hd)
    angle = (position.double()[:, None] * freq)[:, None, :]
    c, s = torch.cos(angle), torch.sin(angle)
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat((a * c - b * s, a * s + b * c), dim=-1)


def _plain_norm(st):
    h = (st.x.float() + st.r.float()).to(st.x.dtype)
    # 64 bits: a code of the quantization hangs on each value
    wide = h.double()
    y = (wide * torch.rsqrt(wide.square().mean(dim=1, keepdim=True) + EPS) * st.w.double()).float()
    amax = y.abs().amax(dim=1, keepdim=True)
    scale = torch.where(amax > 0, amax / torch.full_like(amax, 127.0), torch.ones_like(amax))
    q = (y * (1.0 / scale)).clamp(-127.0, 127.0).round()
    return [h, q * scale, scale[:, 0]]


def _plain_append(st):
    case, hd, kvh = st.case, st.case["head_dim"], st.case["kv_heads"]
    counts = st.starts[1:] - st.starts[:-1]
    seq, at = _rows_of(counts, st.total)
    position = st.past[seq].long() + at
    slot = _slots(case, st.table, seq, position)
    out = []
    q = torch.zeros_like(st.q)
    q[:st.total] = _rotate(st.q[:st.total].reshape(st.total, -1, hd), position).to(st.q.dtype).reshape(st.total, -1)
    k = _rotate(st.k[:st.total].reshape(-1, kvh, hd), position).float()
    v = st.v[:st.total].reshape(-1, kvh, hd).float()
    for x, (codes, scales) in zip((k, v), st.pool):
        c, s = _quantize4(x)
        codes[slot], scales[slot] = _pack(c), s
        back = torch.zeros(st.rows, kvh * hd, device=DEV)
        back[:st.total] = _values(codes[slot], scales[slot], hd).reshape(st.total, -1)
        out.append(back)
    return [q, torch.stack(out)]


def _plain_attention(st):
    case, hd, kvh, heads = st.case, st.case["head_dim"], st.case["kv_heads"], st.case["heads"]
    seqs, page, n = case["seqs"], case["page"], st.new_max
    group = heads // kvh
    counts = st.starts[1:] - st.starts[:-1]
    seq, at = _rows_of(counts, st.total)
    q = torch.zeros(seqs, n, heads, hd, device=DEV)
    q[seq, at] = st.q[:st.total].reshape(-1, heads, hd).float()
    q = q.reshape(seqs, n, kvh, group, hd).permute(0, 2, 1, 3, 4).reshape(seqs, kvh, n * group, hd)
    slot = (st.table.clamp(min=0).long()[:, :, None] * page + torch.arange(page, device=DEV)).reshape(seqs, -1)
    (kc, ks), (vc, vs) = st.pool
    k = _values(kc[slot], ks[slot], hd).permute(0, 2, 3, 1).contiguous()        # [seq][head][channel][slot]
    v = _values(vc[slot], vs[slot], hd).permute(0, 2, 1, 3).contiguous()
    s = torch.matmul(q, k) * hd ** -0.5
    last = st.past[:, None].long() + torch.arange(n, device=DEV)                  # the last slot each row sees
    seen = torch.arange(slot.shape[1], device=DEV) <= last[:, :, None]
    s = s.reshape(seqs, kvh, n, group, -1).masked_fill_(~seen[:, None, :, None, :], -math.inf).reshape(s.shape)
    s = torch.exp(s - s.amax(dim=-1, keepdim=True))
    o = torch.matmul(s, v) / s.sum(dim=-1, keepdim=True)
    o = o.reshape(seqs, kvh, n, group, hd).permute(0, 2, 1, 3, 4).reshape(seqs, n, heads * hd)
    out = torch.zeros_like(st.q)
    out[:st.total] = o[seq, at].to(out.dtype)
    return out


def _plain_logits(st):
    i = st.inp
    rows, vocab = i["x"].shape
    total = i["history"].numel()
    row, at = _rows_of(i["starts"][1:] - i["starts"][:-1], total)
    real = (i["history"] >= 0) & (i["history"] < vocab)
    flat = torch.where(real, row * vocab + i["history"].long(), rows * vocab)
    ones = torch.ones(total, device=DEV, dtype=torch.float64)
    seen = torch.zeros(rows * vocab + 1, device=DEV, dtype=torch.float64).scatter_add_(0, flat, ones)[:-1].reshape(rows, vocab)
    made = torch.zeros(rows * vocab + 1, device=DEV, dtype=torch.float64).scatter_add_(
        0, flat, (at >= i["prompts"][row]).double())[:-1].reshape(rows, vocab)
    # 64 bits, rounded once: the greedy id hangs on the last one
    x = i["x"].double()
    rep = i["repetition"].double()[:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - made * i["frequency"].double()[:, None] - (made > 0) * i["presence"].double()[:, None]
    brow, _ = _rows_of(i["bstarts"][1:] - i["bstarts"][:-1], i["btokens"].numel())
    x = x + torch.zeros(rows * vocab, device=DEV, dtype=torch.float64).scatter_add_(
        0, brow * vocab + i["btokens"].long(), i["bvalues"].double()).reshape(rows, vocab)
    x = x.to(i["x"].dtype)
    if i["mask"] is not None:
        bits = ((i["mask"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1).reshape(i["mask"].shape[0], -1)
        allowed = (bits[i["index"].clamp(min=0).long(), :vocab] > 0) | (i["index"] < 0)[:, None]
        x = x.masked_fill(~allowed, -math.inf)
    best = x.amax(dim=1, keepdim=True)
    ids = torch.where(x == best, torch.arange(vocab, device=DEV), vocab).amin(dim=1).to(torch.int32)
    return [x, torch.where(best[:, 0] > -math.inf, ids, -1)]


# ---- one pass -------------------------------------------------------------------


def run(st):
    op = st.case["op"]
    if not own:
        return {"norm": _plain_norm, "append": _plain_append, "attention": _plain_attention, "logits": _plain_logits}[op](st)
    if op == "norm":
        st.ctx.norm_quantize_device(st.req, stream=st.stream)
        return [st.out, st.q8 * st.scales[:, None], st.scales]
    if op == "append":
        st.ctx.paged_kv_append_device(st.cache, st.req, stream=st.stream)
        st.ctx.paged_kv_read_device(st.cache, st.batch, st.kv[0].data_ptr(), st.kv[1].data_ptr(), stream=st.stream)
        return [st.q_out, st.kv]
    if op == "attention":
        st.ctx.paged_kv_attention_device(st.cache, st.req, stream=st.stream)
        return st.out
    st.ctx.logits_process_device(st.req, stream=st.stream)
    return [st.out, st.ids]


# ---- in 64 bits, from the definitions ---------------------------------------------


def _exact4(x):
    """What the 4-bit cache holds of fp32 x [rows][heads][head_dim], float64: per group of 64
    channels an f16 minimum and an f16 fifteenth of the span, the nearest of 16 levels."""
    x = torch.nan_to_num(torch.where(x.abs() == math.inf, 0.0, x), nan=0.0).clamp(-F16_MAX, F16_MAX)
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for first in range(0, x.shape[-1], GROUP):
        g = x[..., first:first + GROUP]
        m = g.min(dim=-1).values[..., None]
        d = g.max(dim=-1).values[..., None] - m
        d16 = torch.div(d, torch.tensor([15.0], device=d.device)).to(torch.float16).double()
        m16 = m.to(torch.float16).double()
        level = torch.where(d16 > 0, (g.double() - m16) / torch.where(d16 > 0, d16, 1.0), 0.0)
        out[..., first:first + GROUP] = m16 + d16 * torch.clamp(torch.round(level), 0.0, 15.0)
    return out


def _exact_norm(case, seed):
    x, r, w = _norm_inputs(case, seed)
    h64 = x.double() + r.double()
    h = h64.to(x.dtype).double()
    y = h * w.double() / torch.sqrt((h * h).sum(dim=1, keepdim=True) / h.shape[1] + EPS)
    # the int8 step is defined on fp32 values, with fp32 operations
    y32 = y.to(torch.float32)
    top = y32.abs().max(dim=1).values
    scale = torch.where(top > 0, torch.div(top, torch.tensor([127.0], device=DEV)), 1.0)
    inverse = torch.div(torch.tensor([1.0], device=DEV), scale)
    code = torch.round(torch.clamp(y32 * inverse[:, None], -127.0, 127.0))
    return [h64, code.double() * scale.double()[:, None], scale.double()]


def _exact_rotation(x, position):
    rows, heads, hd = x.shape
    x = x.double().reshape(rows, heads, 2, hd // 2)
    i = torch.arange(hd // 2, device=DEV, dtype=torch.float64)
    angle = position.double()[:, None, None] * torch.exp(-2.0 * i / hd * math.log(ROPE_THETA))
    z = torch.complex(x[:, :, 0], x[:, :, 1]) * torch.polar(torch.ones_like(angle), angle)
    return torch.cat((z.real, z.imag), dim=-1)


def _exact_append(case, seed):
    past, new, starts, _ = _batch(case)
    rows, hd, kvh = starts[-1] + case["rows_pad"], case["head_dim"], case["kv_heads"]
    position = torch.tensor([p + j for p, n in zip(past, new) for j in range(n)], device=DEV)
    n = starts[-1]
    k, v = _kv_inputs(case, seed, rows)
    q = torch.zeros(rows, case["heads"] * hd, dtype=torch.float64, device=DEV)
    q[:n] = _exact_rotation(_query(case, seed, rows)[:n].reshape(n, -1, hd), position).reshape(n, -1)
    kv = torch.zeros(2, rows, kvh * hd, dtype=torch.float64, device=DEV)
    kv[0, :n] = _exact4(_exact_rotation(k[:n].reshape(n, kvh, hd), position).float()).reshape(n, -1)
    kv[1, :n] = _exact4(v[:n].reshape(n, kvh, hd).float()).reshape(n, -1)
    return [q, kv]


def _exact_attention(case, seed):
    past, new, starts, _ = _batch(case)
    hd, kvh, heads = case["head_dim"], case["kv_heads"], case["heads"]
    rows = starts[-1] + case["rows_pad"]
    q = _query(case, seed, rows)
    k, v = _kv_inputs(case, seed, sum(past) + sum(new))
    out = torch.zeros(rows, heads * hd, dtype=torch.float64, device=DEV)
    at = 0
    for s, (p, n) in enumerate(zip(past, new)):
        ks = _exact4(k[at:at + p + n].reshape(-1, kvh, hd).float())
        vs = _exact4(v[at:at + p + n].reshape(-1, kvh, hd).float())
        at += p + n
        qs = q[starts[s]:starts[s + 1]].double().reshape(n, heads, hd)
        allowed = torch.arange(p + n, device=DEV)[None, :] <= p + torch.arange(n, device=DEV)[:, None]
        for h in range(heads if n else 0):
            j = h * kvh // heads
            w = torch.softmax((qs[:, h] @ ks[:, j].t().contiguous() / math.sqrt(hd)).masked_fill(~allowed, -math.inf), dim=1)
            out[starts[s]:starts[s + 1], h * hd:(h + 1) * hd] = w @ vs[:, j].contiguous()
    return out


def _exact_logits(case, seed):
    i = _logits_inputs(case, seed)
    x = i["x"].double().clone()
    rows, vocab = x.shape
    starts, bstarts = i["starts"].tolist(), i["bstarts"].tolist()
    for r in range(rows):
        h = i["history"][starts[r]:starts[r + 1]].long()
        prompt = int(i["prompts"][r])
        known = torch.unique(h[(h >= 0) & (h < vocab)])
        rep = float(i["repetition"][r])
        x[r, known] = torch.where(x[r, known] > 0, x[r, known] / rep, x[r, known] * rep)
        tail = h[prompt:]
        made, count = torch.unique(tail[(tail >= 0) & (tail < vocab)], return_counts=True)
        x[r, made] -= count.double() * float(i["frequency"][r]) + float(i["presence"][r])
        b = slice(bstarts[r], bstarts[r + 1])
        x[r].index_add_(0, i["btokens"][b].long(), i["bvalues"][b].double())
        if i["mask"] is not None and int(i["index"][r]) >= 0:
            words = i["mask"][int(i["index"][r])].long() & 0xFFFFFFFF
            token = torch.arange(vocab, device=DEV)
            x[r, ((words[token // 32] >> (token % 32)) & 1) == 0] = -math.inf
    return [x, None]


def exact(case, seed):
    return {"norm": _exact_norm, "append": _exact_append, "attention": _exact_attention, "logits": _exact_logits}[case["op"]](case, seed)
