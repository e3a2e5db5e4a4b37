"""The operators of packed prompts and of beams, as cases that can be timed and checked.

op "rotary"   queries and keys of a step's tokens, each head normed where weights
              are given, rotated by positions with one to three axes (time, height,
              width).
op "prompt"   causal attention of packed sequences over their own keys and values,
              grouped heads.
op "select"   the best continuations of every sequence's beams over the vocabulary,
              and the beams that go on.
op "advance"  what the beams keep (page tables, lengths, token histories, the page
              each writes to, in the caches of all layers) follows them.

With ``own`` false, run() computes them in elementary torch operations; with
``own`` true, it makes the library's calls.
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
GROUP = 64          # channels of a cached token and head that share a scale and a minimum
F16_MAX = 65504.0
END = 7             # a token that ends a beam

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ------------------------------------------------------------------


def listed():
    return [
        # one decoded token of a text: all latency
        dict(name="rotary_token_f32", op="rotary", dtype="f32", tokens=1, rope=128, axes=1, turn=False, norms=False, fused=False,
             **QWEN2_1P5B),
        # a decode batch, heads normed, columns of the projections' one buffer
        dict(name="rotary_61_tokens_f16", op="rotary", dtype="f16", tokens=61, rope=128, axes=3, turn=True, norms=True, fused=True,
             **QWEN3_4B),
        # prompts with images: bytes
        dict(name="rotary_4099_tokens_bf16", op="rotary", dtype="bf16", tokens=4099, rope=128, axes=3, turn=False, norms=True,
             fused=True, **QWEN3_4B),
        # a few short questions at once
        dict(name="prompt_short_f32", op="prompt", dtype="f32", seqs=3, longest=61, mix=1, fused=False, rows_pad=0, **QWEN2_1P5B),
        # prompts of several users, from a line to pages of text, packed
        dict(name="prompt_packed_bf16", op="prompt", dtype="bf16", seqs=9, longest=1777, mix=2, fused=True, rows_pad=5, **QWEN3_4B),
        # one long document
        dict(name="prompt_long_bf16", op="prompt", dtype="bf16", seqs=1, longest=8192, mix=3, fused=True, rows_pad=0, **QWEN3_4B),
        # documents for a model of small heads
        dict(name="prompt_packed_f16", op="prompt", dtype="f16", seqs=3, longest=3000, mix=4, fused=False, rows_pad=0, heads=16,
             kv_heads=4, head_dim=64),
        # fp32 throughout
        dict(name="prompt_packed_f32", op="prompt", dtype="f32", seqs=4, longest=1024, mix=5, fused=False, rows_pad=3, **QWEN2_1P5B),
        # one request's beams
        dict(name="select_4_beams_f32", op="select", dtype="f32", seqs=1, beams=4, vocab=VOCAB, count=8, mix=6, grammar=False),
        # a batch of requests, some with first steps, some under a grammar
        dict(name="select_64_beams_bf16", op="select", dtype="bf16", seqs=16, beams=4, vocab=VOCAB, count=8, mix=7, grammar=True),
        # one request's beams in a model of two layers
        dict(name="advance_4_beams", op="advance", seqs=1, beams=4, layers=2, page=16, past_max=333, mix=8, kv_heads=2, head_dim=128),
        # a batch of requests in all layers of a small model
        dict(name="advance_64_beams", op="advance", seqs=16, beams=4, layers=28, page=64, past_max=6000, mix=9, kv_heads=2,
             head_dim=128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges the listed ones stand for: 1 to 4099 rotated tokens, packed prompts of 1 to 8192 tokens,
    head dims 32 to 256, up to 64 beams in all, vocabularies of 1000 to 152000, caches of 1 to 28 layers."""
    op = rng.choice(["rotary", "prompt", "prompt", "prompt", "select", "advance"])
    kv = rng.choice([1, 2, 4, 8])
    heads = dict(kv_heads=kv, heads=kv * rng.choice([1, 2, 3, 4, 6, 8]), head_dim=rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256]))
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op == "rotary":
        hd = heads["head_dim"]
        most = max(1, min(4099, 21_000_000 // ((heads["heads"] + kv) * hd)))
        return dict(op=op, dtype=dtype, tokens=_log_int(rng, 1, most), rope=rng.choice([hd, hd, hd // 2]), axes=rng.choice([1, 2, 3, 3]),
                    turn=rng.random() < 0.5, norms=rng.random() < 0.5, fused=rng.random() < 0.5, **heads)
    if op == "prompt":
        case = dict(op=op, dtype=dtype, seqs=_log_int(rng, 1, 16), longest=_log_int(rng, 1, 8192), mix=rng.randrange(1 << 20),
                    fused=rng.random() < 0.5, rows_pad=rng.choice([0, 0, 1, 7]), **heads)
        # no dearer than the largest listed one, padded to the longest too
        while case["seqs"] * case["longest"] ** 2 * case["heads"] * max(128, case["head_dim"]) > 2.7e11:
            case["longest"] = max(1, case["longest"] * 3 // 4)
        return case
    if op == "select":
        vocab, beams = _log_int(rng, 1000, VOCAB), rng.choice([1, 2, 3, 4, 4, 5, 8])
        return dict(op=op, dtype=dtype, seqs=_log_int(rng, 1, max(1, min(64 // beams, 9_700_000 // (beams * vocab)))), beams=beams,
                    vocab=vocab, count=rng.choice([2 * beams, 2 * beams, rng.randint(1, 16)]), mix=rng.randrange(1 << 20),
                    grammar=rng.random() < 0.5)
    beams = rng.choice([1, 2, 3, 4, 4, 5, 8])
    return dict(op=op, seqs=_log_int(rng, 1, 64 // beams), beams=beams, layers=_log_int(rng, 1, 28), page=rng.choice([16, 16, 32, 64]),
                past_max=_log_int(rng, 1, 6000), mix=rng.randrange(1 << 20), kv_heads=rng.choice([1, 2]),
                head_dim=rng.choice([64, 80, 128, 128]))


def _lengths(case):
    """Tokens of each sequence: the first the longest, the others spread over the range, some none."""
    rng = random.Random(case["mix"])
    return [case["longest"]] + [_log_int(rng, 1, case["longest"]) if rng.random() < 0.95 else 0 for _ in range(case["seqs"] - 1)]


def _beams(case):
    """(cached tokens of each sequence's beams, this step's among them; the row each row goes on from, -1: from itself, ended)."""
    rng = random.Random(case["mix"])
    cached = [case["past_max"]] + [_log_int(rng, 1, case["past_max"]) for _ in range(case["seqs"] - 1)]
    b = case["beams"]
    parents = []
    for s in range(case["seqs"]):
        # the best beams have most of the next ones
        parents += [s * b + min(b - 1, int(b * rng.random() ** 1.5)) if rng.random() < 0.97 else -1 for _ in range(b)]
    return cached, parents


def _copies(case):
    """Rows whose page in use is copied: of a parent's children all but the first."""
    cached, parents = _beams(case)
    b, seen, rows = case["beams"], set(), []
    for r, p in enumerate(parents):
        p = r if p < 0 else p
        if p in seen and cached[r // b] % case["page"]:
            rows.append(r)
        seen.add(p)
    return rows


def work(case):
    op = case["op"]
    if op == "advance":
        cached, _ = _beams(case)
        b, page, c = case["beams"], case["page"], case["kv_heads"] * case["head_dim"]
        groups = -(-case["head_dim"] // GROUP)
        token = case["kv_heads"] * (case["head_dim"] + 8 * groups)
        tails = sum(b * (n % page) for n in cached)
        copied = sum(cached[r // b] % page for r in _copies(case))
        rows = b * sum(n + -(-n // page) for n in cached)
        # pages copied; the pages in use read back as fp32 values; tables and histories
        return {"bytes": case["layers"] * (2 * copied * token + tails * (token + 8 * c)) + 8 * rows, "flops": case["layers"] * tails * 4 * c}
    size = SIZE[case["dtype"]]
    if op == "rotary":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        return {"bytes": 2 * n * size + 4 * case["axes"] * case["tokens"], "flops": 8 * n}
    if op == "select":
        n = case["seqs"] * case["beams"] * case["vocab"]
        return {"bytes": n * size + case["seqs"] * (case["count"] * 12 + case["beams"] * 16), "flops": 4 * n}
    lengths = _lengths(case)
    rows = sum(lengths) * case["head_dim"]
    return {"bytes": size * rows * 2 * (case["heads"] + case["kv_heads"]),
            "flops": 2 * sum(n * (n + 1) for n in lengths) * case["heads"] * case["head_dim"]}


# ---- inputs ---------------------------------------------------------------------


def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + salt)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _qkv(case, seed, rows):
    """Projections' outputs: channels of their own scale and offset; in one buffer, or in three."""
    g = _gen(seed, 21)
    q, c, dt = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"], DTYPES[case["dtype"]]
    scale = 0.3 + 1.2 * torch.rand(c, generator=g, device=DEV)
    offset = torch.where(torch.rand(c, generator=g, device=DEV) < 0.05, 2.0, 0.3) * _normal(g, c)
    parts = [1.2 * _normal(g, rows, q), _normal(g, rows, c) * scale + offset, _normal(g, rows, c) * scale.flip(0)]
    if case["fused"]:
        return torch.cat(parts, dim=1).to(dt).split([q, c, c], dim=1)
    return tuple(p.to(dt) for p in parts)


def _sections(case):
    """Pairs of each axis: time the fewest, as for images."""
    half, axes = case["rope"] // 2, case["axes"]
    if axes == 1:
        return [half]
    first = half // (axes + 1)
    rest = half - first
    return [first] + [rest // (axes - 1) + (1 if i < rest % (axes - 1) else 0) for i in range(axes - 1)]


def _axis_of_pair(case):
    sections = _sections(case)
    if not case["turn"]:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, order, a = list(sections), [], 0
    while len(order) < sum(sections):
        if left[a]:
            order.append(a)
            left[a] -= 1
        a = (a + 1) % len(left)
    return order


def _positions(case, seed):
    """Text far into a context, then an image's grid: a time for all of it, its rows and columns."""
    t = torch.arange(case["tokens"], device=DEV)
    first = 20000 + 37 * (seed % 1000)
    p = (first + t).repeat(case["axes"], 1)
    image = t % 300 >= 44          # 16 by 16
    at = t % 300 - 44
    start = first + t - at
    for a in range(case["axes"] if case["axes"] > 1 else 0):
        p[a] = torch.where(image, start + (0 if a == 0 else at // 16 if a == 1 else at % 16), p[a])
    return p.to(torch.int32)


def _rotary_inputs(case, seed):
    q, k, _ = _qkv(case, seed, case["tokens"])
    g = _gen(seed, 22)
    norms = [1.0 + 0.2 * _normal(g, case["head_dim"]) for _ in range(2)] if case["norms"] else [None, None]
    return q, k, norms, _positions(case, seed)


def _select_inputs(case, seed):
    g = _gen(seed, 23)
    rng = random.Random(case["mix"])
    seqs, beams, vocab = case["seqs"], case["beams"], case["vocab"]
    x = 2.5 * _normal(g, seqs, 1, vocab) + 1.2 * _normal(g, seqs, beams, vocab)    # beams of a request are alike
    x[:, :, END] += 6.0
    x = x.reshape(seqs * beams, vocab)
    if case["grammar"]:
        open_ = torch.rand(seqs * beams, 1, generator=g, device=DEV) ** 2
        allowed = (torch.rand(seqs * beams, vocab, generator=g, device=DEV) < open_) | (torch.rand(seqs * beams, 1, generator=g, device=DEV) < 0.5)
        allowed[:, END] = True
        x = torch.where(allowed, x, -math.inf)
    scores = -20.0 * torch.rand(seqs, 1, generator=g, device=DEV) - 2.0 * torch.rand(seqs, beams, generator=g, device=DEV)
    # a first step has one beam
    first = torch.tensor([rng.random() < 0.2 for _ in range(seqs)], device=DEV)
    scores = torch.where(first[:, None] & (torch.arange(beams, device=DEV) > 0), -math.inf, scores)
    return x.to(DTYPES[case["dtype"]]), scores


def _advance_inputs(case, seed):
    """Tables whose beams share whole pages and have one of their own, spares, histories; the tokens chosen."""
    g = _gen(seed, 24)
    cached, parents = _beams(case)
    b, page, seqs = case["beams"], case["page"], case["seqs"]
    rows, width = seqs * b, max(cached) // page + 2
    full = torch.tensor([n // page for n in cached], device=DEV).repeat_interleave(b)
    tail = torch.tensor([n % page for n in cached], device=DEV).repeat_interleave(b)
    whole = sum(n // page for n in cached)
    pages = whole + 2 * rows + 3
    order = torch.randperm(pages, generator=g, device=DEV)
    first = torch.tensor([sum(n // page for n in cached[:s]) for s in range(seqs)], device=DEV).repeat_interleave(b)
    column = torch.arange(width, device=DEV)
    row = torch.arange(rows, device=DEV)
    shared = order[(first[:, None] + column).clamp(max=pages - 1)]
    table = torch.where(column < full[:, None], shared, torch.where((column == full[:, None]) & (tail[:, None] > 0), order[whole + row][:, None], -1))
    spare = order[whole + rows + row]
    length = max(cached) + 8
    history = torch.randint(0, VOCAB, (rows, length), generator=g, device=DEV)
    history = torch.where(torch.arange(length, device=DEV) < (full * page + tail)[:, None], history, -1)
    i = lambda t: t.to(torch.int32).contiguous()  # noqa: E731
    return dict(pages=pages, cached=i(full * page + tail), parents=_i32(parents), table=i(table), spare=i(spare), history=i(history),
                tokens=torch.randint(0, VOCAB, (rows,), generator=g, device=DEV, dtype=torch.int32), full=full, tail=tail,
                tails=[n % page for n in cached for _ in range(b)])


def _cached_inputs(case, seed, rows):
    """Keys and values of every layer's pages in use, [layer][2][tokens][channels]."""
    return _normal(_gen(seed, 25), case["layers"], 2, rows, case["kv_heads"] * case["head_dim"])


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


def _ptr(t):
    return None if t is None else t.data_ptr()


def _prepare_rotary(st, seed):
    case = st.case
    st.q, st.k, st.norms, st.positions = _rotary_inputs(case, seed)
    if not own:
        st.axis = torch.tensor(_axis_of_pair(case), device=DEV)
        return
    dt = DTYPES[case["dtype"]]
    st.q_out, st.k_out = (torch.empty(x.shape, device=DEV, dtype=dt) for x in (st.q, st.k))
    st.req = st.open().rotary_request(case["tokens"], case["dtype"], case["head_dim"], case["rope"], ROPE_THETA, _ptr(st.positions),
                                      sections=_sections(case), in_turn=case["turn"], query_heads=case["heads"], q_ptr=_ptr(st.q),
                                      q_out_ptr=_ptr(st.q_out), key_heads=case["kv_heads"], k_ptr=_ptr(st.k), k_out_ptr=_ptr(st.k_out),
                                      q_norm_ptr=_ptr(st.norms[0]), k_norm_ptr=_ptr(st.norms[1]), eps=EPS,
                                      query_stride=st.q.stride(0), key_stride=st.k.stride(0))


def _prepare_prompt(st, seed):
    case = st.case
    lengths = _lengths(case)
    starts = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    st.total, st.longest = starts[-1], max(lengths)
    rows = st.total + case["rows_pad"]
    st.starts = _i32(starts)
    st.q, st.k, st.v = _qkv(case, seed, rows)
    if own:
        st.out = torch.zeros(st.q.shape, device=DEV, dtype=st.q.dtype)
        st.req = st.open().prompt_attention_request(case["seqs"], rows, _ptr(st.starts), case["dtype"], case["heads"], case["kv_heads"],
                                                    case["head_dim"], _ptr(st.q), _ptr(st.k), _ptr(st.v), _ptr(st.out),
                                                    case["head_dim"] ** -0.5, query_stride=st.q.stride(0), key_stride=st.k.stride(0),
                                                    value_stride=st.v.stride(0))


def _prepare_select(st, seed):
    case = st.case
    st.x, st.scores = _select_inputs(case, seed)
    if own:
        seqs, beams, count = case["seqs"], case["beams"], case["count"]
        f = lambda n: torch.empty(seqs, n, device=DEV)  # noqa: E731
        i = lambda n: torch.empty(seqs, n, device=DEV, dtype=torch.int32)  # noqa: E731
        st.values, st.parents, st.tokens, st.next = f(count), i(count), i(count), [f(beams), i(beams), i(beams)]
        ctx = st.open()
        st.work = torch.empty(max(1, ctx.beam_select_workspace_bytes(seqs, beams, case["vocab"], count)), device=DEV, dtype=torch.uint8)
        st.req = ctx.beam_select_request(seqs, beams, case["vocab"], count, case["dtype"], _ptr(st.x), _ptr(st.scores), _ptr(st.values),
                                         _ptr(st.parents), _ptr(st.tokens), _ptr(st.work), end_tokens=[END],
                                         next_scores_ptr=_ptr(st.next[0]), next_parents_ptr=_ptr(st.next[1]),
                                         next_tokens_ptr=_ptr(st.next[2]))


def _prepare_advance(st, seed):
    case = st.case
    st.inp = i = _advance_inputs(case, seed)
    rows, hd, kvh, page = case["seqs"] * case["beams"], case["head_dim"], case["kv_heads"], case["page"]
    st.rows = sum(i["tails"])
    starts = [sum(i["tails"][:r]) for r in range(rows + 1)]
    kv = _cached_inputs(case, seed, max(1, st.rows))
    if not own:
        groups = -(-hd // GROUP)
        slots = i["pages"] * page
        # the pools as [layer][keys, values][slot][head]: two codes a byte, (step, minimum) pairs
        st.codes = torch.zeros(case["layers"], 2, slots, kvh, groups * GROUP // 2, dtype=torch.uint8, device=DEV)
        st.scales = torch.zeros(case["layers"], 2, slots, kvh, groups, 2, dtype=torch.float16, device=DEV)
        slot = _tail_slots(st, i["table"])
        c, s = _quantize4(kv[:, :, :st.rows].reshape(case["layers"], 2, st.rows, kvh, hd))
        st.codes[:, :, slot], st.scales[:, :, slot] = _pack(c), s
        return
    ctx = st.open()
    st.caches = [ctx.paged_kv_create(i["pages"], page, kvh, hd) for _ in range(case["layers"])]
    st.first, st.starts = (i["full"] * page).to(torch.int32), _i32(starts)
    st.out = {n: torch.empty_like(i[n]) for n in ("table", "cached", "spare", "history")}
    st.kv = torch.zeros(case["layers"], 2, max(1, st.rows), kvh * hd, device=DEV)
    fill = ctx.paged_batch(rows, max(1, st.rows), _ptr(st.starts), _ptr(st.first), _ptr(i["table"]), i["table"].shape[1])
    st.back = ctx.paged_batch(rows, max(1, st.rows), _ptr(st.starts), _ptr(st.first), _ptr(st.out["table"]), i["table"].shape[1])
    for h, x in zip(st.caches, kv):
        ctx.paged_kv_append_device(h, ctx.paged_append_request(fill, "f32", k_ptr=_ptr(x[0]), v_ptr=_ptr(x[1])), stream=st.stream)
    torch.cuda.synchronize()
    st.req = ctx.beam_advance_request(case["seqs"], case["beams"], page, i["table"].shape[1], _ptr(i["parents"]), _ptr(i["cached"]),
                                      _ptr(st.out["cached"]), _ptr(i["table"]), _ptr(st.out["table"]), _ptr(i["spare"]),
                                      _ptr(st.out["spare"]), added=0, tokens_ptr=_ptr(i["tokens"]), history_ptr=_ptr(i["history"]),
                                      history_out_ptr=_ptr(st.out["history"]), history_length=i["history"].shape[1])


def prepare(case, seed):
    st = _State(case)
    {"rotary": _prepare_rotary, "prompt": _prepare_prompt, "select": _prepare_select, "advance": _prepare_advance}[case["op"]](st, seed)
    return st


# ---- the plain forms ------------------------------------------------------------


def _rows_of(counts, total):
    """(sequence, index within it) of each of `total` rows laid one sequence after the other."""
    seq = torch.repeat_interleave(torch.arange(counts.numel(), device=DEV), counts.long(), output_size=total)
    first = torch.cumsum(counts.long(), 0) - counts.long()
    return seq, torch.arange(total, device=DEV) - first[seq]


def _plain_rotary(st):
    case, rope = st.case, st.case["rope"]
    half = rope // 2
    # 64 bits: at far positions an fp32 angle is off by hundredths
    freq = ROPE_THETA ** (-2.0 * torch.arange(half, device=DEV, dtype=torch.float64) / rope)
    angle = (st.positions.double()[st.axis].t() * freq)[:, None, :]
    c, s = torch.cos(angle).float(), torch.sin(angle).float()

    def turn(x, norm):
        y = x.reshape(case["tokens"], -1, case["head_dim"]).float()
        if norm is not None:
            y = y * torch.rsqrt(y.square().mean(dim=-1, keepdim=True) + EPS) * norm
        a, b = y[..., :half], y[..., half:rope]
        return torch.cat((a * c - b * s, a * s + b * c, y[..., rope:]), dim=-1).to(x.dtype).reshape(x.shape)

    return [turn(st.q, st.norms[0]), turn(st.k, st.norms[1])]


def _plain_prompt(st):
    case, hd, kvh, heads = st.case, st.case["head_dim"], st.case["kv_heads"], st.case["heads"]
    seqs, n, group = case["seqs"], st.longest, heads // kvh
    seq, at = _rows_of(st.starts[1:] - st.starts[:-1], st.total)

    def padded(x):
        y = torch.zeros(seqs, n, x.shape[1], device=DEV)
        y[seq, at] = x[:st.total].float()
        return y.reshape(seqs, n, kvh, -1, hd)

    q = padded(st.q).permute(0, 2, 1, 3, 4).reshape(seqs, kvh, n * group, hd)
    k = padded(st.k)[:, :, :, 0].permute(0, 2, 3, 1).contiguous()
    v = padded(st.v)[:, :, :, 0].permute(0, 2, 1, 3).contiguous()
    s = torch.matmul(q, k) * hd ** -0.5
    later = torch.arange(n, device=DEV)[None, :] > torch.arange(n, device=DEV)[:, None]
    s = s.reshape(seqs, kvh, n, group, n).masked_fill_(later[:, None], -math.inf).reshape(seqs, kvh, n * group, n)
    s = torch.exp(s - s.amax(dim=-1, keepdim=True))
    o = torch.matmul(s, v) / s.sum(dim=-1, keepdim=True)
    o = o.reshape(seqs, kvh, n, group, hd).permute(0, 2, 1, 3, 4).reshape(seqs, n, heads * hd)
    out = torch.zeros(st.q.shape, device=DEV, dtype=st.q.dtype)
    out[:st.total] = o[seq, at].to(out.dtype)
    return out


def _plain_select(st):
    case = st.case
    seqs, beams, vocab, count = case["seqs"], case["beams"], case["vocab"], case["count"]
    # 64 bits: which of two candidates is the better one hangs on the last one
    x = st.x.double()
    top = x.amax(dim=1, keepdim=True)
    total = top + torch.log(torch.exp(x - top).sum(dim=1, keepdim=True))
    x = (x - total).reshape(seqs, beams, vocab) + st.scores.double()[:, :, None]
    value, at = torch.sort(x.reshape(seqs, -1), dim=1, descending=True, stable=True)
    value, at = value[:, :count], at[:, :count]
    none = value == -math.inf
    parent = torch.where(none, -1, at // vocab + beams * torch.arange(seqs, device=DEV)[:, None])
    token = torch.where(none, -1, at % vocab)
    # the best that do not end come first, in their order
    out = torch.arange(count, device=DEV) + torch.where(none | (token == END), count, 0)
    rank = torch.sort(out, dim=1).values[:, :beams]
    pick = torch.nn.functional.pad(rank, (0, beams - rank.shape[1]), value=count)
    gone, pick = pick >= count, pick.clamp(max=count - 1)
    i32 = torch.int32
    return [value.float(), parent.to(i32), token.to(i32), torch.where(gone, -math.inf, value.gather(1, pick)).float(),
            torch.where(gone, -1, parent.gather(1, pick)).to(i32), torch.where(gone, -1, token.gather(1, pick)).to(i32)]


def _quantize4(x):
    """fp32 [..., head_dim] as 4-bit codes and (step, minimum) of each group, as the cache defines them."""
    x = torch.nn.functional.pad(x, (0, -x.shape[-1] % GROUP), value=math.nan).unflatten(-1, (-1, GROUP))
    real = ~torch.isnan(x)
    lo = torch.where(real, x, math.inf).amin(dim=-1, keepdim=True)
    span = torch.where(real, x, -math.inf).amax(dim=-1, keepdim=True) - lo
    least, step = lo.half(), (span / torch.full_like(span, 15.0)).half()
    # next to a border between codes the quotient decides: 64 bits
    t = (torch.where(real, x, lo).double() - least.double()) / step.double()
    code = torch.where(step > 0, t.round().clamp(0, 15), torch.zeros_like(t)).to(torch.uint8)
    return code.flatten(-2), torch.cat([step, least], dim=-1)


def _pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _values(codes, scales, hd):
    """The fp32 values that packed codes and their (step, minimum) pairs stand for."""
    c = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)[..., :hd].float()
    s = scales.float().repeat_interleave(GROUP, dim=-2)[..., :hd, :]
    return s[..., 0] * c + s[..., 1]


def _tail_slots(st, table):
    """Slots of every row's page in use, a row after the other."""
    i, page = st.inp, st.case["page"]
    row, at = _rows_of(i["tail"], st.rows)
    return table[row, i["full"][row]].long() * page + at


def _plain_advance(st):
    i, case = st.inp, st.case
    beams, page = case["beams"], case["page"]
    rows = case["seqs"] * beams
    row = torch.arange(rows, device=DEV)
    stays = i["parents"] < 0
    parent = torch.where(stays, row, i["parents"].long())
    column = torch.arange(i["table"].shape[1], device=DEV)
    # the first child of a parent takes its page; a later one the spare that it holds, and gets the page of a beam that ended
    same = parent[:, None] == parent[None, :]
    later = (same & (row[None, :] < row[:, None])).any(dim=1)
    childless = ~(parent[:, None] == row).any(dim=0)
    group = row // beams
    before = (group[:, None] == group) & (row < row[:, None])
    nth = (before & later).sum(dim=1)
    rank = (before & childless).sum(dim=1)
    match = (group[:, None] == group) & childless & (rank == nth[:, None])
    left = i["table"].gather(1, i["full"][:, None])[:, 0]
    released = left[match.to(torch.int8).argmax(dim=1)]
    begins = i["tail"] == 0
    spare = torch.where(begins, -1, torch.where(later, released, i["spare"]))
    mine = torch.where(begins | later, i["spare"], left[parent])
    table = torch.where(column < i["full"][:, None], i["table"][parent], torch.where(column == i["full"][:, None], mine[:, None], -1))
    at = torch.arange(i["history"].shape[1], device=DEV)
    history = i["history"][parent]
    history = torch.where((at == i["cached"][:, None]) & ~stays[:, None], i["tokens"][:, None], history)
    src, dst = _tail_slots(st, i["table"][parent]), _tail_slots(st, table)
    codes, scales = st.codes[:, :, src], st.scales[:, :, src]
    st.codes[:, :, dst], st.scales[:, :, dst] = codes, scales
    kv = _values(codes, scales, case["head_dim"]).flatten(-2)
    i32 = torch.int32
    return [table.to(i32), i["cached"][parent], spare.to(i32), history.to(i32), kv]


# ---- one pass -------------------------------------------------------------------


def run(st):
    op = st.case["op"]
    if not own:
        return {"rotary": _plain_rotary, "prompt": _plain_prompt, "select": _plain_select, "advance": _plain_advance}[op](st)
    if op == "rotary":
        st.ctx.rotary_device(st.req, stream=st.stream)
        return [st.q_out, st.k_out]
    if op == "prompt":
        st.ctx.prompt_attention_device(st.req, stream=st.stream)
        return st.out
    if op == "select":
        st.ctx.beam_select_device(st.req, stream=st.stream)
        return [st.values, st.parents, st.tokens, *st.next]
    st.ctx.paged_kv_beam_advance_device(st.caches, st.req, stream=st.stream)
    for h, x in zip(st.caches if st.rows else [], st.kv):
        st.ctx.paged_kv_read_device(h, st.back, x[0].data_ptr(), x[1].data_ptr(), stream=st.stream)
    return [st.out["table"], st.out["cached"], st.out["spare"], st.out["history"], st.kv[:, :, :st.rows]]


# ---- in 64 bits, from the definitions ---------------------------------------------


def _exact_rotary(case, seed):
    q, k, norms, positions = _rotary_inputs(case, seed)
    n, rope = case["tokens"], case["rope"]
    i = torch.arange(rope // 2, device=DEV, dtype=torch.float64)
    p = torch.stack([positions[a] for a in _axis_of_pair(case)], dim=1).double()
    z = torch.polar(torch.ones_like(p), p * torch.exp(-2.0 * i / rope * math.log(ROPE_THETA)))[:, None]
    out = []
    for x, w in ((q, norms[0]), (k, norms[1])):
        y = x.double().reshape(n, -1, case["head_dim"])
        if w is not None:
            y = y / torch.sqrt((y * y).sum(dim=-1, keepdim=True) / y.shape[-1] + EPS) * w.double()
        r = torch.complex(y[..., :rope // 2].contiguous(), y[..., rope // 2:rope].contiguous()) * z
        out.append(torch.cat((r.real, r.imag, y[..., rope:]), dim=-1).reshape(n, -1))
    return out


def _exact_prompt(case, seed):
    lengths, hd = _lengths(case), case["head_dim"]
    rows = sum(lengths) + case["rows_pad"]
    q, k, v = _qkv(case, seed, rows)
    out = torch.zeros(rows, case["heads"] * hd, dtype=torch.float64, device=DEV)
    at = 0
    for n in lengths:
        for h in range(case["heads"] if n else 0):
            j = h * case["kv_heads"] // case["heads"]
            qs, (ks, vs) = q[at:at + n, h * hd:(h + 1) * hd].double(), (x[at:at + n, j * hd:(j + 1) * hd].double() for x in (k, v))
            s = torch.matmul(qs, ks.t().contiguous()) / math.sqrt(hd)
            s = s + torch.full_like(s, -math.inf).triu(1)
            out[at:at + n, h * hd:(h + 1) * hd] = torch.matmul(torch.softmax(s, dim=1), vs)
        at += n
    return out


def _exact_select(case, seed):
    x, scores = _select_inputs(case, seed)
    seqs, beams, count = case["seqs"], case["beams"], case["count"]
    logp = torch.log_softmax(x.double(), dim=1).reshape(seqs, beams, -1)
    value, at = torch.topk((logp + scores.double()[:, :, None]).reshape(seqs, -1), min(count, logp[0].numel()), dim=1)
    goes = torch.full((seqs, beams), -math.inf, dtype=torch.float64, device=DEV)
    for s in range(seqs):
        on = [float(value[s, c]) for c in range(value.shape[1]) if int(at[s, c]) % case["vocab"] != END][:beams]
        goes[s, :len(on)] = torch.tensor(on, dtype=torch.float64)
    return [value, None, None, goes, None, None]


def exact(case, seed):
    op = case["op"]
    # whole numbers and copies have no nearer value
    return None if op == "advance" else {"rotary": _exact_rotary, "prompt": _exact_prompt, "select": _exact_select}[op](case, seed)
