"""Helpers of the serving operators' tests: batches on the GPU, and the
operators' definitions in 64 bits on the host."""
import torch

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half a step of a type's rounding, relative to the value
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
GROUP = 64


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float32)


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    from qwanto_amd import abi
    return torch.cuda.current_stream().cuda_stream or abi.NULL_STREAM


def quantize8(y):
    """The framework's per-token int8 quantization of fp32 y: (codes, scales)."""
    amax = y.abs().amax(dim=1, keepdim=True)
    scale = torch.where(amax > 0, amax / torch.full_like(amax, 127.0), torch.ones_like(amax))
    inv = torch.ones_like(scale) / scale
    return (y * inv).clamp(-127.0, 127.0).round().to(torch.int8), scale[:, 0]


def levels(x):
    """The cache's 4-bit form of fp32 x [..., head_dim]: (values float64, step, minimum of
    every channel, the quotient each code is rounded from)."""
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).clamp(-65504.0, 65504.0)
    values, steps, mins, quotients = [], [], [], []
    for c in range(0, x.shape[-1], GROUP):
        g = x[..., c:c + GROUP]
        lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        m = lo.half().double()
        s = ((hi - lo) / torch.full_like(lo, 15.0)).half().double()
        t = torch.where(s > 0, (g.double() - m) / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(g.double()))
        values.append(m + s * t.round().clamp(0, 15))
        steps.append(s.expand_as(t))
        mins.append(m.expand_as(t))
        quotients.append(t)
    cat = lambda v: torch.cat(v, dim=-1)  # noqa: E731
    return cat(values), cat(steps), cat(mins), cat(quotients)


def rotate(x, positions, rope, theta):
    """[rows][heads][head_dim] rotated in 64 bits: pairs (i, i + rope / 2)."""
    y = x.double().clone()
    half = rope // 2
    if half:
        freq = theta ** (-2.0 * torch.arange(half, dtype=torch.float64) / rope)
        ang = (positions.double()[:, None] * freq)[:, None]
        a, b = x[..., :half].double(), x[..., half:rope].double()
        y[..., :half] = a * ang.cos() - b * ang.sin()
        y[..., half:rope] = a * ang.sin() + b * ang.cos()
    return y


class Cache:
    """A paged cache of the library with its table, filled and read through the
    public calls."""

    def __init__(self, ctx, lengths, kv_heads, head_dim, page=16, rope=0, theta=1.0e6, extra=2, seed=0, width=None):
        """`lengths`: slots each sequence may use."""
        self.ctx, self.kv_heads, self.head_dim, self.page, self.rope, self.theta = ctx, kv_heads, head_dim, page, rope, theta
        need = [-(-n // page) for n in lengths]
        self.pages = sum(need) + extra
        order = torch.randperm(self.pages, generator=gen(seed + 99)).to(torch.int32)
        self.width = width or max(max(need), 1)
        table = torch.full((len(lengths), self.width), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        self.table_host = table
        self.table = table.to(DEV)
        self.h = ctx.paged_kv_create(self.pages, page, kv_heads, head_dim, rope_dims=rope, rope_theta=theta if rope else 0.0)
        self.keep = []

    def batch(self, past, new, pad=0, table=None):
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s = torch.tensor(starts, dtype=torch.int32, device=DEV)
        p = torch.tensor(past, dtype=torch.int32, device=DEV)
        t = self.table if table is None else table
        b = self.ctx.paged_batch(len(past), max(1, starts[-1] + pad), ptr(s), ptr(p), ptr(t), t.shape[1])
        self.keep.append((s, p, t, b))
        return b

    def append(self, batch, k, v, dtype, q=None, q_out=None, heads=0, positions=None, **strides):
        r = self.ctx.paged_append_request(batch, dtype, ptr(k), ptr(v), q_ptr=ptr(q), q_out_ptr=ptr(q_out),
                                          query_heads=heads, positions_ptr=ptr(positions), **strides)
        self.ctx.paged_kv_append_device(self.h, r, stream=stream())

    def read(self, batch, fill=float("nan")):
        out = torch.full((2, batch.tokens, self.kv_heads * self.head_dim), fill, device=DEV)
        self.ctx.paged_kv_read_device(self.h, batch, ptr(out[0]), ptr(out[1]), stream=stream())
        return out.cpu()

    def request(self, batch, q, out, dtype, heads, scale, **strides):
        r = self.ctx.paged_attention_request(batch, dtype, heads, ptr(q), ptr(out), scale, **strides)
        n = self.ctx.paged_attention_workspace_bytes(self.h, r)
        assert n > 0, "request refused"
        work = torch.full((n,), 0xff, dtype=torch.uint8, device=DEV)   # NaN everywhere
        r.workspace = ptr(work)
        self.keep.append((work, r))
        return r

    def attend(self, batch, q, out, dtype, heads, scale, **strides):
        self.ctx.paged_kv_attention_device(self.h, self.request(batch, q, out, dtype, heads, scale, **strides), stream=stream())

    def close(self):
        torch.cuda.synchronize()
        self.ctx.paged_kv_destroy(self.h)


# ---- attention: which kernel takes a batch, and how far a row may be off -----------


def attention_path(dtype, past, new, kv_heads, heads, d, slots, pad=0):
    """(kernel, split) that the library's rules on sizes give a batch whose table rows hold `slots`
    slots: "block" (many bf16 rows), "prompt" or "decode" (16 rows), and whether a context may be
    shared among workgroups."""
    group, tokens, seqs = heads // kv_heads, max(1, sum(new) + pad), len(past)
    width = 64 if d <= 64 else 128 if d <= 128 else 256
    rows, used = tokens * group, min(seqs, tokens)
    many = rows >= 80 * seqs
    if many and dtype == "bf16" and (rows * kv_heads > 8192 or slots > 512):
        block = 64 if width == 256 else 128
        parts = max(1, min(8, 256 // ((rows + used * (block - 1)) // block * kv_heads)))
        longest = max(min(p + n, slots) for p, n in zip(past, new) if n)
        return "block", parts > 1 and -(-(-(-longest // 64)) // 2) > 4
    groups = min(rows, rows // 16 + used) * kv_heads
    eight = not many and width != 256 and groups < 256
    longer = groups >= 256 or (eight and (dtype != "f32" or groups >= 16))
    return "prompt" if many else "decode", slots > (1024 if longer else 512)


def attention_rows(kv, q, past, new, kv_heads, heads, d, scale, dtype, kernel, gone=()):
    """64-bit attention over the cached values kv [2][tokens][..], [rows][heads][d], and how far a row
    of it may be off in the 2-norm, [rows][heads].  `gone`: slots that are left out.

    With scores off by e_t, weights by w_t of themselves and values by y_t, a row o = sum p_t v_t moves
    by sum p_t ((e_t + w_t) (v_t - o) + y_t).  These are roundings: of zero mean and independent from
    token to token, the largest r (r / sqrt 3 in the root mean square), so the sum is held to 6 times
    the root of its squares' sum.  r is
    - of a score: about 20 fp32 sums, 2^-24 each of the magnitudes |q| (|k| + 16 steps) (the matrix
      cores' sums of subnormal codes, 16-bit rows, 2^-22), and fp32's queries in two halves 2^-22 of
      each product; in "block" the keys' rounding to f16, 2^-11 of each product;
    - of a weight: 2^-20 for the exponential and its argument; in "block" 2^-11, f16;
    - of a value: weight times step rounded, 2^-11 (two halves: 2^-22) of what it multiplies, the value
      less the middle of its group; in "block" 2^-11 of the value.
    The sums over n tokens are chains of n / 16 + 64 fp32 sums of magnitudes that grow as the root of
    the squares' sum and as the output; subnormal codes' are off by 2^-22 of a sum of 8 steps.  On top
    of it the output's own rounding."""
    group, half = heads // kv_heads, HALF[dtype]
    out, lim = [], []
    at = row = 0
    for p0, n in zip(past, new):
        total = p0 + n
        k, v = (kv[i, at:at + total].double().reshape(total, kv_heads, d) for i in range(2))
        at += total
        if not n:
            continue
        qs = q[row:row + n].double().reshape(n, heads, d)
        row += n
        see = torch.arange(total)[None] <= p0 + torch.arange(n)[:, None]
        for s in gone:
            see[:, s] = False
        for h in range(heads):
            kh, vh, qh = k[:, h // group], v[:, h // group], qs[:, h]
            s = (qh @ kh.t() * scale).masked_fill(~see, -float("inf"))
            p = torch.nan_to_num(torch.softmax(s, dim=1))
            o = p @ vh
            steps, middle = [], []
            for x in (kh, vh):
                lo = torch.cat([g.amin(1, keepdim=True).expand_as(g) for g in x.split(GROUP, 1)], 1)
                hi = torch.cat([g.amax(1, keepdim=True).expand_as(g) for g in x.split(GROUP, 1)], 1)
                steps.append((hi - lo) / 15)
                middle.append(lo + 8 * (hi - lo) / 15)
            products = ((qh ** 2) @ (kh ** 2).t()).sqrt()
            sums = qh.abs() @ (kh.abs() + 16 * steps[0]).t()
            e = (20 / 3) ** 0.5 * (2.0 ** -24 if dtype == "f32" else 2.0 ** -22) * sums
            e = e + 3 ** -0.5 * (2.0 ** -22 if dtype == "f32" else 2.0 ** -11 if kernel == "block" else 0.0) * products
            e = abs(scale) * e + 3 ** -0.5 * (2.0 ** -11 if kernel == "block" else 2.0 ** -20)
            away = ((vh ** 2).sum(1)[None] - 2 * o @ vh.t() + (o ** 2).sum(1)[:, None]).clamp_min(0)
            value = vh if kernel == "block" else vh - middle[1]
            y = 3 ** -0.5 * (2.0 ** -22 if dtype == "f32" else 2.0 ** -11) * (value ** 2).sum(1).sqrt()
            moved = ((p * e) ** 2 * away).sum(1).sqrt() + ((p * y[None]) ** 2).sum(1).sqrt()
            length = (o ** 2).sum(1).sqrt()
            chain = 2.0 ** -24 * (total / 16 + 64) ** 0.5 * (((p ** 2) @ (vh ** 2).sum(1)).sqrt() + length)
            if dtype != "f32":
                chain = chain + 2.0 ** -22 * p @ (8 * steps[1]).square().sum(1).sqrt()
            out.append(o)
            lim.append((half + 2.0 ** -23) * length + 6 * (moved + chain))
    rows = lambda x, *s: torch.cat([torch.stack(x[i:i + heads], 1) for i in range(0, len(x), heads)])  # noqa: E731
    return rows(out), rows(lim)
