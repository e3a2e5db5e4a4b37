"""Causal attention of packed sequences (qwn_hip_ext_prompt_attention_device), each row against the
definition in 64 bits."""
import math

import pytest
import torch

import serving as sv
from qwanto_amd import abi

pytestmark = pytest.mark.gpu


def rows_of(q, k, v, lengths, heads, kv_heads, d, scale, dtype):
    """64-bit attention of packed q, k, v, and how far each row and head may be off in the 2-norm:
    ([rows][heads][d], [rows][heads]).

    With scores off by e_t and weights by w_t of themselves, a row o = sum p_t v_t moves by
    sum p_t (e_t + w_t) (v_t - o); a weight that is rounded only where it meets a value, by r_t, moves
    it by sum p_t r_t v_t.  These are roundings, of zero mean and independent from token to token, the
    largest r (r / sqrt 3 in the root mean square): the sum is held to 6 times the root of its squares'.
    - a score is a chain of at most d / 2 fp32 sums, 2^-24 each of the magnitudes |q| |k|;
    - an exponent is rounded to fp32: 2^-24 of |log2 p_t|, at most 2^-19 where p_t counts; its
      power of 2 by 2^-23;
    - a probability that meets a value is rounded to the type (fp32's is not).
    The sums over n tokens are chains of n / 2 + 64 fp32 sums of magnitudes that grow as the root of
    the squares' sum and as the output.  On top the output's own rounding."""
    half, group = sv.HALF[dtype], heads // kv_heads
    out, lim, at = [], [], 0
    for n in lengths:
        if not n:
            continue
        qs, ks, vs = (x[at:at + n].double().reshape(n, -1, d) for x in (q, k, v))
        at += n
        later = torch.ones(n, n).triu(1) > 0
        for h in range(heads):
            kh, vh, qh = ks[:, h // group], vs[:, h // group], qs[:, h]
            p = torch.softmax((qh @ kh.t() * scale).masked_fill(later, -math.inf), dim=1)
            o = p @ vh
            e = abs(scale) * (d / 6) ** 0.5 * 2.0 ** -24 * (qh.abs() @ kh.abs().t()) + 2.0 ** -19
            away = ((vh ** 2).sum(1)[None] - 2 * o @ vh.t() + (o ** 2).sum(1)[:, None]).clamp_min(0)
            moved = ((p * e) ** 2 * away).sum(1).sqrt()
            length = (o ** 2).sum(1).sqrt()
            squares = ((p ** 2) @ (vh ** 2).sum(1)).sqrt()
            if dtype != "f32":
                moved = moved + 3 ** -0.5 * half * squares
            chain = 2.0 ** -24 * (n / 2 + 64) ** 0.5 * (squares + length)
            out.append(o)
            lim.append((half + 2.0 ** -23) * length + 6 * (moved + chain))
    rows = lambda x: torch.cat([torch.stack(x[i:i + heads], 1) for i in range(0, len(x), heads)])  # noqa: E731
    return rows(out), rows(lim)


def inputs(seed, rows, heads, kv_heads, d, dtype):
    g = sv.gen(seed)
    scale = 0.3 + 1.2 * torch.rand(kv_heads * d, generator=g)
    dt = sv.DTYPES[dtype]
    return ((1.2 * sv.normal(g, rows, heads * d)).to(dt), (sv.normal(g, rows, kv_heads * d) * scale + 0.3).to(dt),
            (sv.normal(g, rows, kv_heads * d) * scale.flip(0)).to(dt))


def starts_of(lengths):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32)


def attend(ctx, q, k, v, lengths, heads, kv_heads, d, scale, dtype, out=None, starts=None, rows=None, **strides):
    """The output of tensors on the host or the GPU; rows that no sequence has keep 5."""
    dev = [x.to(sv.DEV) for x in (q, k, v)]
    if out is None:
        out = torch.full(dev[0].shape, 5.0, dtype=dev[0].dtype, device=sv.DEV)
    st = (starts if starts is not None else starts_of(lengths)).to(sv.DEV)
    r = ctx.prompt_attention_request(st.numel() - 1, rows or q.shape[0], sv.ptr(st), dtype, heads, kv_heads, d, *(sv.ptr(x) for x in dev),
                                     sv.ptr(out), scale, **strides)
    ctx.prompt_attention_device(r, stream=sv.stream())
    torch.cuda.synchronize()
    return out


def check(got, q, k, v, lengths, heads, kv_heads, d, scale, dtype):
    n = sum(lengths)
    want, lim = rows_of(q, k, v, lengths, heads, kv_heads, d, scale, dtype)
    off = (got[:n].cpu().double().reshape(n, heads, d) - want).square().sum(-1).sqrt()
    assert bool((off <= lim).all()), float((off / lim).max())
    assert bool((got[n:] == 5.0).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,lengths,pad", [
    (1, 1, 64, [1], 0),
    (12, 2, 128, [1, 2, 3], 2),
    (2, 2, 128, [31, 0, 32, 33], 1),
    (4, 2, 64, [63, 64, 65], 0),
    (3, 1, 128, [127, 128, 129, 0], 3),
    (32, 8, 128, [200, 1, 17], 0),
    (4, 1, 32, [150, 9], 0),
    (2, 1, 80, [100, 40], 1),
    (6, 2, 96, [70, 71], 0),
    (2, 1, 256, [90, 161], 0),
    (5, 5, 1, [40], 0),
    (2, 1, 33, [77, 5], 0),
    (2, 1, 200, [65], 0),
    (129, 1, 64, [3, 70], 0),
    (8, 1, 128, [600], 0),
    (2, 2, 64, [1000, 300], 0),
    (1, 1, 128, [2500], 0),
])
def test_sizes(gpu_ctx, dtype, heads, kv_heads, d, lengths, pad):
    q, k, v = inputs(d + sum(lengths), sum(lengths) + pad, heads, kv_heads, d, dtype)
    got = attend(gpu_ctx, q, k, v, lengths, heads, kv_heads, d, d ** -0.5, dtype)
    check(got, q, k, v, lengths, heads, kv_heads, d, d ** -0.5, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,lengths,pad", [(32, 16, 64, [1300, 0, 700, 511, 129], 2), (8, 2, 64, [640, 1, 1100], 0),
                                                          (4, 1, 40, [1029], 1), (40, 40, 56, [515], 0), (3, 1, 63, [900, 127, 640], 3)])
def test_long_sequences_of_small_heads(gpu_ctx, dtype, heads, kv_heads, d, lengths, pad):
    """Sequences of 512 tokens and more on average, heads of up to 64 channels: larger tiles."""
    q, k, v = inputs(sum(lengths) + d, sum(lengths) + pad, heads, kv_heads, d, dtype)
    check(attend(gpu_ctx, q, k, v, lengths, heads, kv_heads, d, d ** -0.5, dtype), q, k, v, lengths, heads, kv_heads, d, d ** -0.5, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_masked_values_in_larger_tiles(gpu_ctx, dtype):
    """Values that are not finite in the last tiles reach the rows that see them, and no other."""
    n, d = 700, 64
    q, k, v = inputs(3, n, 4, 2, d, dtype)
    clean = attend(gpu_ctx, q, k, v, [n], 4, 2, d, 0.125, dtype).cpu()
    for t in (0, 63, 64, 127, 128, 300, 447, 640, 699):
        b = v.clone()
        b[t, 5], b[t, d + 9] = math.inf, math.nan
        got = attend(gpu_ctx, q, k, b, [n], 4, 2, d, 0.125, dtype).cpu()
        assert bool((got[t:, [5, d + 5]] == math.inf).all()) and bool(torch.isnan(got[t:, [2 * d + 9, 3 * d + 9]]).all()), t
        got[t:, [5, d + 5, 2 * d + 9, 3 * d + 9]] = clean[t:, [5, d + 5, 2 * d + 9, 3 * d + 9]]
        assert torch.equal(got, clean), t


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_many_sequences(gpu_ctx, dtype):
    """More sequences than a wave has lanes, most of one token and some of none."""
    lengths = [(i * 7) % 5 for i in range(200)] + [130] + [1] * 70
    q, k, v = inputs(3, sum(lengths), 4, 2, 64, dtype)
    got = attend(gpu_ctx, q, k, v, lengths, 4, 2, 64, 0.125, dtype)
    check(got, q, k, v, lengths, 4, 2, 64, 0.125, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,odd", [(4, 2, 128, 0), (6, 2, 64, 1), (2, 1, 80, 3), (2, 1, 33, 0)])
def test_columns_of_one_buffer(gpu_ctx, dtype, heads, kv_heads, d, odd):
    """Queries, keys and values side by side in a projection's rows, at any alignment, the output in
    a wider one: the same to the bit, and nothing beside it is touched."""
    lengths = [90, 41]
    n = sum(lengths)
    q, k, v = inputs(odd + d, n, heads, kv_heads, d, dtype)
    want = attend(gpu_ctx, q, k, v, lengths, heads, kv_heads, d, 0.1, dtype)
    edge = torch.full((n, odd), float("nan")).to(q.dtype)
    buf = torch.cat([edge, q, k, v, edge], dim=1).to(sv.DEV).contiguous()
    out = torch.full((n, heads * d + 2 * odd + 5), 5.0, dtype=q.dtype, device=sv.DEV)
    w, a, b = buf.shape[1], odd + heads * d, odd + (heads + kv_heads) * d
    attend(gpu_ctx, buf[:, odd:], buf[:, a:], buf[:, b:], lengths, heads, kv_heads, d, 0.1, dtype, out=out[:, odd:], query_stride=w,
           key_stride=w, value_stride=w, output_stride=out.shape[1])
    assert torch.equal(out[:, odd:odd + heads * d], want)
    assert bool((out[:, :odd] == 5.0).all()) and bool((out[:, odd + heads * d:] == 5.0).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_what_is_masked_does_not_count(gpu_ctx, dtype, d):
    """Keys and values that are not finite, or the type's largest, behind a row and in other sequences
    leave it as it was to the bit; in front of it they show in it, values in their channel alone."""
    heads, kv_heads, lengths = 4, 2, [150, 70]
    q, k, v = inputs(d, 221, heads, kv_heads, d, dtype)
    k[220], v[220] = float("nan"), float("nan")                  # of no sequence
    clean = attend(gpu_ctx, q, k, v, lengths, heads, kv_heads, d, 0.1, dtype)
    top = torch.finfo(q.dtype).max
    for t, bad in ((149, float("nan")), (100, float("inf")), (128, -float("inf")), (37, float("nan")), (149, top), (0, float("nan"))):
        kb, vb = k.clone(), v.clone()
        kb[t, :d] = bad
        vb[t, d + 3] = bad
        rows = torch.arange(221)
        before = (rows < t) | (rows >= 150)
        got = attend(gpu_ctx, q, k, vb, lengths, heads, kv_heads, d, 0.1, dtype).cpu()
        assert torch.equal(got[before], clean.cpu()[before]), (t, bad)
        after = got[t:150].reshape(150 - t, heads, d)
        others = torch.ones(heads, d, dtype=torch.bool)
        others[2:, 3] = False
        assert torch.equal(after[:, others], clean[t:150].cpu().reshape(150 - t, heads, d)[:, others]), (t, bad)
        if bad != top:
            assert not bool(torch.isfinite(after[:, 2:, 3]).any()), (t, bad)
            if not math.isnan(bad):
                assert bool((after[:, 2:, 3] == bad).all()), (t, bad)
        got = attend(gpu_ctx, q, kb, v, lengths, heads, kv_heads, d, 0.1, dtype).cpu()
        assert torch.equal(got[before], clean.cpu()[before]), (t, bad)
        assert torch.equal(got[:, 2 * d:], clean[:, 2 * d:].cpu()), (t, bad)      # the other KV head
        if math.isnan(bad):
            assert bool(torch.isnan(got[t:150, :2 * d]).all()), (t, bad)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_values_of_both_infinities(gpu_ctx, dtype):
    q, k, v = inputs(1, 40, 1, 1, 64, dtype)
    v[10, 7], v[20, 7], v[15, 9] = math.inf, -math.inf, -math.inf
    got = attend(gpu_ctx, q, k, v, [40], 1, 1, 64, 0.125, dtype).cpu()
    assert bool(torch.isfinite(got[:10]).all())
    assert bool((got[10:20, 7] == math.inf).all()) and bool(torch.isnan(got[20:, 7]).all())
    assert bool((got[15:, 9] == -math.inf).all())
    rest = [c for c in range(64) if c not in (7, 9)]
    assert bool(torch.isfinite(got[:, rest]).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_size,k_size,scale", [(1.0, 1.0, -0.3), (1.0, 1.0, 0.0), (60.0, 60.0, 1.0), (3e4, 3e4, 1.0), (3e4, 3e4, -1e30),
                                                 (1e-4, 1.0, 1e4), (1.0, 1.0, 1e-40), (1.0, 1.0, 3e38)])
def test_scores_of_any_size(gpu_ctx, dtype, q_size, k_size, scale):
    """Against the definition in 64 bits: softmax of scores whose largest is far from the next is the
    value of one token."""
    lengths, d = [70, 33], 64
    g = sv.gen(5)
    dt = sv.DTYPES[dtype]
    q, k, v = ((s * (2 * torch.rand(103, d, generator=g) - 1)).to(dt) for s in (q_size, k_size, 1.0))
    got = attend(gpu_ctx, q, k, v, lengths, 1, 1, d, scale, dtype)
    scale = float(torch.tensor(scale, dtype=torch.float32))
    want, lim = rows_of(q, k, v, lengths, 1, 1, d, scale, dtype)
    off = (got.cpu().double().reshape(103, 1, d) - want).square().sum(-1).sqrt()
    # where scores are so large that their own roundings decide between tokens, the row is one or the other
    clear = []
    at = 0
    for n in lengths:
        s = (q[at:at + n].double() @ k[at:at + n].double().t() * scale).masked_fill(torch.ones(n, n).triu(1) > 0, -math.inf)
        e = abs(scale) * (d / 2) * 2.0 ** -24 * (q[at:at + n].double().abs() @ k[at:at + n].double().abs().t())
        best = s.topk(min(2, n), dim=1).values
        gap = best[:, 0] - best[:, -1] if n > 1 else torch.full((n,), math.inf, dtype=torch.float64)
        clear.append((gap > 2 * e.max(dim=1).values + 40) | (e.max(dim=1).values < 1e-3))
        at += n
    clear = torch.cat(clear)
    assert bool(clear.float().mean() > 0.9)
    assert bool((off[clear] <= lim[clear] + 1e-9).all())
    assert bool(torch.isfinite(got).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scores_past_fp32(gpu_ctx, dtype):
    """Products past fp32's largest: the row is the value of its best token."""
    d = 64
    g = sv.gen(6)
    dt = sv.DTYPES[dtype]
    q, k, v = ((s * (2 * torch.rand(50, d, generator=g) - 1)).to(dt) for s in (1e37, 1e38, 1.0))
    for scale in (1.0, -1e20, 1e-30):
        got = attend(gpu_ctx, q, k, v, [50], 1, 1, d, scale, dtype).cpu().double()
        s = (q.double() @ k.double().t() * scale).masked_fill(torch.ones(50, 50).triu(1) > 0, -math.inf)
        want = v.double()[s.argmax(dim=1)]
        assert bool(((got - want).abs() <= (sv.HALF[dtype] + 2.0 ** -22) * want.abs()).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q_size,k_size,scale", [(1.0, 1e36, 1e-36), (1e-30, 1e36, 1e-6), (1e-20, 3e37, 1e-18), (1e30, 1e-30, 1.0), (1e-36, 1e36, -1.0),
                                                 (30.0, 3e37, 1e-38), (1e-5, 1e37, 2e-33), (1e38, 1e-34, 1e-4), (1e-38, 1e38, 1.0)])
@pytest.mark.parametrize("d,n", [(64, 150), (128, 70)])
def test_ordinary_scores_of_factors_of_any_size(gpu_ctx, dtype, q_size, k_size, scale, d, n):
    """Queries, keys and a scale of which no product is out of the ordinary, though each may be."""
    g = sv.gen(12)
    dt = sv.DTYPES[dtype]
    q, k, v = ((s * (2 * torch.rand(n, d, generator=g) - 1)).to(dt) for s in (q_size, k_size, 1.0))
    scale = float(torch.tensor(scale, dtype=torch.float32))
    s = q.double() @ k.double().t() * scale
    assert 0.01 < float(s.std()) < 100
    check(attend(gpu_ctx, q, k, v, [n], 1, 1, d, scale, dtype), q, k, v, [n], 1, 1, d, scale, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_queries_and_scales_that_are_not_finite(gpu_ctx, dtype):
    q, k, v = inputs(2, 40, 2, 1, 64, dtype)
    clean = attend(gpu_ctx, q, k, v, [40], 2, 1, 64, 0.125, dtype).cpu()
    for bad in (math.nan, math.inf, -math.inf):
        b = q.clone()
        b[7, 64 + 5] = bad
        got = attend(gpu_ctx, b, k, v, [40], 2, 1, 64, 0.125, dtype).cpu()
        assert bool(torch.isnan(got[7, 64:]).all())
        got[7, 64:] = clean[7, 64:]
        assert torch.equal(got, clean)
        assert bool(torch.isnan(attend(gpu_ctx, q, k, v, [40], 2, 1, 64, bad, dtype)).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,heads,kv_heads,lengths", [(64, 2, 1, [300, 40]), (64, 2, 1, [600]), (128, 2, 2, [300]), (256, 1, 1, [200, 70]),
                                                      (96, 2, 1, [150]), (33, 1, 1, [140]), (64, 80, 80, [200, 190]), (128, 80, 80, [150, 140]),
                                                      (256, 80, 80, [150, 140])])
def test_large_values(gpu_ctx, dtype, d, heads, kv_heads, lengths):
    """Finite values up to the type's largest, scores that rise along the sequence or not: outputs are averages of values,
    so they are finite, and those of other channels are what they were to the bit."""
    n, top = sum(lengths), torch.finfo(sv.DTYPES[dtype]).max
    q, k, v = inputs(d + heads, n, heads, kv_heads, d, dtype)
    t = torch.cat([torch.arange(m) for m in lengths])
    for rise in (0.0, 0.3, 3.0):
        q2, k2 = q.clone(), k.clone()
        if rise:                                                                  # scores of about rise * token, of any query
            q2.reshape(n, heads, d)[:, :, 0] = 4.0
            k2.reshape(n, kv_heads, d)[:, :, 0] = (rise / 0.4 * t)[:, None].to(k.dtype)
        clean = attend(gpu_ctx, q2, k2, v, lengths, heads, kv_heads, d, 0.1, dtype).cpu().reshape(n, heads, d)
        check(clean.reshape(n, -1), q2, k2, v, lengths, heads, kv_heads, d, 0.1, dtype)
        for size in (top, 0.99 * top, 2.0 ** 100 if dtype != "f16" else 2.0 ** 14):
            b = v.clone()
            x = b.reshape(n, kv_heads, d)
            x[:, :, 3] = size                                                     # all alike: the row's, too
            x[:, :, 7] = (size * (2 * torch.rand(n, kv_heads, generator=sv.gen(1)) - 1)).to(v.dtype)
            x[-1, :, 9] = -size
            got = attend(gpu_ctx, q2, k2, b, lengths, heads, kv_heads, d, 0.1, dtype).cpu()
            assert bool(torch.isfinite(got).all())
            got = got.reshape(n, heads, d)
            others = [c for c in range(d) if c not in (3, 7, 9)]
            assert torch.equal(got[:, :, others], clean[:, :, others])
            assert torch.equal(got[:-1, :, 9], clean[:-1, :, 9])
            big = torch.zeros_like(b).reshape(n, kv_heads, d)
            big[:, :, [3, 7, 9]] = x[:, :, [3, 7, 9]]
            alone = torch.zeros_like(got)
            alone[:, :, [3, 7, 9]] = got[:, :, [3, 7, 9]]
            # the large channels by themselves: their sizes, not the others', are what they may be off by
            for ch in (3, 7, 9):
                one, mine = torch.zeros_like(big), torch.zeros_like(alone)
                one[:, :, ch], mine[:, :, ch] = big[:, :, ch], alone[:, :, ch]
                check(mine.reshape(n, -1), q2, k2, one.reshape(n, -1), lengths, heads, kv_heads, d, 0.1, dtype)


def test_large_values_beside_what_is_not_finite(gpu_ctx):
    """A row with an infinite value in one channel and large finite ones in another, in tiles that are masked and
    that are not."""
    n, d = 260, 64
    for dtype in ("f32", "bf16"):
        top = torch.finfo(sv.DTYPES[dtype]).max
        q, k, v = inputs(8, n, 1, 1, d, dtype)
        q[:, 0], k[:, 0] = 4.0, torch.arange(n).to(q.dtype)
        v[:, 5] = top
        v[100, 9], v[230, 11] = math.inf, math.nan
        got = attend(gpu_ctx, q, k, v, [n], 1, 1, d, 0.1, dtype).cpu().double()
        assert bool(((got[:, 5] - top).abs() <= ((2 * sv.HALF[dtype] if dtype == "bf16" else 0) + 2.0 ** -20) * top).all())
        assert bool(torch.isfinite(got[:100]).all()) and bool(torch.isfinite(got[:230, 11]).all())
        assert bool((got[100:, 9] == math.inf).all()) and bool(torch.isnan(got[230:, 11]).all())
        rest = [c for c in range(d) if c not in (9, 11)]
        assert bool(torch.isfinite(got[:, rest]).all())


@pytest.mark.parametrize("d,heads,n,late", [(64, 1, 1500, 0), (64, 48, 1100, 3), (128, 1, 1500, 70), (256, 1, 700, 0), (128, 40, 1100, 0)])
@pytest.mark.parametrize("below", [18.0, 20.5, 23.3, 25.0, 27.7])
def test_small_probabilities_add_up(gpu_ctx, below, d, heads, n, late):
    """One token has nearly all of the weight and a value of nothing, the others 2^-18 of it and less each: what they add
    up to is there in f16, too.  A probability that is rounded to f16 2^6 times as large as it is to the row's largest is
    off by 2^-11 of itself, or by 2^-31 of the largest where it is below f16's normal numbers; beside that the fp32 chains
    and roundings of rows_of, in whole: 2^-16 of a probability."""
    g = sv.gen(int(10 * below) + d)
    q, k = torch.zeros(n, heads, d), torch.zeros(n, 1, d)
    q[:, :, 0], q[:, :, 1] = 1.0, 1.0
    k[:, 0, 0] = -below * math.log(2.0)                                          # scale 1: rounded to f16, and taken as it is
    k[:, 0, 1] = 0.1 * sv.normal(g, n)
    k[late, 0, :2] = 0.0
    v = 0.5 + torch.rand(n, 1, d, generator=g)
    v[late] = 0.0
    q, k, v = (x.half().reshape(n, -1) for x in (q, k, v))
    got = attend(gpu_ctx, q, k, v, [n], heads, 1, d, 1.0, "f16").cpu().double().reshape(n, heads, d)
    s = (q.double()[:, :d] @ k.double().t()).masked_fill(torch.ones(n, n).triu(1) > 0, -math.inf)
    p = torch.softmax(s, dim=1)
    want = (p @ v.double())[:, None]
    size = v.double().abs()
    off = (2.0 ** -11 + 2.0 ** -16) * (p @ size) + 2.0 ** -31 * (p.amax(1, keepdim=True) * torch.tril(torch.ones(n, n)).double()) @ size
    assert bool(((got - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -25 + off[:, None]).all())


def test_query_channels_far_apart(gpu_ctx):
    """f16 queries with a channel of the type's largest and others of its smallest numbers, which decide."""
    d, n = 64, 50
    g = sv.gen(11)
    q, k = torch.zeros(n, d), torch.zeros(n, d)
    q[:, 0] = 65504.0
    q[:, 1:9] = 2.0 ** -24 * torch.randint(1, 8, (n, 8), generator=g)
    k[:, 1:9] = 60000 * (2 * torch.rand(n, 8, generator=g) - 1)
    q, k, v = q.half(), k.half(), sv.normal(g, n, d).half()
    for scale in (1.0, 100.0, -30.0):
        got = attend(gpu_ctx, q, k, v, [n], 1, 1, d, scale, "f16")
        check(got, q, k, v, [n], 1, 1, d, scale, "f16")


def test_starts_that_are_none(gpu_ctx):
    """Sequences whose rows do not lie in the batch are left out, the others are not."""
    q, k, v = inputs(4, 100, 2, 1, 64, "bf16")
    for starts, good in (([0, 30, 101], [(0, 30)]), ([-1, 30, 60], [(30, 60)]), ([40, 10, 60], [(10, 60)]), ([0, 0, 0], []),
                         ([5, 2 ** 31 - 1, 7], []), ([20, 100, 100], [(20, 100)]), ([0, -2 ** 31, 9], [])):
        got = attend(gpu_ctx, q, k, v, None, 2, 1, 64, 0.125, "bf16", starts=torch.tensor(starts, dtype=torch.int32))
        kept = torch.ones(100, dtype=torch.bool)
        for a, b in good:
            part = got[a:b]
            check(part, q[a:b], k[a:b], v[a:b], [b - a], 2, 1, 64, 0.125, "bf16")
            kept[a:b] = False
        assert bool((got.cpu()[kept] == 5.0).all()), starts


def test_rows_far_apart(gpu_ctx):
    """Row offsets past 32 bits."""
    stride, n, d = 2 ** 31 + 8, 5, 64
    q, k, v = inputs(9, n, 1, 1, d, "bf16")
    want = attend(gpu_ctx, q, k, v, [n], 1, 1, d, 0.125, "bf16")
    buf = torch.empty((n - 1) * stride + 4 * d, dtype=torch.bfloat16, device=sv.DEV)
    wide = torch.as_strided(buf, (n, 4 * d), (stride, 1))
    wide.copy_(torch.cat([q, k, v, torch.full_like(q, 5.0)], dim=1))
    cols = [wide[:, i * d:(i + 1) * d] for i in range(4)]
    attend(gpu_ctx, *cols[:3], [n], 1, 1, d, 0.125, "bf16", out=cols[3], query_stride=stride, key_stride=stride, value_stride=stride,
           output_stride=stride)
    assert torch.equal(cols[3], want)


def test_refusals(gpu_ctx):
    n, d = 6, 64
    buf = torch.zeros(n + 1, 6 * d, device=sv.DEV)
    st = torch.tensor([0, n], dtype=torch.int32, device=sv.DEV)
    at = lambda row, col: sv.ptr(buf) + (row * 6 * d + col) * 4  # noqa: E731

    def req(**kw):
        base = dict(sequences=1, tokens=n, starts_ptr=sv.ptr(st), dtype="f32", query_heads=2, kv_heads=1, head_dim=d, q_ptr=at(0, 0),
                    k_ptr=at(0, 2 * d), v_ptr=at(0, 3 * d), out_ptr=at(0, 4 * d), scale=0.1, query_stride=6 * d, key_stride=6 * d,
                    value_stride=6 * d, output_stride=6 * d)
        base.update(kw)
        return gpu_ctx.prompt_attention_request(**base)

    def status(r):
        with pytest.raises(abi.AbiError) as e:
            gpu_ctx.prompt_attention_device(r, stream=sv.stream())
        return e.value.status

    for good in (req(), req(v_ptr=at(0, 2 * d)), req(k_ptr=at(0, 0))):
        gpu_ctx.prompt_attention_device(good, stream=sv.stream())
    for bad in (dict(sequences=0), dict(tokens=0), dict(starts_ptr=None), dict(query_heads=0), dict(kv_heads=0), dict(head_dim=0),
                dict(q_ptr=None), dict(k_ptr=None), dict(v_ptr=None), dict(out_ptr=None), dict(query_stride=d), dict(key_stride=d - 1),
                dict(value_stride=1), dict(output_stride=2 * d - 1), dict(out_ptr=at(0, 0)), dict(out_ptr=at(0, 1)), dict(out_ptr=at(1, d)),
                dict(out_ptr=at(0, 3 * d + 1)), dict(out_ptr=at(0, 2 * d - 1)), dict(out_ptr=sv.ptr(st) - 4, output_stride=2 * d)):
        assert status(req(**bad)) == -1, bad
    for bad in (dict(head_dim=257, query_stride=0, key_stride=0, value_stride=0, output_stride=0), dict(query_heads=3, kv_heads=2, head_dim=16),
                dict(tokens=2 ** 31 - 1, out_ptr=at(0, 0) + 2 ** 50)):
        assert status(req(**bad)) == -5, bad
    r = req()
    r.dtype = 3
    assert status(r) == -1
    r = req()
    r.header.abi_version = 2
    assert status(r) == -1
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_captured_and_on_two_streams(gpu_ctx, dtype):
    """Recorded once and replayed with other sequences, eager calls on another stream between: the same
    to the bit, and rows of no sequence stay."""
    n, heads, kv_heads, d = 400, 4, 2, 128
    q, k, v = (x.to(sv.DEV) for x in inputs(7, n, heads, kv_heads, d, dtype))
    st = torch.zeros(4, dtype=torch.int32, device=sv.DEV)
    out, want = torch.zeros_like(q), torch.zeros_like(q)
    req = lambda o: gpu_ctx.prompt_attention_request(3, n, sv.ptr(st), dtype, heads, kv_heads, d, sv.ptr(q), sv.ptr(k), sv.ptr(v),  # noqa: E731
                                                     sv.ptr(o), 0.1)
    r, e = req(out), req(want)
    gpu_ctx.prompt_attention_device(e, stream=sv.stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu_ctx.prompt_attention_device(r, stream=sv.stream())
    side = torch.cuda.Stream()
    for starts in ([0, 400, 400, 400], [0, 1, 200, 333], [0, 0, 130, 260], [0, 399, 399, 400]):
        st.copy_(torch.tensor(starts, dtype=torch.int32))
        out.fill_(2.0)
        want.fill_(2.0)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            gpu_ctx.prompt_attention_device(e, stream=sv.stream())
        torch.cuda.synchronize()
        assert torch.equal(out, want), starts
        assert bool((out[starts[-1]:] == 2.0).all())


def groups_of(lengths, heads, kv_heads, pad=0):
    """Workgroups that blocks of 128 rows would make: from 320 on these are taken."""
    tokens, group = sum(lengths) + pad, heads // kv_heads
    return (tokens * group + min(len(lengths), tokens) * 127) // 128 * kv_heads


LARGE = [(32, 8, 128, [700, 0, 530, 1, 129], 3), (16, 16, 96, [1300, 1200], 0), (40, 40, 256, [600, 450], 1), (40, 40, 200, [700, 300], 0),
         (36, 36, 33, [640, 500], 2), (32, 32, 80, [257, 900], 0), (64, 32, 64, [100] * 7, 1), (48, 48, 40, [900], 0)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,lengths,pad", LARGE)
def test_blocks_of_128_rows(gpu_ctx, dtype, heads, kv_heads, d, lengths, pad):
    """Batches that fill the GPU, in blocks of 128 rows: every width, heads narrower than it, unaligned rows."""
    assert groups_of(lengths, heads, kv_heads, pad) >= 320
    q, k, v = inputs(d + sum(lengths), sum(lengths) + pad, heads, kv_heads, d, dtype)
    got = attend(gpu_ctx, q, k, v, lengths, heads, kv_heads, d, d ** -0.5, dtype)
    check(got, q, k, v, lengths, heads, kv_heads, d, d ** -0.5, dtype)
    # columns of one buffer, at an odd element
    n = q.shape[0]
    buf = torch.cat([torch.full((n, 3), float("nan")).to(q.dtype), q, k, v], dim=1).to(sv.DEV).contiguous()
    a, b = 3 + heads * d, 3 + (heads + kv_heads) * d
    odd = torch.full_like(got, 5.0)
    attend(gpu_ctx, buf[:, 3:], buf[:, a:], buf[:, b:], lengths, heads, kv_heads, d, d ** -0.5, dtype, out=odd, query_stride=buf.shape[1],
           key_stride=buf.shape[1], value_stride=buf.shape[1], output_stride=heads * d)
    assert torch.equal(odd, got)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,n", [(32, 8, 128, 1280), (40, 40, 256, 1027), (36, 36, 33, 1150), (64, 32, 64, 700), (24, 24, 200, 1707)])
def test_what_is_masked_in_blocks_of_128_rows(gpu_ctx, dtype, heads, kv_heads, d, n):
    """Values and keys that are not finite leave the rows before them, and other heads and channels, as they were to the
    bit; values show in their channel of the rows that see them."""
    assert groups_of([n], heads, kv_heads) >= 320
    group = heads // kv_heads
    q, k, v = (x.to(sv.DEV) for x in inputs(n, n, heads, kv_heads, d, dtype))
    clean = attend(gpu_ctx, q, k, v, [n], heads, kv_heads, d, 0.1, dtype)
    for t in (0, 31, 32, 63, 64, 127, 128, 500, n - 33, n - 1):
        b = v.clone()
        b[t, 5], b[t, (kv_heads - 1) * d + 9] = -math.inf, math.nan
        got = attend(gpu_ctx, q, k, b, [n], heads, kv_heads, d, 0.1, dtype).reshape(n, heads, d)
        assert bool((got[t:, :group, 5] == -math.inf).all()) and bool(torch.isnan(got[t:, heads - group:, 9]).all()), t
        got[t:, :group, 5] = clean.reshape(n, heads, d)[t:, :group, 5]
        got[t:, heads - group:, 9] = clean.reshape(n, heads, d)[t:, heads - group:, 9]
        assert torch.equal(got.reshape(n, -1), clean), t
        b = k.clone()
        b[t, d:] = math.nan                                                      # all KV heads but the first
        got = attend(gpu_ctx, q, b, v, [n], heads, kv_heads, d, 0.1, dtype)
        assert torch.equal(got[:t], clean[:t]) and torch.equal(got[:, :group * d], clean[:, :group * d]), t
        assert bool(torch.isnan(got[t:, group * d:]).all()), t


@pytest.mark.parametrize("dtype,heads,kv_heads,d,n", [("bf16", 32, 8, 128, 1400), ("f16", 64, 32, 64, 800)])
def test_blocks_of_128_rows_captured_and_on_two_streams(gpu_ctx, dtype, heads, kv_heads, d, n):
    q, k, v = (x.to(sv.DEV) for x in inputs(7, n, heads, kv_heads, d, dtype))
    st = torch.zeros(4, dtype=torch.int32, device=sv.DEV)
    out, want = torch.zeros_like(q), torch.zeros_like(q)
    req = lambda o: gpu_ctx.prompt_attention_request(3, n, sv.ptr(st), dtype, heads, kv_heads, d, sv.ptr(q), sv.ptr(k), sv.ptr(v),  # noqa: E731
                                                     sv.ptr(o), 0.1)
    assert groups_of([n, 0, 0], heads, kv_heads) >= 320
    r, e = req(out), req(want)
    gpu_ctx.prompt_attention_device(e, stream=sv.stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu_ctx.prompt_attention_device(r, stream=sv.stream())
    side = torch.cuda.Stream()
    for starts in ([0, n, n, n], [0, 1, 200, n - 70], [0, 0, 130, 260], [0, n - 1, n - 1, n]):
        st.copy_(torch.tensor(starts, dtype=torch.int32))
        out.fill_(2.0)
        want.fill_(2.0)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            gpu_ctx.prompt_attention_device(e, stream=sv.stream())
        torch.cuda.synchronize()
        assert torch.equal(out, want), starts
        assert bool((out[starts[-1]:] == 2.0).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d,lengths,pad", LARGE + [(64, 64, 64, [640], 0), (64, 64, 24, [640], 0)])
def test_large_values_in_blocks_of_128_rows(gpu_ctx, dtype, heads, kv_heads, d, lengths, pad):
    """A channel of the type's largest in every token is that in every row, whatever the weights; the other channels are
    what they are without it, to the bit; eager and replayed."""
    assert groups_of(lengths, heads, kv_heads, pad) >= 320
    n, top = sum(lengths), torch.finfo(sv.DTYPES[dtype]).max
    q, k, v = (x.to(sv.DEV) for x in inputs(d, n + pad, heads, kv_heads, d, dtype))
    q.reshape(n + pad, heads, d)[:, :, 0] = 4.0
    k.reshape(n + pad, kv_heads, d)[:, :, 0] = torch.arange(n + pad, device=sv.DEV)[:, None].to(k.dtype)
    clean = attend(gpu_ctx, q, k, v, lengths, heads, kv_heads, d, 0.1, dtype).reshape(-1, heads, d)
    v.reshape(n + pad, kv_heads, d)[:, -1, 3] = top
    st, out = starts_of(lengths).to(sv.DEV), torch.full_like(q, 5.0)
    r = gpu_ctx.prompt_attention_request(len(lengths), n + pad, sv.ptr(st), dtype, heads, kv_heads, d, sv.ptr(q), sv.ptr(k), sv.ptr(v),
                                         sv.ptr(out), 0.1)
    gpu_ctx.prompt_attention_device(r, stream=sv.stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu_ctx.prompt_attention_device(r, stream=sv.stream())
    last = heads - heads // kv_heads
    for replay in range(3):
        if replay:
            out.fill_(5.0)
            graph.replay()
            torch.cuda.synchronize()
        got = out.reshape(-1, heads, d)
        # every weight is off by half a step of the type, and so is the output; sums and powers by less than 2^-18
        assert bool((got[:n, last:, 3].double() >= top * (1 - 2 * sv.HALF[dtype] - 2.0 ** -18)).all())
        assert bool(torch.isfinite(got).all())
        rest = got.clone()
        rest[:n, last:, 3] = clean[:n, last:, 3]
        assert torch.equal(rest, clean)
