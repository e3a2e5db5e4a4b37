"""The paged 4-bit KV cache: append with rotation, read back, and attention
over it, against their definitions in 64 bits."""
import math

import pytest
import torch

import serving as sv
from qwanto_amd import abi

pytestmark = pytest.mark.gpu


def inputs(seed, rows, kv_heads, head_dim, dtype, heads=0):
    g = sv.gen(seed)
    c = kv_heads * head_dim
    scale = 0.3 + 1.2 * torch.rand(c, generator=g)
    offset = torch.where(torch.rand(c, generator=g) < 0.05, 4.0, 0.3) * sv.normal(g, c)
    dt = sv.DTYPES[dtype]
    k = (sv.normal(g, rows, c) * scale + offset).to(dt)
    v = (sv.normal(g, rows, c) * scale.flip(0)).to(dt)
    q = (1.2 * sv.normal(g, rows, heads * head_dim)).to(dt) if heads else None
    return k, v, q


def positions_of(past, new):
    return torch.tensor([p + i for p, n in zip(past, new) for i in range(n)], dtype=torch.int64)


def check_cached(got, x, rotated):
    """got [rows][heads][dim]: the 4-bit form of fp32 x.  Rotated values may come out of another
    library's sine by an ulp of 64 bits: a code may differ where its quotient lies on a border to
    1e-6, by one step."""
    want, step, _, t = sv.levels(x)
    off = (got.double() - want).abs()
    exact = off <= 2.0 ** -23 * want.abs() + 1e-12   # fp32's rounding of minimum + step * code
    if not rotated:
        assert bool(exact.all())
        return
    border = ((t - t.floor()) - 0.5).abs() < 1e-6
    assert bool((exact | (border & (off <= step * (1 + 1e-6)))).all())
    assert float((~exact).double().mean()) < 1e-3


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv_heads,head_dim,page,rope", [(2, 128, 16, 128), (1, 64, 32, 64), (3, 80, 16, 80), (2, 32, 64, 20),
                                                        (1, 256, 16, 256), (2, 96, 128, 0), (1, 65, 16, 64), (5, 2, 16, 2)])
def test_append_and_read(gpu_ctx, dtype, kv_heads, head_dim, page, rope):
    heads = 2 * kv_heads
    past, new = [0, 5, 15, 33, 7], [1, 3, 18, 0, 1]
    rows, pad = sum(new), 2
    c = sv.Cache(gpu_ctx, [p + n for p, n in zip(past, new)], kv_heads, head_dim, page, rope, seed=head_dim)
    try:
        b = c.batch(past, new, pad=pad)
        k, v, q = inputs(head_dim + rope, rows + pad, kv_heads, head_dim, dtype, heads)
        kd, vd, qd = k.to(sv.DEV), v.to(sv.DEV), q.to(sv.DEV)
        qo = torch.full_like(qd, 3.0)
        c.append(b, kd, vd, dtype, q=qd, q_out=qo, heads=heads)
        got = c.read(b)
        assert bool(torch.isnan(got[:, rows:]).all())               # rows of no sequence: untouched
        assert bool((qo[rows:] == 3.0).all())
        pos = positions_of(past, new)
        shape = (rows, -1, head_dim)
        kr = sv.rotate(k[:rows].reshape(shape), pos, rope, c.theta).float()
        check_cached(got[0, :rows].reshape(shape), kr, rope > 0)
        check_cached(got[1, :rows].reshape(shape), v[:rows].reshape(shape).float(), False)
        qr = sv.rotate(q[:rows].reshape(shape), pos, rope, c.theta)
        # 64 bits rounded to fp32 and to the type
        tol = (2.0 ** -24 + sv.HALF[dtype]) * (1 + 1e-6) * qr.abs() + 2.0 ** -24
        assert bool(((qo[:rows].cpu().reshape(shape).double() - qr).abs() <= tol).all())
        # in place, and with the rows' own positions
        own = torch.randint(0, 200000, (rows + pad,), generator=sv.gen(3), dtype=torch.int32)
        c.append(b, kd, vd, dtype, q=qd, q_out=qd, heads=heads, positions=own.to(sv.DEV))
        qr = sv.rotate(q[:rows].reshape(shape), own[:rows], rope, c.theta)
        tol = (2.0 ** -24 + sv.HALF[dtype]) * (1 + 1e-6) * qr.abs() + 2.0 ** -24
        assert bool(((qd[:rows].cpu().reshape(shape).double() - qr).abs() <= tol).all())
        assert torch.equal(qd[rows:].cpu(), q[rows:])
    finally:
        c.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv_heads,head_dim,rope,odd", [(2, 128, 128, 0), (2, 64, 32, 3), (1, 80, 40, 1), (3, 65, 10, 5)])
def test_append_from_one_buffer(gpu_ctx, dtype, kv_heads, head_dim, rope, odd):
    """Queries, keys and values side by side in a projection's rows, at any alignment: the same codes
    and queries as from tensors of their own."""
    heads, past, new = 3 * kv_heads, [3, 0, 17], [6, 1, 30]
    rows = sum(new)
    k, v, q = inputs(head_dim, rows, kv_heads, head_dim, dtype, heads)
    c = sv.Cache(gpu_ctx, [p + n for p, n in zip(past, new)], kv_heads, head_dim, 16, rope)
    try:
        b = c.batch(past, new)
        qo = torch.zeros(rows, heads * head_dim, dtype=q.dtype, device=sv.DEV)
        c.append(b, k.to(sv.DEV), v.to(sv.DEV), dtype, q=q.to(sv.DEV), q_out=qo, heads=heads)
        want = c.read(b)
        zero = torch.zeros_like(k).to(sv.DEV)
        c.append(b, zero, zero, dtype)
        assert not bool(c.read(b).any())
        buf = torch.cat([torch.full((rows, odd), 9.0).to(q.dtype), q, k, v, torch.full((rows, odd), 9.0).to(q.dtype)], dim=1)
        dev = buf.to(sv.DEV).contiguous()
        w, qc, kc = dev.shape[1], heads * head_dim, kv_heads * head_dim
        at = lambda n: dev[:, n:]  # noqa: E731
        c.append(b, at(odd + qc), at(odd + qc + kc), dtype, q=at(odd), q_out=at(odd), heads=heads, key_stride=w, value_stride=w,
                 query_stride=w, query_out_stride=w)
        assert torch.equal(c.read(b), want)
        got = dev.cpu()
        assert torch.equal(got[:, odd:odd + qc], qo.cpu())                       # in place,
        got[:, odd:odd + qc] = q
        assert torch.equal(got, buf)                                             # and nothing beside it
    finally:
        c.close()


def test_tokens_one_by_one_equal_a_prompt(gpu_ctx):
    """The same slots written a token at a time, in runs of 3 and at once; neighbours in a word keep
    their codes, and other slots of the pool stay as they were."""
    n, hk, d = 37, 2, 128
    k, v, _ = inputs(8, n, hk, d, "f32")
    kd, vd = k.to(sv.DEV), v.to(sv.DEV)
    c = sv.Cache(gpu_ctx, [64, 64, 64, 64], hk, d)
    try:
        whole = c.batch([0, 0, 0, 0], [0, n, 0, 0])
        c.append(whole, kd, vd, "f32")
        want = c.read(whole)
        for i in range(n):
            c.append(c.batch([0, 0, i, 0], [0, 0, 1, 0]), kd[i:], vd[i:], "f32")
        assert torch.equal(c.read(c.batch([0, 0, 0, 0], [0, 0, n, 0])), want)
        for i in range(0, n, 3):
            c.append(c.batch([0, 0, 0, i], [0, 0, 0, min(3, n - i)]), kd[i:], vd[i:], "f32")
        assert torch.equal(c.read(c.batch([0, 0, 0, 0], [0, 0, 0, n])), want)
        assert torch.equal(c.read(whole), want)
        assert not bool(c.read(c.batch([0, n, n, n], [64, 64 - n, 64 - n, 64 - n])).any())
        # written over
        c.append(c.batch([0, 6, 0, 0], [0, 1, 0, 0]), kd[20:], vd[20:], "f32")
        again = c.read(whole)
        want[:, 6] = want[:, 20]
        assert torch.equal(again, want)
    finally:
        c.close()


def test_sequences_that_share_a_page(gpu_ctx):
    """Two sequences of one call whose tokens share a word of a shared page."""
    hk, d = 2, 64
    k, v, _ = inputs(9, 4, hk, d, "bf16")
    kd, vd = k.to(sv.DEV), v.to(sv.DEV)
    c = sv.Cache(gpu_ctx, [16, 16, 16, 16], hk, d)
    try:
        table = c.table[:1].repeat(4, 1).contiguous()
        b = c.batch([4, 5, 6, 7], [1, 1, 1, 1], table=table)
        for _ in range(3):
            c.append(b, kd, vd, "bf16")
            got = c.read(b)
            check_cached(got[0].reshape(4, hk, d), k.reshape(4, hk, d).float(), False)
            check_cached(got[1].reshape(4, hk, d), v.reshape(4, hk, d).float(), False)
            kd, vd, k, v = kd.flip(0).contiguous(), vd.flip(0).contiguous(), k.flip(0), v.flip(0)
    finally:
        c.close()


def test_values_that_are_extreme(gpu_ctx):
    """NaN and infinities are zeros, past f16 clamped; a constant group is its minimum; ties on a
    code's border go to the even code."""
    hk, d, n = 1, 128, 8
    k, v, _ = inputs(10, n, hk, d, "f32")
    k[0, 3], k[0, 70], v[0, 5] = math.nan, math.inf, -math.inf
    k[1] = 1e38 * torch.sign(k[1])
    v[1] = 1e-9 * v[1]
    k[2], v[2] = 2.5, -0.0
    k[3] = torch.arange(d) % 64 * 0.5           # 0 .. 31.5: step 2.1
    v[3] = (torch.arange(d) % 31) * 0.5         # 0 .. 15: step 1, every other value on a border
    k[4, :64] = 1e-6 * k[4, :64]
    kd, vd = k.to(sv.DEV), v.to(sv.DEV)
    c = sv.Cache(gpu_ctx, [n], hk, d)
    try:
        b = c.batch([0], [n])
        c.append(b, kd, vd, "f32")
        got = c.read(b)
        assert bool(torch.isfinite(got).all())
        check_cached(got[0].reshape(n, hk, d), k.reshape(n, hk, d), False)
        check_cached(got[1].reshape(n, hk, d), v.reshape(n, hk, d), False)
    finally:
        c.close()


def test_pages_that_the_table_does_not_name(gpu_ctx):
    """Slots of such pages are not stored, not read and not attended to; the other rows' results stay.
    (That the lookup turns them down is checked on the host.)"""
    hk, d, heads = 1, 64, 2
    k, v, q = inputs(11, 40, hk, d, "f32", heads)
    kd, vd, qd = k.to(sv.DEV), v.to(sv.DEV), q.to(sv.DEV)
    c = sv.Cache(gpu_ctx, [40], hk, d, extra=3)
    try:
        b = c.batch([0], [40])
        c.append(b, kd, vd, "f32")
        before = c.read(b)
        table = c.table.clone()
        table[0, 0], table[0, 1] = c.pages, -5
        bad = c.batch([0], [40], table=table)
        c.append(bad, kd.flip(0).contiguous(), vd.flip(0).contiguous(), "f32")
        after = c.read(b)
        assert torch.equal(after[:, :32], before[:, :32]) and not torch.equal(after[:, 32:], before[:, 32:])
        assert bool(torch.isnan(c.read(bad)[:, :32]).all())
        out = torch.full((40, heads * d), 5.0, device=sv.DEV)
        c.attend(bad, qd, out, "f32", heads, d ** -0.5)
        out = out.cpu()
        assert not bool(out[:32].any())                    # nothing left to attend to
        want, tol = reference(after[:, 32:], q[32:], [0], [8], hk, heads, d, d ** -0.5, "f32")
        assert bool(((out[32:].double() - want).abs() <= tol).all())
        # a table that ends before the sequence does
        short = c.batch([0], [40], table=c.table[:, :1].contiguous())
        c.attend(short, qd, (o := torch.full((40, heads * d), 5.0, device=sv.DEV)), "f32", heads, d ** -0.5)
        want, tol = reference(after, q, [0], [40], hk, heads, d, d ** -0.5, "f32", most=16)
        assert bool(((o.cpu().double() - want).abs() <= tol).all())
    finally:
        c.close()


def reference(kv, q, past, new, kv_heads, heads, d, scale, dtype, most=None, block=False, gone=None):
    """64-bit attention over the cached values kv [2][tokens][..] (whole sequences, one after the
    other), and how far an output may be from it.

    A score is fp32 sums of products of f16 halves: the query's two halves leave 2^-22 of the row's
    largest |q| (2^-25 absolute on one exact half of bf16 and f16), each of at most 8 + 4 + 4 sums in
    a chain rounds by 2^-24 (the matrix cores' own sums of 32 within that), against the sum of
    magnitudes |q| (15 step + |minimum|); its exponential has 2 more ulps and the argument's own
    rounding.  A relative error e of every probability moves the output by at most 2 e max|v|.
    Probabilities times step are halves with 2^-22 (one half: 2^-11) of themselves or 2^-25 of the
    largest; the sums over the tokens round by 2^-24 each, in chains of at most `n` tokens / 32 + 64.
    Where sequences bring many rows (`block`), bf16 ones meet keys and values rounded to f16: 2^-11 of
    each."""
    group, out, tols = heads // kv_heads, [], []
    at = row = 0
    for p, n in zip(past, new):
        k, v = (kv[i, at:at + p + n].double().reshape(p + n, kv_heads, d) for i in range(2))
        at += p + n
        if not n:
            continue
        qs = q[row:row + n].double().reshape(n, heads, d)
        row += n
        see = torch.arange(p + n)[None] <= p + torch.arange(n)[:, None]
        if most is not None:
            see &= torch.arange(p + n)[None] < most
        if gone is not None:
            see &= ~gone
        o, t = torch.zeros(n, heads, d, dtype=torch.float64), torch.zeros(n, heads, d, dtype=torch.float64)
        for h in range(heads):
            kh, vh = k[:, h // group], v[:, h // group]
            s = (qs[:, h] @ kh.t() * scale).masked_fill(~see, -math.inf)
            w = torch.nan_to_num(torch.softmax(s, dim=1))        # a row that sees nothing: zeros
            o[:, h] = w @ vh
            # |minimum| + 15 step of any group is at most 3 times its largest magnitude
            kmag = 3 * kh.abs().amax()
            vmag = 3 * vh.abs().amax()
            size = abs(scale) * qs[:, h].abs().sum(1) * kmag
            lost = 2.0 ** -22 if dtype == "f32" else 2.0 ** -25
            e_s = abs(scale) * qs[:, h].abs().amax(1) * d * lost * kmag + size * 20 * 2.0 ** -24
            e_p = 2.0 ** -22 if dtype == "f32" else 2.0 ** -11
            if block and dtype == "bf16":
                e_s = e_s + 2.0 ** -11 * abs(scale) * (qs[:, h].abs() @ kh.abs().t()).amax(1)
                e_p += 2.0 ** -11
            chain = ((p + n) / 32 + 64) * 2.0 ** -24
            err = (2 * (e_s + 2.0 ** -22) + e_p + 2.0 ** -24 + chain) * vmag
            t[:, h] = err[:, None] + (sv.HALF[dtype] + 2.0 ** -23) * o[:, h].abs()
        out.append(o.reshape(n, heads * d))
        tols.append(t.reshape(n, heads * d))
    return torch.cat(out), torch.cat(tols)


def attention_case(ctx, dtype, past, new, kv_heads, heads, d, page=16, scale=None, pad=0, seed=0, qs=0, os=0, slots=0):
    """`slots`: of a table row at least; a table for long contexts takes other kernels."""
    scale = d ** -0.5 if scale is None else scale
    total = [p + n for p, n in zip(past, new)]
    c = sv.Cache(ctx, total, kv_heads, d, page, seed=seed, width=max(-(-max(total) // page), -(-slots // page)))
    try:
        k, v, _ = inputs(seed + 1, sum(total), kv_heads, d, "f32")
        fill = c.batch([0] * len(total), total)
        c.append(fill, k.to(sv.DEV), v.to(sv.DEV), "f32")
        kv = c.read(fill)
        rows = sum(new)
        q = (1.2 * sv.normal(sv.gen(seed + 2), rows + pad, heads * d + qs)).to(sv.DTYPES[dtype])
        qd = q.to(sv.DEV)
        out = torch.full((rows + pad, heads * d + os), 7.0, dtype=sv.DTYPES[dtype], device=sv.DEV)
        c.attend(c.batch(past, new, pad=pad), qd, out, dtype, heads, scale, query_stride=q.shape[1], output_stride=out.shape[1])
        got = out.cpu()
        assert bool((got[rows:] == 7.0).all()) and bool((got[:, heads * d:] == 7.0).all())
        want, tol = reference(kv, q[:rows, :heads * d], past, new, kv_heads, heads, d, scale, dtype,
                              block=rows * (heads // kv_heads) >= 64 * len(past))
        off = (got[:rows, :heads * d].double() - want).abs()
        assert bool((off <= tol).all()), f"off by {float((off / tol).max()):.2f} of the bound"
        return got
    finally:
        c.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("past,new,kv_heads,heads,d,page", [
    ([0], [1], 1, 1, 64, 16),                                  # a single token
    ([0, 0, 0], [1, 2, 3], 2, 4, 128, 16),
    ([15, 16, 17, 0, 31, 300], [1, 1, 1, 0, 1, 1], 2, 12, 128, 16),
    ([1000, 3, 127, 128, 129], [1, 1, 1, 1, 1], 8, 32, 128, 64),
    ([700, 0, 12], [5, 9, 2], 2, 8, 128, 32),                  # a few drafted tokens each
    ([0, 65], [150, 33], 2, 6, 64, 16),                        # prompts, rows past one block of 16
    ([40, 7], [1, 3], 1, 16, 256, 16),
    ([333], [1], 1, 40, 32, 128),                              # more query heads than a block has rows
    ([200, 90], [2, 1], 3, 3, 80, 16),
    ([77], [4], 5, 15, 96, 32),
    ([50], [3], 2, 2, 65, 16),
    ([5000, 20, 2600], [1, 1, 4], 1, 4, 128, 16),              # one sequence split over many workgroups
    ([1500, 3, 127, 128, 700], [1, 1, 1, 1, 2], 8, 32, 128, 64),
    ([2000, 40, 1029], [3, 1, 1], 2, 8, 64, 16),
    ([1020, 511], [4, 1], 2, 12, 128, 16),                     # as long as contexts get that are not split
])
def test_attention(gpu_ctx, dtype, past, new, kv_heads, heads, d, page):
    attention_case(gpu_ctx, dtype, past, new, kv_heads, heads, d, page, pad=3, seed=sum(past) + d)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("past,new,kv_heads,heads,d,page", [
    ([0], [64], 1, 1, 64, 16),                                 # one chunk
    ([0], [79], 1, 1, 128, 16),                                # a row fewer than the kernel for many takes,
    ([0], [80], 1, 1, 128, 16),                                # and as many: part of a block
    ([0, 64], [96, 64], 1, 1, 64, 16),
    ([0], [65], 1, 1, 128, 16),                                # a row, and a token, more
    ([63, 64, 0, 0], [128, 63, 1, 200], 2, 2, 128, 32),        # chunks that begin and end inside
    ([1000, 0], [40, 300], 2, 12, 128, 16),                    # a group of 6 heads: tokens across blocks
    ([7, 500], [130, 90], 2, 4, 256, 64),
    ([0, 33], [100, 77], 3, 6, 80, 16),
    ([9], [200], 1, 5, 96, 128),
    ([17, 0, 0], [150, 0, 1], 1, 4, 32, 16),
    ([2000], [20], 1, 16, 128, 16),
    ([5], [70], 1, 2, 65, 16),
])
def test_attention_of_prompts(gpu_ctx, dtype, past, new, kv_heads, heads, d, page):
    for slots in (0, 2048):
        attention_case(gpu_ctx, dtype, past, new, kv_heads, heads, d, page, pad=2, seed=sum(past) + d + 1, slots=slots)


def test_attention_of_many_prompts(gpu_ctx):
    """Enough rows for blocks, whatever the contexts may be."""
    attention_case(gpu_ctx, "bf16", [0] * 9, [130, 128, 200, 64, 300, 127, 129, 1, 150], 2, 16, 64, page=64, seed=41)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("past,new,kv_heads,heads,d,page", [
    ([1500], [130], 1, 2, 64, 16),                             # blocks whose context several workgroups share
    ([3000], [20], 2, 8, 128, 32),
    ([900, 0, 1300], [33, 128, 40], 1, 4, 256, 64),            # and others beside them that one does
    ([2100], [64], 1, 1, 80, 16),
    ([700, 1200], [70, 3], 1, 2, 32, 16),
    ([511], [65], 1, 1, 128, 16),                              # from four rounds to a fifth
    ([9000], [33], 1, 2, 128, 1024),
])
def test_attention_of_few_blocks(gpu_ctx, dtype, past, new, kv_heads, heads, d, page):
    attention_case(gpu_ctx, dtype, past, new, kv_heads, heads, d, page, pad=2, seed=sum(past) + d + 2)


def test_few_blocks_with_bad_pages_and_queries(gpu_ctx):
    """Parts of a context that hold nothing to attend to; a row that is not finite."""
    hk, heads, d, past, n = 1, 2, 64, 2000, 64
    k, v, _ = inputs(31, past + n, hk, d, "f32")
    c = sv.Cache(gpu_ctx, [past + n], hk, d)
    try:
        b = c.batch([0], [past + n])
        c.append(b, k.to(sv.DEV), v.to(sv.DEV), "f32")
        kv = c.read(b)
        q = sv.normal(sv.gen(32), n, heads * d).to(torch.bfloat16)
        q[7, 3] = math.nan
        clean = q.clone()
        clean[7] = 0.0
        for first, last in ((0, 700 // 16), (1024 // 16, 2064 // 16), (0, 2064 // 16)):
            table = c.table.clone()
            table[0, first:last] = -1
            gone = torch.zeros(past + n, dtype=torch.bool)
            gone[first * 16:last * 16] = True
            out = torch.full((n, heads * d), 5.0, dtype=torch.bfloat16, device=sv.DEV)
            c.attend(c.batch([past], [n], table=table), q.to(sv.DEV), out, "bf16", heads, d ** -0.5)
            got = out.cpu()
            want, tol = reference(kv, clean, [past], [n], hk, heads, d, d ** -0.5, "bf16", block=True, gone=gone)
            ok = (got.double() - want).abs() <= tol
            ok[7, :d] = torch.isnan(got[7, :d]) if not gone.all() else True
            ok[7, d:] = ~torch.isnan(got[7, d:])
            assert bool(ok.all())
            assert not gone.all() or not bool(torch.nan_to_num(got).any())
    finally:
        c.close()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_attention_of_prompts_scales(gpu_ctx, scale, dtype):
    attention_case(gpu_ctx, dtype, [90], [130], 2, 4, 64, scale=scale, seed=24, qs=3, os=5, slots=1024)


@pytest.mark.parametrize("dtype,slots", [("f16", 0), ("bf16", 0), ("bf16", 2048)])
def test_prompts_with_bad_pages_and_queries(gpu_ctx, dtype, slots):
    """In the kernel for many rows: pages that the table does not name are not attended to, rows before
    them see nothing, and a row that is not finite is NaN by itself."""
    hk, heads, d, n = 1, 2, 64, 130
    k, v, _ = inputs(21, n, hk, d, "f32")
    c = sv.Cache(gpu_ctx, [n], hk, d, width=max(-(-n // 16), slots // 16))
    try:
        b = c.batch([0], [n])
        c.append(b, k.to(sv.DEV), v.to(sv.DEV), "f32")
        kv = c.read(b)
        table = c.table.clone()
        table[0, 0], table[0, 1], table[0, 5] = -1, c.pages, -7          # slots 0 .. 31 and 80 .. 95
        q = sv.normal(sv.gen(22), n, heads * d).to(sv.DTYPES[dtype])
        q[50, 3], q[60, d + 1] = math.nan, math.inf
        out = torch.full((n, heads * d), 5.0, dtype=sv.DTYPES[dtype], device=sv.DEV)
        c.attend(c.batch([0], [n], table=table), q.to(sv.DEV), out, dtype, heads, d ** -0.5)
        got = out.cpu()
        assert not bool(got[:32].any())
        clean = q.clone()
        clean[50], clean[60] = 0.0, 0.0
        gone = torch.zeros(n, dtype=torch.bool)
        gone[:32] = gone[80:96] = True
        want, tol = reference(kv, clean, [0], [n], hk, heads, d, d ** -0.5, dtype, block=True, gone=gone)
        ok = (got.double() - want).abs() <= tol
        ok[50, :d] = torch.isnan(got[50, :d])
        ok[60, d:] = torch.isnan(got[60, d:])
        ok[50, d:] = ~torch.isnan(got[50, d:])
        ok[60, :d] = ~torch.isnan(got[60, :d])
        assert bool(ok[32:].all())
    finally:
        c.close()


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0, 40.0])
def test_attention_scales(gpu_ctx, scale):
    attention_case(gpu_ctx, "f32", [90, 5], [2, 7], 2, 4, 64, scale=scale, seed=4)


def test_attention_strides(gpu_ctx):
    attention_case(gpu_ctx, "bf16", [90, 5], [2, 7], 2, 4, 64, seed=5, qs=3, os=5)


def test_many_sequences(gpu_ctx):
    """More sequences than a search step holds, many of them empty."""
    g = sv.gen(12)
    past = torch.randint(0, 90, (300,), generator=g).tolist()
    new = (torch.rand(300, generator=g) < 0.7).long().tolist()
    attention_case(gpu_ctx, "f16", past, new, 2, 4, 64, seed=6)


def test_long_context_in_64_bits(gpu_ctx):
    """A cache past 4 GB: its last pages, addressed in 64 bits, next to its first."""
    hk, d, heads, page = 8, 128, 8, 1024
    n = 2048
    pages = (5 << 30) // (hk * page // 16 * 2304) + 1
    h = gpu_ctx.paged_kv_create(pages, page, hk, d)
    try:
        assert pages * hk * (page // 16) * 2304 > 1 << 32
        c = sv.Cache.__new__(sv.Cache)
        c.ctx, c.kv_heads, c.head_dim, c.h, c.keep = gpu_ctx, hk, d, h, []
        c.table = torch.tensor([[pages - 1, pages - 2], [0, 1]], dtype=torch.int32, device=sv.DEV)
        k, v, _ = inputs(13, 2 * n, hk, d, "bf16")
        fill = c.batch([0, 0], [n, n])
        c.append(fill, k.to(sv.DEV), v.to(sv.DEV), "bf16")
        kv = c.read(fill)
        check_cached(kv[0].reshape(2 * n, hk, d), k.reshape(2 * n, hk, d).float(), False)
        check_cached(kv[1].reshape(2 * n, hk, d), v.reshape(2 * n, hk, d).float(), False)
        q = sv.normal(sv.gen(14), 2, heads * d)
        out = torch.zeros(2, heads * d, device=sv.DEV)
        c.attend(c.batch([n - 1, n - 1], [1, 1]), q.to(sv.DEV), out, "f32", heads, d ** -0.5)
        want, tol = reference(kv, q, [n - 1, n - 1], [1, 1], hk, heads, d, d ** -0.5, "f32")
        assert bool(((out.cpu().double() - want).abs() <= tol).all())
    finally:
        torch.cuda.synchronize()
        gpu_ctx.paged_kv_destroy(h)


def test_queries_that_are_not_finite(gpu_ctx):
    """Such a row is NaN, and no other row is touched by it; stale slots behind a sequence do not
    count, whatever they hold."""
    hk, heads, d = 1, 4, 64
    k, v, _ = inputs(15, 200, hk, d, "f32")
    c = sv.Cache(gpu_ctx, [200], hk, d)
    try:
        big = c.batch([0], [200])
        stale = torch.full((200, d), 6.0e4, device=sv.DEV) * torch.sign(torch.randn(200, d, device=sv.DEV))
        c.append(big, stale, stale, "f32")
        fill = c.batch([0], [100])
        c.append(fill, k.to(sv.DEV), v.to(sv.DEV), "f32")
        kv = c.read(fill)
        q = sv.normal(sv.gen(16), 3, heads * d)
        q[1, 5], q[1, 2 * d + 1] = math.nan, math.inf
        out = torch.zeros(3, heads * d, device=sv.DEV)
        c.attend(c.batch([97], [3]), q.to(sv.DEV), out, "f32", heads, d ** -0.5)
        got = out.cpu()
        clean = q.clone()
        clean[1] = 0.0
        want, tol = reference(kv, clean, [97], [3], hk, heads, d, d ** -0.5, "f32")
        ok = (got.double() - want).abs() <= tol
        assert bool(ok[0].all()) and bool(ok[2].all())
        assert bool(torch.isnan(got[1, :d]).all()) and bool(torch.isnan(got[1, 2 * d:3 * d]).all())
        assert not bool(torch.isnan(got[1, d:2 * d]).any()) and not bool(torch.isnan(got[1, 3 * d:]).any())
    finally:
        c.close()


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e6, 1e30])
def test_queries_of_any_size(gpu_ctx, size):
    """The row's power of two keeps the halves in range; the scale brings the scores back."""
    hk, heads, d = 1, 2, 128
    c = sv.Cache(gpu_ctx, [150], hk, d)
    try:
        k, v, _ = inputs(17, 150, hk, d, "f32")
        fill = c.batch([0], [150])
        c.append(fill, k.to(sv.DEV), (v * 1e-3).to(sv.DEV), "f32")
        kv = c.read(fill)
        q = sv.normal(sv.gen(18), 1, heads * d) * size
        out = torch.zeros(1, heads * d, device=sv.DEV)
        scale = float(torch.tensor(0.1 / size, dtype=torch.float32))
        c.attend(c.batch([149], [1]), q.to(sv.DEV), out, "f32", heads, scale)
        want, tol = reference(kv, q, [149], [1], hk, heads, d, scale, "f32")
        assert bool(((out.cpu().double() - want).abs() <= tol).all())
    finally:
        c.close()


@pytest.mark.parametrize("new", [1, 90])
def test_large_queries_of_small_scale(gpu_ctx, new):
    """The row's power of two and the scale meet before either leaves fp32's range."""
    hk, heads, d, n = 1, 2, 128, 200
    c = sv.Cache(gpu_ctx, [n], hk, d, width=64)
    try:
        k, v, _ = inputs(27, n, hk, d, "f32")
        fill = c.batch([0], [n])
        c.append(fill, k.to(sv.DEV), v.to(sv.DEV), "f32")
        kv = c.read(fill)
        q = (sv.normal(sv.gen(28), new, heads * d).clamp(-3, 3) * 1e37).to(torch.bfloat16)
        out = torch.zeros(new, heads * d, dtype=torch.bfloat16, device=sv.DEV)
        scale = float(torch.tensor(2e-38, dtype=torch.float32))
        c.attend(c.batch([n - new], [new]), q.to(sv.DEV), out, "bf16", heads, scale)
        want, tol = reference(kv, q, [n - new], [new], hk, heads, d, scale, "bf16", block=new > 40)
        assert bool(((out.cpu().double() - want).abs() <= tol).all())
    finally:
        c.close()


@pytest.mark.parametrize("dtype,heads", [("f32", 2), ("f16", 16), ("bf16", 32)])
def test_starts_that_do_not_ascend(gpu_ctx, dtype, heads):
    """A sequence whose rows do not lie in the batch, or go backwards, is left out; the others' rows are
    what they are without it."""
    hk, d = 2, 64
    c = sv.Cache(gpu_ctx, [64, 64, 64, 64, 64], hk, d, width=64)
    try:
        k, v, q = inputs(29, 40, hk, d, dtype, heads)
        fill = c.batch([0] * 5, [8] * 5)
        c.append(fill, k.to(sv.DEV), v.to(sv.DEV), dtype)
        before = c.read(fill)
        b = c.batch([8] * 5, [8] * 5)
        starts = torch.tensor([0, 8, -3, 16, 41, 30], dtype=torch.int32, device=sv.DEV)   # of five only the first's are rows
        b.starts = sv.ptr(starts)
        out = torch.full_like(q.to(sv.DEV), 3.0)
        c.append(b, k.to(sv.DEV), v.to(sv.DEV), dtype)
        c.attend(b, q.to(sv.DEV), out, dtype, heads, 0.125)
        assert torch.equal(c.read(fill), before)
        got = out.cpu()
        assert bool((got[8:] == 3.0).all())
        one = c.batch([8], [8], table=c.table[:1].contiguous())
        alone = torch.full_like(out, 3.0)
        c.attend(one, q.to(sv.DEV), alone, dtype, heads, 0.125)
        both = torch.cat([before[:, :8], c.read(one)[:, :8]], dim=1)
        want, tol = reference(both, q[:8], [8], [8], hk, heads, d, 0.125, dtype, block=True)
        assert bool(((got[:8].double() - want).abs() <= tol).all())
        assert bool(((alone.cpu()[:8].double() - want).abs() <= tol).all())
    finally:
        c.close()


def test_refusals(gpu_ctx):
    for kw, status in ((dict(pages=0), -1), (dict(kv_heads=0), -1), (dict(head_dim=0), -1), (dict(head_dim=257), -5),
                       (dict(page_tokens=24), -5), (dict(page_tokens=8), -5), (dict(page_tokens=2048), -5),
                       (dict(rope_dims=3, rope_theta=1e4), -5), (dict(rope_dims=66, rope_theta=1e4), -5),
                       (dict(rope_dims=64), -5), (dict(rope_dims=64, rope_theta=math.inf), -5),
                       (dict(pages=0x7fffffff, kv_heads=65535, page_tokens=1024, head_dim=256), -4), (dict(pages=1 << 30), -4)):
        args = dict(pages=4, page_tokens=16, kv_heads=1, head_dim=64) | kw
        with pytest.raises(abi.AbiError) as e:
            gpu_ctx.paged_kv_create(**args)
        assert e.value.status == status, kw
    small = abi.Context(gpu_ctx.lib, device=0, budget=1 << 20)
    with pytest.raises(abi.AbiError) as e:
        small.paged_kv_create(1000, 16, 8, 128)
    assert e.value.status == -4
    c = sv.Cache(small, [64], 2, 64)
    before = small.telemetry().kv_cache_resident_bytes
    x = torch.zeros(4, 8 * 64, device=sv.DEV)
    ok = c.batch([0], [4])

    def refuse(call, *args, **kw):
        with pytest.raises(abi.AbiError) as e:
            call(*args, **kw)
        assert e.value.status == -1

    def app(batch=ok, **kw):
        base = dict(k_ptr=sv.ptr(x), v_ptr=sv.ptr(x))
        base.update(kw)
        return small.paged_append_request(batch, "f32", **base)

    for r in (app(k_ptr=None), app(v_ptr=None), app(key_stride=127), app(value_stride=5), app(q_ptr=sv.ptr(x), query_heads=2),
              app(q_ptr=sv.ptr(x), q_out_ptr=sv.ptr(x)),
              app(q_ptr=sv.ptr(x), q_out_ptr=sv.ptr(x), query_heads=2, query_stride=200)):
        refuse(small.paged_kv_append_device, c.h, r)
    for field in ("sequences", "tokens", "table_stride"):
        b = c.batch([0], [4])
        setattr(b, field, 0)
        refuse(small.paged_kv_append_device, c.h, app(batch=b))
        refuse(small.paged_kv_read_device, c.h, b, sv.ptr(x), None)
        assert small.paged_attention_workspace_bytes(c.h, small.paged_attention_request(b, "f32", 2, sv.ptr(x), sv.ptr(x), 1.0)) == 0
    refuse(small.paged_kv_read_device, c.h, ok, None, None)
    refuse(small.paged_kv_read_device, c.h, ok, sv.ptr(x), None, stride=3)

    def att(heads=2, **kw):
        r = small.paged_attention_request(ok, "f32", heads, sv.ptr(x), sv.ptr(x) + 4096, 0.1, workspace_ptr=sv.ptr(x))
        for k, v in kw.items():
            setattr(r, k, v)
        return r

    for r in (att(3), att(0), att(query=None), att(output=None), att(output=sv.ptr(x)), att(workspace=None), att(workspace=sv.ptr(x) + 4),
              att(dtype=3), att(query_stride=100), att(output_stride=100)):
        refuse(small.paged_kv_attention_device, c.h, r)
    # another context's handle, and one that is gone
    refuse(gpu_ctx.paged_kv_append_device, c.h, app())
    refuse(gpu_ctx.paged_kv_destroy, c.h)
    gone = abi.Handle(opaque=c.h.opaque)
    small.paged_kv_destroy(c.h)
    assert small.telemetry().kv_cache_resident_bytes < before
    refuse(small.paged_kv_append_device, gone, app())
    refuse(small.paged_kv_destroy, gone)
    small.close()
