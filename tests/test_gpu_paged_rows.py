"""Attention over the paged cache held row by row to what its roundings can do (the bound's own test:
test_paged_bounds.py), each case in the kernel that it names."""
import pytest
import torch

import serving as sv
from test_gpu_paged import inputs

pytestmark = pytest.mark.gpu


def check(ctx, kernel, dtype, past, new, kv_heads, heads, d, page=16, slots=0, pad=0, sharp=1.0, seed=0, split=None):
    scale = sharp * d ** -0.5
    total = [p + n for p, n in zip(past, new)]
    width = max(-(-max(total) // page), -(-slots // page))
    got = sv.attention_path(dtype, past, new, kv_heads, heads, d, width * page, pad)
    assert got[0] == kernel and (split is None or got[1] == split), got
    c = sv.Cache(ctx, total, kv_heads, d, page, seed=seed, width=width)
    try:
        k, v, _ = inputs(seed + 1, sum(total), kv_heads, d, "f32")
        fill = c.batch([0] * len(total), total)
        c.append(fill, k.to(sv.DEV), v.to(sv.DEV), "f32")
        kv = c.read(fill)
        rows = sum(new)
        q = (1.2 * sv.normal(sv.gen(seed + 2), rows + pad, heads * d)).to(sv.DTYPES[dtype])
        want, limit = sv.attention_rows(kv, q, past, new, kv_heads, heads, d, scale, dtype, kernel)
        b, first = c.batch(past, new, pad=pad), None
        for _ in range(3):          # the same every time, bit for bit
            out = torch.full((rows + pad, heads * d), 7.0, dtype=sv.DTYPES[dtype], device=sv.DEV)
            c.attend(b, q.to(sv.DEV), out, dtype, heads, scale)
            out = out.cpu()
            assert bool((out[rows:] == 7.0).all())
            first = out if first is None else first
            assert torch.equal(out, first)
        off = ((first[:rows].reshape(want.shape).double() - want) ** 2).sum(2).sqrt() / limit
        assert bool((off <= 1).all()), f"off by {float(off.max()):.2f} of the bound"
    finally:
        c.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("past,new,kv_heads,heads,d,page,slots,sharp", [
    ([0], [1], 1, 1, 64, 16, 0, 1.0),
    ([15, 16, 17, 0, 31, 300], [1, 1, 1, 0, 1, 1], 2, 12, 128, 16, 0, 1.0),
    ([15, 16, 17, 0, 31, 300], [1, 1, 1, 0, 1, 1], 2, 12, 128, 16, 4096, 1.0),
    ([1000, 3, 127, 128, 129], [1, 1, 1, 1, 1], 8, 32, 128, 64, 0, 1.0),
    ([700, 0, 12], [5, 9, 2], 2, 8, 80, 32, 0, 2.0),
    ([40, 700], [1, 3], 1, 16, 256, 16, 0, 1.0),
    ([333], [1], 1, 40, 32, 128, 0, 1.0),
    ([2000], [20], 4, 8, 128, 16, 0, 1.0),
    ([5000, 20, 2600], [1, 1, 4], 1, 4, 128, 16, 0, 1.0),
    ([9000], [33], 1, 2, 128, 1024, 0, 1.0),
    ([511], [65], 1, 1, 128, 16, 0, 1.0),
    ([300], [79], 1, 1, 96, 16, 2048, 1.0),          # a row fewer than a prompt has
])
def test_decode(gpu_ctx, dtype, past, new, kv_heads, heads, d, page, slots, sharp):
    check(gpu_ctx, "decode", dtype, past, new, kv_heads, heads, d, page, slots, sharp=sharp, seed=sum(past) + d)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("past,new,kv_heads,heads,d,page,slots,sharp", [
    ([0], [80], 1, 1, 128, 16, 0, 1.0),
    ([63, 64, 0, 0], [128, 63, 1, 200], 2, 2, 128, 32, 0, 1.0),
    ([63, 64, 0, 0], [128, 63, 1, 200], 2, 2, 128, 32, 2048, 1.0),
    ([1500], [130], 1, 2, 64, 16, 0, 1.0),
    ([2000], [40], 1, 16, 128, 16, 0, 2.0),
    ([900, 0, 1300], [90, 128, 40], 1, 4, 256, 64, 0, 1.0),
    ([0, 33], [100, 77], 3, 6, 80, 16, 0, 1.0),
])
def test_prompts(gpu_ctx, dtype, past, new, kv_heads, heads, d, page, slots, sharp):
    check(gpu_ctx, "prompt", dtype, past, new, kv_heads, heads, d, page, slots, sharp=sharp, seed=sum(past) + d + 1, pad=2)


def test_short_prompts_of_bf16(gpu_ctx):
    """Few rows of short contexts stay in blocks of 16."""
    for past, new, kv_heads, heads, d in (([0], [80], 1, 1, 128), ([63, 64, 0], [128, 100, 40], 2, 2, 128), ([7], [200], 1, 4, 256)):
        check(gpu_ctx, "prompt", "bf16", past, new, kv_heads, heads, d, seed=d + new[0])


@pytest.mark.parametrize("past,new,kv_heads,heads,d,page,slots,split", [
    ([0], [80], 1, 1, 128, 16, 2048, False),                 # as many rows as the kernel takes: part of a block
    ([0], [81], 1, 1, 96, 16, 2048, False),
    ([0, 64], [96, 70], 1, 1, 64, 16, 1024, False),
    ([63, 64, 0, 0], [128, 63, 1, 200], 2, 2, 128, 32, 1024, False),
    ([700, 1200], [150, 30], 1, 2, 32, 16, 0, True),         # contexts that several workgroups share,
    ([2100], [90], 1, 1, 80, 16, 0, True),
    ([1500], [130], 1, 2, 64, 16, 0, True),
    ([900, 0, 1300], [90, 128, 40], 1, 4, 256, 64, 0, True),
    ([9000], [90], 1, 2, 128, 1024, 0, True),
    ([3000], [40], 2, 8, 128, 32, 0, True),
    ([511], [81], 1, 1, 128, 16, 0, True),                   # from five rounds on,
    ([430], [82], 1, 1, 128, 16, 592, False),                # not of four
    ([5], [85], 1, 2, 65, 16, 640, False),
    ([0] * 9, [130, 128, 200, 64, 300, 127, 129, 1, 150], 2, 16, 64, 64, 0, False),
    ([2000], [45], 1, 16, 128, 16, 0, True),
    ([600], [1024], 8, 32, 128, 16, 0, False),               # as many blocks as the GPU has units for
])
def test_blocks_of_many_rows(gpu_ctx, past, new, kv_heads, heads, d, page, slots, split):
    for pad, sharp in ((0, 1.0), (2, 1.0)):
        check(gpu_ctx, "block", "bf16", past, new, kv_heads, heads, d, page, slots, pad, sharp, sum(past) + d + 2, split)


@pytest.mark.parametrize("dtype,kernel", [("f32", "decode"), ("f16", "decode"), ("bf16", "decode"), ("f32", "prompt"), ("f16", "prompt"),
                                          ("bf16", "block")])
def test_every_slot_is_read(gpu_ctx, dtype, kernel):
    """Keys of one direction, each larger than all before it by more than rounding: row i is slot i's
    value, whatever page, tile, piece or part the slot lies in."""
    n, d = 600, 64
    step = 60 if kernel == "decode" else n          # rows of a call
    c = sv.Cache(gpu_ctx, [n], 1, d, 16, width=128)
    try:
        g = sv.gen(5)
        u = torch.where(torch.rand(d, generator=g) < 0.5, -1.0, 1.0)
        u[0], u[1] = 1.0, -1.0
        k = 2.0 ** (-8 + 20 * torch.arange(n) / n)[:, None] * u
        v = sv.normal(g, n, d)
        fill = c.batch([0], [n])
        c.append(fill, k.to(sv.DEV), v.to(sv.DEV), "f32")
        kv = c.read(fill)
        # scores 64 * 2^-8 * 2^14 and up, 2.3 % apart
        q = (u * 2.0 ** 7).repeat(step, 1).to(sv.DTYPES[dtype])
        for first in range(0, n, step):
            assert sv.attention_path(dtype, [first], [step], 1, 1, d, 2048)[0] == kernel
            out = torch.zeros(step, d, dtype=sv.DTYPES[dtype], device=sv.DEV)
            c.attend(c.batch([first], [step]), q.to(sv.DEV), out, dtype, 1, 128.0)
            want = kv[1, first:first + step].double()
            tol = (sv.HALF[dtype] + 2.0 ** -11 + 2.0 ** -20) * want.abs() + 2.0 ** -20 * 3 * v.abs().max()
            assert bool(((out.cpu().double() - want).abs() <= tol).all())
    finally:
        c.close()


@pytest.mark.parametrize("dtype,kernel", [("f32", "prompt"), ("f16", "prompt"), ("bf16", "block")])
def test_single_tokens_beside_a_prompt(gpu_ctx, dtype, kernel):
    """Single tokens behind long contexts and a prompt's rows: in one call, and in a call each over the
    same tensors."""
    past, new, kv_heads, heads, d = [3000, 700, 5, 40], [1, 1, 1, 300], 2, 8, 128
    check(gpu_ctx, kernel, dtype, past, new, kv_heads, heads, d, seed=71, pad=1)
    total = [p + n for p, n in zip(past, new)]
    c = sv.Cache(gpu_ctx, total, kv_heads, d)
    try:
        k, v, _ = inputs(72, sum(total), kv_heads, d, "f32")
        fill = c.batch([0] * 4, total)
        c.append(fill, k.to(sv.DEV), v.to(sv.DEV), "f32")
        kv = c.read(fill)
        rows, one = sum(new), 3
        q = (1.2 * sv.normal(sv.gen(73), rows, heads * d)).to(sv.DTYPES[dtype])
        qd, out = q.to(sv.DEV), torch.full((rows, heads * d), 7.0, dtype=sv.DTYPES[dtype], device=sv.DEV)
        b = c.batch(past, new)
        singles = gpu_ctx.paged_batch(one, one, b.starts, b.past, b.page_table, b.table_stride)
        prompt = gpu_ctx.paged_batch(1, rows, b.starts + 4 * one, b.past + 4 * one, b.page_table + 4 * one * b.table_stride, b.table_stride)
        c.attend(singles, qd, out, dtype, heads, d ** -0.5)
        assert bool((out[one:] == 7.0).all()) and not bool((out[:one] == 7.0).all())
        c.attend(prompt, qd, out, dtype, heads, d ** -0.5)
        want, limit = (torch.cat(x) for x in zip(
            sv.attention_rows(kv, q, past, new[:3] + [0], kv_heads, heads, d, d ** -0.5, dtype, "decode"),
            sv.attention_rows(kv[:, sum(total[:3]):], q[3:], past[3:], new[3:], kv_heads, heads, d, d ** -0.5, dtype, kernel)))
        assert bool((((out.cpu().reshape(want.shape).double() - want) ** 2).sum(2).sqrt() <= limit).all())
    finally:
        c.close()
