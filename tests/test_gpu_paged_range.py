"""Attention over the paged cache where scores are far apart: every finite query and scale has the
softmax of its definition, whatever the scores' size."""
import math

import pytest
import torch

import serving as sv

pytestmark = pytest.mark.gpu


def steep_keys(n, kv_heads, d, octaves, seed):
    """Keys that are multiples of one direction u (+-1) per head: factors from 2^-6 up, each its own,
    in no order.  Returns (keys [n][kv_heads * d], u)."""
    g = sv.gen(seed)
    u = torch.where(torch.rand(kv_heads, d, generator=g) < 0.5, -1.0, 1.0)
    u[:, 0], u[:, -1] = 1.0, -1.0
    c = 2.0 ** (-6 + octaves * torch.randperm(n, generator=g).float() / n)
    return (c[:, None, None] * u).reshape(n, -1), u


def one_of(kv, q, past, new, kv_heads, heads, d, scale):
    """64-bit attention of one sequence; every row's best score stands apart from its second by more
    than any rounding (asserted), so that its output is one token's value."""
    group = heads // kv_heads
    k, v = (x.double().reshape(past + new, kv_heads, d) for x in kv)
    qs = q.double().reshape(new, heads, d)
    out = torch.zeros(new, heads, d, dtype=torch.float64)
    see = torch.arange(past + new)[None] <= past + torch.arange(new)[:, None]
    for h in range(heads):
        s = (qs[:, h, None] * k[None, :, h // group]).sum(-1) * scale
        s = s.masked_fill(~see, -math.inf)
        size = (qs[:, h, None].abs() * k[None, :, h // group].abs()).sum(-1) * abs(scale)
        best = s.argmax(1, keepdim=True)
        # keys rounded to f16 move a score by 2^-11 of its magnitude at most, sums by far less; e^-40
        # of another token is nothing
        gap = s.gather(1, best) - s - 2.0 ** -10 * (size + size.gather(1, best))
        assert bool((gap > 40).scatter(1, best, True).all())
        out[:, h] = v[s.argmax(1), h // group]
    return out.reshape(new, heads * d)


# powers of two of query times scale, and of the scale alone
SIZES = [(16, 0), (24, 4), (28, 0), (30, 12), (33, 0), (45, 0), (70, 40), (100, -20), (115, 0), (118, 0), (121, -3),
         (126, 0), (126, -3), (130, 10), (150, 24), (200, 90)]


def check_sizes(ctx, dtype, past, new, kv_heads, heads, d, slots):
    n, dt = past + new, sv.DTYPES[dtype]
    c = sv.Cache(ctx, [n], kv_heads, d, 16, width=max(-(-n // 16), slots // 16), seed=n)
    try:
        # factors apart by 2^(octaves / n), 1.5 % at least
        k, u = steep_keys(n, kv_heads, d, 16 if n > 300 else 12, n + d)
        v = sv.normal(sv.gen(n), n, kv_heads * d)
        fill = c.batch([0], [n])
        c.append(fill, k.to(sv.DEV), v.to(sv.DEV), "f32")
        kv = c.read(fill)
        b, wrong = c.batch([past], [new]), []
        for both, of_scale in SIZES:
            if dtype == "f16":       # a query of f16 has no such size: all of it in the scale
                of_scale = min(both - 8, 126)
            if both - of_scale > 126 or (dtype == "f16" and both - of_scale > 14):
                continue
            size = 2.0 ** (both - of_scale) * (1 + torch.arange(heads) % 3 / 4)
            lean = u.repeat_interleave(heads // kv_heads, 0) * size[:, None]
            q = lean.reshape(1, -1).repeat(new, 1).to(dt)
            for sign in (1.0, -0.7):
                scale = float(torch.tensor(sign * 2.0 ** of_scale, dtype=torch.float32))
                want = one_of(kv, q, past, new, kv_heads, heads, d, scale)
                # the output's own rounding and that of a value to f16, a few of fp32 of minimum and 15 steps
                tol = (sv.HALF[dtype] + 2.0 ** -11 + 2.0 ** -20) * want.abs() + 2.0 ** -20 * 3 * v.abs().max()
                out = torch.full((new, heads * d), 7.0, dtype=dt, device=sv.DEV)
                c.attend(b, q.to(sv.DEV), out, dtype, heads, scale)
                ok = (out.cpu().double() - want).abs() <= tol
                if not bool(ok.all()):
                    wrong.append((both, of_scale, sign, round(float((~ok).double().mean()), 3)))
        assert not wrong, f"(size, of the scale, sign, share of wrong values): {wrong}"
    finally:
        c.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("past,new,kv_heads,heads,d,slots", [
    (20, 3, 1, 2, 64, 0),            # whole contexts
    (100, 2, 2, 12, 128, 2048),      # a context that several workgroups share
    (600, 1, 1, 1, 256, 1024),
])
def test_scores_of_any_size(gpu_ctx, dtype, past, new, kv_heads, heads, d, slots):
    check_sizes(gpu_ctx, dtype, past, new, kv_heads, heads, d, slots)


PROMPTS = [
    (0, 90, 1, 4, 64, 2048),
    (30, 100, 2, 4, 128, 2048),
    (640, 85, 1, 1, 64, 2048),       # a context that several workgroups share
    (60, 90, 1, 2, 256, 1024),
]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("past,new,kv_heads,heads,d,slots", PROMPTS)
def test_scores_of_any_size_in_prompts(gpu_ctx, dtype, past, new, kv_heads, heads, d, slots):
    check_sizes(gpu_ctx, dtype, past, new, kv_heads, heads, d, slots)


@pytest.mark.parametrize("dtype,new", [("f32", 1), ("f16", 3), ("bf16", 2), ("f32", 90), ("f16", 90), ("bf16", 90)])
def test_scales_next_to_nothing_and_not_finite(gpu_ctx, dtype, new):
    """Rows with queries of all sizes, in one block: a scale that leaves nothing of the scores is a mean,
    one that is not finite makes rows NaN, but for a row that attends to nothing."""
    n, heads, d = 300, 2, 64
    c = sv.Cache(gpu_ctx, [n], 1, d, width=128)
    try:
        k, v = (sv.normal(sv.gen(i), n, d) for i in (1, 2))
        fill = c.batch([0], [n])
        c.append(fill, k.to(sv.DEV), v.to(sv.DEV), "f32")
        kv = c.read(fill)
        dt = sv.DTYPES[dtype]
        sizes = torch.tensor([1.0, 0.0, 2.0 ** -20, 2.0 ** 12] if dtype == "f16" else [1.0, 0.0, 2.0 ** -125, 2.0 ** 100, 2.0 ** -60])
        q = (sv.normal(sv.gen(3), new, heads, d) * sizes[torch.arange(new * heads) % len(sizes)].reshape(new, heads, 1)).reshape(new, -1).to(dt)
        path = sv.attention_path(dtype, [n - new], [new], 1, heads, d, 2048)[0]
        b = c.batch([n - new], [new])
        for scale in (0.0, 1e-45, -1e-40, 1e-36, 2.0 ** -103, 0.125, float("inf"), float("-inf"), float("nan")):
            out = torch.full((new, heads * d), 7.0, dtype=dt, device=sv.DEV)
            c.attend(b, q.to(sv.DEV), out, dtype, heads, scale)
            got = out.cpu().double().reshape(new, heads, d)
            if not math.isfinite(scale):
                assert bool(torch.isnan(got).all()), scale
                continue
            want, limit = sv.attention_rows(kv, q, [n - new], [new], 1, heads, d, scale, dtype, path)
            # rows whose scores are past what the bound's first order holds for are another test's
            held = (scale * q.double().reshape(new, heads, d).abs().amax(2)).abs() < 3
            off = ((got - want) ** 2).sum(2).sqrt() / limit
            assert bool((off[held] <= 1).all()) and bool(torch.isfinite(got).all()), (scale, float(off[held].max()))
        none = c.batch([n - new], [new], table=torch.full_like(c.table, -1))
        for scale in (0.125, float("inf"), float("nan")):
            out = torch.full((new, heads * d), 7.0, dtype=dt, device=sv.DEV)
            c.attend(none, q.to(sv.DEV), out, dtype, heads, scale)
            assert not bool(out.any())
    finally:
        c.close()


@pytest.mark.parametrize("past,new,kv_heads,heads,d,slots", PROMPTS)
def test_scores_of_any_size_in_blocks_of_many_rows(gpu_ctx, past, new, kv_heads, heads, d, slots):
    check_sizes(gpu_ctx, "bf16", past, new, kv_heads, heads, d, slots)
