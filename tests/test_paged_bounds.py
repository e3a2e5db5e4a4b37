"""The bound that attention's rows are held to, on the host: what it lets through and what it does not."""
import pytest
import torch

import serving as sv

CASES = [
    # past, new, kv_heads, heads, head_dim, sharpness
    ([0], [40], 1, 2, 64, 1.0),
    ([200, 0], [3, 20], 2, 6, 80, 1.0),
    ([1500], [130], 1, 2, 64, 1.0),
    ([2000], [20], 1, 16, 128, 1.0),
    ([3000], [20], 2, 4, 128, 3.0),
    ([9000], [33], 1, 2, 128, 1.0),
]


def cached(past, new, kv_heads, heads, d, dtype, seed):
    """Keys and values as the cache holds them, and queries, for whole sequences."""
    from test_gpu_paged import inputs
    total = sum(p + n for p, n in zip(past, new))
    k, v, _ = inputs(seed, total, kv_heads, d, "f32")
    kv = torch.stack([sv.levels(x.reshape(total, kv_heads, d))[0].reshape(total, -1) for x in (k, v)])
    q = (1.2 * sv.normal(sv.gen(seed + 1), sum(new), heads * d)).to(sv.DTYPES[dtype])
    return kv, q


def rounded(x, to):
    return x if to is None else x.to(to).double()


def attend(kv, q, past, new, kv_heads, heads, d, scale, of=None, weights=None, cache=None, gone=()):
    """64-bit attention with queries, weights, and keys and values rounded to those types; `gone`: slots
    of the first sequence that it leaves out.  Also what share of each row's weight those had."""
    out, share, at, row = [], [], 0, 0
    for p0, n in zip(past, new):
        total = p0 + n
        k, v = (rounded(kv[i, at:at + total].double(), cache).reshape(total, kv_heads, d) for i in range(2))
        qs = rounded(q[row:row + n].double(), of).reshape(n, heads, d)
        see = torch.arange(total)[None] <= p0 + torch.arange(n)[:, None]
        left = torch.ones(total)
        left[list(gone) if row == 0 else []] = 0.0
        o, lost = torch.zeros(n, heads, d, dtype=torch.float64), torch.zeros(n, heads, dtype=torch.float64)
        for h in range(heads):
            s = (qs[:, h] @ k[:, h // (heads // kv_heads)].t() * scale).masked_fill(~see, -float("inf"))
            w = rounded(torch.exp(s - s.amax(1, keepdim=True)), weights)
            kept = w * left[None]
            lost[:, h] = 1 - kept.sum(1) / w.sum(1)
            o[:, h] = torch.nan_to_num(kept @ v[:, h // (heads // kv_heads)] / kept.sum(1, keepdim=True))
        out.append(o)
        share.append(lost)
        at, row = at + total, row + n
    return torch.cat(out), torch.cat(share)


def beyond(got, want, limit):
    return ((got - want) ** 2).sum(2).sqrt() > limit


@pytest.mark.parametrize("past,new,kv_heads,heads,d,sharp", CASES)
@pytest.mark.parametrize("dtype,kernel", [("f32", "decode"), ("f16", "decode"), ("bf16", "decode"), ("bf16", "block")])
def test_what_a_row_may_be_off(dtype, kernel, past, new, kv_heads, heads, d, sharp):
    kv, q = cached(past, new, kv_heads, heads, d, dtype, sum(past) + d)
    shape, scale = (past, new, kv_heads, heads, d), sharp * d ** -0.5
    want, limit = sv.attention_rows(kv, q, *shape, scale, dtype, kernel)
    run = lambda **kw: attend(kv, q, *shape, scale, **kw)  # noqa: E731
    off = lambda **kw: beyond(run(**kw)[0], want, limit)  # noqa: E731
    assert torch.allclose(run()[0], want, rtol=1e-9, atol=1e-12)
    # the roundings that a kernel makes pass
    like = dict(weights=None if dtype == "f32" else torch.float16, cache=torch.float16 if kernel == "block" else None)
    assert not bool(beyond(run(**like)[0].to(sv.DTYPES[dtype]).double(), want, limit).any())
    # zeros do not, nor does a chunk of tokens left out where it has a hundredth of the weight
    assert bool(beyond(torch.zeros_like(want), want, limit).all())
    first = max(0, past[0] - 64)
    less, share = run(gone=range(first, first + 64 if past[0] else 8))
    lost = share > 0.01
    assert bool(lost.any()) and float(beyond(less, want, limit)[lost].double().mean()) > 0.98
    if dtype == "f32":
        # nor queries or weights with one f16 half, or in bf16, but for rows that one token has
        for to in (torch.float16, torch.bfloat16):
            assert float(off(of=to).double().mean()) > 0.8, to
            assert sharp > 1 or float(off(weights=to).double().mean()) > 0.8, to


def test_rows_are_told_apart():
    """The kernels' sides as the cases of the GPU tests name them."""
    path = sv.attention_path
    assert path("bf16", [0], [79], 1, 1, 128, 2048) == ("decode", True)
    assert path("bf16", [0], [80], 1, 1, 128, 2048)[0] == "block"
    assert path("bf16", [0], [80], 1, 1, 128, 512)[0] == "prompt"
    assert path("f16", [0], [80], 1, 1, 128, 2048) == ("prompt", True)
    assert path("bf16", [511], [81], 1, 1, 128, 592) == ("block", True) and path("bf16", [430], [81], 1, 1, 128, 592) == ("block", False)
