"""Rotary positions with several axes and the heads' norms (qwn_hip_ext_rotary_device), against the
definition in 64 bits."""
import pytest
import torch

import serving as sv
from qwanto_amd import abi

pytestmark = pytest.mark.gpu
THETA, EPS = 1.0e6, 1e-6


def axis_of(sections, in_turn):
    """The axis of each pair."""
    if not in_turn:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, order = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                order.append(a)
    return order


def reference(x, heads, d, rope, positions, sections, in_turn, norm, theta=THETA, eps=EPS):
    """(64-bit result [rows][heads * d], the size of what each element is computed from)."""
    rows = x.shape[0]
    y = x.double().reshape(rows, heads, d)
    if norm is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * norm.double()
    size = y.abs()
    half = rope // 2
    if half:
        axis = axis_of(sections, in_turn)
        freq = theta ** (-2.0 * torch.arange(half, dtype=torch.float64) / rope)
        ang = (positions[axis].double().t() * freq)[:, None]
        a, b = y[..., :half].clone(), y[..., half:rope].clone()
        y = torch.cat((a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos(), y[..., rope:]), -1)
        pair = a.abs() + b.abs()
        size = torch.cat((pair, pair, size[..., rope:]), -1)
    return y.reshape(rows, -1), size.reshape(rows, -1)


def check(got, want, size, dtype):
    """fp32: 64 bits rounded once, by at most half a step; the angle, of up to 2^18, in 64 bits (2^-33),
    twice over for the frequency's own rounding.  16 bits: fp32, rounded to the type.  A square sum of up
    to 256 channels is off by at most 22 roundings (products, chains of 16, 5 lanes), the root of it
    by half of them and 2; weight, product, angle and two products of the rotation are 5 more: 18 of
    2^-24 of what the element is computed from."""
    tiny = 2.0 ** -25 if dtype == "f16" else 2.0 ** -134 if dtype == "bf16" else 2.0 ** -150
    if dtype == "f32":
        tol = 2.0 ** -24 * (1 + 1e-6) * want.abs() + 2.0 ** -31 * size + tiny
    else:
        tol = sv.HALF[dtype] * want.abs() + (1 + sv.HALF[dtype]) * 18 * 2.0 ** -24 * size + tiny
    assert bool(((got.double() - want).abs() <= tol).all())


def positions_of(g, axes, tokens):
    return torch.randint(-10, 1 << 18, (axes, tokens), generator=g, dtype=torch.int32)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,heads,kv_heads,d,rope,sections,in_turn,norms", [
    (1, 12, 2, 128, 128, [64], False, False),
    (1, 1, 1, 1, 0, [], False, True),
    (3, 2, 1, 2, 2, [1], False, True),
    (5, 32, 8, 128, 128, [16, 24, 24], False, True),
    (5, 32, 8, 128, 128, [24, 20, 20], True, True),
    (7, 3, 1, 80, 80, [10, 15, 15], True, False),
    (2, 6, 3, 65, 40, [4, 0, 16], True, True),
    (4, 4, 2, 256, 256, [32, 32, 32, 32], True, True),
    (4, 2, 2, 256, 2, [1], False, True),
    (3, 5, 5, 96, 50, [5, 20], False, True),
    (61, 0, 4, 64, 64, [0, 32], False, False),
    (61, 16, 0, 64, 32, [8, 4, 4], False, True),
    (4099, 2, 1, 32, 32, [6, 5, 5], True, True),
    (5, 129, 1, 64, 64, [32], False, False),
])
def test_sizes(gpu_ctx, dtype, tokens, heads, kv_heads, d, rope, sections, in_turn, norms):
    g = sv.gen(tokens + d)
    dt = sv.DTYPES[dtype]
    q, k = ((1.2 * sv.normal(g, tokens, h * d) + 0.3).to(dt) for h in (heads, kv_heads))
    w = [1 + 0.2 * sv.normal(g, d) if norms else None for _ in range(2)]
    p = positions_of(g, max(1, len(sections)), tokens)
    qd, kd, pd = q.to(sv.DEV), k.to(sv.DEV), p.to(sv.DEV)
    wd = [x.to(sv.DEV) if x is not None else None for x in w]
    qo, ko = torch.full_like(qd, float("nan")), torch.full_like(kd, float("nan"))

    def req(q_out, k_out):
        return gpu_ctx.rotary_request(tokens, dtype, d, rope, THETA, sv.ptr(pd), sections=sections, in_turn=in_turn, query_heads=heads,
                                      q_ptr=sv.ptr(qd), q_out_ptr=sv.ptr(q_out), key_heads=kv_heads, k_ptr=sv.ptr(kd),
                                      k_out_ptr=sv.ptr(k_out), q_norm_ptr=sv.ptr(wd[0]), k_norm_ptr=sv.ptr(wd[1]), eps=EPS)

    gpu_ctx.rotary_device(req(qo, ko), stream=sv.stream())
    torch.cuda.synchronize()
    for x, o, h, n in ((q, qo, heads, w[0]), (k, ko, kv_heads, w[1])):
        if h:
            check(o.cpu(), *reference(x, h, d, rope, p, sections, in_turn, n), dtype)
    gpu_ctx.rotary_device(req(qd, kd), stream=sv.stream())                       # in place
    torch.cuda.synchronize()
    assert torch.equal(qd, qo) and torch.equal(kd, ko)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("odd", [0, 1, 3])
def test_columns_of_one_buffer(gpu_ctx, dtype, odd):
    """Queries and keys side by side in a projection's rows, at any alignment, one of them normed, in
    place: the same as from tensors of their own, and nothing beside them is touched."""
    tokens, heads, kv_heads, d = 9, 6, 2, 64
    g = sv.gen(odd)
    q, k, v = (sv.normal(g, tokens, h * d).to(sv.DTYPES[dtype]) for h in (heads, kv_heads, kv_heads))
    p, w = positions_of(g, 3, tokens + 4).to(sv.DEV), (1 + 0.1 * sv.normal(g, d)).to(sv.DEV)
    edge = torch.full((tokens, odd), 7.0).to(q.dtype)
    buf = torch.cat([edge, q, k, v, edge], dim=1).to(sv.DEV).contiguous()
    size, width = buf.element_size(), buf.shape[1]
    qo, ko = torch.zeros_like(q).to(sv.DEV), torch.zeros_like(k).to(sv.DEV)
    qd, kd = q.to(sv.DEV), k.to(sv.DEV)
    common = dict(sections=[8, 12, 12], query_heads=heads, key_heads=kv_heads, q_norm_ptr=sv.ptr(w), eps=EPS, position_stride=tokens + 4)
    gpu_ctx.rotary_device(gpu_ctx.rotary_request(tokens, dtype, d, 64, THETA, sv.ptr(p), q_ptr=sv.ptr(qd), q_out_ptr=sv.ptr(qo),
                                                 k_ptr=sv.ptr(kd), k_out_ptr=sv.ptr(ko), **common), stream=sv.stream())
    at = lambda c: sv.ptr(buf) + (odd + c) * size  # noqa: E731
    gpu_ctx.rotary_device(gpu_ctx.rotary_request(tokens, dtype, d, 64, THETA, sv.ptr(p), q_ptr=at(0), q_out_ptr=at(0), k_ptr=at(heads * d),
                                                 k_out_ptr=at(heads * d), query_stride=width, key_stride=width, query_out_stride=width,
                                                 key_out_stride=width, **common), stream=sv.stream())
    torch.cuda.synchronize()
    assert torch.equal(buf.cpu(), torch.cat([edge, qo.cpu(), ko.cpu(), v, edge], dim=1))
    check(qo.cpu(), *reference(q, heads, d, 64, p.cpu()[:, :tokens], [8, 12, 12], False, w.cpu()), dtype)
    check(ko.cpu(), *reference(k, kv_heads, d, 64, p.cpu()[:, :tokens], [8, 12, 12], False, None), dtype)


def test_values_that_are_not_finite_stay_in_their_head(gpu_ctx):
    heads, d = 3, 64
    g = sv.gen(1)
    q = sv.normal(g, 4, heads * d)
    q[1, d + 3] = float("inf")
    q[2, 5] = float("nan")
    q[3, :d] = 0.0
    p, w = positions_of(g, 1, 4), 1 + 0.1 * sv.normal(g, d)
    qd, pd, wd = q.to(sv.DEV), p.to(sv.DEV), w.to(sv.DEV)
    for norm in (None, w):
        out = torch.zeros_like(qd)
        gpu_ctx.rotary_device(gpu_ctx.rotary_request(4, "f32", d, d, THETA, sv.ptr(pd), query_heads=heads, q_ptr=sv.ptr(qd),
                                                     q_out_ptr=sv.ptr(out), q_norm_ptr=sv.ptr(wd) if norm is not None else None, eps=EPS),
                              stream=sv.stream())
        want, size = reference(q, heads, d, d, p, [d // 2], False, norm)
        fine = torch.isfinite(want)
        got = out.cpu()
        assert torch.equal(torch.isfinite(got), fine)
        check(got[fine], want[fine], size[fine], "f32")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,rope", [(128, 128), (256, 64), (80, 80), (1, 0)])
def test_norms_of_any_size(gpu_ctx, dtype, d, rope):
    """Heads whose squares' sum is past fp32's range, or below it, beside ordinary ones and zeros: of each its norm."""
    g = sv.gen(d)
    info = torch.finfo(sv.DTYPES[dtype])
    sizes = [1.0, 0.9 * info.max, info.max ** 0.5, 1e-3 * info.max, info.tiny ** 0.5, 3 * info.tiny, info.tiny / 16, 0.0]
    heads, tokens = len(sizes), 5
    x = 2 * torch.rand(tokens, heads, d, generator=g) - 1
    x = (x * torch.tensor(sizes)[:, None]).to(sv.DTYPES[dtype]).reshape(tokens, heads * d)
    p, w = positions_of(g, 1, tokens), 1 + 0.2 * sv.normal(g, d)
    xd, pd, wd = x.to(sv.DEV), p.to(sv.DEV), w.to(sv.DEV)
    out = torch.zeros_like(xd)
    for eps in (0.0, 1e-30, 1e-6):
        gpu_ctx.rotary_device(gpu_ctx.rotary_request(tokens, dtype, d, rope, THETA, sv.ptr(pd), query_heads=heads, q_ptr=sv.ptr(xd),
                                                     q_out_ptr=sv.ptr(out), q_norm_ptr=sv.ptr(wd), eps=eps), stream=sv.stream())
        eps = float(torch.tensor(eps, dtype=torch.float32))
        want, size = reference(x, heads, d, rope, p, [rope // 2], False, w, eps=eps)
        got = out.cpu()
        zeros = x.reshape(tokens, heads, d).double().square().sum(-1).eq(0).repeat_interleave(d, 1)
        if eps == 0.0:
            assert bool(torch.isnan(got[zeros]).all())                           # 0 / 0
        else:
            assert bool((got[zeros] == 0).all())
        check(got[~zeros], want[~zeros], size[~zeros], dtype)
    # many tokens, the odd ones ordinary: theirs is what it is beside ordinary ones, to the bit; in place
    many = x.repeat(820, 1)
    many[1::2] = (2 * torch.rand(2050, heads * d, generator=g) - 1).to(many.dtype)
    calm = many.clone()
    calm[0::2] = calm[1::2]
    p = positions_of(g, 1, 4100).to(sv.DEV)
    out = [t.to(sv.DEV) for t in (many, calm)]
    for o in out:
        gpu_ctx.rotary_device(gpu_ctx.rotary_request(4100, dtype, d, rope, THETA, sv.ptr(p), query_heads=heads, q_ptr=sv.ptr(o),
                                                     q_out_ptr=sv.ptr(o), q_norm_ptr=sv.ptr(wd), eps=1e-30), stream=sv.stream())
    torch.cuda.synchronize()
    assert torch.equal(out[0][1::2], out[1][1::2])
    want, size = reference(many, heads, d, rope, p.cpu(), [rope // 2], False, w, eps=float(torch.tensor(1e-30)))
    check(out[0].cpu(), want, size, dtype)


def test_axes_without_a_section_have_a_row(gpu_ctx):
    """Positions are found by the axis' number, so an axis without pairs has a row of its own, too, which does not count;
    rows up to the last axis with pairs are an input, which an output may not overlap."""
    tokens, d = 7, 64
    g = sv.gen(3)
    x, p = sv.normal(g, tokens, d), positions_of(g, 4, tokens)
    xd, out = x.to(sv.DEV), torch.zeros(tokens, d, device=sv.DEV)
    for sections in ([4, 0, 28], [0, 0, 0, 32], [0, 32], [16, 0, 0, 16]):
        want, size = reference(x, 1, d, d, p, sections, False, None)
        for other in (0, 2 ** 31 - 1):
            q = p.clone()
            for a, n in enumerate(sections):
                if not n:
                    q[a] = other
            qd = q[:len(sections)].contiguous().to(sv.DEV)
            gpu_ctx.rotary_device(gpu_ctx.rotary_request(tokens, "f32", d, d, THETA, sv.ptr(qd), sections=sections, query_heads=1, q_ptr=sv.ptr(xd),
                                                         q_out_ptr=sv.ptr(out)), stream=sv.stream())
            torch.cuda.synchronize()
            check(out.cpu(), want, size, "f32")
    both = torch.zeros(3 * tokens + tokens * d, dtype=torch.int32, device=sv.DEV)
    req = lambda sections, at: gpu_ctx.rotary_request(tokens, "f32", d, d, THETA, sv.ptr(both), sections=sections, query_heads=1,  # noqa: E731
                                                      q_ptr=sv.ptr(xd), q_out_ptr=sv.ptr(both) + 4 * at)
    gpu_ctx.rotary_device(req([32, 0], tokens), stream=sv.stream())
    gpu_ctx.rotary_device(req([4, 0, 28], 3 * tokens), stream=sv.stream())
    with pytest.raises(abi.AbiError):
        gpu_ctx.rotary_device(req([4, 0, 28], 2 * tokens), stream=sv.stream())
    torch.cuda.synchronize()


def test_refusals(gpu_ctx):
    t, d = 4, 64
    q, k = torch.zeros(t, 2 * d, device=sv.DEV), torch.zeros(t, d, device=sv.DEV)
    qo, ko = torch.zeros_like(q), torch.zeros_like(k)
    p, w = torch.zeros(3, t, dtype=torch.int32, device=sv.DEV), torch.ones(d, device=sv.DEV)

    def req(**kw):
        base = dict(tokens=t, dtype="f32", head_dim=d, rope_dims=d, rope_theta=THETA, positions_ptr=sv.ptr(p), sections=[8, 12, 12],
                    query_heads=2, q_ptr=sv.ptr(q), q_out_ptr=sv.ptr(qo), key_heads=1, k_ptr=sv.ptr(k), k_out_ptr=sv.ptr(ko),
                    q_norm_ptr=sv.ptr(w), eps=EPS)
        base.update(kw)
        return gpu_ctx.rotary_request(**base)

    def status(r):
        with pytest.raises(abi.AbiError) as e:
            gpu_ctx.rotary_device(r, stream=sv.stream())
        return e.value.status

    gpu_ctx.rotary_device(req(), stream=sv.stream())
    for bad in (dict(tokens=0), dict(query_heads=0, key_heads=0), dict(head_dim=0), dict(q_ptr=None), dict(k_out_ptr=None),
                dict(positions_ptr=None), dict(sections=[8, 12, 11]), dict(sections=[8, 12, 12, 1]), dict(sections=[2 ** 32 - 1, 33]),
                dict(query_stride=d), dict(key_out_stride=d - 1), dict(position_stride=t - 1), dict(q_out_ptr=sv.ptr(q), query_out_stride=3 * d),
                dict(q_out_ptr=sv.ptr(q) + 4), dict(q_out_ptr=sv.ptr(k)), dict(q_out_ptr=sv.ptr(ko)), dict(k_out_ptr=sv.ptr(w)),
                dict(k_out_ptr=sv.ptr(p) + 16), dict(k_out_ptr=sv.ptr(q) + 4 * d, key_out_stride=2 * d)):
        assert status(req(**bad)) == -1, bad
    for bad in (dict(head_dim=257, rope_dims=64), dict(rope_dims=63), dict(rope_dims=66), dict(rope_theta=0.0),
                dict(rope_theta=float("inf")), dict(rope_theta=float("nan")), dict(rope_theta=-1.0)):
        assert status(req(**bad)) == -5, bad
    r = req()
    r.dtype = 3
    assert status(r) == -1
    r = req()
    r.header.struct_size -= 1
    assert status(r) == -1
    torch.cuda.synchronize()


def test_captured_with_other_positions(gpu_ctx):
    """Recorded once; each replay, and the eager call between two, take the positions that are there."""
    t, heads, d = 33, 4, 128
    g = sv.gen(2)
    q = sv.normal(g, t, heads * d).to(torch.bfloat16).to(sv.DEV)
    p = torch.zeros(3, t, dtype=torch.int32, device=sv.DEV)
    out, want = torch.zeros_like(q), torch.zeros_like(q)
    req = lambda o: gpu_ctx.rotary_request(t, "bf16", d, d, THETA, sv.ptr(p), sections=[16, 24, 24], in_turn=True, query_heads=heads,  # noqa: E731
                                           q_ptr=sv.ptr(q), q_out_ptr=sv.ptr(o))
    r, e = req(out), req(want)
    gpu_ctx.rotary_device(e, stream=sv.stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu_ctx.rotary_device(r, stream=sv.stream())
    for i in range(4):
        p.copy_(positions_of(sv.gen(i), 3, t))
        graph.replay()
        gpu_ctx.rotary_device(e, stream=sv.stream())
        torch.cuda.synchronize()
        assert torch.equal(out, want)
