"""The residual's addition, RMSNorm and int8 quantization in one pass
(qwn_hip_ext_norm_quantize_device), against the definition in 64 bits."""
import pytest
import torch

import serving as sv
from qwanto_amd import abi

pytestmark = pytest.mark.gpu
EPS = 1e-6


def run(ctx, x, r, w, dtype, q8_pad=0, strides=None, eps=EPS, in_place=None):
    """All outputs, from tensors on the host laid out as given."""
    dev = sv.DEV
    t, c = x.shape[0], w.numel()
    def there(v):   # on the GPU with its strides
        return torch.empty_strided(v.shape, v.stride(), dtype=v.dtype, device=dev).copy_(v)

    xd, wd = there(x), w.to(dev)
    rd = there(r) if r is not None else None
    st = dict(x_stride=x.stride(0), residual_stride=r.stride(0) if r is not None else 0)
    if in_place == "x":
        out = xd
    elif in_place == "residual":
        out = rd
    else:
        out = torch.full((t, c), float("nan"), dtype=sv.DTYPES[dtype], device=dev)
    y = torch.full((t, c), float("nan"), dtype=sv.DTYPES[dtype], device=dev)
    q = torch.full((t, c + q8_pad), 77, dtype=torch.int8, device=dev)
    s = torch.full((t,), -1.0, device=dev)
    req = ctx.norm_request(t, c, dtype, sv.ptr(xd), sv.ptr(wd), eps, residual_ptr=sv.ptr(rd), residual_out_ptr=sv.ptr(out),
                           y_ptr=sv.ptr(y), q8_ptr=sv.ptr(q), scales_ptr=sv.ptr(s), q8_stride=c + q8_pad,
                           residual_out_stride=out.stride(0), **st)
    ctx.norm_quantize_device(req, stream=sv.stream())
    torch.cuda.synchronize()
    return out.cpu()[:, :c], y.cpu(), q.cpu(), s.cpu()


def check(h, y, q, s, x, r, w, dtype, eps=EPS):
    c = w.numel()
    hr = x if r is None else (x.float() + r.float()).to(x.dtype)
    assert torch.equal(h, hr)
    wide = hr.double()
    y64 = wide * w.double() / (wide.square().mean(1, keepdim=True) + eps).sqrt()
    y32 = y64.float()
    # y: the 64-bit value rounded to fp32 and to the type, each by at most half a step
    tol = (2.0 ** -24 + (sv.HALF[dtype] if dtype != "f32" else 0.0)) * (1 + 1e-6)
    tiny = 2.0 ** -25 if dtype == "f16" else 2.0 ** -134 if dtype == "bf16" else 2.0 ** -149
    assert bool(((y.double() - y64).abs() <= tol * y64.abs() + tiny).all())
    q8, scale = sv.quantize8(y32)
    assert torch.equal(s, scale)
    assert torch.equal(q[:, :c], q8)
    assert not bool(q[:, c:].any())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,cols", [(1, 1), (3, 2), (1, 7), (5, 64), (2, 255), (7, 363), (3, 1536), (61, 2560), (2, 4097),
                                         (2, 9728), (1, 16385), (1, 32769), (2, 40000)])
def test_sizes(gpu_ctx, dtype, tokens, cols):
    g = sv.gen(tokens * 131 + cols)
    big = torch.where(torch.rand(cols, generator=g) < 0.02, 20.0, 1.0)
    x = (0.7 * sv.normal(g, tokens, cols)).to(sv.DTYPES[dtype])
    r = (2.0 * sv.normal(g, tokens, cols) * big).to(sv.DTYPES[dtype])
    w = 1.0 + 0.3 * sv.normal(g, cols)
    check(*run(gpu_ctx, x, r, w, dtype, q8_pad=5), x, r, w, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad", [1, 3, 8])
def test_strided_rows_and_no_residual(gpu_ctx, dtype, pad):
    g = sv.gen(5 + pad)
    x = sv.normal(g, 9, 515 + pad).to(sv.DTYPES[dtype])[:, :515]
    w = 1.0 + 0.3 * sv.normal(g, 515)
    check(*run(gpu_ctx, x, None, w, dtype), x, None, w, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("cols", [130, 33000])
@pytest.mark.parametrize("place", ["x", "residual"])
def test_in_place(gpu_ctx, dtype, cols, place):
    g = sv.gen(cols)
    x, r = (sv.normal(g, 4, cols).to(sv.DTYPES[dtype]) for _ in range(2))
    w = 1.0 + 0.3 * sv.normal(g, cols)
    check(*run(gpu_ctx, x, r, w, dtype, in_place=place), x, r, w, dtype)


def test_equals_quantize_device(gpu_ctx):
    """q8 and the scales are those of qwn_hip_ext_quantize_device on y."""
    g = sv.gen(1)
    x = sv.normal(g, 33, 1536)
    w = 1.0 + 0.3 * sv.normal(g, 1536)
    _, y, q, s = run(gpu_ctx, x, None, w, "f32")
    yd = y.to(sv.DEV)
    q2, s2 = torch.empty(33, 1536, dtype=torch.int8, device=sv.DEV), torch.empty(33, device=sv.DEV)
    gpu_ctx.quantize_device(sv.ptr(yd), 33, 1536, 1536, sv.ptr(q2), 1536, sv.ptr(s2), stream=sv.stream())
    torch.cuda.synchronize()
    assert torch.equal(q, q2.cpu()) and torch.equal(s, s2.cpu())


@pytest.mark.parametrize("cols", [200, 33000])
def test_rows_that_are_zero_or_not_finite(gpu_ctx, cols):
    """A zero row has the scale 1; one with an infinity or a NaN, or whose y overflow, has the scale
    NaN and zeros; its neighbours are untouched by it."""
    g = sv.gen(2)
    x = sv.normal(g, 6, cols)
    w = 1.0 + 0.3 * sv.normal(g, cols)
    x[0] = 0.0
    x[1, 3] = float("nan")
    x[3, cols - 1] = float("-inf")
    x[4, 5] = 3.0e38
    w[7] = 1.0e38
    x[4, 7] = 3.0e38          # y of about sqrt(cols / 2) * 1e38
    x[2, 7] = x[5, 7] = 0.0
    h, y, q, s = run(gpu_ctx, x, None, w, "f32")
    assert float(s[0]) == 1.0 and not bool(q[0].any()) and not bool(y[0].any())
    for row in (1, 3, 4):
        assert bool(torch.isnan(s[row])) and not bool(q[row].any())
    for row in (2, 5):
        check(h[row:row + 1], y[row:row + 1], q[row:row + 1], s[row:row + 1], x[row:row + 1], None, w, "f32")


def test_single_outputs(gpu_ctx):
    """Each output alone is what it is among the others."""
    g = sv.gen(3)
    x, w = sv.normal(g, 4, 96), 1.0 + 0.3 * sv.normal(g, 96)
    h, y, q, s = run(gpu_ctx, x, x, w, "f32")
    xd, wd = x.to(sv.DEV), w.to(sv.DEV)
    for name, want in (("y", y), ("residual_out", h), ("q8", q)):
        out = torch.full(want.shape, 9, dtype=want.dtype, device=sv.DEV)
        sc = torch.zeros(4, device=sv.DEV)
        kw = {name + "_ptr": sv.ptr(out)} | ({"scales_ptr": sv.ptr(sc)} if name == "q8" else {})
        gpu_ctx.norm_quantize_device(gpu_ctx.norm_request(4, 96, "f32", sv.ptr(xd), sv.ptr(wd), EPS, residual_ptr=sv.ptr(xd), **kw),
                                     stream=sv.stream())
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), want)


def test_refusals(gpu_ctx):
    x = torch.zeros(4, 64, device=sv.DEV)
    w, q, s = torch.ones(64, device=sv.DEV), torch.zeros(4, 64, dtype=torch.int8, device=sv.DEV), torch.zeros(4, device=sv.DEV)

    def req(**kw):
        base = dict(x_ptr=sv.ptr(x), norm_ptr=sv.ptr(w), eps=EPS, q8_ptr=sv.ptr(q), scales_ptr=sv.ptr(s))
        base.update(kw)
        return gpu_ctx.norm_request(4, 64, "f32", **base)

    gpu_ctx.norm_quantize_device(req(), stream=sv.stream())
    bad = [req(x_ptr=None), req(norm_ptr=None), req(scales_ptr=None), req(q8_ptr=None), req(x_stride=63), req(q8_stride=63),
           req(y_ptr=sv.ptr(x), y_stride=8), req(residual_ptr=sv.ptr(x), residual_stride=5),
           req(residual_out_ptr=sv.ptr(x), residual_out_stride=65), req(y_ptr=sv.ptr(x)),
           req(residual_ptr=sv.ptr(s), y_ptr=sv.ptr(s)), req(residual_out_ptr=sv.ptr(s), y_ptr=sv.ptr(s))]
    for field, value in (("tokens", 0), ("cols", 0), ("dtype", 3), ("tokens", 0x80000000)):
        r = req()
        setattr(r, field, value)
        bad.append(r)
    r = req()
    r.header.struct_size = 16
    bad.append(r)
    for r in bad:
        with pytest.raises(abi.AbiError) as e:
            gpu_ctx.norm_quantize_device(r, stream=sv.stream())
        assert e.value.status == -1
