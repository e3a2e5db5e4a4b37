"""Requests of the serving operators whose outputs share bytes with their inputs or each other are
refused; results in place and columns of one buffer are not."""
import pytest
import torch

import serving as sv
from qwanto_amd import abi

pytestmark = pytest.mark.gpu


def refused(call, *args):
    with pytest.raises(abi.AbiError) as e:
        call(*args)
    assert e.value.status == -1 and "overlap" in str(e.value)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm(gpu_ctx, dtype):
    t, c, dt = 5, 64, sv.DTYPES[dtype]
    size = torch.finfo(dt).bits // 8
    buf = torch.zeros(t + 1, 4 * c, dtype=dt, device=sv.DEV)
    at = lambda row, col: sv.ptr(buf) + (row * 4 * c + col) * size  # noqa: E731
    w, q8 = torch.ones(c, device=sv.DEV), torch.zeros(t, 80, dtype=torch.int8, device=sv.DEV)
    s = torch.zeros(t, device=sv.DEV)

    def req(**kw):
        base = dict(x_ptr=at(0, 0), norm_ptr=sv.ptr(w), eps=1e-6, residual_ptr=at(0, c), residual_out_ptr=at(0, 2 * c), y_ptr=at(0, 3 * c),
                    q8_ptr=sv.ptr(q8), scales_ptr=sv.ptr(s), x_stride=4 * c, residual_stride=4 * c, residual_out_stride=4 * c,
                    y_stride=4 * c, q8_stride=80)
        base.update(kw)
        return gpu_ctx.norm_request(t, c, dtype, **base)

    for good in (req(), req(residual_out_ptr=at(0, 0)), req(residual_out_ptr=at(0, c)), req(residual_ptr=at(0, 0)),
                 req(residual_ptr=at(0, 0), residual_out_ptr=at(0, 0)), req(q8_ptr=None, scales_ptr=sv.ptr(w))):
        gpu_ctx.norm_quantize_device(good, stream=sv.stream())
    torch.cuda.synchronize()
    for bad in (dict(residual_out_ptr=at(1, 0)), dict(residual_out_ptr=at(0, 1)), dict(residual_out_ptr=at(0, 3 * c - 1)),
                dict(y_ptr=at(0, 0)), dict(y_ptr=at(0, c)), dict(y_ptr=at(0, 2 * c)), dict(y_ptr=at(0, 3 * c + 1)),
                dict(q8_ptr=at(0, 0)), dict(q8_ptr=at(t - 1, c + 5)), dict(q8_ptr=at(t - 1, 3 * c)), dict(scales_ptr=at(2, c - 1)),
                dict(scales_ptr=sv.ptr(q8) + 5 * 80 - 4), dict(scales_ptr=sv.ptr(w) + 4), dict(q8_ptr=sv.ptr(w)),
                dict(y_ptr=sv.ptr(w)), dict(residual_out_ptr=sv.ptr(w))):
        refused(gpu_ctx.norm_quantize_device, req(**bad), sv.stream())


def test_logits(gpu_ctx):
    rows, vocab = 3, 70
    x = torch.zeros(rows, 2 * vocab, device=sv.DEV)
    i = {n: torch.zeros(k, dtype=torch.int32, device=sv.DEV) for n, k in
         dict(history=9, history_starts=rows + 1, prompt_counts=rows, bias_tokens=5, bias_starts=rows + 1, mask=2 * 3,
              mask_index=rows, ids=rows).items()}
    f = {n: torch.zeros(k, device=sv.DEV) for n, k in dict(repetition=rows, presence=rows, frequency=rows, bias_values=5).items()}
    f["repetition"] += 1
    work = torch.zeros(gpu_ctx.logits_workspace_bytes(rows, vocab), dtype=torch.uint8, device=sv.DEV)
    given = {n + "_ptr": sv.ptr(t) for n, t in (i | f).items()} | dict(workspace_ptr=sv.ptr(work))

    def req(**kw):
        base = dict(logits_ptr=sv.ptr(x), out_ptr=sv.ptr(x) + 4 * vocab, in_stride=2 * vocab, out_stride=2 * vocab, history_capacity=9,
                    bias_capacity=5, mask_rows=2) | given
        base.update(kw)
        return gpu_ctx.logits_request(rows, vocab, "f32", **base)

    for good in (req(), req(out_ptr=sv.ptr(x)), req(ids_ptr=None, workspace_ptr=sv.ptr(x))):
        gpu_ctx.logits_process_device(good, stream=sv.stream())
    torch.cuda.synchronize()
    refused(gpu_ctx.logits_process_device, req(out_ptr=sv.ptr(x) + 4), sv.stream())
    refused(gpu_ctx.logits_process_device, req(out_ptr=sv.ptr(x) + 8 * vocab), sv.stream())
    refused(gpu_ctx.logits_process_device, req(workspace_ptr=sv.ptr(x)), sv.stream())
    refused(gpu_ctx.logits_process_device, req(workspace_ptr=sv.ptr(x) + 4 * vocab), sv.stream())
    refused(gpu_ctx.logits_process_device, req(ids_ptr=sv.ptr(x)), sv.stream())
    refused(gpu_ctx.logits_process_device, req(ids_ptr=sv.ptr(work)), sv.stream())
    for n in given:
        if n not in ("ids_ptr", "workspace_ptr"):
            refused(gpu_ctx.logits_process_device, req(ids_ptr=given[n]), sv.stream())
            refused(gpu_ctx.logits_process_device, req(**{n: sv.ptr(x) + 4 * vocab}), sv.stream())


def test_cache(gpu_ctx):
    hk, heads, d, rows = 2, 4, 64, 6
    c = sv.Cache(gpu_ctx, [32, 32], hk, d)
    try:
        b = c.batch([0, 0], [4, 2])
        wide = (2 * hk + 2 * heads) * d
        buf = torch.zeros(rows + 1, wide, device=sv.DEV)
        at = lambda row, col: sv.ptr(buf) + (row * wide + col) * 4  # noqa: E731
        q, qo, k, v = 0, heads * d, 2 * heads * d, (2 * heads + hk) * d
        pos = torch.zeros(rows, dtype=torch.int32, device=sv.DEV)

        def app(**kw):
            base = dict(k_ptr=at(0, k), v_ptr=at(0, v), q_ptr=at(0, q), q_out_ptr=at(0, qo), query_heads=heads, positions_ptr=sv.ptr(pos),
                        key_stride=wide, value_stride=wide, query_stride=wide, query_out_stride=wide)
            base.update(kw)
            return gpu_ctx.paged_append_request(b, "f32", **base)

        for good in (app(), app(q_out_ptr=at(0, q)), app(v_ptr=at(0, k)), app(q_ptr=None, q_out_ptr=at(0, k))):
            gpu_ctx.paged_kv_append_device(c.h, good, stream=sv.stream())
        torch.cuda.synchronize()
        starts = b.starts
        for bad in (dict(q_out_ptr=at(0, 1)), dict(q_out_ptr=at(1, q)), dict(q_out_ptr=at(0, k)), dict(q_out_ptr=at(0, qo + 1)),
                    dict(q_out_ptr=at(0, v)), dict(q_out_ptr=sv.ptr(pos)), dict(q_out_ptr=starts), dict(q_out_ptr=b.page_table)):
            refused(gpu_ctx.paged_kv_append_device, c.h, app(**bad), sv.stream())

        out = torch.zeros(2, rows, 2 * hk * d, device=sv.DEV)
        read = lambda kp, vp, stride: gpu_ctx.paged_kv_read_device(c.h, b, kp, vp, stride, stream=sv.stream())  # noqa: E731
        read(sv.ptr(out), sv.ptr(out) + 4 * hk * d, 2 * hk * d)
        torch.cuda.synchronize()
        refused(read, sv.ptr(out), sv.ptr(out), 0)
        refused(read, sv.ptr(out), sv.ptr(out) + 4 * hk * d - 4, 2 * hk * d)
        refused(read, None, starts, 0)
        refused(read, b.past, None, 0)

        def att(**kw):
            r = gpu_ctx.paged_attention_request(b, "f32", heads, at(0, q), at(0, qo), 0.1, workspace_ptr=sv.ptr(work), query_stride=wide,
                                                output_stride=wide)
            for n, p in kw.items():
                setattr(r, n, p)
            return r

        need = gpu_ctx.paged_attention_workspace_bytes(c.h, gpu_ctx.paged_attention_request(b, "f32", heads, at(0, q), at(0, qo), 0.1))
        work = torch.zeros(need + 64, dtype=torch.uint8, device=sv.DEV)
        gpu_ctx.paged_kv_attention_device(c.h, att(), stream=sv.stream())
        torch.cuda.synchronize()
        for bad in (dict(output=at(0, q)), dict(output=at(0, 5)), dict(output=at(1, q)), dict(output=sv.ptr(work) + need - 4),
                    dict(query=sv.ptr(work)), dict(workspace=at(0, 0)), dict(output=starts), dict(output=b.page_table)):
            refused(gpu_ctx.paged_kv_attention_device, c.h, att(**bad), sv.stream())
    finally:
        c.close()
