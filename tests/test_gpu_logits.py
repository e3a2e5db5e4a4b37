"""Penalties, biases and masks on logits, and the greedy ids
(qwn_hip_ext_logits_process_device), against the definition in 64 bits."""
import math

import pytest
import torch

import serving as sv
from qwanto_amd import abi

pytestmark = pytest.mark.gpu


def reference(x, hist, prompts, rep, pres, freq, biases, masks):
    """Row by row on the host: the processed logits in x's type and the ids."""
    out = x.double().clone()
    rows, vocab = x.shape
    for r in range(rows):
        seen, made = set(), {}
        for j, t in enumerate(hist[r]):
            if 0 <= t < vocab:
                seen.add(t)
                if j >= prompts[r]:
                    made[t] = made.get(t, 0) + 1
        for t in seen:
            v = float(out[r, t])
            v = v / rep[r] if v > 0 else v * rep[r]
            if t in made:
                v = v - made[t] * freq[r] - pres[r]
            out[r, t] = v
        add = {}
        for t, b in biases[r]:
            if 0 <= t < vocab:
                add[t] = add.get(t, 0.0) + b
        for t, b in add.items():
            out[r, t] += b
    y = out.float().to(x.dtype)
    for r in range(rows):
        if masks[r] is not None:
            y[r][~masks[r]] = -math.inf
    ids = []
    for r in range(rows):
        v = y[r].float()
        v = torch.where(torch.isnan(v), torch.full_like(v, -math.inf), v)
        top = float(v.max())
        ids.append(int((v == top).nonzero()[0, 0]) if top > -math.inf else -1)
    return y, ids


def pack(mask):
    n = -(-mask.numel() // 32)
    bits = torch.zeros(n * 32, dtype=torch.int64)
    bits[:mask.numel()] = mask.long()
    w = (bits.reshape(n, 32) << torch.arange(32)).sum(1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def run(ctx, x, hist, prompts, rep, pres, freq, biases, masks, dtype, in_place=False, in_stride=None, out_stride=None, ids=True):
    rows, vocab = x.shape
    dev = sv.DEV

    def ragged(lists):
        starts = [0]
        for v in lists:
            starts.append(starts[-1] + len(v))
        flat = [t for v in lists for t in v]
        return flat, torch.tensor(starts, dtype=torch.int32, device=dev)

    si = in_stride or vocab
    xd = torch.full((rows, si), 5.0, dtype=sv.DTYPES[dtype], device=dev)
    xd[:, :vocab] = x.to(dev)
    so = si if in_place else out_stride or vocab
    out = xd if in_place else torch.full((rows, so), 5.0, dtype=sv.DTYPES[dtype], device=dev)
    flat, hs = ragged(hist)
    h = torch.tensor(flat, dtype=torch.int32, device=dev)
    bt, bs = ragged([[t for t, _ in b] for b in biases])
    bv, _ = ragged([[v for _, v in b] for b in biases])
    bt, bv = torch.tensor(bt, dtype=torch.int32, device=dev), torch.tensor(bv, dtype=torch.float32, device=dev)
    f32 = lambda v: torch.tensor(v, dtype=torch.float32, device=dev)  # noqa: E731
    rp, pr, fq = f32(rep), f32(pres), f32(freq)
    pc = torch.tensor(prompts, dtype=torch.int32, device=dev)
    have = [m for m in masks if m is not None]
    mk = torch.stack([pack(m) for m in have]).to(dev) if have else None
    idx, at = [], 0
    for m in masks:
        idx.append(at if m is not None else -1)
        at += m is not None
    mi = torch.tensor(idx, dtype=torch.int32, device=dev)
    idt = torch.full((rows,), -7, dtype=torch.int32, device=dev)
    work = torch.full((max(8, ctx.logits_workspace_bytes(rows, vocab)),), 0xff, dtype=torch.uint8, device=dev)
    req = ctx.logits_request(rows, vocab, dtype, sv.ptr(xd), sv.ptr(out), in_stride=si, out_stride=so,
                             history_ptr=sv.ptr(h) if flat else None, history_starts_ptr=sv.ptr(hs), history_capacity=len(flat),
                             prompt_counts_ptr=sv.ptr(pc), repetition_ptr=sv.ptr(rp), presence_ptr=sv.ptr(pr),
                             frequency_ptr=sv.ptr(fq), bias_tokens_ptr=sv.ptr(bt) if bt.numel() else None,
                             bias_values_ptr=sv.ptr(bv), bias_starts_ptr=sv.ptr(bs), bias_capacity=bt.numel(),
                             mask_ptr=sv.ptr(mk), mask_rows=len(have), mask_index_ptr=sv.ptr(mi) if have else None,
                             ids_ptr=sv.ptr(idt) if ids else None, workspace_ptr=sv.ptr(work))
    ctx.logits_process_device(req, stream=sv.stream())
    torch.cuda.synchronize()
    out = out.cpu()
    assert bool((out[:, vocab:] == 5.0).all())   # behind the rows
    return out[:, :vocab], idt.cpu().tolist()


def case(seed, rows, vocab, dtype, history=40, nbias=9, masked=True):
    g = sv.gen(seed)
    x = (3.0 * sv.normal(g, rows, vocab)).to(sv.DTYPES[dtype])
    ri = lambda hi: int(torch.randint(0, hi, (1,), generator=g))  # noqa: E731
    hist = [[ri(vocab) if ri(10) else ri(max(1, vocab // 50)) for _ in range(ri(history + 1))] for _ in range(rows)]
    for h in hist:
        if len(h) > 4:
            h[1], h[2], h[3] = -1, vocab, h[0]
    prompts = [ri(len(h) + 1) for h in hist]
    u = lambda lo, hi: [lo + (hi - lo) * float(torch.rand(1, generator=g)) for _ in range(rows)]  # noqa: E731
    f32 = lambda v: torch.tensor(v, dtype=torch.float32).tolist()  # noqa: E731
    rep, pres, freq = f32(u(0.8, 1.6)), f32(u(-0.5, 1.0)), f32(u(0.0, 0.7))
    biases = [[(ri(vocab), float(v)) for v in 4.0 * sv.normal(g, ri(nbias + 1))] for _ in range(rows)]
    for b in biases:
        if len(b) > 3:
            b[2] = (b[0][0], b[2][1])        # the same token twice
            b[3] = (-1, 1.0)
    masks = [torch.rand(vocab, generator=g) < (0.02, 0.5, 0.97)[ri(3)] if masked and ri(3) else None for _ in range(rows)]
    return x, hist, prompts, rep, pres, freq, biases, masks


def check(got, want, x):
    (y, ids), (yr, idr) = got, want
    assert torch.equal(torch.isnan(y), torch.isnan(yr))
    # both are the 64-bit value rounded to fp32 and to the type; sums of 64-bit terms in another order
    # move a value by 2^-50, and a rounding next to a border by one step
    fine = ~torch.isnan(yr)
    off = (y.double() - yr.double()).abs()[fine & torch.isfinite(yr)]
    assert torch.equal(y[fine & ~torch.isfinite(yr)], yr[fine & ~torch.isfinite(yr)])
    assert float((off > 0).double().mean() if off.numel() else 0.0) <= 1e-4
    assert bool((off <= 2 * 2.0 ** -8 * yr.double().abs()[fine & torch.isfinite(yr)]).all())
    assert ids == idr


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 5), (3, 33), (2, 4095), (2, 4096), (3, 4097), (1, 20011), (5, 9001)])
def test_against_definition(gpu_ctx, dtype, rows, vocab):
    c = case(rows * 7 + vocab, rows, vocab, dtype)
    check(run(gpu_ctx, *c, dtype), reference(*c), c[0])


def test_large_vocabulary(gpu_ctx):
    c = case(5, 3, 151936, "f32", history=900, nbias=300)
    check(run(gpu_ctx, *c, "f32"), reference(*c), c[0])


@pytest.mark.parametrize("lengths", [(1023, 1024), (1025, 1028), (6001, 2500)])
def test_long_lists(gpu_ctx, lengths):
    """Histories and biases past what a workgroup loads ahead, and at its ends."""
    vocab, rows = 9001, 2
    x, hist, prompts, rep, pres, freq, biases, masks = case(11, rows, vocab, "f32", masked=False)
    g = sv.gen(12)
    for r in range(rows):
        hist[r] = torch.randint(0, vocab, (lengths[r],), generator=g).tolist()
        prompts[r] = lengths[r] // 3
        n = lengths[1 - r]
        biases[r] = list(zip(torch.randint(0, vocab, (n,), generator=g).tolist(), sv.normal(g, n).tolist()))
    c = (x, hist, prompts, rep, pres, freq, biases, masks)
    check(run(gpu_ctx, *c, "f32"), reference(*c), x)


def test_biases_of_one_token(gpu_ctx):
    """Lists that name one token often, across every step of the search for it, sums of very unlike
    sizes among them: added in the list's order."""
    vocab = 5000
    g = sv.gen(9)
    x = sv.normal(g, 3, vocab)
    few = [(int(t), float(b)) for t, b in zip(torch.randint(0, 7, (900,), generator=g), sv.normal(g, 900))]
    one = [(4321, 1e8 if i == 3 else -1e8 if i == 700 else 0.125) for i in range(800)]
    nobody = [[], [], []]
    args = (x, nobody, [0] * 3, [1.0] * 3, [0.0] * 3, [0.0] * 3, [few, one, [(0, 1.0), (2100, 2.0), (0, 3.0)]], [None] * 3)
    check(run(gpu_ctx, *args, "f32"), reference(*args), x)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_in_place(gpu_ctx, dtype):
    c = case(6, 4, 5001, dtype)
    want = reference(*c)
    check(run(gpu_ctx, *c, dtype, in_stride=5003, out_stride=5101), want, c[0])
    check(run(gpu_ctx, *c, dtype, in_stride=5004, in_place=True), want, c[0])
    y, _ = run(gpu_ctx, *c, dtype, ids=False)
    assert torch.equal(y, run(gpu_ctx, *c, dtype)[0])


def test_rows_with_nothing_left(gpu_ctx):
    """A row whose mask allows nothing, or only tokens at -inf or NaN, has the id -1; infinities and
    NaN in masked places do not reach the output; ties and signed zeros go to the first index."""
    x = torch.zeros(7, 200)
    x[:, 150] = 1.0
    x[1, 10] = math.nan
    x[1, 11] = math.inf
    x[2] = -math.inf
    x[3, 40] = x[3, 30] = 2.0
    x[4] = -1.0
    x[4, 20], x[4, 21] = -0.0, 0.0
    x[4, 150] = -1.0
    x[5, 60] = math.inf
    x[6, 0] = math.nan
    allow = torch.ones(200, dtype=torch.bool)
    none = torch.zeros(200, dtype=torch.bool)
    no_10_11 = allow.clone()
    no_10_11[10:12] = False
    only = none.clone()
    only[5] = True
    masks = [none, no_10_11, only, allow, None, None, None]
    nobody = [[] for _ in range(7)]
    args = (x, nobody, [0] * 7, [1.0] * 7, [0.0] * 7, [0.0] * 7, nobody, masks)
    y, ids = run(gpu_ctx, *args, "f32")
    assert ids == [-1, 150, -1, 30, 20, 60, 150]
    assert bool((y[0] == -math.inf).all()) and bool((y[1, 10:12] == -math.inf).all()) and bool(torch.isnan(y[6, 0]))


def test_lists_that_do_not_lie_in_their_capacity_are_left_out(gpu_ctx):
    x = torch.ones(3, 64)
    xd = x.to(sv.DEV)
    out = torch.zeros(3, 64, device=sv.DEV)
    h = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device=sv.DEV)
    starts = torch.tensor([0, 2, 1, 5], dtype=torch.int32, device=sv.DEV)       # one row fits
    rep = torch.full((3,), 2.0, device=sv.DEV)
    idx = torch.tensor([-2, 1, 0], dtype=torch.int32, device=sv.DEV)             # one mask exists
    mask = torch.zeros(1, 2, dtype=torch.int32, device=sv.DEV)
    req = gpu_ctx.logits_request(3, 64, "f32", sv.ptr(xd), sv.ptr(out), history_ptr=sv.ptr(h), history_starts_ptr=sv.ptr(starts),
                                 history_capacity=4, repetition_ptr=sv.ptr(rep), mask_ptr=sv.ptr(mask), mask_rows=1,
                                 mask_index_ptr=sv.ptr(idx))
    gpu_ctx.logits_process_device(req, stream=sv.stream())
    torch.cuda.synchronize()
    want = x.clone()
    want[0, 1:3] = 0.5
    want[2] = -math.inf
    assert torch.equal(out.cpu(), want)


def test_refusals(gpu_ctx):
    x = torch.zeros(2, 64, device=sv.DEV)
    i = torch.zeros(64, dtype=torch.int32, device=sv.DEV)

    def req(**kw):
        base = dict(logits_ptr=sv.ptr(x), out_ptr=sv.ptr(x))
        base.update(kw)
        return gpu_ctx.logits_request(2, 64, "f32", **base)

    gpu_ctx.logits_process_device(req(), stream=sv.stream())
    bad = [req(logits_ptr=None), req(out_ptr=None), req(in_stride=63, out_stride=63), req(out_stride=65), req(history_ptr=sv.ptr(i)),
           req(bias_tokens_ptr=sv.ptr(i), bias_values_ptr=sv.ptr(x)), req(bias_tokens_ptr=sv.ptr(i), bias_starts_ptr=sv.ptr(i)),
           req(mask_ptr=sv.ptr(i), mask_rows=1), req(mask_ptr=sv.ptr(i), mask_rows=2, mask_stride=1),
           req(mask_ptr=sv.ptr(i), mask_index_ptr=sv.ptr(i)), req(ids_ptr=sv.ptr(i)),
           req(ids_ptr=sv.ptr(i), workspace_ptr=sv.ptr(x) + 4)]
    for field, value in (("rows", 0), ("rows", 65536), ("vocab", 0), ("dtype", 9)):
        r = req()
        setattr(r, field, value)
        bad.append(r)
    for r in bad:
        with pytest.raises(abi.AbiError) as e:
            gpu_ctx.logits_process_device(r, stream=sv.stream())
        assert e.value.status == -1
