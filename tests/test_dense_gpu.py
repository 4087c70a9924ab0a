"""The dense operators (8-bit rows, scaled scores, softmax loss over documents with its gradients) against plain
implementations in 64 bits.

Tolerances, from the arithmetic.  A rounding to a type is off by at most u = eps / 2 of the value (bf16 2^-8, f16 2^-11, f32
2^-24).  8-bit rows are exact: whole bytes are compared.  Scores and logits: products of two e4m3 values (or two 16-bit ones)
are exact in fp32, a sum of K of them in fp32 is off by at most K roundings of partial sums, K * 2^-23 * sum |a b| (2^-23: the
tensor core may cut instead of rounding), plus one rounding to the output type."""
import numpy as np
import pytest
import torch

import apoe

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def spread(rows, cols, g, dtype=torch.float32):
    """Values over many binades: every row and block has a size of its own."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    return (x * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g, device=DEV).float())).to(dtype)


# ---- 8-bit rows -----------------------------------------------------------------------------------------------------------
def plain_quantize(x):
    """64 bits, from the definition: the smallest exponent by trial, rounding to e4m3 by hand."""
    x = x.double().cpu()
    rows, dim = x.shape
    blocks = -(-dim // 128)
    q, scale = torch.zeros_like(x), torch.zeros(rows, blocks, dtype=torch.int64)
    for b in range(blocks):
        part = x[:, b * 128:(b + 1) * 128]
        top = torch.where(torch.isnan(part), torch.zeros_like(part), part).abs().amax(1).clamp(max=2.0 ** 128)
        e = torch.full((rows,), -126, dtype=torch.int64)
        for k in range(-126, 122):
            e = torch.where(top > 448.0 * 2.0 ** k, torch.full_like(e, k + 1), e)
        v = part * torch.pow(torch.tensor(2.0, dtype=torch.float64), -e.double())[:, None]
        _, kv = torch.frexp(v.abs().clamp(max=448.0))
        step = torch.pow(torch.tensor(2.0, dtype=torch.float64), ((kv - 1).clamp(min=-6) - 3).double())
        r = torch.round(v / step) * step
        q[:, b * 128:(b + 1) * 128] = torch.where(torch.isinf(v), torch.sign(v) * 448.0, r)
        scale[:, b] = e + 127
    return q, scale


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 127), (5, 128), (64, 1024), (33, 776), (257, 130), (2, 4096 + 5)])
def test_quantize_equals_the_definition(rows, dim, dtype):
    x = spread(rows, dim, gen(rows * 7 + dim), dtype)
    q, scale = apoe.quantize_rows(x)
    want_q, want_s = plain_quantize(x)
    assert torch.equal(scale.cpu().long(), want_s)
    assert torch.equal(q.cpu().double(), want_q)
    assert q.stride(0) % 16 == 0


def test_quantize_borders_and_odd_values():
    x = torch.zeros(12, 128, device=DEV)
    x[0, 5] = 448.0                                   # the largest value of scale 2^0
    x[1, 5] = float(np.nextafter(np.float32(448.0), np.float32(1e9)))   # one step beyond: 2^1
    x[2, 0], x[2, 1] = 3.4028234663852886e38, -1.0    # the largest float
    x[3, 0] = 1e-45                                   # the smallest subnormal: scale stays at 2^-126
    x[4, 3], x[4, 4] = float("nan"), 2.0
    x[5, 3], x[5, 4] = float("inf"), 1.0
    x[6, 3] = float("-inf")
    x[7] = float("nan")
    x[8, :4] = torch.tensor([448.0, 17.0, 19.0, 2.0 ** -10])           # ties: 17 -> 16, 19 -> 20; half the smallest: 0
    x[9, :3] = torch.tensor([448.0, 1.5 * 2.0 ** -9, 2.5 * 2.0 ** -9])  # ties among the subnormals: to even
    x[10] = -0.0
    q, scale = apoe.quantize_rows(x)
    want_q, want_s = plain_quantize(x)
    assert torch.equal(scale.cpu().long(), want_s)
    got = q.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want_q))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want_q))
    assert scale[0, 0] == 127 and scale[1, 0] == 128 and scale[11, 0] == 1
    back = q.float() * (scale.int() << 23).view(torch.float32)
    assert back[5, 3] == float("inf") and back[6, 3] == float("-inf")


def test_quantize_strides_offsets_and_untouched_neighbours():
    g = gen(3)
    wide = spread(40, 300, g)
    for view in (wide[:, 1:258], wide[::2, 3:131], wide[:, :300], wide[5:6, 2:9]):     # unaligned starts, skipped rows
        q, scale = apoe.quantize_rows(view)
        want_q, want_s = plain_quantize(view)
        assert torch.equal(q.cpu().double(), want_q) and torch.equal(scale.cpu().long(), want_s)
    # outputs with rows further apart than they are long: what lies between is left alone
    x = spread(9, 200, g)
    q = torch.full((9, 256), 0x55, dtype=torch.uint8, device=DEV)
    s = torch.full((9, 5), 0x55, dtype=torch.uint8, device=DEV)
    apoe._check(apoe.lib().ap_quantize_rows_device(0, 9, 200, 0, x.data_ptr(), 200, q.data_ptr(), 256, s.data_ptr(), 5,
                                                   torch.cuda.current_stream().cuda_stream))
    want_q, want_s = plain_quantize(x)
    assert torch.equal(q[:, :200].contiguous().view(torch.float8_e4m3fn).cpu().double(), want_q) and bool((q[:, 200:] == 0x55).all())
    assert torch.equal(s[:, :2].cpu().long(), want_s) and bool((s[:, 2:] == 0x55).all())
    empty_q, empty_s = apoe.quantize_rows(torch.empty(0, 64, device=DEV))
    assert empty_q.shape == (0, 64) and empty_s.shape == (0, 1)


# ---- scores ---------------------------------------------------------------------------------------------------------------
def values(q, scale):
    f = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=q.device), scale.double() - 127.0)
    return q.double() * f.repeat_interleave(128, 1)[:, :q.shape[1]]


def check_scores(got, qa, sa, qb, sb, alpha=1.0):
    a, b = values(qa, sa), values(qb, sb)
    want = alpha * (a @ b.t())
    bound = abs(alpha) * (a.abs() @ b.abs().t()) * a.shape[1] * 2.0 ** -23
    u = U[got.dtype]
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[got.dtype]     # half a step of f16's subnormals
    err = (got.double() - want).abs()
    assert bool((err <= bound + u * (want.abs() + bound) + tiny).all()), float((err / (bound + u * want.abs() + 1e-300)).max())
    # and far closer on the whole: roundings add like a walk, not all in one direction
    rms = float((err.square().mean() / want.square().mean().clamp(min=1e-300)).sqrt())
    assert rms <= max(2e-6, 1.2 * u), rms


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,dim", [(1, 1, 16), (1, 1000, 1024), (7, 225, 128), (128, 64, 272), (129, 300, 1024), (200, 33, 100),
                                     (257, 449, 784), (300, 1000, 48), (512, 2048, 1024)])
def test_scores_equal_the_product(m, n, dim, dtype):
    g = gen(m + n + dim)
    qa, sa = apoe.quantize_rows(torch.randn(m, dim, generator=g, device=DEV) * 0.1)
    qb, sb = apoe.quantize_rows(torch.randn(n, dim, generator=g, device=DEV) * 0.1)
    check_scores(apoe.scaled_scores(qa, sa, qb, sb, out_dtype=dtype), qa, sa, qb, sb)
    apoe.dense_check_status()


@pytest.mark.parametrize("m", [5, 300])
def test_scores_use_each_rows_and_blocks_own_scale(m):
    g = gen(9)
    n, dim = 500, 640
    a, b = spread(m, dim, g), spread(n, dim, g)
    for j in range(5):                                # blocks of one row differ as well
        a[:, j * 128:(j + 1) * 128] *= 2.0 ** (3 * j - 7)
        b[:, j * 128:(j + 1) * 128] *= 2.0 ** (5 - 2 * j)
    qa, sa = apoe.quantize_rows(a)
    qb, sb = apoe.quantize_rows(b)
    assert len(torch.unique(sa)) > 10 and len(torch.unique(sb)) > 10
    check_scores(apoe.scaled_scores(qa, sa, qb, sb, alpha=-0.37), qa, sa, qb, sb, alpha=float(np.float32(-0.37)))


@pytest.mark.parametrize("up,down", [(100, -95), (-60, -50), (-110, 115), (60, 55)])
@pytest.mark.parametrize("m", [5, 300])
def test_scores_of_far_apart_scales(m, up, down):
    """Scales whose product is ordinary (or small, or large) although each is near an end of its range."""
    g = gen(14)
    qa, sa = apoe.quantize_rows(torch.randn(m, 200, generator=g, device=DEV) * 2.0 ** up)
    qb, sb = apoe.quantize_rows(torch.randn(90, 200, generator=g, device=DEV) * 2.0 ** down)
    check_scores(apoe.scaled_scores(qa, sa, qb, sb), qa, sa, qb, sb)


def test_scores_wide_narrow_and_many_tiles():
    """More tiles than SMs in every form: wide tiles for few rows, pairs of SMs, groups of row tiles."""
    g = gen(10)
    for m, n, dim in ((3, 148 * 224 + 5, 64), (100, 40000, 256), (1500, 5000, 128), (2300, 3000, 64)):
        qa, sa = apoe.quantize_rows(torch.randn(m, dim, generator=g, device=DEV))
        qb, sb = apoe.quantize_rows(torch.randn(n, dim, generator=g, device=DEV))
        check_scores(apoe.scaled_scores(qa, sa, qb, sb), qa, sa, qb, sb)


def test_scores_strides_and_neighbours():
    g = gen(11)
    m, n, dim = 150, 333, 320
    qa, sa = apoe.quantize_rows(torch.randn(m, 512, generator=g, device=DEV))
    qb, sb = apoe.quantize_rows(torch.randn(2 * n, 512, generator=g, device=DEV))
    va, vsa, vb, vsb = qa[:, 128:448], sa[:, 1:4], qb[::2, 128:448], sb[::2, 1:4]        # 320 values: the last block is short
    for dtype in (torch.float32, torch.float16):
        for off, width in ((0, n + 3), (1, n + 5), (8, n + 11)):                          # unaligned rows take plain stores
            room = torch.full((m, width + off), 7.0, dtype=dtype, device=DEV)
            out = room[:, off:off + n]
            apoe.scaled_scores(va, vsa, vb, vsb, out=out)
            check_scores(out, va, vsa, vb, vsb)
            assert bool((room[:, :off] == 7.0).all()) and bool((room[:, off + n:] == 7.0).all())
    assert apoe.scaled_scores(qa[:0], sa[:0], qb, sb).shape == (0, 2 * n)
    assert apoe.scaled_scores(qa, sa, qb[:0], sb[:0]).shape == (m, 0)


@pytest.mark.parametrize("m", [9, 200])
@pytest.mark.parametrize("dim", [1, 15, 17, 100, 131, 250])
def test_scores_ignore_what_lies_behind_a_row(m, dim):
    g = gen(12)
    qa, sa = apoe.quantize_rows(torch.randn(m, dim, generator=g, device=DEV))
    qb, sb = apoe.quantize_rows(torch.randn(70, dim, generator=g, device=DEV))
    def wide(q, s):                                   # the same rows in the middle of a matrix of the largest values and of NaN
        room = torch.full((q.shape[0], 272), 0x7E, dtype=torch.uint8, device=DEV)
        room[1::2] = 0x7F
        room[:, :dim] = q.view(torch.uint8)
        scales = torch.full((q.shape[0], 8), 254, dtype=torch.uint8, device=DEV)
        scales[:, :s.shape[1]] = s
        return room.view(torch.float8_e4m3fn)[:, :dim], scales[:, :s.shape[1]]
    (wa, wsa), (wb, wsb) = wide(qa, sa), wide(qb, sb)
    got = apoe.scaled_scores(wa, wsa, wb, wsb)
    check_scores(got, qa, sa, qb, sb)
    assert torch.equal(got, apoe.scaled_scores(qa, sa, qb, sb))


# ---- softmax loss ---------------------------------------------------------------------------------------------------------
def loss_case(rows, docs, dim, dtype, seed, scale=20.0, pad=True):
    g = gen(seed)
    d = torch.randn(docs, dim, generator=g, device=DEV)
    d = d / d.norm(dim=1, keepdim=True)
    t = torch.randint(0, docs, (rows,), generator=g, device=DEV)
    q = torch.randn(rows, dim, generator=g, device=DEV)
    q = q / q.norm(dim=1, keepdim=True) + 0.4 * d[t]
    t = t.to(torch.int32)
    if pad and rows > 2:
        t[rows // 2] = -1
        t[-1] = -1
    return q.to(dtype), d.to(dtype), t, scale


def plain_loss(q, d, t, scale, grad=None):
    """64 bits, from the definition; rows without a target are left out."""
    q, d, scale = q.double(), d.double(), float(np.float32(scale))
    kept = t >= 0
    y = t.long().clamp(min=0)
    l = scale * (q @ d.t())
    l = torch.where(kept[:, None], l, torch.zeros_like(l))
    lse = torch.logsumexp(l, 1)
    loss = lse - l.gather(1, y[:, None])[:, 0]
    out = [torch.where(kept, loss, 0.0), torch.where(kept, lse, 0.0)]
    if grad is not None:
        p = torch.exp(l - lse[:, None])
        p.scatter_add_(1, y[:, None], torch.full_like(lse, -1.0)[:, None])
        p *= torch.where(kept, grad.double(), 0.0)[:, None]
        q = torch.where(kept[:, None], q, torch.zeros_like(q))
        out += [scale * (p @ d), scale * (p.t() @ q)]
        out.append(p)
    return out


def logit_bound(q, d, scale):
    """Largest error of a logit: the fp32 sum of dim exact products, the scaling, the exponent's argument."""
    most = float((q.double().abs() @ d.double().abs().t()).amax()) * abs(scale)
    return most * (q.shape[1] * 2.0 ** -23 + 4 * 2.0 ** -24)


LOSS_SIZES = [(1, 1, 8), (1, 2, 64), (2, 300, 72), (32, 256, 1024), (128, 257, 136), (129, 1000, 1024), (300, 513, 776), (513, 5000, 200),
              (1000, 3001, 64)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,docs,dim", LOSS_SIZES)
def test_loss_equals_the_definition(rows, docs, dim, dtype):
    q, d, t, scale = loss_case(rows, docs, dim, dtype, rows + docs)
    loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
    want_loss, want_lse = plain_loss(q, d, t, scale)
    tol = 2 * logit_bound(q, d, scale) + 1e-6            # a shift of every logit by at most that; exp2, log2 and sums below 1e-6
    assert float((loss.double() - want_loss).abs().max()) <= tol
    assert float((lse.double() - want_lse).abs().max()) <= tol + 2.0 ** -22 * float(want_lse.abs().max())
    assert bool((loss[t < 0] == 0).all()) and bool((lse[t < 0] == 0).all())
    apoe.dense_check_status()


@pytest.mark.parametrize("scale", [0.0, -3.0, 1e-6, 400.0])
def test_loss_and_gradients_at_other_scales(scale):
    q, d, t, _ = loss_case(150, 333, 64, torch.float16, 61)
    grad = torch.full((150,), 0.25, device=DEV)
    loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
    want_loss, want_lse = plain_loss(q, d, t, scale)
    tol = 2 * logit_bound(q, d, scale) + 2e-6
    assert float((loss.double() - want_loss).abs().max()) <= tol + 2.0 ** -22 * float(want_loss.abs().max())
    assert float((lse.double() - want_lse).abs().max()) <= tol + 2.0 ** -22 * float(want_lse.abs().max())
    dq, dd = apoe.softmax_loss_backward(q, d, t, loss, lse, grad, scale)
    check_grads(q, d, t, scale, grad, loss, lse, dq, dd)


def check_grads(q, d, t, scale, grad, loss, lse, dq, dd):
    """An element of a gradient is a sum of g * v: each G is rounded to 16 bits once (u) and its exponential is off by the
    logit's error; the sum over N terms in fp32; the result is rounded once.  Rows' own |G| |v| sums bound all of it."""
    _, _, want_q, want_d, p = plain_loss(q, d, t, scale, grad)
    u, eps = U[q.dtype], 2 * logit_bound(q, d, scale) + 2e-6
    kept = (t >= 0)[:, None]
    qz = torch.where(kept, q.double(), torch.zeros_like(q.double()))
    floor = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    for got, want, mass, n in ((dq, want_q, scale * (p.abs() @ d.double().abs()), d.shape[0]), (dd, want_d, scale * (p.abs().t() @ qz.abs()), q.shape[0])):
        err = (got.double() - want).abs()
        tol = abs(mass) * (u + eps + n * 2.0 ** -23) + u * (want.abs() + abs(mass) * u) + floor
        # f16: G is held with its largest possible value at 2^14 (exact power of two): below 2^-14 it steps by 2^-24
        if q.dtype == torch.float16:
            top = float(grad.abs().max())
            other = d if got is dq else qz
            tol = tol + abs(scale) * top * 2.0 ** (-25 - 13) * other.double().abs().sum(0, keepdim=True)
        assert bool((err <= tol).all()), float((err / tol.clamp(min=1e-300)).max())
        # on the whole: a few roundings of u each; f16 results below 2^-14 are rounded to steps of 2^-24, off by at most `floor`
        assert float(err.square().mean().sqrt()) <= 4 * u * float(want.square().mean().sqrt()) + floor
    assert bool((dq[t < 0] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,docs,dim", [s for s in LOSS_SIZES if s[1] > 1])
def test_gradients_equal_the_definition(rows, docs, dim, dtype):
    q, d, t, scale = loss_case(rows, docs, dim, dtype, 3 * rows + docs)
    grad = (torch.rand(rows, generator=gen(5), device=DEV) + 0.5) * (64.0 if dtype == torch.float16 else 1.0) / rows
    loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
    dq, dd = apoe.softmax_loss_backward(q, d, t, loss, lse, grad, scale)
    apoe.dense_check_status()
    check_grads(q, d, t, scale, grad, loss, lse, dq, dd)


def test_gradient_agrees_with_differences():
    """The loss moved along a direction, in 64-bit arithmetic of the forward operator's own outputs: (f(x + h) - f(x - h)) / 2h
    with steps that are exact in f16.  The difference's own error (f''' h^2 and 2^-22 |loss| / h) is counted."""
    rows, docs, dim, scale = 64, 500, 128, 4.0
    q, d, t, _ = loss_case(rows, docs, dim, torch.float16, 77)
    q = (q.float() * 256).round().div(256).half()                     # steps of 1/256: x +- h stays exact
    grad = torch.full((rows,), 1.0, device=DEV)
    loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
    dq, dd = apoe.softmax_loss_backward(q, d, t, loss, lse, grad, scale)
    h = 1.0 / 64
    g = gen(6)
    way = torch.randint(0, 2, q.shape, generator=g, device=DEV).half() * 2 - 1
    up, down = (apoe.softmax_loss_forward(q + s * h * way, d, t, scale)[0].double() for s in (1, -1))
    want = (up - down) / (2 * h)
    got = (dq.double() * way.double()).sum(1)
    # along +-1 directions a logit moves by scale * h * |sum d| : third-order term of log-sum-exp below (that)^3 / h
    move = scale * h * float((d.double() @ way.double().t()).abs().max())
    noise = 2.0 ** -20 * float(lse.abs().max()) / h
    assert float((got - want).abs().max()) <= move ** 3 / h + noise + dim ** 0.5 * 2.0 ** -10 * float(dq.double().abs().max()) * 4
    assert float(want.abs().max()) > 10 * noise


def test_rows_without_a_target_may_hold_anything():
    q, d, t, scale = loss_case(200, 700, 256, torch.bfloat16, 8)
    t[10:20] = -1
    loss0, lse0 = apoe.softmax_loss_forward(q, d, t, scale)
    grad = torch.full((200,), 1 / 200, device=DEV)
    dq0, dd0 = apoe.softmax_loss_backward(q, d, t, loss0, lse0, grad, scale)
    q2, grad2 = q.clone(), grad.clone()
    q2[10:15] = float("nan")
    q2[15:20] = float("inf")
    grad2[12] = float("nan")
    grad2[13] = 1e30
    loss, lse = apoe.softmax_loss_forward(q2, d, t, scale)
    dq, dd = apoe.softmax_loss_backward(q2, d, t, loss, lse, grad2, scale)
    for a, b in ((loss, loss0), (lse, lse0), (dq, dq0), (dd, dd0)):
        assert torch.equal(a, b)
    t[:] = -1                                                          # no row left at all
    loss, lse = apoe.softmax_loss_forward(q2, d, t, scale)
    dq, dd = apoe.softmax_loss_backward(q2, d, t, loss, lse, grad2, scale)
    for a in (loss, lse, dq, dd):
        assert bool((a == 0).all())


@pytest.mark.parametrize("rows,docs,dim", [(5, 70, 3), (40, 301, 101), (200, 300, 70), (300, 1029, 131)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_loss_ignores_what_lies_behind_a_row(rows, docs, dim, dtype):
    """Row lengths that are no multiple of 16 bytes, in rows that are further apart, NaN between them."""
    q, d, t, scale = loss_case(rows, docs, dim, dtype, 15)
    wq = torch.full((rows, 136), float("nan"), dtype=dtype, device=DEV)
    wd = torch.full((docs, 144), float("nan"), dtype=dtype, device=DEV)
    wq[:, :dim], wd[:, :dim] = q, d
    vq, vd = wq[:, :dim], wd[:, :dim]
    grad = torch.full((rows,), (64.0 if dtype == torch.float16 else 1.0) / rows, device=DEV)
    loss, lse = apoe.softmax_loss_forward(vq, vd, t, scale)
    want_loss, _ = plain_loss(q, d, t, scale)
    assert float((loss.double() - want_loss).abs().max()) <= 2 * logit_bound(q, d, scale) + 1e-6
    dq, dd = apoe.softmax_loss_backward(vq, vd, t, loss, lse, grad, scale)
    check_grads(q, d, t, scale, grad, loss, lse, dq, dd)
    # gradients into rows that are further apart: the values between them are left alone (aligned rows, and others)
    for pad, off in ((152, 0), (137 if dim < 137 else 145, 1)):
        gq = torch.full((rows, 152), 3.0, dtype=dtype, device=DEV)
        gd = torch.full((docs * pad + 8,), 3.0, dtype=dtype, device=DEV)[off:off + docs * pad].view(docs, pad)
        size = apoe._workspace_bytes(0, rows, docs, dim, 1)
        ws = torch.empty(size, dtype=torch.uint8, device=DEV)
        apoe._check(apoe.lib().ap_softmax_loss_backward_device(
            0, rows, docs, dim, {torch.float16: 1, torch.bfloat16: 2}[dtype], vq.data_ptr(), 136, vd.data_ptr(), 144, t.data_ptr(), scale, loss.data_ptr(), lse.data_ptr(),
            grad.data_ptr(), gq.data_ptr(), 152, gd.data_ptr(), pad, ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(gq[:, :dim], dq) and torch.equal(gd[:, :dim], dd)
        assert bool((gq[:, dim:] == 3.0).all()) and bool((gd[:, dim:] == 3.0).all())


def test_gradients_scale_with_the_losses_gradient():
    """Times a power of two the same bits (bf16 has f32's range); extreme sizes of it neither overflow nor vanish on the way."""
    q, d, t, scale = loss_case(140, 400, 64, torch.bfloat16, 17)
    grad = torch.rand(140, generator=gen(18), device=DEV) + 0.5
    loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
    dq, dd = apoe.softmax_loss_backward(q, d, t, loss, lse, grad, scale)
    for k in (-90, -20, 3, 100):
        gq, gd = apoe.softmax_loss_backward(q, d, t, loss, lse, grad * 2.0 ** k, scale)
        assert torch.equal(gq.double(), dq.double() * 2.0 ** k) and torch.equal(gd.double(), dd.double() * 2.0 ** k)
    gq, gd = apoe.softmax_loss_backward(q, d, t, loss, lse, torch.zeros_like(grad), scale)
    assert not gq.any() and not gd.any()
    h, e = q.half(), d.half()
    loss, lse = apoe.softmax_loss_forward(h, e, t, scale)
    big = grad * 2e38                                     # below 3e38
    gq, _ = apoe.softmax_loss_backward(h, e, t, loss, lse, big, 1e-36)     # f16 results of ordinary size from gradients near 3e38
    assert bool(torch.isfinite(gq).all()) and bool((gq[t >= 0] != 0).any())


def test_nearly_certain_batches_keep_their_gradients_digits():
    """A batch whose every row is certain (losses near 1e-9): its small G are held as exactly as large ones, so the f16 gradients,
    brought back to ordinary size by the losses' gradient, are off by roundings only."""
    dim, docs = 128, 40
    g = gen(23)
    d = torch.randn(docs, dim, generator=g, device=DEV)
    d = (d / d.norm(dim=1, keepdim=True)).half()
    t = torch.arange(docs, device=DEV, dtype=torch.int32)
    q, scale = d.clone(), 36.0
    loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
    assert float(loss.max()) < 1e-5
    l = float(np.float32(scale)) * (q.double() @ d.double().t())
    p = torch.softmax(l, 1)
    away = torch.logsumexp(l.scatter(1, t.long()[:, None], -torch.inf), 1) - l.gather(1, t.long()[:, None])[:, 0]
    p = p.scatter(1, t.long()[:, None], -torch.sigmoid(away)[:, None])
    grad = (1.0 / loss.double()).float()                  # every row's coefficient near 1
    dq, dd = apoe.softmax_loss_backward(q, d, t, loss, lse, grad, scale)
    p = p * grad.double()[:, None]
    eps = 4 * logit_bound(q, d, scale) + 4e-6             # exponentials: both logits and lse; the coefficient's loss likewise
    for got, want, mass in ((dq, scale * (p @ d.double()), scale * (p.abs() @ d.double().abs())),
                            (dd, scale * (p.t() @ q.double()), scale * (p.abs().t() @ q.double().abs()))):
        u = U[torch.float16]
        # G itself is rounded relative to the largest one of the batch: 2^-24 of 2^14 at the least
        low = scale * 2.0 ** -38 * float(p.abs().max()) * docs
        assert bool(((got.double() - want).abs() <= mass * (u + eps) + u * want.abs() + low + 2.0 ** -25).all())


def test_single_rows_of_any_length():
    g = gen(19)
    for dim in (1, 7, 100, 333):
        x = torch.randn(1, dim, generator=g, device=DEV)
        q, s = apoe.quantize_rows(x)
        check_scores(apoe.scaled_scores(q, s, q, s), q, s, q, s)
        h = x.half()
        t = torch.zeros(1, dtype=torch.int32, device=DEV)
        loss, lse = apoe.softmax_loss_forward(h, h, t, 0.5)
        assert float(loss) == 0.0 and abs(float(lse) - 0.5 * float((h.double() ** 2).sum())) < 1e-4 * float((h.double() ** 2).sum())
        dq, dd = apoe.softmax_loss_backward(h, h, t, loss, lse, torch.ones(1, device=DEV), 0.5)
        assert not dq.any() and not dd.any()


def test_targets_out_of_range_show_and_give_no_gradient():
    q, d, t, scale = loss_case(40, 300, 64, torch.float16, 12, pad=False)
    grad = torch.full((40,), 0.1, device=DEV)
    t2 = t.clone()
    t2[3], t2[7] = 300, -2
    loss, lse = apoe.softmax_loss_forward(q, d, t2, scale)
    assert torch.equal(torch.isnan(loss).nonzero()[:, 0].cpu(), torch.tensor([3, 7])) and torch.equal(torch.isnan(lse), torch.isnan(loss))
    dq, dd = apoe.softmax_loss_backward(q, d, t2, loss, lse, grad, scale)
    t3 = t2.clone()
    t3[3], t3[7] = -1, -1
    loss3, lse3 = apoe.softmax_loss_forward(q, d, t3, scale)
    dq3, dd3 = apoe.softmax_loss_backward(q, d, t3, loss3, lse3, grad, scale)
    assert torch.equal(dq, dq3) and torch.equal(dd, dd3)


def test_certain_and_hopeless_rows_keep_their_digits():
    """Losses from 1e-12 to 100: where the target's logit leads, the loss is the others' weight and must keep its digits."""
    dim, docs = 64, 300
    g = gen(13)
    d = torch.randn(docs, dim, generator=g, device=DEV)
    d = d / d.norm(dim=1, keepdim=True)
    t = torch.arange(64, device=DEV, dtype=torch.int32)
    q = torch.cat([d[:32], -d[32:64]])
    q, d, scale = q.half(), d.half(), 50.0
    loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
    l = scale * (q.double() @ d.double().t())
    at = l.gather(1, t.long()[:, None])
    others = torch.logsumexp(l.scatter(1, t.long()[:, None], -torch.inf), 1)
    want = torch.nn.functional.softplus(others - at[:, 0], threshold=80.0)
    assert float(want.min()) < 1e-9 and float(want.max()) > 50
    # relative: the weight is e^(difference of logits), each logit off by at most logit_bound
    assert float(((loss.double() - want).abs() / want).max()) <= 2 * logit_bound(q, d, scale) + 2e-5
    grad = torch.full((64,), 1.0, device=DEV)
    dq, dd = apoe.softmax_loss_backward(q, d, t, loss, lse, grad, scale)
    # rows as certain as these: their gradient is their loss times vectors; f16 holds it with its scale of 2^14 over |grad|
    p = torch.softmax(l, 1).scatter(1, t.long()[:, None], 0.0)
    p = p.scatter(1, t.long()[:, None], -torch.expm1(-want)[:, None] * -1.0 * -1.0 * -1.0)
    assert float((dq.double() - scale * (p @ d.double())).abs().max()) <= 0.02 * float(dq.abs().max())


@pytest.mark.parametrize("rows,docs", [(8192, 9000), (65000, 8461), (40001, 20011)])
def test_pieces_of_the_documents_join(rows, docs):
    """More rows than one piece of the workspaces covers (from 40 000 rows on): several pieces forward and back, the last one
    short."""
    dim = 64
    q, d, t, scale = loss_case(rows, docs, dim, torch.bfloat16, 21)
    grad = torch.full((rows,), 1.0 / rows, device=DEV)
    loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
    dq, dd = apoe.softmax_loss_backward(q, d, t, loss, lse, grad, scale)
    want_loss, want_lse = plain_loss(q, d, t, scale)
    assert float((loss.double() - want_loss).abs().max()) <= 2 * logit_bound(q, d, scale) + 1e-6
    check_grads(q, d, t, scale, grad, loss, lse, dq, dd)


@pytest.mark.parametrize("rows,docs,dim", [(12, 71344, 144), (4, 55990, 200), (150, 60000, 72), (40, 30000, 328)])
def test_ragged_columns_over_many_tiles(rows, docs, dim):
    """Many tiles per SM whose last columns are written element by element while the others' copies are still on their way:
    every document's gradient, several times over, and the same bits each time."""
    q, d, t, scale = loss_case(rows, docs, dim, torch.bfloat16, 71)
    grad = torch.full((rows,), 1.0 / rows, device=DEV)
    loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
    first = apoe.softmax_loss_backward(q, d, t, loss, lse, grad, scale)
    check_grads(q, d, t, scale, grad, loss, lse, *first)
    for _ in range(8):
        again = apoe.softmax_loss_backward(q, d, t, loss, lse, grad, scale)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", [(30000, 200), (60000, 45), (20000, 233)])
def test_ragged_scores_over_many_tiles(m, n, dtype):
    g = gen(72)
    qa, sa = apoe.quantize_rows(torch.randn(m, 64, generator=g, device=DEV))
    qb, sb = apoe.quantize_rows(torch.randn(n, 64, generator=g, device=DEV))
    first = apoe.scaled_scores(qa, sa, qb, sb, out_dtype=dtype)
    check_scores(first, qa, sa, qb, sb)
    for _ in range(8):
        assert torch.equal(apoe.scaled_scores(qa, sa, qb, sb, out_dtype=dtype), first)


def test_offsets_beyond_32_bits():
    """More than 2^32 values on a side: the rows at the end are as right as those at the start."""
    g = gen(81)
    rows, dim = 4_200_000, 1024                                        # 4.3e9 values of f16
    x = torch.empty(rows, dim, dtype=torch.float16, device=DEV)
    x[:1000] = torch.randn(1000, dim, generator=g, device=DEV).half()
    x[1000:-1000] = 0.5
    x[-1000:] = torch.randn(1000, dim, generator=g, device=DEV).half()
    q, s = apoe.quantize_rows(x)
    for part in (slice(0, 50), slice(rows - 50, rows)):
        want_q, want_s = plain_quantize(x[part])
        assert torch.equal(q[part].cpu().double(), want_q) and torch.equal(s[part].cpu().long(), want_s)
    few_q, few_s = q[-40:].clone(), s[-40:].clone()
    out = apoe.scaled_scores(few_q, few_s, q, s, out_dtype=torch.float16)
    check_scores(out[:, -500:], few_q, few_s, q[-500:], s[-500:])
    del out
    # the loss over these documents: the targets at the end, the gradient of the last rows
    t = torch.arange(rows - 3, rows, device=DEV, dtype=torch.int32)
    few = x[-3:].clone()
    x[1000:-1000] *= 0.125
    loss, lse = apoe.softmax_loss_forward(few, x, t, 0.01)
    l = 0.01 * torch.cat([few.double() @ x[a:a + 400000].double().t() for a in range(0, rows, 400000)], 1)
    want_lse = torch.logsumexp(l, 1)
    bound = 2 * float(l.abs().max()) * (dim + 4) * 2.0 ** -23
    assert float((lse.double() - want_lse).abs().max()) <= bound + 2.0 ** -20 * float(want_lse.abs().max())
    grad = torch.full((3,), 1000.0, device=DEV)
    _, dd = apoe.softmax_loss_backward(few, x, t, loss, lse, grad, 0.01)
    p = torch.exp(l[:, -3:] - want_lse[:, None])
    p -= torch.eye(3, device=DEV, dtype=torch.float64)
    want = 10.0 * (p.t() @ few.double())                                # 0.01 * 1000
    assert float((dd[-3:].double() - want).abs().max()) <= (3 * 2.0 ** -11 + 2 * bound + 1e-5) * 10.0 * float((p.abs().t() @ few.double().abs()).max())
    del q, s, x, dd, l
    # results beyond 2^32 values, on and off 16-byte rows
    a, sa = apoe.quantize_rows(torch.randn(66000, 64, generator=g, device=DEV))
    for n, ld in ((66000, 66000), (66000, 66001)):
        room = torch.empty(66000, ld, dtype=torch.bfloat16, device=DEV)
        apoe.scaled_scores(a, sa, a[:n], sa[:n], out=room[:, :n])
        check_scores(room[-100:, n - 300:n], a[-100:], sa[-100:], a[n - 300:n], sa[n - 300:n])
        check_scores(room[:100, :300], a[:100], sa[:100], a[:300], sa[:300])
        del room


def test_same_call_same_bits_on_any_stream():
    q, d, t, scale = loss_case(700, 3000, 256, torch.bfloat16, 31)
    grad = torch.full((700,), 1 / 700, device=DEV)
    def once():
        loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
        return (loss, lse, *apoe.softmax_loss_backward(q, d, t, loss, lse, grad, scale), *apoe.quantize_rows(q))
    first = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    runs = []
    for s in streams:                                     # calls that overlap, each with its own workspace
        with torch.cuda.stream(s):
            runs.append([once() for _ in range(3)])
    torch.cuda.synchronize()
    for r in runs:
        for out in r:
            assert all(torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a, b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)
                       for a, b in zip(out, first))


def test_calls_are_captured_and_replayed():
    q, d, t, scale = loss_case(260, 1000, 128, torch.float16, 41)
    grad = torch.full((260,), 0.5, device=DEV)
    def step():
        loss, lse = apoe.softmax_loss_forward(q, d, t, scale)
        dq, dd = apoe.softmax_loss_backward(q, d, t, loss, lse, grad, scale)
        q8, sq = apoe.quantize_rows(q)
        d8, sd = apoe.quantize_rows(d)
        return loss, lse, dq, dd, apoe.scaled_scores(q8, sq, d8, sd)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    q2, d2, t2, _ = loss_case(260, 1000, 128, torch.float16, 42)
    q.copy_(q2), d.copy_(d2), t.copy_(t2)                 # new contents, same buffers
    graph.replay()
    torch.cuda.synchronize()
    got = [x.clone() for x in held]
    graph.replay()
    torch.cuda.synchronize()
    want = step()
    for a, b, c in zip(got, held, want):
        assert torch.equal(a, c) and torch.equal(b, c)
    apoe.dense_check_status()


def test_a_wait_that_runs_out_is_reported_once():
    """The error path of the bounded waits, without a fault: a kernel whose wait nothing ends gives up and returns."""
    stream = torch.cuda.current_stream().cuda_stream
    apoe._check(apoe.lib().ap_debug_dense_wait_timeout(0, 64, apoe.C.c_void_p(stream)))
    with pytest.raises(apoe.ApoeError) as e:
        apoe.dense_check_status()
    assert e.value.code == 6 and "error word" in str(e.value)
    apoe.dense_check_status()
    q, s = apoe.quantize_rows(torch.ones(3, 128, device=DEV))          # the context stays usable
    check_scores(apoe.scaled_scores(q, s, q, s), q, s, q, s)


def test_train_pack_and_score_together():
    """The operators as they are used in a row: some steps of descent on the document and query vectors, the vectors packed to
    8 bits, the packed scores close to those of the vectors: each value is off by at most 2^-4 of itself (e4m3)."""
    rows, docs, dim, scale = 256, 2000, 256, 20.0
    q, d, t, _ = loss_case(rows, docs, dim, torch.bfloat16, 51, pad=False)
    q, d = q.float(), d.float()
    grad = torch.full((rows,), 1.0 / rows, device=DEV)
    for _ in range(3):
        qh, dh = q.bfloat16(), d.bfloat16()
        loss, lse = apoe.softmax_loss_forward(qh, dh, t, scale)
        dq, dd = apoe.softmax_loss_backward(qh, dh, t, loss, lse, grad, scale)
        check_grads(qh, dh, t, scale, grad, loss, lse, dq, dd)
        q -= 0.5 * dq.float()
        d -= 0.5 * dd.float()
    q8, sq = apoe.quantize_rows(q)
    d8, sd = apoe.quantize_rows(d)
    got = apoe.scaled_scores(q8, sq, d8, sd).double()
    want = q.double() @ d.double().t()
    # |a8 b8 - a b| <= (2 * 2^-4 + 2^-8) |a b| + 2^-10 of a block's scale for values below e4m3's normal range
    bound = (2 * 2.0 ** -4 + 2.0 ** -8) * (q.double().abs() @ d.double().abs().t())
    bound += 2.0 ** -10 * (values(torch.ones_like(q8, dtype=torch.float32), sq).abs() @ d.double().abs().t()
                           + q.double().abs() @ values(torch.ones_like(d8, dtype=torch.float32), sd).abs().t()) * 1.1
    assert bool(((got - want).abs() <= bound).all())
