"""Dropout, residual + RMS norm (16 and 8 bit) and the e4m3 projection against 64-bit restatements.

Tolerances count roundings.  ``HALF[t]`` is half a step of a type relative to the value.  A result that is computed in
fp32 and rounded once is off by at most HALF times its value plus the fp32 arithmetic's error, taken as ``F32`` = 2^-18
(64 roundings of 2^-24) times the sum of the magnitudes it was formed from: the longest chain, a row's sum, is a tree
over threads on top of at most ~32 sequential additions a thread.  ``TINY`` absorbs results below the smallest normal.
"""

import pytest
import torch

from oracle import rows as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF = {t: torch.finfo(t).eps / 2 for t in DTYPES}
TINY = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24, torch.float32: 2.0**-126}
F32 = 2.0**-18
EPS = 1e-5


@pytest.fixture(scope="module")
def ck():
    import coda_kernels_b200 as ck

    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return ck


def randn(*shape, dtype=torch.bfloat16, seed=0, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype).to(DEV)


def rng_state(seed=1234567890123, step=7):
    return torch.tensor([seed, step], dtype=torch.int64, device=DEV)


def within(got, want, bound, what):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst error {float(err[bad].max()):.3e}, "
        f"bound there {float((bound + 0 * err)[bad].max()):.3e}")


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,p", [((1,), 0.5), ((1, 1), 0.5), ((3, 5), 0.25), ((7, 4), 0.1), ((5, 1023), 0.5), ((33, 512), 0.999),
                                     ((2, 3, 40), 0.1), ((64, 4096), 0.1), ((4, 20001), 0.3)])
def test_dropout_matches_the_generator(ck, dtype, shape, p):
    x = randn(*shape, dtype=dtype).requires_grad_(True)
    rng = rng_state()
    out = ck.dropout(x, p, rng, stream=3)
    rng[1] += 1  # the program moves on before the backward
    dout = randn(*shape, dtype=dtype, seed=1)
    (dx,) = torch.autograd.grad(out, x, dout)
    cols = shape[-1]
    keep = ref.keep_mask(x.numel() // cols, cols, p, 1234567890123, 7, 3).reshape(shape).to(DEV)
    assert out.dtype == dtype and out.shape == x.shape
    for got, src in ((out, x), (dx, dout)):
        want = ref.dropped(src.detach().double(), keep, p)
        within(got.detach(), want, want.abs() * (HALF[dtype] + 2.0**-22) + TINY[dtype], "dropout")
        assert not bool(got[~keep].any()), "a dropped element is zero"


def test_dropout_state_words(ck):
    """Every part of the state changes the mask; step counts modulo 2^32; a negative seed is its 64 bits."""
    x = torch.ones(16, 256, device=DEV)
    base = ck.dropout(x, 0.5, rng_state(5, 1), stream=0)
    assert torch.equal(base, ck.dropout(x, 0.5, rng_state(5, 1 + 2**32), stream=0))
    for other in (ck.dropout(x, 0.5, rng_state(6, 1)), ck.dropout(x, 0.5, rng_state(5 + 2**32, 1)), ck.dropout(x, 0.5, rng_state(5, 2)),
                  ck.dropout(x, 0.5, rng_state(5, 1), stream=1)):
        assert 0.35 < float((other != base).float().mean()) < 0.65
    got = ck.dropout(x, 0.5, rng_state(-3, -1), stream=2**32 - 1) != 0
    assert torch.equal(got.cpu(), ref.keep_mask(16, 256, 0.5, -3 % 2**64, -1, 2**32 - 1))


def test_dropout_edges(ck):
    x = randn(8, 100)
    assert torch.equal(ck.dropout(x, 0.0), x)
    assert ck.dropout(x[:0], 0.5, rng_state()).shape == (0, 100)
    bad = torch.full((64, 64), float("nan"), device=DEV)
    bad[:, ::2] = float("inf")
    out = ck.dropout(bad, 0.5, rng_state())
    keep = ref.keep_mask(64, 64, 0.5, 1234567890123, 7, 0).to(DEV)
    assert bool((out[~keep] == 0).all()) and not bool(torch.isfinite(out[keep]).any())
    # strided and misaligned inputs give what their dense copies give
    wide = randn(32, 129)
    for view in (wide[:, 1:], wide.t(), wide.reshape(-1)[1:4097].view(64, 64)):
        assert torch.equal(ck.dropout(view, 0.3, rng_state()), ck.dropout(view.clone(memory_format=torch.contiguous_format), 0.3, rng_state()))


def test_dropout_beyond_31_bits(ck):
    cols = 4096
    rows = 2**31 // cols + 5
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device=DEV)
    out = ck.dropout(x, 0.5, rng_state())
    keep = ref.keep_mask(7, cols, 0.5, 1234567890123, 7, 0, first_row=rows - 7)
    assert torch.equal(out[-7:].cpu() == 2.0, keep) and torch.equal(out[-7:].cpu() == 0.0, ~keep)


# ------------------------------------------------------------------------------------------------ norm
def norm_case(ck, dtype, rows, cols, p, residual=True, seed=0):
    x = randn(rows, cols, dtype=dtype, seed=seed).requires_grad_(True)
    res = randn(rows, cols, dtype=dtype, seed=seed + 1).requires_grad_(True) if residual else None
    w = randn(cols, dtype=dtype, seed=seed + 2, std=0.2, mean=1.0).requires_grad_(True)
    dout, dh = randn(rows, cols, dtype=dtype, seed=seed + 3), randn(rows, cols, dtype=dtype, seed=seed + 4)
    if residual:
        out, h = ck.add_rms_norm(x, res, w, EPS, p=p, rng=rng_state() if p else None, stream=5)
        dx, dres, dw = torch.autograd.grad((out, h), (x, res, w), (dout, dh))
    else:
        out, h, dh, dres = ck.rms_norm(x, w, EPS), None, None, None
        dx, dw = torch.autograd.grad(out, (x, w), dout)
    return x, res, w, dout, dh, out, h, dx, dres, dw


def check_norm(dtype, p, x, res, w, dout, dh, out, h, dx, dres, dw):
    u, tiny = HALF[dtype], TINY[dtype]
    rows, cols = x.shape
    x64, w64, do64 = x.detach().double(), w.detach().double(), dout.double()
    keep = ref.keep_mask(rows, cols, p, 1234567890123, 7, 5).to(DEV) if p else torch.ones_like(x64, dtype=torch.bool)
    parts = ref.dropped(x64, keep, p)
    h64 = parts if res is None else parts + res.detach().double()
    size = parts.abs() if res is None else parts.abs() + res.detach().double().abs()  # what h was formed from
    want, rstd = ref.norm(h64, w64, EPS)
    # an error of F32 * size in h is one of the same order in rstd (relative to the row's rms) and so in out
    slack = F32 * (rstd * w64.abs() * size + want.abs() * (1 + (rstd * size).square().mean(1, keepdim=True).sqrt()))
    within(out.detach(), want, u * want.abs() + slack + tiny, "out")
    if h is not None:
        within(h.detach(), h64, u * h64.abs() + F32 * size + tiny, "h")
    wres, wdw = ref.norm_backward(do64, None if dh is None else dh.double(), h64, rstd, w64)
    # the backward reads the stored h, half a step off: xh moves by up to u |xh|, the row's mean product by u mean|g xh|
    # (fp32 errors count against xs, what h was formed from: x / (1 - p) is rounded before the residual cancels it, so the
    # error of h is up to 2^-23 of |x / (1 - p)| + |residual| however small h comes out)
    g, xh, xs = (do64 * w64).abs(), (h64 * rstd).abs(), size * rstd
    gx = (g * xh).mean(1, keepdim=True)
    uh = u + F32 * (1 + (rstd * size).square().mean(1, keepdim=True).sqrt())
    moved = rstd * xh * gx * 2 * uh
    formed = (0 if dh is None else dh.double().abs()) + rstd * (g + xs * (g * xs).mean(1, keepdim=True))
    bound = u * wres.abs() + moved + F32 * formed + tiny
    if res is None:
        within(dx, wres, bound, "dx")
    else:
        within(dres, wres, bound, "dresidual")
        within(dx, ref.dropped(wres, keep, p), keep * (bound / (1 - p)) + tiny, "dx")
        assert not bool(dx[~keep].any())
    terms = (do64.abs() * xh)
    within(dw, wdw, u * wdw.abs() + (terms * uh).sum(0) + F32 * (do64.abs() * xs).sum(0) + tiny, "dweight")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,p", [(1, 1, 0.0), (1, 4096, 0.1), (2, 7, 0.5), (33, 64, 0.1), (5, 1000, 0.0), (130, 1531, 0.25),
                                         (1200, 128, 0.1), (700, 2056, 0.0), (9, 8192, 0.1), (3, 20004, 0.1), (2, 33001, 0.0), (30001, 50, 0.1), (2051, 121, 0.2), (10007, 3, 0.5)])
def test_add_rms_norm(ck, dtype, rows, cols, p):
    check_norm(dtype, p, *norm_case(ck, dtype, rows, cols, p))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 8), (65, 513), (300, 4096), (4, 16384), (2, 40000), (2, 60001), (2000, 257), (3000, 250), (4099, 65), (20000, 64), (777, 128), (5003, 13), (700, 8190), (1300, 4095)])
def test_rms_norm(ck, dtype, rows, cols):
    check_norm(dtype, 0.0, *norm_case(ck, dtype, rows, cols, 0.0, residual=False))


def test_add_rms_norm_uses_the_mask_of_dropout(ck):
    x, res, w = randn(40, 260), randn(40, 260, seed=1), randn(260, seed=2)
    rng = rng_state()
    _, h = ck.add_rms_norm(x, torch.zeros_like(res), w, EPS, p=0.3, rng=rng, stream=9)
    assert torch.equal(h, ck.dropout(x, 0.3, rng, stream=9))


def test_norm_gradients_against_differences(ck):
    """Along a direction, (L(+e) - L(-e)) / 2e of the kernel's own fp32 forward.  L sums ~2 * 48 * 100 products of unit
    size: fp32 forward errors of 2^-22 of each leave ~sqrt(9600) * 2^-22 / e = 2.3e-3 at e = 1e-2, and the third-order
    term e^2 L''' / 6 is below 1e-4 of a derivative of order sqrt(9600) = 98."""
    rows, cols, e = 48, 100, 1e-2
    t = torch.float32
    x, res, w = randn(rows, cols, dtype=t), randn(rows, cols, dtype=t, seed=1), randn(cols, dtype=t, seed=2, mean=1.0, std=0.2)
    dout, dh = randn(rows, cols, dtype=t, seed=3), randn(rows, cols, dtype=t, seed=4)
    rng = rng_state()

    def L(x, res, w):
        out, h = ck.add_rms_norm(x, res, w, EPS, p=0.2, rng=rng, stream=1)
        return out, h, float((out.detach().double() * dout).sum() + (h.detach().double() * dh).sum())

    leaves = [v.clone().requires_grad_(True) for v in (x, res, w)]
    out, h, _ = L(*leaves)
    grads = torch.autograd.grad((out, h), leaves, (dout, dh))
    for i, grad in enumerate(grads):
        v = randn(*grad.shape, dtype=t, seed=20 + i)
        args = [x, res, w]
        plus, minus = list(args), list(args)
        plus[i], minus[i] = args[i] + e * v, args[i] - e * v
        numeric = (L(*plus)[2] - L(*minus)[2]) / (2 * e)
        analytic = float((grad.double() * v).sum())
        assert abs(numeric - analytic) <= 0.02 + 2e-3 * 98, (i, numeric, analytic)


def test_norm_partial_gradients_and_repeatability(ck):
    x, res, w = randn(70, 264), randn(70, 264, seed=1), randn(264, seed=2)
    dout, dh = randn(70, 264, seed=3), randn(70, 264, seed=4)
    full = [v.clone().requires_grad_(True) for v in (x, res, w)]
    out, h = ck.add_rms_norm(*full, EPS, p=0.1, rng=rng_state())
    all_grads = torch.autograd.grad((out, h), full, (dout, dh))
    for i in range(3):
        args = [v.clone().requires_grad_(j == i) for j, v in enumerate((x, res, w))]
        o, hh = ck.add_rms_norm(*args, EPS, p=0.1, rng=rng_state())
        (g,) = torch.autograd.grad((o, hh), args[i], (dout, dh))
        assert torch.equal(g, all_grads[i])
    # only one of the two outputs used
    leaves = [v.clone().requires_grad_(True) for v in (x, res, w)]
    out, h = ck.add_rms_norm(*leaves, EPS)
    dx, dres, dw = torch.autograd.grad(h, leaves, dh, allow_unused=True, retain_graph=True)
    assert torch.equal(dx, dh) and torch.equal(dres, dh) and not bool(dw.any())
    a = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    b = torch.autograd.grad((out, h), leaves, (dout, torch.zeros_like(dh)))
    for u, v in zip(a, b):
        assert torch.equal(u, v)
    # distinct buffers: an in-place change of one gradient leaves the other alone
    assert a[0].data_ptr() != a[1].data_ptr()


def test_norm_empty_and_views(ck):
    w = randn(64, seed=2).requires_grad_(True)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    out, h = ck.add_rms_norm(x, torch.empty_like(x), w, EPS)
    dx, dw = torch.autograd.grad((out, h), (x, w), (torch.empty_like(out), torch.empty_like(h)))
    assert out.shape == dx.shape == (0, 64) and not bool(dw.any())
    big = randn(4, 10, 200)
    view = big[:, ::2, 1:130]
    dense = view.clone(memory_format=torch.contiguous_format)
    wv = randn(129, seed=3)
    assert torch.equal(ck.rms_norm(view, wv, EPS), ck.rms_norm(dense, wv, EPS))
    odd = randn(1 + 16 * 64)[1:].view(16, 64)  # dense, but only 2-byte aligned
    w64 = randn(1 + 64, seed=3)[1:]
    o1, h1 = ck.add_rms_norm(odd, odd, w64, EPS)
    o2, h2 = ck.add_rms_norm(odd.clone(), odd.clone(), w64.clone(), EPS)
    assert torch.equal(o1, o2) and torch.equal(h1, h2)


def test_norm_nonfinite_rows_stay_in_their_rows(ck):
    x, res, w = randn(6, 300), randn(6, 300, seed=1), randn(300, seed=2)
    x2 = x.clone()
    x2[1, 5], x2[3, 7] = float("nan"), float("inf")
    a, ha = ck.add_rms_norm(x, res, w, EPS)
    b, hb = ck.add_rms_norm(x2, res, w, EPS)
    rows = [0, 2, 4, 5]
    assert torch.equal(a[rows], b[rows]) and torch.equal(ha[rows], hb[rows])
    assert bool(b[1].isnan().all()) and bool(b[3, 7].isnan())


# ------------------------------------------------------------------------------------------------ e4m3 rows
def check_e4m3(q, scale, want):
    """The scale is the fp32 one; q is off by half a step (2^-4 of the value, or 2^-10 below 2^-6) of the scaled value."""
    ws = ref.row_scale(want)
    within(scale, ws, ws * F32, "scale")
    y = want / ws[..., None]
    within(q.float(), y, y.abs() * (2.0**-4 + 4 * F32) + 2.0**-10, "q")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 7), (64, 128), (37, 1531), (500, 2048), (2, 16384), (3, 20001), (9001, 64), (8191, 57), (3001, 100)])
def test_rows_in_e4m3(ck, dtype, rows, cols):
    x, res, w = randn(rows, cols, dtype=dtype), randn(rows, cols, dtype=dtype, seed=1), randn(cols, dtype=dtype, seed=2, mean=1.0, std=0.2)
    h64 = x.double() + res.double()
    q, scale, h = ck.add_rms_norm_e4m3(x, res, w, EPS)
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32 and scale.shape == (rows,)
    check_e4m3(q, scale, ref.norm(h64, w.double(), EPS)[0])
    within(h, h64, HALF[dtype] * h64.abs() + 2.0**-24 * h64.abs(), "h")
    check_e4m3(*ck.rms_norm_e4m3(x, w, EPS), ref.norm(x.double(), w.double(), EPS)[0])
    check_e4m3(*ck.quantize_e4m3(x), x.double())


@pytest.mark.parametrize("dtype", DTYPES)
def test_e4m3_ties_follow_the_rounded_quotient(ck, dtype):
    """Values of a 2-byte type lie on the middle between two e4m3 values all the time; they go to the even one, as the
    correctly rounded fp32 quotient does."""
    for i, top in enumerate((3.5, 2.625, 21.0, 1.0, 0.7, 5.25, 448.0, 1.3125 * 2.0**-20)):
        x = (randn(64, 2048, dtype=torch.float32, seed=i).clamp(-3.9, 3.9) / 4 * top).to(dtype)
        x[:, 5] = top
        q, scale = ck.quantize_e4m3(x)
        assert bool((scale == scale[0]).all())
        want = (x.float() / scale[:, None]).to(torch.float8_e4m3fn)
        assert torch.equal(q.float(), want.float()), top  # (a zero's sign is no value)


def test_e4m3_edges(ck):
    x = randn(8, 96, dtype=torch.float32)
    x[1] = 0.0
    x[2] *= 1e-37 * 448
    x[3] *= 1e37
    x[4, 9] = float("nan")
    x[5, 9] = float("inf")
    q, scale = ck.quantize_e4m3(x)
    fine = [0, 2, 3, 6, 7]
    check_e4m3(q[fine], scale[fine], x[fine].double())
    assert float(scale[1]) == 2.0**-126 and not bool(q[1].float().any())
    assert bool(scale[4].isnan()) and bool(q[4].float().isnan().all())
    assert float(scale[5]) == float("inf") and bool(q[5, 9].float().isnan()) and not bool(q[5, :9].float().any())
    q, scale, h = ck.add_rms_norm_e4m3(x[:0], x[:0], x[0], EPS)
    assert q.shape == (0, 96) and scale.shape == (0,) and h.shape == (0, 96)
    q, scale = ck.quantize_e4m3(randn(2, 3, 64))
    assert q.shape == (2, 3, 64) and scale.shape == (2, 3)
    zero, one = ck.rms_norm_e4m3(torch.zeros(2, 64, device=DEV), torch.ones(64, device=DEV), EPS)
    assert not bool(zero.float().any()) and float(one[0]) == 2.0**-126


# ------------------------------------------------------------------------------------------------ e4m3 projection
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 8, 16), (1, 4096, 1024), (2, 136, 48), (7, 64, 4096), (8, 1000, 528), (9, 1000, 528), (16, 264, 2064), (17, 512, 512), (32, 72, 1040), (20, 8200, 64), (33, 72, 64), (64, 520, 4096), (40, 6144, 2048), (65, 1032, 8208), (100, 24, 1040), (128, 20000, 512), (129, 512, 2048), (130, 264, 1552),
                                   (256, 256, 256), (333, 2056, 784), (1000, 520, 128)])
def test_linear_e4m3(ck, M, N, K, out_dtype):
    """e4m3 products are exact in fp32; accumulating K of them, 32 an instruction, is off by at most (K / 32 + 1) * 2^-22
    of the sum of their magnitudes (an addition each, and the sum inside an instruction, to 2^-22)."""
    x8, xs = ck.quantize_e4m3(randn(M, K))
    w8, ws = ck.quantize_e4m3(randn(N, K, seed=1, std=K**-0.5))
    out = ck.linear_e4m3(x8, xs, w8, ws, out_dtype)
    a, b = x8.double() * xs.double()[:, None], w8.double() * ws.double()[:, None]
    want, terms = a @ b.T, a.abs() @ b.abs().T
    assert out.dtype == out_dtype and out.shape == (M, N)
    within(out, want, HALF[out_dtype] * want.abs() + ((K / 32 + 1) * 2.0**-22 + 2.0**-22) * terms, "out")
    assert torch.equal(out, ck.linear_e4m3(x8, xs, w8, ws, out_dtype))
    ck.ops.check_device_status(torch.device(DEV))


def test_linear_e4m3_rows_are_independent(ck):
    """A NaN row stays in its row; an all-zero row gives zeros; no row at all gives an empty result."""
    x8, xs = ck.quantize_e4m3(torch.cat([randn(3, 64), torch.zeros(1, 64, dtype=torch.bfloat16, device=DEV), randn(1, 64) * float("nan")]))
    w8, ws = ck.quantize_e4m3(randn(16, 64, seed=1))
    out = ck.linear_e4m3(x8, xs, w8, ws)
    assert bool(out[4].isnan().all()) and not bool(out[3].any()) and bool(torch.isfinite(out[:4]).all())
    assert ck.linear_e4m3(x8[:0], xs[:0], w8, ws).shape == (0, 16)
    # scales and rows that start off a 16-byte boundary, and a strided weight
    odd_scale = torch.cat([ws[:1], ws])[1:]
    assert torch.equal(ck.linear_e4m3(x8[:3], xs[:3], w8, odd_scale), out[:3])
    wide = torch.empty(16, 128, dtype=torch.float8_e4m3fn, device=DEV)
    wide[:, ::2] = w8
    assert torch.equal(ck.linear_e4m3(x8[:3], xs[:3], wide[:, ::2], ws), out[:3])


# ------------------------------------------------------------------------------------------------ streams, graphs, refusals
def test_side_stream_and_graph_with_an_advancing_step(ck):
    x, res, w = randn(64, 512), randn(64, 512, seed=1), randn(512, seed=2)
    rng = rng_state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = ck.add_rms_norm(x, res, w, EPS, p=0.1, rng=rng)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(on_side, ck.add_rms_norm(x, res, w, EPS, p=0.1, rng=rng)):
        assert torch.equal(a, b)

    leaves = [t.clone().requires_grad_(True) for t in (x, res, w)]
    dout, dh = randn(64, 512, seed=3), randn(64, 512, seed=4)

    def step():
        out, h = ck.add_rms_norm(*leaves, EPS, p=0.1, rng=rng, stream=2)
        h2 = ck.dropout(h, 0.2, rng, stream=3)
        grads = torch.autograd.grad((out, h2), leaves, (dout, dh))
        return out.detach(), h2.detach(), *grads

    # (no eager graph of these leaves is kept alive: see the capture test of the cross entropy)
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
        rng[1] += 1
    rng.copy_(rng_state())
    for _ in range(3):
        before = rng.clone()
        graph.replay()
        torch.cuda.synchronize()
        now = rng.clone()
        rng.copy_(before)
        eager = step()
        rng.copy_(now)
        for a, b in zip(static, eager):
            assert torch.equal(a, b)
    assert int(rng[1]) == 10


def test_refusals(ck):
    x, w = randn(4, 64), randn(64)
    rng = rng_state()
    with pytest.raises(ValueError):
        ck.dropout(x, 1.0, rng)
    with pytest.raises(ValueError):
        ck.dropout(x, -0.1, rng)
    with pytest.raises(ValueError):
        ck.dropout(x, float("nan"), rng)
    with pytest.raises(ValueError, match="rng"):
        ck.dropout(x, 0.1)
    with pytest.raises(ValueError, match="rng"):
        ck.dropout(x, 0.1, rng.int())
    with pytest.raises(ValueError, match="rng"):
        ck.dropout(x, 0.1, rng.cpu())
    with pytest.raises(ValueError, match="stream"):
        ck.dropout(x, 0.1, rng, stream=2**32)
    with pytest.raises(NotImplementedError):
        ck.dropout(x.double(), 0.1, rng)
    with pytest.raises(ValueError):
        ck.dropout(torch.zeros((), device=DEV), 0.1, rng)
    with pytest.raises(ValueError, match="weight"):
        ck.rms_norm(x, w[:32], EPS)
    with pytest.raises(ValueError, match="weight"):
        ck.rms_norm(x, w.float(), EPS)
    with pytest.raises(ValueError, match="residual"):
        ck.add_rms_norm(x, x[:3], w, EPS)
    with pytest.raises(ValueError, match="residual"):
        ck.add_rms_norm(x, x.float(), w, EPS)
    leaf = x.clone().requires_grad_(True)
    for call in (lambda: ck.quantize_e4m3(leaf), lambda: ck.rms_norm_e4m3(leaf, w, EPS), lambda: ck.add_rms_norm_e4m3(x, leaf, w, EPS)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad():
            call()
    q, s = ck.quantize_e4m3(x)
    for bad in (lambda: ck.linear_e4m3(x, s, q, s), lambda: ck.linear_e4m3(q, s, x, s)):
        with pytest.raises(NotImplementedError):
            bad()
    w8, ws = ck.quantize_e4m3(randn(16, 64))
    for bad in (lambda: ck.linear_e4m3(q[:, :40], s, w8[:, :40], ws), lambda: ck.linear_e4m3(q, s[:2], w8, ws),
                lambda: ck.linear_e4m3(q, s, w8[:12], ws[:12]), lambda: ck.linear_e4m3(q, s, w8, ws.double()),
                lambda: ck.linear_e4m3(q, s, w8[:, :48], ws), lambda: ck.linear_e4m3(q, s, w8, ws, torch.float16)):
        with pytest.raises(ValueError):
            bad()


def test_row_operators_under_compile(ck):
    def f(x, res, w, rng):
        out, h = ck.add_rms_norm(x, res, w, EPS, p=0.1, rng=rng, stream=1)
        return ck.dropout(out, 0.2, rng, stream=2), h

    leaves = [t.requires_grad_(True) for t in (randn(40, 136), randn(40, 136, seed=1), randn(136, seed=2))]
    douts = randn(40, 136, seed=3), randn(40, 136, seed=4)
    rng = rng_state()
    eager = f(*leaves, rng)
    traced = torch.compile(f, fullgraph=True, dynamic=False)(*leaves, rng)
    for a, b in zip(eager, traced):
        assert torch.equal(a, b)
    for a, b in zip(torch.autograd.grad(eager, leaves, douts), torch.autograd.grad(traced, leaves, douts)):
        assert torch.equal(a, b)


def test_both_bindings_give_the_same_bits(ck):
    """The compiled operators and the Python nodes over the custom ops (what torch.compile traces)."""
    from importlib import import_module

    norm, drop, ce = (import_module(f"coda_kernels_b200.functional.{m}") for m in ("rms_norm", "dropout", "cross_entropy_pieces"))
    rows_ops = import_module("coda_kernels_b200.ops_rows")
    x, res, w = randn(50, 264), randn(50, 264, seed=1), randn(264, seed=2)
    dout, dh = randn(50, 264, seed=3), randn(50, 264, seed=4)

    def grads(outs, leaves, gs):
        outs = outs if isinstance(outs, tuple) else (outs,)
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, gs[: len(outs)]))

    for native, node, args, n in (
        (ck.add_rms_norm, norm.AddRMSNorm, (x, res, w, EPS, 0.1, rng_state(), 3), 3),
        (ck.rms_norm, norm.RMSNorm, (x, w, EPS), 2),
        (ck.dropout, drop.Dropout, (x, 0.4, rng_state(), 1), 1),
    ):
        results = []
        for fn in (native, node.apply):
            leaves = [a.clone().requires_grad_(True) for a in args[:n]]
            results.append(grads(fn(*leaves, *args[n:]), leaves, (dout, dh)))
        for a, b in zip(*results):
            assert torch.equal(a, b)
    t = torch.randint(0, 50, (50,), dtype=torch.int32, device=DEV)
    results = []
    for fn in (lambda a, b: ck.linear_cross_entropy_pieces(a, b, t, piece=24),
               lambda a, b: ce.LinearCrossEntropyPieces.apply(a, b, t, -100, "mean", 24)):
        leaves = [x.clone().requires_grad_(True), res.clone().requires_grad_(True)]
        loss = fn(*leaves)
        results.append([loss.detach(), *torch.autograd.grad(loss, leaves)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    for a, b in zip(ck.add_rms_norm_e4m3(x, res, w, EPS), rows_ops.rows_e4m3(x, res, w, EPS)):
        assert torch.equal(a.float(), b.float())
    q, s = ck.quantize_e4m3(torch.randn(9, 64, device=DEV))
    q2, s2 = ck.quantize_e4m3(torch.randn(16, 64, device=DEV))
    assert torch.equal(ck.linear_e4m3(q, s, q2, s2), rows_ops.gemm_e4m3(q, s, q2, s2))


def test_second_derivative_is_refused(ck):
    x, w = randn(4, 64).requires_grad_(True), randn(64, seed=1).requires_grad_(True)
    for out in (ck.rms_norm(x, w, EPS), ck.dropout(x, 0.5, rng_state()), ck.add_rms_norm(x, x.detach(), w, EPS)[0]):
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(out.sum(), x, create_graph=True)


def test_inference_mode_and_backward_accumulation(ck):
    x, res, w = randn(20, 128), randn(20, 128, seed=1), randn(128, seed=2)
    with torch.inference_mode():
        a = ck.add_rms_norm(x, res, w, EPS)
        q = ck.rms_norm_e4m3(x, w, EPS)
    b = ck.add_rms_norm(x, res, w, EPS)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and q[0].shape == x.shape
    # x used twice: both contributions arrive, through .backward() into .grad
    leaf, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    out, h = ck.add_rms_norm(leaf, leaf, wl, EPS)
    (out.float().sum() + h.float().sum()).backward()
    l1, l2 = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    out, h = ck.add_rms_norm(l1, l2, w, EPS)
    g1, g2 = torch.autograd.grad((out, h), (l1, l2), (torch.ones_like(out), torch.ones_like(h)))
    assert torch.equal(leaf.grad, g1 + g2)


def test_norm_beyond_31_bits(ck):
    """The last rows of a matrix of more than 2^31 elements come out as they do alone."""
    cols = 4096
    rows = 2**31 // cols + 6
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    for i in range(0, rows, 65536):
        x[i:i + 65536].normal_()
    w = randn(cols, seed=2, std=0.2, mean=1.0)
    tail = x[-9:].clone()
    out, h = ck.add_rms_norm(x, x, w, EPS)
    o, hh = ck.add_rms_norm(tail, tail, w, EPS)
    assert torch.equal(out[-9:], o) and torch.equal(h[-9:], hh)
    del out, h
    q, s = ck.quantize_e4m3(x)
    qq, ss = ck.quantize_e4m3(tail)
    assert torch.equal(q[-9:].float(), qq.float()) and torch.equal(s[-9:], ss)
    del q
    leaf = x.requires_grad_(True)
    (dx,) = torch.autograd.grad(ck.rms_norm(leaf, w, EPS), leaf, x.detach())
    lt = tail.requires_grad_(True)
    (dt,) = torch.autograd.grad(ck.rms_norm(lt, w, EPS), lt, tail.detach())
    assert torch.equal(dx[-9:], dt)


def test_e4m3_projection_stores_and_groupings(ck):
    """Per-thread stores give what TMA stores give; one CTA a tile is refused, as it is not built."""
    x8, xs = ck.quantize_e4m3(randn(200, 128))
    w8, ws = ck.quantize_e4m3(randn(328, 128, seed=1))
    for out_dtype in (torch.bfloat16, torch.float32):
        base = ck.linear_e4m3(x8, xs, w8, ws, out_dtype)
        for name, value, default in (("epi_tma", 0, 1), ("tile_n", 64, 0), ("tile_n", 256, 0)):
            ck.set_option(name, value)
            try:
                assert torch.equal(base, ck.linear_e4m3(x8, xs, w8, ws, out_dtype))
            finally:
                ck.set_option(name, default)
    ck.set_option("cta_group", 1)
    try:
        with pytest.raises(ck.CodaB200Error, match="CTA pairs"):
            ck.linear_e4m3(x8, xs, w8, ws)
    finally:
        ck.set_option("cta_group", 2)


def test_inference_operators_under_compile(ck):
    def f(x, res, w, w8, ws):
        q, s, h = ck.add_rms_norm_e4m3(x, res, w, EPS)
        return ck.linear_e4m3(q, s, w8, ws), h, *ck.quantize_e4m3(h)

    x, res, w = randn(20, 128), randn(20, 128, seed=1), randn(128, seed=2)
    w8, ws = ck.quantize_e4m3(randn(72, 128, seed=3))
    with torch.no_grad():
        traced = torch.compile(f, fullgraph=True, dynamic=False)(x, res, w, w8, ws)
        for a, b in zip(f(x, res, w, w8, ws), traced):
            assert torch.equal(a.float(), b.float())
