"""The weight gradient of ``add_rms_norm`` is summed from ``h`` as it was before its rounding, so its error is that of a plain
form in fp32 that is rounded once.

A sum over rows of dout * h * rstd.  ``LOW``: how far the h that the backward works with may be from the unrounded one, relative to
it (four bits below the type in units of 4369 or 546 fp32 steps of 2^-23: half a unit, with a margin of 1.9); an fp16 h below
2^-14, where they do not reach, by the type's half step 2^-25.  ``F32`` = 2^-18 stands for 64 roundings of 2^-24, relative
to the magnitudes that went into h and into the sums."""

import pytest
import torch

from oracle import rows as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
LOW = {torch.bfloat16: 2.0**-11, torch.float16: 2.0**-14, torch.float32: 0.0}
SMALL = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}
TINY = {torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25, torch.float32: 2.0**-126}
F32 = 2.0**-18
EPS = 1e-5


@pytest.fixture(scope="module")
def ck():
    import coda_kernels_b200 as ck

    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return ck


def inputs(dtype, rows, cols, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x, res, dout = (torch.randn(rows, cols, generator=g) for _ in range(3))
    return [(t * s).to(dtype).to(DEV) for t, s in ((x, scale), (res, scale), (dout, 1.0))] + [(torch.rand(cols, generator=g) + 0.5).to(dtype).to(DEV)]


def check(ck, dtype, x, res, dout, w, p):
    rows, cols = x.shape
    rng = torch.tensor([77, 5], dtype=torch.int64, device=DEV)
    leaves = [t.clone().requires_grad_(True) for t in (x, res, w)]
    out, _ = ck.add_rms_norm(*leaves, EPS, p=p, rng=rng if p else None, stream=5)
    (dw,) = torch.autograd.grad(out, leaves[2], dout)
    x64, r64, do64 = x.double(), res.double(), dout.double().abs()
    keep = ref.keep_mask(rows, cols, p, 77, 5, 5).to(DEV) if p else torch.ones_like(x64, dtype=torch.bool)
    part = ref.dropped(x64, keep, p)
    h, size = part + r64, part.abs() + r64.abs()
    rstd = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
    want = (dout.double() * h * rstd).sum(0)
    slack = F32 * (1 + (rstd * size).square().mean(1, keepdim=True).sqrt())  # of rstd
    terms = (do64 * rstd * (h.abs() * (LOW[dtype] + slack) + SMALL[dtype] + F32 * size)).sum(0)
    bound = HALF[dtype] * (want.abs() + terms) + terms + TINY[dtype]
    err = (dw.double() - want).abs()
    assert bool((err <= bound).all()), (float((err - bound).max()), float((err / bound).max()))


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("p", [0.0, 0.2])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (40, 8), (2000, 64), (1000, 65), (777, 128), (600, 249), (500, 1000), (300, 1531),
                                       (2049, 4096), (200, 8190), (200, 8192), (40, 16384), (30, 20004), (20, 51208), (10007, 3)])
def test_against_the_unrounded_sum(ck, dtype, p, rows, cols):
    check(ck, dtype, *inputs(dtype, rows, cols), p)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_half_way_between_two_of_the_type(ck, dtype):
    """x + residual with x half a step of residual, of either sign: the first and the last value of the four bits; and sums that cancel, and small ones."""
    rows, cols = 512, 264
    x, res, dout, w = inputs(dtype, rows, cols)
    step = torch.finfo(dtype).eps
    _, e = torch.frexp(res.float())
    half = torch.ldexp(torch.full_like(res, step / 2, dtype=torch.float32), e - 1)
    x = torch.where(torch.rand(rows, cols, generator=torch.Generator().manual_seed(1)).to(DEV) < 0.5, half, -half).to(dtype)
    x[:64] = -res[:64]
    x[64:128] *= 0.75
    check(ck, dtype, x, res, dout, w, 0.0)
    check(ck, dtype, *inputs(dtype, rows, cols, seed=3, scale=2.0**-13 if dtype == torch.float16 else 2.0**-60), 0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_non_finite_rows(ck, dtype):
    """They make the weight gradient NaN in their column, a neighbour's garbage nowhere; h and the other gradients have the bits
    they have when the weight needs none."""
    for cols in (264, 263):
        x, res, dout, w = inputs(dtype, 9, cols)
        for bad in (float("nan"), float("inf")):
            x2 = x.clone()
            x2[4, 7] = bad
            leaves = [t.clone().requires_grad_(True) for t in (x2, res, w)]
            out, h = ck.add_rms_norm(*leaves, EPS)
            dx, dres, dw = torch.autograd.grad((out, h), leaves, (dout, dout))
            assert bool(dw[7].isnan())
            frozen = [t.clone().requires_grad_(True) for t in (x2, res)]
            out2, h2 = ck.add_rms_norm(*frozen, w, EPS)
            for a, b in zip((out, h, dx, dres), (out2, h2, *torch.autograd.grad((out2, h2), frozen, (dout, dout)))):
                assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
        # the row beside a matrix' end, of columns that share a chunk with their neighbours'
        leaves = [t.clone().requires_grad_(True) for t in (x, res, w)]
        (dw,) = torch.autograd.grad(ck.add_rms_norm(*leaves, EPS)[0], leaves[2], dout)
        assert bool(torch.isfinite(dw).all())


def test_what_is_kept(ck):
    """Beside the outputs and a number a row: half a byte an element of a 2-byte type, nothing of fp32."""
    rows, cols = 512, 2048

    def held(dtype):
        x, res, _, w = inputs(dtype, rows, cols)
        x.requires_grad_(True)
        before = torch.cuda.memory_allocated()
        out, h = ck.add_rms_norm(x, res, w, EPS)
        return torch.cuda.memory_allocated() - before - (out.numel() + h.numel()) * out.element_size() - 4 * rows

    for dtype, extra in ((torch.bfloat16, rows * cols // 2), (torch.float16, rows * cols // 2), (torch.float32, 0)):
        assert extra <= held(dtype) <= extra + 2048, dtype
