"""The norm's backward stays inside the scratch that the library asks for, with every type, with and without dropout."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("rows,cols", [(1, 1), (7, 64), (5000, 64), (5000, 65), (3000, 249), (3000, 256), (3000, 1000), (2000, 2047), (2000, 4096),
                                       (700, 8192), (700, 8195), (400, 20004), (300, 51200), (300, 51208)])
def test_scratch_holds_the_partial_rows(dtype, p, rows, cols):
    import coda_kernels_b200 as ck

    lib = ck._lib.lib
    size = lib.coda_b200_add_rmsnorm_bwd_scratch_bytes(rows, cols)
    assert size % 4 == 0
    floats = size // 4
    # all of what is asked for is memory of the test's own, and so is what lies on both sides of it
    guard = 64 * cols + 64
    guard += -guard % 4
    memory = torch.full((guard + floats + guard,), 7.0, device=DEV)
    scratch = memory[guard:guard + floats]
    g = torch.Generator(device=DEV).manual_seed(0)
    dout, h = (torch.randn(rows, cols, generator=g, device=DEV).to(dtype) for _ in range(2))
    rstd, w = torch.ones(rows, device=DEV), torch.ones(cols, device=DEV).to(dtype)
    dx, dres, dw = torch.empty_like(h), torch.empty_like(h), torch.empty_like(w)
    rng = torch.tensor([3, 4], dtype=torch.int64, device=DEV)
    rc = lib.coda_b200_add_rmsnorm_bwd(dout.data_ptr(), None, h.data_ptr(), rstd.data_ptr(), w.data_ptr(), p, rng.data_ptr() if p else None, 1,
                                       dx.data_ptr(), dres.data_ptr(), dw.data_ptr(), scratch.data_ptr(), size, rows, cols, CODES[dtype],
                                       torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.coda_b200_last_error()
    assert bool((memory[:guard] == 7.0).all()) and bool((memory[guard + floats:] == 7.0).all())
    # rstd = 1: dweight = sum of dout * h, rounded once; products and sums in fp32 are off by at most 2^-18 of the magnitudes
    terms = dout.double() * h.double()
    want = terms.sum(0)
    bound = want.abs() * torch.finfo(dtype).eps / 2 + 2.0**-18 * terms.abs().sum(0) + torch.finfo(dtype).tiny
    assert bool(((dw.double() - want).abs() <= bound).all())
