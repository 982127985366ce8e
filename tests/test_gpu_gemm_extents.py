"""The GEMMs refuse operands whose contiguous extent is no multiple of 8 (the piecewise loss has an entry of its own for them).

Every matrix is whole memory with lines 16 elements apart: a call that were accepted would stay inside of it."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ck():
    import coda_kernels_b200 as ck

    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return ck


def test_contiguous_extents_are_refused(ck):
    lib = ck._lib.lib
    a, b, d, e, c = (torch.zeros(16, 16, dtype=torch.bfloat16, device=DEV) for _ in range(5))
    status = ck.ops.status_word(torch.device(DEV))
    stream = torch.cuda.current_stream().cuda_stream
    a, b, d, e, c, status = (t.data_ptr() for t in (a, b, d, e, c, status))
    M, N, K, ld = 16, 16, 12, 16
    for rc in (lambda: lib.coda_b200_gemm(a, ld, 1, b, 1, ld, d, N, 0, M, N, K, None, status, stream),
               lambda: lib.coda_b200_gemm_add(a, ld, 1, b, 1, ld, c, N, 0, d, N, 0, M, N, K, None, status, stream),
               lambda: lib.coda_b200_gemm_ws(a, 1, ld, b, ld, 1, d, N, 0, 12, N, 16, None, None, 0, status, stream),  # A along M
               lambda: lib.coda_b200_gemm_sigmoid(a, ld, 1, b, 1, ld, d, N, 0, M, N, K, status, stream),
               lambda: lib.coda_b200_gemm_swiglu(a, ld, 1, b, 1, ld, d, N, e, 8, M, N, K, status, stream)):
        assert rc() == -1
        assert b"multiple of 8" in lib.coda_b200_last_error(), lib.coda_b200_last_error()
    x = torch.zeros(16, 16, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: ck.ops.gemm(x[:, :12], x[:12]), lambda: ck.linear_swiglu(x[:, :12], x[:, :12])):
        with pytest.raises(ck.CodaB200Error, match="multiple of 8"):
            call()


@pytest.mark.parametrize("M,N,K", [(16, 16, 12), (13, 40, 64), (37, 264, 1003), (300, 1032, 517), (1, 8, 1), (700, 512, 8200)])
@pytest.mark.parametrize("a_along_m", [False, True])
@pytest.mark.parametrize("with_c", [False, True])
def test_the_entry_for_any_extent(ck, M, N, K, a_along_m, with_c):
    """Elements between an operand's extent and its next line are not used (they hold NaN), nor is anything outside D written.
    bf16 products are exact in fp32; K of them summed 16 an instruction are off by (K / 16 + 2) * 2^-23 of their magnitudes."""
    from coda_kernels_b200.ops_ce import _gemm_ragged

    g = torch.Generator().manual_seed(M + N + K)

    def padded(rows, cols):
        t = torch.full((rows, -(-cols // 8) * 8 + 8), float("nan"))
        t[:, :cols] = torch.randn(rows, cols, generator=g)
        return t.bfloat16().to(DEV)[:, :cols]

    A = padded(K, M).T if a_along_m else padded(M, K)
    B = torch.randn(K, N, generator=g).bfloat16().to(DEV)
    C = torch.randn(M, N, generator=g).to(DEV) if with_c else None
    alpha = torch.tensor([0.5], device=DEV)
    whole = torch.full((M + 2, N), 7.0, device=DEV)
    out = whole[1:-1]
    _gemm_ragged(A, B, C, alpha, out)
    a64, b64 = A.double(), B.double()
    want, terms = 0.5 * (a64 @ b64), 0.5 * (a64.abs() @ b64.abs())
    if with_c:
        want, terms = want + C.double(), terms + C.double().abs()
    assert bool(((out.double() - want).abs() <= ((K / 16 + 2) * 2.0**-23 + 2.0**-23) * terms).all())
    assert bool((whole[[0, -1]] == 7.0).all())
    ck.ops.check_device_status(torch.device(DEV))
