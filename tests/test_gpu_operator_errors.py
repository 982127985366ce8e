"""Errors of the compiled operators on a GPU: running out of memory stays what PyTorch calls it."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_no_memory_is_reported_as_such():
    """Asked for 16 TB, the allocator refuses without touching the device; the next call works."""
    import coda_kernels_b200 as ck

    one = torch.ones(1, 1, dtype=torch.bfloat16, device=DEV)
    huge = one.expand(2**21, 2**22)
    w = torch.ones(2**22, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: ck.dropout(huge, 0.0), lambda: ck.rms_norm(huge, w, 1e-5), lambda: ck.quantize_e4m3(huge),
                 lambda: ck.add_rms_norm(huge, huge, w, 1e-5)):
        with pytest.raises(torch.OutOfMemoryError):
            call()
    assert torch.equal(ck.dropout(one, 0.0), one)


def test_what_the_library_refuses_and_what_the_checks_refuse():
    import coda_kernels_b200 as ck

    x = torch.ones(200, 128, dtype=torch.bfloat16, device=DEV)
    q, s = ck.quantize_e4m3(x)
    ck.set_option("cta_group", 1)
    try:
        with pytest.raises(ck.CodaB200Error, match="CTA pairs"):
            ck.linear_e4m3(q, s, q, s)
    finally:
        ck.set_option("cta_group", 2)
    with pytest.raises(RuntimeError, match="no backward") as caught:
        ck.quantize_e4m3(x.requires_grad_(True))
    assert not isinstance(caught.value, ck.CodaB200Error)
