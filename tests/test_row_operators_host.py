"""Argument checks of the operators around the fused linears, and the oracle's generator: no GPU needed."""

import numpy as np
import pytest
import torch

from oracle import rows as ref


def test_generator_known_answers():
    """The published known-answer vectors of Philox4x32-10."""
    for counter, key, want in (
        ([0] * 4, (0, 0), "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
        ([0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF), "408f276d 41c83b0e a20bc7c6 6d5451fd"),
        ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], (0xA4093822, 0x299F31D0), "d16cfe09 94fdcceb 5001e420 24126ea1"),
    ):
        got = ref.philox([np.array([c], dtype=np.uint64) for c in counter], key)
        assert " ".join(f"{int(v[0]):08x}" for v in got) == want


def test_c_entries_refuse_on_the_host():
    """Fake, aligned, never dereferenced addresses."""
    from coda_kernels_b200 import _lib

    lib, p = _lib.lib, 1 << 20

    def refused(rc, text):
        assert rc == -1 and text in lib.coda_b200_last_error(), (rc, lib.coda_b200_last_error())

    refused(lib.coda_b200_dropout(p, p, 4, 0, 0, 0.1, p, 0, None, None), b"cols")
    refused(lib.coda_b200_dropout(p, p, -1, 8, 0, 0.1, p, 0, None, None), b"rows")
    refused(lib.coda_b200_dropout(p, p, 4, 8, 3, 0.1, p, 0, None, None), b"dtype")
    refused(lib.coda_b200_dropout(p, p, 4, 8, 0, 1.0, p, 0, None, None), b"probability")
    refused(lib.coda_b200_dropout(p, p, 4, 8, 0, float("nan"), p, 0, None, None), b"probability")
    refused(lib.coda_b200_dropout(p, p, 4, 8, 0, 0.1, None, 0, None, None), b"seed")
    refused(lib.coda_b200_dropout(p, p, 4, 8, 0, 0.1, p, 1 << 32, None, None), b"stream")
    refused(lib.coda_b200_dropout(None, p, 4, 8, 0, 0.1, p, 0, None, None), b"NULL")
    assert lib.coda_b200_dropout(None, None, 0, 8, 0, 0.1, p, 0, None, None) == 0  # no rows: nothing to do
    refused(lib.coda_b200_add_rmsnorm_fwd(p, p, None, 1e-5, 0.0, None, 0, None, p, p, p, 4, 8, 0, None), b"NULL")
    refused(lib.coda_b200_rows_e4m3(p, None, None, 0.0, None, p, None, 4, 8, 0, None), b"NULL")
    need = lib.coda_b200_add_rmsnorm_bwd_scratch_bytes(1000, 64)
    assert need > 0 and lib.coda_b200_add_rmsnorm_bwd_scratch_bytes(0, 64) == 0
    refused(lib.coda_b200_add_rmsnorm_bwd(p, p, p, p, p, 0.0, None, 0, p, p, p, p, need - 4, 1000, 64, 0, None), b"scratch")
    refused(lib.coda_b200_gemm_e4m3(p, p, p, p, p, 16, 0, 4, 16, 40, None, 0, p, None), b"multiple of 16")
    refused(lib.coda_b200_gemm_e4m3(p, p, p, p, p, 12, 0, 4, 12, 32, None, 0, p, None), b"multiples of 8")
    refused(lib.coda_b200_gemm_e4m3(p + 8, p, p, p, p, 16, 0, 4, 16, 32, None, 0, p, None), b"16-byte")
    refused(lib.coda_b200_gemm_e4m3(p, p, p, p, p, 16, 0, 0, 16, 32, None, 0, p, None), b"positive")
    refused(lib.coda_b200_gemm_e4m3(p, p, p, p, p, 16, 0, 4, 16, 32, p + 4, 64, p, None), b"16-byte")
    assert lib.coda_b200_gemm_e4m3_workspace_bytes(50, 6144, 4096) > 0 == lib.coda_b200_gemm_e4m3_workspace_bytes(1, 6144, 4096)
    refused(lib.coda_b200_gemm_softmax_grad(p, 64, 1, p, 1, 64, p, p, -100, 0, None, p, 12, 4, 12, 64, p, None), b"ldg")
    refused(lib.coda_b200_gemm_softmax_grad(p, 64, 1, p, 1, 64, p, p, -100, -1, None, p, 16, 4, 12, 64, p, None), b"col0")
    refused(lib.coda_b200_ce_loss(p, 60, 1, p, 1, 60, p, -100, 1, None, p, p, p, p, p, p, p, 4, 12, 60, p, None), b"K must")


def test_products_of_counted_rows_refuse_on_the_host():
    from coda_kernels_b200 import _lib

    lib, p = _lib.lib, 1 << 20

    def refused(rc, text):
        assert rc in (-1, -2) and text in lib.coda_b200_last_error(), (rc, lib.coda_b200_last_error())

    assert lib.coda_b200_ce_compacts(8192, 128256, 4096) == 1 and lib.coda_b200_ce_compacts(256, 8000, 512) == 0
    refused(lib.coda_b200_ce_compact(p, p, -100, p, p, None, p, 4, 64, None), b"NULL")
    refused(lib.coda_b200_ce_compact(p, p, -100, p, p, p, p, 4, 60, None), b"multiple of 8")
    refused(lib.coda_b200_ce_scatter(p + 4, p, p, 4, 64, None), b"16-byte")
    refused(lib.coda_b200_gemm_live(p, 64, p, 64, None, p, 64, 0, None, None, 0, 4, 64, 64, p, None), b"NULL")
    refused(lib.coda_b200_gemm_live(p, 64, p, 60, None, p, 60, 0, None, p, 0, 4, 60, 64, p, None), b"multiples of 8")
    refused(lib.coda_b200_gemm_live(p, 56, p, 64, None, p, 64, 0, None, p, 0, 4, 64, 64, p, None), b"leading")
    refused(lib.coda_b200_gemm_softmax_grad(p, 1, 64, p, 1, 64, p, p, -100, 0, p, p, 16, 64, 16, 64, p, None), b"contiguous along")
    assert lib.coda_b200_set_option(b"cta_group", 1) == 0
    try:
        assert lib.coda_b200_ce_compacts(8192, 128256, 4096) == 0
    finally:
        assert lib.coda_b200_set_option(b"cta_group", 2) == 0


def test_cpu_tensors_are_refused():
    import coda_kernels_b200 as ck

    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    rng = torch.zeros(2, dtype=torch.int64)
    q, s = x.to(torch.float8_e4m3fn), torch.ones(4)
    for call in (lambda: ck.dropout(x, 0.1, rng), lambda: ck.rms_norm(x, w, 1e-5), lambda: ck.add_rms_norm(x, x, w, 1e-5),
                 lambda: ck.rms_norm_e4m3(x, w, 1e-5), lambda: ck.add_rms_norm_e4m3(x, x, w, 1e-5), lambda: ck.quantize_e4m3(x),
                 lambda: ck.linear_e4m3(q, s, q, s),
                 lambda: ck.linear_cross_entropy_pieces(x, x, torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_default_piece():
    from coda_kernels_b200.ops_ce import _PIECE_ELEMENTS, _PIECE_MIN, default_piece

    for rows in (0, 1, 100, 2048, 8192, 100_000):
        for vocab in (1, 7, 8191, 8193, 32003, 128256, 1_000_003):
            piece = default_piece(rows, vocab)
            assert 1 <= piece <= vocab
            assert piece * rows <= max(_PIECE_ELEMENTS, _PIECE_MIN * rows) + 256 * rows
            assert piece == vocab or piece % 256 == 0
