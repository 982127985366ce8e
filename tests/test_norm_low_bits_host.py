"""The bits of ``h`` below its type that ``add_rms_norm`` keeps for its backward: their room, and what is refused.  No GPU needed."""

import torch


def test_room():
    """As the library counts it and as a tracer can: a word for eight elements, one more a row where rows may share eight."""
    from coda_kernels_b200 import _lib
    from coda_kernels_b200.ops_rows import _low_like

    for rows, cols in ((1, 1), (1, 8), (7, 8), (7, 9), (5, 64), (10007, 3), (0, 16), (0, 3), (3, 20004), (2, 51201)):
        room = _low_like(torch.empty(rows, cols, dtype=torch.bfloat16)).numel()
        assert 4 * room == _lib.lib.coda_b200_add_rmsnorm_low_bytes(rows, cols)
        # word of the chunk of row r that begins at element e: e / 8 (+ r); all inside, and no two rows' the same
        words = [{(r * cols + c) // 8 + (r if cols % 8 else 0) for c in range(cols)} for r in range(min(rows, 50))]
        assert len(set().union(*words)) == sum(map(len, words))
        if rows:
            assert (rows * cols - 1) // 8 + (rows - 1 if cols % 8 else 0) < room


def test_refusals():
    """Fake, aligned, never dereferenced addresses."""
    from coda_kernels_b200 import _lib

    lib, p = _lib.lib, 1 << 20
    assert lib.coda_b200_add_rmsnorm_fwd_low(p, p, p, 1e-5, 0.0, None, 0, None, p, p, p, p, 4, 8, 2, None) == -1
    assert b"2-byte" in lib.coda_b200_last_error()
    assert lib.coda_b200_add_rmsnorm_fwd_low(p, p, p, 1e-5, 0.0, None, 0, None, None, p, p, p, 4, 8, 0, None) == -1
    need = lib.coda_b200_add_rmsnorm_bwd_scratch_bytes(4, 8)
    assert lib.coda_b200_add_rmsnorm_bwd_low(p, p, p, p, p, p, 0.0, None, 0, p, p, p, p, need, 4, 8, 2, None) == -1
    assert b"2-byte" in lib.coda_b200_last_error()
    assert lib.coda_b200_add_rmsnorm_bwd_low(p, p, p, p + 8, p, p, 0.0, None, 0, p, p, p, p, need, 4, 8, 0, None) == -1
    assert b"16-byte" in lib.coda_b200_last_error()
