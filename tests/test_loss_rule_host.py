"""The rule by which the piecewise loss leaves ignored rows out, as the library answers it and as a tracer can follow it."""

import pytest
import torch


@pytest.mark.parametrize("option,value,default", [(None, 0, 0), ("ce_compact", 0, 1), ("cta_group", 1, 2)])
def test_both_forms_agree(option, value, default):
    from coda_kernels_b200 import _lib
    from coda_kernels_b200.ops_ce import _compacts

    if option is not None:
        _lib.set_option(option, value)
    try:
        g = torch.Generator().manual_seed(0)
        seen = set()
        sizes = [(1, 8192, 8), (0, 8192, 4096), (1500, 8191, 2048), (1500, 8192, 2048), (3125, 8000, 1000), (3125, 10000, 800),
                 (3125, 10000, 792), (2**31 - 1, 2**31 - 257, 1 << 20)]
        sizes += [tuple(int(10 ** float(v)) for v in torch.rand(3, generator=g) * torch.tensor([4.0, 2.0, 2.0]) + torch.tensor([0.0, 3.3, 1.5]))
                  for _ in range(300)]
        for M, V, K in sizes:
            lib = M > 0 and bool(_lib.lib.coda_b200_ce_compacts(M, V, K))
            assert _compacts(M, V, K) == lib, (M, V, K)
            seen.add(lib)
        assert seen == ({True, False} if option is None else {False})
    finally:
        if option is not None:
            _lib.set_option(option, default)


def test_the_rule_can_be_traced():
    from coda_kernels_b200 import _lib
    from coda_kernels_b200.ops_ce import _compacts

    traced = torch.compile(lambda t, m, v, k: t + int(_compacts(m, v, k)), fullgraph=True, dynamic=False, backend="eager")
    for M, V, K in [(1500, 8195, 2048), (8192, 128256, 4096), (40, 300, 64), (1500, 8191, 2048), (1, 8192, 8), (0, 8192, 4096),
                    (1003, 32003, 1032)]:
        lib = M > 0 and bool(_lib.lib.coda_b200_ce_compacts(M, V, K))
        assert int(traced(torch.zeros((), dtype=torch.int32), M, V, K)) == int(lib)
