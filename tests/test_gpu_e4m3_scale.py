"""The scale of a row of e4m3 values is the fp32 quotient of its largest magnitude and 448, and ties of the values over it go
to the even e4m3 value.

No tolerance: the scale is one division of fp32 numbers, rounded once.  A value over its scale is taken in 64 bits here;
rounding that to fp32 gives what dividing two fp32 numbers in fp32 gives (53 >= 2 * 24 + 2 bits)."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# largest magnitudes whose quotient by 448 = 7 * 64 is exact (they are multiples of 7), and some where it is not
TOPS = [2.625, 5.25, 21.0, 1.3125, 1.53125, 0.4375, 3.5, 448.0, 1.0, 0.69921875, 3.984375, 2.625 * 2.0**-30, 1.53125 * 2.0**60]


@pytest.fixture(scope="module")
def ck():
    import coda_kernels_b200 as ck

    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return ck


def every_bf16(top):
    """All bf16 values of either sign from top / 64 to top."""
    bits = torch.arange(2**15, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    v = bits[(bits <= top) & (bits > top / 64)]
    return torch.cat([v, -v])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", TOPS)
def test_scale_and_ties(ck, top, dtype):
    row = every_bf16(top).to(dtype)
    assert float(row.abs().max()) == top
    x = torch.stack([row, row.flip(0)]).to(DEV)
    for y in (x, torch.nn.functional.pad(x, (0, -x.shape[1] % 8)), x.repeat(1, 12)):  # ragged, whole chunks, a long row
        q, scale = ck.quantize_e4m3(y)
        want = (torch.tensor([top], dtype=torch.float32) / 448.0).to(DEV)
        assert torch.equal(scale, want.expand(2)), (float(scale[0]), float(want))
        quotient = (y.double() / want.double()).float()
        assert torch.equal(q.float(), quotient.to(torch.float8_e4m3fn).float())
        if (torch.tensor(top).double() / 448).item() == want.item():  # the scale is exact: so is the definition
            exact = (y.double() * 448 / top).float().to(torch.float8_e4m3fn)
            assert torch.equal(q.float(), exact.float())


def test_scale_of_random_rows(ck):
    g = torch.Generator().manual_seed(3)
    for cols in (40, 257, 4096, 20000):
        x = (torch.randn(200, cols, generator=g) * torch.exp(4 * torch.randn(200, 1, generator=g))).to(DEV)
        q, scale = ck.quantize_e4m3(x)
        want = x.abs().amax(1).cpu() / 448.0
        assert torch.equal(scale.cpu(), want)
        assert torch.equal(q.float(), (x.double() / scale.double()[:, None]).float().to(torch.float8_e4m3fn).float())
