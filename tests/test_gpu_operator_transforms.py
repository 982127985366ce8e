"""The operators around the fused linears under PyTorch's program transforms: forward-mode derivatives are refused."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5


@pytest.fixture(scope="module")
def ck():
    import coda_kernels_b200 as ck

    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return ck


def randn(*shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def rng_state():
    return torch.tensor([1234567890123, 7], dtype=torch.int64, device=DEV)


def calls(ck, seed=0):
    """name -> (function, its floating-point inputs)"""
    x, res, w = randn(24, 64, seed=seed), randn(24, 64, seed=seed + 1), randn(64, seed=seed + 2)
    x8, xs = ck.quantize_e4m3(x)
    w8, ws = ck.quantize_e4m3(randn(40, 64, seed=seed + 3))
    vocab = randn(72, 64, seed=seed + 4)
    target = torch.randint(0, 72, (24,), generator=torch.Generator().manual_seed(5), dtype=torch.int32).to(DEV)
    rng = rng_state()
    return {
        "dropout": (lambda x: ck.dropout(x, 0.3, rng, stream=2), (x,)),
        "rms_norm": (lambda x, w: ck.rms_norm(x, w, EPS), (x, w)),
        "add_rms_norm": (lambda x, r, w: ck.add_rms_norm(x, r, w, EPS, p=0.2, rng=rng, stream=3), (x, res, w)),
        "linear_cross_entropy_pieces": (lambda x, v: ck.linear_cross_entropy_pieces(x, v, target, piece=32), (x, vocab)),
        "rms_norm_e4m3": (lambda x, w: ck.rms_norm_e4m3(x, w, EPS), (x, w)),
        "add_rms_norm_e4m3": (lambda x, r, w: ck.add_rms_norm_e4m3(x, r, w, EPS), (x, res, w)),
        "quantize_e4m3": (lambda x: ck.quantize_e4m3(x), (x,)),
        "linear_e4m3": (lambda s, t: ck.linear_e4m3(x8, s, w8, t), (xs, ws)),
    }


NAMES = ["dropout", "rms_norm", "add_rms_norm", "linear_cross_entropy_pieces", "rms_norm_e4m3", "add_rms_norm_e4m3", "quantize_e4m3",
         "linear_e4m3"]
DIFFERENTIABLE = NAMES[:4]


@pytest.mark.parametrize("whole_operators", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(ck, monkeypatch, name, whole_operators):
    """A tangent on any input, with and without a gradient beside it: no result that reads as if the derivative were zero."""
    monkeypatch.setattr(ck.ops, "_WHOLE_OPERATORS", whole_operators)
    fn, inputs = calls(ck)[name]
    for i in range(len(inputs)):
        for needs_grad in (False, True) if name in DIFFERENTIABLE else (False,):
            with fwd.dual_level():
                args = [t.clone().requires_grad_(needs_grad) for t in inputs]
                args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError):
                    fn(*args)
                if not needs_grad:
                    with torch.no_grad(), pytest.raises(NotImplementedError):
                        fn(*args)
    fn(*inputs)  # and nothing is refused without one
    with fwd.dual_level():
        fn(*inputs)
