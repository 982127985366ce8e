"""The operators around the fused linears run together, as a program uses them.

Training: norm -> ``linear_swiglu`` -> down projection -> residual + dropout + norm -> dropout -> loss in vocabulary pieces,
against the same formulas in 64 bits with autograd.  Between the bf16 inputs and a gradient lie at most 14 roundings to
bf16 (a, preact, z, y, out, h, its dropout, the logit gradient, and the gradients of the last five); each changes its tensor
by at most 2^-8 of its norm, and no operator here amplifies a relative error of a whole tensor by more than a factor of
about one, so a gradient is off by at most 14 * 2^-8 = 5.5e-2 of its norm.  The loss is a mean over rows of fp32 values
whose inputs carry seven of those roundings; its error in logit units is far below the bound 7 * 2^-8 on a logit of unit size.

Serving: the same sublayer in 8 bits, each step against the exact product of what the step was given.
"""

import pytest
import torch

from oracle import rows as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5
SEED, STEP = 987654321, 3


@pytest.fixture(scope="module")
def ck():
    import coda_kernels_b200 as ck

    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return ck


def randn(*shape, seed=0, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std + mean).bfloat16().to(DEV)


def parameters(M=200, dim=256, ffn=384, vocab=1003):
    p = {
        "x": randn(M, dim),
        "wn0": randn(dim, seed=1, std=0.1, mean=1.0),
        "w_up": randn(2 * ffn, dim, seed=2, std=dim**-0.5),
        "w_down": randn(dim, ffn, seed=3, std=ffn**-0.5),
        "wn1": randn(dim, seed=4, std=0.1, mean=1.0),
        "w_vocab": randn(vocab, dim, seed=5, std=dim**-0.5),
    }
    g = torch.Generator().manual_seed(6)
    t = torch.randint(0, vocab, (M,), generator=g, dtype=torch.int32)
    t[::7] = -100
    return p, t.to(DEV)


def loss_of(ck, p, t, rng):
    a = ck.rms_norm(p["x"], p["wn0"], EPS)
    z = ck.linear_swiglu(a, p["w_up"])
    y = z @ p["w_down"].t()
    out, h = ck.add_rms_norm(y, p["x"], p["wn1"], EPS, p=0.1, rng=rng, stream=4)
    out = ck.dropout(out, 0.2, rng, stream=5)
    return ck.linear_cross_entropy_pieces(out, p["w_vocab"], t, piece=256) + 0.01 * h.float().square().mean()


def loss_in_64_bits(p, t, step):
    def norm(h, w):
        return h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * w

    M, dim = p["x"].shape
    a = norm(p["x"], p["wn0"])
    pre = a @ p["w_up"].T
    z = torch.nn.functional.silu(pre[:, ::2]) * pre[:, 1::2]
    y = z @ p["w_down"].T
    h = p["x"] + ref.dropped(y, ref.keep_mask(M, dim, 0.1, SEED, step, 4).to(DEV), 0.1)
    out = ref.dropped(norm(h, p["wn1"]), ref.keep_mask(M, dim, 0.2, SEED, step, 5).to(DEV), 0.2)
    return torch.nn.functional.cross_entropy(out @ p["w_vocab"].T, t.long(), ignore_index=-100) + 0.01 * h.square().mean()


def test_training_step(ck):
    raw, t = parameters()
    p = {k: v.requires_grad_(True) for k, v in raw.items()}
    rng = torch.tensor([SEED, STEP], dtype=torch.int64, device=DEV)
    loss = loss_of(ck, p, t, rng)
    grads = torch.autograd.grad(loss, list(p.values()))
    p64 = {k: v.detach().double().requires_grad_(True) for k, v in raw.items()}
    want = loss_in_64_bits(p64, t, STEP)
    wgrads = torch.autograd.grad(want, list(p64.values()))
    assert abs(float(loss.detach()) - float(want.detach())) <= 7 * 2.0**-8
    for name, g, w in zip(p, grads, wgrads):
        err = float((g.double() - w).norm() / w.norm())
        assert err <= 14 * 2.0**-8, f"{name}: {err:.3e}"
    ck.ops.check_device_status(torch.device(DEV))


def test_captured_training_steps_draw_new_masks(ck):
    """A replayed step with the state advanced on the device gives what eager steps give, mask by mask."""
    raw, t = parameters(M=64)
    p = {k: v.requires_grad_(True) for k, v in raw.items()}
    rng = torch.tensor([SEED, 0], dtype=torch.int64, device=DEV)

    def step():
        loss = loss_of(ck, p, t, rng)
        grads = torch.autograd.grad(loss, list(p.values()))
        rng[1] += 1
        return loss.detach(), *grads

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    rng[1] = 10
    seen = []
    for _ in range(3):
        graph.replay()
        seen.append([v.clone() for v in static])
    torch.cuda.synchronize()
    assert int(rng[1]) == 13
    rng[1] = 10
    for replayed in seen:
        for a, b in zip(replayed, step()):
            assert torch.equal(a, b)
    assert not torch.equal(seen[0][1], seen[1][1])


@pytest.mark.parametrize("M", [1, 5, 30, 130])
def test_serving_in_8_bits(ck, M):
    """Products are exact in fp32 up to their accumulation (see the projection's own test) and round once to bf16; rows in
    8 bits are checked against the 64-bit norm of the residual stream that came out beside them."""
    raw, _ = parameters(M=M)
    with torch.no_grad():
        up8, up_s = ck.quantize_e4m3(raw["w_up"])
        down8, down_s = ck.quantize_e4m3(raw["w_down"])
        y = randn(M, 256, seed=9)
        q, s, h = ck.add_rms_norm_e4m3(y, raw["x"], raw["wn1"], EPS)
        pre = ck.linear_e4m3(q, s, up8, up_s)
        z = torch.nn.functional.silu(pre[:, ::2]) * pre[:, 1::2]
        z8, z_s = ck.quantize_e4m3(z)
        out = ck.linear_e4m3(z8, z_s, down8, down_s, torch.float32)
    h64 = y.double() + raw["x"].double()
    want = ref.norm(h64, raw["wn1"].double(), EPS)[0]
    got = q.double() * s.double()[:, None]
    assert bool(((got - want).abs() <= want.abs() * (2.0**-4 + 2.0**-16) + s.double()[:, None] * 2.0**-10).all())
    for x8, xs, w8, ws, y, half in ((q, s, up8, up_s, pre, 2.0**-8), (z8, z_s, down8, down_s, out, 2.0**-24)):
        a, b = x8.double() * xs.double()[:, None], w8.double() * ws.double()[:, None]
        exact, terms = a @ b.T, a.abs() @ b.abs().T
        K = a.shape[1]
        assert bool(((y.double() - exact).abs() <= half * exact.abs() + (K / 32 + 2) * 2.0**-22 * terms).all())
    # the whole in 8 bits stays near the whole in 64: every value of q, z8 and the two weights is off by 2^-4 of itself at
    # most; gate and up each carry q's and a weight's, their product both, so 6 * 2^-4 of the norm of the exact result
    pre64 = want @ raw["w_up"].double().T
    z64 = torch.nn.functional.silu(pre64[:, ::2]) * pre64[:, 1::2]
    far = z64 @ raw["w_down"].double().T
    assert float((out.double() - far).norm()) <= 6 * 2.0**-4 * float(far.norm())
