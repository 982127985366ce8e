"""The operators around the fused linears under PyTorch's program transforms: forward-mode derivatives are refused; tracers and
dispatch modes see the computation."""

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


# ------------------------------------------------------------------------------------------------ tracers and modes
def flat(out):
    return [t for t in (out if isinstance(out, tuple) else (out,)) if t is not None]


def step_of(fn, differentiable):
    """The forward, and with gradients for every input where there are any, as a function of plain tensors."""
    if not differentiable:
        return lambda *inputs: flat(fn(*inputs))

    def step(*inputs):
        leaves = [t.detach().requires_grad_(True) for t in inputs]
        outs = flat(fn(*leaves))
        seeds = [torch.ones_like(o) * 0.5 for o in outs]
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, seeds))

    return step


@pytest.mark.parametrize("name", NAMES)
def test_traced_program_computes_on_other_inputs(ck, name):
    """A graph recorded below autograd holds the kernels, not only their allocations."""
    from torch.fx.experimental.proxy_tensor import make_fx

    fn, inputs = calls(ck)[name]
    step = step_of(fn, name in DIFFERENTIABLE)
    graph = make_fx(step)(*inputs)
    for seed in (0, 40):
        _, others = calls(ck, seed)[name]
        want = step(*others)
        filler = [torch.full((64, 64), float("nan"), device=DEV) for _ in range(8)]
        del filler  # what memory the replay gets holds something else
        got = graph(*others)
        assert len(want) == len(got)
        for a, b in zip(want, got):
            assert a.dtype == b.dtype and torch.equal(a.float(), b.float())


@pytest.mark.parametrize("name", NAMES)
def test_dispatch_modes_see_forward_and_backward(ck, name):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    fn, inputs = calls(ck)[name]
    leaves = [t.clone().requires_grad_(name in DIFFERENTIABLE) for t in inputs]
    plain = flat(fn(*leaves))
    with Seen() as forward:
        outs = flat(fn(*leaves))
    assert any(n.startswith("coda_b200") for n in forward.names), forward.names
    for a, b in zip(plain, outs):
        assert torch.equal(a.detach().float(), b.detach().float())
    if name in DIFFERENTIABLE:
        seeds = [torch.ones_like(o) for o in plain]
        want = torch.autograd.grad(plain, leaves, seeds)  # the forward ran outside of the mode
        with Seen() as backward:
            got = torch.autograd.grad(outs, leaves, seeds)
        assert any(n.startswith("coda_b200") for n in backward.names), backward.names
        for a, b in zip(want, got):
            assert torch.equal(a, b)
        outs = flat(fn(*leaves))
        with Seen() as backward:
            torch.autograd.grad(outs, leaves, seeds)
        assert any(n.startswith("coda_b200") for n in backward.names), backward.names


def test_selective_checkpointing_runs_the_policy(ck):
    """A policy that keeps the norm's outputs finds the norm, and the gradients are those without checkpointing."""
    from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts

    if not ck.ops._fast():
        pytest.skip("the Python nodes' ops write into buffers they are given, which a policy cannot keep")
    x, res, w = (randn(*s, seed=i).requires_grad_(True) for i, s in enumerate(((24, 64), (24, 64), (64,))))
    rng, asked = rng_state(), []

    def block(x, res, w):
        out, h = ck.add_rms_norm(x, res, w, EPS, p=0.2, rng=rng)
        return torch.sin(ck.dropout(out, 0.1, rng, stream=1).float()) + h.float()

    def policy(ctx, op, *args, **kwargs):
        asked.append(str(op))
        return CheckpointPolicy.MUST_SAVE if str(op).startswith("coda_b200") else CheckpointPolicy.PREFER_RECOMPUTE

    def context():
        return create_selective_checkpoint_contexts(policy)

    want = torch.autograd.grad(block(x, res, w).sum(), (x, res, w))
    got = torch.autograd.grad(checkpoint(block, x, res, w, use_reentrant=False, context_fn=context).sum(), (x, res, w))
    assert any(n.startswith("coda_b200") for n in asked)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_shapes_without_a_device(ck):
    """Fake tensors: shapes, types and devices of the row operators without a launch."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode() as mode:
        x = torch.empty(6, 5, 64, dtype=torch.bfloat16, device=DEV)
        w = torch.empty(64, dtype=torch.bfloat16, device=DEV)
        rng = torch.empty(2, dtype=torch.int64, device=DEV)
        assert ck.dropout(x, 0.5, rng).shape == x.shape
        out, h = ck.add_rms_norm(x, x, w, EPS, p=0.5, rng=rng)
        assert out.shape == h.shape == x.shape and out.dtype == x.dtype and out.device == x.device
        assert ck.rms_norm(x, w, EPS).shape == x.shape
        q, scale, h = ck.add_rms_norm_e4m3(x, x, w, EPS)
        assert q.shape == x.shape and q.dtype == torch.float8_e4m3fn and scale.shape == (6, 5) and scale.dtype == torch.float32
        leaf = x.clone().requires_grad_(True)
        (grad,) = torch.autograd.grad(ck.rms_norm(leaf, w, EPS).sum(), leaf)
        assert grad.shape == x.shape


def test_recorded_loss_keeps_its_way_when_options_change(ck):
    """Whether the rows that count are put first is decided when a program is recorded, for forward and backward together."""
    from torch.fx.experimental.proxy_tensor import make_fx

    g = torch.Generator().manual_seed(0)
    M, K, V = 1500, 2048, 8195
    x, w = (torch.randn(*s, generator=g).bfloat16().to(DEV) for s in ((M, K), (V, K)))
    w *= K**-0.5
    target = torch.randint(0, V, (M,), generator=g, dtype=torch.int32).to(DEV)
    target[::3] = -100
    assert ck._lib.lib.coda_b200_ce_compacts(M, V, K) == 1
    step = step_of(lambda x, w: ck.linear_cross_entropy_pieces(x, w, target, piece=3000), True)
    for recorded, later in ((1, 0), (0, 1)):
        ck.set_option("ce_compact", recorded)
        try:
            want = step(x, w)
            graph = make_fx(step)(x, w)
            ck.set_option("ce_compact", later)
            for a, b in zip(want, graph(x, w)):
                assert torch.equal(a, b)
        finally:
            ck.set_option("ce_compact", 1)


@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("name", ["add_rms_norm", "rms_norm", "linear_cross_entropy_pieces"])
def test_one_tensor_in_two_places_under_compile(ck, name, dynamic):
    """Its gradient is the sum of both places', as an eager call gives it (two bf16 numbers, added once)."""
    a = randn(40) if name == "rms_norm" else randn(24, 64)
    w, rng = randn(64, seed=1), rng_state()
    target = torch.arange(24, dtype=torch.int32, device=DEV).flip(0)
    fn = {
        "add_rms_norm": lambda a: ck.add_rms_norm(a, a, w, EPS, p=0.2, rng=rng),
        "rms_norm": lambda a: ck.rms_norm(a, a, EPS),
        "linear_cross_entropy_pieces": lambda a: ck.linear_cross_entropy_pieces(a, a, target),
    }[name]
    two = {
        "add_rms_norm": lambda a, b: ck.add_rms_norm(a, b, w, EPS, p=0.2, rng=rng),
        "rms_norm": lambda a, b: ck.rms_norm(a, b, EPS),
        "linear_cross_entropy_pieces": lambda a, b: ck.linear_cross_entropy_pieces(a, b, target),
    }[name]
    a.requires_grad_(True)
    eager = flat(fn(a))
    seeds = [torch.ones_like(o) for o in eager]
    (want,) = torch.autograd.grad(eager, a, seeds)
    b, c = (a.detach().clone().requires_grad_(True) for _ in range(2))
    assert torch.equal(want, sum(torch.autograd.grad(flat(two(b, c)), (b, c), seeds)))
    for traced, args in ((torch.compile(fn, fullgraph=True, dynamic=dynamic), (a,)), (torch.compile(two, fullgraph=True, dynamic=dynamic), (a, a))):
        outs = flat(traced(*args))
        for x, y in zip(outs, eager):
            assert torch.equal(x, y)
        (got,) = torch.autograd.grad(outs, a, seeds)
        assert torch.equal(got, want)


def off_boundary(t):
    """The same values in memory that starts one element behind a 16-byte boundary."""
    whole = torch.empty(t.numel() + 16, dtype=t.dtype, device=DEV)
    view = whole[1:1 + t.numel()].view(t.shape)
    return view.copy_(t)


@pytest.mark.parametrize("large", [False, True])
def test_matrices_off_a_16_byte_boundary_under_compile(ck, large):
    """They are copied there as in an eager call, not refused."""
    M, K, V, piece = (1500, 2048, 8195, 3000) if large else (24, 64, 72, 32)
    g = torch.Generator().manual_seed(0)
    x, w = (off_boundary(torch.randn(*s, generator=g).bfloat16().to(DEV)).requires_grad_(True) for s in ((M, K), (V, K)))
    assert x.data_ptr() % 16 and w.data_ptr() % 16
    target = torch.randint(0, V, (M,), generator=g, dtype=torch.int32).to(DEV)
    target[::3] = -100

    def f(x, w):
        return ck.linear_cross_entropy_pieces(x, w, target, piece=piece)

    want, got = f(x, w), torch.compile(f, fullgraph=True, dynamic=False)(x, w)
    assert torch.equal(want, got)
    for a, b in zip(torch.autograd.grad(want, (x, w)), torch.autograd.grad(got, (x, w))):
        assert torch.equal(a, b)
    if not large:
        q, s = ck.quantize_e4m3(x.detach())
        w8, ws = ck.quantize_e4m3(w.detach())
        q, w8 = (off_boundary(t.view(torch.uint8)).view(t.dtype) for t in (q, w8))
        with torch.no_grad():
            assert torch.equal(ck.linear_e4m3(q, s, w8, ws), torch.compile(ck.linear_e4m3, fullgraph=True, dynamic=False)(q, s, w8, ws))


def test_symbolic_trace_of_a_norm_step_runs_on_other_extents(ck):
    from torch.fx.experimental.proxy_tensor import make_fx

    rng = rng_state()

    def step(x, r, w):
        leaves = [t.detach().requires_grad_(True) for t in (x, r, w)]
        out, h = ck.add_rms_norm(*leaves, EPS, p=0.2, rng=rng)
        return [out.detach(), h.detach(), *torch.autograd.grad((out, h), leaves, (torch.ones_like(out), torch.ones_like(h)))]

    graph = make_fx(step, tracing_mode="symbolic", _allow_non_fake_inputs=True)(randn(24, 64), randn(24, 64, seed=1), randn(64, seed=2))
    for rows in (24, 7, 300):
        args = randn(rows, 64, seed=3), randn(rows, 64, seed=4), randn(64, seed=5)
        for a, b in zip(step(*args), graph(*args)):
            assert torch.equal(a, b)


def test_shapes_of_the_loss_are_refused_as_arguments(ck):
    """Whatever the number of dimensions, with a piece given."""
    x, v, t = randn(24, 64), randn(72, 64, seed=1), torch.zeros(24, dtype=torch.int32, device=DEV)
    for bad in ((x[0], v, t), (x, v[0], t), (x[None], v, t), (x, v[0, 0], t), (x[0, 0], v, t), (x, v, t[None])):
        for grad in (False, True):
            with pytest.raises(ValueError):
                ck.linear_cross_entropy_pieces(*(a.clone().requires_grad_(grad) for a in bad[:2]), bad[2], piece=32)
