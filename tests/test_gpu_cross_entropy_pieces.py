"""``linear_cross_entropy_pieces`` against the 64-bit definition and against ``linear_cross_entropy``.

Tolerances count roundings.  A logit is a K-term fp32 sum, 16 terms an instruction: off by at most
``(K / 16 + 2) * 2^-23`` times the sum of its terms' magnitudes (``zerr``).  The gradient of a logit moves by its
probability times that (twice: the log-sum-exp moves too), by 2^-20 of it for the exponential, and by half a bf16 step
(2^-8) of itself when it is stored; the products behind it sum those with fp32 errors of ``2^-18`` of their terms and
round once more to bf16.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = 2.0**-8
F32 = 2.0**-18


@pytest.fixture(scope="module")
def ck():
    import coda_kernels_b200 as ck

    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return ck


def make(M, K, V, ignored=0.2, seed=0, ignore_index=-100, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, K, generator=g) * scale).bfloat16().to(DEV)
    w = (torch.randn(V, K, generator=g) * K**-0.5).bfloat16().to(DEV)
    t = torch.randint(0, V, (M,), generator=g, dtype=torch.int32)
    t[torch.rand(M, generator=g) < ignored] = ignore_index
    return x.requires_grad_(True), w.requires_grad_(True), t.to(DEV)


def check(x, w, t, loss, dx, dw, reduction, dloss=1.0, ignore_index=-100):
    x64, w64, tl = x.detach().double(), w.detach().double(), t.long()
    K = x.shape[1]
    valid = tl != ignore_index
    z = x64 @ w64.T
    zerr = (K / 16 + 2) * 2.0**-23 * (x64.abs() @ w64.abs().T)
    lse = torch.logsumexp(z, 1, keepdim=True)
    label = torch.where(valid, tl, 0)[:, None]
    rows = (lse - z.gather(1, label))[:, 0]
    n = int(valid.sum())
    a = 1.0 / n if reduction == "mean" else 1.0
    want = (rows * valid).sum() * a
    row_err = 2 * zerr.amax(1) + 2.0**-20 * (1 + lse[:, 0].abs() + rows.abs())
    assert abs(float(loss.detach()) - float(want)) <= float((row_err * valid).sum() * a + F32 * (rows.abs() * valid).sum() * a)
    p = torch.exp(z - lse)
    g = p.clone()
    g.scatter_add_(1, label, torch.full_like(lse, -1.0))
    g, p = g * valid[:, None], p * valid[:, None]
    gerr = p * (2 * zerr + 2.0**-19) + BF * (g.abs() + p * (2 * zerr + 2.0**-19)) + 2.0**-126
    a = abs(a * dloss)
    for name, got, left, lerr, right in (("dx", dx, g, gerr, w64), ("dweight", dw, g.T, gerr.T, x64)):
        if got is None:
            continue
        ref = left @ right * (a if dloss > 0 else -a)
        bound = BF * ref.abs() + a * (lerr @ right.abs()) * (1 + BF) + a * F32 * (left.abs() @ right.abs()) + 2.0**-126
        err = (got.double() - ref).abs()
        assert bool((err <= bound).all()), f"{name}: worst excess {float((err - bound).max()):.3e}"


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("M,K,V,piece", [(1, 8, 1, None), (1, 64, 1000, None), (3, 72, 7, 2), (33, 128, 517, 100), (130, 264, 1003, 256),
                                         (257, 1032, 3001, 777), (300, 64, 4099, 4098), (512, 512, 2048, 1024)])
def test_pieces_against_the_definition(ck, M, K, V, piece, reduction):
    x, w, t = make(M, K, V, ignored=0.2 if M > 1 else 0.0)
    loss = ck.linear_cross_entropy_pieces(x, w, t, reduction=reduction, piece=piece)
    dx, dw = torch.autograd.grad(loss, (x, w), torch.tensor(-1.5, device=DEV))
    assert loss.dtype == torch.float32 and loss.dim() == 0 and dx.dtype == dw.dtype == torch.bfloat16
    check(x, w, t, loss, dx, dw, reduction, dloss=-1.5)
    ck.ops.check_device_status(torch.device(DEV))


def test_steep_rows_and_labels_at_the_ends(ck):
    """Logits far apart (a probability of nearly one), labels at both ends of a piece, ignore_index inside the range."""
    x, w, t = make(64, 128, 1024, ignored=0.0, scale=30.0)
    t[:8] = torch.tensor([0, 255, 256, 511, 512, 767, 1022, 1023], dtype=torch.int32, device=DEV)
    t[8:12] = 5
    loss = ck.linear_cross_entropy_pieces(x, w, t, ignore_index=5, reduction="mean", piece=256)
    dx, dw = torch.autograd.grad(loss, (x, w))
    check(x, w, t, loss, dx, dw, "mean", ignore_index=5)
    assert not bool(dx[8:12].any())


def test_matches_the_stored_form(ck):
    """Same loss as linear_cross_entropy to fp32 rounding (its tiles are the same sums), whatever the piece."""
    x, w, t = make(200, 256, 1024)
    a = ck.linear_cross_entropy(x, w, t)
    losses = [ck.linear_cross_entropy_pieces(x, w, t, piece=p) for p in (None, 128, 1000)]
    for b in losses:
        assert abs(float((a - b).detach())) <= 2.0**-20 * abs(float(a.detach()))
        assert torch.equal(b, losses[0])
    # one piece or many: dweight is the same product; dx differs by the order of an fp32 sum
    (g1, g2, g3) = (torch.autograd.grad(v, (x, w)) for v in losses)
    assert torch.equal(g1[1], g3[1]) and torch.equal(g1[1], g2[1])


def test_masks_that_leave_nothing(ck):
    x, w, t = make(5, 64, 300)
    t[:] = -100
    loss = ck.linear_cross_entropy_pieces(x, w, t, reduction="sum", piece=100)
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert float(loss.detach()) == 0.0 and not bool(dx.any()) and not bool(dw.any())
    assert bool(ck.linear_cross_entropy_pieces(x, w, t).isnan())
    empty = ck.linear_cross_entropy_pieces(x[:0], w, t[:0], reduction="sum")
    dx, dw = torch.autograd.grad(empty, (x, w), allow_unused=True)
    assert float(empty.detach()) == 0.0 and not bool(dw.any())
    assert bool(ck.linear_cross_entropy_pieces(x[:0], w, t[:0]).isnan())


def test_label_outside_the_vocabulary_is_loud(ck):
    x, w, t = make(4, 64, 300, ignored=0.0)
    t[2] = 300
    assert bool(ck.linear_cross_entropy_pieces(x, w, t).isnan())
    t[2] = -1
    assert bool(ck.linear_cross_entropy_pieces(x, w, t).isnan())


def test_ignored_rows_may_hold_anything_for_the_loss_and_dx(ck):
    x, w, t = make(40, 64, 300, ignored=0.0)
    t[7] = -100
    clean = ck.linear_cross_entropy_pieces(x, w, t, piece=128)
    (dx,) = torch.autograd.grad(clean, x)
    bad = x.detach().clone()
    bad[7, 3], bad[7, 9] = float("nan"), float("inf")
    bad.requires_grad_(True)
    loss = ck.linear_cross_entropy_pieces(bad, w, t, piece=128)
    (dbad,) = torch.autograd.grad(loss, bad)
    assert torch.equal(loss, clean) and torch.equal(dx, dbad)


def test_partial_gradients_views_and_streams(ck):
    x, w, t = make(100, 128, 700)
    loss = ck.linear_cross_entropy_pieces(x, w, t, piece=256)
    dx, dw = torch.autograd.grad(loss, (x, w))
    (only_x,) = torch.autograd.grad(ck.linear_cross_entropy_pieces(x, w.detach(), t, piece=256), x)
    (only_w,) = torch.autograd.grad(ck.linear_cross_entropy_pieces(x.detach(), w, t, piece=256), w)
    assert torch.equal(only_x, dx) and torch.equal(only_w, dw)
    xt = x.detach().t().contiguous().t().requires_grad_(True)  # column-major rows
    tt = torch.stack((t, t), 1)[:, 0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss2 = ck.linear_cross_entropy_pieces(xt, w, tt, piece=256)
        dx2, dw2 = torch.autograd.grad(loss2, (xt, w))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(loss, loss2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)


def test_captured_step_replays_on_new_inputs(ck):
    x, w, t = make(96, 128, 700)
    # (no eager graph of these leaves is kept: their gradient nodes would tie the capture to the stream of that graph,
    # which PyTorch answers with an invalidated capture for any operator)

    def step():
        loss = ck.linear_cross_entropy_pieces(x, w, t, piece=300)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    x2, w2, t2 = make(96, 128, 700, seed=5, ignored=0.5)
    with torch.no_grad():
        x.copy_(x2), w.copy_(w2), t.copy_(t2)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(static, step()):
        assert torch.equal(a, b)


def test_memory_stays_bounded(ck):
    """Nothing of size M x V: the peak above the inputs and gradients is the piece buffer, dx in fp32 and the tiles' partials."""
    M, K, V, piece = 4096, 128, 65536, 4096
    x, w, t = make(M, K, V)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = ck.linear_cross_entropy_pieces(x, w, t, piece=piece)
    grads = torch.autograd.grad(loss, (x, w))
    torch.cuda.synchronize()
    own = M * piece * 2 + M * K * 4 + 2 * M * (V // 256) * 4 + sum(g.numel() * 2 for g in grads)
    workspace = 64 << 20  # a GEMM's split tail
    assert torch.cuda.max_memory_allocated() - before <= own + workspace < M * V * 2


def test_refusals(ck):
    x, w, t = make(8, 64, 100)
    with pytest.raises(AssertionError):
        ck.linear_cross_entropy_pieces(x, w, t.long())
    with pytest.raises(AssertionError):
        ck.linear_cross_entropy_pieces(x, w, t, reduction="none")
    for bad in (lambda: ck.linear_cross_entropy_pieces(x, w[:, :32], t), lambda: ck.linear_cross_entropy_pieces(x, w, t[:7]),
                lambda: ck.linear_cross_entropy_pieces(x[:, :60], w[:, :60], t), lambda: ck.linear_cross_entropy_pieces(x, w, t, piece=0),
                lambda: ck.linear_cross_entropy_pieces(x, w, t.cpu()), lambda: ck.linear_cross_entropy_pieces(x, w[:0], t),
                lambda: ck.linear_cross_entropy_pieces(x, w, t, ignore_index=2**31)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        ck.linear_cross_entropy_pieces(x.float(), w.float(), t)


def test_under_compile(ck):
    x, w, t = make(64, 128, 520)

    def f(x, w, t):
        return ck.linear_cross_entropy_pieces(x, w, t, piece=256)

    loss = torch.compile(f, fullgraph=True, dynamic=False)(x, w, t)
    dx, dw = torch.autograd.grad(loss, (x, w))
    check(x, w, t, loss, dx, dw, "mean")


@pytest.mark.parametrize("option,value,default", [("epi_tma", 0, 1), ("cta_group", 1, 2), ("split_tail", 0, 1)])
def test_library_options_leave_the_result(ck, option, value, default):
    """Whatever the stores, the grouping and the schedule, the definition decides."""
    x, w, t = make(300, 136, 1003)
    ck.set_option(option, value)
    try:
        loss = ck.linear_cross_entropy_pieces(x, w, t, piece=300)
        dx, dw = torch.autograd.grad(loss, (x, w))
        torch.cuda.synchronize()
    finally:
        ck.set_option(option, default)
    check(x, w, t, loss, dx, dw, "mean")


def test_second_derivative_is_refused(ck):
    x, w, t = make(20, 64, 300)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(ck.linear_cross_entropy_pieces(x, w, t), x, create_graph=True)


# ------------------------------------------------------------------------------------------------ ignored rows left out
# Large enough for the rows that count to be put together first (2 M V K >= 5e10, V >= 8192).
def large(M=1500, K=2048, V=8195, **kw):
    from coda_kernels_b200._lib import lib

    assert lib.coda_b200_ce_compacts(M, V, K) == 1
    return make(M, K, V, **kw)


@pytest.mark.parametrize("ignored", [0.0, 0.05, 0.6, 0.99])
@pytest.mark.parametrize("M,K,V,piece", [(1500, 2048, 8195, 3000), (65, 4096, 100003, None), (4100, 776, 8200, None)])
def test_counted_rows_against_the_definition(ck, M, K, V, piece, ignored):
    x, w, t = large(M, K, V, ignored=ignored)
    loss = ck.linear_cross_entropy_pieces(x, w, t, piece=piece)
    dx, dw = torch.autograd.grad(loss, (x, w))
    check(x, w, t, loss, dx, dw, "mean")
    assert not bool(dx[t == -100].any())
    with torch.no_grad():
        assert torch.equal(loss, ck.linear_cross_entropy_pieces(x, w, t))
    ck.ops.check_device_status(torch.device(DEV))


@pytest.mark.parametrize("kept", [[], [0], [1499], list(range(64)), list(range(700, 765)), list(range(0, 1500, 7))])
def test_counted_rows_at_the_edges(ck, kept):
    x, w, t = large(ignored=0.0)
    mask = torch.ones(1500, dtype=torch.bool, device=DEV)
    mask[kept] = False
    t = torch.where(mask, torch.full_like(t, -100), t)
    loss = ck.linear_cross_entropy_pieces(x, w, t, reduction="sum", piece=3000)
    dx, dw = torch.autograd.grad(loss, (x, w))
    check(x, w, t, loss, dx, dw, "sum")
    if not kept:
        assert float(loss.detach()) == 0.0 and not bool(dx.any()) and not bool(dw.any())


def test_ignored_rows_are_not_read_by_the_products(ck):
    x, w, t = large(ignored=0.3)
    clean = ck.linear_cross_entropy_pieces(x, w, t, piece=5000)
    grads = torch.autograd.grad(clean, (x, w))
    bad = x.detach().clone()
    bad[t == -100] = float("nan")
    bad.requires_grad_(True)
    loss = ck.linear_cross_entropy_pieces(bad, w, t, piece=5000)
    assert torch.equal(loss, clean)
    for a, b in zip(torch.autograd.grad(loss, (bad, w)), grads):
        assert torch.equal(a, b)


def test_counted_rows_follow_the_labels_of_a_replay(ck):
    """The number of rows that count is read on the device: a captured step takes other masks than it was captured with."""
    x, w, t = large(ignored=0.5)

    def step():
        loss = ck.linear_cross_entropy_pieces(x, w, t, piece=3000)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for seed, ignored in ((5, 0.0), (6, 0.95), (7, 0.2)):
        _, _, t2 = large(ignored=ignored, seed=seed)
        t.copy_(t2)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(static, step()):
            assert torch.equal(a, b)


def test_counted_rows_in_both_bindings_and_with_partial_gradients(ck):
    from importlib import import_module

    node = import_module("coda_kernels_b200.functional.cross_entropy_pieces").LinearCrossEntropyPieces
    x, w, t = large(ignored=0.3)
    loss = ck.linear_cross_entropy_pieces(x, w, t, piece=5000)
    dx, dw = torch.autograd.grad(loss, (x, w))
    other = node.apply(x, w, t, -100, "mean", 5000)
    for a, b in zip((loss, dx, dw), (other, *torch.autograd.grad(other, (x, w)))):
        assert torch.equal(a, b)
    (only_x,) = torch.autograd.grad(ck.linear_cross_entropy_pieces(x, w.detach(), t, piece=5000), x)
    (only_w,) = torch.autograd.grad(ck.linear_cross_entropy_pieces(x.detach(), w, t, piece=5000), w)
    assert torch.equal(only_x, dx) and torch.equal(only_w, dw)
    # with one CTA a tile, or by option, all rows take part: the definition decides
    for option, value, default in (("cta_group", 1, 2), ("ce_compact", 0, 1)):
        ck.set_option(option, value)
        try:
            loss = ck.linear_cross_entropy_pieces(x, w, t, piece=5000)
            grads = torch.autograd.grad(loss, (x, w))
            torch.cuda.synchronize()
        finally:
            ck.set_option(option, default)
        check(x, w, t, loss, *grads, "mean")
