"""``linear_cross_entropy_pieces`` where labels are missing or wrong: gradients of a batch without a label, labels outside the
vocabulary, ignored rows that hold anything; traced programs, and what is held between forward and backward.  Each at a size
whose products run over all rows and at one where the rows that count are put first, through the compiled operators and
through the Python nodes."""

from importlib import import_module

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SIZES = [(40, 64, 300, 128), (1500, 2048, 8195, 3000)]  # rows, dim, vocabulary, piece: all rows; the rows that count


@pytest.fixture(scope="module")
def ck():
    import coda_kernels_b200 as ck

    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return ck


def make(M, K, V, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).bfloat16().to(DEV).requires_grad_(True)
    w = (torch.randn(V, K, generator=g) * K**-0.5).bfloat16().to(DEV).requires_grad_(True)
    return x, w, torch.randint(0, V, (M,), generator=g, dtype=torch.int32).to(DEV)


def loss_of(ck, binding):
    if binding == "compiled":
        return lambda x, w, t, reduction, piece: ck.linear_cross_entropy_pieces(x, w, t, reduction=reduction, piece=piece)
    node = import_module("coda_kernels_b200.functional.cross_entropy_pieces").LinearCrossEntropyPieces
    return lambda x, w, t, reduction, piece: node.apply(x, w, t, -100, reduction, piece)


@pytest.mark.parametrize("binding", ["compiled", "python"])
@pytest.mark.parametrize("M,K,V,piece", SIZES)
def test_no_label_counts(ck, M, K, V, piece, binding):
    """The mean over nothing is NaN, and its gradients are zeros, as those of torch's own cross entropy: a fully masked
    micro-batch adds nothing to the accumulated gradients."""
    assert ck._lib.lib.coda_b200_ce_compacts(M, V, K) == (M > 1000)
    x, w, t = make(M, K, V)
    loss = loss_of(ck, binding)(x, w, torch.full_like(t, -100), "mean", piece)
    assert bool(loss.isnan())
    dx, dw = torch.autograd.grad(loss, (x, w), torch.tensor(0.25, device=DEV))
    assert torch.equal(dx, torch.zeros_like(dx)) and torch.equal(dw, torch.zeros_like(dw))
    total = loss_of(ck, binding)(x, w, torch.full_like(t, -100), "sum", piece)
    assert float(total.detach()) == 0.0
    for g in torch.autograd.grad(total / 0.0, (x, w)):  # a sum divided by the number of labels
        assert not bool(g.any())
    logits = (x.detach().float() @ w.detach().float().T).requires_grad_(True)
    torch.nn.functional.cross_entropy(logits, torch.full_like(t, -100).long()).backward()
    assert not bool(logits.grad.any())  # what is meant by "as those of torch's own"


@pytest.mark.parametrize("binding", ["compiled", "python"])
@pytest.mark.parametrize("label", [-1, -2**31, 2**31 - 1, "V"])
@pytest.mark.parametrize("M,K,V,piece", SIZES)
def test_label_outside_the_vocabulary_reaches_the_gradients(ck, M, K, V, piece, label, binding):
    """The loss is NaN, and so are the row's dx and all of dweight: a program that does not look at the loss sees it there.
    The other rows' dx is what it is with a label in its place."""
    x, w, t = make(M, K, V)
    t[1] = -100
    good = loss_of(ck, binding)(x, w, t, "sum", piece)
    (dx_good,) = torch.autograd.grad(good, x)
    t2 = t.clone()
    t2[2] = V if label == "V" else label
    loss = loss_of(ck, binding)(x, w, t2, "sum", piece)
    assert bool(loss.isnan())
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert bool(dx[2].isnan().all()) and bool(dw.isnan().all())
    rows = [i for i in range(M) if i != 2]
    assert torch.equal(dx[rows], dx_good[rows])


@pytest.mark.parametrize("binding", ["compiled", "python"])
@pytest.mark.parametrize("M,K,V,piece", SIZES)
def test_ignored_rows_may_hold_anything(ck, M, K, V, piece, binding):
    """Rows whose label is ignored take no part in loss, dx or dweight, whatever they hold, at every size."""
    x, w, t = make(M, K, V)
    t[5:9] = -100
    t[M - 1] = -100
    fn = loss_of(ck, binding)
    clean = fn(x, w, t, "mean", piece)
    grads = torch.autograd.grad(clean, (x, w))
    bad = x.detach().clone()
    bad[5], bad[6, 3], bad[M - 1] = float("nan"), float("inf"), float("-inf")
    bad.requires_grad_(True)
    loss = fn(bad, w, t, "mean", piece)
    assert torch.equal(loss, clean)
    for a, b in zip(torch.autograd.grad(loss, (bad, w)), grads):
        assert torch.equal(a, b)
    assert not bool(grads[0][t == -100].any())
    # the weight's gradient alone, and an x that needs none
    loss = fn(bad.detach(), w, t, "mean", piece)
    assert torch.equal(torch.autograd.grad(loss, w)[0], grads[1])


def test_compiled_program_leaves_ignored_rows_out(ck):
    """Traced, the loss takes the same rows into its products as an eager call does: the same bits, and ignored rows may hold
    anything."""
    M, K, V, piece = SIZES[1]
    x, w, t = make(M, K, V)
    t[torch.rand(M, generator=torch.Generator().manual_seed(1)).to(DEV) < 0.4] = -100

    def step(x, w, t):
        return ck.linear_cross_entropy_pieces(x, w, t, piece=piece)

    eager = step(x, w, t)
    want = (eager.detach(), *torch.autograd.grad(eager, (x, w)))
    bad = torch.where((t == -100)[:, None], torch.full_like(x, float("nan")), x.detach()).requires_grad_(True)
    traced = torch.compile(step, fullgraph=True, dynamic=False)
    for rows in (x, bad):
        loss = traced(rows, w, t)
        for a, b in zip((loss.detach(), *torch.autograd.grad(loss, (rows, w))), want):
            assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(traced(bad, w, t), want[0])
    # labels of another call
    t2 = t.roll(7)
    loss, plain = traced(x, w, t2), step(x, w, t2)
    for a, b in zip(torch.autograd.grad(loss, (x, w)), torch.autograd.grad(plain, (x, w))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("binding", ["compiled", "python"])
def test_memory_held_between_forward_and_backward(ck, binding):
    """Beside what the caller holds, and with the rows that count put first for the products: log-sum-exp, labels and positions,
    4 bytes a row each, no copy of the rows (33.5 MB here)."""
    M, K, V, piece = 4096, 4096, 8200, 4096
    assert ck._lib.lib.coda_b200_ce_compacts(M, V, K) == 1
    x, w, t = make(M, K, V)
    t[::5] = -100
    fn = loss_of(ck, binding)
    torch.autograd.grad(fn(x, w, t, "mean", piece), (x, w))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    loss = fn(x, w, t, "mean", piece)
    held = torch.cuda.memory_allocated() - before
    assert held <= 12 * M + 4096, held  # (the allocator rounds each of five tensors up to 512 bytes)
    torch.autograd.grad(loss, (x, w))
