"""The operators between token ids and a model against their formulas in 64 bits, on a B200.

How far a result may be off is counted from roundings: u = eps / 2 of a type is half a step relative to the value.  A sum of tensor-core
products loses at most a step of fp32 (2^-23) of its largest partial sum every 16 elements."""
import math
import threading

import pytest
import torch

from conftest import tiny_vocab

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops(built):
    from graphtok_b200 import vocab_ops
    return vocab_ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def half_step(t):
    return torch.finfo(t).eps / 2


def within(got, want, tol, what=""):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    off = torch.nan_to_num((got - want).abs()) - tol
    assert got.numel() == 0 or off.max().item() <= 0, "%s off by %g more than the bound (largest error %g)" % (
        what, off.max().item(), torch.nan_to_num((got - want).abs()).max().item())


# ---- losses -----------------------------------------------------------------------
def wanted_of_targets(targets, vocab, ignore=-100):
    rows = ((targets >= 0) & (targets != ignore)).nonzero().squeeze(1)
    q = torch.zeros(targets.numel(), vocab, dtype=torch.float64, device="cuda")
    q[rows, targets[rows].long()] = 1.0
    return q, torch.zeros(targets.numel(), dtype=torch.float64, device="cuda")


def wanted_of_teacher(ids, logits, vocab, temperature):
    """(what the softmax should be, sum of q log q over the entries)"""
    l = torch.where(ids >= 0, logits.double() / temperature, -math.inf)
    top = l.max(1, keepdim=True).values
    e = torch.where(torch.isinf(top), 0.0, torch.exp(l - torch.where(torch.isinf(top), 0.0, top)))
    share = e / e.sum(1, keepdim=True).clamp(min=1e-300)
    q = torch.zeros(ids.shape[0], vocab, dtype=torch.float64, device="cuda")
    q.scatter_add_(1, ids.long().clamp(min=0), share)
    return q, torch.xlogy(share, share).sum(1)


class Reference:
    """Losses and gradients of rows with weights `g`, and how far 32-bit sums and 16-bit dZ may take them."""

    def __init__(self, hidden, weight, q, entropy, g, temperature=1.0):
        u = half_step(hidden.dtype)
        h, w, t = hidden.double(), weight.double(), temperature
        vocab, width = w.shape
        active = q.sum(1) > 0
        h = torch.where(active[:, None], h, 0.0)
        z = h @ w.T / t
        # a logit: a step of its largest partial sum each 16 elements, of which the sum of magnitudes is more
        dz = ((width + 15) // 16 + 2) * 2.0 ** -23 * (h.abs() @ w.abs().T / t).max(1).values
        self.lse = torch.where(active, torch.logsumexp(z, 1), 0.0)
        self.losses = torch.where(active, entropy - (q * z).sum(1) + self.lse, 0.0)
        size = self.lse.abs() + (q * z.abs()).sum(1) + entropy.abs() + 1
        # logsumexp moves by no more than its logits; exp2, log and the sums over tiles take some steps of their own
        self.lse_tol = dz + 16 * 2.0 ** -24 * (self.lse.abs() + 1)
        self.loss_tol = 2 * dz + 32 * 2.0 ** -24 * size
        p = torch.softmax(z, 1) * active[:, None]
        gt = (g * active).abs()[:, None] / t
        d = (p - q) * (g * active)[:, None] / t
        # of dZ: p by its exponent (logit, lse and their products), the difference by one step of fp32, and its 16 bits
        dp = p * gt * ((dz + self.lse_tol)[:, None] + 2.0 ** -20 * (1 + z.abs()))
        dd = dp + (p + q) * gt * 2.0 ** -22 + d.abs() * u
        if hidden.dtype == F16:
            dd = dd + 2.0 ** -24 / 32768 * gt.max()              # the least that fp16 holds, at the scale that dZ has
        self.d_hidden, self.d_weight = d @ w, d.T @ h
        least = 2.0 ** -25 if hidden.dtype == F16 else 0.0
        pieces = 2.0 ** -23 * 40                                    # sums over pieces and splits, scale factors
        self.h_tol = dd @ w.abs() + (d.abs() @ w.abs()) * ((vocab + 15) // 16 * 2.0 ** -23 + pieces) + self.d_hidden.abs() * u * 1.01 + least
        self.w_tol = dd.T @ h.abs() + (d.abs().T @ h.abs()) * ((h.shape[0] + 15) // 16 * 2.0 ** -23 + pieces) + self.d_weight.abs() * u * 1.01 + least

    def check(self, losses, lse, d_hidden=None, d_weight=None):
        within(losses, self.losses, self.loss_tol, "losses")
        if lse is not None:
            within(lse, self.lse, self.lse_tol, "lse")
        if d_hidden is not None:
            within(d_hidden, self.d_hidden, self.h_tol, "d_hidden")
        if d_weight is not None:
            within(d_weight, self.d_weight, self.w_tol, "d_weight")


def make(seed, n, vocab, width, dtype, masked=0.25):
    g = gen(seed)
    weight = (randn(g, vocab, width) * (2.0 / math.sqrt(width))).to(dtype)
    targets = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    hidden = (randn(g, n, width) + torch.rand(n, 1, generator=g, device="cuda") * 2 * weight[targets].float()).to(dtype)
    if masked:
        targets[torch.rand(n, generator=g, device="cuda") < masked] = -100
    return hidden, weight, targets, torch.rand(n, generator=g, device="cuda") + 0.1


SHAPES = [(1, 1, 1), (1, 2, 8), (2, 255, 7), (3, 256, 64), (127, 257, 65), (128, 1000, 200), (129, 300, 72), (255, 31, 130), (256, 513, 256), (257, 2049, 264), (513, 5003, 520),
          (1000, 777, 1), (16, 40001, 136), (17, 19000, 64), (33, 18945, 200), (48, 300, 64), (63, 5000, 72), (64, 38000, 264), (65, 38000, 128)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,vocab,width", SHAPES)
def test_cross_entropy(ops, n, vocab, width, dtype):
    hidden, weight, targets, g = make(n + vocab, n, vocab, width, dtype)
    ref = Reference(hidden, weight, *wanted_of_targets(targets, vocab), g.double())
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets)
    d_hidden, d_weight = ops.cross_entropy_grad(hidden, weight, targets, lse, g)
    ref.check(losses, lse, d_hidden, d_weight)


@pytest.mark.parametrize("temperature", [0.5, 3.0])
def test_cross_entropy_with_a_temperature(ops, temperature):
    hidden, weight, targets, g = make(5, 300, 1500, 192, BF16)
    ref = Reference(hidden, weight, *wanted_of_targets(targets, 1500), g.double(), temperature)
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets, temperature=temperature)
    ref.check(losses, lse, *ops.cross_entropy_grad(hidden, weight, targets, lse, g, temperature=temperature))


@pytest.mark.parametrize("n,vocab,width,kept", [(4096, 70000, 64, 1500), (64, 50000, 72, None), (131072, 56 * 256 + 1, 64, 300), (3000, 9000, 264, 40)])
def test_pieces_splits_and_few_active_rows(ops, n, vocab, width, kept):
    """A vocabulary in several pieces; a hidden gradient in many splits; a last piece with fewer columns than splits; rows that are left out."""
    hidden, weight, targets, g = make(n, n, vocab, width, BF16, masked=0.1 if kept is None else 0)
    if kept is not None:
        some = torch.randperm(n, generator=gen(1), device="cuda")[:kept]
        left = torch.full_like(targets, -100)
        left[some] = targets[some]
        targets = left
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets)
    d_hidden, d_weight = ops.cross_entropy_grad(hidden, weight, targets, lse, g)
    rows = (targets >= 0).nonzero().squeeze(1)
    ref = Reference(hidden[rows], weight, *wanted_of_targets(targets[rows], vocab), g[rows].double())
    ref.check(losses[rows], lse[rows], d_hidden[rows], d_weight)
    others = targets < 0
    assert losses[others].eq(0).all() and lse[others].eq(0).all() and d_hidden[others].eq(0).all()


@pytest.mark.parametrize("n", [20, 70])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_that_are_all_masked(ops, dtype, n):
    hidden, weight, targets, g = make(3, n, 600, 96, dtype)
    targets[:] = -100
    hidden[:] = float("nan")
    for reduction, shape in (("none", (n,)), ("mean", ()), ("sum", ())):
        loss, lse = ops.cross_entropy_forward(hidden, weight, targets, reduction=reduction)
        assert loss.shape == shape and loss.eq(0).all()
        grads = ops.cross_entropy_grad(hidden, weight, targets, lse, torch.ones(shape, device="cuda"), reduction=reduction)
        assert all(x.eq(0).all() for x in grads)
    odd = weight[:, :95].contiguous()
    assert ops.cross_entropy_grad(hidden[:, :95].contiguous(), odd, targets, lse, g)[1].eq(0).all()


@pytest.mark.parametrize("n", [50, 400])
def test_nothing_of_masked_rows_is_seen(ops, n):
    hidden, weight, targets, g = make(4, n, 900, 128, BF16, masked=0.4)
    masked = targets < 0
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets)
    grads = ops.cross_entropy_grad(hidden, weight, targets, lse, g)
    for value in (float("nan"), float("inf"), torch.finfo(BF16).min):
        other, og = hidden.clone(), g.clone()
        other[masked] = value
        og[masked] = float("nan")
        l2, s2 = ops.cross_entropy_forward(other, weight, targets)
        assert torch.equal(l2, losses) and torch.equal(s2, lse)
        assert all(torch.equal(a, b) for a, b in zip(ops.cross_entropy_grad(other, weight, targets, lse, og), grads))


@pytest.mark.parametrize("n", [30, 200])
def test_nan_and_far_logits(ops, n):
    hidden, weight, targets, g = make(6, n, 700, 64, BF16, masked=0)
    hidden[17] = float("nan")
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets)
    rest = torch.arange(n, device="cuda") != 17
    assert losses[17].isnan() and lse[17].isnan() and losses[rest].isfinite().all()
    d_hidden, d_weight = ops.cross_entropy_grad(hidden, weight, targets, lse, g)
    assert d_hidden[17].isnan().all() and d_hidden[rest].isfinite().all() and d_weight.isnan().all()
    # logits of tens of thousands, of which one is left
    hidden[17] = 0
    hidden *= 8192
    ref = Reference(hidden, weight, *wanted_of_targets(targets, 700), g.double())
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets)
    ref.check(losses, lse)
    # a table with a row of the lowest value and one of infinities that no hidden state reaches
    hidden, weight, targets, g = make(7, n, 513, 64, BF16, masked=0)
    hidden = hidden.abs()
    weight[512] = torch.finfo(BF16).min
    weight[7] = -float("inf")
    targets[(targets == 512) | (targets == 7)] = 0
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets)
    finite = weight.clone()
    finite[512] = finite[7] = 0
    keep = torch.ones(513, dtype=torch.bool, device="cuda")
    keep[512] = keep[7] = False
    z = hidden.double() @ weight[keep].double().T
    assert (lse.double() - z.logsumexp(1)).abs().max() <= Reference(hidden, finite, *wanted_of_targets(targets, 513), g.double()).lse_tol.max()


@pytest.mark.parametrize("n", [60, 100])
def test_targets_beyond_the_vocabulary(ops, n):
    hidden, weight, targets, g = make(8, n, 300, 64, BF16, masked=0)
    good, lse = ops.cross_entropy_forward(hidden, weight, targets)
    for bad in (300, 2 ** 31 - 1, 2 ** 40):
        wrong = targets.clone()
        wrong[[3, n - 1]] = bad
        losses, lse = ops.cross_entropy_forward(hidden, weight, wrong)
        assert losses[[3, n - 1]].isnan().all() and torch.equal(losses[4:n - 1], good[4:n - 1])
        assert ops.cross_entropy_forward(hidden, weight, wrong, reduction="mean")[0].isnan()
        wrong_grads = ops.cross_entropy_grad(hidden, weight, wrong, lse, g)
        wrong[[3, n - 1]] = -100
        assert all(torch.equal(a, b) for a, b in zip(wrong_grads, ops.cross_entropy_grad(hidden, weight, wrong, lse, g)))
    # an ignored id inside the vocabulary, and other negative ids
    targets[5], targets[6] = 7, -1
    losses, _ = ops.cross_entropy_forward(hidden, weight, targets, ignore_index=7)
    assert losses[(targets == 7) | (targets < 0)].eq(0).all()


def layouts(x):
    """The same values in other layouts."""
    n, width = x.shape
    wide = torch.zeros(n, width + 13, dtype=x.dtype, device=x.device)
    wide[:, 5:5 + width] = x
    yield wide[:, 5:5 + width]                       # lines that begin anywhere
    even = torch.zeros(n, width + 24, dtype=x.dtype, device=x.device)
    even[:, 8:8 + width] = x
    yield even[:, 8:8 + width]
    yield x.t().contiguous().t()                     # columns together
    twice = torch.zeros(2 * n, width, dtype=x.dtype, device=x.device)
    twice[::2] = x
    yield twice[::2]


@pytest.mark.parametrize("width", [64, 100])
def test_layouts_and_shapes(ops, width):
    hidden, weight, targets, g = make(9, 150, 400, width, F16)
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets)
    grads = ops.cross_entropy_grad(hidden, weight, targets, lse, g)
    for h, w in zip(layouts(hidden), layouts(weight)):
        l2, s2 = ops.cross_entropy_forward(h, w, targets)
        assert torch.equal(l2, losses) and torch.equal(s2, lse)
        assert all(torch.equal(a, b) for a, b in zip(ops.cross_entropy_grad(h, w, targets, lse, g), grads))
    l3, s3 = ops.cross_entropy_forward(hidden.view(3, 50, width), weight, targets.view(3, 50).int())
    assert l3.shape == s3.shape == (3, 50) and torch.equal(l3.flatten(), losses)
    d_hidden, d_weight = ops.cross_entropy_grad(hidden.view(3, 50, width), weight, targets.view(3, 50).t().contiguous().t(), s3, g.view(3, 50))
    assert torch.equal(d_hidden.view(150, width), grads[0]) and torch.equal(d_weight, grads[1])
    one = hidden[:1].expand(150, width)              # a row that all positions share
    assert torch.equal(ops.cross_entropy_forward(one, weight, targets)[0], ops.cross_entropy_forward(one.contiguous(), weight, targets)[0])


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("keep", [False, True])
def test_a_calls_memory_is_apart(ops, reduction, keep):
    """What a forward pass writes lies in tensors that live until it is queued, and none of it over another."""
    for n in (1, 50, 700):
        hidden, weight, targets, _ = make(13, n, 900, 64, BF16)
        call = ops._Call(hidden, weight, targets, None, -100, 1.0)
        result, lse = call.forward(reduction, keep=keep, want_lse=not keep)
        a = call.args
        spans = [(a.losses, 4 * n), (a.lse, 4 * n), (a.workspace, a.workspace_bytes)] + [(a.kept, a.kept_bytes)] * keep + [(a.total, 4)] * (reduction != "none")
        spans.sort()
        assert all(x + size <= y for (x, size), (y, _) in zip(spans, spans[1:]))
        owners = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in (result, lse, call.work, getattr(call, "kept", None)) if t is not None]
        assert all(any(lo <= at and at + size <= hi for lo, hi in owners) for at, size in spans)


def test_no_rows(ops):
    hidden, weight = torch.zeros(0, 64, dtype=BF16, device="cuda"), torch.ones(300, 64, dtype=BF16, device="cuda")
    targets = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert ops.cross_entropy(hidden, weight, targets) == 0 and ops.cross_entropy(hidden, weight, targets, reduction="none").shape == (0,)
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets)
    d_hidden, d_weight = ops.cross_entropy_grad(hidden, weight, targets, lse, losses)
    assert d_hidden.shape == (0, 64) and d_weight.eq(0).all()


@pytest.mark.parametrize("factor", [0.0, 1e-42, 1e-20, 1e20])
def test_gradients_of_any_size(ops, factor):
    """The losses' gradients are scaled to 1 on their way; with all of them 0, or next to it, nothing overflows there."""
    hidden, weight, targets, g = make(12, 50, 300, 64, BF16)
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets)
    d_hidden, d_weight = ops.cross_entropy_grad(hidden, weight, targets, lse, g * factor)
    ref = Reference(hidden, weight, *wanted_of_targets(targets, 300), (g * factor).double())
    least = 2.0 ** -126 * 64                # below the least normal number results may be 0
    within(d_hidden, ref.d_hidden, ref.h_tol + least)
    within(d_weight, ref.d_weight, ref.w_tol + least)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_autograd(ops, reduction):
    hidden, weight, targets, g = make(10, 260, 1000, 128, BF16)
    hidden, weight = hidden.requires_grad_(), weight.requires_grad_()
    count = (targets >= 0).sum()
    loss = ops.cross_entropy(hidden, weight, targets, reduction=reduction)
    if reduction == "none":
        weights = g.double()
        (loss * g).sum().backward()
    else:
        weights = torch.full_like(g, 2.5, dtype=torch.float64) / (count if reduction == "mean" else 1)
        (loss * 2.5).backward()
    ref = Reference(hidden.detach(), weight.detach(), *wanted_of_targets(targets, 1000), weights)
    within(hidden.grad, ref.d_hidden, ref.h_tol, "d_hidden")
    within(weight.grad, ref.d_weight, ref.w_tol, "d_weight")
    total = ref.losses.sum() / (count if reduction == "mean" else 1)
    if reduction != "none":
        tol = ref.loss_tol.sum() / (count if reduction == "mean" else 1) + 40 * 2.0 ** -24 * ref.losses.abs().sum()
        within(loss.detach(), total, tol, "loss")
    # one of the two alone, and a gradient that is the same for all rows
    h = hidden.detach().requires_grad_()
    ops.cross_entropy(h, weight.detach(), targets, reduction=reduction).sum().backward()
    w = weight.detach().requires_grad_()
    ops.cross_entropy(hidden.detach(), w, targets, reduction=reduction).sum().backward()
    ref = Reference(hidden.detach(), weight.detach(), *wanted_of_targets(targets, 1000), torch.full_like(g, 1.0, dtype=torch.float64) / (count if reduction == "mean" else 1))
    within(h.grad, ref.d_hidden, ref.h_tol, "d_hidden")
    within(w.grad, ref.d_weight, ref.w_tol, "d_weight")


def test_gradients_by_differences(ops):
    """The losses at two places on a line through the inputs differ by the gradient along it, up to the third derivative: of logsumexp that is at
    most twice the third power of the logits' range along the line."""
    g = gen(11)
    hidden, weight, targets, _ = make(11, 96, 700, 64, BF16)
    hidden, weight = (hidden * 4).round() / 4, (weight * 16).round() / 16         # a step of 1/16 or 1/64 more is exact
    ids = torch.randint(0, 700, (96, 5), generator=g, device="cuda")
    logits = randn(g, 96, 5)
    for which in ("hidden", "weight"):
        for op in ("cross_entropy", "distill"):
            args = (targets,) if op == "cross_entropy" else (ids, logits)
            x = hidden if which == "hidden" else weight
            step = (torch.randint(0, 2, x.shape, generator=g, device="cuda") * 2 - 1).to(BF16) / (16 if which == "hidden" else 64)
            sums, refs = [], []
            for sign in (1, -1):
                h, w = (hidden + sign * step, weight) if which == "hidden" else (hidden, weight + sign * step)
                assert torch.equal((h.double(), w.double())[which == "weight"], x.double() + sign * step.double())
                sums.append(getattr(ops, op + "_forward")(h, w, *args)[0].double().sum().item())
            _, lse = getattr(ops, op + "_forward")(hidden, weight, *args)
            ones = torch.ones(96, device="cuda")
            grads = getattr(ops, op + "_grad")(hidden, weight, *args, lse, ones)
            slope = (grads[which == "weight"].double() * step.double()).sum().item()
            q, entropy = wanted_of_targets(targets, 700) if op == "cross_entropy" else wanted_of_teacher(ids, logits, 700, 1.0)
            ref = Reference(hidden, weight, q, entropy, ones.double())
            move = step.double() @ weight.double().T if which == "hidden" else hidden.double() @ step.double().T
            third = ((move.max(1).values - move.min(1).values) ** 3 * (q.sum(1) > 0)).sum().item() * 2 / 6
            tol = third + 2 * ref.loss_tol.sum().item() + ((ref.h_tol, ref.w_tol)[which == "weight"] * step.double().abs()).sum().item()
            assert abs((sums[0] - sums[1]) / 2 - slope) <= tol and abs(slope) > 3 * tol / 100


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("k,n,vocab,width", [(1, 40, 300, 64), (3, 257, 1000, 128), (20, 301, 4001, 72), (64, 130, 9000, 264), (100, 33, 300, 7), (1000, 20, 5000, 64), (1024, 3, 1025, 8)])
def test_distillation(ops, k, n, vocab, width, dtype):
    hidden, weight, _, g = make(20 + k, n, vocab, width, dtype)
    r = gen(k)
    ids = torch.randint(0, vocab, (n, k), generator=r, device="cuda")             # some come twice
    ids[torch.rand(n, k, generator=r, device="cuda") < 0.2] = -1
    ids[::7] = -1                                                                 # rows of no entries
    logits = randn(r, n, k) * 3
    for kind, temperature in ((F32, 1.0), (BF16, 2.0), (F16, 0.75)):
        t = logits.to(kind)
        ref = Reference(hidden, weight, *wanted_of_teacher(ids, t, vocab, temperature), g.double(), temperature)
        losses, lse = ops.distill_forward(hidden, weight, ids.int() if kind == F32 else ids, t, temperature=temperature)
        d_hidden, d_weight = ops.distill_grad(hidden, weight, ids, t, lse, g, temperature=temperature)
        ref.check(losses, lse, d_hidden, d_weight)
        assert losses[::7].eq(0).all() and d_hidden[::7].eq(0).all()


@pytest.mark.parametrize("k", [1, 2, 7, 8, 9, 15, 16, 24, 63, 64, 65, 128, 511, 512, 1024])
def test_rows_with_all_their_entries(ops, k):
    """Every entry is one, all of them before, in or behind some tile of the vocabulary."""
    n, vocab = 130, 5000
    hidden, weight, _, g = make(33, n, vocab, 72, BF16)
    first = torch.randint(0, vocab - k, (n, 1), generator=gen(k), device="cuda")
    ids = first + torch.arange(k, device="cuda").flip(0)
    spread = torch.rand(n // 2, vocab, generator=gen(k + 1), device="cuda").argsort(1)[:, :k]
    ids[: n // 2] = spread
    logits = randn(gen(k + 2), n, k)
    ref = Reference(hidden, weight, *wanted_of_teacher(ids, logits, vocab, 1.0), g.double())
    losses, lse = ops.distill_forward(hidden, weight, ids, logits)
    ref.check(losses, lse, *ops.distill_grad(hidden, weight, ids, logits, lse, g))


def test_a_teachers_masks(ops):
    hidden, weight, _, g = make(30, 6, 500, 64, BF16)
    ids = torch.arange(24, device="cuda").view(6, 4)
    logits = randn(gen(30), 6, 4)
    low = torch.finfo(F32).min
    logits[0, 1:] = -math.inf          # one is left
    logits[1] = -math.inf              # none is left: no loss
    logits[2] = low                    # all alike
    logits[3, :2] = low
    ids[4] = -1
    ids[5, 2] = 500                    # beyond the vocabulary
    losses, lse = ops.distill_forward(hidden, weight, ids, logits)
    assert losses[5].isnan() and losses[[1, 4]].eq(0).all()
    logits2 = logits.clone()
    logits2[2] = 0
    good = [0, 2, 3]
    q, entropy = wanted_of_teacher(ids[good], logits2[good], 500, 1.0)
    ref = Reference(hidden[good], weight, q, entropy, g[good].double())
    d_hidden, d_weight = ops.distill_grad(hidden, weight, ids, logits, lse, g)
    ref.check(losses[good], lse[good], d_hidden[good], d_weight)
    assert d_hidden[[1, 4, 5]].eq(0).all()
    logits[0, 0] = math.nan          # (not in logits2)
    assert ops.distill_forward(hidden, weight, ids, logits)[0][0].isnan()
    # the order of a row's entries does not matter
    order = torch.tensor([2, 0, 3, 1], device="cuda")
    losses, lse = ops.distill_forward(hidden[good], weight, ids[good][:, order], logits2[good][:, order])
    ref.check(losses, lse, *ops.distill_grad(hidden[good], weight, ids[good][:, order], logits2[good][:, order], lse, g[good]))


def test_distillation_takes_part_in_autograd(ops):
    hidden, weight, _, g = make(31, 90, 800, 128, BF16)
    hidden, weight = hidden.requires_grad_(), weight.requires_grad_()
    ids = torch.randint(-1, 800, (9, 10, 6), generator=gen(31), device="cuda")
    logits = randn(gen(32), 9, 10, 6).requires_grad_()
    loss = ops.distill(hidden.view(9, 10, 128), weight, ids, logits, temperature=2.0, reduction="none")
    (loss * g.view(9, 10)).sum().backward()
    ref = Reference(hidden.detach(), weight.detach(), *wanted_of_teacher(ids.view(90, 6), logits.detach().view(90, 6), 800, 2.0), g.double(), 2.0)
    within(loss.detach().flatten(), ref.losses, ref.loss_tol, "losses")
    within(hidden.grad, ref.d_hidden, ref.h_tol, "d_hidden")
    within(weight.grad, ref.d_weight, ref.w_tol, "d_weight")
    assert logits.grad is None


# ---- lookup -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,vocab,width", [(0, 5, 8), (1, 1, 1), (5, 3, 3), (47, 300, 64), (33, 1000, 100), (1000, 50, 768), (129, 7, 2050), (3, 100, 4096)])
@pytest.mark.parametrize("scale", [1.0, 27.7128])
def test_embed(ops, n, vocab, width, dtype, scale):
    g = gen(n + width)
    table = randn(g, vocab, width).to(dtype)
    ids = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    if n > 4:
        ids[1], ids[3] = -1, -100
    want = torch.where(ids[:, None] >= 0, table[ids.clamp(min=0)].double() * float(torch.tensor(scale, dtype=F32)), 0.0)
    tol = want.abs() * (half_step(dtype) * 1.01 + 2.0 ** -24) + (2.0 ** -25 if dtype == F16 else 0)
    for kind in (torch.int32, torch.int64):
        got = ops.embed(ids.to(kind), table, scale=scale)
        assert got.dtype == dtype
        within(got, want, tol)
    if scale == 1.0:
        assert torch.equal(got, want.to(dtype))
    if n == 1000:
        assert torch.equal(ops.embed(ids.view(10, 100), table, scale=scale).view(n, width), got)
        assert torch.equal(ops.embed(ids.view(10, 100).t(), table, scale=scale), got.view(10, 100, width).transpose(0, 1))
    for other in layouts(table):
        assert torch.equal(ops.embed(ids, other, scale=scale), got)


def test_embed_without_the_extension(ops):
    """The lookup by ctypes gives what it gives by the extension, whichever of the two the installation has."""
    from graphtok_b200.ctypes_host import CtypesHost
    lib, table = ops._lib(), randn(gen(5), 300, 72).to(F16)
    ids = torch.randint(-1, 301, (100,), generator=gen(6), device="cuda")
    host, want = lib.host, ops.embed(ids, table, scale=0.3)
    lib.host = CtypesHost(lib)
    try:
        assert torch.equal(ops.embed(ids, table, scale=0.3).view(torch.int16), want.view(torch.int16))
    finally:
        lib.host = host


def test_embed_beyond_the_table(ops):
    table = randn(gen(1), 300, 64).to(BF16)
    ids = torch.tensor([0, 300, 299, 2 ** 40, -2 ** 40, 2 ** 31 + 5], device="cuda")
    out = ops.embed(ids, table)
    assert out[[1, 3, 5]].isnan().all() and out[4].eq(0).all() and torch.equal(out[[0, 2]], table[[0, 299]])
    assert ops.embed(ids, table[:0])[[0, 1, 2, 3, 5]].isnan().all()
    grad = ops.embed_grad(ids, torch.ones(6, 64, device="cuda", dtype=BF16), 300)
    assert grad[[0, 299]].eq(1).all() and grad.sum() == 128


def embed_grad_bound(ids, grad, vocab, scale, dtype):
    known = (ids >= 0) & (ids < vocab)
    want = torch.zeros(vocab, grad.shape[1], dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    want.index_add_(0, ids[known].long(), grad[known].double())
    size.index_add_(0, ids[known].long(), grad[known].double().abs())
    count = torch.bincount(ids[known].long(), minlength=vocab).double()[:, None]
    scale = float(torch.tensor(scale, dtype=F32))
    want *= scale
    # each addition takes half a step of fp32 of no more than the sum of magnitudes; one product; one rounding
    tol = (count + 1) * 2.0 ** -24 * size * abs(scale) + want.abs() * half_step(dtype) * 1.01 + (2.0 ** -25 if dtype == F16 else 0)
    return want, tol


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,vocab,width", [(0, 5, 8), (1, 1, 1), (31, 40, 3), (32, 2, 64), (33, 300, 256), (2047, 1000, 100), (2048, 513, 264), (2049, 512, 40), (2500, 1, 8),
                                           (5000, 70000, 64), (3000, 300001, 24), (40000, 511, 520), (7, 100003, 16), (100, 6000, 1032), (70000, 3000, 8), (3, 0, 8)])
def test_embed_grad(ops, n, vocab, width, dtype):
    g = gen(n + vocab)
    # frequent ids in long runs, rare ones in between, some outside the table (all of them, where it is empty)
    ids = (torch.exp(torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * math.log(vocab + 1)) - 1).long().clamp(max=max(0, vocab - 1))
    if n > 5:
        ids[2], ids[4] = -1, vocab + 7
    grad = randn(g, n, width).to(dtype)
    want, tol = embed_grad_bound(ids, grad, vocab, 1.5, dtype)
    got = ops.embed_grad(ids, grad, vocab, scale=1.5)
    within(got, want, tol)
    assert torch.equal(ops.embed_grad(ids.int(), grad, vocab, scale=1.5), got)                # and the same each time
    for other in layouts(grad):
        within(ops.embed_grad(ids, other, vocab, scale=1.5), want, tol)
    if not vocab:
        return
    wide = torch.full((vocab, width + 5), 3.0, dtype=dtype, device="cuda")
    assert ops.embed_grad(ids, grad, vocab, scale=1.5, out=wide[:, 2:2 + width]).data_ptr() == wide[:, 2:].data_ptr()
    within(wide[:, 2:2 + width], want, tol)
    assert wide[:, :2].eq(3).all() and wide[:, 2 + width:].eq(3).all()
    # onto what is there: one rounding of the new sum, other rows bit for bit
    base = randn(g, vocab, width).to(dtype)
    both = ops.embed_grad(ids, grad, vocab, scale=1.5, out=base.clone(), accumulate=True)
    total = base.double() + want
    within(both, total, tol + total.abs() * half_step(dtype) * 1.01 + base.double().abs() * 2.0 ** -24)
    untouched = torch.ones(vocab, dtype=torch.bool, device="cuda")
    untouched[ids[(ids >= 0) & (ids < vocab)]] = False
    assert torch.equal(both[untouched], base[untouched])


def test_embed_takes_part_in_autograd(ops):
    table = randn(gen(2), 500, 96).to(BF16).requires_grad_()
    ids = torch.randint(-1, 500, (7, 40), generator=gen(3), device="cuda")
    for make_grad in (lambda o: o.float().sum(), lambda o: (o.float() * randn(gen(4), *o.shape)).sum(), lambda o: o.transpose(0, 1).float().square().sum()):
        table.grad = None
        out = ops.embed(ids, table, scale=2.0)
        out.retain_grad()
        make_grad(out).backward()
        want, tol = embed_grad_bound(ids.flatten(), out.grad.reshape(280, 96), 500, 2.0, BF16)
        within(table.grad, want, tol)
    with torch.no_grad():
        assert not ops.embed(ids, table).requires_grad


def test_offsets_beyond_32_bits(ops):
    """Tables of more than 2^31 elements: rows at their end are looked up, summed and compared like others."""
    vocab, width = 262209, 8200
    table = torch.zeros(vocab, width, dtype=BF16, device="cuda")
    g = gen(80)
    some = torch.tensor([0, 1, 131071, 261900, 262207, 262208], device="cuda")
    table[some] = randn(g, 6, width).to(BF16)
    ids = some[torch.randint(0, 6, (70,), generator=g, device="cuda")]
    assert torch.equal(ops.embed(ids, table), table[ids])
    rows = randn(g, 70, width).to(BF16)
    grad = ops.embed_grad(ids, rows, vocab)
    want, tol = embed_grad_bound(torch.searchsorted(some, ids), rows, 6, 1.0, BF16)
    within(grad[some], want, tol)
    grad[some] = 0
    assert not grad.any()
    del grad
    for n in (40, 70):                   # the form of few rows, and the other
        hidden = (randn(g, n, width) / 32).to(BF16)
        losses, lse = ops.cross_entropy_forward(hidden, table, ids[:n])
        z = hidden.double() @ table[some].double().T
        others = torch.full((n, 1), math.log(vocab - 6), dtype=torch.float64, device="cuda")       # logits of 0
        full = torch.logsumexp(torch.cat([z, others], 1), 1)
        at = torch.searchsorted(some, ids[:n])
        size = ((width + 15) // 16 + 2) * 2.0 ** -23 * (hidden.double().abs() @ table[some].double().abs().T).max(1).values
        # a quarter of a million equal terms are added in fp32, tile by tile and then one tile after the other
        within(lse, full, size + 2000 * 2.0 ** -24 + 16 * 2.0 ** -24 * full.abs(), "lse")
        within(losses, full - z.gather(1, at[:, None])[:, 0], 2 * size + 2000 * 2.0 ** -24 + 32 * 2.0 ** -24 * (full.abs() + z.abs().max(1).values), "losses")
        d_hidden, d_weight = ops.cross_entropy_grad(hidden, table, ids[:n], lse, torch.ones(n, device="cuda"))
        p = torch.exp(z - full[:, None])
        d = p.clone()
        d[torch.arange(n), at] -= 1
        u = half_step(BF16)
        slack = u * 1.1 + size.max() * 4 + 2.0 ** -12
        within(d_hidden, d @ table[some].double(), slack * (d.abs() @ table[some].double().abs()) + (d @ table[some].double()).abs() * u * 1.01, "d_hidden")
        want = d.T @ hidden.double()
        within(d_weight[some], want, slack * (d.abs().T @ hidden.double().abs()) + want.abs() * u * 1.01, "d_weight")
        rest = torch.tensor([2, 100000, 262000, 262206], device="cuda")
        want = (torch.exp(-full)[:, None] * hidden.double()).sum(0)
        within(d_weight[rest], want.expand(4, -1), (slack * (torch.exp(-full)[:, None] * hidden.double().abs()).sum(0) + want.abs() * u * 1.01).expand(4, -1), "d_weight")


# ---- targets --------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(6))
def test_next_targets(ops, seed):
    g = torch.Generator().manual_seed(seed)
    n = [0, 1, 2, 300, 5000, 1025][seed]
    ids = torch.randint(0, 1000, (n,), generator=g, dtype=torch.int32)
    cuts = sorted(torch.randint(0, n + 1, (seed * 5 + 1,), generator=g).tolist())              # empty documents among them
    offsets = cuts if seed % 2 else [0] + cuts + [n]
    mask = torch.rand(n, generator=g) < 0.7
    want = torch.full((n,), -100, dtype=torch.int32)
    for a, b in zip(offsets, offsets[1:]):
        want[a:max(a, b - 1)] = ids[a + 1:b]
    off = torch.tensor(offsets, dtype=torch.int32).cuda()
    assert torch.equal(ops.next_targets(ids.cuda(), off).cpu(), want)
    assert torch.equal(ops.next_targets(ids.cuda(), off, loss_mask=mask.cuda(), ignore_index=-7).cpu(), torch.where(mask & (want >= 0), want, -7))


# ---- streams, graphs, errors -------------------------------------------------------------
def test_on_another_stream_and_captured(ops):
    """Two captured graphs, replayed one inside the other's work with new inputs, and eager calls on a side stream, all against eager results."""
    hidden, weight, targets, g = make(40, 300, 3000, 128, BF16)
    ids = torch.randint(0, 3000, (2500,), generator=gen(40), device="cuda")
    rows = randn(gen(41), 2500, 128).to(BF16)
    teacher = torch.randint(0, 3000, (300, 9), generator=gen(42), device="cuda")
    logits = randn(gen(43), 300, 9)

    def step():
        losses, lse = ops.cross_entropy_forward(hidden, weight, targets)
        soft, soft_lse = ops.distill_forward(hidden, weight, teacher, logits)
        d = ops.cross_entropy_grad(hidden, weight, targets, lse, g)
        e = ops.distill_grad(hidden, weight, teacher, logits, soft_lse, g)
        return [losses, soft, *d, *e, ops.embed(ids, weight.detach()), ops.embed_grad(ids, rows, 3000)]

    @torch.no_grad()
    def renew(seed):
        r = gen(seed)
        hidden.copy_(randn(r, 300, 128).to(BF16))
        targets.copy_(torch.randint(-1, 3000, (300,), generator=r, device="cuda"))
        ids.copy_(torch.randint(0, 40, (2500,), generator=r, device="cuda"))
        teacher.copy_(torch.randint(-1, 3000, (300, 9), generator=r, device="cuda"))

    side = torch.cuda.Stream()
    step()
    # an eager graph of the same leaves that lives all the while
    hidden.requires_grad_()
    weight.requires_grad_()
    alive = ops.cross_entropy(hidden, weight, targets) + ops.embed(ids, weight).float().mean()
    alive.backward(retain_graph=True)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step()
        graphs.append((graph, outs))
    for seed in (50, 51):
        renew(seed)
        want = [x.clone() for x in step()]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = step()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got in [eager] + [outs for _, outs in graphs]:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_from_a_thread_of_its_own(ops):
    """A backward pass in a thread that has not used the GPU yet, as torch's own for backward passes; two at once, and one a second time."""
    hidden, weight, targets, g = make(44, 40, 1000, 64, BF16, masked=0)
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets)
    want = ops.cross_entropy_grad(hidden, weight, targets, lse, g)
    h, w = hidden.clone().requires_grad_(), weight.clone().requires_grad_()
    loss = ops.cross_entropy(h, w, targets, reduction="none")
    torch.cuda.synchronize()
    got = [None] * 3
    def run(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[i] = ops.cross_entropy_grad(hidden, weight, targets, lse, g) if i else torch.autograd.grad(loss, (h, w), g, retain_graph=True)
        stream.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    h.detach().zero_()                  # the graph keeps what it needs of it
    got.append(torch.autograd.grad(loss, (h, w), g))
    torch.cuda.synchronize()
    for pair in got:
        assert all(torch.equal(a, b) for a, b in zip(pair, want))


def test_refusals(ops):
    from graphtok_b200 import GTokError
    hidden, weight, targets, g = make(60, 10, 50, 64, BF16)
    ids, logits = targets[:, None].clamp(min=0), randn(gen(60), 10, 1)
    lse = torch.zeros(10, device="cuda")
    bad = [
        (TypeError, lambda: ops.cross_entropy(hidden.float(), weight.float(), targets)),
        (TypeError, lambda: ops.cross_entropy(hidden, weight.half(), targets)),
        (TypeError, lambda: ops.cross_entropy(hidden, weight, targets.float())),
        (ValueError, lambda: ops.cross_entropy(hidden, weight[:, :32], targets)),
        (ValueError, lambda: ops.cross_entropy(hidden, weight[:0], targets)),
        (ValueError, lambda: ops.cross_entropy(hidden, weight, targets[:9])),
        (ValueError, lambda: ops.cross_entropy(hidden, weight, targets.cpu())),
        (ValueError, lambda: ops.cross_entropy(hidden, weight, targets, reduction="max")),
        (ValueError, lambda: ops.cross_entropy(hidden, weight, targets, temperature=0)),
        (ValueError, lambda: ops.distill(hidden, weight, ids, logits, temperature=math.nan)),
        (ValueError, lambda: ops.distill(hidden, weight, ids, logits[:, :0])),
        (ValueError, lambda: ops.distill(hidden, weight, ids.expand(10, 1025), logits.expand(10, 1025))),
        (TypeError, lambda: ops.distill(hidden, weight, ids, logits.double())),
        (TypeError, lambda: ops.cross_entropy_grad(hidden, weight, targets, lse, g.double())),
        (ValueError, lambda: ops.cross_entropy_grad(hidden, weight, targets, lse, g[:1])),
        (ValueError, lambda: ops.cross_entropy_grad(hidden, weight, targets, lse, g, reduction="mean")),
        (TypeError, lambda: ops.embed(targets.float(), weight)),
        (TypeError, lambda: ops.embed(targets, weight.double())),
        (ValueError, lambda: ops.embed(targets, weight[0])),
        (ValueError, lambda: ops.embed(targets, weight, scale=math.inf)),
        (ValueError, lambda: ops.embed_grad(targets, hidden[:9], 50)),
        (ValueError, lambda: ops.embed_grad(targets, hidden, -1)),
        (ValueError, lambda: ops.embed_grad(targets, hidden, 50, accumulate=True)),
        (ValueError, lambda: ops.embed_grad(targets, hidden, 50, out=weight[:49])),
        (ValueError, lambda: ops.embed_grad(targets, hidden, 50, out=weight.float())),
        (GTokError, lambda: ops.embed_grad(targets, hidden, 50, out=weight[:1].expand(50, 64))),
        (ValueError, lambda: ops.next_targets(targets, targets)),
        (ValueError, lambda: ops.next_targets(targets.int(), targets.int(), loss_mask=targets > 1, ignore_index=3)),
        (ValueError, lambda: ops.next_targets(targets.int(), targets.int(), loss_mask=(targets > 1)[:3])),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


def test_refusals_of_the_c_entries(ops):
    """Workspaces that are too small or missing, addresses on the host, shapes that do not fit: an error code and a message, nothing queued."""
    hidden, weight, targets, g = make(61, 10, 300, 64, BF16)
    lib = ops._lib()
    losses, lse = torch.zeros(10, device="cuda"), torch.zeros(10, device="cuda")
    work = torch.empty(1 << 26, dtype=torch.uint8, device="cuda")
    host = torch.zeros(4096, dtype=torch.uint8)

    def args():
        call = ops._Call(hidden, weight, targets, None, -100, 1.0)
        a = call.args
        a.losses, a.lse, a.workspace, a.workspace_bytes = losses.data_ptr(), lse.data_ptr(), work.data_ptr(), work.numel()
        a.grad, a.grad_stride = g.data_ptr(), 1
        a.d_hidden = ops._matrix(torch.empty_like(hidden))
        a.cuda_stream = torch.cuda.current_stream().cuda_stream
        return a

    assert lib.gtok_x_vocab_loss_forward(args()) == 0 and lib.gtok_x_vocab_loss_backward(args()) == 0
    # the mean has one gradient, whatever the stride says
    one, got = torch.full((), 0.5, device="cuda"), torch.empty_like(hidden)
    a = args()
    a.mean, a.grad, a.d_hidden = 1, one.data_ptr(), ops._matrix(got)
    assert lib.gtok_x_vocab_loss_backward(a) == 0
    assert torch.equal(got, ops.cross_entropy_grad(hidden, weight, targets, lse, one, reduction="mean")[0])
    need = lib.gtok_x_vocab_loss_workspace(args(), 0)
    changes = [("workspace_bytes", need - 1), ("workspace", None), ("workspace", work.data_ptr() + 16), ("workspace", host.data_ptr()), ("losses", None),
               ("losses", host.data_ptr()), ("lse", None), ("targets", host.data_ptr()), ("targets", None), ("targets", targets.data_ptr() + 4), ("target_bits", 16),
               ("total", host.data_ptr()), ("hidden", ops._Matrix(hidden.data_ptr() + 1, 10, 64, 64, 1)), ("hidden", ops._Matrix(host.data_ptr(), 10, 64, 64, 1)),
               ("hidden", ops._Matrix(None, 10, 64, 64, 1)), ("weight", ops._Matrix(weight.data_ptr(), 300, 64, 63, 1)), ("weight", ops._Matrix(weight.data_ptr(), 300, 64, -64, 1))]
    for name, value in changes:
        a = args()
        setattr(a, name, value)
        assert lib.gtok_x_vocab_loss_forward(a) == -1, name
        assert lib.gtok_x_last_error()
    for name, value in (("grad", None), ("grad", host.data_ptr()), ("grad_stride", -1), ("lse", None), ("d_hidden", ops._Matrix(hidden.data_ptr(), 10, 64, 32, 1)),
                        ("d_hidden", ops._Matrix(hidden.data_ptr(), 9, 64, 64, 1)), ("d_hidden", ops._Matrix(hidden.data_ptr(), 10, 64, 64, 2)), ("d_weight", ops._matrix(hidden)),
                        ("workspace_bytes", 100)):
        a = args()
        setattr(a, name, value)
        assert lib.gtok_x_vocab_loss_backward(a) == -1, name
    torch.cuda.synchronize()


# ---- as they are used together ------------------------------------------------------------
@pytest.mark.parametrize("family", ["llama3", "gemma"])
def test_text_to_gradients_of_a_tied_table(ops, family):
    """Texts to ids, ids to rows of a table, a layer of a model, and the loss against the same table: gradients of the table and the layer against
    the formulas in 64 bits."""
    from graphtok_b200.gpu_bpe_tokenizer import Tokenizer
    tok = Tokenizer(tiny_vocab(family))
    texts = ["The first document, of some length.", "", "A second one; shorter!", "éè and 123 others\n\n", "x"]
    width, vocab = 64, tok.vocab_size
    table = (randn(gen(70), vocab, width) / 8).to(BF16).requires_grad_()
    layer = (randn(gen(71), width, width) / 8).to(BF16).requires_grad_()
    scale = 8.0 if family == "gemma" else 1.0
    rows, ids, offsets, targets = tok.encode_batch_for_model(texts, table, scale=scale)
    want_ids, want_offsets = tok.encode_batch(texts)
    assert ids.tolist() == want_ids.tolist() and offsets.tolist() == want_offsets.tolist()
    n = ids.numel()
    rows.retain_grad()
    hidden = torch.tanh(rows @ layer) * 3
    hidden.retain_grad()
    loss = ops.cross_entropy(hidden, table, targets)
    loss.backward()
    # every part by its formula, from the 16-bit values that the part before gave
    last = {b - 1 for a, b in zip(want_offsets.tolist(), want_offsets.tolist()[1:]) if b > a}
    expect = torch.tensor([-100 if i in last else int(want_ids[i + 1]) for i in range(n)], device="cuda")
    assert torch.equal(targets.long(), expect)
    within(rows.detach(), table.detach()[ids.long()].double() * scale, (table.detach()[ids.long()].double() * scale).abs() * half_step(BF16))
    count = int((expect >= 0).sum())
    assert count == n - len(last)
    ref = Reference(hidden.detach(), table.detach(), *wanted_of_targets(expect, vocab), torch.full((n,), 1.0 / count, dtype=torch.float64, device="cuda"))
    within(loss.detach(), ref.losses.sum() / count, ref.loss_tol.sum() / count + 40 * 2.0 ** -24 * ref.losses.abs().mean())
    within(hidden.grad, ref.d_hidden, ref.h_tol, "d_hidden")
    lookup, lookup_tol = embed_grad_bound(ids.long(), rows.grad, vocab, scale, BF16)
    total = lookup + ref.d_weight
    # torch adds the two gradients of the shared table: each rounded, then their sum
    within(table.grad, total, lookup_tol + ref.w_tol + total.abs() * half_step(BF16) * 1.01 + (lookup_tol + ref.w_tol) * half_step(BF16), "table")
    assert layer.grad.isfinite().all() and layer.grad.abs().sum() > 0
