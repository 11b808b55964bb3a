"""Cases at the borders of the operators between token ids and a model, on a B200: long running sums, exact logits, gradients that are not finite,
results that another party looks at."""
import math

import pytest
import torch

from conftest import tiny_vocab
from test_vocab_ops import BF16, F16, Reference, gen, make, ops, randn, wanted_of_targets, wanted_of_teacher, within     # noqa: F401  (ops is a fixture)

pytestmark = pytest.mark.gpu


def exact_logits(n, vocab):
    """Rows whose products and sums of products are small whole numbers, exact in any order: a leading logit of 40 to 100 (of 0 in every eighth row) at an
    id in the first tile that a pair of blocks takes (256 ids a tile, 74 pairs take them in turn), the others between -4 and 4."""
    width = 64                                   # (a logit is scaled by 1 + 2^-24 for it, which is 1 in fp32)
    g = gen(n)
    weight = torch.zeros(vocab, width, device="cuda")
    weight[:, 60:] = torch.randint(-1, 2, (vocab, 4), generator=g, device="cuda").float()
    leads = torch.arange(60, device="cuda") * 256 + torch.randint(0, 256, (60,), generator=g, device="cuda")
    weight[leads, 60:] = 0
    weight[leads, torch.arange(60, device="cuda")] = 10
    row = torch.arange(n, device="cuda")
    hidden = torch.zeros(n, width, device="cuda")
    hidden[row, row % 60] = (3 + row % 8).float() * (row % 8 > 0)
    hidden[:, 60:] = torch.randint(0, 2, (n, 4), generator=g, device="cuda").float() * (row % 16 > 0)[:, None]
    targets = leads[row % 60].clone()
    targets[::5] = torch.randint(0, vocab, ((n + 4) // 5,), generator=g, device="cuda")
    return hidden.to(BF16), weight.to(BF16), targets


@pytest.mark.parametrize("n", [1, 37, 64, 65, 200, 256, 300])
def test_long_running_sums(ops, n):  # noqa: F811
    """A row's sum over 151,665 ids with its maximum at the front, whatever number of rows it is computed among.  The terms' sum S in units of
    the largest is off by what its additions round, at most 2^-24 S each, and never by more than what they add; lse is maximum + log S.

    Additions one after the other: 8 + 2 of a step of 32 columns, 36 steps, 8 + 5 to join them, and 43 in the form of few rows.  Where the maximum moves
    (in whole numbers from -4 to 4, so at most 8 times) a power of 2 and a product, 2^-22 + 2^-24; three powers of 2 of each term and the sum."""
    vocab = 151665
    hidden, weight, targets = exact_logits(n, vocab)
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets)
    z = hidden.double() @ weight.double().T
    want = torch.logsumexp(z, 1)
    rest = torch.exp(want - z.max(1).values) - 1                # beside the largest term, in its units
    total = torch.minimum((59 + 8 * 5) * 2.0 ** -24 * (1 + rest), 2 * rest) + 3 * 2.0 ** -22 * (1 + rest)
    step = 2.0 ** -24
    # a term's exponent is rounded by half a step of 16 at most, log2(e) in it by half a step of its own
    tol = total / (1 + rest) + 16 * step + 2 * step * torch.log1p(rest) + step * want.abs()
    within(lse, want, tol, "lse")
    at = z.gather(1, targets[:, None])[:, 0]
    within(losses, want - at, tol + step * (want - at).abs(), "losses")


@pytest.mark.parametrize("n", [37, 200, 300])
def test_gradients_of_confident_rows(ops, n):  # noqa: F811
    """Where a row's target is its far logit, p - 1 is next to nothing, and what lse is off by would be all of it.  With the logits exact, the exponent of p
    is off by half a step each of lse, of its power of 2 and of their difference, log2(e) in the difference by half a step more; then a power of 2."""
    vocab = 151665
    hidden, weight, targets = exact_logits(n, vocab)
    _, lse = ops.cross_entropy_forward(hidden, weight, targets)
    d_hidden, d_weight = ops.cross_entropy_grad(hidden, weight, targets, lse, torch.ones(n, device="cuda"))
    h, w = hidden.double(), weight.double()
    z = h @ w.T
    want = torch.logsumexp(z, 1, keepdim=True)
    rest = torch.exp(want - z.max(1, keepdim=True).values) - 1
    step, u = 2.0 ** -24, torch.finfo(BF16).eps / 2
    lse_off = torch.minimum((59 + 8 * 5) * step * (1 + rest), 2 * rest) / (1 + rest) + 3 * 2.0 ** -22 + 16 * step + 2 * step * torch.log1p(rest) + step * want.abs()
    p = torch.exp(z - want)
    q = torch.zeros_like(p).scatter_(1, targets[:, None], 1.0)
    d = p - q
    # three products and a difference in fp32, 16 bits, and the sums of the two products (a step every 16 elements, 40 more for pieces and splits)
    least = 2.0 ** -126                    # powers of 2 below the least normal number are 0, and a product or a sum may lose as much
    off = p * (lse_off + step * (want.abs() + 2 * (z - want).abs()) + 2.0 ** -22) + 4 * step * (p + q) + d.abs() * u + least
    for got, a, b, o, m in ((d_hidden, d, w, off, vocab), (d_weight, d.T, h, off.T, n)):
        size = a.abs() @ b.abs()
        within(got, a @ b, o @ b.abs() + size * (m / 16 + 40) * 2.0 ** -23 + (a @ b).abs() * u * 1.01 + least)


@pytest.mark.parametrize("n", [9, 64])
@pytest.mark.parametrize("temperature", [0.4, 2.5])
def test_a_temperature_with_few_rows(ops, n, temperature):  # noqa: F811
    hidden, weight, targets, g = make(90 + n, n, 40000, 136, BF16)
    ref = Reference(hidden, weight, *wanted_of_targets(targets, 40000), g.double(), temperature)
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets, temperature=temperature)
    ref.check(losses, lse, *ops.cross_entropy_grad(hidden, weight, targets, lse, g, temperature=temperature))


@pytest.mark.parametrize("n", [20, 300])
@pytest.mark.parametrize("width", [64, 4096])
def test_exact_logits(ops, n, width):  # noqa: F811
    """Hidden states with one element: every logit is one product.  It is taken 2^-26 a step of 16 elements too large, and no more."""
    g = gen(n + width)
    weight = randn(g, 500, width).to(BF16)
    column = torch.randint(0, width, (n,), generator=g, device="cuda")
    hidden = torch.zeros(n, width, dtype=BF16, device="cuda")
    hidden[torch.arange(n, device="cuda"), column] = (randn(g, n) * 4).to(BF16)
    targets = torch.randint(0, 500, (n,), generator=g, device="cuda")
    losses, lse = ops.cross_entropy_forward(hidden, weight, targets)
    z = hidden.double() @ weight.double().T
    dz = z.abs().max(1).values * (width / 16 * 2.0 ** -26 + 2.0 ** -24)
    want = torch.logsumexp(z, 1)
    # sums of 500 terms: 12 powers of 2 and 60 additions at most, logarithm and last sum
    tol = dz + (12 * 4 + 60) * 2.0 ** -24 + 2.0 ** -22 * (want.abs() + z.abs().max(1).values)
    within(lse, want, tol, "lse")
    within(losses, want - z.gather(1, targets[:, None])[:, 0], tol + dz, "losses")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("op", ["cross_entropy", "distill"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_gradient_that_is_not_finite_stays_in_its_row(ops, value, op, dtype):  # noqa: F811
    """dH_i = g_i dz_i W depends on its own row's gradient alone; dW takes part of every row."""
    n, vocab = 300, 700
    hidden, weight, targets, g = make(95, n, vocab, 64, dtype)
    if op == "cross_entropy":
        args, (q, entropy) = (targets,), wanted_of_targets(targets, vocab)
    else:
        ids, logits = torch.randint(0, vocab, (n, 6), generator=gen(96), device="cuda"), randn(gen(97), n, 6)
        args, (q, entropy) = (ids, logits), wanted_of_teacher(ids, logits, vocab, 1.0)
    forward, backward = getattr(ops, op + "_forward"), getattr(ops, op + "_grad")
    _, lse = forward(hidden, weight, *args)
    active = (q.sum(1) > 0).nonzero().squeeze(1)
    wrong = active[[3, 100]]
    bad = g.clone()
    bad[wrong] = value
    d_hidden, d_weight = backward(hidden, weight, *args, lse, bad)
    assert not d_hidden[wrong].isfinite().any() and not d_weight.isfinite().any()
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[wrong] = False
    g[wrong] = 0
    ref = Reference(hidden, weight, q, entropy, g.double())
    within(d_hidden[rest], ref.d_hidden[rest], ref.h_tol[rest], "d_hidden")
    # all of them: nothing finite is made up
    d_hidden, d_weight = backward(hidden, weight, *args, lse, torch.full_like(g, value))
    assert not d_hidden[active].isfinite().any() and not d_weight.isfinite().any()
    others = torch.ones(n, dtype=torch.bool, device="cuda")
    others[active] = False
    assert d_hidden[others].eq(0).all()


@pytest.mark.parametrize("n,vocab,width", [(50, 3000, 64), (2100, 140000, 584), (300, 500, 65)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_an_error_makes_every_gradient_nan(ops, n, vocab, width, dtype):  # noqa: F811
    """The flag that a kernel raises when a wait of its has run out, here set where a forward pass keeps it for the backward one; d_hidden finished by the
    last product and by a launch of its own, the table's gradient in one piece and in several, by tiles and by threads."""
    hidden, weight, targets, g = make(98, n, vocab, width, dtype)
    call = ops._Call(hidden, weight, targets, None, -100, 1.0)
    call.forward("none", keep=True)
    good = call.again(weight, call.kept).backward(None, g, "none", True, True)
    assert all(x.isfinite().all() for x in good)
    call.kept[4:8].view(torch.int32).fill_(1)
    for want_hidden, want_weight in ((True, True), (True, False), (False, True)):
        d_hidden, d_weight = call.again(weight, call.kept).backward(None, g, "none", want_hidden, want_weight)
        if want_hidden:
            assert d_hidden[targets >= 0].isnan().all() and d_hidden[targets < 0].eq(0).all()
        if want_weight:
            assert d_weight.isnan().all()


def test_autograd_sees_what_embed_grad_writes(ops):  # noqa: F811
    ids = torch.tensor([1, 3], device="cuda")
    grad, out = torch.ones(2, 8, device="cuda"), torch.ones(5, 8, device="cuda")
    x = torch.ones(5, 8, device="cuda", requires_grad=True)
    product = x * out
    ops.embed_grad(ids, grad, 5, out=out, accumulate=True)
    assert out._version == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    with torch.inference_mode():
        ops.embed_grad(ids, grad, 5, out=torch.zeros(5, 8, device="cuda"))


def test_embed_grad_onto_its_own_input_is_refused(ops):  # noqa: F811
    ids = torch.arange(5, device="cuda")
    both = torch.ones(6, 16, device="cuda")
    for out in (both[:5], both[1:], both[:5, :16]):
        with pytest.raises(ValueError, match="overlap"):
            ops.embed_grad(ids, both[:5], 5, out=out)
    with pytest.raises(ValueError, match="overlap"):
        ops.embed_grad(ids, both[:5, :8], 5, out=both[:5, 4:12])
    # columns beside one another are apart, and so are rows behind one another
    got = ops.embed_grad(ids, both[:5, :8], 5, out=both[:5, 8:])
    assert got.eq(1).all()
    two = torch.ones(10, 16, device="cuda")
    assert ops.embed_grad(ids, two[:5], 5, out=two[5:], accumulate=True).eq(2).all() and two[:5].eq(1).all()


@pytest.mark.parametrize("family", ["llama3", "gemma"])
def test_texts_with_a_mask(ops, family):  # noqa: F811
    """A mask is made of the ids that the call makes: here prompts whose positions carry no loss, by their lengths in ids."""
    from graphtok_b200.gpu_bpe_tokenizer import Tokenizer
    tok = Tokenizer(tiny_vocab(family))
    prompts, answers = ["A question? ", "", "Another, longer question:\n"], ["An answer.", "No prompt.", "42"]
    table = randn(gen(72), tok.vocab_size, 64).to(BF16)
    lengths = torch.tensor([len(tok.encode(p)) for p in prompts], device="cuda")
    seen = []

    def answers_only(ids, offsets):
        seen.append((ids, offsets))
        at = torch.arange(ids.numel(), device="cuda")
        doc = torch.searchsorted(offsets[1:].contiguous(), at.int(), right=True)
        return at - offsets[doc] + 1 >= lengths[doc]

    rows, ids, offsets, targets = tok.encode_batch_for_model([p + a for p, a in zip(prompts, answers)], table, loss_mask=answers_only)
    assert len(seen) == 1 and seen[0][0] is ids and seen[0][1] is offsets
    want = [-100] * ids.numel()
    o = offsets.tolist()
    for d in range(3):
        for i in range(o[d], o[d + 1] - 1):
            if i - o[d] + 1 >= lengths[d]:
                want[i] = int(ids[i + 1])
    assert targets.tolist() == want and 0 < sum(t >= 0 for t in want) < len(want) - 3
    assert torch.equal(rows, table[ids.long()])
    mask = answers_only(ids, offsets)                    # one that is there already is taken as it is
    assert torch.equal(tok.encode_batch_for_model([p + a for p, a in zip(prompts, answers)], table, loss_mask=mask)[3], targets)
    with pytest.raises(ValueError, match="loss_mask"):
        tok.encode_batch_for_model(prompts, table, loss_mask=lambda ids, offsets: torch.ones(1, dtype=torch.bool, device="cuda"))


def test_no_texts(ops):  # noqa: F811
    from graphtok_b200.gpu_bpe_tokenizer import Tokenizer
    tok = Tokenizer(tiny_vocab("llama3"))
    table = torch.ones(tok.vocab_size, 64, dtype=BF16, device="cuda", requires_grad=True)
    for texts in ([], [""], ["", ""]):
        rows, ids, offsets, targets = tok.encode_batch_for_model(texts, table)
        assert rows.shape == (0, 64) and ids.numel() == targets.numel() == 0 and offsets.tolist() == [0] * (len(texts) + 1)
        table.grad = None
        loss = ops.cross_entropy(rows, table, targets)
        loss.backward()
        assert loss == 0 and table.grad.eq(0).all()


def test_numbers_at_odd_addresses_are_refused(ops):  # noqa: F811
    """Losses, lse, their total and their gradient are whole fp32 numbers to the kernels: a message in place of a misaligned access."""
    hidden, weight, targets, g = make(99, 10, 300, 64, BF16)
    lib, room = ops._lib(), torch.zeros(64, device="cuda")
    work = torch.empty(1 << 26, dtype=torch.uint8, device="cuda")

    def args():
        a = ops._Call(hidden, weight, targets, None, -100, 1.0).args
        a.losses, a.lse, a.total, a.workspace, a.workspace_bytes = room.data_ptr(), room.data_ptr() + 64, room.data_ptr() + 128, work.data_ptr(), work.numel()
        a.grad, a.grad_stride, a.cuda_stream = g.data_ptr(), 1, torch.cuda.current_stream().cuda_stream
        a.d_weight = ops._matrix(torch.empty_like(weight))
        return a

    assert lib.gtok_x_vocab_loss_forward(args()) == 0 and lib.gtok_x_vocab_loss_backward(args()) == 0
    for entry, names in ((lib.gtok_x_vocab_loss_forward, ("losses", "lse", "total")), (lib.gtok_x_vocab_loss_backward, ("lse", "grad"))):
        for name in names:
            for odd in (1, 2, 3):
                a = args()
                setattr(a, name, getattr(a, name) + odd)
                assert entry(a) == -1 and b"aligned" in lib.gtok_x_last_error(), name
    torch.cuda.synchronize()


@pytest.mark.parametrize("temperature", [1e-40, 1.1e-38, 1e39, 0.0, -1.0, math.inf, math.nan])
def test_temperatures_that_float32_does_not_hold(ops, temperature):  # noqa: F811
    hidden, weight, targets, _ = make(100, 10, 300, 64, BF16)
    with pytest.raises(ValueError, match="temperature"):
        ops.cross_entropy(hidden, weight, targets, temperature=temperature)
    least = 2.0 ** -126
    assert ops.cross_entropy(torch.zeros_like(hidden), weight, targets, temperature=least, reduction="none")[targets >= 0].sub(math.log(300)).abs().max() < 1e-5


@pytest.mark.parametrize("scale", [1e39, -1e39, 3.5e38, math.inf, math.nan])
def test_scales_that_float32_does_not_hold(ops, scale):  # noqa: F811
    ids, table = torch.tensor([1, 2], device="cuda"), torch.zeros(5, 8, device="cuda")
    for call in (lambda: ops.embed(ids, table, scale=scale), lambda: ops.embed_grad(ids, table[:2], 5, scale=scale)):
        with pytest.raises(ValueError, match="scale"):
            call()
    assert ops.embed(ids, table, scale=torch.finfo(torch.float32).max).eq(0).all()


def test_captured_behind_copies_and_on_forked_streams(ops):  # noqa: F811
    """In a graph whose nodes in front of the kernels are copies and fills, and with two passes side by side."""
    hidden, weight, targets, g = make(101, 300, 3000, 128, BF16)
    ids, rows = torch.randint(0, 3000, (2500,), generator=gen(102), device="cuda"), randn(gen(103), 2500, 128).to(BF16)

    def step(h, w):
        losses, lse = ops.cross_entropy_forward(h, w, targets)
        return [losses, lse, *ops.cross_entropy_grad(h, w, targets, lse, g), ops.embed(ids, w), ops.embed_grad(ids, rows, 3000)]

    want = [x.clone() for x in step(hidden, weight)]
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        h, w = torch.empty_like(hidden).copy_(hidden), torch.zeros_like(weight).copy_(weight)
        first = ops.embed(ids, w)
        other.wait_stream(side)
        with torch.cuda.stream(other):
            there = step(h, w)
        here = step(h, w)
        side.wait_stream(other)
        joined = ops.embed(ids, w)
        onto = ops.embed_grad(ids, rows, 3000, out=torch.zeros_like(weight), accumulate=True)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for outs in (here, there) for a, b in zip(outs, want))
        assert torch.equal(first, want[4]) and torch.equal(joined, want[4]) and torch.equal(onto, want[5])


def test_from_compiled_code(ops):  # noqa: F811
    """torch.compile does not look into the operators; called through torch.compiler.disable they run between its graphs."""
    hidden, weight, targets, _ = make(104, 70, 900, 64, BF16)
    embed, loss_of = torch.compiler.disable(ops.embed), torch.compiler.disable(ops.cross_entropy)

    @torch.compile(backend="eager")
    def step(ids, table, layer):
        return loss_of(embed(ids, table) @ layer, table, targets) * 2

    ids = torch.randint(0, 900, (70,), generator=gen(105), device="cuda")
    layer = (randn(gen(106), 64, 64) / 8).to(BF16)
    got, want = [], []
    for outs, f in ((got, step), (want, lambda i, t, m: ops.cross_entropy(ops.embed(i, t) @ m, t, targets) * 2)):
        t, m = weight.clone().requires_grad_(), layer.clone().requires_grad_()
        loss = f(ids, t, m)
        loss.backward()
        outs += [loss.detach(), t.grad, m.grad]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def negated(*shape):
    """(values as a view whose memory holds their negatives, as torch gives for parts of complex gradients; the same in memory of their own)"""
    x = torch.complex(torch.zeros(shape, device="cuda"), torch.randn(shape, generator=gen(107), device="cuda")).conj().imag
    assert x.is_neg()
    return x, x.clone()


def test_views_of_negated_values(ops):  # noqa: F811
    hidden, weight, targets, _ = make(108, 300, 700, 64, BF16)
    _, lse = ops.cross_entropy_forward(hidden, weight, targets)
    view, plain = negated(300)
    assert all(torch.equal(a, b) for a, b in zip(ops.cross_entropy_grad(hidden, weight, targets, lse, view), ops.cross_entropy_grad(hidden, weight, targets, lse, plain)))
    view, plain = negated()
    assert all(torch.equal(a, b) for a, b in zip(ops.cross_entropy_grad(hidden, weight, targets, lse, view, reduction="sum"),
                                                 ops.cross_entropy_grad(hidden, weight, targets, lse, plain, reduction="sum")))
    # through autograd: the losses as the imaginary part of a complex number
    grads = []
    for part in (lambda x: torch.complex(torch.zeros_like(x), x).conj().imag, lambda x: -x):
        h = hidden.clone().requires_grad_()
        part(ops.cross_entropy(h, weight, targets, reduction="none")).sum().backward()
        grads.append(h.grad)
    assert torch.equal(*grads)
    ids = torch.randint(0, 300, (50,), generator=gen(109), device="cuda")
    for width in (1, 8):
        view, plain = negated(300, width)
        assert torch.equal(ops.embed(ids, view), ops.embed(ids, plain))
        assert torch.equal(ops.embed_grad(ids, view[:50], 300), ops.embed_grad(ids, plain[:50], 300))
    view, plain = negated(300, 1)
    with pytest.raises(ValueError, match="negated"):
        ops.embed_grad(ids, plain[:50], 300, out=view)
