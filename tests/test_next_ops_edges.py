"""The operators from hidden states to ids where it is easy to go wrong: the largest vocabularies, arguments that lie over one another, on a B200."""
import math
import os
import textwrap

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from test_next_ops import check_draw, check_logits, model_logits
from test_vocab_ops import BF16, F16, F32, gen, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(built):
    from graphtok_b200 import next_ops
    return next_ops


# ---- an id a row -----------------------------------------------------------------------
@pytest.mark.parametrize("vocab,depth", [(1 << 24, 25.0), (1 << 24, 17.25), (3000001, 20.0), ((1 << 19) + 1, 18.0), (1 << 19, 18.0)])
def test_a_flat_tail_far_below_one_logit(ops, vocab, depth):
    """One likely id, and all others alike and so unlikely that a mass is a few units or none: their share is drawn and cut as it should be, and whatever the number of rows.

    A mass is rounded to a unit of the largest, which is 2^-43 up to 2^19 ids and 2^-50 here beyond (the total is near 1): together they are off by
    at most 2^19 * 2^-44 and 2^24 * 2^-51, both within 2^-25; masses and u * total are off by 2^-43 and 2^-53 relative."""
    likely, off = vocab // 13, 2.0 ** -25
    row = torch.full((1, vocab), -depth, device="cuda")
    row[0, likely] = 0.0
    m = math.exp(-depth)
    total = 1 + (vocab - 1) * m
    tail = 1 - 1 / total
    upto = lambda i: ((i + 1) * m + (1 - m if i >= likely else 0)) / total          # noqa: E731
    points = [0.0, tail / 20, 0.5, 1 - 0.8 * tail, 1 - tail / 3, 1 - 2.0 ** -53]
    seen = {}
    for n in (1, 3, 148):
        u = torch.tensor([points[i % len(points)] for i in range(n)], dtype=torch.float64, device="cuda")
        ids, logprobs = ops.sample(row.expand(n, vocab), u)
        for i, (got, logprob) in enumerate(zip(ids.tolist(), logprobs.tolist())):
            at = points[i % len(points)]
            assert upto(got - 1) <= at + off and upto(got) >= at - off, (n, at, got)
            want = math.log((1.0 if got == likely else m) / total)
            assert abs(logprob - want) <= 1.01 * off + abs(want) * 2.0 ** -24 * 1.01
            assert seen.setdefault(at, (got, logprob)) == (got, logprob)
    # a cut inside the tail: the last kept id says where
    share = float(torch.tensor(1 - 0.4 * tail, dtype=F32))
    for n in (1, 148):
        ids, _ = ops.sample(row.expand(n, vocab), torch.full((n,), 1 - 2.0 ** -53, dtype=torch.float64, device="cuda"), top_p=share)
        got = ids.tolist()
        assert len(set(got)) == 1 and abs((1 + (got[0] + (got[0] < likely)) * m) / total - share) <= off + 2 * m
        assert seen.setdefault("cut", got[0]) == got[0]


# (blocks of a row for each: 1, 1, 2, 2, 4, 4, 8; none of the shares fits into shared memory)
@pytest.mark.parametrize("n,vocab,dtype", [(251, 30000, BF16), (160, 50257, F32), (100, 60000, F32), (40, 100000, BF16), (30, 100000, F32), (20, 151665, BF16), (3, 262144, F32)])
def test_shares_that_are_read_again_from_memory(ops, n, vocab, dtype):
    """In each number of blocks: flat rows of which much is kept, and rows that begin anywhere in 16 bytes."""
    for i, wish in enumerate(((1.0, 0, 0.9, 0.0), (0.9, 40, 0.95, 0.0), (1.0, 0, 1.0, 0.0))):
        logits = model_logits(n + i, n, vocab, dtype)
        logits[::7] *= 0.01                                  # next to flat
        u = torch.rand(n, generator=gen(i), device="cuda")
        ids = check_draw(ops, logits, u, *wish)
        room = torch.empty(n, vocab + 3, dtype=dtype, device="cuda")
        room[:, 1:1 + vocab] = logits
        assert torch.equal(ops.sample(room[:, 1:1 + vocab], u, temperature=wish[0], top_k=wish[1], top_p=wish[2], min_p=wish[3])[0], ids)


@pytest.mark.parametrize("n,vocab", [(5, 128256), (5, 151665), (3, 50256), (200, 40000), (4, 7), (2, 600000)])
def test_no_logprob_is_above_0(ops, n, vocab):
    """An id that is alone, as a grammar often leaves one, has all of the mass: logprob 0 to the bit, whatever the logit; and others' are not above it."""
    logits = torch.full((n, vocab), -math.inf, device="cuda")
    value = torch.tensor([0.0, 7.3, -100.1, 3e38, -3.4e38], device="cuda")[torch.arange(n, device="cuda") % 5]
    place = torch.randint(0, vocab, (n,), generator=gen(n), device="cuda")
    logits[torch.arange(n, device="cuda"), place] = value
    u = torch.rand(n, generator=gen(n + 1), device="cuda")
    for wish in (dict(), dict(top_k=1), dict(top_k=50, top_p=0.9), dict(top_p=0.9, temperature=0.7), dict(min_p=0.1), dict(top_p=0.0)):
        ids, logprobs = ops.sample(logits, u, **wish)
        assert torch.equal(ids.long(), place) and (logprobs.view(torch.int32) == 0).all(), wish
    # all but the least that numbers tell apart
    logits.fill_(-36.0)
    logits[torch.arange(n, device="cuda"), place] = 0.0
    for wish in (dict(), dict(top_k=1), dict(top_p=0.9), dict(temperature=0.2)):
        assert (ops.sample(logits, u, **wish)[1] <= 0).all(), wish


# ---- tables in 4 bits -----------------------------------------------------------------------
def test_a_table_is_a_constant(ops):
    """Of weights that are being trained, and of no dual ones."""
    weight = randn(gen(1), 40, 64)
    want = ops.quantize_table(weight).data
    assert torch.equal(ops.quantize_table(torch.nn.Parameter(weight)).data, want)
    codes, scales = torch.zeros(40, 64, dtype=torch.uint8, device="cuda"), torch.ones(40, 1, device="cuda").to(BF16)
    with forward_ad.dual_level():
        for call in (lambda: ops.quantize_table(forward_ad.make_dual(weight, weight)), lambda: ops.pack_table(codes, forward_ad.make_dual(scales, scales))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


# ---- penalties, biases, masks -----------------------------------------------------------------
def test_one_row_in_place_through_two_views(ops):
    """The last positions of one text: a view of [1, positions, vocab] and one of a single row have different strides."""
    room = randn(gen(2), 1, 3, 1001)
    logits, out = room[:, -1], room[0, -1:]
    allowed = torch.randint(-2 ** 31, 2 ** 31, (32,), generator=gen(3), device="cuda", dtype=torch.int64).int()
    want = ops.adjust_logits(logits, allowed=allowed)
    rest = room[:, :-1].clone()
    assert logits.stride() != out.stride() and ops.adjust_logits(logits, allowed=allowed, out=out) is out
    assert torch.equal(out, want) and torch.equal(room[:, :-1], rest) and torch.isinf(want).any()


# ---- together -----------------------------------------------------------------------------------
@pytest.mark.parametrize("where", ["INTEGRATION.md", "docstring"])
def test_the_step_that_is_shown_runs(ops, where):
    """As it is written, for two requests of which one's mask leaves nothing, and ids that are not whole characters."""
    from conftest import ROOT, tiny_vocab
    from graphtok_b200.gpu_bpe_tokenizer import Tokenizer
    if where == "docstring":
        lines = [line for line in ops.__doc__.splitlines() if line.startswith("    ")]
        shown = textwrap.dedent("\n".join(lines))
    else:
        with open(os.path.join(ROOT, where)) as f:
            shown = next(block.split("```")[0] for block in f.read().split("```python\n") if "next_ops.sample" in block.split("```")[0])
    tok = Tokenizer(tiny_vocab("llama3"))
    ids, offsets = tok.encode_batch_to_device(["some text to go on from", "and another one"])
    some = next(i for i in range(tok.vocab_size) if tok.decode_bytes([i])[0] >= 0x80)
    weight = randn(gen(5), tok.vocab_size, 64) * 0.3
    masks = torch.zeros(2, -(-tok.vocab_size // 32), dtype=torch.int32, device="cuda")
    masks[0, some // 32] = 1 << (some % 32) if some % 32 < 31 else -2 ** 31
    names = dict(vars(ops), next_ops=ops, torch=torch, tokenizer=tok, ids=ids, offsets=offsets, hidden=randn(gen(6), 2, 64).to(BF16), out_table=weight, answers=[[], []], masks=masks,
                 states=torch.arange(2, dtype=torch.int32, device="cuda"), prompts=offsets.diff().int(), heat=torch.ones(2, device="cuda"))
    if where == "docstring":
        names["tokenizer"].decode = tok.decode_bytes           # (of a whole answer, which one id is not)
    exec(shown, names)
    answers = names["answers"]
    if where == "docstring":
        assert [len(a) for a in answers] == [1, 1] and names["text"] == tok.decode_bytes(answers[0])
    else:
        assert answers == [[some], []] and names["part"] == tok.decode_bytes([some]) and names["new"].tolist() == [some, -1] and names["logprobs"].tolist() == [0.0, -math.inf]


@pytest.mark.parametrize("zeros", [False, True])
def test_groups_whose_scale_is_too_large(ops, zeros):
    """Weights of fp32 beyond what scales in fp16 can say: NaN for the whole group, as where a weight is infinite, and the largest that can be said is."""
    weight = randn(gen(8), 64, 256)
    bad = weight.clone()
    least = 65520.0 * (15 if zeros else 7)                     # rounds to infinity in fp16, what is below does not
    bad[3, 64:128] = least * 1.0001
    bad[40, 192] = -1e38
    weight[3, 70] = weight[40, 200] = math.nan
    got, want = ops.quantize_table(bad, group=64, zeros=zeros, dtype=F16), ops.quantize_table(weight, group=64, zeros=zeros, dtype=F16)
    eye = torch.eye(256, device="cuda").half()
    rows = torch.zeros(64, dtype=torch.bool, device="cuda")
    rows[3] = rows[40] = True
    for table in (got, want):
        values = ops.table_logits(eye, table).T
        assert values[rows].isnan().all() and values[~rows].isfinite().all()
    assert torch.equal(got.data, want.data)                    # (a group that is NaN is one whatever it was)
    bad[3, 64:128] = least * 0.9999
    bad[40, 192] = 1.0
    values = ops.table_logits(eye, ops.quantize_table(bad, group=64, zeros=zeros, dtype=F16)).T
    assert values.isfinite().all() and ((values - bad).abs()[3, 64:128] <= 65504.0 * (1.0 if zeros else 0.5) + least * 2.0 ** -11).all()


# ---- the largest, and what every share of a row takes part in ---------------------------------------
@pytest.mark.parametrize("n,vocab,dtype", [(1, 128256, BF16), (20, 50257, F32), (70, 9000, F16), (60, 100001, BF16), (251, 20000, BF16), (251, 50257, F32), (2, 600001, F32)])
def test_greedy_rows_in_every_number_of_blocks(ops, n, vocab, dtype):
    """The first of the largest, wherever it lies: at both ends, once and many times."""
    logits = randn(gen(n), n, vocab).to(dtype)
    rows = torch.arange(n, device="cuda")
    top = float(logits.max()) + 1
    logits[rows[::3], torch.randint(0, vocab, (len(rows[::3]),), generator=gen(n + 1), device="cuda")] = top
    logits[rows[1::3], vocab - 1] = top
    logits[::5, 0] = top
    u = torch.rand(n, generator=gen(n + 2), device="cuda")
    want = (logits == logits.amax(1, keepdim=True)).int().argmax(1)
    shares = torch.log_softmax(logits.double(), 1)[rows, want]
    for wish, logprobs in ((dict(temperature=0.0), torch.zeros_like(shares)), (dict(temperature=0.0, top_k=5, top_p=0.5, min_p=0.3), torch.zeros_like(shares)), (dict(top_k=1), shares),
                           (dict(top_p=0.0), shares), (dict(min_p=1.5), shares)):
        ids, got = ops.sample(logits, u, **wish)
        assert torch.equal(ids.long(), want), wish
        # (2^-25 of the total in whole numbers; the softmax in 64 bits)
        assert ((got.double() - logprobs).abs() <= logprobs.abs() * 2.0 ** -24 * 1.01 + 1.01 * 2.0 ** -25).all(), wish


def test_as_many_rows_as_there_may_be(ops):
    n = 1 << 20
    logits = randn(gen(4), n, 3)
    u = torch.rand(n, generator=gen(5), device="cuda", dtype=torch.float64)
    ids, _ = ops.sample(logits, u)
    ends = torch.softmax(logits.double(), 1).cumsum(1)
    sure = (ends - u[:, None]).abs().amin(1) > 1e-9              # (the others are borders, of which 64 bits may say either)
    assert torch.equal(ids.long()[sure], (ends <= u[:, None]).sum(1)[sure]) and sure.sum() > n - 100
    allowed = torch.randint(0, 8, (n, 1), generator=gen(6), device="cuda").int()
    got = ops.adjust_logits(logits, torch.arange(n, device="cuda").int() % 3, torch.arange(n + 1, device="cuda").int(), presence=1.0, allowed=allowed)
    want = logits.clone()
    want[torch.arange(n, device="cuda"), torch.arange(n, device="cuda") % 3] -= 1
    assert torch.equal(got, want.masked_fill((allowed >> torch.arange(3, device="cuda").int()) % 2 == 0, -math.inf))
    more = torch.zeros(n + 1, 1, device="cuda")
    for call in (lambda: ops.sample(more, more[:, 0]), lambda: ops.adjust_logits(more)):
        with pytest.raises(ValueError, match="2\\^20"):
            call()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adjust_logits_of_the_largest_vocabulary(ops, dtype):
    n, vocab = 2, 1 << 24
    logits = randn(gen(7), n, vocab).to(dtype)
    ends = torch.tensor([0, 1, 15, 16383, 16384, 16391, vocab // 2, vocab - 16385, vocab - 9, vocab - 1], dtype=torch.int32, device="cuda")
    ids = torch.cat([ends, ends, ends.flip(0), torch.randint(0, vocab, (5000,), generator=gen(8), device="cuda").int()])
    allowed = torch.randint(-2 ** 31, 2 ** 31, (1, vocab // 32), generator=gen(9), device="cuda", dtype=torch.int64).int()
    bias = torch.arange(10, device="cuda") * 0.5
    got = ops.adjust_logits(logits, ids, torch.tensor([0, 10, len(ids)], dtype=torch.int32, device="cuda"), frequency=0.25, bias_ids=ends, bias=bias, allowed=allowed,
                            allowed_rows=torch.tensor([-1, 0], dtype=torch.int32, device="cuda"))
    want = logits.float()
    for r, some in enumerate((ids[:10], ids[10:])):
        want[r] -= 0.25 * torch.bincount(some, minlength=vocab)
        want[r, ends.long()] += bias
    bit = (allowed[0, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32) & 1).flatten() != 0
    want[1].masked_fill_(~bit, -math.inf)
    # (frequencies and biases are quarters: one rounding of fp32 at each of two steps, in the same order, and one to the type)
    assert torch.equal(got, want.to(dtype))


@pytest.mark.parametrize("n", [1, 12, 40])
def test_tables_of_more_than_4_gib(ops, n):
    """Places of codes and scales beyond 32 bits: rows all over the table against the formula."""
    vocab, width = (1 << 23) + 77, 1024
    codes = torch.randint(0, 16, (vocab, width), generator=gen(10), device="cuda", dtype=torch.uint8)
    scales = (torch.rand(vocab, width // 64, generator=gen(11), device="cuda") + 0.5).to(BF16)
    table = ops.pack_table(codes, scales, group=64)
    assert table.data.numel() > 1 << 32
    hidden = randn(gen(12), n, width).to(BF16)
    rows = torch.cat([torch.arange(2000, device="cuda"), torch.randint(0, vocab, (4000,), generator=gen(13), device="cuda"), torch.arange(vocab - 2000, vocab, device="cuda")])
    got = ops.table_logits(hidden, table)[:, rows]
    values = scales[rows].double().repeat_interleave(64, 1) * (codes[rows].double() - 8)
    check_logits(got, hidden, values, 64)


@pytest.mark.parametrize("n,vocab", [(6, 600001), (6, (1 << 21) + 5)])
def test_rows_with_units_of_their_own(ops, n, vocab):
    """More than 2^19 ids: all alike, infinities, lowest values, few ids left, nothing left and a NaN, in one call."""
    g = gen(vocab)
    logits = randn(g, n, vocab) * 3
    logits[0] = 2.5
    logits[1, torch.randint(0, vocab, (1000,), generator=g, device="cuda")] = math.inf
    logits[2] = torch.where(torch.rand(vocab, generator=g, device="cuda") < 1e-4, logits[2], torch.finfo(F32).min)
    logits[3] = -math.inf
    logits[4, vocab // 2] = math.nan
    u = torch.tensor([0.3, 0.71, 0.5, 0.5, 0.5, 0.93], device="cuda")
    for wish in ((1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.0, 0, 0.75, 0.0), (1.0, 100000, 1.0, 0.0), (1.5, 0, 1.0, 0.02), (1e-30, 0, 0.9, 0.0), (1e30, 0, 0.4, 0.0), (1.0, 1, 1.0, 0.0)):
        check_draw(ops, logits, u, *wish)
