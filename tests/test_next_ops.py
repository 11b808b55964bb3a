"""The operators from hidden states to ids against their formulas in 64 bits, on a B200.

How far a result may be off is counted from roundings: u = eps / 2 of a type is half a step relative to the value.  A sum of tensor-core
products loses at most a step of fp32 (2^-23) of its largest partial sum every 16 elements."""
import math

import pytest
import torch

from test_vocab_ops import BF16, F16, F32, gen, half_step, randn, within

pytestmark = pytest.mark.gpu

LEAST = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -25}          # what rounding takes from numbers below the normal ones


@pytest.fixture(scope="module")
def ops(built):
    from graphtok_b200 import next_ops
    return next_ops


# ---- tables in 4 bits -------------------------------------------------------------
def spread(t, group, width):
    return t.double().repeat_interleave(group, 1)[:, :width]


def make_table(seed, vocab, width, group, dtype, zeros):
    g = gen(seed)
    codes = torch.randint(0, 16, (vocab, width), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand(vocab, -(-width // group), generator=g, device="cuda") * 0.1 + 0.01).to(dtype)
    scales *= torch.where(torch.rand(scales.shape, generator=g, device="cuda") < 0.1, -1, 1).to(dtype)
    z = torch.randint(0, 16, scales.shape, generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    values = spread(scales, group, width) * (codes.double() - (8 if z is None else spread(z, group, width)))
    return codes, scales, z, values


def check_logits(got, hidden, values, group):
    h = hidden.double()
    want = h @ values.T
    size = h.abs() @ values.abs().T
    width = values.shape[1]
    tol = size * ((width + 15) // 16 + -(-width // group) + 20) * 2.0 ** -23
    if got.dtype != F32:
        tol = tol + want.abs() * half_step(got.dtype) * 1.01 + LEAST[got.dtype]
    within(got, want, tol, "logits")


SHAPES = [(1, 1, 1), (1, 31, 64), (2, 32, 63), (3, 33, 65), (7, 100, 128), (8, 1000, 200), (9, 257, 320), (15, 5003, 1000), (16, 64, 1024), (17, 777, 130), (31, 4096, 512),
          (33, 300, 2049), (47, 9001, 96), (64, 1024, 4096), (65, 129, 256), (127, 2000, 333), (128, 515, 640), (129, 258, 257), (300, 4801, 72), (5, 70000, 64), (4, 40, 13000),
          (40, 40, 13000), (1, 300, 65536), (12, 129, 8192), (20, 4000, 7)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,vocab,width", SHAPES)
def test_table_logits(ops, n, vocab, width, dtype):
    for group, zeros in ((32, False), (64, True), (128, False), (32, True), (192, True), (8192, False)):
        codes, scales, z, values = make_table(n + vocab + width + group, vocab, width, group, dtype, zeros)
        hidden = randn(gen(n), n, width).to(dtype)
        table = ops.pack_table(codes, scales, z, group=group)
        assert table.shape == (vocab, width)
        check_logits(ops.table_logits(hidden, table), hidden, values, group)
        if group == 64:
            got = ops.table_logits(hidden, table, dtype=dtype)
            assert got.dtype == dtype
            check_logits(got, hidden, values, group)


@pytest.mark.parametrize("n", [1, 5, 16, 40, 130])
def test_rows_do_not_touch_one_another(ops, n):
    """NaN and infinities in one row stay there, and a row is the same whatever else is in the batch of its size; calls repeat to the bit."""
    codes, scales, z, _ = make_table(3, 1500, 500, 64, BF16, True)
    table = ops.pack_table(codes, scales, z, group=64)
    hidden = randn(gen(4), n, 500).to(BF16)
    want = ops.table_logits(hidden, table)
    assert torch.equal(want, ops.table_logits(hidden, table))
    for bad in (math.nan, math.inf, -math.inf):
        other = hidden.clone()
        other[n // 2, 17] = bad
        got = ops.table_logits(other, table)
        keep = torch.arange(n, device="cuda") != n // 2
        assert torch.equal(got[keep], want[keep]) and not got[n // 2].isfinite().any()


def test_strides_offsets_and_shapes_of_hidden_states(ops):
    codes, scales, z, values = make_table(5, 700, 300, 128, F16, False)
    strided = torch.zeros(700, 900, dtype=torch.uint8, device="cuda")
    strided[:, 37:337] = codes
    wide = torch.zeros(700, 11, dtype=F16, device="cuda")
    wide[:, 4:7] = scales
    table = ops.pack_table(strided[:, 37:337], wide[:, 4:7], group=128)
    assert torch.equal(table.data, ops.pack_table(codes, scales, group=128).data)
    assert torch.equal(table.data, ops.pack_table(codes.t().contiguous().t(), scales, group=128).data)
    big = randn(gen(6), 6, 20, 301).to(F16)
    for hidden in (big[:, :, 1:], big[0, :, :300], big[2:3, 1:2, :300], big[0, 0, 1:], big[:, 0, :300], big[1, :1, :300].expand(9, 300), big[0, :, :300].contiguous().t().contiguous().t()):
        got = ops.table_logits(hidden, table)
        assert got.shape == (*hidden.shape[:-1], 700)
        check_logits(got.reshape(-1, 700), hidden.reshape(-1, 300), values, 128)
    assert ops.table_logits(big[:0, 0, :300], table).shape == (0, 700)
    # another storage offset: rows at odd addresses
    flat = randn(gen(7), 4 * 300 + 3).to(F16)
    check_logits(ops.table_logits(flat[3:].view(4, 300), table), flat[3:].view(4, 300), values, 128)


def quantized(weight, group, zeros, dtype):
    """(codes, scales, zeros) from the formulas; quotients in 64 bits and then 32, which is the quotient rounded once to 32 (torch divides by a number by multiplying with its inverse)."""
    over = lambda a, b: (a.double() / b).float()       # noqa: E731
    vocab, width = weight.shape
    groups = -(-width // group)
    w = torch.zeros(vocab, groups * group, device="cuda")
    w[:, :width] = weight.float()
    w = w.view(vocab, groups, group)
    if zeros:
        low, high = w.amin(2).clamp(max=0), w.amax(2).clamp(min=0)
        s = (over(high, 15) - over(low, 15)).to(dtype).float()
        b = torch.where(s > 0, over(-low, s).round().clamp(0, 15), 0.0)
    else:
        s = over(w.abs().amax(2), 7).to(dtype).float()
        b = torch.full_like(s, 8)
    q = torch.where(s[:, :, None] > 0, (over(w, s[:, :, None]).round() + b[:, :, None]).clamp(0, 15), 0)
    return q.flatten(1)[:, :width].to(torch.uint8), s.to(dtype), b.to(torch.uint8)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("source,dtype", [(F32, BF16), (BF16, BF16), (F16, F16), (F32, F16), (BF16, F16)])
@pytest.mark.parametrize("vocab,width,group", [(1, 1, 32), (40, 64, 32), (33, 100, 64), (100, 1000, 128), (65, 700, 192), (31, 3000, 1024), (10, 5000, 8192), (2000, 96, 64)])
def test_quantize_table(ops, vocab, width, group, source, dtype, zeros):
    weight = (randn(gen(vocab), vocab, width) * 0.05 + (0.03 if zeros else 0)).to(source)
    if vocab > 8:
        weight[2] = 0
        weight[3] = weight[3].abs()
        weight[4] = -weight[4].abs()
        weight[5, ::3] = 0.25
    table = ops.quantize_table(weight, group=group, zeros=zeros, dtype=dtype)
    codes, scales, b = quantized(weight, group, zeros, dtype)
    want = ops.pack_table(codes, scales, b if zeros else None, group=group)
    # what the parts beyond the last row and column hold does not matter
    eye = torch.eye(width, device="cuda").to(dtype)
    got, want = ops.table_logits(eye, table), ops.table_logits(eye, want)
    # a quotient next to a tie may round to either side of it: nowhere else may a code differ
    step = spread(scales, group, width).T.abs()
    assert (((got - want).abs() / step.clamp(min=1e-30)).round() <= 1).all() and (got != want).double().mean() < 1e-3
    off = (got.double().T - weight.double()).abs()
    # half a step, a step at the ends where scale or zero have been rounded, and what rounding the scale makes of 15 steps
    limit = spread(scales, group, width) * (1.0 if zeros else 0.5) + 16 * spread(scales, group, width) * half_step(dtype) + 2.0 ** -23
    assert (off <= limit * 1.001).all()


def test_quantized_groups_that_are_not_finite(ops):
    weight = randn(gen(1), 64, 256)
    weight[3, 70], weight[5, 0], weight[40, 255] = math.nan, math.inf, -math.inf
    for zeros in (False, True):
        table = ops.quantize_table(weight, group=64, zeros=zeros)
        values = ops.table_logits(torch.eye(256, device="cuda").to(BF16), table).T
        bad = torch.zeros(64, 4, dtype=torch.bool, device="cuda")
        bad[3, 1] = bad[5, 0] = bad[40, 3] = True
        # (a hidden state of 0 times NaN is NaN: the whole row)
        assert values[bad.any(1)].isnan().all() and values[~bad.any(1)].isfinite().all()


# ---- penalties, biases, masks --------------------------------------------------------
def adjusted(logits, rows, repetition, presence, frequency, biases, masks):
    """(what should come, how far it may be off, which logits may change) from lists: rows of (prompt ids, further ids), of (id, bias), of allowed ids or None."""
    x = logits.double().cpu()
    size = x.abs()
    touched = torch.zeros(x.shape, dtype=torch.bool)
    roundings = torch.zeros(x.shape, dtype=torch.float64)
    n, vocab = x.shape
    for i in range(n):
        prompt, rest = rows[i]
        count = {}
        for v in rest:
            if 0 <= v < vocab:
                count[v] = count.get(v, 0) + 1
        for v in set(prompt) | set(rest):
            if 0 <= v < vocab:
                rho = float(repetition[i])
                x[i, v] = x[i, v] / rho if x[i, v] > 0 else x[i, v] * rho
                size[i, v] = x[i, v].abs()
                touched[i, v] = True
                roundings[i, v] += 1
                if v in count:
                    x[i, v] = x[i, v] - float(frequency[i]) * count[v] - float(presence[i])
                    size[i, v] += abs(float(frequency[i])) * count[v] + abs(float(presence[i]))
                    roundings[i, v] += 3
        for v, b in biases[i]:
            if 0 <= v < vocab:
                x[i, v] += b
                size[i, v] += abs(b)
                touched[i, v] = True
                roundings[i, v] += 1
        if masks[i] is not None:
            out = torch.ones(vocab, dtype=torch.bool)
            out[list(masks[i])] = False
            x[i, out] = -math.inf
            touched[i, out] = True
    u = half_step(logits.dtype)
    tol = roundings * 2.0 ** -24 * torch.nan_to_num(size, posinf=0) + torch.where(touched, torch.nan_to_num(x, posinf=0, neginf=0).abs() * u * 1.01 + LEAST[logits.dtype], 0.0)
    return x.cuda(), tol.cuda(), touched.cuda()


def pack_bits(masks, vocab):
    words = -(-vocab // 32)
    bits = torch.zeros(len(masks), words * 32, dtype=torch.int64)
    for i, m in enumerate(masks):
        bits[i, list(m)] = 1
    whole = (bits.view(len(masks), words, 32) << torch.arange(32)).sum(2)
    return torch.where(whole >= 2 ** 31, whole - 2 ** 32, whole).int().cuda()


def close(got, want, tol):
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf].double(), want[inf])
    within(torch.where(inf, 0.0, got.double()), torch.where(inf, 0.0, want), tol, "logits")


def a_batch(seed, n, vocab, longest, entries, dtype, share_masks):
    import random
    rng = random.Random(seed)
    pick = lambda: rng.choice((rng.randrange(vocab), rng.randrange(min(vocab, 9)), rng.randrange(vocab)))     # noqa: E731
    rows = []
    for i in range(n):
        length = rng.choice((0, 1, longest, rng.randint(0, longest)))
        ids = [pick() for _ in range(length)]
        for _ in range(length // 50):
            ids[rng.randrange(length)] = rng.choice((-1, vocab, vocab + 5, -2 ** 31, 2 ** 31 - 1))
        cut = rng.choice((0, length, rng.randint(0, length)))
        rows.append((ids[:cut], ids[cut:]))
    biases = [[(rng.choice((pick(), -1)), rng.choice((rng.gauss(0, 5), -100.0, -math.inf))) for _ in range(entries)] for _ in range(n)]
    for b in biases:
        if len(b) > 3:
            b[1] = (b[0][0], 1.5)              # the same id twice, and not next to one another
            b[-1] = (b[0][0], -0.25)
    masks = [rng.choice((None, set(), {0}, {vocab - 1}, {v for v in range(vocab) if rng.random() < 0.5})) for _ in range(n)]
    logits = (randn(gen(seed), n, vocab) * 6).to(dtype)
    return rows, biases, masks, logits, [1 + rng.random() for _ in range(n)], [rng.uniform(-1, 2) for _ in range(n)], [rng.uniform(-1, 1) for _ in range(n)]


def arguments(rows, biases, masks, n, vocab, bits):
    flat = [v for a, b in rows for v in a + b]
    offsets = [0]
    for a, b in rows:
        offsets.append(offsets[-1] + len(a) + len(b))
    named = dict(ids=torch.tensor(flat, dtype=torch.int64).to(bits).cuda(), offsets=torch.tensor(offsets, dtype=torch.int32).cuda(),
                 prompt_lengths=torch.tensor([len(a) for a, _ in rows], dtype=torch.int32).cuda())
    if biases[0]:
        named |= dict(bias_ids=torch.tensor([[v for v, _ in b] for b in biases], dtype=torch.int32).cuda(), bias=torch.tensor([[x for _, x in b] for b in biases]).cuda())
    real = [m for m in masks if m is not None]
    if real:
        places, k = [], 0
        for m in masks:
            places.append(-1 if m is None else k)
            k += m is not None
        named |= dict(allowed=pack_bits(real, vocab), allowed_rows=torch.tensor(places, dtype=torch.int32).cuda())
    return named


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,vocab,longest,entries", [(1, 1, 3, 0), (2, 31, 40, 5), (3, 32, 0, 1), (5, 33, 500, 4), (4, 2047, 100, 0), (3, 2048, 300, 7), (2, 2049, 100, 1024), (7, 5000, 2000, 20),
                                                      (1, 16384, 20, 3), (40, 1001, 60, 3), (2, 40001, 5000, 33), (150, 2100, 9, 2)])
def test_adjust_logits(ops, n, vocab, longest, entries, dtype):
    rows, biases, masks, logits, rho, presence, frequency = a_batch(n * vocab, n, vocab, longest, entries, dtype, False)
    column = lambda v: torch.tensor(v, device="cuda")          # noqa: E731
    want, tol, touched = adjusted(logits, rows, column(rho).double(), column(presence).double(), column(frequency).double(),
                                  [[(v, float(torch.tensor(x, dtype=F32))) for v, x in b] for b in biases], masks)
    for bits in (torch.int32, torch.int64):
        named = arguments(rows, biases, masks, n, vocab, bits)
        before = logits.clone()
        got = ops.adjust_logits(logits, repetition=column(rho), presence=column(presence), frequency=column(frequency), **named)
        assert torch.equal(logits, before) and got.dtype == dtype
        close(got, want, tol)
        assert torch.equal(got[~touched], logits[~touched])
        # in place, and rows that lie apart at odd places: the same to the bit
        here = logits.clone()
        assert ops.adjust_logits(here, repetition=column(rho), presence=column(presence), frequency=column(frequency), out=here, **named) is here
        assert torch.equal(here, got)
        for left, right in ((1, 2), (0, 5), (3, 5)):
            room = torch.full((n, vocab + left + right), 7.0, device="cuda", dtype=dtype)
            view = room[:, left:left + vocab]
            view.copy_(logits)
            to = torch.full((n, vocab + 4), 9.0, device="cuda", dtype=dtype)
            ops.adjust_logits(view, repetition=column(rho), presence=column(presence), frequency=column(frequency), out=to[:, 2:2 + vocab], **named)
            assert torch.equal(to[:, 2:2 + vocab], got) and (to[:, :2] == 9).all() and (to[:, 2 + vocab:] == 9).all() and torch.equal(view, logits)
            ops.adjust_logits(view, repetition=column(rho), presence=column(presence), frequency=column(frequency), out=view, **named)
            assert torch.equal(view, got) and (room[:, :left] == 7).all() and (room[:, left + vocab:] == 7).all()


def test_one_number_for_all_and_one_list_for_all(ops):
    rows, biases, _, logits, _, _, _ = a_batch(8, 6, 3000, 200, 9, F32, False)
    masks = [{1, 5, 2999}] * 6
    want, tol, _ = adjusted(logits, rows, [float(torch.tensor(1.3))] * 6, [0.5] * 6, [0.25] * 6, [[(v, float(torch.tensor(x))) for v, x in biases[0]]] * 6, masks)
    named = arguments(rows, biases, masks, 6, 3000, torch.int32)
    named["bias_ids"], named["bias"] = named["bias_ids"][0], named["bias"][0]
    named["allowed"] = named["allowed"][0]
    del named["allowed_rows"]
    got = ops.adjust_logits(logits, repetition=1.3, presence=0.5, frequency=0.25, **named)
    close(got, want, tol)
    # without prompt lengths all of the history counts; masks of each row's own without allowed_rows
    del named["prompt_lengths"]
    named["allowed"] = named["allowed"].expand(6, -1).contiguous()
    want, tol, _ = adjusted(logits, [([], a + b) for a, b in rows], [float(torch.tensor(1.3))] * 6, [0.5] * 6, [0.25] * 6, [[(v, float(torch.tensor(x))) for v, x in biases[0]]] * 6, masks)
    close(ops.adjust_logits(logits, repetition=1.3, presence=0.5, frequency=0.25, **named), want, tol)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_nothing_asked_for_is_a_copy(ops, dtype):
    logits = randn(gen(1), 5, 4001).to(dtype)
    logits[1, 3], logits[2, 4], logits[3, 5], logits[0, 0] = math.nan, math.inf, -math.inf, -0.0
    got = ops.adjust_logits(logits)
    assert got.data_ptr() != logits.data_ptr() and torch.equal(got.view(torch.uint8), logits.view(torch.uint8))
    assert torch.equal(ops.adjust_logits(logits, out=logits).view(torch.uint8), got.view(torch.uint8))
    assert ops.adjust_logits(logits[:0]).shape == (0, 4001)


def test_masked_places_hold_anything(ops):
    """NaN, infinities and the type's lowest value where nothing is allowed become -inf; what is allowed stays; a mask that is not there allows nothing."""
    logits = torch.tensor([[math.nan, math.inf, -math.inf, torch.finfo(F32).min, 1.0, math.nan]], device="cuda").repeat(4, 1)
    allowed = pack_bits([{4, 5}], 6)
    got = ops.adjust_logits(logits, allowed=allowed, allowed_rows=torch.tensor([0, -1, 1, -7], dtype=torch.int32, device="cuda"))
    assert torch.equal(got[0, :5], torch.tensor([-math.inf] * 4 + [1.0], device="cuda")) and got[0, 5].isnan()
    for r in (1, 3):
        assert torch.equal(got[r].view(torch.int32), logits[r].view(torch.int32))
    assert (got[2] == -math.inf).all()
    empty = torch.empty(0, 1, dtype=torch.int32, device="cuda")
    assert (ops.adjust_logits(logits, allowed=empty, allowed_rows=torch.tensor([0, 0, 0, -1], dtype=torch.int32, device="cuda"))[:3] == -math.inf).all()


def test_offsets_that_lead_outside_are_held_to_the_ids(ops):
    logits = randn(gen(2), 3, 100)
    ids = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")
    got = ops.adjust_logits(logits, ids, torch.tensor([-4, 1, 2, 900], dtype=torch.int32, device="cuda"), presence=1.0)
    want = logits.clone()
    for r, v in ((0, 5), (1, 6), (2, 7)):
        want[r, v] -= 1
    assert torch.equal(got, want)


def test_a_long_history_of_one_id(ops):
    logits = torch.ones(2, 300, device="cuda")
    ids = torch.full((300000,), 7, dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 200001, 300000], dtype=torch.int32, device="cuda")
    got = ops.adjust_logits(logits, ids, offsets, frequency=0.5, prompt_lengths=torch.tensor([1, 0], dtype=torch.int32, device="cuda"))
    assert got[:, 7].tolist() == [1 - 0.5 * 200000, 1 - 0.5 * 99999] and (got[:, :7] == 1).all() and (got[:, 8:] == 1).all()


# ---- an id a row -----------------------------------------------------------------------
def drawn(logits, u, temperature, top_k, top_p, min_p):
    """(ids, logprobs) by the definition, in 64 bits on the host, a row at a time."""
    ids, logs = [], []
    x = logits.double().cpu()
    for i in range(x.shape[0]):
        t, k, p, m, ui = float(temperature[i]), int(top_k[i]), float(top_p[i]), float(min_p[i]), float(u[i])
        row = x[i]
        top = row.max()
        if row.isnan().any() or not (0 <= t < math.inf) or not (0 <= ui < 1) or p != p or m != m:
            ids.append(-1), logs.append(math.nan)
            continue
        if top == -math.inf:
            ids.append(-1), logs.append(-math.inf)
            continue
        order = torch.sort(row, descending=True, stable=True).indices
        if t == 0:
            ids.append(int(order[0])), logs.append(0.0)
            continue
        mass = (row == top).double() if top == math.inf else torch.exp((row - top) / t)
        order = order[row[order] > -math.inf]
        if k > 0:
            order = order[:k]
        if p < 1:
            run = mass[order].cumsum(0)
            before = torch.cat([torch.zeros(1, dtype=torch.float64), run[:-1]])
            order = order[:max(1, int((before < p * run[-1]).sum()))]
        if m > 0:
            order = order[:max(1, int((mass[order] >= m).sum()))]
        kept = order.sort().values
        run = mass[kept].cumsum(0)
        at = int(kept[torch.searchsorted(run, ui * run[-1], right=True).clamp(max=kept.numel() - 1)])
        ids.append(at), logs.append(float(torch.log(mass[at] / mass.sum())))
    return torch.tensor(ids, dtype=torch.int32), torch.tensor(logs, dtype=torch.float64)


def check_draw(ops, logits, u, temperature, top_k, top_p, min_p):
    n = logits.shape[0]
    column = lambda v, t: v if isinstance(v, torch.Tensor) else torch.full((n,), v, dtype=t, device="cuda")      # noqa: E731
    temperature, top_k, top_p, min_p = column(temperature, F32), column(top_k, torch.int32), column(top_p, F32), column(min_p, F32)
    ids, logprobs = ops.sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    want, logs = drawn(logits, u, temperature, top_k, top_p, min_p)
    assert ids.dtype == torch.int32 and logprobs.dtype == F32
    assert torch.equal(ids.cpu(), want), (ids.cpu() != want).nonzero().flatten().tolist()[:10]
    # masses are off by 2^-40 relative or a unit of their sum's 2^-38; the rest is the rounding to fp32
    got = logprobs.cpu().double()
    inf = torch.isinf(logs)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got.isnan(), logs.isnan())
    off = torch.nan_to_num((got - logs).abs(), nan=0.0)[~inf]
    assert (off <= torch.nan_to_num(logs.abs())[~inf] * 2.0 ** -24 * 1.01 + 2.0 ** -30).all()
    return ids


def model_logits(seed, n, vocab, dtype, sharp=1.8):
    g = gen(seed)
    x = randn(g, n, vocab) * sharp
    x[:, torch.randint(0, vocab, (30,), generator=g, device="cuda")] += 6 * torch.rand(n, 30, generator=g, device="cuda")
    return x.to(dtype)


WISHES = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.8, 40, 0.95, 0.0), (1.3, 0, 1.0, 0.05), (0.9, 20, 0.8, 0.1), (0.0, 5, 0.5, 0.5), (1.0, 1, 1.0, 0.0), (0.01, 0, 0.9, 0.0),
          (3.0, 0, 0.5, 0.0), (100.0, 700, 0.3, 0.0), (1.0, 10 ** 6, 0.999, 1e-6), (2.0, 300, 0.9999, 0.0), (0.6, 0, 1e-9, 0.0), (1.0, 3, 1.0, 1.0), (1.0, -5, 1.5, -1.0), (1.0, 0, 0.0, 0.0),
          (1.0, 0, -3.0, 0.0), (1.0, 0, 1.0, 2.0), (1e-30, 0, 0.9, 0.1), (1e30, 0, 0.4, 0.0)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,vocab", [(1, 1), (3, 2), (9, 31), (5, 33), (6, 1000), (4, 4096), (3, 4097), (2, 50256), (7, 20011)])
def test_sample(ops, n, vocab, dtype):
    for i, wish in enumerate(WISHES):
        logits = model_logits(100 * i + n, n, vocab, dtype)
        check_draw(ops, logits, torch.rand(n, generator=gen(i), device="cuda"), *wish)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_their_own_wishes(ops, dtype):
    n = 4 * len(WISHES)
    logits = model_logits(5, n, 30011, dtype)
    logits[::3] = logits[::3].masked_fill(torch.rand(logits[::3].shape, generator=gen(6), device="cuda") < 0.99, -math.inf)
    logits[7], logits[8, 5], logits[9, 77] = -math.inf, math.nan, math.inf
    t, k, p, m = (torch.tensor([w[j] for w in WISHES] * 4, device="cuda") for j in range(4))
    check_draw(ops, logits, torch.rand(n, generator=gen(7), device="cuda"), t.float(), k.int(), p.float(), m.float())


def test_numbers_are_the_same_as_tensors(ops):
    logits = model_logits(3, 6, 5000, F32)
    u = torch.rand(6, generator=gen(4), device="cuda")
    for t, k, p, m in WISHES:
        one = ops.sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)
        all_ = ops.sample(logits, u, temperature=torch.full((6,), t, device="cuda"), top_k=torch.full((6,), k, device="cuda", dtype=torch.int32),
                          top_p=torch.full((6,), p, device="cuda"), min_p=torch.full((6,), m, device="cuda"))
        assert torch.equal(one[0], all_[0]) and torch.equal(one[1], all_[1])


@pytest.mark.parametrize("value", [0.0, -3.5, 1e30, -1e-40, math.inf, -65504.0])
@pytest.mark.parametrize("vocab", [1, 7, 600, 5001, 40000])
def test_equal_logits_are_cut_in_the_order_of_ids(ops, vocab, value):
    logits = torch.full((8, vocab), value, device="cuda")
    logits[4:, : vocab // 3] = -math.inf
    u = torch.tensor([0.0, 0.25, 0.5, 1 - 2.0 ** -24] * 2, device="cuda")
    for wish in ((1.0, 0, 1.0, 0.0), (1.0, 300, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 5, 0.5, 0.0), (1.0, 0, 0.75, 1.0), (0.0, 0, 1.0, 0.0), (1.0, 4999, 0.25, 0.0)):
        check_draw(ops, logits, u, *wish)


def test_logits_of_every_size(ops):
    """Values over all of fp32's range, many next to 0, and steps of one unit in the last place at a cut."""
    g = gen(11)
    bits = torch.randint(-2 ** 31, 2 ** 31, (6, 20000), generator=g, device="cuda", dtype=torch.int64).int()
    anything = bits.view(F32)
    anything = torch.where(anything.isnan() | anything.isinf(), 0.0, anything)
    tiny = randn(g, 3, 20000) * 1e-39
    fine = torch.nextafter(torch.ones(3, 20000, device="cuda"), torch.tensor(2.0, device="cuda")) + torch.randint(0, 3000, (3, 20000), generator=g, device="cuda") * 2.0 ** -23
    zeros = torch.where(torch.rand(3, 20000, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    logits = torch.cat([anything, tiny, fine, zeros])
    u = torch.rand(15, generator=g, device="cuda")
    for wish in ((1.0, 0, 1.0, 0.0), (1.0, 777, 1.0, 0.0), (1e38, 0, 0.5, 0.0), (1e-39, 5000, 0.5, 0.0), (1e-3, 10000, 0.9, 0.0), (1.0, 12345, 0.37, 0.0)):
        check_draw(ops, logits, u, *wish)


@pytest.mark.parametrize("vocab,dtype", [(262144, F32), (300001, BF16), (700001, F32), (1 << 20, F16)])
def test_large_vocabularies(ops, vocab, dtype):
    logits = model_logits(vocab, 3, vocab, dtype)
    u = torch.tensor([0.1, 0.5, 0.9999], device="cuda")
    for wish in ((1.0, 0, 1.0, 0.0), (0.8, 50, 0.9, 0.0), (1.2, 0, 0.9, 0.0)):
        check_draw(ops, logits, u, *wish)


def test_random_numbers_at_their_ends(ops):
    logits = model_logits(8, 6, 3000, F32)
    logits[0, 0] = logits[1, 0] = -math.inf
    u = torch.tensor([0.0, 0.0, 1 - 2.0 ** -53, 1.0, -0.1, math.nan], dtype=torch.float64, device="cuda")
    for wish in ((1.0, 0, 1.0, 0.0), (0.5, 30, 0.9, 0.0), (0.0, 0, 1.0, 0.0)):
        ids = check_draw(ops, logits, u, *wish)
        assert ids[3:].tolist() == [-1, -1, -1]


def test_bad_wishes_of_a_row_are_that_row_s(ops):
    logits = model_logits(9, 7, 2000, F32)
    nan, inf = math.nan, math.inf
    t = torch.tensor([-1.0, nan, inf, 1, 1, 1, 1], device="cuda")
    p = torch.tensor([0.9, 0.9, 0.9, nan, 0.9, 0.9, inf], device="cuda")
    m = torch.tensor([0.0, 0, 0, 0, nan, 0, -inf], device="cuda")
    ids = check_draw(ops, logits, torch.full((7,), 0.3, device="cuda"), t, 0, p, m)
    assert (ids[:5] == -1).all() and (ids[5:] >= 0).all()


def test_strides_of_logits(ops):
    base = model_logits(12, 9, 4001, F32)
    u = torch.rand(9, generator=gen(13), device="cuda")
    want = ops.sample(base, u, top_p=0.9)
    room = torch.zeros(9, 4010, device="cuda")
    room[:, 3:4004] = base
    for view in (room[:, 3:4004], base.t().contiguous().t()):
        got = ops.sample(view, u, top_p=0.9)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    same = ops.sample(base[2:3].expand(5, 4001), u[2:3].expand(5), top_p=0.9)
    assert (same[0] == want[0][2]).all()
    none = ops.sample(base[:0], u[:0])
    assert none[0].shape == (0,) and none[1].shape == (0,)


# ---- together ----------------------------------------------------------------------------
def a_step(ops, hidden, table, ids, offsets, u, allowed):
    logits = ops.table_logits(hidden, table)
    ops.adjust_logits(logits, ids, offsets, repetition=1.2, frequency=0.1, allowed=allowed, out=logits)
    return (logits, *ops.sample(logits, u, temperature=0.8, top_k=100, top_p=0.9))


def step_inputs(seed, n=5, vocab=9001, width=320):
    g = gen(seed)
    hidden = randn(g, n, width).to(BF16)
    ids = torch.randint(0, vocab, (n * 40,), generator=g, device="cuda").int()
    offsets = (torch.arange(n + 1, device="cuda") * 40).int()
    allowed = torch.randint(-2 ** 31, 2 ** 31, (n, -(-vocab // 32)), generator=g, device="cuda", dtype=torch.int64).int()
    return hidden, ids, offsets, torch.rand(n, generator=g, device="cuda"), allowed


def test_a_decoding_step(ops):
    """From hidden states to ids, as a server runs it: against the formulas, and every id allowed."""
    weight = randn(gen(20), 9001, 320) * 0.06
    table = ops.quantize_table(weight)
    hidden, ids, offsets, u, allowed = step_inputs(21)
    logits, got, _ = a_step(ops, hidden, table, ids, offsets, u, allowed)
    column = lambda v, t=F32: torch.full((5,), v, dtype=t, device="cuda")           # noqa: E731
    want, _ = drawn(logits, u, column(0.8), column(100, torch.int32), column(0.9), column(0.0))
    assert torch.equal(got.cpu(), want)
    codes, scales, _ = quantized(weight, 128, False, BF16)
    values = spread(scales, 128, 320) * (codes.double() - 8)
    z = hidden.double() @ values.T
    for i in range(5):
        some = torch.unique(ids[40 * i:40 * i + 40].long(), return_counts=True)
        z[i, some[0]] = torch.where(z[i, some[0]] > 0, z[i, some[0]] / 1.2, z[i, some[0]] * 1.2) - 0.1 * some[1]
        bit = (allowed[i].long()[:, None] >> torch.arange(32, device="cuda") & 1).flatten()[:9001] != 0
        z[i, ~bit] = -math.inf
        assert bit[got[i].long()]
    assert torch.equal(torch.isinf(z), torch.isinf(logits)) and (logits.double() - z)[~torch.isinf(z)].abs().max() < 0.05


def test_captured_and_replayed_steps(ops):
    table = ops.quantize_table(randn(gen(30), 9001, 320) * 0.06, zeros=True)
    first, second = step_inputs(31), step_inputs(32)
    want = [a_step(ops, i[0], table, *i[1:]) for i in (first, second)]
    held = [t.clone() for t in first]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a_step(ops, held[0], table, *held[1:])
    for inputs, w in ((second, want[1]), (first, want[0]), (second, want[1])):
        for h, t in zip(held, inputs):
            h.copy_(t)
        graph.replay()
        for got, expected in zip(out, w):
            assert torch.equal(got, expected)


def test_two_streams_at_once(ops):
    table = ops.quantize_table(randn(gen(40), 9001, 320) * 0.06)
    inputs = [step_inputs(41 + i) for i in range(4)]
    want = [a_step(ops, i[0], table, *i[1:]) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(5):
        got = []
        for s, i in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append(a_step(ops, i[0], table, *i[1:]))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for a, b in zip(g, w):
                assert torch.equal(a, b)


def test_from_text_to_text(ops):
    """Ids of texts as the history, answers as ids that decode."""
    from conftest import tiny_vocab
    from graphtok_b200.gpu_bpe_tokenizer import Tokenizer
    tok = Tokenizer(tiny_vocab("llama3"))
    ids, offsets = tok.encode_batch_to_device(["some text to go on from", "and another one"])
    table = ops.quantize_table(randn(gen(50), tok.vocab_size, 64) * 0.3)
    hidden = randn(gen(51), 2, 64).to(BF16)
    logits = ops.adjust_logits(ops.table_logits(hidden, table), ids, offsets, repetition=1.5)
    got, logprobs = ops.sample(logits, torch.rand(2, generator=gen(52), device="cuda"), top_p=0.5)
    assert ((got >= 0) & (got < tok.vocab_size)).all() and (logprobs <= 0).all()
    assert isinstance(tok.decode_bytes(got.tolist()), bytes)


def test_refusals(ops):
    cuda = dict(device="cuda")
    weight = torch.zeros(40, 128, **cuda)
    table = ops.quantize_table(weight)
    hidden = torch.zeros(2, 128, dtype=BF16, **cuda)
    for call, kind, words in (
            (lambda: ops.table_logits(hidden.half(), table), TypeError, "bfloat16"), (lambda: ops.table_logits(hidden[:, :127], table), ValueError, "128"),
            (lambda: ops.table_logits(hidden, weight), TypeError, "QuantizedTable"), (lambda: ops.table_logits(hidden, table, dtype=F16), TypeError, "float32"),
            (lambda: ops.table_logits(hidden.cpu(), table), ValueError, "on"), (lambda: ops.table_logits(hidden.clone().requires_grad_(), table), NotImplementedError, "gradient"),
            (lambda: ops.quantize_table(weight, group=100), ValueError, "group"), (lambda: ops.quantize_table(weight[0]), ValueError, "weight"),
            (lambda: ops.quantize_table(weight.double()), TypeError, "float"), (lambda: ops.quantize_table(weight, dtype=F32), TypeError, "dtype"),
            (lambda: ops.quantize_table(weight[:0]), ValueError, "empty"),
            (lambda: ops.pack_table(weight, torch.zeros(40, 1, dtype=F16, **cuda)), TypeError, "uint8"),
            (lambda: ops.pack_table(weight.byte(), torch.zeros(40, 2, dtype=F16, **cuda)), ValueError, "scales"),
            (lambda: ops.pack_table(weight.byte(), torch.zeros(40, 1, **cuda)), TypeError, "scales"),
            (lambda: ops.pack_table(weight.byte(), torch.zeros(40, 1, dtype=F16, **cuda), torch.zeros(39, 1, dtype=torch.uint8, **cuda)), ValueError, "zeros")):
        with pytest.raises(kind, match=words):
            call()
    logits = torch.zeros(3, 50, **cuda)
    ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32, **cuda)        # noqa: E731
    room = torch.zeros(300, **cuda)
    for named, kind in ((dict(ids=ints(4)), ValueError), (dict(offsets=ints(4)), ValueError), (dict(ids=ints(4), offsets=ints(3)), ValueError), (dict(ids=ints(4).float(), offsets=ints(4)), TypeError),
                        (dict(ids=ints(2, 2), offsets=ints(4)), ValueError), (dict(ids=ints(4), offsets=ints(4).long()), TypeError),
                        (dict(ids=ints(4), offsets=ints(4), prompt_lengths=ints(2)), ValueError), (dict(prompt_lengths=ints(3)), ValueError),
                        (dict(ids=ints(4), offsets=ints(4), repetition=0.0), ValueError), (dict(ids=ints(4), offsets=ints(4), repetition=-1.0), ValueError),
                        (dict(ids=ints(4), offsets=ints(4), presence=math.nan), ValueError), (dict(ids=ints(4), offsets=ints(4), frequency=math.inf), ValueError),
                        (dict(ids=ints(4), offsets=ints(4), frequency=torch.zeros(2, **cuda)), ValueError), (dict(ids=ints(4), offsets=ints(4), repetition=torch.ones(3, **cuda).double()), ValueError),
                        (dict(bias=torch.zeros(3, 2, **cuda)), ValueError), (dict(bias_ids=ints(3, 2), bias=torch.zeros(3, 3, **cuda)), ValueError),
                        (dict(bias_ids=ints(2, 2), bias=torch.zeros(2, 2, **cuda)), ValueError), (dict(bias_ids=ints(3, 1025), bias=torch.zeros(3, 1025, **cuda)), ValueError),
                        (dict(bias_ids=ints(3, 2), bias=torch.zeros(3, 2, **cuda).half()), TypeError), (dict(allowed=ints(3, 1)), ValueError), (dict(allowed=ints(2, 2)), ValueError),
                        (dict(allowed=ints(3, 2).bool()), TypeError), (dict(allowed=ints(2), allowed_rows=ints(3)), ValueError), (dict(allowed_rows=ints(3)), ValueError),
                        (dict(allowed=ints(2, 2), allowed_rows=ints(2)), ValueError), (dict(out=torch.zeros(3, 49, **cuda)), ValueError), (dict(out=torch.zeros(3, 50, **cuda).half()), ValueError),
                        (dict(out=torch.zeros(50, 3, **cuda).t()), ValueError), (dict(out=torch.zeros(50, **cuda).expand(3, 50)), ValueError), (dict(ids=ints(4).cpu(), offsets=ints(4)), ValueError)):
        with pytest.raises(kind):
            ops.adjust_logits(logits, **named)
    with pytest.raises(ValueError, match="overlap"):
        ops.adjust_logits(room[:150].view(3, 50), out=room[20:170].view(3, 50))
    u = torch.zeros(3, **cuda)
    for args, named, kind in (((logits[0], u), {}, ValueError), ((logits, u[:2]), {}, ValueError), ((logits, u.half()), {}, ValueError), ((logits.double(), u), {}, TypeError),
                              ((logits, u), dict(temperature=-1.0), ValueError), ((logits, u), dict(temperature=math.inf), ValueError), ((logits, u), dict(temperature=math.nan), ValueError),
                              ((logits, u), dict(top_p=math.nan), ValueError), ((logits, u), dict(min_p=math.nan), ValueError), ((logits, u), dict(top_k=torch.zeros(3, **cuda)), ValueError),
                              ((logits, u), dict(top_p=torch.zeros(2, **cuda)), ValueError), ((logits, u.cpu()), {}, ValueError), ((logits[:, :0], u), {}, ValueError)):
        with pytest.raises(kind):
            ops.sample(*args, **named)


def test_a_least_share_far_below_a_huge_logit(ops):
    """The border of min_p among logits next to 0, where floating numbers lie so dense that their distance to the largest is the same for millions of them."""
    logits = torch.cat([torch.tensor([1e10, 0.0, 1e-38, -1e-7, -1e-5, -1.0, -10.0]), torch.linspace(-3e-6, 3e-6, 2000)]).cuda().repeat(6, 1)
    u = torch.tensor([0.0, 0.3, 0.6, 0.9, 0.99, 0.9999], device="cuda")
    for heat in (1e10 / math.log(10), 1e10 / math.log(10) * (1 + 2.0 ** -23), 5e9):
        check_draw(ops, logits, u, heat, 0, 1.0, 0.1)


def test_tables_are_copied_and_kept(ops, tmp_path):
    import copy
    table = ops.quantize_table(randn(gen(60), 300, 200), zeros=True, dtype=F16)
    hidden = randn(gen(61), 3, 200).to(F16)
    want = ops.table_logits(hidden, table)
    other = copy.deepcopy(table)
    assert other.data.data_ptr() != table.data.data_ptr() and torch.equal(ops.table_logits(hidden, other), want)
    torch.save(table, tmp_path / "table")
    kept = torch.load(tmp_path / "table", weights_only=False, map_location="cpu")
    with pytest.raises(ValueError, match="is on"):
        ops.table_logits(hidden, kept)
    assert torch.equal(ops.table_logits(hidden, kept.to("cuda")), want) and table.to("cuda") is table
    with pytest.raises(AttributeError):
        table.data = kept.data


def test_in_inference_mode(ops):
    with torch.inference_mode():
        table = ops.quantize_table(randn(gen(70), 5000, 64))
        logits = ops.table_logits(randn(gen(71), 4, 64).to(BF16), table)
        assert ops.adjust_logits(logits, bias_ids=torch.tensor([7], dtype=torch.int32, device="cuda"), bias=torch.tensor([99.0], device="cuda"), out=logits) is logits
        assert ops.sample(logits, torch.rand(4, generator=gen(72), device="cuda"), temperature=0.0)[0].tolist() == [7] * 4


@pytest.mark.parametrize("n", [9, 16, 17, 33, 64, 65, 97, 128, 129, 200])
def test_table_logits_of_more_rows_and_odd_lines(ops, n):
    """Rows of hidden states that begin at odd addresses, for every number of columns that the kernels are made for."""
    for width, group in ((130, 32), (191, 64), (320, 192)):
        codes, scales, z, values = make_table(n + width, 601, width, group, BF16, True)
        table = ops.pack_table(codes, scales, z, group=group)
        room = randn(gen(n), n, width + 3).to(BF16)
        for hidden in (room[:, 1:1 + width], room[:, :width].contiguous(), room[:1, :width].expand(n, width)):
            check_logits(ops.table_logits(hidden, table), hidden, values, group)


def test_c_entries_take_hidden_states_at_any_address(ops):
    """Through the C entry, which makes no copies: more rows than a pass, odd addresses and strides, rows of the output apart."""
    codes, scales, z, values = make_table(5, 333, 100, 64, F16, True)
    table = ops.pack_table(codes, scales, z, group=64)
    room = randn(gen(6), 70, 103).to(F16)
    hidden = room[:, 2:102]
    out = torch.full((70, 340), 5.0, device="cuda")
    lib = ops._lib()
    assert lib.gtok_x_table4_logits(ops._Matrix(hidden.data_ptr(), 70, 100, 103, 2), table._args, ops._Matrix(out.data_ptr() + 4, 70, 333, 340, 0), torch.cuda.current_stream().cuda_stream) == 0
    check_logits(out[:, 1:334], hidden, values, 64)
    assert (out[:, 0] == 5).all() and (out[:, 334:] == 5).all()
    # and what they refuse
    good = ops._Matrix(hidden.data_ptr(), 70, 100, 103, 2)
    for m, o in ((ops._Matrix(hidden.data_ptr() + 1, 70, 100, 103, 2), ops._Matrix(out.data_ptr(), 70, 333, 340, 0)), (ops._Matrix(hidden.data_ptr(), 70, 99, 103, 2), ops._Matrix(out.data_ptr(), 70, 333, 340, 0)),
                 (ops._Matrix(hidden.data_ptr(), 70, 100, 103, 1), ops._Matrix(out.data_ptr(), 70, 333, 340, 0)), (good, ops._Matrix(out.data_ptr(), 70, 333, 332, 0)),
                 (good, ops._Matrix(out.data_ptr(), 70, 333, 340, 1)), (good, ops._Matrix(out.data_ptr() + 2, 70, 333, 340, 0)), (good, ops._Matrix(0, 70, 333, 340, 0)),
                 (good, ops._Matrix(out.data_ptr(), 69, 333, 340, 0))):
        assert lib.gtok_x_table4_logits(m, table._args, o, None) == -1
    for change in (dict(data=table.data.data_ptr() + 16), dict(bytes=table.data.numel() - 1), dict(group=48), dict(type=0), dict(zeros=2), dict(data=0)):
        bad = ops._Table4(table.data.data_ptr(), table.data.numel(), 333, 100, 64, 2, 1)
        for k, v in change.items():
            setattr(bad, k, v)
        assert lib.gtok_x_table4_logits(good, bad, ops._Matrix(out.data_ptr(), 70, 333, 340, 0), None) == -1
    logits = torch.zeros(3, 50, device="cuda")
    a = ops._Adjustment()
    a.logits, a.out, a.offsets, a.ids, a.id_bits, a.n_ids = ops._Matrix(logits.data_ptr(), 3, 50, 50, 0), ops._Matrix(logits.data_ptr(), 3, 50, 50, 0), 0, 0, 32, 0
    assert lib.gtok_x_adjust_logits(a) == 0
    for change in (dict(entries=1025), dict(entries=3), dict(offsets=logits.data_ptr() + 2), dict(repetition=logits.data_ptr() + 1), dict(allowed=12), dict(id_bits=16, offsets=logits.data_ptr()),
                   dict(out=ops._Matrix(logits.data_ptr(), 3, 50, 60, 0)), dict(out=ops._Matrix(logits.data_ptr(), 3, 50, 50, 1)), dict(logits=ops._Matrix(logits.data_ptr(), 3, 0, 50, 0))):
        b = ops._Adjustment()
        b.logits, b.out, b.id_bits = a.logits, a.out, 32
        for k, v in change.items():
            setattr(b, k, v)
        assert lib.gtok_x_adjust_logits(b) == -1, change
    u, ids, logprobs = torch.zeros(3, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, device="cuda")
    d = dict(logits=a.logits, u=u.data_ptr(), u_bits=32, one_temperature=1.0, one_top_p=1.0, ids=ids.data_ptr(), logprobs=logprobs.data_ptr())
    for change, code in (({}, 0), (dict(u_bits=16), -1), (dict(u=0), -1), (dict(u=u.data_ptr() + 4, u_bits=64), -1), (dict(ids=0), -1), (dict(logprobs=logprobs.data_ptr() + 1), -1),
                         (dict(temperature=u.data_ptr() + 2), -1), (dict(logits=ops._Matrix(logits.data_ptr(), 3, (1 << 24) + 1, 50, 0)), -1), (dict(logits=ops._Matrix(logits.data_ptr(), -1, 50, 50, 0)), -1)):
        c = ops._Draw()
        for k, v in (d | change).items():
            setattr(c, k, v)
        assert lib.gtok_x_sample(c) == code, change


@pytest.mark.parametrize("n,vocab", [(1, 128256), (16, 20000), (17, 20000), (40, 9000), (70, 9000), (150, 5000), (300, 3000)])
def test_every_share_of_a_row(ops, n, vocab):
    """As many rows as make one to eight blocks of a row, held in shared memory or not."""
    for i, wish in enumerate(((1.0, 0, 1.0, 0.0), (0.9, 30, 0.9, 0.0), (1.5, 0, 0.95, 0.0), (1.0, 900, 0.97, 0.0))):
        check_draw(ops, model_logits(7 * n + i, n, vocab, BF16 if i % 2 else F32), torch.rand(n, generator=gen(i + n), device="cuda"), *wish)


def test_rows_with_few_logits_left(ops):
    """Masks that leave a few ids, fewer than top_k or hardly more, and lowest finite values in place of -inf."""
    g = gen(80)
    logits = randn(g, 40, 30000) * 2
    lowest = torch.finfo(F32).min
    for i in range(40):
        keep = torch.randint(0, 30000, ((1, 2, 5, 39, 40, 41, 500, 2500)[i % 8],), generator=g, device="cuda")
        masked = torch.full((30000,), -math.inf if i % 3 else lowest, device="cuda")
        masked[keep] = logits[i, keep]
        logits[i] = masked
    u = torch.rand(40, generator=g, device="cuda")
    for wish in ((1.0, 0, 1.0, 0.0), (0.8, 40, 1.0, 0.0), (0.8, 40, 0.9, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 0, 0.999, 0.0), (1.0, 0, 0.9, 0.2), (1e38, 0, 0.9, 0.0)):
        check_draw(ops, logits, u, *wish)


@pytest.mark.parametrize("n", [1, 3, 60])
def test_long_histories_of_every_kind(ops, n):
    """Histories that pass a block's steps, with the ids that come most often at the beginning of the vocabulary, at its end, and all the same."""
    g = gen(90 + n)
    vocab = 50257
    logits = randn(g, n, vocab)
    parts = [torch.randint(0, 40, (4000,), generator=g, device="cuda"), vocab - 1 - torch.randint(0, 40, (4000,), generator=g, device="cuda"), torch.full((4001,), 7, device="cuda"),
             torch.randint(0, vocab, (9000,), generator=g, device="cuda")]
    row = torch.cat(parts)
    ids = row.repeat(n)
    offsets = (torch.arange(n + 1, device="cuda") * row.numel()).int()
    prompts = torch.randint(0, row.numel() + 1, (n,), generator=g, device="cuda").int()
    got = ops.adjust_logits(logits, ids, offsets, prompt_lengths=prompts, repetition=1.25, frequency=0.5, presence=2.0)
    for i in range(n):
        said = torch.zeros(vocab, dtype=torch.bool, device="cuda")
        said[row] = True
        times = torch.bincount(row[prompts[i]:], minlength=vocab).double()
        x = logits[i].double()
        want = torch.where(said, torch.where(x > 0, x / 1.25, x * 1.25), x) - 0.5 * times - 2.0 * (times > 0)
        within(got[i], want, 4 * 2.0 ** -24 * (x.abs() * 1.25 + 0.5 * times + 2) * said, "logits")


def test_the_version_of_what_is_written(ops):
    logits = randn(gen(1), 2, 100)
    before = logits._version
    ops.adjust_logits(logits, allowed=torch.zeros(4, dtype=torch.int32, device="cuda"), out=logits)
    assert logits._version == before + 1 and (logits == -math.inf).all()
