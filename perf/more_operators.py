"""The way from a model's last hidden states to the ids that it answers with, for timing it.

A server that decodes has, for each of its requests, one hidden state a step.  It multiplies it with the output table, which is held in
4 bits; changes the logits as the request asks (penalties for what has been said, biases, what its grammar allows); and draws an id.
A case is one pass through one of these three:

    logits      products of some hidden states with a table of 4-bit codes, a scale (and a zero) for each group of a row
    adjust      penalties, biases and grammar masks
    sample      an id for each row of logits: temperature, top-k, top-p, min-p and a random number that is given

`run` computes them in plain form from elementary operations, or with `own` by the calls of `graphtok_b200.next_ops`.

    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) tensors on the GPU, as a program has them in hand before the call
    run(state)          the pass
    work(case)          bytes and operations that the pass cannot do without
    exact(case, seed)   its outputs from the definitions in 64 bits
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
#: Ids of the synthetic vocabularies of the GPT-2, Llama-3 and Qwen2.5 shapes.
GPT2, LLAMA3, QWEN25 = 50256, 128256, 151665


def listed():
    return [
        # One request to a small model: the smallest call, all latency.
        {"name": "logits_small", "op": "logits", "type": "fp16", "rows": 1, "vocab": GPT2, "width": 768, "group": 64, "zeros": False},
        # One request to a large model: the table has to be read.
        {"name": "logits_chat", "op": "logits", "type": "bf16", "rows": 1, "vocab": LLAMA3, "width": 4096, "group": 128, "zeros": False},
        # The drafts of a few requests checked at once; codes as a calibrated quantisation gives them, with zeros.
        {"name": "logits_drafts", "op": "logits", "type": "fp16", "rows": 13, "vocab": QWEN25, "width": 2560, "group": 64, "zeros": True},
        # A server with some dozens of requests.
        {"name": "logits_step", "op": "logits", "type": "bf16", "rows": 47, "vocab": LLAMA3, "width": 4096, "group": 128, "zeros": True},
        # A full one; the most operations.
        {"name": "logits_full", "op": "logits", "type": "bf16", "rows": 125, "vocab": QWEN25, "width": 2048, "group": 32, "zeros": False},
        # A conversation with penalties.
        {"name": "adjust_chat", "op": "adjust", "type": "fp32", "rows": 1, "vocab": LLAMA3, "history": 911, "bias": 0, "grammar": 0.0},
        # Some dozens of requests: a part of them have to answer in a format, and each has a few biases.
        {"name": "adjust_step", "op": "adjust", "type": "fp32", "rows": 47, "vocab": QWEN25, "history": 4093, "bias": 21, "grammar": 0.5},
        # Many, with long documents behind them, logits in 16 bits.
        {"name": "adjust_full", "op": "adjust", "type": "bf16", "rows": 251, "vocab": LLAMA3, "history": 20011, "bias": 300, "grammar": 1.0},
        # An answer's next id, as interfaces ask for it by default.
        {"name": "sample_chat", "op": "sample", "type": "fp32", "rows": 1, "vocab": GPT2, "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "mixed": False},
        # Rollouts of a policy: the whole distribution, as it is.
        {"name": "sample_rollouts", "op": "sample", "type": "fp32", "rows": 64, "vocab": QWEN25, "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "mixed": False},
        # A server's requests, each with its own wishes, greedy ones and ones with a grammar among them.
        {"name": "sample_step", "op": "sample", "type": "fp32", "rows": 47, "vocab": LLAMA3, "temperature": 0.7, "top_k": 40, "top_p": 0.9, "min_p": 0.05, "mixed": True},
        # A full one, in 16 bits, where many logits are alike.
        {"name": "sample_full", "op": "sample", "type": "bf16", "rows": 251, "vocab": LLAMA3, "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "mixed": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("logits", "logits", "adjust", "sample", "sample"))
    while True:
        vocab = rng.choice((GPT2, LLAMA3, QWEN25, _log(rng, 3000, 200000)))
        if op == "logits":
            case = {"op": op, "type": rng.choice(("bf16", "fp16")), "rows": _log(rng, 1, 128), "vocab": vocab,
                    "width": rng.choice((_log(rng, 64, 8192), 8 * _log(rng, 8, 1024))), "group": rng.choice((32, 64, 128)), "zeros": rng.random() < 0.5}
            most = (work(listed()[1]), work(listed()[3]))
        elif op == "adjust":
            case = {"op": op, "type": rng.choice(tuple(TYPES)), "rows": _log(rng, 1, 256), "vocab": vocab, "history": _log(rng, 1, 32768),
                    "bias": rng.choice((0, _log(rng, 1, 300))), "grammar": rng.choice((0.0, 0.3, 1.0))}
            most = (work(listed()[7]),) * 2
        else:
            case = {"op": op, "type": rng.choice(tuple(TYPES)), "rows": _log(rng, 1, 256), "vocab": vocab, "temperature": round(rng.uniform(0.3, 1.5), 2),
                    "top_k": rng.choice((0, 0, 1, _log(rng, 2, 1000))), "top_p": rng.choice((1.0, round(rng.uniform(0.5, 0.99), 2))),
                    "min_p": rng.choice((0.0, 0.0, round(rng.uniform(0.01, 0.3), 2))), "mixed": rng.random() < 0.4}
            most = (work(listed()[11]),) * 2
        got = work(case)
        if got["bytes"] <= most[0]["bytes"] * 1.2 and got["flops"] <= most[1]["flops"]:
            return case


def _generator(seed, what):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + what)


def _ids(gen, n, vocab):
    """Ids as frequent as their place in the vocabulary says (Zipf): merges learned first stand for the commonest text."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(vocab)) - 1.0).int().clamp_(0, vocab - 1)


def _model_logits(gen, n, vocab, dtype):
    """Logits of a model that has learned something: noise, above it some dozens of ids that could follow, and one or two that likely do."""
    x = torch.randn(n, vocab, generator=gen, device="cuda") * 1.8
    near = torch.randint(0, vocab, (n, 40), generator=gen, device="cuda")
    level = 13.0 - 3.0 * torch.rand(n, 1, generator=gen, device="cuda") - 9.0 * torch.rand(n, 40, generator=gen, device="cuda").sqrt()
    return x.scatter_reduce_(1, near, level, "amax").to(dtype)      # (the same whatever order it is done in)


def prepare(case, seed):
    gen = _generator(seed, case["rows"] + 7 * case["vocab"])
    n, vocab, dtype = case["rows"], case["vocab"], TYPES[case["type"]]
    state = {"op": case["op"]}
    if case["op"] == "logits":
        width, group = case["width"], case["group"]
        groups = -(-width // group)
        codes = torch.empty(vocab, width, dtype=torch.uint8, device="cuda")
        for at in range(0, vocab, 16384):          # (bounds what 32-bit noise takes)
            some = codes[at:at + 16384]
            some.copy_(torch.randn(some.shape, generator=gen, device="cuda").mul_(2.5).add_(8.0).round_().clamp_(0.0, 15.0))
        scales = (torch.rand(vocab, groups, generator=gen, device="cuda") * 0.006 + 0.005).to(dtype)
        zeros = torch.randint(5, 11, (vocab, groups), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        state |= {"codes": codes, "scales": scales, "zeros": zeros, "group": group}
        state["hidden"] = (torch.randn(n, width, generator=gen, device="cuda") * (1.5 / (0.02 * math.sqrt(width)))).to(dtype)
        if own:        # the table as a server keeps it, laid out when it is loaded
            from graphtok_b200 import next_ops
            state["table"] = next_ops.pack_table(codes, scales, zeros, group=group)
        return state
    state["logits"] = _model_logits(gen, n, vocab, dtype)
    if case["op"] == "adjust":
        lengths = (torch.rand(n, generator=gen, device="cuda") * 0.75 + 0.25).mul(case["history"]).int().clamp_(min=1)
        state["offsets"] = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)]).int()
        state["ids"] = _ids(gen, int(state["offsets"][-1]), vocab)
        state["prompt_lengths"] = (torch.rand(n, generator=gen, device="cuda") * lengths).int()
        state["repetition"] = 1.0 + 0.3 * torch.rand(n, generator=gen, device="cuda")
        state["presence"] = 0.8 * torch.rand(n, generator=gen, device="cuda")
        state["frequency"] = 0.5 * torch.rand(n, generator=gen, device="cuda")
        state["bias_ids"] = state["bias"] = state["allowed"] = state["allowed_rows"] = None
        if case["bias"]:
            # lists are as long as the longest of them; what an entry of -1 stands for is left out
            kept = torch.arange(case["bias"], device="cuda") < torch.randint(0, case["bias"] + 1, (n, 1), generator=gen, device="cuda")
            state["bias_ids"] = torch.where(kept, torch.randint(0, vocab, kept.shape, generator=gen, device="cuda"), -1).int()
            state["bias"] = torch.randn(kept.shape, generator=gen, device="cuda") * 4.0
        if case["grammar"]:
            # a grammar allows little most of the time, and nearly all of it within a string; requests share its states
            states, words = max(1, n // 3), -(-vocab // 32)
            bits = torch.randint(-2 ** 31, 2 ** 31, (3, states, words), generator=gen, device="cuda")
            free = torch.rand(states, 1, generator=gen, device="cuda") < 0.3
            state["allowed"] = torch.where(free, bits[0] | bits[1] | bits[2], bits[0] & bits[1] & bits[2]).int()
            rows = torch.randint(0, states, (n,), generator=gen, device="cuda")
            state["allowed_rows"] = torch.where(torch.rand(n, generator=gen, device="cuda") < case["grammar"], rows, -1).int()
        return state
    spread = lambda low, high: low + (high - low) * torch.rand(n, generator=gen, device="cuda")     # noqa: E731
    alike = torch.ones(n, device="cuda")
    state |= {"u": torch.rand(n, generator=gen, device="cuda"), "temperature": alike * case["temperature"], "top_k": (alike * case["top_k"]).int(),
              "top_p": alike * case["top_p"], "min_p": alike * case["min_p"]}
    if case["mixed"]:
        on = lambda share: torch.rand(n, generator=gen, device="cuda") < share      # noqa: E731
        state["temperature"] = torch.where(on(0.2), 0.0, state["temperature"] * spread(0.6, 1.4))
        state["top_k"] = torch.where(on(0.5), state["top_k"], 0)
        state["top_p"] = torch.where(on(0.5), state["top_p"], 1.0)
        state["min_p"] = torch.where(on(0.5), state["min_p"], 0.0)
        few = torch.rand(n, vocab, generator=gen, device="cuda") < 0.02
        state["logits"] = state["logits"].masked_fill(~few & on(0.3)[:, None], -math.inf)
    return state


def _plain_logits(s):
    codes, groups = s["codes"], s["scales"].shape[1]
    spread = lambda t: t.float().repeat_interleave(s["group"], 1)[:, :codes.shape[1]] if groups > 1 else t.float()     # noqa: E731
    weight = codes.float()
    weight -= 8.0 if s["zeros"] is None else spread(s["zeros"])
    weight *= spread(s["scales"])
    return s["hidden"].float() @ weight.T


def _plain_adjust(s):
    x = s["logits"].float()
    n, vocab = x.shape
    lengths = s["offsets"].diff().long()
    row = torch.repeat_interleave(torch.arange(n, device=x.device), lengths)
    behind = torch.arange(row.numel(), device=x.device) - s["offsets"][:-1].long()[row] >= s["prompt_lengths"].long()[row]
    place = row * vocab + s["ids"].long()
    said = torch.zeros(n * vocab, device=x.device).index_add_(0, place, torch.ones_like(place, dtype=torch.float32)).view(n, vocab) > 0
    count = torch.zeros(n * vocab, device=x.device).index_add_(0, place, behind.float()).view(n, vocab)
    rho = s["repetition"][:, None]
    x = torch.where(said, torch.where(x > 0, x / rho, x * rho), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias_ids"] is not None:
        x = x.scatter_add(1, s["bias_ids"].long().clamp(min=0), torch.where(s["bias_ids"] >= 0, s["bias"], 0.0))
    if s["allowed"] is not None:
        bits = (s["allowed"][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        allowed = bits.flatten(1)[:, :vocab][s["allowed_rows"].long().clamp(min=0)] != 0
        x = torch.where(allowed | (s["allowed_rows"] < 0)[:, None], x, -math.inf)
    return x.to(s["logits"].dtype)


def _plain_sample(s):
    logits = s["logits"].double()
    n, vocab = logits.shape
    heat, greedy = s["temperature"].double()[:, None], s["temperature"] == 0
    top = logits.max(1, keepdim=True).values
    mass = torch.exp((logits - top) / torch.where(heat == 0, 1.0, heat))
    total = mass.sum(1, keepdim=True)
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices
    ranked = mass.gather(1, order)
    kept = torch.arange(vocab, device=logits.device) < torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    ranked *= kept
    running = ranked.cumsum(1)
    before = torch.cat([running.new_zeros(n, 1), running[:, :-1]], 1)
    kept &= (before < s["top_p"].double()[:, None] * running[:, -1:]) & (ranked >= s["min_p"].double()[:, None] * ranked[:, :1])
    kept[:, 0] = True
    running = (mass * torch.zeros_like(mass).scatter_(1, order, kept.double())).cumsum(1)
    ids = (running <= s["u"].double()[:, None] * running[:, -1:]).sum(1)
    ids = torch.where(greedy, order[:, 0], ids)
    logprobs = torch.where(greedy, 0.0, (mass.gather(1, ids[:, None]) / total).log()[:, 0])
    return {"ids": ids.int(), "logprobs": logprobs.float()}


def _plain(s):
    return {"logits": _plain_logits, "adjust": _plain_adjust, "sample": _plain_sample}[s["op"]](s)


def _own(s):
    from graphtok_b200 import next_ops
    if s["op"] == "logits":
        return next_ops.table_logits(s["hidden"], s["table"])
    if s["op"] == "adjust":
        return next_ops.adjust_logits(s["logits"], s["ids"], s["offsets"], prompt_lengths=s["prompt_lengths"], repetition=s["repetition"], presence=s["presence"],
                                      frequency=s["frequency"], bias_ids=s["bias_ids"], bias=s["bias"], allowed=s["allowed"], allowed_rows=s["allowed_rows"])
    ids, logprobs = next_ops.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return {"ids": ids, "logprobs": logprobs}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    n, vocab, size = case["rows"], case["vocab"], SIZE[case["type"]]
    if case["op"] == "logits":
        width = case["width"]
        groups = -(-width // case["group"])
        return {"bytes": vocab * (width / 2 + groups * (2.5 if case["zeros"] else 2)) + n * (2.0 * width + 4.0 * vocab), "flops": 2.0 * n * vocab * width}
    if case["op"] == "adjust":
        masks = min(n * case["grammar"], max(1, n // 3)) * vocab / 8
        return {"bytes": n * (2.0 * vocab * size + 2.5 * case["history"] + 8 * case["bias"]) + masks, "flops": 1.0 * n * vocab}
    return {"bytes": n * (1.0 * vocab * size + 28), "flops": 2.0 * n * vocab}


def exact(case, seed):
    state = prepare(case, seed)
    n, vocab = case["rows"], case["vocab"]
    if case["op"] == "logits":
        out = torch.zeros(n, vocab, dtype=torch.float64, device="cuda")
        for g in range(state["scales"].shape[1]):          # a group of columns at a time
            some = slice(g * case["group"], (g + 1) * case["group"])
            zero = state["zeros"][:, g, None].double() if case["zeros"] else 8.0
            out += (state["hidden"][:, some].double() @ (state["codes"][:, some].double() - zero).T) * state["scales"][:, g].double()
        return out
    x = state["logits"].double()
    if case["op"] == "adjust":
        edges, prompts = state["offsets"].tolist(), state["prompt_lengths"].tolist()
        bits = 1 << torch.arange(32, device="cuda")
        for i in range(n):
            ids = state["ids"][edges[i]:edges[i + 1]].long()
            anywhere = torch.unique(ids)
            old = x[i, anywhere]
            rho = state["repetition"][i].double()
            x[i, anywhere] = torch.minimum(old * rho, old / rho)         # (rho is 1 at least here)
            new, times = torch.unique(ids[prompts[i]:], return_counts=True)
            x[i, new] -= state["frequency"][i].double() * times + state["presence"][i].double()
            if case["bias"]:
                real = state["bias_ids"][i] >= 0
                x[i].index_put_((state["bias_ids"][i][real].long(),), state["bias"][i][real].double(), accumulate=True)
            if case["grammar"] and int(state["allowed_rows"][i]) >= 0:
                allowed = (state["allowed"][state["allowed_rows"][i]].long()[:, None] & bits).flatten()[:vocab] != 0
                x[i, ~allowed] = -math.inf
        return x
    ids, logprobs = [], []
    for i in range(n):
        heat, k, p, least = (state[name][i].item() for name in ("temperature", "top_k", "top_p", "min_p"))
        if heat == 0:
            ids.append(int((x[i] == x[i].max()).nonzero()[0]))
            logprobs.append(0.0)
            continue
        z = x[i] / heat
        share = torch.softmax(z, 0)
        # ids from the likeliest on; among equals the lower first, as the sort by id comes before the sort by value
        rank = torch.argsort(-x[i], stable=True)
        if k > 0:
            rank = rank[:k]
        some = share[rank] / share[rank].sum()
        keep = int((some.cumsum(0) < p).sum()) + 1 if p < 1 else rank.numel()
        rank = rank[:keep]
        rank = rank[share[rank] >= least * share[rank[0]]].sort().values
        ends = share[rank].cumsum(0)
        pick = rank[torch.searchsorted(ends, state["u"][i].double() * ends[-1], right=True)]
        ids.append(int(pick))
        logprobs.append(float(z[pick] - torch.logsumexp(z, 0)))
    return {"ids": torch.tensor(ids, dtype=torch.int32, device="cuda"), "logprobs": torch.tensor(logprobs, dtype=torch.float64, device="cuda")}
