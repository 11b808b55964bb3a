"""The two ends of a language model that are as wide as the vocabulary, for timing them.

Token ids come from the tokenizer packed: the documents of a batch one after another, with the place at which each begins.
A model looks each id up in its embedding table and, at the other end, compares what it made of each position with the id
that follows there.  A case is one pass through one of the operators between ids and such a model:

    embed        rows of the embedding table, scaled
    embed_grad   the table's gradient: the rows that a step's ids were looked up from, summed for each id
    score        loss of every position against the next id, from hidden states and the output table, without gradients
    train        the mean of that loss with the gradients of hidden states and output table
    distill      the same against a teacher's top logits

`run` computes them in plain form from elementary operations in 32 bits, or with `own` by the calls of `graphtok_b200.vocab_ops`.

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
IGNORE = -100


def listed():
    return [
        # One decoding step of a server with some dozens of requests: the last id of each, looked up.
        {"name": "embed_step", "op": "embed", "type": "bf16", "tokens": 47, "vocab": LLAMA3, "width": 4096, "scale": 1.0, "wide_ids": False},
        # The prompts that a scheduler packed together, straight from the tokenizer; a family that scales by the root of the width.
        {"name": "embed_prompts", "op": "embed", "type": "bf16", "tokens": 32749, "vocab": QWEN25, "width": 2560, "scale": 50.59644256269407, "wide_ids": False},
        # The table's gradient in a training step of a large model: tens of thousands of ids, most of them frequent ones.
        {"name": "embed_grad_step", "op": "embed_grad", "type": "bf16", "tokens": 16384, "vocab": LLAMA3, "width": 4096, "scale": 1.0, "wide_ids": False},
        # The same of a small model in 32 bits, as it is fine-tuned on one document; ids as a data loader has them, in 64 bits.
        {"name": "embed_grad_small", "op": "embed_grad", "type": "fp32", "tokens": 2047, "vocab": GPT2, "width": 768, "scale": 27.712812921102035, "wide_ids": True},
        # The answers to a question ranked by their likelihood: a few positions against the whole table, which has to be read.
        {"name": "score_answers", "op": "score", "type": "bf16", "docs": 3, "tokens": 37, "vocab": QWEN25, "width": 2048},
        # Perplexity of some documents under a large model.
        {"name": "score_documents", "op": "score", "type": "bf16", "docs": 11, "tokens": 4093, "vocab": LLAMA3, "width": 4096},
        # A step of a small model.
        {"name": "train_small", "op": "train", "type": "fp16", "docs": 5, "tokens": 1021, "vocab": GPT2, "width": 768, "prompt": 0.0},
        # Fine-tuning on answers: the prompts' positions carry no loss.
        {"name": "train_answers", "op": "train", "type": "bf16", "docs": 23, "tokens": 4099, "vocab": QWEN25, "width": 1024, "prompt": 0.6},
        # A pre-training step, the largest call.
        {"name": "train_step", "op": "train", "type": "bf16", "docs": 9, "tokens": 8192, "vocab": LLAMA3, "width": 2048, "prompt": 0.0},
        # A student of one short conversation, from the few logits that a serving interface gives.
        {"name": "distill_chat", "op": "distill", "type": "fp16", "tokens": 301, "vocab": LLAMA3, "width": 1024, "top": 20, "temperature": 1.0, "prompt": 0.3},
        # Distillation proper: a stored set of a teacher's top logits, softened.
        {"name": "distill_step", "op": "distill", "type": "bf16", "tokens": 2048, "vocab": QWEN25, "width": 2048, "top": 64, "temperature": 2.0, "prompt": 0.1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("embed", "embed_grad", "score", "train", "train", "distill", "distill"))
    while True:
        vocab = rng.choice((GPT2, LLAMA3, QWEN25, _log(rng, 3000, 200000)))
        case = {"op": op, "type": rng.choice(("bf16", "fp16")), "tokens": _log(rng, 1 if op == "embed" else 8, 32768), "vocab": vocab}
        if op.startswith("embed"):
            case |= {"type": rng.choice(tuple(TYPES)), "width": rng.choice((_log(rng, 64, 8192), 8 * _log(rng, 8, 1024))),
                     "scale": rng.choice((1.0, 0.25, 45.25)), "wide_ids": rng.random() < 0.5}
        else:
            case |= {"width": 8 * _log(rng, 32, 640)}
            if op != "distill":
                case["docs"] = min(case["tokens"] // 2, _log(rng, 1, 40))
            else:
                case |= {"top": _log(rng, 1, 100), "temperature": rng.choice((1.0, 2.0, 4.0, 0.7))}
            if op != "score":
                case["prompt"] = rng.choice((0.0, 0.3, 0.8)) if case["tokens"] >= 512 else 0.0
        got, most = work(case), work(listed()[8])
        if got["flops"] <= most["flops"] and got["bytes"] <= most["bytes"] * 2 and case["tokens"] * vocab <= 8192 * LLAMA3:
            return case


def _generator(seed, what):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + what)


def _ids(gen, n, vocab):
    """Ids as frequent as their place in the vocabulary says (Zipf): merges learned first stand for the commonest text."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(vocab)) - 1.0).long().clamp_(0, vocab - 1)


def _hidden(gen, weight, ids, dtype):
    """Hidden states of a model that has learned something: noise, and of the row of the next id as much as a logit of 0 to 12 takes."""
    n, width = ids.numel(), weight.shape[1]
    lead = 12.0 * torch.rand(n, 1, generator=gen, device="cuda") / (0.02 * 0.02 * width)
    noise = torch.randn(n, width, generator=gen, device="cuda") * (1.5 / (0.02 * math.sqrt(width)))
    return (noise + lead * weight[ids].float()).to(dtype)


def prepare(case, seed):
    gen = _generator(seed, case["tokens"] + 7 * case["width"])
    n, vocab, width, dtype = case["tokens"], case["vocab"], case["width"], TYPES[case["type"]]
    ids = _ids(gen, n, vocab)
    state = {"op": case["op"], "vocab": vocab}
    if case["op"].startswith("embed"):
        rows = n if case["op"] == "embed_grad" else vocab
        state["rows"] = (torch.randn(rows, width, generator=gen, device="cuda") * 0.02).to(dtype)   # gradient, or table
        state["scale"] = case["scale"]
        state["ids"] = ids if case["wide_ids"] else ids.int()
        return state
    weight = (torch.randn(vocab, width, generator=gen, device="cuda") * 0.02).to(dtype)
    state["weight"], state["grads"] = weight, case["op"] != "score"
    # positions of prompts, which carry no loss, come in stretches
    masked = (torch.rand(n // 16 + 1, generator=gen, device="cuda") < case.get("prompt", 0.0)).repeat_interleave(16)[:n]
    if case["op"] == "distill":
        top = case["top"]
        # distinct ids: the likeliest one is that of the text, the others lie anywhere
        gaps = torch.randint(1, vocab // (top + 1) + 1, (n, top), generator=gen, device="cuda")
        gaps[:, 0] = 0
        teacher = (ids[:, None] + gaps.cumsum(1)) % vocab
        logits = 18.0 - 2.5 * torch.log1p(torch.arange(top, device="cuda")) - torch.rand(n, top, generator=gen, device="cuda").cumsum(1) * 0.2
        # a teacher's list ends where little probability is left; of a prompt's position there is none
        kept = torch.randint((top + 1) // 2, top + 1, (n, 1), generator=gen, device="cuda") * ~masked[:, None]
        teacher = torch.where(torch.arange(top, device="cuda") < kept, teacher, -1)
        state |= {"hidden": _hidden(gen, weight, ids, dtype), "teacher_ids": teacher.int(), "teacher_logits": logits.float(),
                  "temperature": case["temperature"]}
    else:
        cuts = torch.rand(case["docs"] - 1, generator=gen, device="cuda").mul(n - 1).long().add(1).sort().values
        state["offsets"] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), n)]).int()
        state["ids"] = ids.int()
        state["hidden"] = _hidden(gen, weight, torch.cat([ids[1:], ids[:1]]), dtype)
        state["loss_mask"] = ~masked if state["grads"] else None
    if state["grads"]:
        state["hidden"].requires_grad_()
        state["weight"].requires_grad_()
    return state


def _next(ids, offsets, loss_mask):
    """The id that follows each position in its document, IGNORE at a document's end and where no loss is wanted."""
    ends = torch.zeros(ids.numel() + 1, dtype=torch.bool, device=ids.device)
    ends[offsets.long()] = True
    targets = torch.where(ends[1:], IGNORE, torch.cat([ids[1:], ids[:1]]).long())
    return targets if loss_mask is None else torch.where(loss_mask, targets, IGNORE)


def _plain(s):
    if s["op"] == "embed":
        return (s["rows"][s["ids"].long()].float() * s["scale"]).to(s["rows"].dtype)
    if s["op"] == "embed_grad":
        total = torch.zeros(s["vocab"], s["rows"].shape[1], dtype=torch.float32, device="cuda")
        total.index_add_(0, s["ids"].long(), s["rows"].float())
        return (total * s["scale"]).to(s["rows"].dtype)
    hidden, weight = s["hidden"].detach().float(), s["weight"].detach().float()
    if s["op"] == "distill":
        given = s["teacher_ids"] >= 0
        active = given.any(1)
        index = s["teacher_ids"].long().clamp(min=0)
        share = torch.softmax(torch.where(given, s["teacher_logits"] / s["temperature"], -1e30), 1) * given
        heat = s["temperature"]
    else:
        targets = _next(s["ids"], s["offsets"], s["loss_mask"])
        active = targets >= 0
        index = targets.clamp(min=0)[:, None]
        share = active[:, None].float()
        heat = 1.0
    logits = (hidden @ weight.T) / heat
    lse = torch.logsumexp(logits, 1, keepdim=True)
    picked = torch.gather(logits, 1, index) - lse
    losses = (share * (torch.where(share > 0, share, 1.0).log() - picked)).sum(1)
    losses = torch.where(active, losses, 0.0)
    if not s["grads"]:
        return losses
    count = active.sum().clamp(min=1)
    delta = torch.exp(logits - lse) * active[:, None]
    delta.scatter_add_(1, index, -share)
    delta /= heat * count
    return {"loss": losses.sum() / count, "d_hidden": (delta @ weight).to(s["hidden"].dtype), "d_weight": (delta.T @ hidden).to(s["weight"].dtype)}


def _own(s):
    from graphtok_b200 import vocab_ops
    if s["op"] == "embed":
        return vocab_ops.embed(s["ids"], s["rows"], scale=s["scale"])
    if s["op"] == "embed_grad":
        return vocab_ops.embed_grad(s["ids"], s["rows"], s["vocab"], scale=s["scale"])
    if s["op"] == "distill":
        loss = vocab_ops.distill(s["hidden"], s["weight"], s["teacher_ids"], s["teacher_logits"], temperature=s["temperature"])
    else:
        targets = vocab_ops.next_targets(s["ids"], s["offsets"], loss_mask=s["loss_mask"])
        loss = vocab_ops.cross_entropy(s["hidden"], s["weight"], targets, reduction="mean" if s["grads"] else "none")
    if not s["grads"]:
        return loss
    d_hidden, d_weight = torch.autograd.grad(loss, (s["hidden"], s["weight"]))
    return {"loss": loss.detach(), "d_hidden": d_hidden, "d_weight": d_weight}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    n, vocab, width, size = case["tokens"], case["vocab"], case["width"], SIZE[case["type"]]
    if case["op"] == "embed":
        return {"bytes": n * (2.0 * width * size + (8 if case["wide_ids"] else 4)), "flops": 1.0 * n * width}
    if case["op"] == "embed_grad":
        return {"bytes": (n + vocab) * 1.0 * width * size + n * (8 if case["wide_ids"] else 4), "flops": 1.0 * n * width}
    product = 2.0 * n * vocab * width
    tables = 1.0 * (n + vocab) * width * size
    if case["op"] == "score":
        return {"bytes": tables + 8.0 * n, "flops": product}
    # logits, the hidden states' gradient and the table's, at the positions that carry a loss
    return {"bytes": 2.0 * tables + n * 8.0 * case.get("top", 1), "flops": 3.0 * product * (1.0 - case["prompt"])}


def exact(case, seed):
    state = prepare(case, seed)
    ids = state.get("ids")
    if case["op"] == "embed":
        return torch.nn.functional.embedding(ids.long(), state["rows"].double()) * case["scale"]
    if case["op"] == "embed_grad":
        order = ids.long().argsort(stable=True)
        rows, counts = torch.unique_consecutive(ids.long()[order], return_counts=True)
        total = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device="cuda")
        total[rows] = torch.segment_reduce(state["rows"].double()[order], "sum", lengths=counts, axis=0) * case["scale"]
        return total
    hidden, weight = state["hidden"].detach().double(), state["weight"].detach().double()
    n = case["tokens"]
    heat = case.get("temperature", 1.0)
    wanted = torch.zeros(n, case["vocab"], dtype=torch.float64, device="cuda")     # what the softmax should be
    if case["op"] == "distill":
        row, entry = (state["teacher_ids"] >= 0).nonzero(as_tuple=True)
        raw = torch.exp((state["teacher_logits"].double()[row, entry] - 18.0) / heat)
        wanted.index_put_((row, state["teacher_ids"].long()[row, entry]), raw, accumulate=True)
    else:
        inner = torch.ones(n, dtype=torch.bool, device="cuda")
        inner[state["offsets"][1:].long() - 1] = False
        if state["loss_mask"] is not None:
            inner &= state["loss_mask"]
        row = inner.nonzero().squeeze(1)
        wanted[row, ids.long()[row + 1]] = 1.0
    mass = wanted.sum(1)
    wanted /= mass.clamp(min=1e-300)[:, None]
    active = mass > 0
    spread = torch.log_softmax(hidden @ weight.T / heat, 1)
    losses = (torch.xlogy(wanted, wanted) - wanted * spread).sum(1)
    if case["op"] == "score":
        return losses
    count = max(1, int(active.sum()))
    delta = spread.exp_().sub_(wanted).mul_(active[:, None] / (heat * count))
    return {"loss": losses.sum() / count, "d_hidden": delta @ weight, "d_weight": delta.T @ hidden}
