"""The vocabulary operators of clip_amd.losses on one MI355X: what is timed, in a plain form and through the library.

Three operators of an LM head's training and evaluation, over hidden rows [n, H], a decoder weight [V, H] and its
bias [V] (BERT-base: H 768, V 30 522):

  ce        softmax cross entropy of hidden @ weight.T + bias against labels, rows with label -100 left out
  distill   T^2 KL(teacher || student) at temperature T, the teacher given by its top logits and their vocabulary ids
  topk      a row's largest k logits with their ids, ties to the lowest id (what a teacher hands to `distill`)

A "loss" case is the forward pass alone (one loss per row), a "train" case the loss with the gradients of hidden
rows, weight and bias."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
IGNORE = -100


def listed():
    return [
        # one masked token scored on its own: pure latency, the decoder weight read once
        {"name": "ce loss, one row", "op": "ce", "train": False, "n": 1, "h": 768, "v": 30522, "dtype": "bf16", "labelled": 1.0,
         "reduction": "none"},
        # evaluation over whole batches: 32 rows of 512 tokens, 15 % of the tokens carry an MLM label
        {"name": "ce loss, 15 % of 16384", "op": "ce", "train": False, "n": 16384, "h": 768, "v": 30522, "dtype": "f16", "labelled": 0.15,
         "reduction": "none"},
        # the small test geometry: everything is launch latency
        {"name": "ce train, 37 rows tiny", "op": "ce", "train": True, "n": 37, "h": 128, "v": 2000, "dtype": "bf16", "labelled": 1.0,
         "reduction": "mean"},
        # a pre-training step on the reference's batch of 8 rows of 256 tokens, 15 % labelled
        {"name": "ce train, 15 % of 2048", "op": "ce", "train": True, "n": 2048, "h": 768, "v": 30522, "dtype": "bf16", "labelled": 0.15,
         "reduction": "mean"},
        # the labelled rows of a larger step, already picked out
        {"name": "ce train, 4096 rows", "op": "ce", "train": True, "n": 4096, "h": 768, "v": 30522, "dtype": "bf16", "labelled": 1.0,
         "reduction": "mean"},
        # every token of 64 rows of 256 tokens labelled (a causal or full-reconstruction objective): the largest
        {"name": "ce train, 16384 rows", "op": "ce", "train": True, "n": 16384, "h": 768, "v": 30522, "dtype": "bf16", "labelled": 1.0,
         "reduction": "mean"},
        # a wider encoder with an expanded vocabulary (odd), fp16 operands, rows weighted one by one
        {"name": "ce train, 2500 rows f16 wide", "op": "ce", "train": True, "n": 2500, "h": 1024, "v": 31019, "dtype": "f16", "labelled": 1.0,
         "reduction": "none"},
        # a distillation loss watched during evaluation, ragged teacher lists
        {"name": "distill loss, 777 rows", "op": "distill", "train": False, "n": 777, "h": 768, "v": 30522, "dtype": "f16", "k": 32, "temperature": 2.0,
         "ragged": True, "reduction": "none"},
        # the masked tokens of one small batch
        {"name": "distill train, 19 rows", "op": "distill", "train": True, "n": 19, "h": 768, "v": 30522, "dtype": "bf16", "k": 8, "temperature": 1.0,
         "ragged": False, "reduction": "mean"},
        # a student half as wide learning from 64 teacher logits per row
        {"name": "distill train, 4096 rows", "op": "distill", "train": True, "n": 4096, "h": 512, "v": 30522, "dtype": "bf16", "k": 64, "temperature": 2.0,
         "ragged": True, "reduction": "mean"},
        # a teacher's scores for the masked tokens of one short row
        {"name": "topk, 5 rows", "op": "topk", "n": 5, "v": 30522, "dtype": "f32", "k": 10},
        # a teacher's scores for a large step, 64 kept of each row
        {"name": "topk, 8192 rows", "op": "topk", "n": 8192, "v": 30522, "dtype": "f32", "k": 64},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["ce", "ce", "distill", "distill", "topk"])
    if op == "topk":
        return {"op": op, "n": _log_int(rng, 1, 4096), "v": _log_int(rng, 300, 50000), "dtype": rng.choice(["f32", "f32", "bf16", "f16"]),
                "k": _log_int(rng, 1, 128)}
    case = {"op": op, "train": rng.random() < 0.7, "n": _log_int(rng, 1, 8192), "h": rng.choice([128, 256, 512, 768, 1024]),
            "v": _log_int(rng, 1000, 40000), "dtype": rng.choice(["bf16", "f16"]), "reduction": rng.choice(["mean", "none"])}
    if op == "ce":
        return dict(case, labelled=rng.choice([1.0, 1.0, 0.5, 0.15]))
    return dict(case, k=_log_int(rng, 1, 128), temperature=rng.choice([1.0, 1.5, 2.0, 4.0]), ragged=rng.random() < 0.5)


def _labelled(case):
    return max(1, round(case["n"] * case["labelled"])) if case["op"] == "ce" else case["n"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    n, v, dtype = case["n"], case["v"], DTYPES[case["dtype"]]
    if case["op"] == "topk":
        # the spread of an LM head's scores; 16-bit scores hold many ties
        return {"case": case, "logits": (2.5 * normal(n, v)).to(dtype)}
    h = case["h"]
    weight = 0.05 * normal(v, h)
    # word frequencies fall off like 1 / rank: ids spread over the vocabulary, frequent ones more often
    ids = torch.exp(torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * math.log(v)).long().clamp_(1, v) - 1
    # LayerNorm output of a partly trained head: the right word scores between an average one and a likely one
    lift = 0.9 * math.log(v) * torch.rand(n, 1, generator=gen, device="cuda")
    hidden = normal(n, h) + lift * weight[ids] / (0.05 ** 2 * h)
    hidden = (hidden - hidden.mean(1, keepdim=True)) / hidden.std(1, keepdim=True)
    state = {"case": case, "hidden": hidden.to(dtype), "weight": weight.to(dtype), "bias": 0.5 * normal(v)}
    if case["op"] == "ce":
        order = torch.rand(n, generator=gen, device="cuda").argsort()
        state["labels"] = ids.index_fill(0, order[_labelled(case):], IGNORE)
    else:
        scores = 2.0 * normal(n, v)
        scores.scatter_(1, ids[:, None], 9.0)
        values, index = scores.topk(min(case["k"], v), dim=1)
        if case["ragged"]:   # lists cut at 95 % of the listed probability: the rest is marked with id -1
            share = torch.softmax(values, 1).cumsum(1)
            index = index.masked_fill(torch.nn.functional.pad(share[:, :-1], (1, 0)) > 0.95, -1)
        state["values"], state["index"] = values.contiguous(), index.contiguous()
    if case["reduction"] == "none" and case["train"]:
        state["row_weight"] = torch.rand(n, generator=gen, device="cuda") / n
    for name in ("hidden", "weight", "bias"):
        state[name].requires_grad_(case["train"])
    return state


def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    with torch.no_grad():
        return {"ce": _plain_ce, "distill": _plain_distill, "topk": _plain_topk}[case["op"]](case, state)


def _own(case, state):
    from clip_amd import losses

    if case["op"] == "topk":
        return losses.topk_logits(state["logits"], case["k"])
    if case["op"] == "ce":
        loss = losses.linear_cross_entropy(state["hidden"], state["weight"], state["bias"], state["labels"], ignore_index=IGNORE,
                                           reduction=case["reduction"])
    else:
        loss = losses.linear_distillation(state["hidden"], state["weight"], state["bias"], state["values"], state["index"],
                                          temperature=case["temperature"], reduction=case["reduction"])
    if not case["train"]:
        return loss
    grads = torch.autograd.grad(loss, (state["hidden"], state["weight"], state["bias"]), state.get("row_weight"))
    return (loss.detach(), *grads)


def _softmax(z):
    top = z.amax(1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(1, keepdim=True)
    return e / total, (top + total.log())[:, 0]


def _finish(case, state, row_loss, live, dz):
    """Reduces the rows' losses; dz: the gradient of each row's loss in its logits, which it overwrites."""
    count = live.sum()
    loss = row_loss if case["reduction"] == "none" else row_loss.sum() / count
    if not case["train"]:
        return loss
    scale = live / count if case["reduction"] == "mean" else live * state["row_weight"]
    dz *= scale[:, None]
    hidden, weight = state["hidden"], state["weight"]
    return loss, (dz @ weight.float()).to(hidden.dtype), (dz.t() @ hidden.float()).to(weight.dtype), dz.sum(0)


def _plain_ce(case, state):
    labels = state["labels"]
    live = (labels != IGNORE).float()
    z = state["hidden"].float() @ state["weight"].float().t() + state["bias"]
    p, lse = _softmax(z)
    at = labels.clamp(min=0)[:, None]
    row_loss = (lse - z.gather(1, at)[:, 0]) * live
    p.scatter_add_(1, at, torch.full_like(at, -1, dtype=p.dtype))
    return _finish(case, state, row_loss, live, p)


def _plain_distill(case, state):
    t, index = case["temperature"], state["index"]
    there = index >= 0
    live = there.any(1).float()
    z = (state["hidden"].float() @ state["weight"].float().t() + state["bias"]) / t
    q, lse = _softmax(z)
    at = index.clamp(min=0)
    p, teacher_lse = _softmax((state["values"] / t).masked_fill(~there, -math.inf))
    log_p = (state["values"] / t - teacher_lse[:, None]).masked_fill(~there, 0.0)
    row_loss = t * t * (p * (log_p - z.gather(1, at) + lse[:, None])).sum(1)
    q.scatter_add_(1, at, -p)
    return _finish(case, state, row_loss, live, q.mul_(t))


def _plain_topk(case, state):
    values, index = state["logits"].sort(dim=1, descending=True, stable=True)
    return values[:, :case["k"]].contiguous(), index[:, :case["k"]].contiguous()


def work(case):
    n, v = case["n"], case["v"]
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "topk":
        return {"bytes": n * v * size + n * min(case["k"], v) * (size + 8), "flops": n * v}
    rows, h = _labelled(case), case["h"]
    given = rows * h * size + v * h * size + 4 * v + (8 * n if case["op"] == "ce" else 12 * n * case["k"])
    if not case["train"]:
        return {"bytes": given + 4 * n, "flops": 2 * rows * v * h}
    return {"bytes": given + n * h * size + v * h * size + 4 * v + 4 * n, "flops": 6 * rows * v * h}


def exact(case, seed):
    """The definitions in 64 bits: the losses by log_softmax, the gradients by automatic differentiation."""
    state = prepare(case, seed)
    if case["op"] == "topk":
        return state["logits"].double().topk(case["k"], dim=1).values, None
    hidden, weight, bias = (state[name].detach().double().requires_grad_(case["train"]) for name in ("hidden", "weight", "bias"))
    t = case.get("temperature", 1.0)
    log_q = torch.log_softmax(torch.addmm(bias, hidden, weight.t()) / t, 1)
    if case["op"] == "ce":
        kept = state["labels"] != IGNORE
        row_loss = torch.where(kept, -log_q[torch.arange(case["n"], device="cuda"), state["labels"].where(kept, 0)], 0.0)
    else:
        listed_ = state["index"] >= 0
        kept = listed_.any(1)
        log_p = torch.log_softmax(torch.where(listed_, state["values"].double() / t, -math.inf), 1)
        gap = log_p.masked_fill(~listed_, 0.0) - torch.gather(log_q, 1, state["index"].where(listed_, 0))
        row_loss = t ** 2 * (log_p.exp() * gap).sum(1)
    loss = row_loss if case["reduction"] == "none" else row_loss.sum() / kept.sum()
    if not case["train"]:
        return loss
    weights = state["row_weight"].double() if case["reduction"] == "none" else None
    return (loss.detach(), *torch.autograd.grad(loss, (hidden, weight, bias), weights))
