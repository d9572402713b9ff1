"""The losses of the language-model head: what is measured of them, their plain forms and their values in 64 bits.

Three operators: softmax cross entropy of hidden states against a vocabulary matrix without keeping the logits
(`Tensor.linear_cross_entropy`), distillation from a teacher's top logits on given student logits
(`Tensor.topk_distillation`), and the two joined (`Tensor.linear_topk_distillation`).

For token t and word v, with the temperature T (1 for cross entropy): z_tv = (x_t . w_v) / T, or logit_tv / T;
p = softmax over v of z.  Targets are sparse, (id, q) pairs: cross entropy has one with q = 1, distillation has the softmax of
the teacher's top logits / T over the entries in use (id >= 0, logit above -inf).  A row with no target in use counts for nothing.
    loss_t = T^2 sum_k q_tk (log q_tk - log p_t,id_tk);    loss = sum of loss_t / n     n: the rows that count
    d loss / d logit_tv = T (p_tv - sum of q_tk with id_tk = v) / n =: G    (0 in rows that do not count)
and through the product dx = G W, dW = G^T x.  Cases with gradients take the mean loss; those without take the rows' own.
"""
import math

import torch

own = False

IGNORE = -100
#: Work of the largest listed case, which no drawn one exceeds.
LARGEST = 8192 * 768 * 50257


def listed():
    return [
        # a model of the size that tests train: latency is all that counts
        {"name": "ce_tiny", "op": "ce", "rows": 48, "width": 64, "words": 500, "grad": True, "ignored": 0.0},
        # one token scored and learned from: the vocabulary matrix is read and its gradient written for a single row
        {"name": "ce_one_token", "op": "ce", "rows": 1, "width": 768, "words": 50257, "grad": True, "ignored": 0.0},
        # ragged everything: rows, width and words share no factor with any tile
        {"name": "ce_odd", "op": "ce", "rows": 777, "width": 203, "words": 10007, "grad": True, "ignored": 0.2},
        # the evaluation loss of one sequence of GPT-2 small, forward alone
        {"name": "ce_gpt2_eval", "op": "ce", "rows": 1024, "width": 768, "words": 50257, "grad": False, "ignored": 0.0},
        # a padded batch, most of it padding, over a rounder vocabulary
        {"name": "ce_padded", "op": "ce", "rows": 2048, "width": 512, "words": 32000, "grad": True, "ignored": 0.6},
        # the training step of GPT-2 small: 8 sequences of 1024 tokens
        {"name": "ce_gpt2_step", "op": "ce", "rows": 8192, "width": 768, "words": 50257, "grad": True, "ignored": 0.0},
        # distillation on logits: a handful of rows
        {"name": "kd_small", "op": "kd", "rows": 16, "words": 1000, "top": 5, "temperature": 1.0, "grad": True, "ragged": False},
        # odd row length, long teacher lists of uneven lengths, empty ones among them
        {"name": "kd_ragged", "op": "kd", "rows": 1001, "words": 32003, "top": 100, "temperature": 2.0, "grad": True, "ragged": True},
        # GPT-2 small taught by a larger model's top 32: the training step's logits
        {"name": "kd_gpt2_step", "op": "kd", "rows": 8192, "words": 50257, "top": 32, "temperature": 2.0, "grad": True, "ragged": False},
        # hidden states of a small model
        {"name": "linear_kd_small", "op": "linear_kd", "rows": 64, "width": 128, "words": 2000, "top": 8, "temperature": 1.0, "grad": True,
         "ragged": False},
        # evaluation against the teacher, forward alone, ragged sizes
        {"name": "linear_kd_odd", "op": "linear_kd", "rows": 513, "width": 250, "words": 20011, "top": 17, "temperature": 1.5, "grad": False,
         "ragged": True},
        # GPT-2 small taught without its logits: 4 sequences of 1024 tokens
        {"name": "linear_kd_gpt2", "op": "linear_kd", "rows": 4096, "width": 768, "words": 50257, "top": 32, "temperature": 2.0, "grad": True,
         "ragged": False},
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["ce", "ce", "kd", "linear_kd"])
    while True:
        rows, width, words = _spread(rng, 1, 8192), _spread(rng, 16, 1100), _spread(rng, 200, 60000)
        if rows * words <= 8192 * 50257 and (op == "kd" or rows * width * words <= LARGEST):
            break
    case = {"op": op, "rows": rows, "words": words, "grad": rng.random() < 0.75}
    if op != "kd":
        case["width"] = width
    if op == "ce":
        case["ignored"] = rng.choice([0.0, 0.0, 0.1, 0.7])
    else:
        case["top"] = _spread(rng, 1, min(128, words))
        case["temperature"] = rng.choice([0.7, 1.0, 2.0, 4.0])
        case["ragged"] = rng.random() < 0.5
    return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=gen, device="cuda") * std

    rows, words = case["rows"], case["words"]
    state = dict(case)
    if case["op"] == "kd":
        logits = state["logits"] = normal(rows, words, std=2.5)
    else:
        # hidden states as a final layer norm leaves them, leaning towards some word's vector as those of a trained model do
        width = case["width"]
        w = state["w"] = normal(words, width, std=2.5 / math.sqrt(width))
        word = torch.randint(0, words, (rows,), generator=gen, device="cuda")
        x = state["x"] = normal(rows, width) + w[word]
        logits = x @ w.T if case["op"] == "linear_kd" else None
    if case["op"] == "ce":
        targets = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.5, word, torch.randint(0, words, (rows,), generator=gen, device="cuda"))
        padding = torch.rand(rows, generator=gen, device="cuda") < case["ignored"]
        state["targets"] = torch.where(padding, IGNORE, targets).float()        # the framework's ids are float-encoded
    else:
        # the teacher agrees with the student in part, and so do its top words
        top = (logits + normal(rows, words, std=2.0)).topk(case["top"], dim=1)
        ids, teacher = top.indices.float(), top.values.contiguous()
        if case["ragged"]:
            length = torch.randint(0, case["top"] + 1, (rows, 1), generator=gen, device="cuda")
            unused = torch.arange(case["top"], device="cuda") >= length
            ids, teacher = torch.where(unused, -1.0, ids), torch.where(unused, float("nan"), teacher)
        state["ids"], state["teacher"] = ids, teacher
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _sparse_targets(state, dtype):
    """Ids (0 in unused places), their q (0 there) and sum of q log q of each row, and whether the row counts."""
    if state["op"] == "ce":
        ids = state["targets"].long()[:, None]
        used = ids != IGNORE
        q = used.to(dtype)
        return ids.clamp(min=0), q, torch.zeros_like(q[:, 0]), used[:, 0]
    ids, t = state["ids"].long(), state["teacher"].to(dtype) / state["temperature"]
    used = (ids >= 0) & (t > -math.inf)
    t = torch.where(used, t, -math.inf)
    t = t - torch.where(used.any(1, keepdim=True), t.amax(1, keepdim=True), 0.0)
    e = torch.exp(t)
    total = e.sum(1, keepdim=True)
    q = e / torch.where(total > 0, total, 1.0)
    entropy = torch.where(q > 0, q * torch.log(torch.where(q > 0, q, 1.0)), 0.0).sum(1)
    return ids.clamp(min=0), q, entropy, used.any(1)


def _run_plain(state):
    temperature = state.get("temperature", 1.0)
    ids, q, entropy, counts = _sparse_targets(state, torch.float32)
    logits = state["logits"] if state["op"] == "kd" else state["x"] @ state["w"].T
    z = logits / temperature if temperature != 1.0 else logits
    shifted = z - z.amax(1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(1, keepdim=True)
    log_p = torch.gather(shifted, 1, ids) - torch.log(total)
    row = entropy - torch.where(q > 0, q * log_p, 0.0).sum(1)
    row = temperature ** 2 * torch.where(counts, row, 0.0)
    if not state["grad"]:
        return {"losses": row}
    n = counts.sum().clamp(min=1)
    loss = (row.double().sum() / n).float().reshape(1)
    g = (e / total).scatter_add_(1, ids, -q)
    g = g * (torch.where(counts, temperature, 0.0) / n)[:, None]
    if state["op"] == "kd":
        return {"loss": loss, "dlogits": g}
    return {"loss": loss, "dx": g @ state["w"], "dw": g.T @ state["x"]}


class _Memory:
    """A tensor of the framework, as torch reads it without a copy."""

    def __init__(self, t):
        self.keep = t
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": "<f4", "data": (t.ptr, False), "version": 3, "strides": None}


def _run_own(state):
    from gradtuity_b200 import Tensor

    def given(name, grad=False):
        t = state[name]
        return Tensor._from_ptr(t.data_ptr(), tuple(t.shape), owns_memory=False, requires_grad=grad and state["grad"])

    def out(t):
        return torch.as_tensor(_Memory(t), device="cuda")

    how = "mean" if state["grad"] else "none"
    # 3xtf32: products as exact as 32-bit sums, as the plain form's are
    if state["op"] == "kd":
        logits = given("logits", grad=True)
        loss = logits.topk_distillation(given("ids"), given("teacher"), temperature=state["temperature"], reduction=how)
        grads = {"dlogits": logits}
    else:
        x, w = given("x", grad=True), given("w", grad=True)
        if state["op"] == "ce":
            loss = x.linear_cross_entropy(w, given("targets"), reduction=how, ignore_index=IGNORE, precision="3xtf32")
        else:
            loss = x.linear_topk_distillation(w, given("ids"), given("teacher"), temperature=state["temperature"], reduction=how,
                                               precision="3xtf32")
        grads = {"dx": x, "dw": w}
    if not state["grad"]:
        return {"losses": out(loss)}
    loss.backward()
    return {"loss": out(loss), **{name: out(t.grad) for name, t in grads.items()}}


def work(case):
    rows, words, flops = case["rows"], case["words"], 0
    if case["op"] == "kd":
        data = 4 * rows * words * (2 if case["grad"] else 1)
        flops = rows * words * (8 if case["grad"] else 5)
    else:
        data = 4 * case["width"] * (rows + words) * (2 if case["grad"] else 1)
        flops = 2 * rows * words * case["width"] * (3 if case["grad"] else 1)
    data += 4 * rows if case["op"] == "ce" else 8 * rows * case["top"]
    return {"bytes": data, "flops": flops}


def exact(case, seed):
    """The same in 64 bits, a few hundred rows at a time, from log-probabilities and dense targets."""
    state = prepare(case, seed)
    rows, words, temperature = case["rows"], case["words"], case.get("temperature", 1.0)
    dtype = torch.float64
    n = 0
    losses, grads, dx, dw = [], [], [], 0.0
    w = state["w"].to(dtype) if "w" in state else None
    for at in range(0, rows, 512):
        part = slice(at, min(rows, at + 512))
        z = state["logits"][part].to(dtype) if w is None else state["x"][part].to(dtype) @ w.T
        log_p = torch.log_softmax(z / temperature, dim=1)
        dense = torch.zeros_like(log_p)                      # the target distribution over all words
        if case["op"] == "ce":
            target = state["targets"][part].long()
            counted = target != IGNORE
            dense[counted.nonzero()[:, 0], target[counted]] = 1.0
        else:
            ids, t = state["ids"][part].long(), state["teacher"][part].to(dtype)
            used = ids >= 0
            counted = used.any(1)
            q = torch.softmax(torch.where(used, t / temperature, -math.inf), dim=1)
            dense.scatter_add_(1, torch.where(used, ids, 0), torch.where(used, q, 0.0))
        losses.append(temperature ** 2 * counted * (torch.special.xlogy(dense, dense) - dense * log_p).sum(1))
        n += int(counted.sum())
        if case["grad"]:
            g = temperature * (log_p.exp() - dense) * counted[:, None]
            if w is None:
                grads.append(g)
            else:
                dx.append(g @ w)
                dw = dw + g.T @ state["x"][part].to(dtype)
    losses = torch.cat(losses)
    if not case["grad"]:
        return {"losses": losses}
    n = max(1, n)
    out = {"loss": (losses.sum() / n).reshape(1)}
    out.update({"dlogits": torch.cat(grads) / n} if w is None else {"dx": torch.cat(dx) / n, "dw": dw / n})
    return out
