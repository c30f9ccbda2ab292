"""The vocabulary operators of the masked-token head and what they are measured on: cross entropy and distillation over a large
vocabulary (forward and backward, from hidden states and the decoder's rows) and the selection of a teacher's top logits.

`own` False: the operators in their plain form (elementary torch operations in fp32); True: the calls a user makes.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
MOST = 8192 * 131072 * 2048           # rows x vocabulary x hidden of the largest listed case
MOST_LOGITS = 4096 * 131072           # rows x vocabulary of the largest selection


def listed():
    ce = dict(op="cross_entropy", k=0, temperature=1.0)
    kd = dict(op="distillation", ignored=0.0)
    top = dict(op="top_logits", hidden=0, bias=False, ignored=0.0, grads="none", temperature=1.0)
    return [
        # the pre-training step's masked-token head: 32 instructions of 80 tokens, 15 % masked, the others ignored
        dict(ce, name="ce mlm step fp32", rows=2560, vocab=30522, hidden=768, dtype="fp32", bias=True, ignored=0.85, grads="all"),
        # one masked token of one instruction, scored only: latency
        dict(ce, name="ce one token fp32", rows=1, vocab=30522, hidden=768, dtype="fp32", bias=True, ignored=0.0, grads="none"),
        # a reduced head, as the tests' configurations have it, trained on a few tokens
        dict(ce, name="ce reduced head fp32", rows=37, vocab=1000, hidden=256, dtype="fp32", bias=True, ignored=0.1, grads="all"),
        # a long-context batch over a large vocabulary, half precision, whole training step: the largest
        dict(ce, name="ce large step bf16", rows=8192, vocab=131072, hidden=2048, dtype="bf16", bias=False, ignored=0.02, grads="all"),
        # validation: losses only, odd vocabulary
        dict(ce, name="ce validation fp16", rows=3001, vocab=50021, hidden=1024, dtype="fp16", bias=True, ignored=0.0, grads="none"),
        # the encoder is trained under a frozen decoder; a hidden size that fills no tile
        dict(ce, name="ce frozen decoder bf16", rows=1535, vocab=32003, hidden=1032, dtype="bf16", bias=False, ignored=0.3, grads="hidden"),
        # the masked tokens of a step against a teacher's 32 top logits
        dict(kd, name="kd mlm step fp32", rows=384, vocab=30522, hidden=768, dtype="fp32", bias=True, k=32, temperature=2.0, grads="all"),
        # one token per call: a handful of rows
        dict(kd, name="kd few tokens bf16", rows=5, vocab=30522, hidden=768, dtype="bf16", bias=True, k=8, temperature=1.0, grads="all"),
        # a long batch, many slots
        dict(kd, name="kd large step bf16", rows=4099, vocab=65537, hidden=2048, dtype="bf16", bias=False, k=128, temperature=1.5, grads="all"),
        # the teacher's scores of a pre-training step
        dict(top, name="top mlm step fp32", rows=384, vocab=30522, dtype="fp32", k=32),
        # one token's scores
        dict(top, name="top one token bf16", rows=1, vocab=131071, dtype="bf16", k=64),
        # a teacher's pass over a long batch
        dict(top, name="top large bf16", rows=4096, vocab=131072, dtype="bf16", k=128),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(("cross_entropy", "cross_entropy", "distillation", "distillation", "top_logits"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    vocab = _log(rng, 300, 131072)
    if op == "top_logits":
        rows = min(_log(rng, 1, 4096), MOST_LOGITS // (vocab * (2 if dtype == "fp32" else 1)))
        return dict(op=op, rows=rows, vocab=vocab, hidden=0, dtype=dtype, bias=False, ignored=0.0, k=_log(rng, 1, 256),
                    temperature=1.0, grads="none")
    hidden = _log(rng, 64, 4096)
    if rng.random() < 0.6:
        hidden = max(64, hidden // 64 * 64)
    rows = max(1, min(_log(rng, 1, 8192), MOST // (vocab * hidden * (4 if dtype == "fp32" else 1))))
    common = dict(op=op, rows=rows, vocab=vocab, hidden=hidden, dtype=dtype, bias=rng.random() < 0.5,
                  grads=rng.choice(("all", "all", "hidden", "none")))
    if op == "cross_entropy":
        return dict(common, ignored=rng.choice((0.0, 0.15, 0.85)), k=0, temperature=1.0)
    return dict(common, ignored=0.0, k=_log(rng, 1, 256), temperature=rng.choice((0.5, 1.0, 2.0, 4.0)))


def _counted(case):
    """Rows that are not ignored."""
    return max(1, case["rows"] - int(case["rows"] * case["ignored"]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, R, V, K = DTYPES[case["dtype"]], case["rows"], case["vocab"], case["hidden"]

    def normal(*shape, std=1.0):
        return torch.empty(shape, dtype=dt, device="cuda").normal_(0.0, std, generator=g)

    s = dict(case=case)
    if case["op"] == "top_logits":
        s["logits"] = normal(R, V, std=2.5)
        return s
    # hidden states behind a LayerNorm; decoder rows that give logits of a trained head's spread
    s["hidden"] = normal(R, K).requires_grad_(case["grads"] != "none")
    s["weight"] = normal(V, K, std=2.0 / math.sqrt(K)).requires_grad_(case["grads"] == "all")
    s["bias"] = normal(V, std=0.5).requires_grad_(case["grads"] == "all") if case["bias"] else None
    if case["grads"] != "none":
        # what the mean over the counted rows hands down, times a weight of each row
        s["grad"] = torch.rand(R, device="cuda", generator=g).add_(0.5).div_(_counted(case))
    if case["op"] == "cross_entropy":
        labels = torch.randint(0, V, (R,), device="cuda", generator=g)
        drop = torch.randperm(R, device="cuda", generator=g)[: R - _counted(case)]
        labels[drop] = -1
        s["labels"] = labels
        return s
    # a teacher's top logits: falling values, ids that are distinct within a row (a stride that is prime to V walks through them)
    k = min(case["k"], V)
    stride = next(p for p in (7919, 7907, 7901) if V % p)
    first = torch.randint(0, V, (R, 1), device="cuda", generator=g)
    s["ids"] = (first + stride * torch.arange(k, device="cuda")) % V
    s["values"] = (torch.rand(R, k, device="cuda", generator=g) * 8.0).sort(1, descending=True)[0]
    return s


def _plain_scores(s, rows=None):
    """z = h W^T + b in fp32, and its factors."""
    h = s["hidden"].detach()
    h = (h if rows is None else h[rows]).float()
    w = s["weight"].detach().float()
    z = h @ w.t()
    return h, w, z if s["bias"] is None else z + s["bias"].detach().float()


def _plain_grads(s, out, d, h, w, rows=None):
    """The gradients of hidden, weight and bias from d = the gradient of z."""
    dt = s["hidden"].dtype
    if rows is None:
        out["d_hidden"] = (d @ w).to(dt)
    else:
        full = torch.zeros(s["hidden"].shape, dtype=dt, device=d.device)
        full[rows] = (d @ w).to(dt)
        out["d_hidden"] = full
    if s["case"]["grads"] == "all":
        out["d_weight"] = (d.t() @ h).to(dt)
        if s["bias"] is not None:
            out["d_bias"] = d.sum(0).to(dt)
    return out


def _plain_cross_entropy(s):
    rows = (s["labels"] != -1).nonzero().squeeze(1)
    y = s["labels"][rows].unsqueeze(1)
    h, w, z = _plain_scores(s, rows)
    top = z.amax(1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(1, keepdim=True)
    loss = torch.zeros(s["case"]["rows"], device=z.device)
    loss[rows] = ((top - z.gather(1, y)) + total.log()).squeeze(1)
    out = dict(loss=loss)
    if s["case"]["grads"] == "none":
        return out
    d = e.div_(total)
    d.scatter_add_(1, y, torch.full(y.shape, -1.0, device=d.device))
    d.mul_(s["grad"][rows].unsqueeze(1))
    return _plain_grads(s, out, d, h, w, rows)


def _plain_distillation(s):
    T, ids = s["case"]["temperature"], s["ids"]
    h, w, z = _plain_scores(s)
    z = z / T
    top = z.amax(1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(1, keepdim=True)
    lse = top + total.log()
    t = s["values"].float() / T
    t = t - t.amax(1, keepdim=True)
    log_p = t - t.exp().sum(1, keepdim=True).log()
    p = log_p.exp()
    out = dict(loss=T * T * (p * (log_p - (z.gather(1, ids) - lse))).sum(1))
    if s["case"]["grads"] == "none":
        return out
    d = e.div_(total)
    d.scatter_add_(1, ids, -p)
    d.mul_((s["grad"] * T).unsqueeze(1))
    return _plain_grads(s, out, d, h, w)


def _plain_top(s):
    x, k = s["logits"], min(s["case"]["k"], s["case"]["vocab"])
    values, ids = x.sort(dim=1, descending=True, stable=True)      # ties: the lowest id first
    z = x.float()
    top = z.amax(1, keepdim=True)
    return dict(values=values[:, :k].contiguous(), ids=ids[:, :k].contiguous(), lse=(top + (z - top).exp().sum(1, keepdim=True).log()).squeeze(1))


def _own(s):
    from gridmm_amd import vocab
    case = s["case"]
    if case["op"] == "top_logits":
        values, ids, lse = vocab.top_logits(s["logits"], min(case["k"], case["vocab"]))
        return dict(values=values, ids=ids, lse=lse)
    if case["op"] == "cross_entropy":
        loss = vocab.vocab_cross_entropy(s["hidden"], s["weight"], s["labels"], bias=s["bias"], ignore_index=-1)
    else:
        loss = vocab.vocab_distillation(s["hidden"], s["weight"], s["ids"], s["values"], bias=s["bias"],
                                        temperature=case["temperature"])
    out = dict(loss=loss.detach())
    if case["grads"] == "none":
        return out
    leaves = {"d_hidden": s["hidden"]}
    if case["grads"] == "all":
        leaves["d_weight"] = s["weight"]
        if s["bias"] is not None:
            leaves["d_bias"] = s["bias"]
    out.update(zip(leaves, torch.autograd.grad(loss, list(leaves.values()), s["grad"])))
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"cross_entropy": _plain_cross_entropy, "distillation": _plain_distillation,
                "top_logits": _plain_top}[state["case"]["op"]](state)


def work(case):
    b, R, V, K = SIZE[case["dtype"]], _counted(case), case["vocab"], case["hidden"]
    if case["op"] == "top_logits":
        return {"bytes": R * V * b + R * min(case["k"], V) * (b + 8) + 4 * R, "flops": 3 * R * V}
    n = R * K * b + V * K * b + case["bias"] * V * b + 4 * case["rows"]
    n += 8 * case["rows"] if case["op"] == "cross_entropy" else R * min(case["k"], V) * 12
    products = 1
    if case["grads"] != "none":
        n, products = n + case["rows"] * (K * b + 4), 2
    if case["grads"] == "all":
        n, products = n + V * K * b + case["bias"] * V * b, 3
    return {"bytes": n, "flops": products * 2 * R * V * K}


def exact(case, seed):
    """From the definitions, in 64 bits, by torch's own differentiation of them."""
    s = prepare(case, seed)
    if case["op"] == "top_logits":
        x = s["logits"].double()
        order = torch.argsort(x, dim=1, descending=True, stable=True)[:, : min(case["k"], case["vocab"])]
        return dict(values=torch.gather(x, 1, order), ids=None, lse=torch.logsumexp(x, 1))
    h = s["hidden"].detach().double().requires_grad_()
    w = s["weight"].detach().double().requires_grad_(case["grads"] == "all")
    b = None if s["bias"] is None else s["bias"].detach().double().requires_grad_(case["grads"] == "all")
    z = torch.nn.functional.linear(h, w, b)
    if case["op"] == "cross_entropy":
        loss = torch.nn.functional.cross_entropy(z, s["labels"], ignore_index=-1, reduction="none")
    else:
        T = case["temperature"]
        log_q = torch.log_softmax(z / T, 1).gather(1, s["ids"])
        log_p = torch.log_softmax(s["values"].double() / T, 1)
        loss = T * T * (log_p.exp() * (log_p - log_q)).sum(1)
    out = dict(loss=loss.detach())
    if case["grads"] != "none":
        names = ["d_hidden"] + (["d_weight"] + (["d_bias"] if b is not None else []) if case["grads"] == "all" else [])
        leaves = [h] + ([w] + ([b] if b is not None else []) if case["grads"] == "all" else [])
        out.update(zip(names, torch.autograd.grad(loss, leaves, s["grad"].double())))
    return out
