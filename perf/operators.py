"""The operators at the two ends of a language model's training step, as a user calls them: the rows of an
embedding table and their gradient, and the loss against a teacher's top logits with its gradient.

``own`` False: elementary torch operations in 32 bits, rounded once.  ``own`` True: ``raf_b200.op``.
Tables and vocabularies are those of the BERT-large and GPT-2-medium parameter lists (30522 and 50257 rows
of 1024, 512 positions, 2 segment types); tokens are drawn as words are, a few of them very often.
"""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16,
         "int32": torch.int32, "int64": torch.int64}
IGNORE = -100


def listed():
    lookup = {"op": "lookup", "dtype": "bfloat16", "out": "bfloat16", "ids": "int64", "scale": 1.0}
    grad = {"op": "gradient", "dtype": "bfloat16", "out": "bfloat16", "ids": "int64", "scale": 1.0, "accumulate": False,
            "padding": -1}
    loss = {"dtype": "bfloat16", "ids": "int64", "pad": 0, "temperature": 1.0, "alpha": 1.0, "labels": False, "grad_scale": 1.0}
    return [
        # one sequence of a fine-tuning step: latency
        dict(lookup, name="lookup-sequence", n=128, v=30522, h=1024),
        # a whole batch from the fp32 master table into the model's type, scaled by the root of the width,
        # with a width that leaves no row on a wide boundary but the first
        dict(lookup, name="lookup-master-ragged", dtype="float32", ids="int32", n=20011, v=30522, h=1023, scale=31.984),
        # the largest batch a GPU takes at once
        dict(lookup, name="lookup-batch", n=65536, v=50257, h=1024, scale=32.0),
        # position embeddings of one sequence: latency
        dict(grad, name="gradient-positions", n=512, v=512, h=1024),
        # word embeddings of an ordinary batch, padding tokens left out, into the flat 16-bit gradient
        dict(grad, name="gradient-words", n=16384, v=30522, h=1024, padding=0),
        # a further micro-batch, added to the fp32 gradient that the optimizer reads
        dict(grad, name="gradient-accumulate", out="float32", ids="int32", n=65536, v=50257, h=1024, scale=32.0, accumulate=True),
        # segment types: two rows that take every token
        dict(grad, name="gradient-types", out="float32", n=65536, v=2, h=1024),
        # the loss of a few scored tokens, fp32 logits: latency
        dict(loss, op="loss", name="loss-few", dtype="float32", n=4, v=50257, k=16),
        # the loss of a batch (the masked words of BERT), softened, with the hard labels beside the teacher
        dict(loss, op="loss", name="loss-batch", n=4096, v=30522, k=64, temperature=2.0, alpha=0.5, labels=True),
        # the gradient of an fp16 run with its loss scale; odd rows, so that they start anywhere
        dict(loss, op="dpred", name="dpred-ragged", dtype="float16", ids="int32", n=777, v=50257, k=32, grad_scale=65536.0),
        # loss and gradient at once, a few rows of logits whose rows are padded for the matrix product in front
        dict(loss, op="both", name="both-few", n=31, v=50257, k=16, pad=47),
        # loss and gradient of the largest batch
        dict(loss, op="both", name="both-batch", n=8192, v=50257, k=64, temperature=2.0, alpha=0.5, labels=True, pad=47),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["lookup", "gradient", "loss", "dpred", "both"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    ids = rng.choice(["int32", "int64"])
    if op in ("lookup", "gradient"):
        case = {"op": op, "dtype": dtype, "out": rng.choice([dtype, "float32", "bfloat16"]), "ids": ids,
                "scale": rng.choice([1.0, round(rng.uniform(0.1, 50.0), 3)]), "n": _spread(rng, 1, 65536),
                "v": _spread(rng, 2, 50257), "h": _spread(rng, 16, 1024)}
        if rng.random() < 0.5:  # most widths are multiples of eight
            case["h"] = max(16, case["h"] // 8 * 8)
        if op == "gradient":
            case.update(accumulate=rng.random() < 0.4, padding=rng.choice([-1, 0]))
        return case
    labels = rng.random() < 0.5
    n = _spread(rng, 1, 2048)
    # 16-bit floats need a loss scale, or what divides by the number of tokens falls below their smallest normal value
    scale = min(65536.0, 1024.0 * 2 ** int(math.log2(n))) if dtype == "float16" else rng.choice([1.0, 128.0])
    return {"op": op, "dtype": dtype, "ids": ids, "n": n, "v": _spread(rng, 64, 50257),
            "k": _spread(rng, 1, 64), "pad": rng.choice([0, 0, 7, 64]),
            "temperature": rng.choice([1.0, 2.0, round(rng.uniform(0.5, 8.0), 2)]),
            "alpha": round(rng.uniform(0.1, 0.9), 2) if labels else 1.0, "labels": labels,
            "grad_scale": scale}


def _tokens(case, g):
    """Ids whose frequency falls with the inverse of their rank, ranks dealt out at random."""
    n, v = case["n"], case["v"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
    return torch.randperm(v, generator=g, device="cuda")[rank].to(TYPES[case["ids"]])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    dtype = TYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "lookup":
        s["x"] = (normal(case["v"], case["h"]) * 0.02).to(dtype)
        s["indices"] = _tokens(case, g)
    elif case["op"] == "gradient":
        s["dy"] = (normal(case["n"], case["h"]) * 1e-3).to(dtype)
        s["indices"] = _tokens(case, g)
        if case["accumulate"]:
            s["dx"] = (normal(case["v"], case["h"]) * 1e-3).to(TYPES[case["out"]])
    else:
        n, v, k = case["n"], case["v"], min(case["k"], case["v"])
        logits = normal(n, v) * 2.0
        teacher, ids = (logits + normal(n, v)).topk(k, dim=1)
        absent = torch.rand(n, k, generator=g, device="cuda") < 0.02  # fewer entries than the list has room for
        s["teacher_logits"] = teacher.to(dtype)
        s["teacher_ids"] = torch.where(absent, torch.full_like(ids, -1), ids).to(TYPES[case["ids"]])
        buffer = torch.zeros(n, v + case["pad"], dtype=dtype, device="cuda")
        buffer[:, :v] = logits
        s["pred"] = buffer[:, :v]
        s["labels"] = None
        if case["labels"]:
            labels = torch.randint(0, v, (n,), generator=g, device="cuda")
            out = torch.rand(n, generator=g, device="cuda") < 0.1  # tokens that carry no loss
            s["labels"] = torch.where(out, torch.full_like(labels, IGNORE), labels).to(TYPES[case["ids"]])
        s["dy"] = torch.rand(n, generator=g, device="cuda") / n
        s["how"] = {"labels": s["labels"], "temperature": case["temperature"], "alpha": case["alpha"], "ignore_index": IGNORE}
        if case["op"] == "dpred":  # the forward pass has left max and sum of each row
            s["stats"] = _stats(s["pred"], case["temperature"])
    return s


def _stats(pred, temperature):
    """What the forward pass hands to the backward pass: each row's maximum, and its sums of exponentials at the
    temperature and at one."""
    z = pred.float()
    top = z.amax(1, keepdim=True)
    return torch.stack([top[:, 0], torch.exp((z - top) / temperature).sum(1), torch.exp(z - top).sum(1), torch.zeros_like(top[:, 0])], 1)


def run(s):
    c = s["case"]
    if own:
        from raf_b200 import op

        if c["op"] == "lookup":
            return op.embedding(s["x"], s["indices"], c["scale"], dtype=TYPES[c["out"]])
        if c["op"] == "gradient":
            return op.embedding_dx(s["dy"], s["indices"], c["v"], c["scale"], padding_idx=c["padding"],
                                   dtype=TYPES[c["out"]], out=s.get("dx"), accumulate=c["accumulate"])
        if c["op"] == "loss":
            return op.distill_loss(s["pred"], s["teacher_logits"], s["teacher_ids"], **s["how"])[0]
        if c["op"] == "dpred":
            return op.distill_loss_dpred(s["dy"], s["pred"], s["teacher_logits"], s["teacher_ids"], s["stats"],
                                         grad_scale=c["grad_scale"], **s["how"])
        return op.distill_loss_with_dpred(s["dy"], s["pred"], s["teacher_logits"], s["teacher_ids"],
                                          grad_scale=c["grad_scale"], **s["how"])
    if c["op"] == "lookup":
        return (s["x"][s["indices"].long()].float() * c["scale"]).to(TYPES[c["out"]])
    if c["op"] == "gradient":
        return _gradient(s, c)
    return _distill(s, c)


def _gradient(s, c):
    ids = s["indices"].long()
    ids = torch.where(ids == c["padding"], torch.full_like(ids, c["v"]), ids)  # a row that is cut off again
    total = torch.zeros(c["v"] + 1, c["h"], device="cuda")
    total.index_add_(0, ids, s["dy"].float())
    total = total[:-1] * c["scale"]
    if c["accumulate"]:
        return s["dx"].copy_(s["dx"].float() + total)
    return total.to(TYPES[c["out"]])


def _distill(s, c):
    temp, alpha = c["temperature"], c["alpha"]
    z = s["pred"].float()
    ids = s["teacher_ids"].long()
    here = ids >= 0
    at = ids.clamp(min=0)
    t = torch.where(here, s["teacher_logits"].float() / temp, torch.full((), -math.inf, device="cuda"))
    t = t - t.amax(1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(t)
    total = p.sum(1, keepdim=True)
    some = (total > 0).float()
    total = total.clamp(min=1e-30)
    log_p = torch.where(here, t - torch.log(total), torch.zeros_like(t))
    p = p / total

    top = z.amax(1, keepdim=True)
    soft = torch.exp((z - top) / temp)
    soft_sum = soft.sum(1, keepdim=True)
    log_q = (z.gather(1, at) - top) / temp - torch.log(soft_sum)
    loss = alpha * temp * temp * (p * (log_p - log_q)).sum(1)
    labels = s["labels"]
    if labels is not None:
        keep = labels >= 0
        label = labels.long().clamp(min=0)[:, None]
        hard = torch.exp(z - top)
        hard_sum = hard.sum(1, keepdim=True)
        loss = loss + (1 - alpha) * (torch.log(hard_sum) - (z.gather(1, label) - top))[:, 0]
        loss = torch.where(keep, loss, torch.zeros_like(loss))
    if c["op"] == "loss":
        return loss
    grad = soft * (alpha * temp * some / soft_sum)
    grad.scatter_add_(1, at, p * (-alpha * temp))
    if labels is not None:
        grad += hard * ((1 - alpha) / hard_sum)
        grad.scatter_add_(1, label, torch.full_like(label, alpha - 1, dtype=torch.float32))
        grad = torch.where(keep[:, None], grad, torch.zeros_like(grad))
    grad = (grad * (s["dy"] * c["grad_scale"])[:, None]).to(TYPES[c["dtype"]])
    return grad if c["op"] == "dpred" else (loss, grad)


def exact(case, seed):
    """The definitions, in 64 bits."""
    s, c = prepare(case, seed), case
    if c["op"] == "lookup":
        return torch.index_select(s["x"], 0, s["indices"].long()).double() * c["scale"]
    if c["op"] == "gradient":
        # every row of the table: the sum over the tokens that name it, as differences of running sums
        order = torch.sort(s["indices"].long(), stable=True)
        running = torch.cat([torch.zeros(1, c["h"], dtype=torch.float64, device="cuda"),
                             s["dy"].double()[order.indices].cumsum(0)])
        rows = torch.arange(c["v"], device="cuda")
        ends = torch.searchsorted(order.values, rows, right=True)
        result = (running[ends] - running[torch.searchsorted(order.values, rows)]) * c["scale"]
        if c["padding"] >= 0:
            result[c["padding"]] = 0
        return result + s["dx"].double() if c["accumulate"] else result
    parts = [_exact_rows(s, c, rows) for rows in torch.arange(c["n"], device="cuda").split(1024)]
    loss = torch.cat([part[0] for part in parts])
    if c["op"] == "loss":
        return loss
    grad = torch.cat([part[1] for part in parts])
    return grad if c["op"] == "dpred" else (loss, grad)


def _exact_rows(s, c, rows):
    temp, alpha = c["temperature"], c["alpha"]
    z = s["pred"][rows].double()
    ids = s["teacher_ids"][rows].long()
    t = s["teacher_logits"][rows].double() / temp
    t[ids < 0] = -math.inf
    p_top = torch.nan_to_num(torch.softmax(t, 1))  # a row without a teacher: zeros
    log_p = torch.where(p_top > 0, torch.log_softmax(t, 1), torch.zeros_like(t))
    p = torch.zeros_like(z).scatter_add_(1, ids.clamp(min=0), torch.where(ids < 0, torch.zeros_like(p_top), p_top))
    log_q = torch.log_softmax(z / temp, 1)
    loss = alpha * temp ** 2 * ((p_top * log_p).sum(1) - (p * log_q).sum(1))
    grad = alpha * temp * (log_q.exp() * p.sum(1, keepdim=True) - p)
    if s["labels"] is not None:
        labels = s["labels"][rows].long()
        log_r = torch.log_softmax(z, 1)
        onehot = torch.zeros_like(z).scatter_(1, labels.clamp(min=0)[:, None], 1.0)
        loss = (loss - (1 - alpha) * (onehot * log_r).sum(1)) * (labels != IGNORE)
        grad = (grad + (1 - alpha) * (log_r.exp() - onehot)) * (labels != IGNORE)[:, None]
    return loss, grad * (s["dy"][rows].double() * c["grad_scale"])[:, None]


def work(case):
    c = case
    size = {"float32": 4, "float16": 2, "bfloat16": 2, "int32": 4, "int64": 8}
    n, v = c["n"], c["v"]
    if c["op"] in ("lookup", "gradient"):
        h = c["h"]
        distinct = min(n, v, math.ceil(_distinct(n, v)))  # rows of the table that this many tokens name
        if c["op"] == "lookup":
            return {"bytes": distinct * h * size[c["dtype"]] + n * h * size[c["out"]] + n * size[c["ids"]], "flops": n * h}
        table = 2 * distinct if c["accumulate"] else v
        return {"bytes": n * h * size[c["dtype"]] + table * h * size[c["out"]] + n * size[c["ids"]], "flops": n * h + distinct * h}
    passes = 1 if c["op"] == "loss" else 2
    exps = 2 if c["labels"] and c["temperature"] != 1.0 else 1
    rows = n * (c["k"] * (size[c["dtype"]] + size[c["ids"]]) + 8 + (size[c["ids"]] if c["labels"] else 0))
    return {"bytes": n * v * size[c["dtype"]] * passes + rows, "flops": n * v * (3 * exps + 1) * passes}


def _distinct(n, v):
    """Expected number of different ids among n tokens of _tokens()."""
    p = [(math.log(r + 2.0) - math.log(r + 1.0)) / math.log(v + 1.0) for r in range(v)]
    return sum(-math.expm1(n * math.log1p(-min(q, 1 - 1e-12))) for q in p)
