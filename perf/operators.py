"""Cases, plain forms and 64-bit values of the vocabulary operators: the token embedding with its
gradient, and the distillation loss against a teacher's top logits with its gradient.

    embedding      y[t]  = scale * x[ids[t] - first_row], a row of zeros for an id outside the table
    embedding_dx   dx[r] = scale * sum of dy[t] over the tokens t with ids[t] - first_row == r, added to a
                   gradient that is there already if one is given; tokens of the padding id have no part
    topk_distill   loss  = soft * T^2 * KL(p || softmax(z / T)) + hard * CE(label, softmax(z)), where p is
                   the softmax of the teacher's top logits over T; a negative index is an absent entry
    topk_distill_dx, topk_distill_step    d loss / d z, the second together with the loss
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4, "i64": 8}
_IDS = {"i32": torch.int32, "i64": torch.int64}


def _embedding(name, vocab, width, batch, length, table="bf16", out="bf16", ids="i64", scale=1.0, shards=1, pad=0.0):
    return {"name": name, "kind": "embedding", "vocab": vocab, "width": width, "batch": batch, "length": length,
            "table": table, "out": out, "ids": ids, "scale": scale, "shards": shards, "pad": pad}


def _embedding_dx(name, vocab, width, batch, length, dy="bf16", out="f32", ids="i64", scale=1.0, shards=1, pad=0.0,
                  accumulate=False):
    return {"name": name, "kind": "embedding_dx", "vocab": vocab, "width": width, "batch": batch, "length": length,
            "dy": dy, "out": out, "ids": ids, "scale": scale, "shards": shards, "pad": pad, "accumulate": accumulate}


def _distill(name, what, rows, vocab, topk, logits="bf16", teacher="f32", ids="i64", temperature=1.0, hard=0.0,
             padded=0, masked=0.0, short=0.0):
    return {"name": name, "kind": what, "rows": rows, "vocab": vocab, "topk": topk, "logits": logits, "teacher": teacher,
            "ids": ids, "temperature": temperature, "hard": hard, "padded": padded, "masked": masked, "short": short}


def listed():
    return [
        # one new token for each of eight sequences, a GPT-2 1.5B table: launch and call latency
        _embedding("embedding_decode", 50257, 1600, 8, 1, scale=40.0),
        # a training batch of BERT-large over its fp32 master table, narrowed to the model's type
        _embedding("embedding_batch", 30522, 1024, 64, 512, table="f32", out="bf16", ids="i32", scale=32.0, pad=0.2),
        # one short sequence into the gradient that a tied output projection has left already
        _embedding_dx("embedding_dx_short", 30522, 768, 1, 37, out="f32", accumulate=True),
        # an odd batch on one of two vocabulary shards, fp32 throughout, a width with no wide accesses
        _embedding_dx("embedding_dx_shard", 50257, 513, 3, 1001, dy="f32", out="f32", ids="i32", scale=22.5, shards=2),
        # the batch of BERT-large, a quarter of it padding, into the fp32 gradient that the optimizer reads
        _embedding_dx("embedding_dx_batch", 30522, 1024, 32, 512, pad=0.25),
        # a long batch of GPT-2 1.5B into a 16-bit gradient
        _embedding_dx("embedding_dx_long", 50257, 1600, 64, 1024, out="bf16", scale=40.0),
        # a few rows: one has to be spread over the GPU
        _distill("distill_few", "distill", 3, 50257, 10, logits="f32", temperature=2.0),
        # the masked positions of a BERT batch, some without a target
        _distill("distill_masked", "distill", 4913, 30522, 32, temperature=2.0, masked=0.1, short=0.2),
        # a short sequence with labels, the vocabulary padded to a multiple of 64
        _distill("distill_dx_short", "distill_dx", 129, 50257, 16, logits="f16", teacher="f16", temperature=2.0, hard=0.1, padded=47),
        # a GPT-2 batch with unpadded rows, so that no two start alike in a 16-byte word
        _distill("distill_dx_batch", "distill_dx", 4096, 50257, 64, teacher="bf16", ids="i32", temperature=1.5, masked=0.05),
        # a fine-tuning micro-batch in fp32, loss and gradient at once
        _distill("distill_step_small", "distill_step", 64, 30522, 100, logits="f32", temperature=4.0, hard=0.5, short=0.1),
        # the large batch of a GPT-2 student, loss and gradient at once
        _distill("distill_step_batch", "distill_step", 8192, 50257, 64, teacher="f16", temperature=2.0, hard=0.25, padded=47, masked=0.05),
    ]


def _log_size(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["embedding", "embedding_dx", "embedding_dx", "distill", "distill_dx", "distill_step"])
    most = 1.5e9  # bytes: under the largest listed case of either family
    if kind.startswith("embedding"):
        most = 3e8
        while True:
            width = rng.choice([_log_size(rng, 48, 4096), 64 * _log_size(rng, 1, 64)])
            batch = rng.randint(1, 64)
            c = dict(_embedding("", _log_size(rng, 900, 200000), width, batch, _log_size(rng, 1, 2048),
                                table=rng.choice(list(_TYPES)), out=rng.choice(list(_TYPES)), ids=rng.choice(list(_IDS)),
                                scale=rng.choice([1.0, math.sqrt(width), 0.5]), shards=rng.choice([1, 1, 1, 2, 4]),
                                pad=rng.choice([0.0, 0.0, 0.3, 0.6])))
            if kind == "embedding_dx":
                c["dy"] = c.pop("table")
                c["accumulate"] = rng.random() < 0.4
                c["kind"] = kind
            del c["name"]
            if work(c)["bytes"] <= most:
                return c
    while True:
        c = _distill("", kind, _log_size(rng, 1, 16384), _log_size(rng, 2000, 160000), _log_size(rng, 1, 256),
                     logits=rng.choice(list(_TYPES)), teacher=rng.choice(list(_TYPES)), ids=rng.choice(list(_IDS)),
                     temperature=rng.choice([1.0, 1.0, 2.0, 3.5]), hard=rng.choice([0.0, 0.0, 0.3]),
                     padded=rng.choice([0, 0, rng.randint(1, 127)]), masked=rng.choice([0.0, 0.1, 0.4]),
                     short=rng.choice([0.0, 0.2]))
        del c["name"]
        if work(c)["bytes"] <= most:
            return c


# ------------------------------------------------------------------------------------------- inputs
def _tokens(case, gen):
    """Token ids as text has them: frequency falls with the rank (log-uniform) and ranks are ids,
    counted from the other end where the vocabulary is sharded, since the last shard is the one that
    is looked at; the end of each sequence is padding (id 0)."""
    b, s, v = case["batch"], case["length"], case["vocab"]
    u = torch.rand((b, s), device="cuda", generator=gen, dtype=torch.float64)
    ids = (torch.exp(u * math.log(v)).to(torch.int64) - 1).clamp_(0, v - 1)
    if case["shards"] > 1:
        ids = v - 1 - ids
    if case["pad"] > 0:
        used = torch.rand((b, 1), device="cuda", generator=gen) * 2 * case["pad"]
        at = torch.arange(s, device="cuda")[None, :]
        ids = torch.where(at < (s * (1 - used)).ceil(), ids, torch.zeros_like(ids))
    return ids.to(_IDS[case["ids"]])


def _shard(case):
    """(rows, first row) of the last vocabulary shard, the one that may be smaller than the others."""
    per = -(-case["vocab"] // case["shards"])
    first = per * (case["shards"] - 1)
    return case["vocab"] - first, first


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, to="f32", std=1.0):
        return torch.randn(shape, device="cuda", generator=gen).mul_(std).to(_TYPES[to])

    s = {"case": case}
    if case["kind"].startswith("embedding"):
        rows, first = _shard(case)
        s.update(ids=_tokens(case, gen), rows=rows, first=first, padding=0 if case["pad"] > 0 else None)
        if case["kind"] == "embedding":
            s["table"] = normal(rows, case["width"], to=case["table"], std=0.02)
        else:
            s["dy"] = normal(case["batch"], case["length"], case["width"], to=case["dy"], std=0.01)
            s["grad"] = normal(rows, case["width"], to=case["out"], std=0.01) if case["accumulate"] else None
        return s
    n, v, k = case["rows"], case["vocab"], case["topk"]
    start = torch.randint(0, v, (n, 1), device="cuda", generator=gen)
    index = (start + torch.arange(k, device="cuda")[None, :] * max(v // k, 1)) % v  # distinct
    teacher = torch.sort(normal(n, k, std=2.0) + 8.0, dim=1, descending=True).values
    logits = normal(n, v + case["padded"], std=2.0)
    logits.scatter_(1, index, teacher + normal(n, k, std=0.7))  # the student has learned some of it
    logits = logits.to(_TYPES[case["logits"]])
    label = torch.where(torch.rand(n, device="cuda", generator=gen) < 0.7, index[:, 0],
                        torch.randint(0, v, (n,), device="cuda", generator=gen))
    if case["short"] > 0:  # a teacher cut by probability leaves fewer than k entries
        kept = (k * (1 - case["short"] * 2 * torch.rand((n, 1), device="cuda", generator=gen))).ceil()
        index = torch.where(torch.arange(k, device="cuda")[None, :] < kept, index, torch.full_like(index, -1))
    if case["masked"] > 0:  # rows without a target
        off = torch.rand(n, device="cuda", generator=gen) < case["masked"]
        index = torch.where(off[:, None], torch.full_like(index, -1), index)
        label = torch.where(off, torch.full_like(label, -100), label)
    # a mean over the rows, or for fp16 a sum times a loss scale, without which most gradients would vanish
    weight = 16.0 if case["logits"] == "f16" else 2.0 / n
    s.update(logits=logits, index=index.to(_IDS[case["ids"]]), teacher=teacher.to(_TYPES[case["teacher"]]),
             labels=label.to(_IDS[case["ids"]]) if case["hard"] > 0 else None,
             dloss=torch.rand(n, device="cuda", generator=gen) * weight)
    if case["kind"] == "distill_dx":  # the forward pass has left the softmax statistics behind
        s["stats"] = _plain_stats(s)
    return s


# ------------------------------------------------------------------------------------- plain forms
def _plain_embedding(s):
    c, x = s["case"], s["table"]
    local = s["ids"].long() - s["first"]
    inside = (local >= 0) & (local < s["rows"])
    y = x[torch.where(inside, local, torch.zeros_like(local))].float() * c["scale"]
    return torch.where(inside[..., None], y, torch.zeros_like(y)).to(_TYPES[c["out"]])


def _plain_embedding_dx(s):
    c = s["case"]
    ids = s["ids"].long().reshape(-1)
    keep = (ids >= s["first"]) & (ids < s["first"] + s["rows"])
    if s["padding"] is not None:
        keep &= ids != s["padding"]
    dy = s["dy"].reshape(-1, c["width"])[keep].float()
    dx = torch.zeros((s["rows"], c["width"]), device=dy.device).index_add_(0, ids[keep] - s["first"], dy) * c["scale"]
    if s["grad"] is None:
        return dx.to(_TYPES[c["out"]])
    return s["grad"].copy_(s["grad"].float() + dx)


def _present(s):
    """Per teacher entry whether it is there, per row whether any is, per row whether it has a label."""
    there = (s["index"] >= 0) & (s["index"] < s["case"]["vocab"])
    labelled = torch.zeros_like(there[:, 0])
    if s["labels"] is not None:
        labelled = (s["labels"] >= 0) & (s["labels"] < s["case"]["vocab"])
    return there, there.any(1), labelled


def _plain_stats(s):
    """[rows, 3]: the largest logit m, log sum exp((z - m) / T) for the rows with a teacher and
    log sum exp(z - m) for the rows with a label, zero where a row has no use for it."""
    c = s["case"]
    _, soft, labelled = _present(s)
    z = s["logits"][:, :c["vocab"]].float()
    m = z.max(dim=1).values
    none = torch.zeros_like(m)
    d = z - m[:, None]
    first = torch.where(soft, (d / c["temperature"]).exp().sum(dim=1).log(), none)
    second = torch.where(labelled, d.exp().sum(dim=1).log(), none) if c["hard"] > 0 else none
    return torch.stack([torch.where(soft | labelled, m, none), first, second], dim=1)


def _plain_teacher(s):
    """p of every entry, zero where it is absent, and log p there."""
    there, soft, _ = _present(s)
    t = torch.where(there, s["teacher"].float() / s["case"]["temperature"], torch.full((), -math.inf, device="cuda"))
    top = torch.where(soft, t.max(dim=1).values, torch.zeros_like(t[:, 0]))[:, None]
    total = (t - top).exp().sum(dim=1, keepdim=True)
    logp = torch.where(there, t - top - torch.where(total > 0, total, torch.ones_like(total)).log(), torch.zeros_like(t))
    return torch.where(there, logp.exp(), torch.zeros_like(logp)), logp


def _plain_loss(s, stats):
    c = s["case"]
    there, soft, labelled = _present(s)
    p, logp = _plain_teacher(s)
    at = torch.where(there, s["index"].long(), torch.zeros_like(s["index"], dtype=torch.int64))
    logq = (s["logits"].gather(1, at).float() - stats[:, :1]) / c["temperature"] - stats[:, 1:2]
    loss = (p * (logp - logq)).sum(dim=1) * c["temperature"] ** 2
    if c["hard"] > 0:
        at = torch.where(labelled, s["labels"].long(), torch.zeros_like(s["labels"], dtype=torch.int64))
        ce = stats[:, 2] - (s["logits"].gather(1, at[:, None]).float().squeeze(1) - stats[:, 0])
        loss = loss + torch.where(labelled, ce, torch.zeros_like(ce)) * c["hard"]
    return loss


def _plain_dlogits(s, stats):
    c = s["case"]
    there, soft, labelled = _present(s)
    p, _ = _plain_teacher(s)
    z = s["logits"][:, :c["vocab"]].float() - stats[:, :1]
    a = (s["dloss"] * c["temperature"])[:, None]
    d = torch.zeros(s["logits"].shape, device=z.device)
    inner = d[:, :c["vocab"]]
    inner += (z / c["temperature"] - stats[:, 1:2]).exp() * torch.where(soft[:, None], a, torch.zeros_like(a))
    d.scatter_add_(1, torch.where(there, s["index"].long(), torch.zeros_like(s["index"], dtype=torch.int64)), -p * a)
    if c["hard"] > 0:
        h = torch.where(labelled, s["dloss"] * c["hard"], torch.zeros_like(s["dloss"]))[:, None]
        inner += (z - stats[:, 2:]).exp() * h
        d.scatter_add_(1, torch.where(labelled, s["labels"].long(), torch.zeros_like(s["labels"], dtype=torch.int64))[:, None], -h)
    return d.to(s["logits"].dtype)


def run(s):
    c = s["case"]
    if own:
        return _own(s)
    if c["kind"] == "embedding":
        return _plain_embedding(s)
    if c["kind"] == "embedding_dx":
        return _plain_embedding_dx(s)
    stats = s["stats"] if c["kind"] == "distill_dx" else _plain_stats(s)
    if c["kind"] == "distill":
        return {"loss": _plain_loss(s, stats), "stats": stats}
    if c["kind"] == "distill_dx":
        return _plain_dlogits(s, stats)
    return {"loss": _plain_loss(s, stats), "dlogits": _plain_dlogits(s, stats)}


def _own(s):
    from raf_amd import op

    c = s["case"]
    if c["kind"] == "embedding":
        return op.embedding(s["table"], s["ids"], scale=c["scale"], first_row=s["first"], out_dtype=_TYPES[c["out"]])
    if c["kind"] == "embedding_dx":
        return op.embedding_dx(s["dy"], s["ids"], s["rows"], scale=c["scale"], padding_idx=s["padding"], first_row=s["first"],
                               out_dtype=_TYPES[c["out"]], grad=s["grad"])
    more = dict(temperature=c["temperature"], labels=s["labels"], hard_weight=c["hard"], vocab_size=c["vocab"])
    if c["kind"] == "distill":
        loss, stats = op.topk_distill(s["logits"], s["index"], s["teacher"], **more)
        return {"loss": loss, "stats": stats}
    if c["kind"] == "distill_dx":
        return op.topk_distill_dx(s["dloss"], s["logits"], s["index"], s["teacher"], s["stats"], **more)
    loss, dlogits = op.topk_distill_step(s["logits"], s["index"], s["teacher"], s["dloss"], **more)
    return {"loss": loss, "dlogits": dlogits}


# -------------------------------------------------------------------------------------------- work
def _distinct(vocab, tokens):
    """Expected number of distinct ids among that many tokens of _tokens' distribution."""
    r = np.arange(1, vocab + 1, dtype=np.float64)
    p = np.log1p(1 / r) / math.log(vocab)
    return float(-np.expm1(tokens * np.log1p(-np.minimum(p, 1 - 1e-12))).sum())


def work(case):
    if case["kind"].startswith("embedding"):
        rows, _ = _shard(case)
        n, w = case["batch"] * case["length"], case["width"]
        live = n * (1 - case["pad"])
        inside = min(1.0, math.log(rows + 1) / math.log(case["vocab"]))
        touched = min(rows, _distinct(case["vocab"], live) * inside)
        ids = n * _BYTES[case["ids"]]
        if case["kind"] == "embedding":
            return {"bytes": ids + touched * w * _BYTES[case["table"]] + n * w * _BYTES[case["out"]], "flops": n * w}
        # the gradient is written whole, or read and written where tokens fall if it is added to
        out = (2 * touched if case["accumulate"] else rows) * w * _BYTES[case["out"]]
        return {"bytes": ids + live * inside * w * _BYTES[case["dy"]] + out, "flops": live * inside * w}
    n, v, k = case["rows"], case["vocab"], case["topk"]
    live = n * (1 - case["masked"])
    targets = n * (k * (_BYTES[case["ids"]] + _BYTES[case["teacher"]]) + (_BYTES[case["ids"]] if case["hard"] > 0 else 0) + 4)
    read = live * v * _BYTES[case["logits"]]
    write = 0 if case["kind"] == "distill" else n * (v + case["padded"]) * _BYTES[case["logits"]]
    sums = 2 if case["hard"] > 0 and case["temperature"] != 1.0 else 1
    passes = 2 if case["kind"] == "distill_step" else 1
    return {"bytes": targets + read + write + n * (16 if case["kind"] == "distill" else 4), "flops": live * v * 3 * sums * passes}


# ------------------------------------------------------------------------------------------- exact
def _exact_target(s):
    """p as a dense row over the vocabulary, and each row's teacher and label weights, in 64 bits."""
    c = s["case"]
    n, v = c["rows"], c["vocab"]
    index = s["index"].long()
    there = (index >= 0) & (index < v)
    t = (s["teacher"].double() / c["temperature"]).masked_fill(~there, -math.inf)
    some = there.any(1)
    p = torch.softmax(t.masked_fill(~some[:, None], 0.0), dim=1).masked_fill(~there, 0.0)
    label = s["labels"].long() if s["labels"] is not None else torch.full((n,), -1, device="cuda")
    return p, index.clamp(0, v - 1), some.double(), label.clamp(0, v - 1), ((label >= 0) & (label < v)).double()


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["kind"].startswith("embedding"):
        local = s["ids"].long() - s["first"]
        inside = ((local >= 0) & (local < s["rows"])).double()
        local = local.clamp(0, s["rows"] - 1)
        if c["kind"] == "embedding":
            return torch.nn.functional.embedding(local, s["table"].double()) * (inside * c["scale"])[..., None]
        if s["padding"] is not None:
            inside = inside * (s["ids"] != s["padding"])
        order = torch.argsort(local.reshape(-1), stable=True)
        weighted = (s["dy"].double() * (inside * c["scale"])[..., None]).reshape(-1, c["width"])[order]
        runs, counts = torch.unique_consecutive(local.reshape(-1)[order], return_counts=True)
        dx = s["grad"].double() if s["grad"] is not None else torch.zeros((s["rows"], c["width"]), device="cuda", dtype=torch.float64)
        dx[runs] += torch.segment_reduce(weighted, "sum", lengths=counts, axis=0, unsafe=True)
        return dx
    t, v = c["temperature"], c["vocab"]
    p, index, some, label, labelled = _exact_target(s)
    loss, stats, grads = [], [], []
    for at in range(0, c["rows"], 1024):  # 64 bits of everything at once would not leave room for the rest
        cut = slice(at, at + 1024)
        z = s["logits"][cut, :v].double()
        logq, logq1 = torch.log_softmax(z / t, dim=1), torch.log_softmax(z, dim=1)
        pi, ii, li = p[cut], index[cut], label[cut][:, None]
        kl = (torch.xlogy(pi, pi) - pi * logq.gather(1, ii)).sum(1)
        loss.append(t * t * kl - c["hard"] * labelled[cut] * logq1.gather(1, li).squeeze(1))
        m = z.amax(1)
        hard = labelled[cut] * (1.0 if c["hard"] > 0 else 0.0)
        stats.append(torch.stack([m * torch.maximum(some[cut], hard), (torch.logsumexp(z / t, 1) - m / t) * some[cut],
                                  (torch.logsumexp(z, 1) - m) * hard], 1))
        if c["kind"] == "distill":
            continue
        g = logq.exp_().mul_(t * some[cut][:, None]).scatter_add_(1, ii, -t * pi)
        g += logq1.exp_().scatter_add_(1, li, torch.full_like(li, -1, dtype=torch.float64)).mul_(c["hard"] * labelled[cut][:, None])
        g *= s["dloss"][cut].double()[:, None]
        grads.append(torch.nn.functional.pad(g, (0, c["padded"])))
        del z, logq, logq1, g
    if c["kind"] == "distill":
        return {"loss": torch.cat(loss), "stats": torch.cat(stats)}
    if c["kind"] == "distill_dx":
        return torch.cat(grads)
    return {"loss": torch.cat(loss), "dlogits": torch.cat(grads)}
