"""Workloads of the vocabulary-row operators: token scores (log probability of a given token,
entropy, top alternatives) with their gradient, and distillation from a teacher's top entries
with its gradient. Every case works on a [rows, vocab] matrix of logits that lives on the GPU.

`run` computes a case with elementary torch operations, or, when `own` is set, through
`see_ml_b200.token_ops`.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _case(name, kind, rows, vocab, dtype, k=0, pad=0, temperature=1.0, masked=0.0, tail=False, teacher="f32"):
    return {"name": name, "kind": kind, "rows": rows, "vocab": vocab, "dtype": dtype, "k": k, "pad": pad,
            "temperature": temperature, "masked": masked, "tail": tail, "teacher": teacher}


def listed():
    return [
        # one generated token: its log probability and the alternatives shown beside it
        _case("scores_one_token", "scores", 1, 32000, "f32", k=8, temperature=0.7),
        # a decoding batch under a grammar that masks a part of the vocabulary
        _case("scores_decode_batch", "scores", 48, 131072, "bf16", k=20, temperature=0.8, masked=0.3),
        # the 16384-row chunk of the 32000-token decoder that bench.py trains, scored in the plan's f32
        _case("scores_chunk", "scores", 16384, 32000, "f32", k=16),
        # a teacher's pass that keeps the top 64 of a large vocabulary
        _case("scores_teacher", "scores", 2048, 131072, "bf16", k=64),
        # an odd vocabulary in rows of an odd stride
        _case("scores_odd", "scores", 777, 50001, "f16", k=5, pad=7),
        # a policy gradient with an entropy term on half a chunk
        _case("scores_grad_chunk", "scores_grad", 8192, 32000, "f32"),
        # the same in 16 bits, odd in both sizes
        _case("scores_grad_odd", "scores_grad", 1001, 100003, "bf16", temperature=1.3),
        # a training step of the chunk against a stored teacher of 32 entries and their tail
        _case("distill_step_chunk", "distill_step", 16384, 32000, "f32", k=32, temperature=2.0, tail=True),
        # a training step in 16 bits over a large vocabulary, the teacher renormalised over its 64 entries
        _case("distill_step_large", "distill_step", 2048, 131072, "bf16", k=64, teacher="bf16"),
        # a step of a few tokens, where launches are what it costs
        _case("distill_step_small", "distill_step", 8, 5000, "f32", k=10, temperature=1.5),
        # the loss alone on a validation batch
        _case("distill_eval_odd", "distill", 513, 50001, "f16", k=17, tail=True),
        # the backward pass on its own, behind a loss that weighs its rows elsewhere
        _case("distill_grad", "distill_grad", 4096, 65537, "bf16", k=128, tail=True),
    ]


def draw(rng):
    kind = rng.choice(["scores", "scores", "scores_grad", "distill_step", "distill_step", "distill", "distill_grad"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    vocab = int(round(math.exp(rng.uniform(math.log(300), math.log(140000)))))
    rows = int(round(math.exp(rng.uniform(0.0, math.log(min(20000.0, 2.0 ** 27 / vocab))))))
    k = int(round(math.exp(rng.uniform(0.0, math.log(128)))))
    if kind == "scores_grad" or (kind == "scores" and rng.random() < 0.2):
        k = 0
    return {"kind": kind, "rows": max(1, rows), "vocab": vocab, "dtype": dtype, "k": k, "pad": rng.choice([0, 0, 0, 1, 8, 13]),
            "temperature": rng.choice([0.5, 1.0, 1.0, 2.0, 3.0]),
            "masked": rng.choice([0.0, 0.5]) if kind == "scores" else 0.0, "tail": rng.random() < 0.5,
            "teacher": rng.choice(["f32", "bf16", "f16"])}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, vocab, k, dtype = case["rows"], case["vocab"], case["k"], DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    # a trained model's logits: a broad normal body and a handful of likely tokens above it
    buf = torch.empty((rows, vocab + case["pad"]), dtype=dtype, device="cuda")
    logits = buf[:, :vocab]
    step = max(1, (1 << 28) // vocab)
    likely = torch.randint(vocab, (rows, 6), generator=g, device="cuda")
    for r in range(0, rows, step):
        n = min(step, rows - r)
        x = normal(n, vocab).mul_(2.0)
        x.scatter_add_(1, likely[r:r + n], normal(n, 6).mul_(2.0).add_(6.0))
        if case["masked"]:
            x.masked_fill_(torch.rand((n, vocab), generator=g, device="cuda") < case["masked"], -math.inf)
        logits[r:r + n] = x
        del x
    state = {"case": case, "logits": logits}
    if case["kind"].startswith("scores"):
        labels = likely[:, 0].to(torch.int32)
        labels[torch.rand(rows, generator=g, device="cuda") < 0.05] = -1          # rows without a token
        state["labels"] = labels
    if case["kind"] == "scores_grad":
        state["dlogprob"] = normal(rows).div_(rows)
        state["dentropy"] = torch.full((rows,), -0.01 / rows, device="cuda")
        stats = torch.empty((rows, 2), device="cuda")
        entropy = torch.empty(rows, device="cuda")
        for r in range(0, rows, step):
            x = logits[r:r + step].float()
            top = x.amax(1)
            y = (x - top[:, None]) / case["temperature"]
            e = torch.exp(y)
            total = e.sum(1)
            stats[r:r + step, 0], stats[r:r + step, 1] = top, total
            entropy[r:r + step] = torch.log(total) - (e * y).sum(1) / total
            del x, y, e
        state["stats"], state["entropy"] = stats, entropy
    if case["kind"].startswith("distill"):
        # the teacher's entries: distinct tokens with falling log probabilities that hold most of the
        # mass; short lists end in entries of id -1
        first = torch.randint(vocab, (rows, 1), generator=g, device="cuda")
        ids = (first + torch.arange(k, device="cuda") * (vocab // k)) % vocab
        v = normal(rows, k).mul_(1.5).sort(1, descending=True).values
        v = torch.log_softmax(v, 1) + math.log(0.93)
        # the student has learned a part of it: most of its mass lies on the same tokens
        t = case["temperature"]
        learned = t * (v + normal(rows, k).mul_(0.5) + math.log(vocab) + 2.0 / t ** 2 + 1.5)
        logits.scatter_(1, ids, learned.to(dtype))
        short = torch.randint(1, k + 1, (rows, 1), generator=g, device="cuda")
        short = torch.where(torch.rand((rows, 1), generator=g, device="cuda") < 0.1, short, k)
        ids = torch.where(torch.arange(k, device="cuda") < short, ids, -1)
        state["teacher_id"] = ids.to(torch.int32).contiguous()
        state["teacher_logprob"] = v.to(DTYPES[case["teacher"]]).contiguous()
        weight = torch.ones(rows, device="cuda")
        weight[torch.rand(rows, generator=g, device="cuda") < 0.1] = 0.0           # padded rows
        state["weight"] = weight
    if case["kind"] == "distill_grad":
        state["drow_loss"] = weight / rows
        saved = torch.empty((rows, 4), device="cuda")
        for r in range(0, rows, step):
            x = logits[r:r + step].float()
            top = x.amax(1)
            total = torch.exp((x - top[:, None]) / case["temperature"]).sum(1)
            i = state["teacher_id"][r:r + step].long()
            wide = torch.cat([x, torch.zeros_like(x[:, :1])], 1)
            wide.scatter_(1, torch.where(i < 0, vocab, i), -math.inf)
            rest = wide[:, :vocab]
            rest_top = rest.amax(1)
            rest_total = torch.exp((rest - rest_top[:, None]) / case["temperature"]).sum(1)
            saved[r:r + step] = torch.stack([rest_top, rest_total, top, total], 1)
            del x, wide, rest
        state["saved"] = saved
    return state


def _softmax(x, temperature):
    """(x - max) / T, its exponentials and their sum, of each row."""
    y = (x - x.amax(1, keepdim=True)) / temperature
    e = torch.exp(y)
    return y, e, e.sum(1, keepdim=True)


def _plain_scores(s):
    case, logits, labels = s["case"], s["logits"], s["labels"]
    y, e, total = _softmax(logits.float(), case["temperature"])
    logsum = torch.log(total)
    picked = y.gather(1, labels.clamp(min=0).long()[:, None]) - logsum
    out = {"logprob": torch.where(labels < 0, 0.0, picked[:, 0]),
           "entropy": (logsum - torch.where(e > 0, e * y, 0.0).sum(1, keepdim=True) / total)[:, 0]}
    if case["k"]:
        k = min(case["k"], case["vocab"])
        ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
        out["top_logprob"] = y.gather(1, ids) - logsum
        out["top_id"] = ids.to(torch.int32)
    return out


def _plain_scores_grad(s):
    logits, labels, t = s["logits"], s["labels"], s["case"]["temperature"]
    y = (logits.float() - s["stats"][:, :1]) / t
    p = torch.exp(y) / s["stats"][:, 1:]
    logp = y - torch.log(s["stats"][:, 1:])
    there = labels >= 0
    gl = torch.where(there, s["dlogprob"], 0.0)[:, None]
    d = -gl * p - s["dentropy"][:, None] * p * (logp + s["entropy"][:, None])
    d.scatter_add_(1, labels.clamp(min=0).long()[:, None], gl)
    return {"dlogits": (d / t).to(logits.dtype)}


def _teacher(s):
    """Present entries, their probabilities (64 bits), the tail's, and the columns that the entries name."""
    ids, v = s["teacher_id"].long(), s["teacher_logprob"].double()
    present = ids >= 0
    v = torch.where(present, v, -math.inf)
    if s["case"]["tail"]:
        q = torch.exp(v)
        rest = (1.0 - q.sum(1, keepdim=True)).clamp(min=0.0)
    else:
        q = torch.softmax(v, 1)
        rest = torch.zeros_like(q[:, :1])
    return ids, present, q, rest


def _members(ids, present, rows, vocab):
    member = torch.zeros((rows, vocab + 1), dtype=torch.bool, device=ids.device)
    member.scatter_(1, torch.where(present, ids, vocab), True)
    return member[:, :vocab]


def _plain_distill(s, gradient, upstream=None):
    case, logits = s["case"], s["logits"]
    rows, vocab, t = case["rows"], case["vocab"], case["temperature"]
    ids, present, q, rest = _teacher(s)
    member = _members(ids, present, rows, vocab)
    y, e, total = _softmax(logits.float(), t)
    rest_sum = torch.where(member, 0.0, e).sum(1, keepdim=True)
    out = {}
    if upstream is None:
        logsum = torch.log(total.double())
        lp = y.gather(1, ids.clamp(min=0)).double() - logsum
        terms = torch.where(q > 0, q * (torch.log(q) - lp), 0.0).sum(1)
        far = rest * (torch.log(rest) - torch.log(rest_sum.double()) + logsum)
        row_loss = terms + torch.where((rest > 0) & (rest_sum > 0), far, 0.0)[:, 0]
        row_loss = torch.where(s["weight"] == 0, 0.0, row_loss)
        scale = 1.0 / rows
        out["loss"] = ((row_loss * s["weight"].double()).sum() * scale).float()
        out["row_loss"] = row_loss.float()
        upstream = s["weight"] * scale
    if gradient:
        d = e / total * (q.sum(1, keepdim=True) + rest).float()
        share = torch.where(rest_sum > 0, (rest / rest_sum).float(), 0.0)
        d -= torch.where(member, 0.0, e * share)
        d.scatter_add_(1, ids.clamp(min=0), -q.float())
        d *= upstream[:, None] / t
        out["dlogits"] = d.to(logits.dtype)
    return out


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        from see_ml_b200 import token_ops
        t = case["temperature"]
        if kind == "scores":
            r = token_ops.token_scores(state["logits"], state["labels"], top_k=min(case["k"], case["vocab"]), temperature=t)
            out = {"logprob": r.logprob, "entropy": r.entropy}
            if case["k"]:
                out["top_logprob"], out["top_id"] = r.top_logprob, r.top_id
            return out
        if kind == "scores_grad":
            return {"dlogits": token_ops.token_scores_backward(
                state["logits"], state["labels"], state["stats"], state["entropy"], state["dlogprob"], state["dentropy"],
                temperature=t)}
        if kind == "distill_grad":
            return {"dlogits": token_ops.distill_topk_backward(
                state["logits"], state["teacher_id"], state["teacher_logprob"], state["saved"], state["drow_loss"],
                temperature=t, tail=case["tail"])}
        r = token_ops.distill_topk(state["logits"], state["teacher_id"], state["teacher_logprob"], row_weight=state["weight"],
                                   scale=1.0 / case["rows"], temperature=t, tail=case["tail"], grad=kind == "distill_step")
        out = {"loss": r.loss, "row_loss": r.row_loss}
        if kind == "distill_step":
            out["dlogits"] = r.dlogits
        return out
    if kind == "scores":
        return _plain_scores(state)
    if kind == "scores_grad":
        return _plain_scores_grad(state)
    if kind == "distill_grad":
        return _plain_distill(state, True, state["drow_loss"])
    return _plain_distill(state, kind == "distill_step")


def work(case):
    rows, n, k = case["rows"], case["rows"] * case["vocab"], case["k"]
    logits = n * BYTES[case["dtype"]]
    kind = case["kind"]
    entries = rows * k * (4 + BYTES[case["teacher"]])
    if kind == "scores":
        return {"bytes": logits + rows * 12 + rows * k * 8, "flops": 6 * n}
    if kind == "scores_grad":
        return {"bytes": 2 * logits + rows * 24, "flops": 6 * n}
    if kind == "distill":
        return {"bytes": logits + entries + rows * 8, "flops": 4 * n}
    return {"bytes": 2 * logits + entries + rows * (20 if kind == "distill_grad" else 8), "flops": 6 * n}


def exact(case, seed):
    s = prepare(case, seed)
    rows, vocab, t, kind = case["rows"], case["vocab"], case["temperature"], case["kind"]
    parts, step = [], max(1, (1 << 26) // vocab)
    for r in range(0, rows, step):
        x = s["logits"][r:r + step].double() / t
        n = x.shape[0]
        lse = torch.logsumexp(x, 1, keepdim=True)
        lp = x - lse
        p = lp.exp()
        every = torch.arange(n, device=x.device)
        part = {}
        if kind.startswith("scores"):
            lab = s["labels"][r:r + step].long()
            ent = -torch.special.xlogy(p, p).sum(1)
            if kind == "scores":
                part["logprob"] = torch.where(lab < 0, 0.0, lp[every, lab.clamp(min=0)])
                part["entropy"] = ent
                if case["k"]:
                    v, i = torch.sort(lp, dim=1, descending=True, stable=True)
                    part["top_logprob"], part["top_id"] = v[:, :case["k"]].clone(), i[:, :case["k"]].to(torch.int32)
                    del v, i
            else:
                gl = torch.where(lab < 0, 0.0, s["dlogprob"][r:r + step].double())
                d = p * (-gl - s["dentropy"][r:r + step].double() * ent)[:, None]
                d -= s["dentropy"][r:r + step].double()[:, None] * torch.special.xlogy(p, p)
                d[every, lab.clamp(min=0)] += gl
                part["dlogits"] = d / t
        else:
            ids = s["teacher_id"][r:r + step].long()
            v = s["teacher_logprob"][r:r + step].double()
            v = v.masked_fill(ids < 0, -math.inf)
            q = v.exp() if case["tail"] else torch.softmax(v, 1)
            target = torch.zeros((n, vocab + 1), dtype=torch.float64, device=x.device)
            target.scatter_add_(1, ids.masked_fill(ids < 0, vocab), q)
            named = torch.zeros((n, vocab + 1), dtype=torch.bool, device=x.device)
            named.scatter_(1, ids.masked_fill(ids < 0, vocab), True)
            target, named = target[:, :vocab], named[:, :vocab]
            q_rest = (1.0 - q.sum(1)).clamp(min=0.0) if case["tail"] else torch.zeros(n, dtype=torch.float64, device=x.device)
            lp_rest = torch.logsumexp(lp.masked_fill(named, -math.inf), 1)
            w = s["weight"][r:r + step].double()
            if kind != "distill_grad":
                terms = torch.special.xlogy(q, q) - q * lp.gather(1, ids.clamp(min=0)).masked_fill(ids < 0, 0.0)
                far = torch.where((q_rest > 0) & torch.isfinite(lp_rest), torch.special.xlogy(q_rest, q_rest) - q_rest * lp_rest, 0.0)
                part["row_loss"] = torch.where(w == 0, 0.0, terms.sum(1) + far)
            if kind != "distill":
                up = s["drow_loss"][r:r + step].double() if kind == "distill_grad" else w / rows
                rest = torch.where(torch.isfinite(lp_rest), q_rest, 0.0)[:, None] * torch.exp(lp - lp_rest[:, None]).masked_fill(named, 0.0)
                rest = torch.nan_to_num(rest)
                d = p * (q.sum(1) + q_rest)[:, None] - target - rest
                part["dlogits"] = d * (up / t)[:, None]
        parts.append(part)
    out = {name: torch.cat([part[name] for part in parts]) for name in parts[0]}
    if kind in ("distill", "distill_step"):
        out = {"loss": (out["row_loss"] * s["weight"].double()).sum() / rows, **out}
    return out
