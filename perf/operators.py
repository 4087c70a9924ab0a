"""The operators over dense query and document vectors, as a user calls them and in plain torch: 8-bit rows with a scale for
each block of 128 values, the scores of such rows against each other, and the softmax loss of queries over all documents
with its gradients.  `listed` and `draw` give the sizes they are measured at, `run` one pass through an operator."""
import os
import sys

import torch

own = False
BLOCK = 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # a batch of query vectors on its way to the scorer: the smallest call, latency counts
        {"name": "quantize 64 queries", "op": "quantize", "rows": 64, "dim": 1024, "type": "f32"},
        # a corpus of 200 000 documents packed to 8 bits once, from the fp32 rows the index is given
        {"name": "quantize 200k docs", "op": "quantize", "rows": 200000, "dim": 1024, "type": "f32"},
        # vectors of another encoder, half precision, rows that end inside a block
        {"name": "quantize 30011 x 776", "op": "quantize", "rows": 30011, "dim": 776, "type": "f16"},
        # one query against a small corpus: the online form
        {"name": "scores 1 x 10k", "op": "scores", "rows": 1, "docs": 10000, "dim": 1024, "type": "f32"},
        # a batch of 100 queries against 200 000 documents: as much reading and writing as arithmetic
        {"name": "scores 100 x 200k", "op": "scores", "rows": 100, "docs": 200000, "dim": 1024, "type": "f32"},
        # odd sizes and another encoder's width
        {"name": "scores 1001 x 10007", "op": "scores", "rows": 1001, "docs": 10007, "dim": 784, "type": "bf16"},
        # a large batch against a large corpus: the product itself
        {"name": "scores 8k x 64k", "op": "scores", "rows": 8192, "docs": 65536, "dim": 1024, "type": "bf16"},
        # every query of a batch of 1000 against the 10 000-document corpus, half precision, loss only (evaluation)
        {"name": "loss 1000 x 10007", "op": "loss", "rows": 1000, "docs": 10007, "dim": 1024, "type": "f16", "scale": 50.0},
        # a large batch against 100 000 documents
        {"name": "loss 8k x 100k", "op": "loss", "rows": 8192, "docs": 100003, "dim": 1024, "type": "bf16", "scale": 20.0},
        # in-batch negatives of a small training batch: 32 queries, eight documents each
        {"name": "step 32 x 256", "op": "step", "rows": 32, "docs": 256, "dim": 1024, "type": "bf16", "scale": 20.0},
        # a training batch with mined negatives, half precision, sizes that end inside every tile
        {"name": "step 1001 x 10007", "op": "step", "rows": 1001, "docs": 10007, "dim": 776, "type": "f16", "scale": 50.0},
        # a large training batch against 50 000 documents
        {"name": "step 4k x 50k", "op": "step", "rows": 4096, "docs": 50021, "dim": 1024, "type": "bf16", "scale": 20.0},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["quantize", "scores", "loss", "step"])
    dim = 8 * rng.randrange(8, 161)          # 64 to 1280 values, in steps of 16 bytes of half precision
    if op == "quantize":
        return {"op": op, "rows": _log_int(rng, 1, 150000), "dim": dim, "type": rng.choice(["f32", "f16", "bf16"])}
    rows, docs = _log_int(rng, 1, 8192), _log_int(rng, 1 if op == "scores" else 2, 100000)
    most = {"scores": 1 << 29, "loss": 3 << 28, "step": 3 << 26}[op]      # query-document pairs: never more than the listed ones
    docs = max(2, min(docs, most // rows, most * 1024 // (rows * (dim + 8))))
    case = {"op": op, "rows": rows, "docs": docs, "dim": dim, "type": rng.choice(["f16", "bf16"])}
    if op == "scores":
        case["dim"] = dim + 8 * (dim // 8 % 2)                            # bytes: rows in steps of 16
        case["type"] = rng.choice(["f32", "f16", "bf16"])
    else:
        case["scale"] = rng.choice([1.0, 20.0, 50.0])
    return case


def _unit(rows, dim, gen):
    x = torch.randn(rows, dim, generator=gen, device="cuda")
    return x.mul_(x.square().sum(1, keepdim=True).rsqrt())


def _quantize(x):
    """The plain quantiser: exponents in 64 bits (a block's largest value may sit on the border), values in 32."""
    rows, dim = x.shape
    blocks = -(-dim // BLOCK)
    x = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - dim)).view(rows, blocks, BLOCK)
    most = x.abs().amax(2).double()
    e = torch.ceil(torch.log2(most / 448.0)).clamp_(-126, 120)
    e = e + (most > 448.0 * torch.exp2(e)).double()
    e = (e - (most <= 448.0 * torch.exp2(e - 1)).double()).clamp_(min=-126).to(torch.int32)
    down = ((127 - e) << 23).view(torch.float32)
    q = (x * down[:, :, None]).view(rows, blocks * BLOCK)[:, :dim].to(torch.float8_e4m3fn)
    return q.contiguous(), (e + 127).to(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, rows, dim = case["op"], case["rows"], case["dim"]
    kind = TYPES[case["type"]]
    if op == "quantize":
        return {"op": op, "x": _unit(rows, dim, gen).to(kind)}
    docs = _unit(case["docs"], dim, gen)
    target = torch.randint(0, case["docs"], (rows,), generator=gen, device="cuda")
    queries = _unit(rows, dim, gen) + 0.35 * docs[target]                 # each query leans to its document, as in training
    queries.mul_(queries.square().sum(1, keepdim=True).rsqrt())
    if op == "scores":
        qa, sa = _quantize(queries)
        qb, sb = _quantize(docs)
        return {"op": op, "qa": qa, "sa": sa, "qb": qb, "sb": sb, "kind": kind}
    target = target.to(torch.int32)
    if rows >= 8:
        target[-(rows // 16 + 1):] = -1                                   # the last rows of a batch are padding
    state = {"op": op, "queries": queries.to(kind), "docs": docs.to(kind), "target": target, "scale": case["scale"]}
    if op == "step":                                                      # mean over the batch; half precision with a loss scale
        state["grad"] = torch.full((rows,), (1024.0 if case["type"] == "f16" else 1.0) / rows, device="cuda")
    return state


def _own_run(s):
    here = os.path.join(os.getcwd(), "allan-poe_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import apoe
    if s["op"] == "quantize":
        q, scale = apoe.quantize_rows(s["x"])
        return {"q": q, "scale": scale}
    if s["op"] == "scores":
        return apoe.scaled_scores(s["qa"], s["sa"], s["qb"], s["sb"], out_dtype=s["kind"])
    loss, lse = apoe.softmax_loss_forward(s["queries"], s["docs"], s["target"], s["scale"])
    if s["op"] == "loss":
        return {"loss": loss, "lse": lse}
    dq, dd = apoe.softmax_loss_backward(s["queries"], s["docs"], s["target"], loss, lse, s["grad"], s["scale"])
    return {"loss": loss, "dqueries": dq, "ddocs": dd}


def run(state):
    if own:
        return _own_run(state)
    s = state
    if s["op"] == "quantize":
        q, scale = _quantize(s["x"])
        return {"q": q, "scale": scale}
    if s["op"] == "scores":
        a, b = (q.float() * _spread(e, q.shape[1]) for q, e in ((s["qa"], s["sa"]), (s["qb"], s["sb"])))
        return (a @ b.t()).to(s["kind"])
    x, w, scale = s["queries"].float(), s["docs"].float(), s["scale"]
    kept = s["target"] >= 0
    y = s["target"].clamp(min=0).long()[:, None]
    logits = (x @ w.t()).mul_(scale)
    logits.scatter_(1, y, -torch.inf)
    top = logits.amax(1, keepdim=True).clamp(min=-1e30)
    # the target's own logit in 64 bits, and the other documents' weight against it: where a row is nearly certain its loss
    # is that weight, and a rounding of a large logit would be a large part of it
    at = scale * (s["queries"].double() * s["docs"].double()[y[:, 0]]).sum(1, keepdim=True)
    p = logits.sub_(top).exp_()
    others = p.sum(1, keepdim=True)
    away = (others.log() + (top - at).float())
    loss = away.clamp(min=0) + (-away.abs()).exp().log1p()
    lse = torch.where(kept, (loss + at)[:, 0].float(), 0.0)
    kept_loss = torch.where(kept, loss[:, 0], 0.0)
    if s["op"] == "loss":
        return {"loss": kept_loss, "lse": lse}
    g = p.mul_((top - at).float().sub_(loss).exp_())
    g.scatter_(1, y, (-loss).expm1())
    g.mul_(torch.where(kept, s["grad"], 0.0)[:, None])
    kind = s["queries"].dtype
    return {"loss": kept_loss, "dqueries": ((g @ w) * scale).to(kind), "ddocs": ((g.t() @ x) * scale).to(kind)}


def _spread(exponent, dim):
    """One factor for each value from the scale byte of its block."""
    return (exponent.to(torch.int32) << 23).view(torch.float32).repeat_interleave(BLOCK, 1)[:, :dim]


def work(case):
    op, rows, dim = case["op"], case["rows"], case["dim"]
    blocks, size = -(-dim // BLOCK), BYTES[case["type"]]
    if op == "quantize":
        return {"bytes": rows * (dim * (size + 1) + blocks), "flops": 2 * rows * dim}
    docs = case["docs"]
    if op == "scores":
        return {"bytes": (rows + docs) * (dim + blocks) + rows * docs * size, "flops": 2 * rows * docs * dim}
    if op == "loss":
        return {"bytes": (rows + docs) * dim * size + 12 * rows, "flops": 2 * rows * docs * dim}
    return {"bytes": 2 * (rows + docs) * dim * size + 12 * rows, "flops": 6 * rows * docs * dim}   # scores once, two gradients


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "quantize":
        x = s["x"].double()
        rows, dim = x.shape
        q, scale = torch.zeros_like(x), []
        for b in range(0, dim, BLOCK):
            part = x[:, b:b + BLOCK]
            f, k = torch.frexp(part.abs().amax(1))                        # largest = f 2^k, f in [0.5, 1); 448 = 0.875 2^9
            e = torch.where(f > 0.875, k - 8, k - 9)
            e = torch.where(f == 0, torch.full_like(e, -126), e).clamp(min=-126)
            v = torch.ldexp(part, -e[:, None])
            _, kv = torch.frexp(v)
            step = torch.ldexp(torch.ones_like(v), (kv - 1).clamp(min=-6) - 3)
            q[:, b:b + BLOCK] = torch.round(v / step) * step
            scale.append((e + 127).to(torch.uint8))
        return {"q": q, "scale": torch.stack(scale, 1)}
    if s["op"] == "scores":
        out = torch.zeros(case["rows"], case["docs"], dtype=torch.float64, device="cuda")
        for b in range(s["sa"].shape[1]):
            k = slice(b * BLOCK, (b + 1) * BLOCK)
            fa, fb = (torch.ldexp(torch.ones_like(e, dtype=torch.float64), e.to(torch.int32) - 127) for e in (s["sa"][:, b], s["sb"][:, b]))
            out += (s["qa"][:, k].double() * fa[:, None]) @ (s["qb"][:, k].double() * fb[:, None]).t()
        return out
    x, w, t, scale = s["queries"].double(), s["docs"].double(), s["target"].long(), s["scale"]
    loss, lse = torch.zeros(x.shape[0], dtype=torch.float64, device="cuda"), torch.zeros(x.shape[0], dtype=torch.float64, device="cuda")
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for a in range(0, x.shape[0], 1024):                                  # by rows: the whole matrix in 64 bits is not held
        rows = slice(a, a + 1024)
        kept = torch.nonzero(t[rows] >= 0)[:, 0] + a
        if not kept.numel():
            continue
        logit = scale * (x[kept] @ w.t())
        lse[kept] = torch.logsumexp(logit, 1)
        each = torch.arange(kept.numel(), device="cuda")
        margin = logit - logit[each, t[kept]][:, None]
        margin[each, t[kept]] = -torch.inf
        away = torch.logsumexp(margin, 1)                                 # log of the others' weight against the target's
        loss[kept] = torch.nn.functional.softplus(away, threshold=60.0)
        if s["op"] == "step":
            g = torch.exp(logit - lse[kept][:, None])
            g[each, t[kept]] = -torch.sigmoid(away)
            g *= s["grad"].double()[kept][:, None]
            dx[kept] = scale * (g @ w)
            dw += scale * (g.t() @ x[kept])
    return {"loss": loss, "lse": lse} if s["op"] == "loss" else {"loss": loss, "dqueries": dx, "ddocs": dw}
