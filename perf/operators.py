"""Cases of the operators at the end of a training step and of scoring: the log-probabilities of given classes with their
entropy and best alternatives, their gradient, the clipping of gradients by their global norm, and the Adam update that clips.

``own`` False: plain torch in 32 bits.  ``own`` True: the package's entry points on the same inputs.
"""
import itertools
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
IGNORE = -100
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 1e-2
# Clipping in place leaves gradients whose norm IS the bound: a second pass on them would have nothing to scale.  Every pass
# therefore asks for a bound a little under the last one's, and scales as a training step with large gradients does.
SHRINK = 0.999


def listed():
    return [
        # one decoding step of one sequence: the launch and its latency are all there is
        dict(name="score-token", op="score", rows=1, classes=50021, dtype="bf16", top=8, ignored=False, masked=False, pad=0),
        # a decoding step of a batch that answers with alternatives, part of the classes forbidden
        dict(name="score-batch", op="score", rows=96, classes=131072, dtype="fp16", top=20, ignored=False, masked=True, pad=0),
        # scoring a prompt: many rows over an odd number of classes, no alternatives asked for
        dict(name="score-prompt", op="score", rows=4000, classes=65537, dtype="fp32", top=0, ignored=False, masked=False, pad=0),
        # labels of eight outdoor sweeps (20 classes, label 0 not scored) with the three best classes of each point
        dict(name="score-points", op="score", rows=400070, classes=20, dtype="fp32", top=3, ignored=True, masked=False, pad=0),
        # training on points with 55 classes, the logits a column slice of a wider matrix
        dict(name="train-points", op="train", rows=220011, classes=55, dtype="fp32", top=0, ignored=True, masked=False, pad=9),
        # training a classifier over a middling number of classes, alternatives and all of their gradients
        dict(name="train-classes", op="train", rows=1031, classes=8191, dtype="fp16", top=4, ignored=True, masked=True, pad=0),
        # training on tokens: the largest logits, in 16 bits
        dict(name="train-tokens", op="train", rows=4096, classes=131072, dtype="bf16", top=0, ignored=True, masked=False, pad=0),
        # the gradients of one small block: the latency of the launches
        dict(name="clip-block", op="clip", tensors=6, total=9001, dtype="fp32", norm="two", align=1),
        # a segmentation network of this package's size: hundreds of tensors, a few million values, slots of four values
        dict(name="clip-network", op="clip", tensors=310, total=5300000, dtype="fp32", norm="two", align=4),
        # a large model in 16 bits, the norm the largest magnitude
        dict(name="clip-large", op="clip", tensors=120, total=400000003, dtype="bf16", norm="max", align=1),
        # the optimiser's step over three of the gradient all-reduce's buckets
        dict(name="adam-buckets", op="adam", tensors=3, total=19700000),
        # the same over a model whose state is far larger than any cache
        dict(name="adam-large", op="adam", tensors=40, total=260000000),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["score", "train", "clip", "adam"])
    if op == "adam":
        return dict(op=op, tensors=rng.randint(1, 40), total=_log_uniform(rng, 20000, 2.5e8))
    if op == "clip":
        tensors = _log_uniform(rng, 1, 600)
        return dict(op=op, tensors=tensors, total=_log_uniform(rng, max(3000, 8 * tensors), 4e8), dtype=rng.choice(sorted(DTYPES)),
                    norm=rng.choice(["two", "two", "max", "one"]), align=rng.choice([1, 4]))
    classes = _log_uniform(rng, 2, 262144)
    top = min(classes, rng.choice([0, 1, 5, rng.randint(2, 32)]))
    most = (2 ** 26 if top else 2 ** 28) if op == "score" else 2 ** 26
    rows = _log_uniform(rng, 1, max(2, min(500000, most // classes)))
    return dict(op=op, rows=rows, classes=classes, dtype=rng.choice(sorted(DTYPES)), top=top, ignored=rng.random() < 0.5,
                masked=rng.random() < 0.3, pad=rng.choice([0, 0, 1, 8]))


def _cuts(case, align):
    """Where the tensors of a list start in their common buffer, how long they are, and how long the buffer is: sizes over
    three orders of magnitude, every start a multiple of ``align`` values."""
    rng = random.Random("%d/%d" % (case["tensors"], case["total"]))
    share = [math.exp(rng.uniform(0.0, 7.0)) for _ in range(case["tensors"])]
    scale = case["total"] / sum(share)
    sizes = [max(1, int(s * scale)) for s in share]
    ends = list(itertools.accumulate(-(-n // align) * align for n in sizes))
    return list(zip([0] + ends, sizes)), ends[-1]


def _flat_normal(size, dtype, gen):
    return torch.empty(size, dtype=dtype, device="cuda").normal_(generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] in ("score", "train"):
        rows, c = case["rows"], case["classes"]
        dtype = DTYPES[case["dtype"]]
        wide = torch.empty(rows, c + case["pad"], dtype=dtype, device="cuda").normal_(0.0, 2.5, generator=gen)
        logits = wide[:, :c]
        target = torch.randint(0, c, (rows,), device="cuda", generator=gen)
        if case["masked"]:      # three of ten classes are forbidden, other ones for each eighth row; the given class is not
            forbidden = torch.rand(min(rows, 8), c, device="cuda", generator=gen) < 0.3
            for k in range(forbidden.size(0)):
                logits[k::8].masked_fill_(forbidden[k], float("-inf"))
        # a trained model prefers the given class in many rows
        lift = 12.0 * torch.rand(rows, 1, device="cuda", generator=gen)
        logits.scatter_(1, target[:, None], lift.to(dtype))
        if case["ignored"]:
            target = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.1, IGNORE, target)
        state = dict(op=case["op"], logits=logits, target=target, top=case["top"])
        if case["op"] == "train":
            state["logits"] = logits.detach().requires_grad_(True)
            state["g_logprob"] = torch.randn(rows, device="cuda", generator=gen) - 1.0
            state["g_entropy"] = 0.1 * torch.randn(rows, device="cuda", generator=gen)
            state["g_top"] = torch.randn(rows, case["top"], device="cuda", generator=gen) if case["top"] else None
        return state
    if case["op"] == "clip":
        cuts, size = _cuts(case, case["align"])
        dtype = DTYPES[case["dtype"]]
        flat, params = torch.zeros(size, dtype=dtype, device="cuda"), []
        values = torch.zeros_like(flat)
        scales = (0.1 + 0.9 * torch.rand(len(cuts), device="cuda", generator=gen)).tolist()
        for (at, n), scale in zip(cuts, scales):
            p = values[at: at + n].requires_grad_(True)
            p.grad = flat[at: at + n].normal_(0.0, scale, generator=gen)
            params.append(p)
        norm = {"one": 1.0, "two": 2.0, "max": math.inf}[case["norm"]]
        bound = {"one": 0.2 * size, "two": 0.25 * math.sqrt(size), "max": 1.0}[case["norm"]]
        return dict(op="clip", flat=flat, params=params, norm=norm, bound=bound)
    cuts, size = _cuts(case, 4)
    flats = dict(p=_flat_normal(size, torch.float32, gen).mul_(0.05), g=_flat_normal(size, torch.float32, gen).mul_(0.01),
                 m=_flat_normal(size, torch.float32, gen).mul_(0.003), v=_flat_normal(size, torch.float32, gen).square_().mul_(1e-4))
    state = dict(op="adam", step=100, bound=0.005 * math.sqrt(size), **flats)
    for k in "pgmv":
        state["list_" + k] = [flats[k][at: at + -(-n // 4) * 4] for at, n in cuts]
    return state


# ---- the plain forms


def _plain_scores(x, target, top):
    """x (rows, classes) in 32 bits."""
    x = x + 0.0
    best = x.amax(1, keepdim=True)
    off = x - best
    e = torch.exp(off)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    entropy = (log_total - torch.where(e > 0, e * off, 0.0).sum(1, keepdim=True) / total).squeeze(1)
    scored = target != IGNORE
    at = torch.where(scored, target, 0)[:, None]
    logprob = torch.where(scored, (off.gather(1, at) - log_total).squeeze(1), 0.0)
    if not top:
        return logprob, entropy, None, None, best + log_total
    order = torch.sort(x, dim=1, descending=True, stable=True)
    return logprob, entropy, (order.values[:, :top] - best) - log_total, order.indices[:, :top].contiguous(), best + log_total


def _plain_gradient(x, lse, s, entropy, top_index):
    """d / d logits of sum(g_logprob * logprob) + sum(g_entropy * entropy) + sum(g_top * top_logprob)."""
    scored = s["target"] != IGNORE
    g = torch.where(scored, s["g_logprob"], 0.0)[:, None]
    given = torch.where(scored, s["target"], 0)[:, None]
    total = g if top_index is None else g + s["g_top"].sum(1, keepdim=True)
    logp = x - lse
    p = torch.exp(logp)
    d = torch.where(p > 0, p * (-total - s["g_entropy"][:, None] * (logp + entropy[:, None])), 0.0)
    d.scatter_add_(1, given, g)
    if top_index is not None:
        d.scatter_add_(1, top_index, s["g_top"])
    return d


def _plain_norm(flat, kind):
    x = flat.to(torch.float32)
    if kind == 2.0:
        return torch.sqrt((x * x).sum())
    return x.abs().sum() if kind == 1.0 else x.abs().amax()


def _run_plain(s):
    if s["op"] in ("score", "train"):
        x = s["logits"].detach().to(torch.float32)
        logprob, entropy, top_logprob, top_index, lse = _plain_scores(x, s["target"], s["top"])
        out = [logprob, entropy] + ([top_logprob, top_index] if s["top"] else [])
        if s["op"] == "train":
            out.append(_plain_gradient(x, lse, s, entropy, top_index).to(s["logits"].dtype))
        return out
    if s["op"] == "clip":
        grads = [p.grad for p in s["params"]]
        norm = _plain_norm(torch.cat(grads), s["norm"])
        scale = (s["bound"] / (norm + 1e-6)).clamp(max=1.0)
        torch._foreach_mul_(grads, scale)           # (a product in 32 bits, rounded once)
        s["bound"] *= SHRINK
        return [norm, s["flat"]]
    s["step"] += 1
    norm = _plain_norm(s["g"], 2.0)
    g = s["g"] * (s["bound"] / (norm + 1e-6)).clamp(max=1.0) + DECAY * s["p"]
    s["m"].mul_(BETA1).add_(g * (1.0 - BETA1))
    s["v"].mul_(BETA2).add_(g * g * (1.0 - BETA2))
    size, root = LR / (1.0 - BETA1 ** s["step"]), math.sqrt(1.0 - BETA2 ** s["step"])
    s["p"].sub_(size * (s["m"] / (torch.sqrt(s["v"]) / root + EPS)))
    return [norm, s["p"], s["m"], s["v"]]


# ---- the package's operators


def _run_own(s):
    if s["op"] in ("score", "train"):
        from curvecloudnet_amd.loss import token_logprobs
        r = token_logprobs(s["logits"], s["target"], top=s["top"], ignore_index=IGNORE)
        if s["op"] == "score":
            return [r.logprob, r.entropy] + ([r.top_logprob, r.top_index] if s["top"] else [])
        outs, gs = [r.logprob, r.entropy], [s["g_logprob"], s["g_entropy"]]
        if s["top"]:
            outs.append(r.top_logprob)
            gs.append(s["g_top"])
        grad = torch.autograd.grad(outs, s["logits"], gs)[0]
        return outs + ([r.top_index] if s["top"] else []) + [grad]
    if s["op"] == "clip":
        from curvecloudnet_amd.parallel import clip_grad_norm_
        norm = clip_grad_norm_(s["params"], s["bound"], norm_type=s["norm"])
        s["bound"] *= SHRINK
        return [norm, s["flat"]]
    from curvecloudnet_amd.parallel import adam_step_
    s["step"] += 1
    norm = adam_step_(s["list_p"], s["list_g"], s["list_m"], s["list_v"], s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS,
                      weight_decay=DECAY, max_norm=s["bound"])
    return [norm, s["p"], s["m"], s["v"]]


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


def work(case):
    if case["op"] in ("score", "train"):
        rows, c = case["rows"], case["classes"]
        size = DTYPES[case["dtype"]].itemsize
        nbytes = rows * c * size + rows * (8 + 4 + 4 + case["top"] * 12)
        flops = 6 * rows * c
        if case["op"] == "train":
            nbytes += rows * c * size + rows * (4 + 4 + case["top"] * 4)
            flops += 7 * rows * c
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "clip":
        n = sum(k for _, k in _cuts(case, case["align"])[0])
        return {"bytes": 2 * n * DTYPES[case["dtype"]].itemsize, "flops": 3 * n}
    n = _cuts(case, 4)[1]
    return {"bytes": 28 * n, "flops": 18 * n}


# ---- the definitions in 64 bits


def _exact_rows(x, target, top, g_logprob, g_entropy, g_top):
    """One block of rows, x in 64 bits: probabilities first, everything else from them."""
    z = torch.logsumexp(x, 1, keepdim=True)
    logp = x - z
    p = logp.exp()
    entropy = -torch.special.xlogy(p, p).sum(1)
    scored = (target != IGNORE).double()
    onehot = torch.zeros_like(p).scatter_(1, target.clamp(min=0)[:, None], scored[:, None])
    logprob = torch.where(onehot > 0, logp, 0.0).sum(1)
    best = torch.topk(x, top, dim=1) if top else None
    out = [logprob, entropy] + ([best.values - z, None] if top else [])
    if g_logprob is not None:
        # through p: d logp_j / d x_i = [i = j] - p_i, d H / d x_i = -p_i (log p_i + H)
        weight = onehot * g_logprob.double()[:, None]
        if top:
            ordered = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
            weight.scatter_add_(1, ordered, g_top.double())
        slope = torch.where(p > 0, p * (logp.clamp(min=-1e300) + entropy[:, None]), 0.0)
        out.append(weight - p * weight.sum(1, keepdim=True) - slope * g_entropy.double()[:, None])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("score", "train"):
        x, block = s["logits"].detach(), max(1, (1 << 25) // case["classes"])
        train = case["op"] == "train"
        parts = []
        for i in range(0, case["rows"], block):
            cut = slice(i, i + block)
            parts.append(_exact_rows(x[cut].double(), s["target"][cut], s["top"], s["g_logprob"][cut] if train else None,
                                     s["g_entropy"][cut] if train else None, s["g_top"][cut] if train and s["top"] else None))
        return [None if parts[0][k] is None else torch.cat([part[k] for part in parts]) for k in range(len(parts[0]))]
    if case["op"] == "clip":
        x = s["flat"].double()
        norm = torch.linalg.vector_norm(x, ord=s["norm"])
        return [norm, x * min(1.0, s["bound"] / (float(norm) + 1e-6))]
    p, g, m, v = (s[k].double() for k in "pgmv")
    norm = torch.linalg.vector_norm(g)
    t = s["step"] + 1
    g = g * min(1.0, s["bound"] / (float(norm) + 1e-6)) + DECAY * p
    m = BETA1 * m + (1.0 - BETA1) * g
    v = BETA2 * v + (1.0 - BETA2) * g * g
    p = p - LR * (m / (1.0 - BETA1 ** t)) / (torch.sqrt(v / (1.0 - BETA2 ** t)) + EPS)
    return [norm, p, m, v]
