"""Cases of the operators around a training step's two ends: log probabilities of given tokens (with entropy and the top
alternatives) and their gradient, orthogonalised updates and the optimizer step that applies them.

``run`` takes the plain form (elementary torch operations in 32 bits or more) or, where ``own`` is set, the framework's calls.
"""
import math

import torch

own = False

DEV = "cuda"
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, MOMENTUM, DECAY, LOSS_SCALE = 0.02, 0.95, 0.01, 1024.0

DTYPE = {"f16": torch.float16, "f32": torch.float32}

MOST_LOGITS = 16384 * 32768 * 2            # bytes of logits
MOST_FLOPS = 5 * (3 * 2048 * 2048 * 8192 + 2048 ** 3)


def resnet50_layers():
    """Every parameter of the ResNet-50 of the training step, matrices as [c_out, c_in * kh * kw], vectors as such."""
    layers, c_in = ["64x147", "64", "64"], 64
    for stage, blocks in enumerate((3, 4, 6, 3)):
        mid = 64 * 2 ** stage
        for b in range(blocks):
            layers += ["%dx%d" % (mid, c_in), "%d" % mid, "%d" % mid, "%dx%d" % (mid, 9 * mid), "%d" % mid, "%d" % mid,
                       "%dx%d" % (4 * mid, mid), "%d" % (4 * mid), "%d" % (4 * mid)]
            if b == 0:
                layers += ["%dx%d" % (4 * mid, c_in), "%d" % (4 * mid), "%d" % (4 * mid)]
            c_in = 4 * mid
    return " ".join(layers + ["1000x2048", "1000"])


def mlp_layers(width, blocks):
    """Up and down projections of blocks of the Linear benchmark's width, with their biases."""
    return " ".join(["%dx%d" % (4 * width, width), "%d" % (4 * width), "%dx%d" % (width, 4 * width), "%d" % width] * blocks)


def shapes_of(text):
    return [tuple(int(v) for v in s.split("x")) for s in text.split()]


def listed():
    return [
        # the 1000-way head of an image classifier at its global batch: loss and top-5 accuracy in one pass
        {"name": "log_probs classes", "op": "log_probs", "rows": 2048, "vocab": 1000, "dtype": "f16", "top": 5},
        # one decoded token, with the alternatives that a server reports beside it: latency
        {"name": "log_probs decode", "op": "log_probs", "rows": 1, "vocab": 131072, "dtype": "f32", "top": 20},
        # scoring a batch of sequences; an odd vocabulary, so no row but the first starts on a vector
        {"name": "log_probs odd", "op": "log_probs", "rows": 4096, "vocab": 50021, "dtype": "f16", "top": 0},
        # a training batch's loss with a report of alternatives
        {"name": "log_probs large", "op": "log_probs", "rows": 16384, "vocab": 32768, "dtype": "f16", "top": 8},
        # one GPU's share of the image classifier's batch: latency
        {"name": "backward classes", "op": "backward", "rows": 256, "vocab": 1000, "dtype": "f16", "entropy": False},
        # policy gradient with an entropy bonus
        {"name": "backward odd", "op": "backward", "rows": 4096, "vocab": 50021, "dtype": "f16", "entropy": True},
        # fp32 logits of a large vocabulary
        {"name": "backward large", "op": "backward", "rows": 2048, "vocab": 131072, "dtype": "f32", "entropy": True},
        # the 7 x 7 stem of an image net: a small update, launches and latency
        {"name": "orthogonalize stem", "op": "orthogonalize", "count": 1, "rows": 64, "cols": 147, "dtype": "f32"},
        # the same projection of eight layers, half precision
        {"name": "orthogonalize stack", "op": "orthogonalize", "count": 8, "rows": 2048, "cols": 512, "dtype": "f16"},
        # the widest layer of the Linear benchmark
        {"name": "orthogonalize wide", "op": "orthogonalize", "count": 1, "rows": 8192, "cols": 2048, "dtype": "f32"},
        # every parameter of the ResNet-50 step
        {"name": "muon resnet50", "op": "muon", "layers": resnet50_layers()},
        # four blocks of the Linear benchmark's width 1024
        {"name": "muon mlp", "op": "muon", "layers": mlp_layers(1024, 4)},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["log_probs", "backward", "orthogonalize", "muon"])
    dtype = rng.choice(["f16", "f32"])
    if op in ("log_probs", "backward"):
        size = 2 if dtype == "f16" else 4
        vocab = _log_uniform(rng, 2, 131072)
        rows = _log_uniform(rng, 1, max(1, min(16384, MOST_LOGITS // size // vocab)))
        case = {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype}
        if op == "log_probs":
            return dict(case, top=min(vocab, rng.choice([0, 0, 1, 5, 8, 20, 32])))
        return dict(case, entropy=rng.random() < 0.5)
    if op == "orthogonalize":
        while True:
            count, rows, cols = _log_uniform(rng, 1, 16), _log_uniform(rng, 1, 8192), _log_uniform(rng, 1, 8192)
            if count * _flops(rows, cols) <= MOST_FLOPS:
                return {"op": op, "count": count, "rows": rows, "cols": cols, "dtype": dtype}
    layers = []
    for _ in range(_log_uniform(rng, 1, 24)):
        rows = _log_uniform(rng, 1, 2048)
        layers += ["%dx%d" % (rows, _log_uniform(rng, 1, 2048)), "%d" % rows][:rng.choice([1, 2])]
    return {"op": op, "layers": " ".join(layers)}


def _flops(rows, cols):
    """Per step the product of a matrix with its transpose and the square of the result (both symmetric: half of each), and the
    product that makes the next iterate."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (3 * m * m * n + m ** 3)


def work(case):
    if case["op"] in ("log_probs", "backward"):
        n, size = case["rows"] * case["vocab"], 2 if case["dtype"] == "f16" else 4
        if case["op"] == "log_probs":
            return {"bytes": n * size + case["rows"] * (8 + 8 + 12 * case["top"]), "flops": 5 * n}
        return {"bytes": 2 * n * size + case["rows"] * (8 + 16 + (4 if case["entropy"] else 0)), "flops": 8 * n}
    if case["op"] == "orthogonalize":
        n, size = case["count"] * case["rows"] * case["cols"], 2 if case["dtype"] == "f16" else 4
        return {"bytes": 2 * n * size, "flops": case["count"] * _flops(case["rows"], case["cols"])}
    shapes = shapes_of(case["layers"])
    # parameter and momentum read and written, gradient read, fp16 copy written
    return {"bytes": 22 * sum(math.prod(s) for s in shapes), "flops": sum(_flops(*s) if len(s) == 2 else 6 * s[0] for s in shapes)}


# ------------------------------------------------------------------ inputs --
def _logits(case, gen):
    """Logits as a model gives them: a spread of a few units and a few likely tokens a row; some rows with most of the vocabulary
    masked (by -inf, or by the type's lowest value), the last of more than two rows with nothing left."""
    rows, vocab, dtype = case["rows"], case["vocab"], DTYPE[case["dtype"]]
    x = torch.empty(rows, vocab, dtype=dtype, device=DEV)
    x.normal_(0.0, 2.5, generator=gen)
    likely = torch.randint(0, vocab, (rows, 4), device=DEV, generator=gen)
    x.scatter_(1, likely, (8.0 + 2.0 * torch.randn(rows, 4, device=DEV, generator=gen)).to(dtype))
    masked = torch.arange(0, rows, 61, device=DEV)[1:]
    if masked.numel():
        keep = torch.rand(masked.numel(), vocab, device=DEV, generator=gen) < 0.1
        keep.scatter_(1, likely[masked], True)
        lowest = torch.finfo(dtype).min if vocab >= 1024 else -math.inf   # (so that what is asked for is not masked itself)
        low = torch.where(torch.arange(masked.numel(), device=DEV) % 2 == 0, -math.inf, lowest)[:, None].to(dtype)
        x[masked] = torch.where(keep, x[masked], low)
    if rows > 2:
        x[-1] = -math.inf
    targets = torch.where(torch.rand(rows, device=DEV, generator=gen) < 0.7, likely[:, 0],
                          torch.randint(0, vocab, (rows,), device=DEV, generator=gen))
    targets[masked] = likely[masked, 0]
    targets[3::17] = -100   # padding
    return x, targets


def _gradient(shape, gen, dtype=torch.float32):
    """A weight gradient: a few dozen directions carry most of it."""
    rows, cols = shape[-2:]
    rank = min(32, rows, cols)
    decay = torch.logspace(0, -1, rank, device=DEV)
    a = torch.randn(*shape[:-2], rows, rank, device=DEV, generator=gen)
    b = torch.randn(*shape[:-2], rank, cols, device=DEV, generator=gen)
    return (0.02 * ((a * decay) @ b / math.sqrt(rank) + 0.2 * torch.randn(*shape, device=DEV, generator=gen))).to(dtype)


def _statistics(x):
    """Largest logit and logarithm of the sum of exponentials against it, and the entropy: what the forward pass has left."""
    m = x.amax(dim=1).float()
    stats, entropy = torch.empty(x.shape[0], 2, device=DEV), torch.empty(x.shape[0], device=DEV)
    for lo in range(0, x.shape[0], 1024):
        d = (x[lo:lo + 1024].double() - m[lo:lo + 1024, None].double()).nan_to_num(nan=-math.inf, neginf=-math.inf)
        e = d.exp()
        s = e.sum(1)
        empty = s == 0
        s = torch.where(empty, 1.0, s)
        stats[lo:lo + 1024, 1] = s.log().float()
        entropy[lo:lo + 1024] = torch.where(empty, 0.0, s.log() - torch.where(e > 0, d * e, 0.0).sum(1) / s).float()
    stats[:, 0] = m
    return stats, entropy


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    if case["op"] == "log_probs":
        x, targets = _logits(case, gen)
        return {"case": case, "logits": x, "targets": targets}
    if case["op"] == "backward":
        x, targets = _logits(case, gen)
        stats, entropy = _statistics(x)
        rows = case["rows"]
        return {"case": case, "logits": x, "targets": targets, "stats": stats, "entropy": entropy,
                "d_log_probs": LOSS_SCALE / 16 * torch.randn(rows, device=DEV, generator=gen),
                "d_entropy": torch.full((rows,), LOSS_SCALE / 64, device=DEV) if case["entropy"] else None}
    if case["op"] == "orthogonalize":
        shape = (case["rows"], case["cols"])
        return {"case": case, "g": _gradient(shape if case["count"] == 1 else (case["count"],) + shape, gen, DTYPE[case["dtype"]])}
    shapes = shapes_of(case["layers"])
    starts, n = [], 0
    for s in shapes:   # every parameter on a 256-byte boundary of one flat buffer, as the training steps keep them
        starts.append(n)
        n += (math.prod(s) + 63) // 64 * 64
    flat = {k: torch.zeros(n, device=DEV) for k in ("params", "grads", "momenta")}
    flat["params_f16"] = torch.zeros(n, dtype=torch.float16, device=DEV)
    views = {k: [f[a:a + math.prod(s)].view(s) for a, s in zip(starts, shapes)] for k, f in flat.items()}
    for i, s in enumerate(shapes):
        views["params"][i].normal_(0.0, s[-1] ** -0.5, generator=gen)
        if len(s) == 2:
            views["grads"][i].copy_(_gradient(s, gen) * LOSS_SCALE)
            views["momenta"][i].copy_(_gradient(s, gen))
        else:
            views["grads"][i].normal_(0.0, 0.02 * LOSS_SCALE, generator=gen)
            views["momenta"][i].normal_(0.0, 0.02, generator=gen)
    flat["params_f16"].copy_(flat["params"])
    return {"case": case, "flat": flat, "views": views}


# ------------------------------------------------------------------ plain forms --
def _log_probs(x, targets, top):
    x = x.float()
    m = x.amax(dim=1, keepdim=True)
    d = torch.where(x == -math.inf, x, x - m)   # (a row of -inf alone keeps them)
    e = d.exp()
    s = e.sum(dim=1, keepdim=True)
    some = s > 0
    s = torch.where(some, s, 1.0)
    lp = d - s.log()
    entropy = torch.where(some, s.log() - torch.where(e > 0, d * e, 0.0).sum(dim=1, keepdim=True) / s, 0.0)[:, 0]
    token = lp.gather(1, targets.clamp(min=0)[:, None])[:, 0]
    out = {"log_probs": torch.where(targets < 0, 0.0, token), "entropy": entropy}
    if top:
        bits = (x + 0.0).view(torch.int32).long()   # keys in the order of the values, ties to the lowest index
        key = ((bits ^ ((bits >> 31) & 0x7fffffff)) << 32) + (0xffffffff - torch.arange(x.shape[1], device=x.device))
        index = 0xffffffff - (key.topk(top, dim=1).values & 0xffffffff)
        out["top_indices"] = index
        out["top_log_probs"] = lp.gather(1, index)
    return out


def _backward(x, targets, stats, entropy, d_log_probs, d_entropy):
    dtype, x = x.dtype, x.float()
    m, log_sum = stats[:, :1], stats[:, 1:]
    lp = torch.where(x == -math.inf, x, x - m) - log_sum
    p = lp.exp()
    g = torch.where(targets < 0, 0.0, d_log_probs)[:, None]
    dx = -g * p
    if d_entropy is not None:
        dx = dx - torch.where(p > 0, p * (lp + entropy[:, None]), 0.0) * d_entropy[:, None]
    dx.scatter_add_(1, targets.clamp(min=0)[:, None], g)
    return torch.where(m == -math.inf, 0.0, dx).to(dtype)


def _orthogonalize(g):
    x = g.float()
    if g.shape[-2] > g.shape[-1]:
        x = x.mT
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.mT if g.shape[-2] > g.shape[-1] else x).to(g.dtype)


def _muon(views):
    for p, g, v, h in zip(views["params"], views["grads"], views["momenta"], views["params_f16"]):
        g = g * (1.0 / LOSS_SCALE)
        v.mul_(MOMENTUM).add_(g)
        u = g + MOMENTUM * v
        if p.dim() == 2:
            u = _orthogonalize(u) * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        p.mul_(1.0 - LR * DECAY).sub_(LR * u)
        h.copy_(p)


def run(state):
    case = state["case"]
    if own:
        from nectarml_b200 import ops
    if case["op"] == "log_probs":
        if own:
            r = ops.token_log_probs(state["logits"], state["targets"], top=case["top"])
            out = {"log_probs": r.log_probs, "entropy": r.entropy}
            return dict(out, top_indices=r.top_indices, top_log_probs=r.top_log_probs) if case["top"] else out
        return _log_probs(state["logits"], state["targets"], case["top"])
    if case["op"] == "backward":
        args = [state[k] for k in ("logits", "targets", "stats", "entropy", "d_log_probs", "d_entropy")]
        return ops.token_log_probs_backward(*args) if own else _backward(*args)
    if case["op"] == "orthogonalize":
        return ops.orthogonalize(state["g"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS) if own else _orthogonalize(state["g"])
    v = state["views"]
    if own:
        ops.muon_step(v["params"], v["grads"], v["momenta"], v["params_f16"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY,
                      inv_scale=1.0 / LOSS_SCALE, steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    else:
        _muon(v)
    return {k: state["flat"][k] for k in ("params", "momenta", "params_f16")}


# ------------------------------------------------------------------ 64 bits --
def _exact_polar(g):
    """The same polynomial of the singular values, on the eigenvectors' side of the smaller Gram matrix's recurrence."""
    g = g.double()
    tall = g.shape[-2] > g.shape[-1]
    x = g.transpose(-2, -1) if tall else g
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + EPS)
    one = torch.eye(x.shape[-2], dtype=torch.float64, device=x.device)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        s = torch.matmul(x, x.transpose(-2, -1))
        x = torch.matmul(a * one + torch.matmul(s, b * one + c * s), x)
    return x.transpose(-2, -1) if tall else x


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "log_probs":
        x, t = state["logits"], state["targets"]
        lps, ents = [], []
        for lo in range(0, case["rows"], 512):
            lp = torch.log_softmax(x[lo:lo + 512].double(), dim=1)
            lp = torch.where(torch.isneginf(x[lo:lo + 512]), -math.inf, lp)
            tt = t[lo:lo + 512]
            lps.append(torch.where(tt < 0, 0.0, lp[torch.arange(len(tt), device=DEV), tt.clamp(min=0)]))
            ents.append(torch.special.entr(lp.exp()).sum(1))
        out = {"log_probs": torch.cat(lps), "entropy": torch.cat(ents)}
        if case["top"]:
            best = [torch.log_softmax(x[lo:lo + 512].double(), dim=1).sort(dim=1, descending=True).values[:, :case["top"]]
                    for lo in range(0, case["rows"], 512)]
            best = torch.cat(best)
            dead = torch.isneginf(x).all(dim=1)
            out.update(top_indices=None, top_log_probs=torch.where(dead[:, None], -math.inf, best))
        return out
    if case["op"] == "backward":
        x, t = state["logits"], state["targets"]
        parts = []
        for lo in range(0, case["rows"], 512):
            xs, ts = x[lo:lo + 512].double(), t[lo:lo + 512]
            dead = torch.isneginf(xs).all(dim=1, keepdim=True)
            p = torch.softmax(xs, dim=1).masked_fill(dead, 0.0)
            one = torch.zeros_like(p)
            one[torch.arange(len(ts), device=DEV), ts.clamp(min=0)] = 1.0
            d = (one - p) * torch.where(ts < 0, 0.0, state["d_log_probs"][lo:lo + 512].double())[:, None]
            if case["entropy"]:
                h = torch.special.entr(p)
                d += (h - p * h.sum(1, keepdim=True)) * state["d_entropy"][lo:lo + 512, None].double()
            # (the operator's result is the gradient to this precision; a half result is rounded once)
            parts.append(d.masked_fill(dead, 0.0).float() if case["dtype"] == "f16" else d.masked_fill(dead, 0.0))
        return torch.cat(parts)
    if case["op"] == "orthogonalize":
        return _exact_polar(state["g"])
    v = state["views"]
    out = {k: state["flat"][k].double() for k in ("params", "momenta", "params_f16")}
    lo = 0
    for p, g, b in zip(v["params"], v["grads"], v["momenta"]):
        n = p.numel()
        grad = g.double() / LOSS_SCALE
        momentum = MOMENTUM * b.double() + grad
        update = grad + MOMENTUM * momentum
        if p.dim() == 2:
            update = _exact_polar(update) * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        new = p.double() - LR * (DECAY * p.double() + update)
        out["params"][lo:lo + n] = out["params_f16"][lo:lo + n] = new.reshape(-1)
        out["momenta"][lo:lo + n] = momentum.reshape(-1)
        lo += (n + 63) // 64 * 64
    return out
