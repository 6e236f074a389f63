"""Measured cases of four operators around the tied head, with their plain forms.

* ``logprobs``  — ``losses.token_logprobs``: log probabilities of given tokens over logits that exist, the entropy
  of each row and its top alternatives, with the gradient of the first two.
* ``tied``      — ``losses.tied_token_logprobs``: the same two numbers straight from the hidden states and the tied
  matrix, with no logits kept, and both gradients.
* ``layernorm`` — ``norm.layer_norm``: layer norm with the gradients of its input, weight and bias.
* ``adamw``     — ``embedding_grad.adamw_step_many``: one AdamW step over many tensors, moments in 32 or in 8 bits.

``run`` computes the plain form with elementary torch operations, or, where ``own`` is true, makes the calls that a
user makes of this package.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
IGNORE = -100
BLOCK = 128        # elements that share a scale in the 8-bit moments
E4M3_MAX = 448.0   # largest e4m3 value
E4M3_MIN = 2.0 ** -9  # smallest positive e4m3 value
HYPER = dict(learning_rate=3e-4, beta1=0.9, beta2=0.95, epsilon=1e-8, weight_decay=0.1)


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # A decoding step of 8 sequences: the sampled token's log probability and 20 alternatives for the answer.
        dict(name="logprobs_decode", op="logprobs", rows=8, vocab=50257, dtype="bfloat16", top_k=20, masked=True,
             backward=False),
        # A policy update on a tiny-vocabulary model that holds its logits, both gradients back to them.
        dict(name="logprobs_train", op="logprobs", rows=2048, vocab=32000, dtype="float16", top_k=0, masked=False,
             backward=True),
        # Scoring a prompt: log probabilities of its own tokens with 5 alternatives a position.
        dict(name="logprobs_score", op="logprobs", rows=4096, vocab=128256, dtype="bfloat16", top_k=5, masked=False,
             backward=False),
        # Scoring a handful of new tokens from their hidden states.
        dict(name="tied_decode", op="tied", rows=7, d=1024, vocab=50257, dtype="bfloat16", backward=False),
        # One micro-batch of a policy update, two sequences of 1024 tokens.
        dict(name="tied_train", op="tied", rows=2048, d=768, vocab=50257, dtype="float16", backward=True),
        # The same for a large vocabulary.
        dict(name="tied_train_large", op="tied", rows=4096, d=4096, vocab=128256, dtype="bfloat16", backward=True),
        # The final norm while decoding 8 sequences.
        dict(name="layernorm_decode", op="layernorm", rows=8, d=1024, dtype="float16", backward=False),
        # Training, 8 sequences of 1024 tokens.
        dict(name="layernorm_train", op="layernorm", rows=8192, d=1024, dtype="float16", backward=True),
        # Training, 4 sequences of 8192 tokens of a wide model.
        dict(name="layernorm_train_large", op="layernorm", rows=32768, d=4096, dtype="bfloat16", backward=True),
        # The optimizer of the smallest GPT, where the launches count.
        dict(name="adamw_tiny", op="adamw", layers=2, d=64, vocab=256, bits=32, grad="float32", copy="none", align=1),
        # The optimizer of a 24-layer GPT with 16-bit gradients and a 16-bit copy for the products.
        dict(name="adamw_gpt", op="adamw", layers=24, d=1024, vocab=50257, bits=32, grad="float16", copy="float16",
             align=128),
        # The same with its moments in 8 bits.
        dict(name="adamw_gpt_8bit", op="adamw", layers=24, d=1024, vocab=50257, bits=8, grad="float16",
             copy="float16", align=128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "tied", "layernorm", "adamw"])
    dtype = rng.choice(["float16", "bfloat16"])
    backward = rng.random() < 0.6
    if op == "logprobs":
        vocab = _log_int(rng, 100, 128256)
        rows = _log_int(rng, 1, min(16384, 4096 * 128256 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["float32", "float16", "bfloat16"]),
                    top_k=rng.choice([0, 1, 5, 20, 64]), masked=rng.random() < 0.5, backward=backward)
    if op == "tied":
        return dict(op=op, rows=_log_int(rng, 1, 4096), d=8 * _log_int(rng, 8, 512), vocab=_log_int(rng, 200, 128256),
                    dtype=dtype, backward=backward)
    if op == "layernorm":
        return dict(op=op, rows=_log_int(rng, 1, 32768), d=_log_int(rng, 16, 4096),
                    dtype=rng.choice(["float32", "float16", "bfloat16"]), backward=backward)
    bits = rng.choice([32, 8])
    return dict(op=op, layers=rng.randint(1, 24), d=_log_int(rng, 32, 1024), vocab=_log_int(rng, 200, 50257), bits=bits,
                grad=rng.choice(["float32", "float16", "bfloat16"]), copy=rng.choice(["none", "float16", "bfloat16"]),
                align=128 if bits == 8 else rng.choice([1, 128]))


# ---------------------------------------------------------------------------------------------------- the inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _tokens(rows, vocab, g):
    """Tokens of a batch whose padding (one row in nine) is ignored."""
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    if rows > 8:
        tokens[8::9] = IGNORE
    return tokens


def _upstream(rows, g):
    """Gradients that reach the log probabilities (advantages) and the entropies (a bonus)."""
    return (torch.randn(rows, generator=g, device=DEV),
            0.01 * (1.0 + 0.1 * torch.randn(rows, generator=g, device=DEV)))


def _shapes(case):
    """The parameter shapes of a GPT with biases, in order."""
    d, shapes = case["d"], [(case["vocab"], case["d"])]
    for _ in range(case["layers"]):
        shapes += [(d,), (d,)] + 4 * [(d, d), (d,)] + [(d,), (d,), (4 * d, d), (4 * d,), (d, 4 * d), (d,)]
    return shapes + [(d,), (d,)]


def _spans(case):
    """(start, elements) of each tensor in the flat buffers, and the buffers' length."""
    at, spans = 0, []
    for s in _shapes(case):
        n = math.prod(s)
        spans.append((at, n))
        at += -(-n // case["align"]) * case["align"]
    return spans, at


def _encode(x, root=False):
    """x (a multiple of BLOCK elements) as e4m3 codes and one fp32 scale a block. A positive root never becomes zero."""
    b = x.view(-1, BLOCK)
    top = b.abs().amax(dim=1, keepdim=True)
    live = top >= 2.0 ** -100
    up = torch.where(live, torch.div(torch.full_like(top, E4M3_MAX), top), torch.zeros_like(top))
    y = b * up
    if root:
        y = torch.where((b > 0) & (y < E4M3_MIN), torch.full_like(y, E4M3_MIN), y)
    scale = torch.where(live, top * (1.0 / E4M3_MAX), torch.zeros_like(top))
    return y.to(torch.float8_e4m3fn).view(-1), scale.view(-1)


def _decode(codes, scales):
    return (codes.float().view(-1, BLOCK) * scales.view(-1, 1)).view(-1)


def prepare(case, seed):
    g = _gen(seed)
    op, s = case["op"], {"case": case}
    if op == "logprobs":
        rows, vocab, dt = case["rows"], case["vocab"], TYPES[case["dtype"]]
        pitch = -(-vocab // 8) * 8  # the tied head writes its logits with rows of whole 16 bytes
        buf = torch.empty(rows, pitch, dtype=dt, device=DEV)
        for lo in range(0, rows, 1024):
            part = torch.randn(min(1024, rows - lo), pitch, generator=g, device=DEV)
            part *= 2.5
            buf[lo:lo + 1024] = part
        logits = buf[:, :vocab]
        s["tokens"] = _tokens(rows, vocab, g)
        if case["masked"]:  # a grammar that rules tokens out
            out = torch.rand(vocab, generator=g, device=DEV) < 0.3
            logits[:, out] = -math.inf
            logits[torch.arange(rows, device=DEV), s["tokens"].clamp(min=0)] = 1.0
        s["logits"] = logits.requires_grad_(case["backward"])
        s["up"] = _upstream(rows, g)
    elif op == "tied":
        rows, d, vocab, dt = case["rows"], case["d"], case["vocab"], TYPES[case["dtype"]]
        h = torch.randn(rows, d, generator=g, device=DEV)
        h /= h.square().mean(dim=1, keepdim=True).sqrt()
        s["hidden"] = h.to(dt).requires_grad_(case["backward"])
        s["weights"] = (0.02 * torch.randn(vocab, d, generator=g, device=DEV)).to(dt).requires_grad_(case["backward"])
        s["tokens"] = _tokens(rows, vocab, g)
        s["up"] = _upstream(rows, g)
    elif op == "layernorm":
        rows, d, dt = case["rows"], case["d"], TYPES[case["dtype"]]
        s["x"] = (1.5 * torch.randn(rows, d, generator=g, device=DEV) + 0.3).to(dt).requires_grad_(case["backward"])
        s["gamma"] = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)).requires_grad_(case["backward"])
        s["beta"] = (0.1 * torch.randn(d, generator=g, device=DEV)).requires_grad_(case["backward"])
        s["grad"] = torch.randn(rows, d, generator=g, device=DEV).to(dt)
    else:
        spans, n = _spans(case)
        w = torch.zeros(n, device=DEV)
        gr = torch.zeros(n, dtype=TYPES[case["grad"]], device=DEV)
        m, r = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
        for at, k in spans:  # the gaps between the tensors stay zero
            size = 10 ** float(torch.empty(()).uniform_(-3, -1, generator=torch.Generator().manual_seed(seed + at)))
            w[at:at + k].normal_(0, 0.02, generator=g)
            raw = size * torch.randn(k, generator=g, device=DEV)
            gr[at:at + k] = raw
            m[at:at + k] = 0.2 * raw + 0.3 * size * torch.randn(k, generator=g, device=DEV)
            r[at:at + k] = size * (0.3 + torch.rand(k, generator=g, device=DEV))
        cut = lambda flat: [flat[at:at + k] for at, k in spans]  # noqa: E731
        s.update(step=100, w=w, g=gr, ws=cut(w), gs=cut(gr), spans=spans)
        if case["bits"] == 8:
            s["m"], s["v"] = _encode(m), _encode(r, root=True)
            blocks = lambda q: [(q[0][at:at + k], q[1][at // BLOCK:-(-(at + k) // BLOCK)]) for at, k in spans]  # noqa: E731
            s["ms"], s["vs"] = blocks(s["m"]), blocks(s["v"])
        else:
            s["m"], s["v"] = m, r.square_()
            s["ms"], s["vs"] = cut(s["m"]), cut(s["v"])
        s["copy"], s["copies"] = None, None
        if case["copy"] != "none":
            s["copy"] = torch.zeros(n, dtype=TYPES[case["copy"]], device=DEV)
            s["copies"] = cut(s["copy"])
    return s


# -------------------------------------------------------------------------------------------------- the operators
def _rows(x, tokens, top_k, up):
    """(outputs, gradient of the logits or None) for fp32 logits x: log probabilities, entropies, alternatives."""
    live = tokens != IGNORE
    at = tokens.clamp(min=0).unsqueeze(1)
    top = x.amax(dim=1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(dim=1, keepdim=True)
    lse = top + total.log()
    logp = x - lse
    p = e / total
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    entropy = -plogp.sum(dim=1)
    out = {"logprobs": torch.where(live, logp.gather(1, at).squeeze(1), torch.zeros_like(entropy)),
           "entropy": torch.where(live, entropy, torch.zeros_like(entropy))}
    if top_k:
        bits = (x + 0.0).view(torch.int32)  # ordered as whole numbers, equal values by the lowest index
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2 ** 32
        key += 2 ** 32 - 1 - torch.arange(x.shape[1], device=x.device)
        ids = 2 ** 32 - 1 - (key.topk(top_k, dim=1).values & (2 ** 32 - 1))
        out["top_ids"] = torch.where(live.unsqueeze(1), ids, torch.full_like(ids, -1))
        out["top_logprobs"] = torch.where(live.unsqueeze(1), logp.gather(1, ids), torch.full((), -math.inf, device=x.device))
    if up is None:
        return out, None
    a, b = up[0].unsqueeze(1), up[1].unsqueeze(1)
    grad = -(p * (a + b * entropy.unsqueeze(1)) + b * plogp)
    grad.scatter_add_(1, at, a)
    return out, torch.where(live.unsqueeze(1), grad, torch.zeros_like(grad))


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "logprobs":
        out, grad = _rows(s["logits"].detach().float(), s["tokens"], min(case["top_k"], case["vocab"]),
                          s["up"] if case["backward"] else None)
        if grad is not None:
            out["grad_logits"] = grad.to(s["logits"].dtype)
        return out
    if op == "tied":
        h, w = s["hidden"].detach().float(), s["weights"].detach().float()
        out, grad = _rows(h @ w.t(), s["tokens"], 0, s["up"] if case["backward"] else None)
        if grad is not None:
            out["grad_hidden"] = (grad @ w).to(s["hidden"].dtype)
            out["grad_weights"] = (grad.t() @ h).to(s["weights"].dtype)
        return out
    if op == "layernorm":
        x, gamma, beta = s["x"].detach().float(), s["gamma"].detach(), s["beta"].detach()
        centred = x - x.mean(dim=1, keepdim=True)
        rstd = 1.0 / (centred.square().mean(dim=1, keepdim=True) + 1e-5).sqrt()
        xhat = centred * rstd
        out = {"y": (xhat * gamma + beta).to(s["x"].dtype)}
        if case["backward"]:
            gy = s["grad"].float()
            gg = gy * gamma
            gx = rstd * (gg - gg.mean(dim=1, keepdim=True) - xhat * (gg * xhat).mean(dim=1, keepdim=True))
            out["grad_x"] = gx.to(s["x"].dtype)
            out["grad_gamma"] = (gy * xhat).sum(dim=0)
            out["grad_beta"] = gy.sum(dim=0)
        return out
    # adamw: the flat buffers hold zeros between the tensors, and those stay zero.
    s["step"] += 1
    c = _scalars(s["step"])
    g = s["g"].float()
    eight = case["bits"] == 8
    m = _decode(*s["m"]) if eight else s["m"]
    v = _decode(*s["v"]).square() if eight else s["v"]
    m = c["b1"] * m + c["omb1"] * g
    v = c["b2"] * v + c["omb2"] * (g * g)
    root = v.sqrt()
    w = s["w"] * c["decay"] - (m * c["c1"]) / (root * c["c2"] + c["eps"])
    s["w"].copy_(w)
    if s["copy"] is not None:
        s["copy"].copy_(w)
    if eight:
        for q, new in ((s["m"], _encode(m)), (s["v"], _encode(root, root=True))):
            q[0].copy_(new[0])
            q[1].copy_(new[1])
        m, v = _decode(*s["m"]), _decode(*s["v"]).square()
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
        m, v = s["m"], s["v"]
    return {"weights": s["w"], "copy": s["copy"], "exp_avg": m, "exp_avg_sq": v}


def _scalars(step):
    b1, b2 = HYPER["beta1"], HYPER["beta2"]
    return dict(b1=b1, omb1=1 - b1, b2=b2, omb2=1 - b2, decay=1 - HYPER["learning_rate"] * HYPER["weight_decay"],
                c1=HYPER["learning_rate"] / (1 - b1 ** step), c2=1 / math.sqrt(1 - b2 ** step), eps=HYPER["epsilon"])


def _framework(s):
    case = s["case"]
    op = case["op"]
    if op == "logprobs":
        from nimbleml_b200.losses import token_logprobs

        r = token_logprobs(s["logits"], s["tokens"], IGNORE, top_k=min(case["top_k"], case["vocab"]))
        out = {"logprobs": r.logprobs, "entropy": r.entropy}
        if case["top_k"]:
            out.update(top_ids=r.top_ids, top_logprobs=r.top_logprobs)
        if case["backward"]:
            (out["grad_logits"],) = torch.autograd.grad((r.logprobs, r.entropy), (s["logits"],), s["up"])
        return out
    if op == "tied":
        from nimbleml_b200.losses import tied_token_logprobs

        r = tied_token_logprobs(s["hidden"], s["weights"], s["tokens"], IGNORE)
        out = {"logprobs": r.logprobs, "entropy": r.entropy}
        if case["backward"]:
            out["grad_hidden"], out["grad_weights"] = torch.autograd.grad(
                (r.logprobs, r.entropy), (s["hidden"], s["weights"]), s["up"])
        return out
    if op == "layernorm":
        from nimbleml_b200.norm import layer_norm

        y = layer_norm(s["x"], s["gamma"], s["beta"], 1e-5)
        out = {"y": y}
        if case["backward"]:
            out["grad_x"], out["grad_gamma"], out["grad_beta"] = torch.autograd.grad(
                y, (s["x"], s["gamma"], s["beta"]), s["grad"])
        return out
    from nimbleml_b200.embedding_grad import adamw_step_many, dequantize_moment

    s["step"] += 1
    adamw_step_many(s["ws"], s["gs"], s["ms"], s["vs"], step=s["step"], copies=s["copies"], **HYPER)
    m, v = s["m"], s["v"]
    if case["bits"] == 8:
        m, v = dequantize_moment(*m), dequantize_moment(*v, root=True)
    return {"weights": s["w"], "copy": s["copy"], "exp_avg": m, "exp_avg_sq": v}


def run(state):
    return _framework(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------- the work
def work(case):
    op = case["op"]
    if op == "logprobs":
        n, es = case["rows"] * case["vocab"], TYPES[case["dtype"]].itemsize
        # Per element: a product-add and an exponential, two sums; the gradient: the exponential again and two products.
        return {"bytes": n * es * (3 if case["backward"] else 1) + case["rows"] * (16 + 12 * case["top_k"]),
                "flops": n * (12 if case["backward"] else 6)}
    if op == "tied":
        rows, d, vocab, es = case["rows"], case["d"], case["vocab"], TYPES[case["dtype"]].itemsize
        return {"bytes": (rows + vocab) * d * es * (2 if case["backward"] else 1) + 16 * rows,
                "flops": 2 * rows * d * vocab * (3 if case["backward"] else 1)}
    if op == "layernorm":
        n, es = case["rows"] * case["d"], TYPES[case["dtype"]].itemsize
        return {"bytes": n * es * (4 if case["backward"] else 2) + case["d"] * (16 if case["backward"] else 8),
                "flops": n * (20 if case["backward"] else 8)}
    n = sum(math.prod(s) for s in _shapes(case))
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8  # the 8-bit moments' values are outputs too
    copy = 0 if case["copy"] == "none" else 2
    return {"bytes": n * (8 + TYPES[case["grad"]].itemsize + copy + state), "flops": n * 16}


# --------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "logprobs":
        return _exact_logprobs(s, case)
    if op == "tied":
        return _exact_tied(s, case)
    if op == "layernorm":
        return _exact_layernorm(s, case)
    return _exact_adamw(s, case)


def _exact_chunk(x, tokens, up):
    """Softmax quantities of 64-bit logits x, from their log-softmax; the gradients by differentiating it."""
    x = x.detach().requires_grad_(up is not None)
    logq = torch.log_softmax(x, dim=1)
    masked = torch.isneginf(x.detach())
    q = logq.exp()
    ent = -(q * logq.masked_fill(masked, 0.0)).sum(dim=1)
    used = tokens != IGNORE
    lp = logq[torch.arange(len(tokens), device=x.device), tokens.clamp(min=0)]
    lp, ent = lp.masked_fill(~used, 0.0), ent.masked_fill(~used, 0.0)
    grad = None
    if up is not None:
        (grad,) = torch.autograd.grad((lp, ent), (x,), (up[0].double(), up[1].double()))
        grad = grad.masked_fill(~used.unsqueeze(1), 0.0)
    return lp.detach(), ent.detach(), logq.detach(), grad


def _exact_logprobs(s, case):
    got = {k: [] for k in ("logprobs", "entropy", "top_ids", "top_logprobs", "grad_logits")}
    k, tokens = min(case["top_k"], case["vocab"]), s["tokens"]
    for lo in range(0, case["rows"], 512):
        cut = slice(lo, lo + 512)
        x, t = s["logits"].detach()[cut].double(), tokens[cut]
        up = (s["up"][0][cut], s["up"][1][cut]) if case["backward"] else None
        lp, ent, logq, grad = _exact_chunk(x, t, up)
        got["logprobs"].append(lp)
        got["entropy"].append(ent)
        if k:
            ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
            gone = (t == IGNORE).unsqueeze(1)
            got["top_ids"].append(ids.masked_fill(gone, -1))
            got["top_logprobs"].append(logq.gather(1, ids).masked_fill(gone, -math.inf))
        if grad is not None:
            got["grad_logits"].append(grad)
    return {name: torch.cat(v) for name, v in got.items() if v}


def _exact_tied(s, case):
    h, w, tokens = s["hidden"].detach().double(), s["weights"].detach().double(), s["tokens"]
    lps, ents, ghs, gw = [], [], [], torch.zeros_like(w) if case["backward"] else None
    for lo in range(0, case["rows"], 1024):
        cut = slice(lo, lo + 1024)
        up = (s["up"][0][cut], s["up"][1][cut]) if case["backward"] else None
        lp, ent, _, grad = _exact_chunk(h[cut] @ w.t(), tokens[cut], up)
        lps.append(lp)
        ents.append(ent)
        if grad is not None:
            ghs.append(grad @ w)
            gw += grad.t() @ h[cut]
    out = {"logprobs": torch.cat(lps), "entropy": torch.cat(ents)}
    if case["backward"]:
        out.update(grad_hidden=torch.cat(ghs), grad_weights=gw)
    return out


def _exact_layernorm(s, case):
    x = s["x"].detach().double().requires_grad_()
    gamma, beta = (s[k].detach().double().requires_grad_() for k in ("gamma", "beta"))
    var, mean = torch.var_mean(x, dim=1, keepdim=True, correction=0)
    y = (x - mean) * torch.rsqrt(var + 1e-5) * gamma + beta
    out = {"y": y.detach()}
    if case["backward"]:
        out["grad_x"], out["grad_gamma"], out["grad_beta"] = torch.autograd.grad(y, (x, gamma, beta), s["grad"].double())
    return out


def _exact_adamw(s, case):
    t, (b1, b2) = s["step"] + 1, (HYPER["beta1"], HYPER["beta2"])
    lr, eps, wd = HYPER["learning_rate"], HYPER["epsilon"], HYPER["weight_decay"]
    g = s["g"].double()
    if case["bits"] == 8:
        m = (s["m"][0].double().view(-1, BLOCK) * s["m"][1].double().unsqueeze(1)).flatten()
        v = (s["v"][0].double().view(-1, BLOCK) * s["v"][1].double().unsqueeze(1)).flatten().square_()
    else:
        m, v = s["m"].double(), s["v"].double()
    m = m.mul_(b1).add_(g, alpha=1 - b1)
    v = v.mul_(b2).addcmul_(g, g, value=1 - b2)
    step = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps)
    w = s["w"].double() * (1 - lr * wd) - lr * step
    # A value at the border of two 8-bit codes has no code of its own in 64 bits: those moments are left out.
    eight = case["bits"] == 8
    return {"weights": w, "copy": w if case["copy"] != "none" else None, "exp_avg": None if eight else m,
            "exp_avg_sq": None if eight else v}
