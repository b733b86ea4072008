"""The operators at the two ends of a language model's step, as cases to time: the embedding of its tokens, the log
probabilities (with entropy and top alternatives) of the tokens it is asked about, and the global norm by which the
gradients are clipped.

    embed   rows of the embedding table by token, times a scale; `backward`: the table's gradient, summed by token
    linear  log probability and entropy from activations and head weight, without logits in memory; `backward`: both
            gradients, as a policy-gradient loss with an entropy bonus has them formed
    logits  the same from logits, with the `top` most probable tokens; `backward`: the logits' gradient
    norm    2-norm over all gradients of a model
    clip    an AdamW step on gradients clipped to a global norm

A token of -1 names none (the padding of a ragged batch): its row has log probability and entropy 0 and no gradient.
Model shapes are those of the README model (width 512, inner width 1024) and of the 1.35 B model (2048, 6144), both with
a vocabulary of 32000, 16 gate blocks and 4 convolution taps.
"""
import functools
import math
import os
import sys

import torch

own = False

DEV = "cuda"
VOCAB, BLOCKS, CONV = 32000, 16, 4
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
LR, BETAS, EPS, DECAY, MAX_NORM = 3e-4, (0.9, 0.999), 1e-8, 0.1, 1.0


def listed():
    return [
        # the embedding of one token for each of a full decoding batch of the 1.35 B model
        dict(name="embed_decode", kind="embed", tokens=256, vocab=VOCAB, width=2048, dtype="bf16", backward=False),
        # a few short sequences of odd length through the README model, as in fine-tuning: the table's gradient is
        # mostly rows that no token names
        dict(name="embed_ragged", kind="embed", tokens=3 * 517, vocab=VOCAB, width=512, dtype="f32", backward=True),
        # the training batch of the 1.35 B model: 8 sequences of 4096 tokens
        dict(name="embed_train_1b", kind="embed", tokens=8 * 4096, vocab=VOCAB, width=2048, dtype="f32", backward=True),
        # policy-gradient fine-tuning: short sequences of odd length, a fifth of the positions padding
        dict(name="linear_ragged", kind="linear", rows=3 * 516, vocab=VOCAB, width=512, padded=0.2, backward=True),
        # scoring four prompts of 777 tokens with the 1.35 B model
        dict(name="linear_score", kind="linear", rows=4 * 777, vocab=VOCAB, width=2048, padded=0.0, backward=False),
        # a full training batch of the 1.35 B model
        dict(name="linear_train_1b", kind="linear", rows=8 * 4095, vocab=VOCAB, width=2048, padded=0.1, backward=True),
        # serving: the token just chosen and five alternatives, for one user and for a full decoding batch
        dict(name="logits_single", kind="logits", rows=1, vocab=VOCAB, dtype="bf16", top=5, padded=0.0, backward=False),
        dict(name="logits_batch", kind="logits", rows=256, vocab=VOCAB, dtype="bf16", top=20, padded=0.0, backward=False),
        # logits of an odd vocabulary in fp32, in training: the rows start at odd addresses
        dict(name="logits_train_odd", kind="logits", rows=3 * 517, vocab=31999, dtype="f32", top=0, padded=0.2, backward=True),
        # the gradients of the README model, 107 tensors from 512 values to 16 million
        dict(name="norm_readme", kind="norm", width=512, inner=1024, layers=8, vocab=VOCAB, dtype="f32"),
        # the gradients of the 1.35 B model, 315 tensors, in bf16
        dict(name="norm_1b", kind="norm", width=2048, inner=6144, layers=24, vocab=VOCAB, dtype="bf16"),
        # a clipped optimiser step: table, head and a layer of the 1.35 B model
        dict(name="clip_step_1b", kind="clip", width=2048, inner=6144, layers=1, vocab=VOCAB, dtype="f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges; sizes are spread over their logarithm, and any whole number where the operator
    takes one (the head's width is a multiple of 8)."""
    kind = rng.choice(["embed", "linear", "logits", "logits", "norm", "clip"])
    vocab = rng.choice([VOCAB, _log_int(rng, 1000, VOCAB)])
    if kind == "embed":
        return dict(kind=kind, tokens=_log_int(rng, 1, 32768), vocab=vocab, width=_log_int(rng, 64, 2048),
                    dtype=rng.choice(["f32", "bf16"]), backward=rng.random() < 0.7)
    padded = rng.choice([0.0, 0.1, 0.3])
    if kind == "linear":
        return dict(kind=kind, rows=_log_int(rng, 1, 32760), vocab=vocab, width=8 * _log_int(rng, 8, 256), padded=padded,
                    backward=rng.random() < 0.6)
    if kind == "logits":
        backward = rng.random() < 0.3
        return dict(kind=kind, rows=_log_int(rng, 1, 4096), vocab=vocab, dtype=rng.choice(["f32", "bf16"]),
                    top=rng.choice([0, 1, 5, 20]), padded=padded, backward=backward)
    width = BLOCKS * _log_int(rng, 16, 128)
    return dict(kind=kind, width=width, inner=width * rng.choice([2, 3]), layers=1 if kind == "clip" else rng.randint(1, 24),
                vocab=_log_int(rng, 1000, VOCAB), dtype="f32" if kind == "clip" else rng.choice(["f32", "bf16"]))


# ---- inputs ----------------------------------------------------------------------------------------------------
def _tokens(n, vocab):
    """Token ids as text has them: the k-th most frequent about 1/k as often as the first, whose share is 7 %."""
    return (float(vocab) ** torch.rand(n, device=DEV, dtype=torch.float64)).long().sub_(1).clamp_(0, vocab - 1)


def _asked(rows, vocab, padded):
    """Tokens asked about; the padded share of the rows names none."""
    return torch.where(torch.rand(rows, device=DEV) < padded, -1, torch.randint(0, vocab, (rows,), device=DEV))


def _upstream(rows):
    """Gradients of a policy-gradient loss: advantages over the number of rows, and an entropy bonus."""
    return torch.randn(rows, device=DEV) / rows, torch.rand(rows, device=DEV) * (-0.02 / rows)


def _shapes(case):
    """Parameters of a model, or of its table, head and some layers."""
    h, i, v = case["width"], case["inner"], case["vocab"]
    layer = [(h,), (2 * h, h), (BLOCKS, h // BLOCKS, h // BLOCKS), (BLOCKS, h // BLOCKS), (BLOCKS, h // BLOCKS, h // BLOCKS),
             (BLOCKS, h // BLOCKS), (h, h), (CONV, h), (h,), (2 * i, h), (h, i), (h,), (h,)]
    return [(v, h), *(layer * case["layers"]), (h,), (v, h)]


def prepare(case, seed):
    torch.manual_seed(seed)
    kind = case["kind"]
    dtype = DTYPES[case.get("dtype", "bf16")]
    if kind == "embed":
        n, v, h = case["tokens"], case["vocab"], case["width"]
        weight = (torch.randn(v, h, device=DEV) / math.sqrt(h)).to(dtype).requires_grad_(case["backward"])
        return dict(kind=kind, ids=_tokens(n, v), weight=weight, scale=math.sqrt(h), backward=case["backward"],
                    go=torch.randn(n, h, device=DEV).to(dtype) if case["backward"] else None)
    if kind == "linear":
        n, v, h = case["rows"], case["vocab"], case["width"]
        weight = torch.randn(v, h, device=DEV) / math.sqrt(h)
        tokens = _asked(n, v, case["padded"])
        # some tokens that the model expects (up to near certainty) and some that surprise it
        act = torch.randn(n, h, device=DEV) + weight[tokens.clamp(min=0)] * (16 * torch.rand(n, 1, device=DEV))
        return dict(kind=kind, weight=weight.bfloat16().requires_grad_(case["backward"]),
                    act=act.bfloat16().requires_grad_(case["backward"]), tokens=tokens, go=_upstream(n), backward=case["backward"])
    if kind == "logits":
        n, v = case["rows"], case["vocab"]
        tokens = _asked(n, v, case["padded"])
        logits = 2.5 * torch.randn(n, v, device=DEV)
        logits[torch.arange(n, device=DEV), tokens.clamp(min=0)] += 20 * torch.rand(n, device=DEV)
        return dict(kind=kind, logits=logits.to(dtype).requires_grad_(case["backward"]), tokens=tokens, top=case["top"],
                    go=_upstream(n), backward=case["backward"])
    grads = [(torch.randn(s, device=DEV) * 10 ** (-2 - 2 * torch.rand((), device=DEV))).to(dtype) for s in _shapes(case)]
    if kind == "norm":
        return dict(kind=kind, grads=grads)
    params = [torch.nn.Parameter(torch.randn_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    return dict(kind=kind, params=params, moments=[torch.zeros_like(g) for g in grads + grads], step=0, opt=None)


# ---- the framework's operators ---------------------------------------------------------------------------------
@functools.lru_cache(None)
def _package():
    sys.path.insert(0, os.path.join(os.getcwd(), "hawk-pytorch_b200"))
    import hawk_b200
    from hawk_b200 import train
    return hawk_b200, train


def _run_own(state):
    hawk, train = _package()
    kind = state["kind"]
    if kind == "embed":
        out = hawk.embedding(state["ids"], state["weight"], state["scale"])
        return [out, *(torch.autograd.grad(out, [state["weight"]], state["go"]) if state["backward"] else ())]
    if kind == "linear":
        out = hawk.linear_logprobs(state["weight"], state["act"], state["tokens"])
        return [*out, *(torch.autograd.grad(out, [state["weight"], state["act"]], state["go"]) if state["backward"] else ())]
    if kind == "logits":
        out = hawk.token_logprobs(state["logits"], state["tokens"], state["top"])
        return [*out, *(torch.autograd.grad(out[:2], [state["logits"]], state["go"]) if state["backward"] else ())]
    if kind == "norm":
        return [hawk.grad_norm(state["grads"])]
    params = state["params"]
    if state["opt"] is None:  # an optimiser lives as long as its parameters
        state["opt"] = train.FusedAdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, max_grad_norm=MAX_NORM)
    opt = state["opt"]
    opt.step()
    return [opt.grad_norm, *(p.detach() for p in params), *(opt.state[p]["exp_avg"] for p in params),
            *(opt.state[p]["exp_avg_sq"] for p in params)]


# ---- the plain forms -------------------------------------------------------------------------------------------
def _log_softmax(x):
    x = x - x.amax(-1, keepdim=True)
    return x - x.exp().sum(-1, keepdim=True).log()


def _scores(logp, tokens):
    """Log probability and entropy for the rows that name a token, and those rows."""
    named = tokens >= 0
    lp = logp.gather(-1, tokens.clamp(min=0)[:, None])[:, 0]
    return torch.where(named, lp, 0), torch.where(named, -(logp.exp() * logp).sum(-1), 0), named


def _logits_gradient(logp, entropy, tokens, named, go):
    """d lp = onehot - p; d entropy = -p (log p + entropy)."""
    p = logp.exp()
    d = -(go[0][:, None] * p) - go[1][:, None] * (p * (logp + entropy[:, None]))
    d.scatter_add_(1, tokens.clamp(min=0)[:, None], go[0][:, None])
    return torch.where(named[:, None], d, 0)


def _norm(grads):
    return torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()


def _adamw(p, g, m, v, step):
    m.mul_(BETAS[0]).add_(g * (1 - BETAS[0]))
    v.mul_(BETAS[1]).add_(g * g * (1 - BETAS[1]))
    p.mul_(1 - LR * DECAY).sub_(m / (1 - BETAS[0] ** step) / ((v / (1 - BETAS[1] ** step)).sqrt() + EPS) * LR)


def _run_plain(state):
    kind = state["kind"]
    if kind == "embed":
        ids, w = state["ids"], state["weight"]
        out = [(w.float()[ids] * state["scale"]).to(w.dtype)]
        if state["backward"]:
            dw = torch.zeros(w.shape, device=DEV).index_add_(0, ids, state["go"].float() * state["scale"])
            out.append(dw.to(w.dtype))
        return out
    if kind == "linear":
        w, act = state["weight"].float(), state["act"].float()
        logp = _log_softmax(act @ w.T)
        lp, entropy, named = _scores(logp, state["tokens"])
        if not state["backward"]:
            return [lp, entropy]
        d = _logits_gradient(logp, entropy, state["tokens"], named, state["go"])
        return [lp, entropy, (d.T @ act).bfloat16(), (d @ w).bfloat16()]
    if kind == "logits":
        x, top = state["logits"].float(), state["top"]
        logp = _log_softmax(x)
        lp, entropy, named = _scores(logp, state["tokens"])
        if top:
            ids = x.sort(dim=-1, descending=True, stable=True)[1][:, :top]
            best = [torch.where(named[:, None], logp.gather(-1, ids), -math.inf), torch.where(named[:, None], ids, -1)]
        else:
            best = [x[:, :0], state["tokens"][:, None][:, :0]]
        if not state["backward"]:
            return [lp, entropy, *best]
        d = _logits_gradient(logp, entropy, state["tokens"], named, state["go"])
        return [lp, entropy, *best, d.to(state["logits"].dtype)]
    if kind == "norm":
        return [_norm(state["grads"])]
    params, (k, moments) = state["params"], (len(state["params"]), state["moments"])
    state["step"] += 1
    norm = _norm([p.grad for p in params])
    coef = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
    [_adamw(p, p.grad * coef, m, v, state["step"]) for p, m, v in zip(params, moments[:k], moments[k:])]
    return [norm, *(p.detach() for p in params), *moments]


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------
def work(case):
    kind, es = case["kind"], 4 if case.get("dtype") == "f32" else 2
    if kind == "embed":
        n, v, h = case["tokens"], case["vocab"], case["width"]
        named = v * (1 - math.exp(-n / v))  # rows that are read, about (each once)
        back = n * h * es + v * h * es if case["backward"] else 0  # the upstream gradient; the table's
        return {"bytes": 8 * n + min(n, named) * h * es + n * h * es + back, "flops": (2 if case["backward"] else 1) * n * h}
    if kind == "linear":
        n, v, h = case["rows"], case["vocab"], case["width"]
        return {"bytes": (2 if case["backward"] else 1) * 2 * (n + v) * h + 16 * n, "flops": (6 if case["backward"] else 2) * n * h * v}
    if kind == "logits":
        n, v = case["rows"], case["vocab"]
        return {"bytes": (2 if case["backward"] else 1) * es * n * v + (16 + 12 * case["top"]) * n, "flops": 6 * n * v}
    size = sum(math.prod(s) for s in _shapes(case))
    return {"bytes": es * size, "flops": 2 * size} if kind == "norm" else {"bytes": 28 * size, "flops": 16 * size}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------
def _exact_rows(x, tokens, go, top, backward):
    """The outputs of one block of rows of logits x (64 bits), and the logits' gradient."""
    named = tokens >= 0
    p = torch.softmax(x, -1)
    lse = torch.logsumexp(x, -1)
    entropy = lse - (p * x).sum(-1)
    at = tokens.clamp(min=0)[:, None]
    lp = x.gather(1, at)[:, 0] - lse
    keep = named.double()
    out = [lp * keep, entropy * keep]
    if top is not None:
        ids = x.sort(dim=-1, descending=True, stable=True).indices[:, :top]
        out += [(x.gather(1, ids) - lse[:, None]).masked_fill(~named[:, None], -math.inf), ids.masked_fill(~named[:, None], -1)]
    if not backward:
        return out, None
    hot = torch.zeros_like(x).scatter_(1, at, 1.0)
    d_entropy = p * (lse[:, None] - x - entropy[:, None])
    return out, (go[0].double()[:, None] * (hot - p) + go[1].double()[:, None] * d_entropy) * keep[:, None]


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    with torch.no_grad():
        if kind == "embed":
            w, ids, scale = state["weight"].double(), state["ids"], state["scale"]
            out = [w.index_select(0, ids) * scale]
            if case["backward"]:
                out.append(torch.zeros_like(w).index_add(0, ids, state["go"].double(), alpha=scale))
            return out
        if kind in ("linear", "logits"):
            n, tokens, go = case["rows"], state["tokens"], state["go"]
            top = case.get("top") if kind == "logits" else None
            parts, grads = [], []
            dw = torch.zeros(case["vocab"], case.get("width", 1), dtype=torch.float64, device=DEV)
            for r in (slice(i, i + 2048) for i in range(0, n, 2048)):
                x = (torch.nn.functional.linear(state["act"][r].double(), state["weight"].double()) if kind == "linear"
                     else state["logits"][r].double())
                out, d = _exact_rows(x, tokens[r], (go[0][r], go[1][r]), top, case["backward"])
                parts.append(out)
                if d is not None and kind == "linear":
                    dw.addmm_(d.T, state["act"][r].double())
                    grads.append(d.mm(state["weight"].double()))
                elif d is not None:
                    grads.append(d)
            outs = [torch.cat(o) for o in zip(*parts)]
            if not case["backward"]:
                return outs
            return [*outs, dw, torch.cat(grads)] if kind == "linear" else [*outs, torch.cat(grads)]
        grads = state["grads"] if kind == "norm" else [p.grad for p in state["params"]]
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g.double()) for g in grads]))
        if kind == "norm":
            return [norm]
        scaled = [g.double() * min(1.0, MAX_NORM / (float(norm) + 1e-6)) for g in grads]
        # the first step: both moments start at zero, and their bias corrections undo the (1 - beta) factors
        new = [p.double() * (1 - LR * DECAY) - LR * g / (g.abs() + EPS) for p, g in zip(state["params"], scaled)]
        return [norm, *new, *((1 - BETAS[0]) * g for g in scaled), *((1 - BETAS[1]) * g * g for g in scaled)]
