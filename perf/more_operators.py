"""The operators of training on a large vocabulary, as measurable cases.

  ce      cross entropy of labels over a vocabulary from hidden states and head weights, the logits
          never kept, with its gradient (functional.linear_cross_entropy)
  kl      distillation on a teacher's distribution over the vocabulary, from the hidden states and
          head weights of both, with its gradient (functional.linear_distill)
  norm    the global norm of many gradients (ops.grad_norm)
  clip    ... and the gradients scaled by it, from accumulators into gradients of the parameters'
          types (ops.clip_grads)

  x bf16 [tokens, hidden], weight bf16 [vocabulary, hidden], labels int64 [tokens]
  z = x weight^T;  ce: loss_n = log sum_v exp z_nv - z_n,label;  rows of ignore_index take no part
  kl: loss_n = sum_v p_nv (log p_nv - log q_nv), p = softmax(z_teacher / T), q = softmax(z / T);
      rows that a mask leaves out take no part
  mean: over the rows that take part

The hidden width and vocabulary are those of the decoder layer here and its model's, and generic ones
of the same ranges.
"""
import math
import os
import sys

import torch

own = False

_mods = None


def _lib():
    """The framework's (functional, ops), imported at the first call that needs them."""
    global _mods
    if _mods is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "qwen-palettize_amd"))
        from palettize_hip import functional, ops
        _mods = functional, ops
    return _mods


# ---- the cases ------------------------------------------------------------------------------
def listed():
    return [
        # a few tokens scored under a small model: the smallest call, where latency counts
        dict(name="ce_eval_t17_v32000_h1024", kind="ce", tokens=17, vocab=32000, hidden=1024,
             ignored=0.0, grads="none"),
        # one answer of 16 tokens scored under the model: a pass over the head's weights
        dict(name="ce_eval_t16_v151936", kind="ce", tokens=16, vocab=151936, hidden=2560,
             ignored=0.0, grads="none"),
        # perplexity of four documents of 2048 tokens
        dict(name="ce_eval_t8192_v151936", kind="ce", tokens=8192, vocab=151936, hidden=2560,
             ignored=0.0, grads="none"),
        # a training step of 8 x 512 tokens, the head trained too; padding at the ends: the largest
        dict(name="ce_step_t4096_v151936", kind="ce", tokens=4096, vocab=151936, hidden=2560,
             ignored=0.05, grads="both"),
        # tuning of adapters on question and answer: a frozen head, labels on the answers only
        dict(name="ce_frozen_t4096_v50257_h1600", kind="ce", tokens=4096, vocab=50257, hidden=1600,
             ignored=0.6, grads="x"),
        # a micro-batch of a small model, nothing of it a round number
        dict(name="ce_step_t777_v32001_h1000", kind="ce", tokens=777, vocab=32001, hidden=1000,
             ignored=0.1, grads="both"),
        # the last block of layers distilled through the model's frozen head, which both sides share
        dict(name="kl_frozen_t2048_v151936", kind="kl", tokens=2048, vocab=151936, hidden=2560,
             teacher_hidden=0, ignored=0.0, temperature=1.0, grads="x"),
        # a small student with a head of its own and a wider teacher, softened
        dict(name="kl_step_t1500_v32000_h1024", kind="kl", tokens=1500, vocab=32000, hidden=1024,
             teacher_hidden=2560, ignored=0.2, temperature=2.0, grads="both"),
        # a few tokens of a small model
        dict(name="kl_frozen_t100_v8003_h512", kind="kl", tokens=100, vocab=8003, hidden=512,
             teacher_hidden=0, ignored=0.1, temperature=1.0, grads="x"),
        # palettes and adapters of 36 layers: many small tensors of two types
        dict(name="norm_adapters_36_layers", kind="norm", tensors="adapters", layers=36,
             hidden=2560, intermediate=9728),
        # the head's gradient, and those of a layer's dense weights
        dict(name="norm_head_v151936", kind="norm", tensors="head", layers=1, hidden=2560,
             intermediate=9728, vocab=151936),
        # a layer's gradients, summed over micro-batches in fp32, into bf16 ones
        dict(name="clip_layer", kind="clip", tensors="layer", layers=1, hidden=2560,
             intermediate=9728),
    ]


def _log(rng, lo, hi):
    """A whole number whose logarithm is uniform over lo..hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng):
    """The model's width, or a multiple of 8 of the usual range."""
    return 2560 if rng.random() < 0.3 else 8 * _log(rng, 32, 640)


def draw(rng):
    kind = rng.choice(("ce", "ce", "ce", "kl", "kl", "norm", "clip"))
    if kind in ("norm", "clip"):
        tensors = rng.choice(("adapters", "layer"))
        # clipped gradients all come back: of two layers at most
        layers = _log(rng, 1, 36 if kind == "norm" else 2) if tensors == "adapters" else 1
        return dict(kind=kind, tensors=tensors, layers=layers, hidden=8 * _log(rng, 16, 320),
                    intermediate=8 * _log(rng, 16, 1216))
    hidden = _width(rng)
    vocab = _log(rng, 1000, 152000 * 2560 // max(hidden, 2560))
    # no more products than the largest listed case, and no more logits
    work = 4096 * 151936 * 2560
    teacher = 0 if kind == "ce" or rng.random() < 0.5 else _width(rng)
    per = vocab * (3 * hidden if kind == "ce" else 2 * hidden + 2 * max(teacher, hidden))
    tokens = _log(rng, 1, max(1, min(16384, 3 * work // per, 4096 * 151936 // vocab)))
    case = dict(kind=kind, tokens=tokens, vocab=vocab, hidden=hidden,
                ignored=rng.choice((0.0, 0.0, 0.1, 0.6)),
                grads=rng.choice(("none", "x", "both", "both")))
    if kind == "kl":
        case.update(teacher_hidden=teacher, temperature=rng.choice((1.0, 1.0, 2.0, 0.7)))
    return case


# ---- the inputs -------------------------------------------------------------------------------
def _shapes(case):
    """(shape, dtype) of the gradients that a case sums."""
    h, f = case["hidden"], case["intermediate"]
    q, kv = 4096 * h // 2560 // 8 * 8, 1024 * h // 2560 // 8 * 8
    linears = [(q, h), (kv, h), (kv, h), (h, q), (f, h), (f, h), (h, f)]
    if case["tensors"] == "adapters":
        # a linear's palettes (fp32, four values for 256 weights) and the two factors of its adapter
        one = [t for n, k in linears for t in (((n, -(-k // 256), 4), torch.float32),
                                               ((16, k), torch.bfloat16), ((n, 16), torch.bfloat16))]
        return one * case["layers"]
    dtype = torch.float32 if case["kind"] == "clip" else torch.bfloat16
    one = [(s, dtype) for s in linears] + [((h,), dtype)] * 2
    head = [((case["vocab"], h), torch.bfloat16)] if case["tensors"] == "head" else []
    return head + one


def _taking_part(case, g):
    """Which tokens take part: all but stretches at random places, one of them at least."""
    n = case["tokens"]
    if not case["ignored"]:
        return torch.ones(n, dtype=torch.bool, device="cuda")
    run = torch.rand(n // 16 + 1, generator=g, device="cuda") >= case["ignored"]
    keep = run.repeat_interleave(16)[:n]
    keep[-1] = True
    return keep


def _head(g, vocab, hidden):
    """Weights that give logits of a spread of 2.5 from hidden states of unit spread."""
    return (torch.randn(vocab, hidden, generator=g, device="cuda") * (2.5 * hidden ** -0.5)).bfloat16()


def _states(g, weight, words):
    """Hidden states that lean towards a word each: some clearly, some hardly."""
    n, h = words.numel(), weight.shape[1]
    lean = 3 * torch.rand(n, 1, generator=g, device="cuda")
    return (torch.randn(n, h, generator=g, device="cuda") + lean * weight[words].float()).bfloat16()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind in ("norm", "clip"):
        shapes = _shapes(case)
        # the spread of gradients differs from tensor to tensor
        spread = (10 ** (-4 + 3 * torch.rand(len(shapes), generator=g, device="cuda"))).tolist()
        grads = [(torch.randn(s, generator=g, device="cuda") * w).to(t)
                 for (s, t), w in zip(shapes, spread)]
        out = [torch.empty(s, dtype=torch.bfloat16, device="cuda") for s, _ in shapes]
        return dict(kind=kind, grads=grads, out=out, max_norm=1.0)
    n, vocab = case["tokens"], case["vocab"]
    words = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    keep = _taking_part(case, g)
    weight = _head(g, vocab, case["hidden"])
    s = dict(kind=kind, weight=weight, grads=case["grads"], keep=keep)
    if kind == "ce":
        s.update(x=_states(g, weight, words), labels=torch.where(keep, words, -100))
    else:
        wide = case["teacher_hidden"]
        s["teacher_weight"] = _head(g, vocab, wide) if wide else weight.clone()
        s["teacher_x"] = _states(g, s["teacher_weight"], words)
        # a student that is near the teacher where it can be
        s["x"] = _states(g, weight, words) if wide else (
            0.9 * s["teacher_x"].float()
            + 0.3 * torch.randn(n, case["hidden"], generator=g, device="cuda")).bfloat16()
        s.update(mask=keep if case["ignored"] else None, temperature=case["temperature"])
    s["x"].requires_grad_(case["grads"] != "none")
    s["weight"].requires_grad_(case["grads"] == "both")
    return s


# ---- the plain forms ----------------------------------------------------------------------------
def _log_softmax(z):
    z = z - z.amax(-1, keepdim=True)
    return z - torch.log(torch.exp(z).sum(-1, keepdim=True))


def _grads(s, dz, scale):
    """Gradients of x (nothing for rows that take no part) and of the head's weights from those of
    the logits of the rows that do."""
    live = s["keep"]
    grad_x = torch.zeros_like(s["x"])
    grad_x[live] = ((dz @ s["weight"].float()) * scale).bfloat16()
    if s["grads"] == "x":
        return (grad_x,)
    return grad_x, ((dz.T @ s["x"][live].float()) * scale).bfloat16()


@torch.no_grad()
def _ce(s):
    live, (x, w) = s["keep"], (s["x"], s["weight"])
    labels = s["labels"][live]
    logp = _log_softmax(x[live].float() @ w.float().T)
    rows = -logp.gather(1, labels[:, None])[:, 0]
    if s["grads"] == "none":
        loss = torch.zeros(x.shape[0], device=x.device)
        loss[live] = rows
        return loss
    dz = torch.exp(logp)
    dz.scatter_add_(1, labels[:, None], -torch.ones_like(rows)[:, None])
    return rows.mean(), *_grads(s, dz, 1 / rows.numel())


@torch.no_grad()
def _kl(s):
    live, T = s["keep"], s["temperature"]
    logp = _log_softmax(s["teacher_x"][live].float() @ s["teacher_weight"].float().T / T)
    logq = _log_softmax(s["x"][live].float() @ s["weight"].float().T / T)
    p = torch.exp(logp)
    rows = (p * (logp - logq)).sum(-1)
    if s["grads"] == "none":
        loss = torch.zeros(s["x"].shape[0], device=logp.device)
        loss[live] = rows
        return loss
    return rows.mean(), *_grads(s, torch.exp(logq) - p, 1 / (T * rows.numel()))


def _norm(grads):
    return torch.sqrt(torch.stack([(v.float() * v.float()).sum() for v in grads]).double().sum()).float()


def _clip(s):
    norm = _norm(s["grads"])
    scale = (s["max_norm"] / (norm + 1e-6)).clamp(max=1)
    return norm, *[(v.float() * scale).to(o.dtype) for v, o in zip(s["grads"], s["out"])]


# ---- one pass -------------------------------------------------------------------------------------
def run(s):
    kind = s["kind"]
    if kind in ("norm", "clip"):
        if own:
            if kind == "norm":
                return _lib()[1].grad_norm(s["grads"])
            return _lib()[1].clip_grads(s["grads"], s["max_norm"], out=s["out"]), *s["out"]
        return _norm(s["grads"]) if kind == "norm" else _clip(s)
    if not own:
        return _ce(s) if kind == "ce" else _kl(s)
    reduction = "none" if s["grads"] == "none" else "mean"
    if kind == "ce":
        loss = _lib()[0].linear_cross_entropy(s["x"], s["weight"], s["labels"], reduction=reduction)
    else:
        loss = _lib()[0].linear_distill(s["x"], s["weight"], s["teacher_x"], s["teacher_weight"],
                                        mask=s["mask"], temperature=s["temperature"],
                                        reduction=reduction)
    if s["grads"] == "none":
        return loss
    wanted = (s["x"],) if s["grads"] == "x" else (s["x"], s["weight"])
    return loss.detach(), *torch.autograd.grad(loss, wanted)


def _part(case):
    """The rows that take part, about."""
    return max(1, round(case["tokens"] * (1 - case["ignored"])))


def work(case):
    if case["kind"] in ("norm", "clip"):
        size = {torch.float32: 4, torch.bfloat16: 2}
        elements = sum(math.prod(s) for s, _ in _shapes(case))
        read = sum(math.prod(s) * size[t] for s, t in _shapes(case))
        # the norm is known only when all has been read: what clips it reads it again
        return dict(bytes=read if case["kind"] == "norm" else 2 * read + 2 * elements,
                    flops=(2 if case["kind"] == "norm" else 3) * elements)
    n, part, V, h = case["tokens"], _part(case), case["vocab"], case["hidden"]
    wide = 0 if case["kind"] == "ce" else case["teacher_hidden"] or h
    passes = {"none": 1, "x": 2, "both": 3}[case["grads"]]
    values = part * (h + wide) + V * (h + (wide if wide else 0))
    values += {"none": 0, "x": n * h, "both": (n + V) * h}[case["grads"]]
    return dict(bytes=2 * values + 8 * n + (4 * n if case["grads"] == "none" else 4),
                flops=2 * part * V * (passes * h + wide))


# ---- 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] in ("norm", "clip"):
        total = sum(torch.linalg.vector_norm(v.double()).item() ** 2 for v in s["grads"])
        norm = torch.tensor(math.sqrt(total), dtype=torch.float64, device="cuda")
        if s["kind"] == "norm":
            return norm
        factor = min(1.0, s["max_norm"] / (math.sqrt(total) + 1e-6))
        return norm, *[v.double() * factor for v in s["grads"]]
    with torch.no_grad():
        at = s["keep"].nonzero()[:, 0]
        x, w = s["x"].double(), s["weight"].double()
        loss = torch.zeros(x.shape[0], dtype=torch.float64, device="cuda")
        grad_x, grad_w = torch.zeros_like(x), torch.zeros_like(w)
        for rows in at.split(512):
            if s["kind"] == "ce":
                z = x[rows] @ w.T
                loss[rows] = torch.logsumexp(z, 1) - z[torch.arange(rows.numel()), s["labels"][rows]]
                dz = torch.softmax(z, 1)
                dz[torch.arange(rows.numel()), s["labels"][rows]] -= 1
            else:
                T = s["temperature"]
                q = torch.log_softmax(x[rows] @ w.T / T, 1)
                p = torch.log_softmax(s["teacher_x"][rows].double()
                                      @ s["teacher_weight"].double().T / T, 1)
                loss[rows] = (torch.exp(p) * (p - q)).sum(1)
                dz = (torch.exp(q) - torch.exp(p)) / T
            if s["grads"] != "none":
                grad_x[rows] = dz @ w / at.numel()
            if s["grads"] == "both":
                grad_w += dz.T @ x[rows] / at.numel()
    if s["grads"] == "none":
        return loss
    return loss.sum() / at.numel(), grad_x, *((grad_w,) if s["grads"] == "both" else ())
