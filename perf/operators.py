"""The operators of decoding over a paged key-value cache, as measurable cases.

  step       one scheduler step on the GPU: pages handed back and taken, block table, slot map and
             positions from the requests' lengths (ops.paged_step)
  write      a step's q, k, v rows: per-head norm and rotation at each token's position, q out, k and
             v into their slots of the cache (ops.paged_rope_write)
  attend     attention of one new token a request over its pages (ops.paged_attn)

The cache of one layer, with pages of P tokens:
  k_cache  bf16 [pages, kv heads, D / 8, P, 8]   value d of a token at [d // 8, token, d % 8]
  v_cache  bf16 [pages, kv heads, P, D]
  block_table int32 [B, W]: page w of request b holds its tokens w P .. w P + P - 1
  a slot is page * P + offset, -1 a token that is stored nowhere

Heads and widths are those of the decoder layer here (32 query and 8 kv heads of 128) and generic
ones of the same ranges.
"""
import math
import os
import sys

import torch

own = False

_ops = None


def _lib():
    """The framework's operators, imported at the first call that needs them."""
    global _ops
    if _ops is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "qwen-palettize_amd"))
        from palettize_hip import ops
        _ops = ops
    return _ops


# ---- the cases ------------------------------------------------------------------------------
def listed():
    return [
        # the first words of one chat: the smallest call, where latency counts
        dict(name="attend_b1_len37", kind="attend", B=1, longest=37, mixed=False, idle=0, heads=32,
             kv_heads=8, head_dim=128, page=64),
        # one request with a long document in its cache: all of the card for eight kv heads
        dict(name="attend_b1_len32768", kind="attend", B=1, longest=32768, mixed=False, idle=0,
             heads=32, kv_heads=8, head_dim=128, page=64),
        # an ordinary batch of chats of very different lengths
        dict(name="attend_b32_mix4096", kind="attend", B=32, longest=4096, mixed=True, idle=0,
             heads=32, kv_heads=8, head_dim=128, page=64),
        # a full batch of long contexts, the largest
        dict(name="attend_b64_len8192", kind="attend", B=64, longest=8192, mixed=False, idle=0,
             heads=32, kv_heads=8, head_dim=128, page=64),
        # a large batch of short chats on small pages, padded: every eighth row is empty
        dict(name="attend_b256_mix1024", kind="attend", B=256, longest=1024, mixed=True, idle=8,
             heads=32, kv_heads=8, head_dim=128, page=16),
        # a small model: heads of 64, seven query heads on a kv head, odd lengths
        dict(name="attend_b48_mix3001_d64", kind="attend", B=48, longest=3001, mixed=True, idle=0,
             heads=14, kv_heads=2, head_dim=64, page=32),
        # one decoded token of one request
        dict(name="write_t1", kind="write", tokens=1, dead=0, heads=32, kv_heads=8, head_dim=128,
             page=64, norm=True, fused=False),
        # the prompts of a batch of 32 x 512 tokens
        dict(name="write_t16384", kind="write", tokens=16384, dead=0, heads=32, kv_heads=8,
             head_dim=128, page=64, norm=True, fused=False),
        # a ragged prefill of a small model without per-head norms, q, k and v side by side in one
        # projection's output, the last rows of the buffer without a slot
        dict(name="write_t3001_d64", kind="write", tokens=3001, dead=37, heads=14, kv_heads=2,
             head_dim=64, page=32, norm=False, fused=True),
        # the step of a small decode batch: one token each
        dict(name="step_b8", kind="step", B=8, longest=2000, width=64, page=64, window=1, fresh=0,
             prompt=0, idle=0),
        # continuous batching: every sixteenth request has ended and its row takes a new prompt,
        # the others one token, every ninth row idle
        dict(name="step_b256_mix", kind="step", B=256, longest=4000, width=128, page=64, window=1,
             fresh=16, prompt=2048, idle=9),
        # the first step of a batch: every row a new prompt, small pages
        dict(name="step_b32_prompts", kind="step", B=32, longest=0, width=512, page=16, window=1,
             fresh=1, prompt=8000, idle=0),
    ]


def _log(rng, lo, hi):
    """A whole number whose logarithm is uniform over lo..hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    """(query heads, kv heads, head dim) of the layer here, or generic ones."""
    if rng.random() < 0.5:
        return 32, 8, 128
    kv = rng.choice((1, 2, 3, 4, 8))
    return kv * rng.choice((1, 2, 4, 5, 7, 8, 16, 20)), kv, rng.choice((64, 128, 128, 256))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "write", "write", "step"))
    page = rng.choice((16, 32, 64, 64, 128))
    if kind == "step":
        width = 16384 // page
        fresh = rng.choice((0, 1, 4, 16))
        B = _log(rng, 1, 32 if fresh == 1 else 1024)
        return dict(kind="step", B=B, longest=_log(rng, 16, 8000), width=width, page=page,
                    window=rng.choice((1, 1, 2, 5)), fresh=fresh,
                    prompt=_log(rng, 16, 8000 if B <= 64 else 1024) if fresh else 0,
                    idle=rng.choice((0, 0, 5)))
    heads, kv, dim = _heads(rng)
    if kind == "write":
        most = min(16384, 16384 * 48 * 128 // ((heads + 2 * kv) * dim))
        return dict(kind="write", tokens=_log(rng, 1, most), dead=rng.choice((0, 0, 3, 64)),
                    heads=heads, kv_heads=kv, head_dim=dim, page=page, norm=rng.random() < 0.7,
                    fused=rng.random() < 0.5)
    B = _log(rng, 1, 256)
    # no more cached values, and no more products, than the largest listed case
    most = min(32768, 64 * 8192 * 8 * 128 // (B * max(kv, -(-heads // 4)) * dim))
    return dict(kind="attend", B=B, longest=_log(rng, 1, most), mixed=rng.random() < 0.6,
                idle=rng.choice((0, 0, 4)), heads=heads, kv_heads=kv, head_dim=dim, page=page)


# ---- the inputs -------------------------------------------------------------------------------
def _spread(n, longest):
    """n lengths spread over 1..longest by their logarithm, the longest among them."""
    return [max(1, round(math.exp((i + 1) / n * math.log(max(longest, 1))))) for i in range(n)]


def _lengths(case):
    """The cached tokens of an attend case's rows (in an order of their own, not the seed's)."""
    B = case["B"]
    lens = _spread(B, case["longest"]) if case["mixed"] else [case["longest"]] * B
    return [0 if case["idle"] and b % case["idle"] == case["idle"] - 1 else lens[b]
            for b in range(B)]


def _rows(case):
    """(cached, kept, new) tokens of a step case's rows: fresh rows drop what they had and take a
    prompt, idle rows are empty, the others take a window of tokens (a window over one token follows
    a guess of which the last ones were wrong: those are dropped first)."""
    B, f, idle = case["B"], case["fresh"], case["idle"]
    cached = _spread(B, case["longest"]) if case["longest"] else [0] * B
    prompts = _spread(B, case["prompt"]) if f else [0] * B
    rows = []
    for b in range(B):
        if idle and b % idle == idle - 1:
            rows.append((0, 0, 0))
        elif f and b % f == f - 1:
            rows.append((cached[b], 0, prompts[b]))
        else:
            rows.append((cached[b], max(0, cached[b] - b % case["window"]), case["window"]))
    return rows


def _pages(n, page):
    return -(-n // page)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16)


def _tables(tokens, dim):
    """cos and sin of the rotation, fp32 [tokens, dim], theta 1e6."""
    inv = 1e6 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    angle = torch.outer(torch.arange(tokens, device="cuda", dtype=torch.float64), inv)
    angle = torch.cat([angle, angle], -1)
    return angle.cos().float(), angle.sin().float()


def _block_table(lens, page, width, order):
    """The block table of rows that hold lens tokens, their pages taken from `order` one after
    another (unused entries 0), and how many pages that took."""
    n = torch.tensor([_pages(x, page) for x in lens], device="cuda")
    end = n.cumsum(0)
    w = torch.arange(width, device="cuda")
    at = (end - n)[:, None] + w
    table = torch.where(w < n[:, None], order[at.clamp(max=order.numel() - 1)], 0)
    return table.to(torch.int32), int(end[-1])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "step":
        rows = _rows(case)
        B, P, W = case["B"], case["page"], case["width"]
        held = sum(_pages(c, P) for c, _, _ in rows)
        total = sum(n for _, _, n in rows)
        F = held + sum(_pages(k + n, P) for _, k, n in rows) + 8
        order = torch.randperm(F, generator=g, device="cuda")
        mixed = torch.randperm(B, generator=g, device="cuda")
        cached, keep, new = (torch.tensor(v, device="cuda", dtype=torch.int32)[mixed]
                             for v in zip(*rows))
        table, used = _block_table(cached.tolist(), P, W, order)
        free = torch.cat([order[used:], order.new_zeros(used)]).to(torch.int32)
        return dict(kind="step", lens=cached, keep=keep, new=new, table=table, free=free, page=P,
                    count=torch.tensor([F - used], device="cuda", dtype=torch.int32),
                    # the buffer of token rows that such a program keeps, in steps of 64
                    rows=-(-max(total, 1) // 64) * 64)
    H, Hkv, D, P = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    if case["kind"] == "write":
        T, live = case["tokens"], max(1, case["tokens"] - case["dead"])
        pages = _pages(live, P) + 3
        order = torch.randperm(pages, generator=g, device="cuda")
        # requests of up to 512 tokens one after another, each at positions of its own
        t = torch.arange(T, device="cuda")
        first = torch.randint(0, 3500, (T // 512 + 1,), generator=g, device="cuda")
        pos = torch.where(t < live, first[t // 512] + t % 512, 0).to(torch.int32)
        slots = torch.where(t < live, order[(t // P).clamp(max=pages - 1)] * P + t % P, -1)
        if case["fused"]:
            qkv = _normal(g, T, (H + 2 * Hkv) * D)
            q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([H * D, Hkv * D, Hkv * D], 1))
        else:
            q, k, v = (_normal(g, T, h, D) for h in (H, Hkv, Hkv))
        qw, kw = ((1 + 0.2 * _normal(g, D) if case["norm"] else None) for _ in range(2))
        cos, sin = _tables(4096, D)
        return dict(kind="write", q=q, k=k, v=v, qw=qw, kw=kw, cos=cos, sin=sin, pos=pos,
                    slots=slots.to(torch.int32), eps=1e-6,
                    kc=torch.zeros(pages, Hkv, D // 8, P, 8, device="cuda", dtype=torch.bfloat16),
                    vc=torch.zeros(pages, Hkv, P, D, device="cuda", dtype=torch.bfloat16))
    lens = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
    lens = lens[torch.randperm(case["B"], generator=g, device="cuda")]
    W = _pages(case["longest"], P)
    n = sum(_pages(x, P) for x in lens.tolist()) + 3
    order = torch.randperm(n, generator=g, device="cuda")
    table, _ = _block_table(lens.tolist(), P, W, order)
    # queries a little longer than a norm leaves them: a softmax with some weight on few tokens
    return dict(kind="attend", q=1.5 * _normal(g, case["B"], H, D), lens=lens, table=table,
                kc=_normal(g, n, Hkv, D // 8, P, 8), vc=_normal(g, n, Hkv, P, D))


# ---- the plain forms ----------------------------------------------------------------------------
def _step(s):
    P, B, W, F, rows = s["page"], s["lens"].numel(), s["table"].shape[1], s["free"].numel(), s["rows"]
    table, free = s["table"], s["free"]
    cached = s["lens"].long().clamp(0, W * P)
    keep = torch.minimum(s["keep"].long().clamp(min=0), cached)
    ends = s["new"].long().clamp(min=0).cumsum(0).clamp(max=rows)
    starts = torch.cat([ends.new_zeros(1), ends])
    new = ends - starts[:-1]
    have, hold = (cached + P - 1) // P, (keep + P - 1) // P
    w = torch.arange(W, device=table.device)
    # pages handed back: onto the stack, in order of the rows
    back = have - hold
    count = s["count"].long().clamp(0, F)
    at = count + (back.cumsum(0) - back)[:, None] + (w - hold[:, None])
    gone = (w >= hold[:, None]) & (w < have[:, None]) & (at < F)
    stack = torch.cat([free, free.new_zeros(1)])
    stack.scatter_(0, torch.where(gone, at, F).flatten(), table.flatten())
    pool = (count + back.sum()).clamp(max=F)
    # pages taken: off the stack's top, in order of the rows, while they last
    want = (torch.minimum(keep + new, keep.new_tensor(W * P)) + P - 1) // P - hold
    want = want.clamp(min=0)
    before = want.cumsum(0) - want
    given = torch.minimum((pool - before).clamp(min=0), want)
    top = pool - 1 - before[:, None] - (w - hold[:, None])
    taken = (w >= hold[:, None]) & (w < (hold + given)[:, None])
    table.copy_(torch.where(taken, stack[top.clamp(0, F)], table))
    free.copy_(stack[:F])
    lens = torch.minimum(keep + new, (hold + given) * P)
    # the tokens' rows
    t = torch.arange(rows, device=table.device)
    b = torch.searchsorted(ends, t, right=True).clamp(max=B - 1)
    live = t < ends[-1]
    pos = torch.where(live, keep[b] + t - starts[b], 0)
    page = table[b, (pos // P).clamp(max=W - 1)].long()
    stored = live & (pos < lens[b]) & (page >= 0) & (page < F)
    slots = torch.where(stored, page * P + pos % P, -1)
    return (slots.int(), pos.int(), starts.int(), lens.int(),
            (pool - torch.minimum(pool, want.sum())).int(), table, free)


def _rope(x, weight, eps, cos, sin):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()
    half = x.shape[-1] // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    return (x * cos[:, None] + turned * sin[:, None]).to(torch.bfloat16)


def _write(s):
    pos, P = s["pos"].long(), s["vc"].shape[2]
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rope(s["q"], s["qw"], s["eps"], cos, sin)
    k = _rope(s["k"], s["kw"], s["eps"], cos, sin)
    live = s["slots"] >= 0
    slot = s["slots"][live].long()
    page, at = slot // P, slot % P
    s["kc"][page, :, :, at] = k[live].unflatten(-1, (-1, 8))
    s["vc"][page, :, at] = s["v"][live]
    return q, s["kc"], s["vc"]


def _attend(s):
    q, kc, vc, lens = s["q"], s["kc"], s["vc"], s["lens"]
    (B, H, D), (_, Hkv, _, P, _) = q.shape, kc.shape
    N = s["table"].shape[1] * P
    pages = s["table"].long()
    k = kc[pages].permute(0, 2, 3, 5, 1, 4).float().reshape(B, Hkv, D, N)
    v = vc[pages].permute(0, 2, 1, 3, 4).float().reshape(B, Hkv, N, D)
    score = (q.float().view(B, Hkv, H // Hkv, D) * D ** -0.5) @ k
    dead = torch.arange(N, device=q.device) >= lens[:, None]
    score = score.masked_fill(dead[:, None, None], -math.inf)
    empty = (lens == 0)[:, None, None, None]
    top = score.amax(-1, keepdim=True).masked_fill(empty, 0)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = ((p @ v) / total).masked_fill(empty, 0)
    lse = top + torch.log(total)
    return o.reshape(B, H, D).to(torch.bfloat16), lse.reshape(B, H)


# ---- one pass -------------------------------------------------------------------------------------
def run(s):
    if s["kind"] == "step":
        if own:
            slots, pos, starts, lens, count = _lib().paged_step(
                s["lens"], s["new"], s["table"], s["free"], s["count"], s["page"], keep=s["keep"],
                rows=s["rows"])
            return slots, pos, starts, lens, count, s["table"], s["free"]
        return _step(s)
    if s["kind"] == "write":
        if own:
            q = _lib().paged_rope_write(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["pos"],
                                        s["slots"], s["kc"], s["vc"], s["qw"], s["kw"], s["eps"])
            return q, s["kc"], s["vc"]
        return _write(s)
    if own:
        return _lib().paged_attn(s["q"], s["kc"], s["vc"], s["table"], s["lens"])
    return _attend(s)


def work(case):
    if case["kind"] == "step":
        rows, P = _rows(case), case["page"]
        moved = sum(_pages(c, P) - 2 * _pages(k, P) + _pages(k + n, P) for c, k, n in rows)
        total = sum(n for _, _, n in rows)
        # lens, keep, new in, starts, lens out; slot and position a token; each page that changes
        # hands read once and written once
        return dict(bytes=20 * len(rows) + 8 * total + 8 * moved, flops=0)
    H, Hkv, D = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "write":
        T, live = case["tokens"], max(1, case["tokens"] - case["dead"])
        elements = T * H * D + 2 * live * Hkv * D
        # a rotation row is read once for each of at most 4096 positions
        return dict(bytes=4 * elements + 8 * T + 8 * D * min(T, 4096),
                    flops=(10 if case["norm"] else 6) * (T * H + live * Hkv) * D)
    lens = _lengths(case)
    tokens = sum(lens)
    return dict(bytes=4 * tokens * Hkv * D + 4 * len(lens) * H * D + 4 * len(lens) * H
                + 4 * sum(_pages(n, case["page"]) for n in lens) + 4 * len(lens),
                flops=4 * tokens * H * D)


# ---- 64 bits ------------------------------------------------------------------------------------------
def _exact_rope(x, weight, eps, cos, sin):
    """The rotation of (x_j, x_{j + D/2}) as a plane turned by the tables' angle."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + eps) * weight.double()
    a, b = x.chunk(2, -1)
    (ca, cb), (sa, sb) = cos.double()[:, None].chunk(2, -1), sin.double()[:, None].chunk(2, -1)
    return torch.cat([a * ca - b * sa, b * cb + a * sb], -1)


def exact(case, seed):
    if case["kind"] == "step":
        return None  # whole numbers: the plain form's are the values
    s = prepare(case, seed)
    if case["kind"] == "write":
        T, Hkv, D = s["k"].shape
        P, pages = s["vc"].shape[2], s["vc"].shape[0]
        cos, sin = s["cos"].index_select(0, s["pos"]), s["sin"].index_select(0, s["pos"])
        # by token first, then into the cache's order
        live = s["slots"] >= 0
        k = torch.zeros(pages * P, Hkv, D, device="cuda", dtype=torch.float64)
        v = torch.zeros_like(k)
        k.index_copy_(0, s["slots"][live].long(), _exact_rope(s["k"], s["kw"], s["eps"], cos, sin)[live])
        v.index_copy_(0, s["slots"][live].long(), s["v"][live].double())
        k = k.view(pages, P, Hkv, D // 8, 8).permute(0, 2, 3, 1, 4)
        return (_exact_rope(s["q"], s["qw"], s["eps"], cos, sin), k,
                v.view(pages, P, Hkv, D).transpose(1, 2))
    B, H, D = s["q"].shape
    Hkv, P = s["vc"].shape[1], s["vc"].shape[2]
    o = torch.zeros(B, H, D, device="cuda", dtype=torch.float64)
    lse = torch.full((B, H), -math.inf, device="cuda", dtype=torch.float64)
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        t = torch.arange(n, device="cuda")
        page, at = s["table"][b].long()[t // P], t % P
        for h in range(Hkv):
            q = s["q"][b].view(Hkv, -1, D)[h].double()
            k = s["kc"][page, h, :, at].reshape(n, D).double()
            score = (k @ q.T) / math.sqrt(D)
            lse[b].view(Hkv, -1)[h] = torch.logsumexp(score, 0)
            weight = torch.softmax(score, 0).T.contiguous()
            o[b].view(Hkv, -1, D)[h] = weight @ s["vc"][page, h, at].double()
    return o, lse
