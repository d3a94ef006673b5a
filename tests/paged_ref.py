"""Plain references of the paged-cache operators: Python integers for the scheduler step, 64 bits for
the cache write and the attention, with bounds for the kernels' rounding derived beside each."""
import math

import torch


def pages(n, P):
    return -(-n // P)


def step(lens, keep, new, table, free, count, P, rows, each=0):
    """paged_step on lists, literally: (slots, positions, starts, lens, count, table, free)."""
    table, free = [list(r) for r in table], list(free)
    W, F = len(table[0]) if table else 0, len(free)
    count = min(max(count, 0), F)
    kept = []
    for b, L in enumerate(lens):
        L = min(max(L, 0), W * P)
        k = L if keep is None else min(max(keep[b], 0), L)
        kept.append(k)
        for w in range(pages(k, P), pages(L, P)):
            if count < F:
                free[count] = table[b][w]
                count += 1
    slots, positions, starts, out = [-1] * rows, [0] * rows, [0], []
    for b, k in enumerate(kept):
        a = min(max(new[b], 0), each or rows - starts[-1])
        have = pages(k, P)
        while have < pages(min(k + a, W * P), P) and count > 0:
            count -= 1
            table[b][have] = free[count]
            have += 1
        out.append(min(k + a, W * P, have * P))
        for i in range(a):
            pos = k + i
            positions[starts[-1] + i] = pos
            if pos < out[b] and 0 <= table[b][pos // P] < F:
                slots[starts[-1] + i] = table[b][pos // P] * P + pos % P
        starts.append(starts[-1] + (each or a))
    return slots, positions, starts, out, count, table, free


def rope(x, weight, eps, cos, sin):
    """(y in 64 bits, a bound, |a| + |b| of its two products). The bound is for a kernel that computes in fp32 and rounds once to bf16): the sum of
    D squares and the factors of the norm are off by at most (D / 2 + 16) 2^-24 of a value (half of a
    sum's error passes the square root; 16 steps for everything else), which the rotation adds up over
    its two products; the last rounding is half a step of bf16, 2^-8 of the value."""
    x, D = x.double(), x.shape[-1]
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    a, b = x.chunk(2, -1)
    (ca, cb), (sa, sb) = cos.double()[:, None].chunk(2, -1), sin.double()[:, None].chunk(2, -1)
    y = torch.cat([a * ca - b * sa, b * cb + a * sb], -1)
    size = torch.cat([(a * ca).abs() + (b * sa).abs(), (b * cb).abs() + (a * sb).abs()], -1)
    return y, (D / 2 + 16) * 2.0 ** -24 * size + 2.0 ** -8 * y.abs(), size


def rows_of(k_cache, v_cache, table_row, n):
    """K and V [n, kv_heads, D] of the first n tokens of a request."""
    P, D = v_cache.shape[2:]
    t = torch.arange(n, device=v_cache.device)
    page, at = table_row.to(t.device).long()[t // P], t % P
    return (k_cache[page, :, :, at].reshape(n, v_cache.shape[1], D), v_cache[page, :, at])


def attend(q, k, v, scale):
    """One request: q [H, D], k, v [n, Hkv, D] -> (o, lse, bound of o, bound of lse) in 64 bits.

    A score of a kernel is off by at most e = scale D 2^-24 sum_d |q_d k_d| (D products, each exact in
    fp32, summed in any order) + 4 2^-24 |s| (the scaling), so a weight's ratio to another by 2 e. The
    weights enter their products as fp32 or as two bf16 pieces, which lose at most 2^-16 of them; their
    sums of n terms at most n 2^-24; exp and the rest 2^-18. So o is off by (2 e + 2^-15 + 2 n 2^-24)
    sum p |v|, and by half a step of bf16 (2^-8 of the value) in the end; lse by e + (n + 8) 2^-24 and
    4 2^-24 of itself."""
    H, D = q.shape
    n, Hkv = k.shape[:2]
    if n == 0:
        zero = torch.zeros(H, D, dtype=torch.float64, device=q.device)
        return zero, torch.full((H,), -math.inf, dtype=torch.float64, device=q.device), zero, zero[:, 0]
    o, lse, bo, bl = [], [], [], []
    for h in range(H):
        hk = h // (H // Hkv)
        qd, kd, vd = q[h].double(), k[:, hk].double(), v[:, hk].double()
        s = (kd * qd).sum(1) * scale
        e = (scale * D * 2.0 ** -24 * (kd * qd).abs().sum(1) + 4 * 2.0 ** -24 * s.abs()).max()
        p = torch.softmax(s, 0)
        o.append((p[:, None] * vd).sum(0))
        lse.append(torch.logsumexp(s, 0))
        size = (p[:, None] * vd.abs()).sum(0)
        bo.append((2 * e + 2.0 ** -15 + 2 * n * 2.0 ** -24) * size + 2.0 ** -8 * o[-1].abs())
        bl.append(e + (n + 8) * 2.0 ** -24 + 4 * 2.0 ** -24 * lse[-1].abs())
    return tuple(torch.stack(x) for x in (o, lse, bo, bl))
