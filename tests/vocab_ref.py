"""The losses over a vocabulary in 64 bits, from their definitions, with bounds of what bf16 and fp32
arithmetic may leave: every sum of n fp32 terms is off by at most n 2^-24 of the sum of their
magnitudes, a rounding to bf16 by 2^-8 of the value (half a step of 2^-7)."""
import torch

U32, U16 = 2.0 ** -24, 2.0 ** -8


def logits(x, w, T=1.0):
    """(z, bound of an fp32 z's error) of x w^T / T."""
    x, w = x.double(), w.double()
    mag = x.abs() @ w.abs().T / T
    return x @ w.T / T, (x.shape[1] + 4) * U32 * mag


def reference(x, w, labels=None, ignore_index=-100, tx=None, tw=None, mask=None, T=1.0,
              reduction="mean", upstream=None, kept=None, top=False):
    """A dict of the loss and gradients of `reduction` in 64 bits and the bounds of their errors
    (loss_tol, gx_tol, gw_tol), and every row's loss (rows, rows_tol). upstream: the gradient of the
    loss, a number or one of every row. kept: the gradient is of a cross entropy that kept its
    exponentials in fp16, relative to the greatest of 256 words (a sum or mean of linear_cross_entropy).
    top: the greatest gradient of each row's logits is in two bf16."""
    kept = labels is not None and reduction != "none" if kept is None else kept
    N, V = x.shape[0], w.shape[0]
    dev = x.device
    keep = (labels != ignore_index) if labels is not None else (
        mask if mask is not None else torch.ones(N, dtype=torch.bool, device=dev))
    at = keep.nonzero()[:, 0]
    rows, rows_tol = (torch.zeros(N, dtype=torch.float64, device=dev) for _ in range(2))
    gx, gx_tol = (torch.zeros(x.shape, dtype=torch.float64, device=dev) for _ in range(2))
    gw, gw_tol = (torch.zeros(w.shape, dtype=torch.float64, device=dev) for _ in range(2))
    n = max(1, at.numel())
    if reduction == "none":
        g = (torch.ones(N, device=dev) if upstream is None else upstream).double()
    else:
        one = 1.0 if upstream is None else float(upstream)
        g = torch.full((N,), one / (n if reduction == "mean" else 1), dtype=torch.float64, device=dev)
    # a sum of exponentials: 16 words in one register block, then joins over blocks, waves, tiles and
    # threads, each of a few roundings, and exponentials of one step (2^-23)
    steps = (64 + 8 * 8 + 8 * (V // 256 + 1) + 4) * U32
    for r in at.split(1024):
        z, dz = logits(x[r], w, T)
        lse = torch.logsumexp(z, 1)
        off = dz.max(1).values + steps  # of a normaliser
        q = torch.softmax(z, 1)
        # a probability: its logit's and normaliser's errors, the argument's rounding (both are rounded
        # values of their own size) and the exponential's
        q_tol = q * (dz + off[:, None] + 4 * U32 * (z.abs() + lse.abs()[:, None] + 4))
        if labels is not None:
            l = labels[r].long()
            i = torch.arange(r.numel(), device=dev)
            rows[r] = lse - z[i, l]
            rows_tol[r] = off + dz[i, l] + 4 * U32 * (lse.abs() + z[i, l].abs())
            d = q.clone()
            d[i, l] -= 1
            if kept:  # half a step of fp16, or of its subnormals (of 2^15 times the value)
                q_tol = q_tol + 2.0 ** -11 * q + 2.0 ** -40 * q.max(1, keepdim=True).values
        else:
            zt, dzt = logits(tx[r], tw, T)
            lt = torch.logsumexp(zt, 1)
            p = torch.softmax(zt, 1)
            off_t = dzt.max(1).values + steps
            rows[r] = (p * (torch.log_softmax(zt, 1) - torch.log_softmax(z, 1))).sum(1)
            far = (zt - z).abs()
            rows_tol[r] = ((p * (dz + dzt + far * 2 * (off_t[:, None] + steps))).sum(1) + off + off_t
                           + 8 * U32 * (far.max(1).values + 4))
            q_tol = q_tol + p * (dzt + off_t[:, None] + 4 * U32 * (zt.abs() + lt.abs()[:, None] + 4))
            d = (q - p) / T
            q_tol = q_tol / T
        d, q_tol = d * g[r][:, None], q_tol * g[r][:, None].abs()
        # rounded to bf16 (a value below the type's range, 2^-133, is not met), of up to 128 rows to two,
        # then fp32 sums
        part = torch.full_like(d, U16 * U16 if N <= 128 else U16)
        if top:
            part.scatter_(1, d.abs().argmax(1, keepdim=True), U16 * U16)
        d_tol = part * d.abs() + 2 * q_tol + 8 * U32 * d.abs()
        gx[r] = d @ w.double()
        gx_tol[r] = (d_tol + (V + 64) * U32 * d.abs()) @ w.double().abs()
        gw += d.T @ x[r].double()
        gw_tol += (d_tol + (N + 64) * U32 * d.abs()).T @ x[r].double().abs()
    # rounded to bf16; a sum's or mean's that the forward computed is multiplied by an upstream gradient
    # afterwards and rounded once more: r(r(g) u) is off by (1 + 2^-8)^2 - 1 = 2 * 2^-8 + 2^-16 of g u
    last = U16 if upstream is None or reduction == "none" else 2 * U16 + U16 * U16
    gx_tol += (last + 4 * U32) * (gx.abs() + gx_tol)
    gw_tol += (last + 4 * U32) * (gw.abs() + gw_tol)
    loss, tol = rows, rows_tol
    if reduction != "none":
        k = n if reduction == "mean" else 1
        loss, tol = rows.sum() / k, rows_tol.sum() / k + 2 * U32 * rows.sum().abs() / k
    return dict(loss=loss, loss_tol=tol + 2 * U32 * loss.abs(), rows=rows, rows_tol=rows_tol, gx=gx,
                gx_tol=gx_tol, gw=gw, gw_tol=gw_tol, keep=keep)


def inputs(N, V, H, seed=0, ignored=0.0, dtype=torch.int64, device="cuda", lean=2.0):
    """x, w, labels: logits of a spread of about 2.5, some rows close to their label."""
    g = torch.Generator(device=device).manual_seed(seed)
    w = (torch.randn(V, H, generator=g, device=device) * (2.5 * H ** -0.5)).bfloat16()
    labels = torch.randint(0, V, (N,), generator=g, device=device)
    x = torch.randn(N, H, generator=g, device=device)
    x = x + lean * torch.rand(N, 1, generator=g, device=device) * w[labels].float()
    if ignored:
        labels[torch.rand(N, generator=g, device=device) < ignored] = -100
    return x.bfloat16(), w, labels.to(dtype)


def close(got, want, tol, what):
    """got within tol of want, element by element; NaN and infinities are not close."""
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    if bool(bad.any()):
        i = int(bad.flatten().nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: "
                             f"{float(got.flatten()[i])} for {float(want.flatten()[i])}, "
                             f"may be off by {float(tol.flatten()[i])}")
