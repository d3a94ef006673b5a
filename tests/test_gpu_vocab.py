"""Losses over a large vocabulary against their definitions in 64 bits (GPU)."""
import pytest
import torch

from vocab_ref import close, inputs, logits, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu(dev):
    pass


@pytest.fixture(scope="module")
def F():
    from palettize_hip import functional
    return functional


@pytest.fixture(scope="module")
def ops():
    from palettize_hip import ops
    return ops


SIZES = [(1, 1, 8), (1, 5, 8), (2, 256, 64), (3, 257, 72), (17, 1000, 128), (64, 1003, 200),
         (255, 511, 64), (256, 512, 256), (257, 2049, 136), (300, 4099, 1000), (777, 3001, 512)]


def run_ce(F, x, w, labels, reduction="mean", upstream=None, **kw):
    x, w = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    loss = F.linear_cross_entropy(x, w, labels, reduction=reduction, **kw)
    g = None if upstream is None and reduction != "none" else (
        torch.ones_like(loss) if upstream is None else
        torch.as_tensor(upstream, dtype=torch.float32, device=loss.device).reshape(loss.shape))
    return (loss.detach(), *torch.autograd.grad(loss, (x, w), g))


def check(got, ref):
    loss, gx, gw = got
    assert loss.dtype == torch.float32 and gx.dtype == gw.dtype == torch.bfloat16
    close(loss, ref["loss"], ref["loss_tol"], "loss")
    close(gx, ref["gx"], ref["gx_tol"], "grad_x")
    close(gw, ref["gw"], ref["gw_tol"], "grad_weight")
    assert not gx[~ref["keep"]].any()


@pytest.mark.parametrize("N,V,H", SIZES)
@pytest.mark.parametrize("ignored", [0.0, 0.5])
def test_ce_mean(F, N, V, H, ignored):
    x, w, labels = inputs(N, V, H, seed=N + V, ignored=ignored)
    check(run_ce(F, x, w, labels), reference(x, w, labels))


@pytest.mark.parametrize("N,V,H", [(17, 1000, 128), (300, 777, 72)])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("reduction,upstream", [("sum", None), ("sum", 0.37), ("mean", -3.0), ("none", None)])
def test_ce_reductions(F, N, V, H, dtype, reduction, upstream):
    x, w, labels = inputs(N, V, H, seed=1, ignored=0.3, dtype=dtype)
    check(run_ce(F, x, w, labels, reduction, upstream),
          reference(x, w, labels, reduction=reduction, upstream=upstream))


def test_ce_upstream_of_every_row(F):
    x, w, labels = inputs(130, 900, 96, seed=2, ignored=0.2)
    up = torch.randn(130, device="cuda")
    up[5] = 0
    check(run_ce(F, x, w, labels, "none", up), reference(x, w, labels, reduction="none", upstream=up))


def run_kl(F, x, w, tx, tw, reduction="mean", upstream=None, **kw):
    x, w = x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    loss = F.linear_distill(x, w, tx, tw, reduction=reduction, **kw)
    g = None if reduction != "none" else torch.ones_like(loss) if upstream is None else upstream
    return (loss.detach(), *torch.autograd.grad(loss, (x, w), g))


def kl_inputs(N, V, H, Ht, seed, ignored):
    x, w, labels = inputs(N, V, H, seed=seed, ignored=ignored)
    if Ht:
        tx, tw, _ = inputs(N, V, Ht, seed=seed + 1)
    else:
        tx, tw = (x.float() + 0.3 * torch.randn(N, H, device="cuda")).bfloat16(), w
    return x, w, tx, tw, (labels != -100) if ignored else None


@pytest.mark.parametrize("N,V,H", SIZES)
@pytest.mark.parametrize("Ht,ignored,T", [(0, 0.0, 1.0), (72, 0.4, 2.0), (640, 0.0, 0.7)])
def test_kl_mean(F, N, V, H, Ht, ignored, T):
    x, w, tx, tw, mask = kl_inputs(N, V, H, Ht, N + V, ignored)
    check(run_kl(F, x, w, tx, tw, mask=mask, temperature=T),
          reference(x, w, tx=tx, tw=tw, mask=mask, T=T))


@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_kl_reductions(F, reduction):
    x, w, tx, tw, mask = kl_inputs(150, 1030, 128, 0, 7, 0.3)
    up = torch.randn(150, device="cuda") if reduction == "none" else None
    check(run_kl(F, x, w, tx, tw, reduction, up, mask=mask),
          reference(x, w, tx=tx, tw=tw, mask=mask, reduction=reduction, upstream=up))


def test_kl_of_itself_is_zero(F):
    x, w, _ = inputs(70, 3000, 256, seed=3)
    loss, gx, gw = run_kl(F, x, w, x, w, "none")
    # both sides' sums are the same instructions on the same values
    assert float(loss.abs().max()) == 0 and not gx.any() and not gw.any()


# ---- forward and backward as two calls, which compute the logits twice ----------------------------------
def two_calls_ce(ops, x, w, labels, reduction="mean", upstream=1.0):
    _, lse, total = ops.linear_ce_fwd(x, w, labels)
    grad = torch.tensor([upstream], device="cuda")
    return (total[0 if reduction == "sum" else 1], *ops.linear_ce_bwd(x, w, labels, lse, grad, reduction))


def two_calls_kl(ops, x, w, tx, tw, mask=None, T=1.0, reduction="mean"):
    _, lse, total = ops.linear_kl_fwd(x, w, tx, tw, mask, T)
    grad = torch.ones(1, device="cuda")
    return (total[0 if reduction == "sum" else 1],
            *ops.linear_kl_bwd(x, w, tx, tw, lse, grad, reduction, mask, T))


@pytest.mark.parametrize("N,V,H", SIZES)
def test_two_calls(ops, N, V, H):
    x, w, labels = inputs(N, V, H, seed=N + V, ignored=0.3)
    check(two_calls_ce(ops, x, w, labels), reference(x, w, labels, kept=False))
    check(two_calls_ce(ops, x, w, labels, "sum", -0.7),
          reference(x, w, labels, reduction="sum", upstream=-0.7, kept=False))
    x, w, tx, tw, mask = kl_inputs(N, V, H, 136, N + V, 0.3)
    check(two_calls_kl(ops, x, w, tx, tw, mask, 1.5),
          reference(x, w, tx=tx, tw=tw, mask=mask, T=1.5))


@pytest.mark.parametrize("kind", ["ce", "kl"])
def test_two_calls_over_pieces(ops, kind):
    """More words than a piece of the backward holds for so many rows, and the last piece odd."""
    x, w, labels = inputs(16384, 33333, 64, seed=12, ignored=0.1)
    if kind == "ce":
        check(two_calls_ce(ops, x, w, labels), reference(x, w, labels, kept=False))
    else:
        tx, mask = (x.float() * 0.8).bfloat16(), labels != -100
        check(two_calls_kl(ops, x, w, tx, w, mask), reference(x, w, tx=tx, tw=w, mask=mask))


@pytest.mark.parametrize("kind", ["ce", "kl"])
def test_second_backward(F, kind):
    """The first backward hands over what the forward computed; another one computes it again."""
    x, w, labels = inputs(200, 1500, 128, seed=20, ignored=0.2)
    tx, tw, _ = inputs(200, 1500, 72, seed=21)
    x.requires_grad_(), w.requires_grad_()
    if kind == "ce":
        loss, ref = F.linear_cross_entropy(x, w, labels), dict(labels=labels)
    else:
        loss, ref = F.linear_distill(x, w, tx, tw), dict(tx=tx, tw=tw)
    for g in (1.0, -0.6, 2.0):
        got = torch.autograd.grad(loss, (x, w), torch.tensor(g, device="cuda"), retain_graph=True)
        want = reference(x.detach(), w.detach(), upstream=g, **ref)
        # a factor other than 1 rounds what the first one hands over again
        for a, n in zip(got, ("gx", "gw")):
            close(a, want[n], want[n + "_tol"] + 2.0 ** -8 * 1.01 * want[n].abs(), n)
    loss.backward(retain_graph=True)
    first = x.grad.clone()
    loss.backward()
    close(x.grad, 2 * first.double(), 2.0 ** -7 * first.double().abs() + 1e-30, "accumulated")


def test_gradients_that_a_step_leaves_out(F):
    x, w, labels = inputs(150, 700, 64, seed=22, ignored=0.2)
    want = run_ce(F, x, w, labels)
    for wants_x in (True, False):
        xs, ws = x.detach().clone().requires_grad_(wants_x), w.detach().clone().requires_grad_(not wants_x)
        loss = F.linear_cross_entropy(xs, ws, labels)
        loss.backward()
        assert torch.equal(loss, want[0])
        assert (ws if wants_x else xs).grad is None
        assert torch.equal((xs if wants_x else ws).grad, want[1 if wants_x else 2])
    with torch.no_grad():
        assert torch.equal(F.linear_cross_entropy(xs, ws, labels), want[0])


@pytest.mark.parametrize("kind", ["ce", "kl"])
def test_step_captured_and_replayed(ops, kind):
    N, V, H = 300, 3001, 136
    x, w, labels = inputs(N, V, H, seed=23)
    tx = torch.zeros_like(x)
    mask = torch.ones(N, dtype=torch.bool, device="cuda")
    up = torch.ones(1, device="cuda")

    def step():
        out = (ops.linear_ce_step(x, w, labels) if kind == "ce" else
               ops.linear_kl_step(x, w, tx, w, mask=mask))
        ops.scale_grads(out[3:], up)
        return out

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        nx, _, nl = inputs(N, V, H, seed=30 + seed, ignored=0.25 * seed)
        x.copy_(nx)
        labels.copy_(nl)
        mask.copy_(nl != -100)
        tx.copy_(nx.flip(0))
        up.fill_(1.0 + seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


# ---- more tiles than a CU has workgroups for: 256 x 256 of them ------------------------------------------
WIDE = [(300, 40001, 136), (129, 70000, 72), (257, 33000, 64), (700, 17003, 200), (1025, 15000, 576)]


@pytest.mark.parametrize("N,V,H", WIDE)
def test_wide_ce(F, ops, N, V, H):
    x, w, labels = inputs(N, V, H, seed=N, ignored=0.2)
    check(run_ce(F, x, w, labels), reference(x, w, labels))
    check(run_ce(F, x, w, labels, "none"), reference(x, w, labels, reduction="none"))
    check(two_calls_ce(ops, x, w, labels), reference(x, w, labels, kept=False))


@pytest.mark.parametrize("N,V,H", WIDE)
@pytest.mark.parametrize("Ht", [64, 328])
def test_wide_kl(F, N, V, H, Ht):
    x, w, tx, tw, mask = kl_inputs(N, V, H, Ht, N, 0.2)
    check(run_kl(F, x, w, tx, tw, mask=mask, temperature=1.3),
          reference(x, w, tx=tx, tw=tw, mask=mask, T=1.3))
    check(run_kl(F, x, w, tx, tw, "none", mask=mask),
          reference(x, w, tx=tx, tw=tw, mask=mask, reduction="none"))


# ---- what takes no part -------------------------------------------------------------------------------
@pytest.mark.parametrize("N", [1, 40, 300])
def test_ce_no_row_takes_part(F, N):
    x, w, labels = inputs(N, 700, 64)
    labels[:] = -100
    for reduction in ("mean", "sum", "none"):
        loss, gx, gw = run_ce(F, x, w, labels, reduction)
        assert not loss.any() and not gx.any() and not gw.any()


def test_no_rows(F):
    x, w, labels = inputs(0, 700, 64)
    for reduction in ("mean", "sum"):
        loss, gx, gw = run_ce(F, x, w, labels, reduction)
        assert float(loss) == 0 and gx.shape == (0, 64) and not gw.any()
    loss, gx, gw = run_ce(F, x, w, labels, "none")
    assert loss.shape == (0,) and not gw.any()
    loss, gx, gw = run_kl(F, x, w, x, w)
    assert float(loss) == 0 and not gw.any()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_rows_without_part_may_hold_anything(F, value):
    x, w, labels = inputs(333, 1500, 136, seed=5, ignored=0.4)
    want = run_ce(F, x, w, labels)
    bad = x.clone()
    bad[labels == -100] = value
    for a, b in zip(run_ce(F, bad, w, labels), want):
        assert torch.equal(a, b)
    mask = labels != -100
    tx = (x.float() * 0.9).bfloat16()
    want = run_kl(F, x, w, tx, w, mask=mask)
    tbad = tx.clone()
    tbad[~mask] = value
    for a, b in zip(run_kl(F, bad, w, tbad, w, mask=mask), want):
        assert torch.equal(a, b)


def test_another_ignore_index(F):
    x, w, labels = inputs(90, 300, 64, seed=6)
    labels[::3] = 7
    check(run_ce(F, x, w, labels, ignore_index=7), reference(x, w, labels, ignore_index=7))


@pytest.mark.parametrize("bad", [-1, 300, 2 ** 31, 2 ** 40, -2 ** 33])
def test_labels_outside_the_vocabulary_are_nan(F, bad):
    x, w, labels = inputs(90, 300, 64, seed=6)
    want = run_ce(F, x, w, labels, "none")
    labels[17] = bad
    loss, gx, gw = run_ce(F, x, w, labels, "none")
    others = torch.arange(90, device="cuda") != 17
    assert torch.isnan(loss[17]) and torch.equal(loss[others], want[0][others])
    assert torch.isnan(gx[17]).all() and torch.equal(gx[others], want[1][others])
    assert torch.isnan(gw).all()
    assert torch.isnan(run_ce(F, x, w, labels)[0])


# ---- extreme values -------------------------------------------------------------------------------------
@pytest.mark.parametrize("shift", [60.0, -60.0, 3000.0])
def test_far_logits(F, shift):
    """All logits of a row moved by the same amount, far past what exp takes by itself."""
    x, w, labels = inputs(64, 1000, 128, seed=8)
    x[:, -8:] = 1.0
    w[:, -8:] = shift / 8
    check(run_ce(F, x, w, labels), reference(x, w, labels))


def test_one_word_holds_all(F):
    x, w, labels = inputs(64, 1000, 128, seed=9, lean=60.0)
    check(run_ce(F, x, w, labels), reference(x, w, labels))


def test_a_word_that_cannot_be(F):
    """Logits of minus infinity: no weight, finite loss for the other words' rows."""
    x, w, labels = inputs(40, 520, 64, seed=10)
    x[:, 0] = 1.0
    dead = torch.tensor([3, 300, 519], device="cuda")
    w[dead] = 0
    w[dead, 0] = -float("inf")
    live = torch.ones(520, dtype=torch.bool, device="cuda")
    live[dead] = False
    labels = live.nonzero()[:, 0][labels % 517]
    loss = F.linear_cross_entropy(x, w, labels, reduction="none")
    index = torch.cumsum(live, 0) - 1
    ref = reference(x, w[live], index[labels], reduction="none")
    close(loss, ref["rows"], ref["rows_tol"], "loss")
    labels[4] = 300
    assert F.linear_cross_entropy(x, w, labels, reduction="none")[4] == float("inf")


def test_nan_in_a_row_stays_in_its_row(F):
    x, w, labels = inputs(50, 700, 64, seed=11)
    want = F.linear_cross_entropy(x, w, labels, reduction="none")
    x[9, 5] = float("nan")
    got = F.linear_cross_entropy(x, w, labels, reduction="none")
    others = torch.arange(50, device="cuda") != 9
    assert torch.isnan(got[9]) and torch.equal(got[others], want[others])


# ---- pieces, splits, shapes -----------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["ce", "kl"])
def test_pieces_of_the_vocabulary(F, kind):
    """More words than a piece of the backward holds for so many rows (32768), and the last piece odd."""
    x, w, labels = inputs(16384, 33333, 64, seed=12, ignored=0.1)
    if kind == "ce":
        check(run_ce(F, x, w, labels), reference(x, w, labels))
    else:
        tx = (x.float() * 0.8).bfloat16()
        check(run_kl(F, x, w, tx, w, mask=labels != -100),
              reference(x, w, tx=tx, tw=w, mask=labels != -100))


def test_many_words_for_one_row(F):
    """dx in many splits of the vocabulary."""
    x, w, labels = inputs(1, 100003, 64, seed=13)
    check(run_ce(F, x, w, labels), reference(x, w, labels))


def test_leading_dimensions_and_strides(F):
    x, w, labels = inputs(60, 500, 64, seed=14, ignored=0.2)
    want = run_ce(F, x, w, labels, "none")
    wide = torch.zeros(60, 2, 64, dtype=torch.bfloat16, device="cuda")
    wide[:, 1] = x
    got = run_ce(F, wide[:, 1].reshape(3, 20, 64), w, labels.reshape(3, 20), "none")
    assert got[0].shape == (3, 20) and got[1].shape == (3, 20, 64)
    assert torch.equal(got[0].flatten(), want[0]) and torch.equal(got[1].reshape(60, 64), want[1])
    # weights that start off 16 bytes, rows in another order
    off = torch.empty(500 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(500, 64)
    off.copy_(w)
    loss = F.linear_cross_entropy(x.t().contiguous().t(), off, labels, reduction="none")
    assert torch.equal(loss, want[0])


def test_only_the_gradients_that_are_wanted(ops):
    x, w, labels = inputs(100, 900, 64, seed=15)
    _, lse, _ = ops.linear_ce_fwd(x, w, labels)
    one = torch.ones(1, device="cuda")
    both = ops.linear_ce_bwd(x, w, labels, lse, one)
    gx, none = ops.linear_ce_bwd(x, w, labels, lse, one, grad_weight=False)
    assert none is None and torch.equal(gx, both[0])
    none, gw = ops.linear_ce_bwd(x, w, labels, lse, one, grad_x=False)
    assert none is None and torch.equal(gw, both[1])


def test_same_bits_every_time(F):
    x, w, labels = inputs(700, 3000, 256, seed=16, ignored=0.3)
    first = run_ce(F, x, w, labels)
    for _ in range(3):
        for a, b in zip(run_ce(F, x, w, labels), first):
            assert torch.equal(a, b)


# ---- gradients against differences ------------------------------------------------------------------------
def test_gradients_against_differences(F):
    """Differences of the kernel's own sums of losses along the signs of its gradient, in steps of about
    2^-6 of every value, between two bf16 points. Along a line on which a row's logits move by at most a,
    the loss's second and third derivatives are at most a^2 and a^3, and the losses are fp32 sums off by
    rows_tol each."""
    x, w, labels = inputs(48, 700, 64, seed=17)
    _, gx, gw = run_ce(F, x, w, labels, "sum")
    ref = reference(x, w, labels, reduction="sum")
    for t, grad, tol in ((x, gx, ref["gx_tol"]), (w, gw, ref["gw_tol"])):
        step = grad.float().sign() * t.float().abs() * 2 ** -6
        up, down = (t.float() + step).bfloat16(), (t.float() - step).bfloat16()
        hi, lo = (F.linear_cross_entropy(*((v, w) if t is x else (x, v)), labels, reduction="none")
                  for v in (up, down))
        d = up.double() - down.double()
        mid = ((up.double() + down.double()) / 2 - t.double()).abs()
        moved, skew = ((v @ w.double().abs().T if t is x else x.double().abs() @ v.T).max(1).values
                       for v in (d.abs(), mid))
        bound = float((moved ** 3 / 24 + moved * skew).sum() + 3 * ref["rows_tol"].sum()
                      + (tol * d.abs()).sum())
        change = float((hi.double() - lo.double()).sum())
        assert abs(change - float((grad.double() * d).sum())) <= bound < 0.2 * change


# ---- streams, graphs, refusals ------------------------------------------------------------------------------
def test_other_stream(F):
    x, w, labels = inputs(200, 2000, 128, seed=18)
    want = run_ce(F, x, w, labels)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run_ce(F, x, w, labels)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["ce", "kl"])
def test_captured_and_replayed(ops, kind):
    """Forward and backward in a graph; replays on other inputs and other masks than the captured."""
    N, V, H = 300, 3001, 136
    x, w, labels = inputs(N, V, H, seed=19)
    tx = torch.zeros_like(x)
    mask = torch.ones(N, dtype=torch.bool, device="cuda")
    one = torch.ones(1, device="cuda")

    def step():
        if kind == "ce":
            loss, lse, total = ops.linear_ce_fwd(x, w, labels)
            return (loss, total, *ops.linear_ce_bwd(x, w, labels, lse, one))
        loss, lse, total = ops.linear_kl_fwd(x, w, tx, w, mask)
        return (loss, total, *ops.linear_kl_bwd(x, w, tx, w, lse, one, mask=mask))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        nx, _, nl = inputs(N, V, H, seed=30 + seed, ignored=0.25 * seed)
        x.copy_(nx)
        labels.copy_(nl)
        mask.copy_(nl != -100)
        tx.copy_(nx.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_refusals(F, ops):
    x, w, labels = inputs(10, 50, 64)
    with pytest.raises(ValueError, match="reduction"):
        F.linear_cross_entropy(x, w, labels, reduction="average")
    with pytest.raises(ValueError, match="labels"):
        F.linear_cross_entropy(x, w, labels[:9])
    with pytest.raises(TypeError, match="bfloat16"):
        F.linear_cross_entropy(x.float(), w, labels)
    with pytest.raises(TypeError, match="bfloat16"):
        F.linear_cross_entropy(x, w.half(), labels)
    with pytest.raises(TypeError, match="labels"):
        F.linear_cross_entropy(x, w, labels.float())
    with pytest.raises(ValueError, match="width"):
        F.linear_cross_entropy(x, w[:, :56], labels)
    with pytest.raises(ValueError, match="multiple of 8"):
        F.linear_cross_entropy(x[:, :60].contiguous(), w[:, :60].contiguous(), labels)
    with pytest.raises(ValueError, match="word"):
        F.linear_cross_entropy(x, w[:0], labels)
    with pytest.raises(ValueError, match="2 dimensions"):
        F.linear_cross_entropy(x, w.reshape(2, 25, 64), labels)
    with pytest.raises(ValueError, match="2 dimensions"):
        F.linear_distill(x, w, x, w.reshape(2, 25, 64))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        F.linear_cross_entropy(x.cpu(), w, labels)
    with pytest.raises(ValueError, match="temperature"):
        F.linear_distill(x, w, x, w, temperature=0.0)
    with pytest.raises(TypeError, match="mask"):
        F.linear_distill(x, w, x, w, mask=torch.ones(10, device="cuda"))
    with pytest.raises(ValueError, match="leading"):
        F.linear_distill(x, w, x[:9], w)
    with pytest.raises(ValueError, match="words"):
        F.linear_distill(x, w, x, w[:49])
    with pytest.raises(ValueError, match="grad"):
        ops.linear_ce_bwd(x, w, labels, torch.zeros(2, 10, device="cuda"), torch.ones(2, device="cuda"))
    with pytest.raises(ValueError, match="lse"):
        ops.linear_ce_bwd(x, w, labels, torch.zeros(2, 9, device="cuda"), torch.ones(1, device="cuda"))


# ---- as they are used together --------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["ce", "kl"])
def test_last_layer_through_the_head(F, kind):
    """A palettized layer trained through the model's final norm and frozen head: the loss over the
    vocabulary, its gradient at the layer's output, the layer's own gradients clipped and applied."""
    from palettize_hip import layer
    from palettize_hip.optim import FusedAdamW, clip_grad_norm_
    cfg = layer.LayerConfig(hidden=512, heads=4, kv_heads=2, head_dim=128, intermediate=1024,
                            lora_rank=16)
    student = layer.PalettizedDecoderLayer(cfg, seed=0, device="cuda", lora_b_std=0.02)
    teacher = layer.DenseDecoderLayer(cfg, seed=1, device="cuda")
    norm = layer.RMSNorm(512, cfg.eps, "cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    head = (torch.randn(3001, 512, generator=g, device="cuda") * 0.1).bfloat16()
    hs = torch.randn(2, 96, 512, generator=g, device="cuda").bfloat16()
    labels = torch.randint(0, 3001, (2, 96), generator=g, device="cuda")
    labels[:, 70:] = -100
    cos, sin = layer.rope_tables(96, 128, cfg.rope_theta, "cuda")
    out = norm(student(hs, cos, sin))
    out.retain_grad()
    with torch.no_grad():
        t_out = norm(teacher(hs, cos, sin))
    if kind == "ce":
        loss = F.linear_cross_entropy(out, head, labels)
        ref = reference(out.detach().view(-1, 512), head, labels.flatten())
    else:
        loss = F.linear_distill(out, head, t_out, head, mask=labels != -100)
        ref = reference(out.detach().view(-1, 512), head, tx=t_out.view(-1, 512), tw=head,
                        mask=(labels != -100).flatten())
    loss.backward()
    close(loss.detach(), ref["loss"], ref["loss_tol"], "loss")
    close(out.grad.view(-1, 512), ref["gx"], ref["gx_tol"], "gradient of the layer's output")
    params = [p for lin in student.linears() for p in (lin.palette, lin.lora_a, lin.lora_b, lin.index_logits)]
    grads = [p.grad.clone() for p in params]
    assert all(torch.isfinite(v).all() and v.any() for v in grads)
    total = float(sum(v.double().pow(2).sum() for v in grads)) ** 0.5
    got = clip_grad_norm_(params, total / 2)
    assert abs(float(got) - total) <= 2.0 ** -22 * total
    for p, v in zip(params, grads):
        # half, but for the roundings of the factor and of the value
        want = v.double() * (total / 2 / (total + 1e-6))
        eps = torch.finfo(v.dtype).eps / 2
        assert bool(((p.grad.double() - want).abs() <= (eps + 2.0 ** -21) * want.abs() + 2.0 ** -133).all())
    before = [p.detach().clone() for p in params]
    FusedAdamW([{"params": params, "lr": 1e-3}]).step()
    assert all(torch.isfinite(p).all() for p in params)
    assert any(not torch.equal(p, b) for p, b in zip(params, before))


# ---- calls beside each other, captured, past 32 bits -------------------------------------------------------
def test_two_calls_at_once(F):
    """Steps on two streams, each with a workspace of its own."""
    sides = []
    for k in range(2):
        x, w, labels = inputs(300 + 200 * k, 20000, 320, seed=40 + k, ignored=0.1 * k)
        sides.append((x, w, labels, run_ce(F, x, w, labels), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for k, (x, w, labels, _, s) in enumerate(sides):
            with torch.cuda.stream(s):
                got[k].append(run_ce(F, x, w, labels))
    torch.cuda.synchronize()
    for k, (_, _, _, want, _) in enumerate(sides):
        for out in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("kind", ["ce", "kl"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_autograd_captured_and_replayed(F, kind, reduction):
    """Loss and backward through autograd in a graph; no eager graph of its leaves is alive meanwhile."""
    N, V, H = 200, 2500, 136
    x, w, labels = inputs(N, V, H, seed=50)
    tx = x.flip(0).contiguous()

    def step(x, w):
        if kind == "ce":
            loss = F.linear_cross_entropy(x, w, labels, reduction=reduction)
        else:
            loss = F.linear_distill(x, w, tx, w.detach(), mask=labels != -100, reduction=reduction)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w), torch.full_like(loss, 1.5)))

    cx, cw = x.clone().requires_grad_(), w.clone().requires_grad_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(cx, cw)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cx, cw)
    for seed in range(3):
        nx, nw, nl = inputs(N, V, H, seed=60 + seed, ignored=0.3 * seed)
        with torch.no_grad():
            cx.copy_(nx)
            cw.copy_(nw)
        labels.copy_(nl)
        tx.copy_(nx.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = step(nx.clone().requires_grad_(), nw.clone().requires_grad_())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_many_rows_of_few_words(F):
    """More rows than are packed four or eight a workgroup, long runs of them without part."""
    x, w, labels = inputs(20011, 301, 64, seed=51, ignored=0.3)
    labels[5000:9000] = -100
    check(run_ce(F, x, w, labels), reference(x, w, labels))
    check(run_ce(F, x, w, labels, "none"), reference(x, w, labels, reduction="none"))


def test_head_of_more_than_two_to_the_31_values(F, ops):
    """Offsets into the head and its gradient pass 32 bits; pieces of the vocabulary, no step."""
    N, V, H = 3, 900001, 2400
    assert V * H > 2 ** 31 and not ops.vocab_step_fits(N, V, H)
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.empty(V, H, dtype=torch.bfloat16, device="cuda").normal_(0, 0.05, generator=g).requires_grad_()
    x = torch.randn(N, H, generator=g, device="cuda").bfloat16().requires_grad_()
    labels = torch.tensor([5, V - 1, V // 2 + 77], device="cuda")
    loss = F.linear_cross_entropy(x, w, labels, reduction="sum")
    gx, gw = torch.autograd.grad(loss, (x, w))
    with torch.no_grad():
        cuts = range(0, V, 100000)
        part = [x.double() @ w[c:c + 100000].double().T for c in cuts]
        z = torch.cat(part, 1)
        # logits of 2400 products of about 1 * 0.05 each, off by at most this
        off = (H + 4) * 2.0 ** -24 * float((x.double().abs().sum(1) * float(w.abs().max())).max())
        dz = torch.softmax(z, 1)
        lse = torch.logsumexp(z, 1)
        rows = lse - z[torch.arange(3), labels]
        tol = 2 * off + (200 + V // 128) * 2.0 ** -24 + 8 * 2.0 ** -24 * lse.abs()
        assert abs(float(loss) - float(rows.sum())) <= float(tol.sum())
        dz[torch.arange(3), labels] -= 1
        # rounding to bf16, and the logits' and normalisers' errors
        dz_tol = dz.abs() * (2.0 ** -8 + 3 * off + 2 * tol.max())
        want, bound = torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(x, dtype=torch.float64)
        for c in cuts:
            d, t, wd = dz[:, c:c + 100000], dz_tol[:, c:c + 100000], w[c:c + 100000].double()
            want += d @ wd
            bound += (t + V * 2.0 ** -24 * d.abs()) @ wd.abs()
            e = d.T @ x.double()
            te = (t + 67 * 2.0 ** -24 * d.abs()).T @ x.double().abs()
            close(gw[c:c + 100000], e, te + (2.0 ** -8 + 2.0 ** -20) * (e.abs() + te), f"grad_weight from {c}")
        close(gx, want, bound + (2.0 ** -8 + 2.0 ** -20) * (want.abs() + bound), "grad_x")


@pytest.mark.parametrize("kind", ["ce", "kl"])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_loss_divided_in_place(F, kind, reduction):
    """As a loop over micro-batches does; 8 is a power of two, so nothing is rounded by it."""
    x, w, labels = inputs(150, 1000, 96, seed=52)
    x, w = x.requires_grad_(), w.requires_grad_()
    tx, tw = x.detach().flip(0).contiguous(), w.detach().flip(0).contiguous()

    def loss():
        if kind == "ce":
            return F.linear_cross_entropy(x, w, labels, reduction=reduction)
        return F.linear_distill(x, w, tx, tw, reduction=reduction)

    whole, part = loss(), loss()
    part /= 8
    assert torch.equal(part * 8, whole)
    for a, b in zip(torch.autograd.grad(part, (x, w)), torch.autograd.grad(whole, (x, w))):
        assert torch.equal(a * 8, b)


@pytest.mark.parametrize("N", [4, 300])
def test_unlikely_words_beside_a_likely_one(F, N):
    """Every row's label has a probability of about 1, the other words of its tile 10^-4 to 10^-8: their
    rows of the weight's gradient are sums of those alone, and as exact as any."""
    V, H = 256, 64
    g = torch.Generator(device="cuda").manual_seed(53)
    x = torch.zeros(N, H, device="cuda")
    x[:, 0] = 1
    x[:, 1:] = torch.rand(N, H - 1, generator=g, device="cuda")
    w = torch.zeros(V, H, device="cuda")
    w[:, 0] = -torch.linspace(9, 18, V, device="cuda")
    w[100, 0] = 0
    x, w = x.bfloat16(), w.bfloat16()
    labels = torch.full((N,), 100, device="cuda")
    ref = reference(x, w, labels)
    check(run_ce(F, x, w, labels), ref)
    some = ref["gw"].abs() > 0
    assert float((ref["gw_tol"][some] / ref["gw"][some].abs()).median()) < 0.02


def test_more_than_four_gib_of_logits_kept(F, ops):
    """A distillation's step that keeps 6.6 GB of both sides' logits (N past the rows of a tile too)."""
    N, V, H = 4100, 190000, 64
    assert ops.vocab_step_fits(N, V, H, H)
    x, w, _ = inputs(N, V, H, seed=54)
    tx, tw, _ = inputs(N, V, H, seed=55)
    check(run_kl(F, x, w, tx, tw), reference(x, w, tx=tx, tw=tw))


@pytest.mark.parametrize("N", [1, 2, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129])
@pytest.mark.parametrize("on", ["all", "odd", "first", "last", "late", "none"])
def test_few_rows_that_take_part(ops, N, on):
    """Forwards of few rows: any of them may take part, the others hold NaN."""
    V, H = 700, 72
    i = torch.arange(N, device="cuda")
    keep = {"all": i >= 0, "odd": i % 2 == 1, "first": i == 0, "last": i == N - 1, "late": i >= 64,
            "none": i < 0}[on]
    x, w, labels = inputs(N, V, H, seed=56)
    labels = torch.where(keep, labels, torch.full_like(labels, -100))
    ref = reference(x, w, labels)
    bad = torch.where(keep[:, None], x, torch.full_like(x, float("nan")))
    for kind in (labels, labels.int()):
        loss, lse, total = ops.linear_ce_fwd(bad, w, kind)
        close(loss, ref["rows"], ref["rows_tol"], "loss")
        close(total[1], ref["loss"], ref["loss_tol"], "mean")
        assert float(total[2]) == int(keep.sum()) and not lse[:, ~keep].any()
        _, _, total, gx, gw = ops.linear_ce_step(bad, w, kind, grad_weight=False)
        close(total[1], ref["loss"], ref["loss_tol"], "mean")
        close(gx, ref["gx"], ref["gx_tol"], "grad_x")
        assert gw is None and not gx[~keep].any()
    tx, tw, _ = inputs(N, V, 136, seed=57)
    ref = reference(x, w, tx=tx, tw=tw, mask=keep)
    bad_tx = torch.where(keep[:, None], tx, torch.full_like(tx, float("nan")))
    loss, lse, total = ops.linear_kl_fwd(bad, w, bad_tx, tw, keep)
    close(loss, ref["rows"], ref["rows_tol"], "loss")
    close(total[1], ref["loss"], ref["loss_tol"], "mean")
    assert float(total[2]) == int(keep.sum()) and not lse[:, ~keep].any()
    _, _, total, gx, gw = ops.linear_kl_step(bad, w, bad_tx, tw, mask=keep, grad_weight=False)
    close(total[1], ref["loss"], ref["loss_tol"], "mean")
    close(gx, ref["gx"], ref["gx_tol"], "grad_x")
    assert gw is None and not gx[~keep].any()


@pytest.mark.parametrize("others", [5.1875, 5.90625, 6.1875, 6.40625])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_word_that_holds_nearly_all(F, others, reduction):
    """Its gradient is a small difference, of logits that are exact here: 20, the last of its lane, and
    others. The sum of exponentials is 1 and little more from there on: six more additions (a half wave,
    three waves, two joins) of at most 2^-24 each, then the rounding of the result. (A normaliser of 20
    rounded to fp32 is off by 8.5 to 9.5 times 10^-7 with these others.)"""
    V, H, at = 40, 8, 27
    x = torch.zeros(1, H, device="cuda")
    x[0, 0] = 1
    w, tw = torch.zeros(V, H, device="cuda"), torch.zeros(V, H, device="cuda")
    w[:, 0], tw[:, 0] = others, others + 0.25
    w[at, 0] = tw[at, 0] = 20
    x, w, tw = x.bfloat16(), w.bfloat16(), tw.bfloat16()
    q, p = (1 - torch.softmax(t[:, 0].double(), 0)[at] for t in (w, tw))
    wg = w.clone().requires_grad_()
    labels = torch.full((1,), at, device="cuda")
    loss = F.linear_cross_entropy(x, wg, labels, reduction=reduction)
    (got,) = torch.autograd.grad(loss, wg, torch.ones_like(loss))
    assert abs(got[at, 0].double() + q) <= (2.0 ** -8 + 2.0 ** -12) * q + 7 * 2.0 ** -24
    # both sides' sums, and their exponentials: two steps of 2^-24 each
    loss = F.linear_distill(x, wg, x, tw, reduction=reduction)
    (got,) = torch.autograd.grad(loss, wg, torch.ones_like(loss))
    assert abs(got[at, 0].double() - (p - q)) <= (2.0 ** -8 + 2.0 ** -12) * (p - q).abs() + 16 * 2.0 ** -24


@pytest.mark.parametrize("N,V,H,Ht,words", [(129, 300, 64, 64, 300), (400, 5003, 200, 136, 5003),
                                            (1300, 2048, 72, 64, 3), (900, 40000, 128, 128, 40000)])
def test_the_word_that_dominates(F, N, V, H, Ht, words):
    """A distillation of more than 128 rows whose sides lean to different words: what rounding the
    greatest gradient of a row's logits leaves is added. words: the sides lean to the first ones (of 3: many
    rows share one)."""
    x, w, labels = inputs(N, V, H, seed=58, lean=0.0)
    tx, tw, _ = inputs(N, V, Ht, seed=59, lean=0.0)
    g = torch.Generator(device="cuda").manual_seed(60)
    a = torch.randint(0, words, (N,), generator=g, device="cuda")
    b = (a + 1) % words
    x = (x.float() + 1.5 * w[a].float()).bfloat16()
    tx = (tx.float() + 1.5 * tw[b].float()).bfloat16()
    q, p = (torch.softmax(s.double() @ t.double().T, 1) for s, t in ((x, w), (tx, tw)))
    most = (q - p).abs().argmax(1)
    some = torch.zeros(N, V, dtype=torch.bool, device="cuda")
    for side in (q, p):  # the tiles that are looked at
        some |= torch.arange(V, device="cuda") // 256 == (side.argmax(1) // 256)[:, None]
    assert bool(some.gather(1, most[:, None]).all())
    check(run_kl(F, x, w, tx, tw), reference(x, w, tx=tx, tw=tw, top=True))


# ---- a distillation's loss alone ----------------------------------------------------------------------
def exact_inputs(N, V, H, seed):
    """x, w of multiples of 1/4 up to 2: logits, and those moved by up to 2^16, are exact in fp32."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return tuple((torch.randint(-8, 9, (n, H), generator=g, device="cuda") / 4).bfloat16() for n in (N, V))


@pytest.mark.parametrize("N,V", [(3, 700), (130, 1003), (300, 40001), (16384, 33333)])
@pytest.mark.parametrize("shift", [2.0 ** 10, -2.0 ** 14])
def test_what_all_logits_of_a_row_share_is_no_part_of_a_distillation(ops, N, V, shift):
    """The student's logits moved by the same amount: exact ones, so every difference is the same and the loss
    is the same to the last bit. (Of 16384 rows the words come in pieces.)"""
    x, w = exact_inputs(N, V, 16, 70)
    tx, tw = exact_inputs(N, V, 16, 71)
    x[:, -1] = 1
    w[:, -1] = 0
    want = ops.linear_kl_fwd(x, w, tx, tw)[0]
    w[:, -1] = shift
    assert torch.equal(ops.linear_kl_fwd(x, w, tx, tw)[0], want)
    # a teacher that is the student but for that
    same, ws = x.clone(), w.clone()
    ws[:, -1] = 0
    assert not ops.linear_kl_fwd(x, w, same, ws)[0].any()


@pytest.mark.parametrize("N", [3, 150, 700])
def test_words_that_cannot_be_distilled(ops, N):
    """Logits of minus infinity, of whole tiles too: where the teacher's are, the words count for nothing;
    where only the student's are, the loss is infinite."""
    V, H = 1100, 64
    x, w, _ = inputs(N, V, H, seed=72)
    tx, tw, _ = inputs(N, V, H, seed=73)
    x[:, 0] = tx[:, 0] = 1
    i = torch.arange(V, device="cuda")
    dead = (i < 131) | ((i >= 256) & (i < 512)) | (i == V - 1)
    kill = lambda t: torch.where(dead[:, None], torch.where(torch.arange(H, device="cuda") == 0,
                                                            -float("inf"), 0.0), t.float()).bfloat16()
    both = reference(x, w[~dead], tx=tx, tw=tw[~dead], reduction="none")
    close(ops.linear_kl_fwd(x, kill(w), tx, kill(tw))[0], both["rows"], both["rows_tol"], "of neither side")
    # the student's probabilities are of all words: its normaliser is another
    got = ops.linear_kl_fwd(x, w, tx, kill(tw))[0]
    z, dz = logits(x, w)
    apart = torch.logsumexp(z, 1) - torch.logsumexp(z[:, ~dead], 1)
    tol = both["rows_tol"] + 2 * dz.max(1).values + 256 * 2.0 ** -24
    close(got, both["rows"] + apart, tol, "of the teacher's words alone")
    assert bool((ops.linear_kl_fwd(x, kill(w), tx, tw)[0] == float("inf")).all())


# ---- what rounding the logits' gradients may leave -------------------------------------------------------
def single_terms(N, D, at, seed):
    """Inputs whose gradients are one product each: the rows `at` hold one value each, in a column of its own,
    and the head's words too, so that neither gradient sums over words or rows and the roundings of the
    logits' gradient and of the result show as they are. The other rows hold NaN and take no part."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = torch.arange(at.numel(), device="cuda")
    x, tx = (torch.full((N, D), float("nan"), device="cuda") for _ in range(2))
    keep = torch.zeros(N, dtype=torch.bool, device="cuda")
    keep[at] = True
    w, tw = (torch.diag(0.5 + 1.5 * torch.rand(D, generator=g, device="cuda")).bfloat16() for _ in range(2))
    for t in (x, tx):
        t[at] = 0
        t[at, k] = 6 * torch.rand(at.numel(), generator=g, device="cuda")
    labels = torch.full((N,), -100, device="cuda")
    labels[at] = k
    return x.bfloat16(), w, tx.bfloat16(), tw, labels, keep


def check_rows(got, ref, at):
    """check() of gradients of which only the rows `at` took part, against a reference of those alone."""
    loss, gx, gw = got
    close(loss if loss.dim() == 0 else loss[at], ref["loss"], ref["loss_tol"], "loss")
    close(gx[at], ref["gx"], ref["gx_tol"], "grad_x")
    close(gw, ref["gw"], ref["gw_tol"], "grad_weight")


@pytest.mark.parametrize("N,part,D", [(300, 13, 64), (1000, 100, 128), (200, 128, 136), (4099, 3, 64)])
@pytest.mark.parametrize("kind", ["ce", "kl"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_few_rows_of_many_take_part(F, N, part, D, kind, reduction):
    """Where up to 128 rows take part, the logits' gradients are in two bf16 however many rows were given."""
    at = torch.randperm(N, generator=torch.Generator().manual_seed(N))[:part].sort().values.cuda()
    x, w, tx, tw, labels, keep = single_terms(N, D, at, N + part)
    up = None
    if reduction == "none":
        up = torch.rand(N, device="cuda") + 0.5
    kw = dict(reduction=reduction, upstream=None if up is None else up[at])
    if kind == "ce":
        check_rows(run_ce(F, x, w, labels, reduction, up), reference(x[at], w, labels[at], **kw), at)
    else:
        check_rows(run_kl(F, x, w, tx, tw, reduction, up, mask=keep), reference(x[at], w, tx=tx[at], tw=tw, **kw), at)


@pytest.mark.parametrize("N,part,D", [(200, 200, 200), (300, 150, 152), (520, 520, 520), (1500, 1100, 1104)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_the_label_s_gradient_in_two_parts(F, ops, N, part, D, reduction):
    """Of more than 128 rows, what rounding the greatest gradient of a row's logits leaves, the label's, is
    added to both products; in a step, and where the backward computes the logits again."""
    at = torch.randperm(N, generator=torch.Generator().manual_seed(N)).sort().values[-part:].cuda()
    x, w, _, _, labels, _ = single_terms(N, D, at, N + part)
    up = torch.rand(N, device="cuda") + 0.5 if reduction == "none" else None
    ref = reference(x[at], w, labels[at], reduction=reduction, top=True, upstream=None if up is None else up[at])
    check_rows(run_ce(F, x, w, labels, reduction, up), ref, at)
    if reduction != "none":
        check_rows(two_calls_ce(ops, x, w, labels, reduction), ref, at)


@pytest.mark.parametrize("N,part,D", [(200, 200, 200), (300, 150, 152), (520, 520, 520), (1500, 1100, 1104)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_distillation_s_backward_adds_what_its_step_adds(F, ops, N, part, D, reduction):
    """Of more than 128 rows, what rounding the greatest gradient of a row's logits leaves is added, whether a
    step or a backward of its own computes them."""
    at = torch.randperm(N, generator=torch.Generator().manual_seed(N)).sort().values[-part:].cuda()
    x, w, tx, tw, _, keep = single_terms(N, D, at, N + part)
    up = torch.rand(N, device="cuda") - 0.5 if reduction == "none" else None
    ref = reference(x[at], w, tx=tx[at], tw=tw, reduction=reduction, top=True, upstream=None if up is None else up[at])
    check_rows(run_kl(F, x, w, tx, tw, reduction, up, mask=keep), ref, at)
    if reduction != "none":
        check_rows(two_calls_kl(ops, x, w, tx, tw, keep), ref, at)


@pytest.mark.parametrize("kind", ["ce", "kl"])
def test_the_greatest_gradients_over_pieces(ops, kind):
    """As those, of a vocabulary in four pieces: a piece's dW adds its own, dx the greatest of all. 200 words
    anywhere hold one value each, in a column of its own; the other words' logits are 0."""
    N, part, V, H = 16384, 200, 25011, 200
    g = torch.Generator(device="cuda").manual_seed(80)
    at = torch.randperm(N, generator=torch.Generator().manual_seed(81))[:part].sort().values.cuda()
    _, dw, _, dtw, _, keep = single_terms(N, H, at, 82)
    words = torch.randperm(V, generator=torch.Generator().manual_seed(83))[:H].cuda()
    x, tx = (torch.full((N, H), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    w, tw = (torch.zeros(V, H, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    k = torch.arange(part, device="cuda")
    # the sides lean to other words, of other pieces
    for t, d, m, l in ((x, dw, w, k), (tx, dtw, tw, (k + 77) % part)):
        t[at] = 0
        t[at, l] = (9 + 3 * torch.rand(part, generator=g, device="cuda")).bfloat16()
        m[words] = d
    labels = torch.full((N,), -100, device="cuda")
    labels[at] = words[k]
    if kind == "ce":
        ref = reference(x[at], w, labels[at], kept=False, top=True)
        check_rows(two_calls_ce(ops, x, w, labels), ref, at)
    else:
        ref = reference(x[at], w, tx=tx[at], tw=tw, top=True)
        check_rows(two_calls_kl(ops, x, w, tx, tw, keep), ref, at)


# ---- the logits computed again instead of what a step keeps ----------------------------------------------
@pytest.mark.parametrize("N,part,D", [(13, 13, 64), (300, 200, 200), (700, 520, 520)])
@pytest.mark.parametrize("kind", ["ce", "kl"])
def test_recompute_rounds_once(F, N, part, D, kind):
    """Gradients for an upstream gradient of 0.37: those of every row's loss times 0.37 over the rows, rounded
    once (what the forward computed would be rounded before, too)."""
    at = torch.randperm(N, generator=torch.Generator().manual_seed(N)).sort().values[-part:].cuda()
    x, w, tx, tw, labels, keep = single_terms(N, D, at, N + part)
    up = torch.full((part,), 0.37 / part, device="cuda", dtype=torch.float64)
    kw = dict(labels=labels[at]) if kind == "ce" else dict(tx=tx[at], tw=tw)
    ref = reference(x[at], w, reduction="none", upstream=up, top=True, **kw)
    mean = reference(x[at], w, **kw)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    if kind == "ce":
        loss = F.linear_cross_entropy(a, b, labels, recompute=True)
    else:
        loss = F.linear_distill(a, b, tx, tw, mask=keep, recompute=True)
    close(loss.detach(), mean["loss"], mean["loss_tol"], "loss")
    for _ in range(2):  # a second backward is the same
        gx, gw = torch.autograd.grad(loss, (a, b), torch.tensor(0.37, device="cuda"), retain_graph=True)
        # (0.37 in fp32, and over the rows: two roundings more)
        close(gx[at], ref["gx"], ref["gx_tol"] + 2.0 ** -22 * ref["gx"].abs(), "grad_x")
        close(gw, ref["gw"], ref["gw_tol"] + 2.0 ** -22 * ref["gw"].abs(), "grad_weight")


@pytest.mark.parametrize("kind", ["ce", "kl"])
def test_recompute_takes_a_piece_of_memory(F, ops, kind):
    """4096 rows of 150000 words: 1.1 GiB kept by a step (5.7 a distillation's), 1 GiB in pieces, and nothing
    but the rows' normalisers from the forward to the backward."""
    N, V, H = 4096, 150000, 64
    x, w, labels = inputs(N, V, H, seed=90, ignored=0.1)
    tx = x.flip(0).contiguous()
    assert ops.vocab_step_fits(N, V, H, 0 if kind == "ce" else H)

    def peaks(recompute):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        if kind == "ce":
            loss = F.linear_cross_entropy(a, b, labels, recompute=recompute)
        else:
            loss = F.linear_distill(a, b, tx, w, mask=labels != -100, recompute=recompute)
        forward = torch.cuda.max_memory_allocated() - before
        held = torch.cuda.memory_allocated() - before
        grads = torch.autograd.grad(loss, (a, b))
        return (loss.detach(), *grads), forward, held, torch.cuda.max_memory_allocated() - before

    want, forward, held, _ = peaks(False)
    got, less, row, peak = peaks(True)
    gib = 2 ** 30
    assert forward > (1.1 if kind == "ce" else 5.7) * gib and held > 2 * (w.numel() + x.numel())
    assert less < (0.1 if kind == "ce" else 1.1) * gib and row < 64 * N and peak < 1.2 * gib
    ref = dict(labels=labels) if kind == "ce" else dict(tx=tx, tw=w, mask=labels != -100)
    check(want, reference(x, w, **ref))
    check(got, reference(x, w, kept=False, **ref))


@pytest.mark.parametrize("kind,N,V", [("kl", 16384, 60001), ("ce", 33000, 66001)])
def test_a_loss_beyond_a_step_s_limit(F, ops, kind, N, V):
    """The mean and sum of more logits than a step keeps: pieces of the vocabulary through autograd, for an
    upstream gradient that is no power of two."""
    H = 64
    assert not ops.vocab_step_fits(N, V, H, H if kind == "kl" else 0)
    x, w, labels = inputs(N, V, H, seed=91, ignored=0.3)
    tx, mask = (x.float() * 0.8).bfloat16(), labels != -100
    for reduction, up in (("mean", 3.0), ("sum", 0.37)):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        if kind == "kl":
            loss, ref = F.linear_distill(a, b, tx, w, mask=mask, reduction=reduction), dict(tx=tx, tw=w, mask=mask)
        else:
            loss, ref = F.linear_cross_entropy(a, b, labels, reduction=reduction), dict(labels=labels, kept=False)
        grads = torch.autograd.grad(loss, (a, b), torch.tensor(up, device="cuda"))
        check((loss.detach(), *grads), reference(x, w, reduction=reduction, upstream=up, **ref))


def test_a_step_of_a_head_past_two_gib(F, ops):
    """Offsets of the head's copies pass 31 bits, and its last tile of columns is not whole."""
    N, V, H = 130, 240007, 4504
    assert V * H * 2 > 2 ** 31 and H % 256 and ops.vocab_step_fits(N, V, H)
    g = torch.Generator(device="cuda").manual_seed(92)
    w = torch.empty(V, H, dtype=torch.bfloat16, device="cuda").normal_(0, 0.03, generator=g).requires_grad_()
    x = torch.randn(N, H, generator=g, device="cuda").bfloat16().requires_grad_()
    labels = torch.randint(0, V, (N,), generator=g, device="cuda")
    labels[-1] = V - 1
    loss = F.linear_cross_entropy(x, w, labels, reduction="sum")
    gx, gw = torch.autograd.grad(loss, (x, w))
    with torch.no_grad():
        cuts = range(0, V, 40000)
        z = torch.cat([x.double() @ w[c:c + 40000].double().T for c in cuts], 1)
        # of a logit: products of magnitudes of at most this sum, and the normaliser's
        off = (H + 4) * 2.0 ** -24 * float((x.double().abs().sum(1) * float(w.abs().max())).max())
        lse = torch.logsumexp(z, 1)
        rows = lse - z[torch.arange(N), labels]
        tol = 2 * off + (200 + V // 128) * 2.0 ** -24 + 8 * 2.0 ** -24 * lse.abs()
        assert abs(float(loss) - float(rows.sum())) <= float(tol.sum()) + 2 * 2.0 ** -24 * float(rows.sum())
        dz = torch.exp(z - lse[:, None])
        dz[torch.arange(N), labels] -= 1
        # rounded to bf16, kept in fp16 before, from logits and normalisers that are off
        dz_tol = dz.abs() * (2.0 ** -8 + 2.0 ** -11 + 3 * off + 2 * float(tol.max())) + 2.0 ** -40
        want, bound = (torch.zeros_like(x, dtype=torch.float64) for _ in range(2))
        for c in cuts:
            d, t, wd = dz[:, c:c + 40000], dz_tol[:, c:c + 40000], w[c:c + 40000].double()
            want += d @ wd
            bound += (t + V * 2.0 ** -24 * d.abs()) @ wd.abs()
            e, te = d.T @ x.double(), (t + (N + 64) * 2.0 ** -24 * d.abs()).T @ x.double().abs()
            close(gw[c:c + 40000], e, te + (2.0 ** -8 + 2.0 ** -20) * (e.abs() + te), f"grad_weight from {c}")
        close(gx, want, bound + (2.0 ** -8 + 2.0 ** -20) * (want.abs() + bound), "grad_x")


@pytest.mark.parametrize("N,part", [(5, 5), (100, 100), (300, 90), (300, 300)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_label_that_cannot_be(F, N, part, reduction):
    """A label whose logit is minus infinity, of one row: its loss and its gradient along the infinite weight
    are infinite, as the formula's are (dz is -1 there and 0 elsewhere; 0 times infinity is NaN in the other
    rows, as it is in any product)."""
    V, H, dead, row = 700, 64, 301, 3
    x, w, labels = inputs(N, V, H, seed=95)
    labels[part:] = -100
    x[:, 0] = 1
    labels[labels == dead] = 5
    labels[row] = dead
    w[dead] = 0
    w[dead, 0] = -float("inf")
    loss, gx, gw = run_ce(F, x, w, labels, reduction)
    assert float(loss if reduction == "mean" else loss[row]) == float("inf")
    assert float(gx[row, 0]) == float("inf") and torch.isfinite(gx[row, 1:]).all()
    others = torch.arange(part, device="cuda") != row
    assert torch.isnan(gx[:part][others][:, 0]).all() and torch.isfinite(gx[:part, 1:]).all()
    assert torch.isfinite(gw).all()


@pytest.mark.parametrize("N,part", [(5, 5), (100, 100), (300, 90), (300, 300)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_word_that_only_the_student_cannot_say(F, N, part, reduction):
    """Its logit is minus infinity, the teacher's is not: infinite losses, and gradients of -p times minus
    infinity along the infinite weight."""
    V, H, dead = 700, 64, 301
    x, w, _ = inputs(N, V, H, seed=96)
    tx, tw, _ = inputs(N, V, H, seed=97)
    mask = torch.arange(N, device="cuda") < part
    x[:, 0] = 1
    w[dead] = 0
    w[dead, 0] = -float("inf")
    tx[:, 1], tw[dead, 1] = 1, 8.0  # the teacher's likeliest word, so the greatest gradient of each row
    loss, gx, gw = run_kl(F, x, w, tx, tw, reduction, mask=mask)
    assert bool((loss if reduction == "mean" else loss[:part] == float("inf")).all())
    assert bool((gx[:part, 0] == float("inf")).all()) and torch.isfinite(gx[:part, 1:]).all()
    assert torch.isfinite(gw).all() and not gx[part:].any()
