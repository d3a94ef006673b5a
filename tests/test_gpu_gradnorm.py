"""The global gradient norm and clipping against 64 bits (GPU).

The norm is a 64-bit sum rounded to fp32 once: off by 2^-24 of its value, and the sum's own errors, of
64-bit operations, are far below. A clipped value is rounded to fp32 in the factor and in the product
(2^-24 each, and the norm's part in the factor is of 64 bits), then to its type: bf16 2^-8, fp16 2^-11."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# the least steps of the types, of which a rounded subnormal is off by half
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}
TYPES = list(HALF)


@pytest.fixture(autouse=True)
def _gpu(dev):
    pass


@pytest.fixture(scope="module")
def ops():
    from palettize_hip import ops
    return ops


def grads_of(sizes, types, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, generator=g, device="cuda") * scale * 10 ** (-(i % 4))).to(types[i % len(types)])
            for i, s in enumerate(sizes)]


def norm_of(grads):
    return float(sum(float(g.double().pow(2).sum()) for g in grads)) ** 0.5


def check_norm(got, grads):
    assert got.dtype == torch.float32 and got.shape == ()
    want = norm_of(grads)
    assert abs(float(got) - want) <= 2 * 2.0 ** -24 * want


def check_clipped(out, grads, max_norm):
    factor = min(1.0, max_norm / (norm_of(grads) + 1e-6))
    for o, g in zip(out, grads):
        want = g.double() * factor
        tol = (HALF[o.dtype] + 3 * 2.0 ** -24) * want.abs() + TINY[o.dtype]
        assert o.shape == g.shape and bool(((o.double() - want).abs() <= tol).all())


SIZES = [
    [(1,)], [(7,)], [(8,)], [()], [(0,), (3,)], [(2047,), (2049,)], [(32768,)], [(32769,), (5,)],
    [(100003,)], [(3, 5, 7), (64, 129), (1,)], [(17,)] * 300, [(40000,)] * 140]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("types", [TYPES[:1], TYPES[1:2], TYPES[2:], TYPES])
def test_norm_and_clip(ops, sizes, types):
    grads = grads_of(sizes, types)
    check_norm(ops.grad_norm(grads), grads)
    for max_norm in (0.0, 0.3, 1e6):
        for out_type in TYPES:
            out = [torch.full(g.shape, 5.0, dtype=out_type, device="cuda") for g in grads]
            check_norm(ops.clip_grads(grads, max_norm, out=out), grads)
            check_clipped(out, grads, max_norm)
        mine = [g.clone() for g in grads]
        check_norm(ops.clip_grads(mine, max_norm), grads)
        check_clipped(mine, grads, max_norm)


def test_large(ops):
    grads = grads_of([(70_000_001,), (3000, 3001)], [torch.bfloat16, torch.float32])
    check_norm(ops.grad_norm(grads), grads)
    out = [torch.empty(g.shape, dtype=torch.bfloat16, device="cuda") for g in grads]
    ops.clip_grads(grads, 1.0, out=out)
    check_clipped(out, grads, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_off_16_bytes(ops, dtype):
    """Views that start anywhere, between values that stay as they are."""
    for first in (1, 2, 3, 5):
        base = torch.randn(70000, device="cuda").to(dtype)
        keep, view = base.clone(), base[first:first + 65537]
        grads = [view.clone()]
        check_norm(ops.grad_norm([view]), grads)
        ops.clip_grads([view], 0.5)
        check_clipped([view], grads, 0.5)
        assert torch.equal(base[:first], keep[:first])
        assert torch.equal(base[first + 65537:], keep[first + 65537:])


def test_beyond_the_types_squares(ops):
    """Squares that fp32 does not hold."""
    for scale in (1e30, 1e-30):
        for dtype in (torch.float32, torch.bfloat16):
            grads = [(torch.randn(5000, device="cuda") * scale).to(dtype)]
            check_norm(ops.grad_norm(grads), grads)
    grads = [torch.randn(64, device="cuda") * 1e37]
    out = [torch.empty(64, device="cuda")]
    check_norm(ops.clip_grads(grads, 10.0, out=out), grads)
    check_clipped(out, grads, 10.0)
    huge = [torch.full((4096,), 3e38, device="cuda")]
    assert float(ops.grad_norm(huge)) == float("inf")  # the norm itself is past fp32


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_not_finite_as_torch(ops, value):
    grads = grads_of([(1000,), (70,)], [torch.float32])
    grads[1][3] = value
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g.clone()
    want = torch.nn.utils.clip_grad_norm_(params, 1.0)
    got = ops.clip_grads(grads, 1.0)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    for g, p in zip(grads, params):
        assert torch.allclose(g, p.grad, rtol=0, atol=0, equal_nan=True)


def test_untouched_below_the_limit(ops):
    grads = grads_of([(1000,), (33,)], [torch.bfloat16])
    keep = [g.clone() for g in grads]
    ops.clip_grads(grads, 1e9)
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))


def test_clip_grad_norm_of_parameters(ops):
    from palettize_hip.optim import clip_grad_norm_
    params = [torch.nn.Parameter(torch.zeros(s, device="cuda", dtype=t))
              for s, t in (((64, 32), torch.bfloat16), ((100,), torch.float32), ((9, 9), torch.float16),
                           ((5,), torch.float32))]
    for p, g in zip(params, grads_of([p.shape for p in params], [p.dtype for p in params])):
        p.grad = g
    params[2].grad = params[2].grad.t().contiguous().t()
    params[3].grad = None
    before = [p.grad.clone() for p in params[:3]]
    check_norm(clip_grad_norm_(params + params[:1], 0.25), before)  # tied: once
    check_clipped([p.grad for p in params[:3]], before, 0.25)
    assert params[3].grad is None
    assert float(clip_grad_norm_(params[3], 1.0)) == 0


def test_after_a_loss_over_the_vocabulary(ops):
    """A training step of a head: loss, gradients, clipped, FusedAdamW with the clipped ones."""
    from palettize_hip.functional import linear_cross_entropy
    from palettize_hip.optim import FusedAdamW, clip_grad_norm_
    from vocab_ref import inputs, reference
    x, w, labels = inputs(96, 1200, 128, seed=4, ignored=0.2)
    head = torch.nn.Parameter(w)
    x.requires_grad_()
    linear_cross_entropy(x, head, labels).backward()
    ref = reference(x.detach(), w, labels)
    grads = [x.grad.clone(), head.grad.clone()]
    norm = clip_grad_norm_([x, head], 1e-3)
    check_norm(norm, grads)
    check_clipped([x.grad, head.grad], grads, 1e-3)
    want = float(ref["gx"].pow(2).sum() + ref["gw"].pow(2).sum()) ** 0.5
    off = float(ref["gx_tol"].pow(2).sum() + ref["gw_tol"].pow(2).sum()) ** 0.5
    assert abs(float(norm) - want) <= off + 2.0 ** -22 * want
    before = head.detach().clone()
    FusedAdamW([{"params": [head], "lr": 1e-2}]).step()
    assert torch.isfinite(head).all() and not torch.equal(head, before)


def test_captured_and_replayed(ops):
    grads = grads_of([(5000,), (33,), (70000,)], [torch.float32])
    out = [torch.empty(g.shape, dtype=torch.bfloat16, device="cuda") for g in grads]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.clip_grads(grads, 1.0, out=out)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grads(grads, 1.0, out=out)
    for seed in range(4):
        for g, n in zip(grads, grads_of([g.shape for g in grads], [torch.float32], seed, 10.0 ** seed)):
            g.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        check_norm(norm, grads)
        check_clipped(out, grads, 1.0)


def test_scale(ops):
    grads = grads_of([(5000,), (33,), (0,), (70001,)], TYPES)
    keep = [g.clone() for g in grads]
    ops.scale_grads(grads, torch.ones((), device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))
    ops.scale_grads(grads, torch.tensor(-2.0, device="cuda"))
    assert all(torch.equal(a, -2 * b) for a, b in zip(grads, keep))
    ops.scale_grads([], torch.ones((), device="cuda"))
    with pytest.raises(ValueError, match="written twice"):
        ops.scale_grads([grads[0], grads[0]], torch.ones((), device="cuda"))
    with pytest.raises(ValueError, match="one value"):
        ops.scale_grads(grads, torch.ones(2, device="cuda"))
    with pytest.raises(TypeError, match="factor"):
        ops.scale_grads(grads, torch.ones((), device="cuda", dtype=torch.float64))


def test_refusals(ops):
    a, b = (torch.ones(10, device="cuda") for _ in range(2))
    with pytest.raises(ValueError, match="at least one"):
        ops.grad_norm([])
    with pytest.raises(TypeError, match="tensors expected"):
        ops.grad_norm([a.double()])
    with pytest.raises(TypeError, match="tensors expected"):
        ops.grad_norm([a, 3.0])
    with pytest.raises(RuntimeError, match="GPU"):
        ops.grad_norm([a.cpu()])
    with pytest.raises(ValueError, match="contiguous"):
        ops.grad_norm([torch.ones(4, 4, device="cuda").t()])
    with pytest.raises(RuntimeError, match="no backward"):
        ops.grad_norm([a.clone().requires_grad_()])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            ops.clip_grads([a], bad)
    with pytest.raises(ValueError, match="written twice"):
        ops.clip_grads([a, a], 1.0)
    with pytest.raises(ValueError, match="written twice"):
        ops.clip_grads([a, b], 1.0, out=[a, a])
    with pytest.raises(ValueError, match="another gradient"):
        ops.clip_grads([a, b], 1.0, out=[b, a])
    with pytest.raises(ValueError, match="another gradient"):
        ops.clip_grads([a], 1.0, out=[a.view(torch.bfloat16)[:10]])
    with pytest.raises(ValueError, match="shape"):
        ops.clip_grads([a], 1.0, out=[torch.ones(11, device="cuda")])
    with pytest.raises(ValueError, match="outputs"):
        ops.clip_grads([a], 1.0, out=[])
    assert torch.equal(a, torch.ones_like(a))


# ---- what else knows of the gradients -----------------------------------------------------------------
def test_autograd_sees_what_was_written(ops):
    """A tensor that a graph saved and that is clipped or scaled before the backward: refused, as after any
    in-place operation. A gradient that is only read may still be used."""
    def saved(t):
        leaf = torch.ones(16, device="cuda", requires_grad=True)
        return (leaf * t).sum()

    one = torch.full((), 0.5, device="cuda")
    read, written = torch.full((16,), 2.0, device="cuda"), torch.full((16,), 2.0, device="cuda")
    for call, t in ((lambda: ops.clip_grads([written], 1.0), written),
                    (lambda: ops.clip_grads([read], 1.0, out=[written]), written),
                    (lambda: ops.scale_grads([written], one), written)):
        loss, other, before = saved(t), saved(read), t._version
        call()
        assert t._version > before
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
        other.backward()


def test_clipped_between_backward_and_update(ops):
    """The trainer's update takes the squared sums that the backward wrote beside the gradients only while
    those are as they were: of clipped ones it reports the norm of what they are now."""
    from palettize_hip import layer
    from palettize_hip.optim import clip_grad_norm_
    cfg = layer.LayerConfig(hidden=512, heads=4, kv_heads=2, head_dim=128, intermediate=1024, lora_rank=16)
    tr = layer.LayerTrainer(cfg, "cuda", seed=0, lora_b_std=0.02)
    g = torch.Generator(device="cuda").manual_seed(1)
    tr.forward_backward(torch.randn(2, 64, 512, generator=g, device="cuda").bfloat16())
    before = norm_of([p.grad for p in tr.logits])
    clip_grad_norm_(tr.logits, before / 8)
    want = [norm_of([p.grad for p in params]) for params in (tr.logits, tr.others)]
    assert want[0] < before / 4
    tr.update()
    for got, w in zip(tr.opt.last_norms.tolist(), want):
        # the optimizer's own sum, in fp32, of positive terms: a thread's 32 squares (64 roundings), then
        # fewer than 64 additions of partial sums
        assert abs(got - w) <= 128 * 2.0 ** -24 * w


def test_clip_grad_norm_keeps_the_gradients_memory(ops):
    """Gradients of other orders and strides are scaled where they are: who holds them, or what they are
    views of, holds the clipped values, and what lies between them stays."""
    from palettize_hip.optim import clip_grad_norm_
    bucket = torch.randn(40, 24, device="cuda")
    turned = torch.randn(24, 40, device="cuda").bfloat16()
    params = [torch.nn.Parameter(torch.zeros(40, 12, device="cuda")),
              torch.nn.Parameter(torch.zeros(40, 24, device="cuda", dtype=torch.bfloat16)),
              torch.nn.Parameter(torch.zeros(7, device="cuda")),
              torch.nn.Parameter(torch.zeros(5, 3, device="cuda"))]
    held = [bucket[:, ::2], turned.t(), torch.randn(7, device="cuda"), torch.ones(3, device="cuda").expand(5, 3)]
    for p, g in zip(params, held):
        p.grad = g
    before, rest = [g.clone() for g in held], bucket[:, 1::2].clone()
    check_norm(clip_grad_norm_(params, 0.25), before)
    check_clipped([p.grad for p in params], before, 0.25)
    for p, g in zip(params[:3], held):
        assert p.grad is g
    check_clipped([bucket[:, ::2], turned.t()], before[:2], norm_of(before[:2]) * 0.25 / norm_of(before))
    assert torch.equal(bucket[:, 1::2], rest)
