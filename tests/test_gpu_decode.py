"""GPU: palettized layers that answer token by token over a paged cache (palettize_hip.decode) against
the same layers in 64 bits over whole sequences."""
import math

import pytest
import torch

from helpers import assert_close, f32

pytestmark = pytest.mark.gpu
decode = pytest.importorskip("palettize_hip.decode")
layer = pytest.importorskip("palettize_hip.layer")

CFGS = {"d128": dict(hidden=256, heads=4, kv_heads=2, head_dim=128, intermediate=512),
        "d64": dict(hidden=256, heads=8, kv_heads=2, head_dim=64, intermediate=512)}


def _layers(dev, kw, n=2):
    cfg = layer.LayerConfig(**kw)
    soft = [layer.PalettizedDecoderLayer(cfg, seed=i, device=dev, lora_b_std=0.02) for i in range(n)]
    for i, s in enumerate(soft):  # the logits away from their one-hot start, norms away from one
        g = torch.Generator().manual_seed(50 + i)
        for lin in s.linears():
            lin.index_logits.data.copy_(torch.randn(lin.index_logits.shape, generator=g))
        for nm in decode.HardDecoderLayer.NORMS:
            w = getattr(s, nm).weight
            w.data.copy_(1 + 0.2 * torch.randn(w.shape, generator=g))
    return cfg, [decode.HardDecoderLayer.from_soft(s) for s in soft], soft


def _norm(x, w, eps):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def _reference(cfg, soft, hs, cos, sin):
    """The layers on one sequence [S, hidden] in 64 bits, weights dequantised as bf16."""
    S, D, G = hs.shape[0], cfg.head_dim, cfg.heads // cfg.kv_heads
    c, s = cos[:S, None].double(), sin[:S, None].double()
    mask = torch.triu(torch.ones(S, S, dtype=torch.bool, device=hs.device), 1)
    for l in soft:
        def lin(name, x):
            p = getattr(l, name)
            idx = p.index_logits.argmax(-1)
            pal = p.palette.to(torch.bfloat16).repeat_interleave(256, 1)
            w = torch.gather(pal, 2, idx[..., None])[..., 0].double()
            return x @ w.T + p.lora_scale * (x @ p.lora_a.double().T) @ p.lora_b.double().T

        def rope(x):
            a, b = x.chunk(2, -1)
            return x * c + torch.cat([-b, a], -1) * s

        x = _norm(hs, l.input_layernorm.weight, cfg.eps)
        q = rope(_norm(lin("q_proj", x).view(S, -1, D), l.q_norm.weight, cfg.eps))
        k = rope(_norm(lin("k_proj", x).view(S, -1, D), l.k_norm.weight, cfg.eps))
        v = lin("v_proj", x).view(S, -1, D)
        k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
        score = torch.stack([q[:, h] @ k[:, h].T for h in range(cfg.heads)]) / math.sqrt(D)
        p = torch.softmax(score.masked_fill(mask, -math.inf), -1)
        o = torch.stack([p[h] @ v[:, h] for h in range(cfg.heads)], 1).reshape(S, -1)
        hs = hs + lin("o_proj", o)
        x = _norm(hs, l.post_attention_layernorm.weight, cfg.eps)
        g = lin("gate_proj", x)
        hs = hs + lin("down_proj", g * torch.sigmoid(g) * lin("up_proj", x))
    return hs


@pytest.mark.parametrize("kw", CFGS.values(), ids=CFGS.keys())
def test_prompts_then_tokens(dev, kw):
    """Prompts of 5, 130 and 64 tokens, then eleven steps in which a request ends, its row takes a new
    prompt, and one row pauses: every row of every step against the whole sequence so far."""
    cfg, hard, soft = _layers(dev, kw)
    cos, sin = layer.rope_tables(256, cfg.head_dim, cfg.rope_theta, dev)
    cache = decode.PagedKVCache(2, 3, 256, cfg.kv_heads, cfg.head_dim, page_size=16, device=dev)
    g = torch.Generator().manual_seed(1)
    seqs = [torch.zeros(0, cfg.hidden, dtype=torch.bfloat16, device=dev) for _ in range(3)]

    def tokens(n):
        return torch.randn(n, cfg.hidden, generator=g).to(torch.bfloat16).to(dev)

    def prefill(lens, keep=None):
        step = cache.step(lens, keep)
        parts = [tokens(n) for n in lens]
        for b, n in enumerate(lens):
            if n:
                seqs[b] = parts[b]
        hs = torch.cat(parts)
        for i, l in enumerate(hard):
            hs = l.prefill(hs, cache, i, step, lens, cos, sin)
        row = 0
        for b, n in enumerate(lens):
            if n:
                assert_close(f32(hs[row:row + n]), f32(_reference(cfg, soft, seqs[b].double(), cos, sin)),
                             what=f"prompt of {n}")
            row += n

    prefill([5, 130, 64])
    for t in range(11):
        if t == 6:  # request 0 ends; its row starts again
            prefill([33, 0, 0], keep=[0] + cache.lens.tolist()[1:])
        new = [1, 1, 0 if t % 4 == 2 else 1]
        step = cache.step(new, rows_each=1)
        hs = tokens(3)
        for b in range(3):
            if new[b]:
                seqs[b] = torch.cat([seqs[b], hs[b:b + 1]])
        for i, l in enumerate(hard):
            hs = l.decode(hs, cache, i, step, cos, sin)
        assert cache.lens.tolist() == [len(s) for s in seqs]
        for b in range(3):
            if new[b]:
                want = _reference(cfg, soft, seqs[b].double(), cos, sin)[-1:]
                assert_close(f32(hs[b:b + 1]), f32(want), what=f"step {t} request {b}")
    held = sum(-(-len(s) // 16) for s in seqs)
    assert int(cache.free_count) == cache.num_pages - held


def test_captured_step(dev):
    """A step of two layers captured once and replayed with other tokens and counts, eager steps of
    another batch and synchronisations in between, against the same steps run eagerly, bit for bit."""
    cfg, hard, _ = _layers(dev, CFGS["d128"])
    cos, sin = layer.rope_tables(128, cfg.head_dim, cfg.rope_theta, dev)
    caches = [decode.PagedKVCache(2, 4, 128, cfg.kv_heads, cfg.head_dim, page_size=16, device=dev)
              for _ in range(3)]
    new = torch.ones(4, dtype=torch.int32, device=dev)
    hs = torch.zeros(4, cfg.hidden, dtype=torch.bfloat16, device=dev)

    def one(cache, x, n):
        step = cache.step(n, rows_each=1)
        for i, l in enumerate(hard):
            x = l.decode(x, cache, i, step, cos, sin)
        return x

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(caches[2], hs, new)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one(caches[0], hs, new)
    g = torch.Generator().manual_seed(4)
    for t in range(30):
        x = torch.randn(4, cfg.hidden, generator=g).to(torch.bfloat16).to(dev)
        n = torch.tensor([1, t % 2, 1, 1 if t > 9 else 0], dtype=torch.int32, device=dev)
        want = one(caches[1], x, n)
        hs.copy_(x)
        new.copy_(n)
        graph.replay()
        if t % 3 == 0:
            one(caches[2], x, n)
        if t % 5 == 0:
            torch.cuda.synchronize()
        live = n.bool()
        assert torch.equal(out[live], want[live]), t
        assert torch.equal(caches[0].lens, caches[1].lens)


def test_layer_without_lora(dev):
    """A layer whose linears have no LoRA equals one whose LoRA is zero, bit for bit."""
    cfg, hard, _ = _layers(dev, CFGS["d128"], 1)
    cos, sin = layer.rope_tables(64, cfg.head_dim, cfg.rope_theta, dev)
    names, norms = decode.HardDecoderLayer.NAMES, decode.HardDecoderLayer.NORMS
    parts = {n: [getattr(hard[0], f"{n}_{p}") for p in ("packed", "palette", "lora_a", "lora_b")]
             for n in names}
    norms = {n: getattr(hard[0], n) for n in norms}
    outs = []
    for lora in (False, True):
        l = decode.HardDecoderLayer(cfg, {n: (*p[:2], p[2] if lora else None,
                                              torch.zeros_like(p[3]) if lora else None)
                                          for n, p in parts.items()}, norms)
        cache = decode.PagedKVCache(1, 2, 64, cfg.kv_heads, cfg.head_dim, device=dev)
        g = torch.Generator().manual_seed(9)
        out = []
        for _ in range(3):
            step = cache.step([1, 1], rows_each=1)
            hs = torch.randn(2, cfg.hidden, generator=g).to(torch.bfloat16).to(dev)
            out.append(l.decode(hs, cache, 0, step, cos, sin))
        outs.append(torch.cat(out))
    assert torch.equal(*outs)


def test_pages_run_out_and_come_back(dev):
    """A pool smaller than its requests: what found no page is not in lens, and a request that ends
    makes room."""
    cache = decode.PagedKVCache(1, 3, 64, 2, 64, page_size=16, num_pages=4, device=dev)
    cache.step([40, 20, 5])
    assert cache.lens.tolist() == [40, 16, 0] and int(cache.free_count) == 0
    step = cache.step([0, 4, 5], keep=[0, 16, 0])
    assert cache.lens.tolist() == [0, 20, 5] and int(cache.free_count) == 1
    assert int((step.slots >= 0).sum()) == 9


@pytest.mark.parametrize("kw", CFGS.values(), ids=CFGS.keys())
def test_prompts_without_room(dev, kw):
    """Prompts of 40, 20 and 5 tokens on a pool of four pages of 16: the second has room for 16, the third
    for none. Rows with room are the rows of a pool with room for all, bit for bit, and right in 64 bits;
    the others are NaN, whatever other requests have in the pages that stale table entries name."""
    cfg, hard, soft = _layers(dev, kw)
    cos, sin = layer.rope_tables(64, cfg.head_dim, cfg.rope_theta, dev)
    lens, have = [40, 20, 5], [40, 16, 0]
    g = torch.Generator().manual_seed(3)
    hs = torch.randn(sum(lens), cfg.hidden, generator=g).to(torch.bfloat16).to(dev)
    outs = []
    for pages in (None, 4):
        cache = decode.PagedKVCache(2, 3, 64, cfg.kv_heads, cfg.head_dim, page_size=16, num_pages=pages,
                                    device=dev)
        step, x = cache.step(lens), hs
        for i, l in enumerate(hard):
            x = l.prefill(x, cache, i, step, lens, cos, sin)
        assert cache.lens.tolist() == (have if pages else lens)
        outs.append(x)
    full, got = outs
    row = 0
    for n, m in zip(lens, have):
        assert torch.equal(got[row:row + m], full[row:row + m])
        assert bool(torch.isnan(got[row + m:row + n]).all())
        if m:
            want = _reference(cfg, soft, hs[row:row + m].double(), cos, sin)
            assert_close(f32(got[row:row + m]), f32(want), what=f"prompt of {n}")
        row += n


@pytest.mark.parametrize("kw", CFGS.values(), ids=CFGS.keys())
def test_prompts_over_cached_tokens_are_marked(dev, kw):
    """prefill is for requests without cached tokens: the rows of one that has some are NaN, the others
    as they are alone."""
    cfg, hard, _ = _layers(dev, kw, 1)
    cos, sin = layer.rope_tables(64, cfg.head_dim, cfg.rope_theta, dev)
    g = torch.Generator().manual_seed(7)
    hs = torch.randn(29, cfg.hidden, generator=g).to(torch.bfloat16).to(dev)
    outs = []
    for first in ([0, 0], [3, 0]):
        cache = decode.PagedKVCache(1, 2, 64, cfg.kv_heads, cfg.head_dim, page_size=16, device=dev)
        step = cache.step(first)
        hard[0].prefill(hs[:sum(first)], cache, 0, step, first, cos, sin) if sum(first) else None
        step = cache.step([12, 17])
        outs.append(hard[0].prefill(hs, cache, 0, step, [12, 17], cos, sin))
    assert bool(torch.isfinite(outs[0]).all())
    assert bool(torch.isnan(outs[1][:12]).all())
    assert torch.equal(outs[1][12:], outs[0][12:])


def test_layers_refuse_gradients(dev):
    """decode and prefill have no backward: a hidden state, or a table, that needs a gradient is refused
    where gradients are on, and taken under no_grad."""
    cfg, hard, _ = _layers(dev, CFGS["d128"], 1)
    cos, sin = layer.rope_tables(64, cfg.head_dim, cfg.rope_theta, dev)
    cache = decode.PagedKVCache(1, 2, 64, cfg.kv_heads, cfg.head_dim, page_size=16, device=dev)
    hs = torch.randn(5, cfg.hidden, device=dev).to(torch.bfloat16)
    step = cache.step([3, 2])
    first = hard[0].prefill(hs, cache, 0, step, [3, 2], cos, sin)
    needs = hs.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        hard[0].prefill(needs, cache, 0, step, [3, 2], cos, sin)
    with pytest.raises(RuntimeError, match="no backward"):
        hard[0].prefill(hs, cache, 0, step, [3, 2], cos=cos.clone().requires_grad_(), sin=sin)
    with torch.no_grad():
        assert torch.equal(hard[0].prefill(needs, cache, 0, step, [3, 2], cos, sin), first)
    step = cache.step([1, 1], rows_each=1)
    with pytest.raises(RuntimeError, match="no backward"):
        hard[0].decode(needs[:2], cache, 0, step, cos, sin)
    with torch.no_grad():
        got = hard[0].decode(needs[:2], cache, 0, step, cos, sin)
    assert not got.requires_grad
    assert torch.equal(got, hard[0].decode(hs[:2], cache, 0, step, cos, sin))


def test_captured_prompts(dev):
    """A step of prompts (of 20, 0 and 7 tokens, on rows that had others) and two layers over them, captured
    once and replayed with other hidden states, eager work and synchronisations in between, against the same
    run eagerly, bit for bit; with a pool that has room for all, and one in which the last finds none."""
    cfg, hard, _ = _layers(dev, CFGS["d128"])
    cos, sin = layer.rope_tables(64, cfg.head_dim, cfg.rope_theta, dev)
    lens = [20, 0, 7]
    new = torch.tensor(lens, dtype=torch.int32, device=dev)
    keep = torch.zeros_like(new)
    for pages in (8, 2):
        caches = [decode.PagedKVCache(2, 3, 64, cfg.kv_heads, cfg.head_dim, page_size=16, num_pages=pages,
                                      device=dev) for _ in range(2)]
        hs = torch.zeros(27, cfg.hidden, dtype=torch.bfloat16, device=dev)

        def one(cache, x):
            step = cache.step(new, keep, rows=27)
            for i, l in enumerate(hard):
                x = l.prefill(x, cache, i, step, lens, cos, sin)
            return x

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            one(caches[1], hs)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = one(caches[0], hs)
        g = torch.Generator().manual_seed(6)
        for t in range(12):
            x = torch.randn(27, cfg.hidden, generator=g).to(torch.bfloat16).to(dev)
            want = one(caches[1], x)
            hs.copy_(x)
            graph.replay()
            if t % 3 == 0:
                torch.cuda.synchronize()
            rows = 27 if pages == 8 else 20
            assert torch.equal(out[:rows], want[:rows]), t
            assert bool(torch.isfinite(out[:rows]).all()) and bool(torch.isnan(out[rows:]).all())
            assert torch.equal(caches[0].lens, caches[1].lens)
