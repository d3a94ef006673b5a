"""Decoding with palettized decoder layers over a paged key-value cache.

  PagedKVCache      the pages of a batch of requests, who holds which, and the layers' keys and values
  HardDecoderLayer  a PalettizedDecoderLayer for inference: indices frozen to 2 bits (packed), LoRA
                    beside them, prompts through the layer step's causal attention, new tokens through
                    attention over the cache

One step of a batch (B requests, one new token each; row b of every tensor is request b):

  step = cache.step(new, rows_each=1)            # pages, slots and positions for the new tokens
  for i, layer in enumerate(layers):
      hs = layer.decode(hs, cache, i, step, cos, sin)

All of it runs on the device and in the same buffers every time, so a step can be captured into a graph
(new: a device tensor that the caller fills). There is no backward.
"""
from __future__ import annotations

import functools
from collections import namedtuple

import torch
import torch.nn as nn

from . import ops
from .layer import LayerConfig, PalettizedDecoderLayer, attention

# where a step's token rows go (ops.paged_step): int32 [rows], [rows], [batch + 1]
Step = namedtuple("Step", "slots positions starts")


def _no_grad(*args):
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in args):
        raise RuntimeError("decoding has no backward: call it under torch.no_grad()")


def _inference(fn):
    """The method under no_grad, after a refusal of arguments that need a gradient where they are on."""
    @functools.wraps(fn)
    def run(self, *args, **kw):
        _no_grad(*args, *kw.values())
        with torch.no_grad():
            return fn(self, *args, **kw)
    return run


class PagedKVCache:
    """Keys and values of `layers` layers for up to `batch` requests of up to `max_tokens` tokens, in
    `num_pages` pages of `page_size` tokens that the requests share (default: enough for all at their
    longest). lens [batch] are the tokens that each request has; a request starts with its first new
    tokens and ends with keep = 0, which hands its pages back."""

    def __init__(self, layers, batch, max_tokens, kv_heads, head_dim, page_size=64, num_pages=None,
                 device="cuda"):
        width = -(-max_tokens // page_size)
        num_pages = batch * width if num_pages is None else num_pages
        if layers < 1 or batch < 1 or max_tokens < 1 or num_pages < 1:
            raise ValueError("a cache needs layers, requests, tokens and pages")
        self.page_size, self.num_pages = page_size, num_pages
        caches = [ops.paged_cache(num_pages, page_size, kv_heads, head_dim, device)
                  for _ in range(layers)]
        self.k, self.v = [list(c) for c in zip(*caches)]
        kw = dict(dtype=torch.int32, device=device)
        self.block_table = torch.zeros(batch, width, **kw)
        self.lens = torch.zeros(batch, **kw)
        self.free_pages = torch.arange(num_pages, **kw)
        self.free_count = torch.full((1,), num_pages, **kw)

    def _ints(self, v):
        return v if v is None or isinstance(v, torch.Tensor) else torch.tensor(
            v, dtype=torch.int32, device=self.lens.device)

    def step(self, new_tokens, keep=None, rows=None, rows_each=0):
        """Room for new_tokens [batch] (int32 tensor, or a list) more tokens of each request, of whose
        cached ones the first keep [batch] stay (None: all). The tokens' rows follow each other in the
        order of the requests (rows of them; default: their sum for lists, batch for tensors), or every
        request owns rows_each rows. Updates lens; a request that found no page has fewer tokens than
        asked for there."""
        if rows is None and not rows_each and not isinstance(new_tokens, torch.Tensor):
            rows = sum(max(0, n) for n in new_tokens)
        slots, positions, starts, _, _ = ops.paged_step(
            self.lens, self._ints(new_tokens), self.block_table, self.free_pages, self.free_count,
            self.page_size, keep=self._ints(keep), rows=rows, rows_each=rows_each,
            lens_out=self.lens, free_count_out=self.free_count)
        return Step(slots, positions, starts)

    def write(self, layer, q, k, v, cos, sin, step, q_weight=None, k_weight=None, eps=1e-6):
        """The step's q, k, v rows [rows, heads, head_dim] through norm and rotation, k and v into layer
        `layer`'s pages; returns q (ops.paged_rope_write)."""
        _no_grad(q, k, v)
        return ops.paged_rope_write(q, k, v, cos, sin, step.positions, step.slots, self.k[layer],
                                    self.v[layer], q_weight, k_weight, eps)

    def attend(self, layer, q, scale=None):
        """Attention of one new token a request, q [batch, heads, head_dim], over layer `layer`'s cached
        tokens (ops.paged_attn); zeros for requests without tokens."""
        _no_grad(q)
        return ops.paged_attn(q, self.k[layer], self.v[layer], self.block_table, self.lens, scale)[0]

    def tokens(self, layer, request, n):
        """Keys and values [n, kv_heads, head_dim] of the first n tokens of a request, copied out. Rows
        past the tokens that it has are zeros: its table's entries there name nothing, or pages of
        others."""
        batch, width = self.block_table.shape
        if not (0 <= request < batch and 0 <= n <= width * self.page_size):
            raise ValueError(f"no {n} tokens of request {request} in a cache of {batch} requests of "
                             f"{width * self.page_size}")
        k, v = self.k[layer], self.v[layer]
        t = torch.arange(n, device=v.device)
        page = self.block_table[request, t // self.page_size].long().clamp(0, self.num_pages - 1)
        at, none = t % self.page_size, (t >= self.lens[request])[:, None, None]
        return (k[page, :, :, at].reshape(n, v.shape[1], v.shape[3]).masked_fill_(none, 0),
                v[page, :, at].masked_fill_(none, 0))


class HardDecoderLayer(nn.Module):
    """One decoder layer on packed 2-bit weights for inference.

    ``linears``: {name: (packed int32 [N, K/16], palette fp32 [N, K/256, 4], lora_a bf16 [r, K] or None,
    lora_b bf16 [N, r] or None)} for PalettizedDecoderLayer.NAMES; ``norms``: bf16 weights of
    input_layernorm, post_attention_layernorm, q_norm and k_norm."""

    NAMES = PalettizedDecoderLayer.NAMES
    NORMS = ("input_layernorm", "post_attention_layernorm", "q_norm", "k_norm")

    def __init__(self, cfg: LayerConfig, linears, norms, lora_scale=1.0):
        super().__init__()
        self.cfg, self.lora_scale = cfg, float(lora_scale)
        for name in self.NAMES:
            for part, t in zip(("packed", "palette", "lora_a", "lora_b"), linears[name]):
                self.register_buffer(f"{name}_{part}", None if t is None else t.detach().contiguous())
        for name in self.NORMS:
            self.register_buffer(name, norms[name].detach().contiguous())

    @classmethod
    @torch.no_grad()
    def from_soft(cls, layer: PalettizedDecoderLayer):
        """The trained layer with its indices frozen: the largest logit of each weight, the first of
        equal ones (as extract_hard_indices takes it), LoRA kept apart."""
        linears = {}
        for name in cls.NAMES:
            lin = getattr(layer, name)
            packed = ops.pack_indices(lin.index_logits.argmax(-1).to(torch.uint8))
            linears[name] = (packed, lin.palette.clone(), lin.lora_a.clone(), lin.lora_b.clone())
        norms = {n: getattr(layer, n).weight.clone() for n in cls.NORMS}
        return cls(layer.cfg, linears, norms, layer.q_proj.lora_scale)

    def _linear(self, name, x, residual=None):
        a, b = getattr(self, name + "_lora_a"), getattr(self, name + "_lora_b")
        t = None if a is None else ops.lora_project(x, a, self.lora_scale)
        y = ops.lut_linear_fwd(x, getattr(self, name + "_packed"), getattr(self, name + "_palette"), None,
                               t, b)
        return y if residual is None else y + residual

    def _rows(self, hs, cache, index, step, cos, sin, attend):
        """The layer on token rows hs [rows, hidden]; attend(q, v) is the attention's part."""
        cfg = self.cfg
        hs = hs.contiguous()
        x, _ = ops.rmsnorm_fwd(hs, self.input_layernorm, cfg.eps)
        q, k, v = (self._linear(n, x).view(-1, h, cfg.head_dim)
                   for n, h in (("q_proj", cfg.heads), ("k_proj", cfg.kv_heads),
                                ("v_proj", cfg.kv_heads)))
        q = cache.write(index, q, k, v, cos, sin, step, self.q_norm, self.k_norm, cfg.eps)
        o = self._linear("o_proj", attend(q, v).reshape(-1, cfg.heads * cfg.head_dim))
        hs, x, _ = ops.add_rmsnorm_fwd(hs, o, self.post_attention_layernorm, cfg.eps)
        h = ops.swiglu_fwd(self._linear("gate_proj", x), self._linear("up_proj", x))
        return self._linear("down_proj", h, hs)

    @_inference
    def decode(self, hs, cache, index, step, cos, sin):
        """One new token a request: hs bf16 [batch, hidden], step from cache.step(..., rows_each=1),
        cos, sin fp32 [positions, head_dim] (layer.rope_tables). A request that got no token in this
        step has its row computed from its cached tokens alone; that row means nothing."""
        return self._rows(hs, cache, index, step, cos, sin, lambda q, v: cache.attend(index, q))

    @_inference
    def prefill(self, hs, cache, index, step, lens, cos, sin):
        """Prompts: hs bf16 [sum(lens), hidden], the requests' rows one after another; lens, a list, is
        what cache.step was given as new_tokens for requests without cached tokens. Whole sequences go
        through the training layers' causal attention on the keys that the cache holds. Rows of tokens that
        found no room (slot -1) are NaN: their keys are nowhere, and later tokens would lack them. So are
        the rows of a request that had cached tokens: its prompt's tokens are not its first ones."""
        cfg = self.cfg
        if hs.shape[0] != sum(lens):
            raise ValueError(f"hs has {hs.shape[0]} rows, the prompts have {sum(lens)} tokens")

        def attend(q, v):
            # rows that are not their request's first tokens, or have no slot
            at = torch.arange(q.shape[0], dtype=torch.int32, device=q.device)
            if len([n for n in lens if n]) > 1:
                at = at - step.starts[torch.searchsorted(step.starts, at, right=True) - 1]
            slots = step.slots.long()
            dead = (step.positions != at).logical_or_(slots < 0)[:, None, None]
            # the other rows' keys back from their slots; what is 0 times a dead row's value has to be 0
            k, P = cache.k[index], cache.page_size
            slots.clamp_(0, cache.num_pages * P - 1)
            k = k[slots // P, :, :, slots % P].view(v.shape).masked_fill_(dead, 0)
            v.masked_fill_(dead, 0)
            o, row = [q[:0]], 0
            for n in lens:
                if n == 0:
                    continue
                # the kernel takes multiples of 128; rows behind a sequence's last do not reach it
                pad = -n % 128 if cfg.head_dim == 128 else 0
                qkv = [nn.functional.pad(t[row:row + n], (0, 0, 0, 0, 0, pad))[None] for t in (q, k, v)]
                y = attention(*qkv, cfg.heads, cfg.kv_heads)
                o.append(y[0, :n].view(n, cfg.heads, cfg.head_dim))
                row += n
            return torch.cat(o).masked_fill_(dead, float("nan"))

        return self._rows(hs, cache, index, step, cos, sin, attend)
