"""Tensor-level wrappers of the C ABI (one function per entry point).

PyTorch provides device memory and the current HIP stream; all arithmetic runs in the HIP
kernels of libpalettize_hip.so. Outputs and workspaces are allocated here (the library
never allocates). Inputs must be CUDA (HIP) tensors; nothing falls back to the CPU.

Native layout (the one the kernels use):
  packed  int32 [N, K/16]      2-bit indices, 16 per word along K, LSB first
  palette fp32  [N, K/256, 4]  per output row and per 256 input columns
  logits  bf16/fp16 [N, K, 4], noise fp32 [N, K, 4]
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib
from ._lib import call, query

_DT = {torch.bfloat16: _lib.PLZ_DT_BF16, torch.float16: _lib.PLZ_DT_FP16,
       torch.float32: _lib.PLZ_DT_FP32}


def _stream(t: torch.Tensor) -> int:
    # the raw handle, without a Stream object (2 us less per call)
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _on_gpu(t: torch.Tensor) -> bool:
    return t.is_cuda


def _need(t: torch.Tensor, name: str, dtype=None, ndim=None) -> torch.Tensor:
    if (isinstance(t, torch.Tensor) and t.is_cuda and (dtype is None or t.dtype == dtype)
            and (ndim is None or t.dim() == ndim) and t.is_contiguous()):
        return t
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not _on_gpu(t):
        raise RuntimeError(f"{name} must be a GPU tensor (palettize_hip has no CPU path)")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must be {ndim}-D, got shape {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=device)


def _opt_workspace(nbytes: int, device):
    """An optional workspace: None (NULL) when the query asks for none."""
    return torch.empty(int(nbytes), dtype=torch.uint8, device=device) if nbytes > 0 else None


def _numel(t) -> int:
    return 0 if t is None else t.numel()


def _bias(bias, N: int):
    """bias must be None or bf16 [N]: the C ABI takes no bias length, the epilogue reads N."""
    if bias is None:
        return None
    _need(bias, "bias", torch.bfloat16, 1)
    if bias.numel() != N:
        raise ValueError(f"bias has {bias.numel()} elements, the output has N={N} columns")
    return bias


# ---- formats ------------------------------------------------------------------------
def pack_indices(idx: torch.Tensor) -> torch.Tensor:
    """uint8 [rows, cols] (0..3) -> int32 [rows, cols/16], LSB first."""
    _need(idx, "idx", torch.uint8, 2)
    rows, cols = idx.shape
    out = torch.empty((rows, cols // 16), dtype=torch.int32, device=idx.device)
    call("plz_pack_indices", _ptr(idx), _ptr(out), rows, cols, _stream(idx))
    return out


def unpack_indices(packed: torch.Tensor) -> torch.Tensor:
    _need(packed, "packed", torch.int32, 2)
    rows, words = packed.shape
    out = torch.empty((rows, words * 16), dtype=torch.uint8, device=packed.device)
    call("plz_unpack_indices", _ptr(packed), _ptr(out), rows, words * 16, _stream(packed))
    return out


def _wshape(packed: torch.Tensor, palette: torch.Tensor):
    _need(packed, "packed", torch.int32, 2)
    _need(palette, "palette", torch.float32, 3)
    N, K = packed.shape[0], packed.shape[1] * 16
    if tuple(palette.shape) != (N, K // 256, 4):
        raise ValueError(f"palette shape {tuple(palette.shape)} != {(N, K // 256, 4)}")
    return N, K


def dequant(packed: torch.Tensor, palette: torch.Tensor) -> torch.Tensor:
    N, K = _wshape(packed, palette)
    w = torch.empty((N, K), dtype=torch.bfloat16, device=packed.device)
    call("plz_dequant", _ptr(packed), _ptr(palette), _ptr(w), N, K, _stream(packed))
    return w


# ---- reference-layout palettes ----------------------------------------------------------
def palette_expand(palette, N: int, kg: int, group_size: int):
    """(G, 4) palette -> native fp32 [N, kg, 4], row n from group n // group_size."""
    _need(palette, "palette", None, 2)
    if palette.dtype not in _DT or palette.shape[1] != 4:
        raise TypeError("palette must be (G, 4) bf16, fp16 or fp32")
    if palette.shape[0] * int(group_size) < N:
        raise ValueError(f"palette has {palette.shape[0]} groups of {group_size} for {N} rows")
    out = torch.empty((N, kg, 4), dtype=torch.float32, device=palette.device)
    call("plz_palette_expand", _ptr(palette), _DT[palette.dtype], _ptr(out), N, kg,
         int(group_size), _stream(palette))
    return out


def palette_fold(grad, n_groups: int, group_size: int, dtype=torch.float32):
    """native fp32 [N, kg, 4] -> (n_groups, 4): the sum over a group's rows and over kg, in fp32;
    groups without rows are zero."""
    _need(grad, "grad", torch.float32, 3)
    N, kg = grad.shape[0], grad.shape[1]
    if n_groups * int(group_size) < N:
        raise ValueError(f"{n_groups} groups of {group_size} for {N} rows")
    out = torch.empty((n_groups, 4), dtype=dtype, device=grad.device)
    call("plz_palette_fold", _ptr(grad), _ptr(out), _DT[dtype], int(n_groups), N, kg,
         int(group_size), _stream(grad))
    return out


# ---- hard linear --------------------------------------------------------------------
def _lora_pair(a, b, first: str, second: str, rows_a: int, rows_b: int):
    if (a is None) != (b is None):
        raise ValueError(f"{first} and {second} must be given together")
    if a is None:
        return 0
    _need(a, first, torch.bfloat16, 2)
    _need(b, second, torch.bfloat16, 2)
    r = a.shape[1]
    if a.shape[0] != rows_a or b.shape[1] != r or b.shape[0] != rows_b:
        raise ValueError(f"{first} {tuple(a.shape)} / {second} {tuple(b.shape)} mismatch")
    return r


def lut_linear_staged(M: int, N: int, K: int, grad_x: bool = False) -> bool:
    """True when the hard forward at this size is fastest with W dequantised once and a dense GEMM
    on it (grad_x by itself: lut_linear_staged(M, K, N)); grad_x: that W serves the pass's grad_x
    too."""
    return query("plz_lut_linear_staged_pair" if grad_x else "plz_lut_linear_staged", M, N, K) != 0


def lut_linear_fwd(x, packed, palette, bias=None, lora_t=None, lora_b=None, staged=True):
    """y = x W^T (+ bias) (+ lora_t lora_b^T).

    staged: W dequantised into the workspace and a dense GEMM on it where that is faster
    (lut_linear_staged); False keeps the one-pass LUT GEMM (workspace for its tail partials
    only)."""
    N, K = _wshape(packed, palette)
    _need(x, "x", torch.bfloat16, 2)
    M = x.shape[0]
    if x.shape[1] != K:
        raise ValueError(f"x has {x.shape[1]} columns, W has K={K}")
    _bias(bias, N)
    rank = _lora_pair(lora_t, lora_b, "lora_t", "lora_b", M, N)
    y = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    q = "plz_lut_linear_fwd_tiled_workspace" if staged else "plz_linear_fwd_dense_workspace"
    ws = _opt_workspace(query(q, M, N, K), x.device)
    call("plz_lut_linear_fwd_tiled" if staged else "plz_lut_linear_fwd", _ptr(x), _ptr(packed), _ptr(palette), _ptr(bias), _ptr(lora_t),
         _ptr(lora_b), rank, _ptr(y), _ptr(ws), _numel(ws), M, N, K, _stream(x))
    return y


def lut_linear_bwd_x(grad_y, packed, palette, lora_gt=None, lora_a=None, staged=True):
    """grad_x = grad_y W (+ lora_gt lora_a).

    staged: W dequantised into the workspace and a dense GEMM on it where that is faster
    (lut_linear_staged); False keeps the one-pass LUT GEMM (workspace for its tail partials
    only)."""
    N, K = _wshape(packed, palette)
    _need(grad_y, "grad_y", torch.bfloat16, 2)
    M = grad_y.shape[0]
    if grad_y.shape[1] != N:
        raise ValueError("grad_y columns != N")
    rank = 0
    if lora_gt is not None or lora_a is not None:
        if lora_gt is None or lora_a is None:
            raise ValueError("lora_gt and lora_a must be given together")
        _need(lora_gt, "lora_gt", torch.bfloat16, 2)
        _need(lora_a, "lora_a", torch.bfloat16, 2)
        rank = lora_gt.shape[1]
        if lora_gt.shape[0] != M or tuple(lora_a.shape) != (rank, K):
            raise ValueError("lora_gt / lora_a shape mismatch")
    gx = torch.empty((M, K), dtype=torch.bfloat16, device=grad_y.device)
    q = "plz_lut_linear_bwd_x_tiled_workspace" if staged else "plz_linear_bwd_x_dense_workspace"
    ws = _opt_workspace(query(q, M, N, K), grad_y.device)
    call("plz_lut_linear_bwd_x_tiled" if staged else "plz_lut_linear_bwd_x", _ptr(grad_y), _ptr(packed), _ptr(palette), _ptr(lora_gt),
         _ptr(lora_a), rank, _ptr(gx), _ptr(ws), _numel(ws), M, N, K, _stream(grad_y))
    return gx


def lut_linear_bwd_palette(x, grad_y, packed):
    """fp32 [N, K/256, 4]: per-class sums of (grad_y^T x)[n, k] over each 256-k group."""
    _need(packed, "packed", torch.int32, 2)
    _need(x, "x", torch.bfloat16, 2)
    _need(grad_y, "grad_y", torch.bfloat16, 2)
    N, K = packed.shape[0], packed.shape[1] * 16
    M = x.shape[0]
    if x.shape[1] != K or tuple(grad_y.shape) != (M, N):
        raise ValueError("x / grad_y shape mismatch")
    out = torch.empty((N, K // 256, 4), dtype=torch.float32, device=x.device)
    nbytes = query("plz_lut_linear_bwd_palette_workspace", M, N, K)
    ws = _workspace(nbytes, x.device)
    call("plz_lut_linear_bwd_palette", _ptr(x), _ptr(grad_y), _ptr(packed), _ptr(out), _ptr(ws),
         ws.numel(), M, N, K, _stream(x))
    return out


def lut_linear_bwd_palette_lora(x, grad_y, packed, lora_a, lora_b, scale: float = 1.0,
                                out_dtype=torch.bfloat16):
    """(grad_palette, grad_a [r, K], grad_b [N, r]) from one dW GEMM: the palette gradient as
    lut_linear_bwd_palette, and the LoRA weight gradients scale * lora_b^T dW and
    scale * dW lora_a^T (dW = grad_y^T x), which lora_weight_grads computes from t and gt."""
    _need(packed, "packed", torch.int32, 2)
    for name, v in (("x", x), ("grad_y", grad_y), ("lora_a", lora_a), ("lora_b", lora_b)):
        _need(v, name, torch.bfloat16, 2)
    N, K = packed.shape[0], packed.shape[1] * 16
    M = x.shape[0]
    r = lora_a.shape[0]
    if x.shape[1] != K or tuple(grad_y.shape) != (M, N):
        raise ValueError("x / grad_y shape mismatch")
    if tuple(lora_a.shape) != (r, K) or tuple(lora_b.shape) != (N, r):
        raise ValueError("lora_a must be [r, K] and lora_b [N, r]")
    out = torch.empty((N, K // 256, 4), dtype=torch.float32, device=x.device)
    ga = torch.empty((r, K), dtype=out_dtype, device=x.device)
    gb = torch.empty((N, r), dtype=out_dtype, device=x.device)
    ws = _workspace(query("plz_lut_linear_bwd_palette_lora_workspace", M, N, K, r), x.device)
    call("plz_lut_linear_bwd_palette_lora", _ptr(x), _ptr(grad_y), _ptr(packed), _ptr(lora_a),
         _ptr(lora_b), r, float(scale), _ptr(out), _ptr(ga), _ptr(gb), _DT[out_dtype], _ptr(ws),
         ws.numel(), M, N, K, _stream(x))
    return out, ga, gb


def lut_linear_bwd_palette_noalloc(x, grad_y, packed, out=None):
    """lut_linear_bwd_palette through the entry point that allocates nothing (its split-M
    partials live in a fixed device array of the library; calls that overlap on one GPU race).
    ``out`` (fp32 [N, K/256, 4]) may be passed in so that the call allocates nothing here
    either."""
    _need(packed, "packed", torch.int32, 2)
    _need(x, "x", torch.bfloat16, 2)
    _need(grad_y, "grad_y", torch.bfloat16, 2)
    N, K = packed.shape[0], packed.shape[1] * 16
    M = x.shape[0]
    if x.shape[1] != K or tuple(grad_y.shape) != (M, N):
        raise ValueError("x / grad_y shape mismatch")
    if out is None:
        out = torch.empty((N, K // 256, 4), dtype=torch.float32, device=x.device)
    _need(out, "out", torch.float32, 3)
    if tuple(out.shape) != (N, K // 256, 4):
        raise ValueError(f"out must be [{N}, {K // 256}, 4]")
    call("plz_lut_linear_bwd_palette_noalloc", _ptr(x), _ptr(grad_y), _ptr(packed), _ptr(out),
         M, N, K, _stream(x))
    return out


def bias_grad(grad_y):
    _need(grad_y, "grad_y", torch.bfloat16, 2)
    M, N = grad_y.shape
    out = torch.empty((N,), dtype=torch.float32, device=grad_y.device)
    call("plz_bias_grad", _ptr(grad_y), _ptr(out), M, N, _stream(grad_y))
    return out


# ---- dense linear -----------------------------------------------------------------------
def swiglu_weight(w_gate, w_up):
    """[N, K] gate and up weights -> the [2N, K] interleave of plz_linear_fwd_dense_swiglu
    (128 gate rows, the 128 matching up rows, ...). N must be a multiple of 128."""
    N, K = w_gate.shape
    if w_up.shape != (N, K) or N % 128:
        raise ValueError("gate / up must be the same [N, K] with N a multiple of 128")
    return torch.stack([w_gate.reshape(N // 128, 128, K), w_up.reshape(N // 128, 128, K)],
                       dim=1).reshape(2 * N, K).contiguous()


def linear_fwd_dense_swiglu(x, w_gate_up):
    """h = silu(x Wg^T) * (x Wu^T) in one GEMM (w_gate_up from swiglu_weight)."""
    _need(x, "x", torch.bfloat16, 2)
    _need(w_gate_up, "w_gate_up", torch.bfloat16, 2)
    M, K = x.shape
    N = w_gate_up.shape[0] // 2
    if w_gate_up.shape[1] != K:
        raise ValueError("x / w shape mismatch")
    h = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    call("plz_linear_fwd_dense_swiglu", _ptr(x), _ptr(w_gate_up), _ptr(h), M, N, K, _stream(x))
    return h


def linear_fwd_dense_swiglu_cat(x, w, lora_t=None, lora_b=None, keep_pre=True):
    """(y, h): y = x w^T (+ lora_t lora_b^T) for w = [Wg; Wu] of 2F rows, and h = silu(y[:, :F])
    * y[:, F:] from the same GEMM (plz_linear_fwd_dense_swiglu_cat); y is None unless
    keep_pre. Bit-equal to linear_fwd_dense followed by swiglu_fwd_cat."""
    _need(x, "x", torch.bfloat16, 2)
    _need(w, "w", torch.bfloat16, 2)
    M, K = x.shape
    F = w.shape[0] // 2
    if w.shape[1] != K or w.shape[0] != 2 * F:
        raise ValueError("x / w shape mismatch")
    rank = _lora_pair(lora_t, lora_b, "lora_t", "lora_b", M, 2 * F)
    y = torch.empty((M, 2 * F), dtype=torch.bfloat16, device=x.device) if keep_pre else None
    h = torch.empty((M, F), dtype=torch.bfloat16, device=x.device)
    call("plz_linear_fwd_dense_swiglu_cat", _ptr(x), _ptr(w), _ptr(lora_t), _ptr(lora_b), rank,
         _ptr(y), _ptr(h), M, F, K, _stream(x))
    return y, h


def linear_fwd_dense(x, w, bias=None, lora_t=None, lora_b=None, residual=None, tiled=False):
    """y = x w^T (+ bias) (+ lora_t lora_b^T); with residual (bf16 [M, N]) y = residual + that,
    added in the GEMM's epilogue with the rounding of a separate bf16 add
    (plz_linear_fwd_dense_residual). tiled: on whichever GEMM core is the faster one for the shape
    (plz_linear_fwd_tiled), whose sums over K may run in another order."""
    _need(x, "x", torch.bfloat16, 2)
    _need(w, "w", torch.bfloat16, 2)
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError("x / w shape mismatch")
    _bias(bias, N)
    rank = _lora_pair(lora_t, lora_b, "lora_t", "lora_b", M, N)
    y = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    if residual is not None:
        _need(residual, "residual", torch.bfloat16, 2)
        if tuple(residual.shape) != (M, N):
            raise ValueError(f"residual must be [M, N] = [{M}, {N}]")
    if tiled:
        ws = _opt_workspace(query("plz_linear_tiled_workspace", M, N, K), x.device)
        call("plz_linear_fwd_tiled", _ptr(x), _ptr(w), _ptr(bias), _ptr(lora_t), _ptr(lora_b),
             rank, _ptr(residual), _ptr(y), _ptr(ws), _numel(ws), M, N, K, _stream(x))
        return y
    ws = _opt_workspace(query("plz_linear_fwd_dense_workspace", M, N, K), x.device)
    if residual is not None:
        call("plz_linear_fwd_dense_residual", _ptr(x), _ptr(w), _ptr(bias), _ptr(lora_t),
             _ptr(lora_b), rank, _ptr(residual), _ptr(y), _ptr(ws), _numel(ws), M, N, K,
             _stream(x))
        return y
    call("plz_linear_fwd_dense", _ptr(x), _ptr(w), _ptr(bias), _ptr(lora_t), _ptr(lora_b), rank,
         _ptr(y), _ptr(ws), _numel(ws), M, N, K, _stream(x))
    return y


def linear_fwd_dense_kn(x, w, bias=None):
    """y = x w (+ bias) for a weight stored [K, N]."""
    _need(x, "x", torch.bfloat16, 2)
    _need(w, "w", torch.bfloat16, 2)
    M, K = x.shape
    N = w.shape[1]
    if w.shape[0] != K:
        raise ValueError("x / w shape mismatch")
    _bias(bias, N)
    y = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    ws = _opt_workspace(query("plz_linear_tiled_workspace", M, N, K), x.device)
    call("plz_linear_fwd_dense_kn", _ptr(x), _ptr(w), _ptr(bias), _ptr(y), _ptr(ws), _numel(ws), M,
         N, K, _stream(x))
    return y


def linear_bwd_x_dense(grad_y, w, lora_gt=None, lora_a=None, tiled=False):
    """grad_x = grad_y w (+ lora_gt lora_a); tiled as in linear_fwd_dense."""
    _need(grad_y, "grad_y", torch.bfloat16, 2)
    _need(w, "w", torch.bfloat16, 2)
    M, N = grad_y.shape
    K = w.shape[1]
    if w.shape[0] != N:
        raise ValueError("grad_y / w shape mismatch")
    rank = 0
    if lora_gt is not None or lora_a is not None:
        if lora_gt is None or lora_a is None:
            raise ValueError("lora_gt and lora_a must be given together")
        _need(lora_gt, "lora_gt", torch.bfloat16, 2)
        _need(lora_a, "lora_a", torch.bfloat16, 2)
        rank = lora_gt.shape[1]
        if lora_gt.shape[0] != M or tuple(lora_a.shape) != (rank, K):
            raise ValueError("lora_gt / lora_a shape mismatch")
    gx = torch.empty((M, K), dtype=torch.bfloat16, device=grad_y.device)
    if tiled:
        ws = _opt_workspace(query("plz_linear_tiled_workspace", M, K, N), grad_y.device)
        call("plz_linear_bwd_x_tiled", _ptr(grad_y), _ptr(w), _ptr(lora_gt), _ptr(lora_a), rank,
             _ptr(gx), _ptr(ws), _numel(ws), M, N, K, _stream(grad_y))
        return gx
    ws = _opt_workspace(query("plz_linear_bwd_x_dense_workspace", M, N, K), grad_y.device)
    call("plz_linear_bwd_x_dense", _ptr(grad_y), _ptr(w), _ptr(lora_gt), _ptr(lora_a), rank,
         _ptr(gx), _ptr(ws), _numel(ws), M, N, K, _stream(grad_y))
    return gx


def linear_bwd_x_dense_swiglu(grad_y, w, gate_up, lora_gt=None, lora_a=None):
    """[grad_gate | grad_up] [M, 2K] of h = silu(gate) * up (gate_up [M, 2K] its pre-activations)
    for grad_h = grad_y w (+ lora_gt lora_a), with the SwiGLU backward in the GEMM's epilogue:
    bit for bit swiglu_bwd_cat(gate_up, linear_bwd_x_dense(...)), grad_h never stored."""
    _need(grad_y, "grad_y", torch.bfloat16, 2)
    _need(w, "w", torch.bfloat16, 2)
    _need(gate_up, "gate_up", torch.bfloat16, 2)
    M, N = grad_y.shape
    K = w.shape[1]
    if w.shape[0] != N or tuple(gate_up.shape) != (M, 2 * K):
        raise ValueError("grad_y [M, N], w [N, K] and gate_up [M, 2K] expected")
    rank = 0
    if lora_gt is not None or lora_a is not None:
        if lora_gt is None or lora_a is None:
            raise ValueError("lora_gt and lora_a must be given together")
        _need(lora_gt, "lora_gt", torch.bfloat16, 2)
        _need(lora_a, "lora_a", torch.bfloat16, 2)
        rank = lora_gt.shape[1]
        if lora_gt.shape[0] != M or tuple(lora_a.shape) != (rank, K):
            raise ValueError("lora_gt / lora_a shape mismatch")
    out = torch.empty((M, 2 * K), dtype=torch.bfloat16, device=grad_y.device)
    ws = _opt_workspace(query("plz_linear_bwd_x_dense_workspace", M, N, K), grad_y.device)
    call("plz_linear_bwd_x_dense_swiglu", _ptr(grad_y), _ptr(w), _ptr(lora_gt), _ptr(lora_a),
         rank, _ptr(gate_up), _ptr(out), _ptr(ws), _numel(ws), M, N, K, _stream(grad_y))
    return out


# ---- soft path ------------------------------------------------------------------------
def gumbel_philox(shape, seed: int, offset: int = 0, device="cuda"):
    n = 1
    for s in shape:
        n *= int(s)
    out = torch.empty(tuple(shape), dtype=torch.float32, device=device)
    call("plz_gumbel_philox", _ptr(out), n, int(seed) & (2**64 - 1), int(offset) & (2**64 - 1),
         _stream(out))
    return out


def gumbel_lcg(N: int, K: int, seed: int, device="cuda", variant: str = "cuda"):
    """The reference's LCG Gumbel noise [N, K, 4], element (n, k, c) drawn at
    idx (k*N + n)*4 + c: the CUDA hash (variant "cuda") or the Triton one ("triton")."""
    if variant not in ("cuda", "triton"):
        raise ValueError(f"unknown LCG variant {variant!r}")
    out = torch.empty((N, K, 4), dtype=torch.float32, device=device)
    call("plz_gumbel_lcg_triton" if variant == "triton" else "plz_gumbel_lcg", _ptr(out),
         int(seed) & 0xFFFFFFFF, N, K, _stream(out))
    return out


def soft_pw_reference_batched(logits_list, palette_list, group_size: int, tau: float,
                              step_seed: int):
    """[P_aos_0, W_0, P_aos_1, W_1, ...] of the reference's fused_compute_P_W_batched
    (fused_lut_linear_cuda.py:513-607) from one launch: logits (4, K, N) fp16 and palettes
    (G, 4) bf16 with G = N / group_size, in and out in the reference's layouts; layer i draws
    its LCG noise with seed step_seed ^ (i * 0x9E3779B9)."""
    n = len(logits_list)
    if n == 0:
        raise ValueError("logits_list must be non-empty")
    if len(palette_list) != n:
        raise ValueError("palette_list size must match logits_list size")
    if n > 64:
        raise ValueError(f"max 64 layers in batched kernel (got {n})")
    group_size = int(group_size)
    if group_size <= 0:
        raise ValueError("group_size must be positive")
    descs = (_lib.PwRefDesc * n)()
    outs, held = [], []  # held: realigned palette copies, alive until the launch is queued
    dev = logits_list[0].device
    for i, (lg, pal) in enumerate(zip(logits_list, palette_list)):
        _need(lg, f"logits[{i}]", torch.float16, 3)
        _need(pal, f"palette[{i}]", torch.bfloat16, 2)
        if lg.shape[0] != 4:
            raise ValueError(f"logits[{i}] must be (4, K, N)")
        if pal.shape[1] != 4:
            raise ValueError(f"palette[{i}] must be (G, 4)")
        if lg.device != dev or pal.device != dev:
            raise ValueError("all tensors must be on one device")
        K, N = lg.shape[1], lg.shape[2]
        if N % group_size:
            raise ValueError(f"layer {i}: N={N} not divisible by group_size={group_size}")
        if N // group_size != pal.shape[0]:
            raise ValueError(f"layer {i}: G mismatch (N/GS={N // group_size} vs "
                             f"palette.size(0)={pal.shape[0]})")
        if pal.data_ptr() % 8:
            pal = pal.clone()
            held.append(pal)
        P = torch.empty((K, N, 4), dtype=torch.float16, device=dev)
        w = torch.empty((K, N), dtype=torch.bfloat16, device=dev)
        outs += [P, w]
        descs[i] = _lib.PwRefDesc(lg.data_ptr(), pal.data_ptr(), P.data_ptr(), w.data_ptr(), K, N,
                                  0, i, 0)
    total = _lib.lib().plz_pw_ref_plan(descs, n, group_size)
    if total < 0:
        raise _lib.PalettizeError("plz_pw_ref_plan failed: " + _lib.lib().plz_last_error().decode())
    raw = bytes(C.string_at(C.addressof(descs), C.sizeof(descs)))
    table = torch.frombuffer(bytearray(raw), dtype=torch.uint8).to(dev)
    call("plz_soft_pw_ref_batched", table.data_ptr(), n, int(total), group_size, float(tau),
         int(step_seed) & 0xFFFFFFFF, torch.cuda.current_stream(dev).cuda_stream)
    return outs


def _soft_ref_shapes(logits, palette, group_size):
    """(K, N) of reference-layout logits (4, K, N) and palette (G, 4)."""
    if logits.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("logits must be bf16 or fp16")
    _need(logits, "logits", None, 3)
    _need(palette, "palette", None, 2)
    if palette.dtype not in _DT:
        raise TypeError("palette must be bf16, fp16 or fp32")
    if logits.shape[0] != 4 or palette.shape[1] != 4:
        raise ValueError("logits (4, K, N) and palette (G, 4) expected")
    K, N = logits.shape[1], logits.shape[2]
    if palette.shape[0] * int(group_size) < N:
        raise ValueError(f"palette has {palette.shape[0]} groups of {group_size} for {N} columns")
    return K, N


def soft_ref_build_w(logits, palette, group_size: int, seed: int, tau: float, mode: int,
                     variant: str = "cuda", copy=None):
    """W [K, N] bf16 of reference-layout logits (4, K, N) and palette (G, 4), the LCG noise of
    gumbel_lcg(variant=...) drawn in the kernel: the transpose of what soft_build_w makes of the
    native-layout tensors. K and N multiples of 8. copy (like logits): the logits as read."""
    K, N = _soft_ref_shapes(logits, palette, group_size)
    if copy is not None:
        _need(copy, "copy", logits.dtype, 3)
        if copy.shape != logits.shape:
            raise ValueError("copy must have the logits' shape")
    w = torch.empty((K, N), dtype=torch.bfloat16, device=logits.device)
    call("plz_soft_ref_build_w_copy", _ptr(logits), _DT[logits.dtype], _ptr(palette),
         _DT[palette.dtype], int(group_size), int(variant == "triton"), int(seed) & 0xFFFFFFFF,
         float(tau), int(mode), _ptr(w), _ptr(copy), K, N, _stream(logits))
    return w


def soft_ref_bwd(x, grad_y, logits, palette, group_size: int, seed: int, tau: float,
                 variant: str = "cuda", want_logits: bool = True):
    """(grad_logits (4, K, N) or None, grad_palette (G, 4)) of the reference-layout soft linear, in
    the logits' and the palette's types: soft_bwd with the noise drawn again in the kernel."""
    K, N = _soft_ref_shapes(logits, palette, group_size)
    _need(x, "x", torch.bfloat16, 2)
    _need(grad_y, "grad_y", torch.bfloat16, 2)
    M = x.shape[0]
    if x.shape[1] != K or tuple(grad_y.shape) != (M, N):
        raise ValueError("x / grad_y shape mismatch")
    gl = torch.empty_like(logits) if want_logits else None
    gp = torch.empty_like(palette)
    ws = _workspace(query("plz_soft_ref_bwd_workspace", M, N, K), x.device)
    call("plz_soft_ref_bwd", _ptr(x), _ptr(grad_y), _ptr(logits), _DT[logits.dtype], _ptr(palette),
         _DT[palette.dtype], palette.shape[0], int(group_size), int(variant == "triton"),
         int(seed) & 0xFFFFFFFF, float(tau), 0, _ptr(gl), _ptr(gp), _ptr(ws), ws.numel(), M, N, K,
         _stream(x))
    return gl, gp


class PhiloxNoise:
    """Gumbel noise drawn inside the soft kernels instead of a tensor: the values
    gumbel_philox(shape, seed, offset) would hold (Philox counter offset + n*K + k for the 4
    classes of weight (n, k)). Accepted wherever a noise tensor [N, K, 4] is."""

    def __init__(self, seed: int, offset: int):
        self.seed, self.offset = int(seed), int(offset)

    def materialize(self, N: int, K: int, device):
        return gumbel_philox((N, K, 4), seed=self.seed, offset=self.offset, device=device)


def _soft_shapes(logits, noise, palette, probs=None):
    """noise may be None only where the forward's P (probs) replaces it."""
    if logits.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("logits must be bf16 or fp16")
    _need(logits, "logits", None, 3)
    _need(palette, "palette", torch.float32, 3)
    N, K, four = logits.shape
    if noise is None:
        if probs is None:
            raise ValueError("noise is needed unless the forward's P (probs) is given")
    elif not isinstance(noise, PhiloxNoise):
        _need(noise, "noise", torch.float32, 3)
        if tuple(noise.shape) != (N, K, 4):
            raise ValueError("logits [N,K,4], noise [N,K,4], palette [N,K/256,4] expected")
    if four != 4 or tuple(palette.shape) != (N, K // 256, 4):
        raise ValueError("logits [N,K,4], noise [N,K,4], palette [N,K/256,4] expected")
    return N, K


def soft_build_w(logits, noise, palette, tau: float, mode: int = _lib.PLZ_W_HARD_NOISY,
                 want_soft: bool = False, probs=None):
    """(w, w_soft or None). probs (optional fp16 [N, K, 4]) also receives
    P = softmax((logits + noise) / tau), which soft_bwd(probs=...) reads in the backward."""
    N, K = _soft_shapes(logits, noise, palette)
    if probs is not None:
        _need(probs, "probs", torch.float16, 3)
        if tuple(probs.shape) != (N, K, 4):
            raise ValueError(f"probs must be [N, K, 4] = [{N}, {K}, 4]")
    w = torch.empty((N, K), dtype=torch.bfloat16, device=logits.device)
    ws = torch.empty((N, K), dtype=torch.bfloat16, device=logits.device) if want_soft else None
    if isinstance(noise, PhiloxNoise):
        call("plz_soft_build_w_philox", _ptr(logits), _DT[logits.dtype], noise.seed, noise.offset,
             _ptr(palette), float(tau), int(mode), _ptr(w), _ptr(ws), _ptr(probs), N, K,
             _stream(logits))
    else:
        call("plz_soft_build_w", _ptr(logits), _DT[logits.dtype], _ptr(noise), _ptr(palette),
             float(tau), int(mode), _ptr(w), _ptr(ws), _ptr(probs), N, K, _stream(logits))
    return w, ws


class SoftBuildGroup:
    """The forward weights of several soft linears built by one launch
    (plz_soft_build_w_batched_philox). ``items`` is a list of (logits, noise, palette), where
    noise is an fp32 [N, K, 4] tensor or a ``PhiloxNoise`` whose seed is that linear's Philox
    key (its noise is then drawn in the kernel at the counter offset given to ``run``). The
    outputs (w and, with want_soft, w_soft) are allocated once and rewritten by every run;
    ``generation`` counts the runs. With want_probs, every run also writes each linear's
    P = softmax((logits + noise) / tau) as fp16 [N, K, 4] into ``probs[i]``, which
    soft_bwd_lora(probs=...) reads in the backward."""

    def __init__(self, items, mode: int = _lib.PLZ_W_HARD_NOISY, want_soft: bool = False,
                 want_probs: bool = False):
        if not items:
            raise ValueError("empty build group")
        self.mode = int(mode)
        self.device = items[0][0].device
        self.outputs = []
        self.probs = []
        self.generation = 0
        descs = (_lib.BuildWDesc * len(items))()
        for i, (logits, noise, palette) in enumerate(items):
            N, K = _soft_shapes(logits, noise, palette)
            w = torch.empty((N, K), dtype=torch.bfloat16, device=self.device)
            ws = torch.empty((N, K), dtype=torch.bfloat16, device=self.device) if want_soft else None
            pr = (torch.empty((N, K, 4), dtype=torch.float16, device=self.device) if want_probs
                  else None)
            self.outputs.append((w, ws))
            self.probs.append(pr)
            philox = isinstance(noise, PhiloxNoise)
            descs[i] = _lib.BuildWDesc(logits.data_ptr(), None if philox else noise.data_ptr(),
                                       palette.data_ptr(), w.data_ptr(),
                                       ws.data_ptr() if ws is not None else None,
                                       N, K, _DT[logits.dtype], 0, 0,
                                       (noise.seed & (2**64 - 1)) if philox else 0, 0,
                                       pr.data_ptr() if pr is not None else None)
        self._keep = items
        total = _lib.lib().plz_build_w_plan(descs, len(items))
        if total < 0:
            raise _lib.PalettizeError(
                "plz_build_w_plan failed: " + _lib.lib().plz_last_error().decode())
        self.total_blocks = int(total)
        raw = bytes(C.string_at(C.addressof(descs), C.sizeof(descs)))
        self.table = torch.frombuffer(bytearray(raw), dtype=torch.uint8).to(self.device)
        self.n = len(items)

    def run(self, tau: float, noise_offset: int = 0):
        call("plz_soft_build_w_batched_philox", self.table.data_ptr(), self.n, self.total_blocks,
             int(noise_offset) & (2**64 - 1), float(tau), self.mode,
             torch.cuda.current_stream(self.device).cuda_stream)
        self.generation += 1
        return self.outputs


def soft_bwd(x, grad_y, logits, noise, palette, tau: float, scale_by_inv_tau: bool = False,
             probs=None):
    """(grad_logits, grad_palette). probs (optional fp16 [N, K, 4], the forward's P from
    soft_build_w(probs=...)) is read instead of logits and noise (plz_soft_bwd_probs), as the
    reference's backward reads its saved P_aos; logits and noise then give only the shapes and
    the gradient's dtype (noise may then be None)."""
    N, K = _soft_shapes(logits, noise, palette, probs)
    _need(x, "x", torch.bfloat16, 2)
    _need(grad_y, "grad_y", torch.bfloat16, 2)
    M = x.shape[0]
    if x.shape[1] != K or tuple(grad_y.shape) != (M, N):
        raise ValueError("x / grad_y shape mismatch")
    gl = torch.empty_like(logits)
    gp = torch.empty((N, K // 256, 4), dtype=torch.float32, device=x.device)
    ws = _workspace(query("plz_soft_bwd_workspace", M, N, K), x.device)
    if probs is not None:
        _need(probs, "probs", torch.float16, 3)
        if tuple(probs.shape) != (N, K, 4):
            raise ValueError(f"probs must be [N, K, 4] = [{N}, {K}, 4]")
        call("plz_soft_bwd_probs", _ptr(x), _ptr(grad_y), _ptr(probs), _ptr(palette), float(tau),
             int(bool(scale_by_inv_tau)), _ptr(gl), _DT[logits.dtype], _ptr(gp), _ptr(ws),
             ws.numel(), M, N, K, _stream(x))
    elif isinstance(noise, PhiloxNoise):
        call("plz_soft_bwd_philox", _ptr(x), _ptr(grad_y), _ptr(logits), _DT[logits.dtype],
             noise.seed, noise.offset, _ptr(palette), float(tau), int(bool(scale_by_inv_tau)),
             _ptr(gl), _ptr(gp), _ptr(ws), ws.numel(), M, N, K, _stream(x))
    else:
        call("plz_soft_bwd", _ptr(x), _ptr(grad_y), _ptr(logits), _DT[logits.dtype], _ptr(noise),
             _ptr(palette), float(tau), int(bool(scale_by_inv_tau)), _ptr(gl), _ptr(gp), _ptr(ws),
             ws.numel(), M, N, K, _stream(x))
    return gl, gp


def soft_bwd_lora(x, grad_y, logits, noise, palette, tau: float, lora_a, lora_b,
                  scale: float = 1.0, scale_by_inv_tau: bool = False, out_dtype=torch.bfloat16,
                  grad_sq=None, probs=None):
    """(grad_logits, grad_palette, grad_a [r, K], grad_b [N, r]) from one dW GEMM: the soft
    backward as soft_bwd (bit for bit), and the LoRA weight gradients scale * lora_b^T dW and
    scale * dW lora_a^T (dW = grad_y^T x), which lora_weight_grads computes from t and gt.
    grad_sq (optional fp32 [N * K / 128]) receives the sum of squares of each 512 consecutive
    grad_logits values, for FusedAdamW.step(grad_sq=...). probs (optional fp16 [N, K, 4]): the
    forward's P (SoftBuildGroup(want_probs=True)), read instead of redrawing the noise (noise
    may then be None)."""
    N, K = _soft_shapes(logits, noise, palette, probs)
    if probs is not None:
        _need(probs, "probs", torch.float16, 3)
        if tuple(probs.shape) != (N, K, 4):
            raise ValueError(f"probs must be [N, K, 4] = [{N}, {K}, 4]")
    if grad_sq is not None:
        _need(grad_sq, "grad_sq", torch.float32, 1)
        if grad_sq.numel() != N * K // 128:
            raise ValueError(f"grad_sq must hold N*K/128 = {N * K // 128} floats")
    for name, v in (("x", x), ("grad_y", grad_y), ("lora_a", lora_a), ("lora_b", lora_b)):
        _need(v, name, torch.bfloat16, 2)
    M = x.shape[0]
    r = lora_a.shape[0]
    if x.shape[1] != K or tuple(grad_y.shape) != (M, N):
        raise ValueError("x / grad_y shape mismatch")
    if tuple(lora_a.shape) != (r, K) or tuple(lora_b.shape) != (N, r):
        raise ValueError("lora_a must be [r, K] and lora_b [N, r]")
    gl = torch.empty_like(logits)
    gp = torch.empty((N, K // 256, 4), dtype=torch.float32, device=x.device)
    ga = torch.empty((r, K), dtype=out_dtype, device=x.device)
    gb = torch.empty((N, r), dtype=out_dtype, device=x.device)
    ws = _workspace(query("plz_soft_bwd_lora_workspace", M, N, K, r), x.device)
    philox = isinstance(noise, PhiloxNoise)
    call("plz_soft_bwd_lora", _ptr(x), _ptr(grad_y), _ptr(logits), _DT[logits.dtype],
         None if philox else _ptr(noise), noise.seed if philox else 0,
         noise.offset if philox else 0, _ptr(probs), _ptr(palette), float(tau),
         int(bool(scale_by_inv_tau)), _ptr(lora_a), _ptr(lora_b), r, float(scale), _ptr(gl),
         _ptr(gp), _ptr(ga), _ptr(gb), _DT[out_dtype], _ptr(grad_sq), _ptr(ws), ws.numel(), M, N,
         K, _stream(x))
    return gl, gp, ga, gb


# ---- LoRA -----------------------------------------------------------------------------
def lora_project(x, lora_a, scale: float):
    """t = scale * x lora_a^T, lora_a [r, K]."""
    _need(x, "x", torch.bfloat16, 2)
    _need(lora_a, "lora_a", torch.bfloat16, 2)
    M, K = x.shape
    r = lora_a.shape[0]
    if lora_a.shape[1] != K:
        raise ValueError("lora_a must be [r, K]")
    t = torch.empty((M, r), dtype=torch.bfloat16, device=x.device)
    call("plz_lora_project", _ptr(x), _ptr(lora_a), float(scale), _ptr(t), M, K, r, _stream(x))
    return t


def lora_grad_t(grad_y, lora_b, scale: float):
    """gt = scale * grad_y lora_b, lora_b [N, r]."""
    _need(grad_y, "grad_y", torch.bfloat16, 2)
    _need(lora_b, "lora_b", torch.bfloat16, 2)
    M, N = grad_y.shape
    r = lora_b.shape[1]
    if lora_b.shape[0] != N:
        raise ValueError("lora_b must be [N, r]")
    gt = torch.empty((M, r), dtype=torch.bfloat16, device=grad_y.device)
    call("plz_lora_grad_t", _ptr(grad_y), _ptr(lora_b), float(scale), _ptr(gt), M, N, r,
         _stream(grad_y))
    return gt


def lora_weight_grads(x, grad_y, t, gt, scale: float = 1.0, out_dtype=torch.float32):
    """grad_a [r, K] = gt^T x ; grad_b [N, r] = scale * grad_y^T t."""
    for name, v in (("x", x), ("grad_y", grad_y), ("t", t), ("gt", gt)):
        _need(v, name, torch.bfloat16, 2)
    M, K = x.shape
    N = grad_y.shape[1]
    r = t.shape[1]
    ga = torch.empty((r, K), dtype=out_dtype, device=x.device)
    gb = torch.empty((N, r), dtype=out_dtype, device=x.device)
    ws = _workspace(query("plz_lora_weight_grads_workspace", M, N, K, r), x.device)
    call("plz_lora_weight_grads", _ptr(x), _ptr(grad_y), _ptr(t), _ptr(gt), float(scale),
         _ptr(ga), _ptr(gb), _DT[out_dtype], _ptr(ws), ws.numel(), M, N, K, r, _stream(x))
    return ga, gb


# ---- decode GEMV ------------------------------------------------------------------------
def lut_gemv(x, packed, palette):
    N, K = _wshape(packed, palette)
    _need(x, "x", torch.bfloat16, 2)
    M = x.shape[0]
    if x.shape[1] != K:
        raise ValueError("x / W shape mismatch")
    y = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    call("plz_lut_gemv", _ptr(x), _ptr(packed), _ptr(palette), _ptr(y), M, N, K, _stream(x))
    return y


def gemv_pack_palettes(palette):
    """One-time decode layout of a palette [N, K/256, 4] (plz_gemv_pack_palettes): per 128-row
    item, group and row the two 32-bit lookup words of the bf16-rounded entries (low bytes, then
    high bytes), [ceil(N/128), K/256, 128, 2]. Returned as a flat int32 tensor."""
    _need(palette, "palette", torch.float32, 3)
    N, G = palette.shape[0], palette.shape[1]
    nbytes = query("plz_gemv_palette_items_bytes", N, G * 256)
    out = torch.empty(max(nbytes // 4, 4), dtype=torch.int32, device=palette.device)
    call("plz_gemv_pack_palettes", _ptr(palette), _ptr(out), N, G * 256, _stream(palette))
    return out


def gemv_pack_indices(packed):
    """One-time decode layout of packed indices [N, K/16] (plz_gemv_pack_indices): one
    contiguous 8 KB block per 128-row item and 256-k stage, fields permuted for natural-order
    dequantisation. Returned as a flat int32 tensor."""
    _need(packed, "packed", torch.int32, 2)
    N, K = packed.shape[0], packed.shape[1] * 16
    nbytes = query("plz_gemv_packed_items_bytes", N, K)
    out = torch.empty(max(nbytes // 4, 4), dtype=torch.int32, device=packed.device)
    call("plz_gemv_pack_indices", _ptr(packed), _ptr(out), N, K, _stream(packed))
    return out


def gemv_pack_planes(packed):
    """One-time planes layout of packed indices [N, K/16] (plz_gemv_pack_planes) for the
    bit-plane GEMV: the decode layout's 8 KB blocks per 128-row item and 256-k stage, each
    lane's words those of k = 128h + 32j .. +31 (h = 0, 1), a word's nibble i holding the
    indices of k0 + i and k0 + 8 + i. Returned as a flat int32 tensor."""
    _need(packed, "packed", torch.int32, 2)
    N, K = packed.shape[0], packed.shape[1] * 16
    nbytes = query("plz_gemv_packed_items_bytes", N, K)
    out = torch.empty(max(nbytes // 4, 4), dtype=torch.int32, device=packed.device)
    call("plz_gemv_pack_planes", _ptr(packed), _ptr(out), N, K, _stream(packed))
    return out


def lut_gemv_planes(x, planes_items, palette_items, N):
    """lut_gemv on weights in the planes layout (gemv_pack_planes, gemv_pack_palettes): the
    bit-plane FP8 x FP4 MFMA GEMV, with its x pieces in a workspace allocated here."""
    _need(x, "x", torch.bfloat16, 2)
    M, K = x.shape
    if planes_items.numel() * 4 < query("plz_gemv_packed_items_bytes", N, K) or \
            palette_items.numel() * 4 < query("plz_gemv_palette_items_bytes", N, K):
        raise ValueError("planes-layout weights smaller than N x K needs")
    y = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    ws = _opt_workspace(query("plz_gemv_planes_workspace", 1, K, M), x.device)
    call("plz_lut_gemv_planes", _ptr(x), _ptr(planes_items), _ptr(palette_items), _ptr(y), M, N,
         K, _ptr(ws), _numel(ws), _stream(x))
    return y


def lut_gemv_decode(x, packed_items, palette_items, N):
    """lut_gemv on weights in the decode layouts (gemv_pack_indices, gemv_pack_palettes)."""
    _need(x, "x", torch.bfloat16, 2)
    M, K = x.shape
    if packed_items.numel() * 4 < query("plz_gemv_packed_items_bytes", N, K) or \
            palette_items.numel() * 4 < query("plz_gemv_palette_items_bytes", N, K):
        raise ValueError("decode-layout weights smaller than N x K needs")
    y = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    call("plz_lut_gemv_decode", _ptr(x), _ptr(packed_items), _ptr(palette_items), _ptr(y), M, N,
         K, _stream(x))
    return y


class GemvGroup:
    """A fixed set of independent GEMVs (same M) run by one grouped launch.

    ``items`` is a list of (x [M,K] bf16, packed, palette); outputs are allocated once and
    reused by every ``run()``. The descriptor table lives in device memory. ``layout``:
    "auto" (default: "planes" up to 8 tokens, where one FP8 operand holds every token's two x
    pieces, "decode" above), "decode" (indices and palettes repacked once into the decode
    layouts, plz_gemv_pack_indices / plz_gemv_pack_palettes, streamed contiguously and
    dequantised to bf16), "planes" (the bit-plane MFMA GEMV on plz_gemv_pack_planes indices, with
    a workspace for the x pieces) or "native" (the packed indices and fp32 palettes as given).
    ``prepack=False`` is "native".
    """

    LAYOUTS = {"native": _lib.PLZ_GEMV_NATIVE, "decode": _lib.PLZ_GEMV_DECODE,
               "planes": _lib.PLZ_GEMV_PLANES}

    def __init__(self, items, prepack=True, layout=None):
        if not items:
            raise ValueError("empty GEMV group")
        self.M = items[0][0].shape[0]
        if layout is None:
            layout = "auto" if prepack else "native"
        if layout == "auto":
            layout = "planes" if self.M <= 8 else "decode"
        if layout not in self.LAYOUTS:
            raise ValueError(f"layout must be one of {sorted(self.LAYOUTS)}")
        prepack = layout != "native"
        self.M = items[0][0].shape[0]
        self.device = items[0][0].device
        self.outputs = []
        self._packed_palettes = []
        self._packed_indices = []
        descs = (_lib.GemvDesc * len(items))()
        for i, (x, packed, palette) in enumerate(items):
            N, K = _wshape(packed, palette)
            _need(x, "x", torch.bfloat16, 2)
            if x.shape != (self.M, K):
                raise ValueError(f"item {i}: x must be [{self.M}, {K}]")
            y = torch.empty((self.M, N), dtype=torch.bfloat16, device=self.device)
            self.outputs.append(y)
            pre = gemv_pack_palettes(palette) if prepack and N > 0 and K > 0 else None
            pack_i = gemv_pack_planes if layout == "planes" else gemv_pack_indices
            pri = pack_i(packed) if prepack and N > 0 and K > 0 else None
            self._packed_palettes.append(pre)
            self._packed_indices.append(pri)
            descs[i] = _lib.GemvDesc(x.data_ptr(), packed.data_ptr(), palette.data_ptr(),
                                     y.data_ptr(), N, K, 0, 0,
                                     pre.data_ptr() if pre is not None else None,
                                     pri.data_ptr() if pri is not None else None)
        self._keep = items
        self.layout = self.LAYOUTS[layout]
        self.max_K = max(int(it[1].shape[1]) * 16 for it in items)
        self.workspace = None
        if layout == "planes":
            self.workspace = _opt_workspace(
                query("plz_gemv_planes_workspace", len(items), self.max_K, self.M), self.device)
        total = _lib.lib().plz_gemv_plan(descs, len(items), self.M, self.layout)
        if total < 0:
            raise _lib.PalettizeError(
                "plz_gemv_plan failed: " + _lib.lib().plz_last_error().decode())
        self.total_blocks = int(total)
        raw = bytes(C.string_at(C.addressof(descs), C.sizeof(descs)))
        host = torch.frombuffer(bytearray(raw), dtype=torch.uint8)
        self.table = host.to(self.device)
        self.n = len(items)

    def run(self):
        stream = torch._C._cuda_getCurrentRawStream(self.device.index)
        if self.layout == _lib.PLZ_GEMV_PLANES:
            call("plz_lut_gemv_grouped_planes", self.table.data_ptr(), self.n, self.total_blocks,
                 self.M, self.max_K, _ptr(self.workspace), _numel(self.workspace), stream)
        else:
            call("plz_lut_gemv_grouped", self.table.data_ptr(), self.n, self.total_blocks,
                 self.M, self.layout, stream)
        return self.outputs


# ---- RMSNorm / SwiGLU -----------------------------------------------------------------------
def _norm_weight(weight, cols: int):
    _need(weight, "weight", torch.bfloat16, 1)
    if weight.numel() != cols:
        raise ValueError(f"weight has {weight.numel()} elements, rows have {cols} columns")


def rmsnorm_fwd(x, weight, eps: float):
    _need(x, "x", torch.bfloat16, 2)
    rows, cols = x.shape
    _norm_weight(weight, cols)
    y = torch.empty_like(x)
    rstd = torch.empty((rows,), dtype=torch.float32, device=x.device)
    call("plz_rmsnorm_fwd", _ptr(x), _ptr(weight), _ptr(y), _ptr(rstd), rows, cols, float(eps),
         _stream(x))
    return y, rstd


def add_rmsnorm_fwd(x, residual, weight, eps: float):
    """(sum = x + residual, rmsnorm(sum), rstd) in one pass; bf16 [rows, cols] inputs."""
    _need(x, "x", torch.bfloat16, 2)
    _need(residual, "residual", torch.bfloat16, 2)
    if residual.shape != x.shape:
        raise ValueError("x / residual shape mismatch")
    rows, cols = x.shape
    _norm_weight(weight, cols)
    s, y = torch.empty_like(x), torch.empty_like(x)
    rstd = torch.empty((rows,), dtype=torch.float32, device=x.device)
    call("plz_add_rmsnorm_fwd", _ptr(x), _ptr(residual), _ptr(weight), _ptr(s), _ptr(y),
         _ptr(rstd), rows, cols, float(eps), _stream(x))
    return s, y, rstd


def rmsnorm_bwd_add(x, weight, rstd, grad_y, grad_add):
    """rmsnorm_bwd's grad_x (bf16) + grad_add, without the weight gradient."""
    _need(x, "x", torch.bfloat16, 2)
    _need(grad_y, "grad_y", torch.bfloat16, 2)
    _need(grad_add, "grad_add", torch.bfloat16, 2)
    rows, cols = x.shape
    _norm_weight(weight, cols)
    if grad_y.shape != x.shape or grad_add.shape != x.shape or rstd.numel() != rows:
        raise ValueError("grad_y / grad_add / rstd do not match x")
    gx = torch.empty_like(x)
    call("plz_rmsnorm_bwd_add", _ptr(x), _ptr(weight), _ptr(rstd), _ptr(grad_y), _ptr(grad_add),
         _ptr(gx), rows, cols, _stream(x))
    return gx


def rmsnorm_bwd(x, weight, rstd, grad_y):
    _need(x, "x", torch.bfloat16, 2)
    _need(grad_y, "grad_y", torch.bfloat16, 2)
    rows, cols = x.shape
    _norm_weight(weight, cols)
    _need(rstd, "rstd", torch.float32, 1)
    if rstd.numel() != rows or grad_y.shape != x.shape:
        raise ValueError("rstd must be [rows] and grad_y the shape of x")
    gx = torch.empty_like(x)
    gw = torch.empty((cols,), dtype=torch.float32, device=x.device)
    ws = _workspace(query("plz_rmsnorm_bwd_workspace", rows, cols), x.device)
    call("plz_rmsnorm_bwd", _ptr(x), _ptr(weight), _ptr(rstd), _ptr(grad_y), _ptr(gx), _ptr(gw),
         _ptr(ws), ws.numel(), rows, cols, _stream(x))
    return gx, gw


def swiglu_fwd(gate, up):
    _need(gate, "gate", torch.bfloat16)
    _need(up, "up", torch.bfloat16)
    h = torch.empty_like(gate)
    call("plz_swiglu_fwd", _ptr(gate), _ptr(up), _ptr(h), gate.numel(), _stream(gate))
    return h


def swiglu_bwd(gate, up, grad_h):
    _need(gate, "gate", torch.bfloat16)
    _need(up, "up", torch.bfloat16)
    _need(grad_h, "grad_h", torch.bfloat16)
    gg = torch.empty_like(gate)
    gu = torch.empty_like(up)
    call("plz_swiglu_bwd", _ptr(gate), _ptr(up), _ptr(grad_h), _ptr(gg), _ptr(gu), gate.numel(),
         _stream(gate))
    return gg, gu


def swiglu_fwd_cat(gate_up):
    """h [..., F] = silu(gate) * up from a fused projection's output [..., 2F] = [gate | up]."""
    _need(gate_up, "gate_up", torch.bfloat16)
    F2 = gate_up.shape[-1]
    if F2 % 16:
        raise ValueError("gate_up: the last dimension must be 2F with F a multiple of 8")
    F = F2 // 2
    g = gate_up.reshape(-1, F2)
    h = torch.empty(gate_up.shape[:-1] + (F,), dtype=torch.bfloat16, device=gate_up.device)
    call("plz_swiglu_fwd_rows", _ptr(g), _ptr(g) + 2 * F, F2, _ptr(h), F, g.shape[0], F,
         _stream(gate_up))
    return h


def swiglu_bwd_cat(gate_up, grad_h):
    """[grad_gate | grad_up] [..., 2F] of swiglu_fwd_cat for the gradient grad_h [..., F]."""
    _need(gate_up, "gate_up", torch.bfloat16)
    _need(grad_h, "grad_h", torch.bfloat16)
    F2 = gate_up.shape[-1]
    F = F2 // 2
    if F2 % 16 or tuple(grad_h.shape) != tuple(gate_up.shape[:-1]) + (F,):
        raise ValueError("gate_up [..., 2F] and grad_h [..., F] expected, F a multiple of 8")
    g = gate_up.reshape(-1, F2)
    out = torch.empty_like(g)
    call("plz_swiglu_bwd_rows", _ptr(g), _ptr(g) + 2 * F, F2, _ptr(grad_h), F, _ptr(out),
         _ptr(out) + 2 * F, F2, g.shape[0], F, _stream(gate_up))
    return out.reshape(gate_up.shape)


# ---- layer step: RoPE and the distillation loss ----------------------------------------------
def _rope(name, x, cos, sin):
    _need(x, "x", torch.bfloat16)
    if x.dim() < 3 or not x.is_contiguous():
        raise ValueError("x must be contiguous [..., seq, heads, head_dim]")
    seq, heads, hd = x.shape[-3], x.shape[-2], x.shape[-1]
    for t, nm in ((cos, "cos"), (sin, "sin")):
        _need(t, nm, torch.float32, 2)
        if tuple(t.shape) != (seq, hd):
            raise ValueError(f"{nm} must be [seq={seq}, head_dim={hd}]")
    y = torch.empty_like(x)
    rows = x.numel() // (heads * hd)
    call(name, _ptr(x), _ptr(cos), _ptr(sin), _ptr(y), rows, seq, heads, hd, _stream(x))
    return y


def rope_fwd(x, cos, sin):
    """x bf16 [..., seq, heads, head_dim] -> x cos + rotate_half(x) sin (fp32 math, bf16 out)."""
    return _rope("plz_rope_fwd", x, cos, sin)


def rope_bwd(grad_y, cos, sin):
    return _rope("plz_rope_bwd", grad_y, cos, sin)


def _head_rows(x, cos, sin, what):
    _need(x, what, torch.bfloat16)
    if x.dim() < 3 or not x.is_contiguous():
        raise ValueError(f"{what} must be contiguous [..., seq, heads, head_dim]")
    seq, heads, hd = x.shape[-3], x.shape[-2], x.shape[-1]
    for t, nm in ((cos, "cos"), (sin, "sin")):
        _need(t, nm, torch.float32, 2)
        if tuple(t.shape) != (seq, hd):
            raise ValueError(f"{nm} must be [seq={seq}, head_dim={hd}]")
    return x.numel() // (heads * hd), seq, heads, hd


def head_norm_rope_fwd(x, weight, cos, sin, eps: float):
    """rope_fwd(rmsnorm over each head's head_dim values) in one pass, bit-identical to the two:
    x bf16 [..., seq, heads, 128] -> (y like x, rstd fp32 [x.numel() / 128])."""
    rows, seq, heads, hd = _head_rows(x, cos, sin, "x")
    _norm_weight(weight, hd)
    y = torch.empty_like(x)
    rstd = torch.empty((rows * heads,), dtype=torch.float32, device=x.device)
    call("plz_head_norm_rope_fwd", _ptr(x), _ptr(weight), _ptr(cos), _ptr(sin), _ptr(y),
         _ptr(rstd), rows, seq, heads, hd, float(eps), _stream(x))
    return y, rstd


def head_norm_rope_bwd(x, weight, rstd, cos, sin, grad_y):
    """grad_x of head_norm_rope_fwd (rope_bwd then rmsnorm_bwd, bit for bit; no weight gradient)."""
    rows, seq, heads, hd = _head_rows(x, cos, sin, "x")
    _norm_weight(weight, hd)
    _need(rstd, "rstd", torch.float32, 1)
    if grad_y.shape != x.shape or not grad_y.is_contiguous() or rstd.numel() != rows * heads:
        raise ValueError("grad_y / rstd do not match x")
    gx = torch.empty_like(x)
    call("plz_head_norm_rope_bwd", _ptr(x), _ptr(weight), _ptr(rstd), _ptr(cos), _ptr(sin),
         _ptr(grad_y), _ptr(gx), rows, seq, heads, hd, _stream(x))
    return gx


def distill_loss_fwd(student, teacher, w_cos=0.5, w_mse=0.5, eps=1e-4):
    """Returns (out4 fp32 [4] = loss, l_cos, t_var, l_mse; workspace for the backward)."""
    _need(student, "student", torch.bfloat16)
    _need(teacher, "teacher", torch.bfloat16)
    if student.shape != teacher.shape:
        raise ValueError("student / teacher shape mismatch")
    dim = student.shape[-1]
    rows = student.numel() // dim
    out = torch.empty(4, dtype=torch.float32, device=student.device)
    ws = _workspace(query("plz_distill_loss_workspace", rows), student.device)
    call("plz_distill_loss_fwd", _ptr(student), _ptr(teacher), float(w_cos), float(w_mse),
         float(eps), _ptr(out), _ptr(ws), ws.numel(), rows, dim, _stream(student))
    return out, ws


def distill_loss_bwd(student, teacher, out4, ws, grad_loss, w_cos=0.5, w_mse=0.5, eps=1e-4):
    dim = student.shape[-1]
    rows = student.numel() // dim
    gl = grad_loss.reshape(1).to(torch.float32).contiguous()
    gs = torch.empty_like(student)
    call("plz_distill_loss_bwd", _ptr(student), _ptr(teacher), _ptr(out4), _ptr(gl),
         float(w_cos), float(w_mse), float(eps), _ptr(gs), _ptr(ws), ws.numel(), rows, dim,
         _stream(student))
    return gs


# ---- attention ---------------------------------------------------------------------------------
def attn_fwd(q, k, v, scale=None):
    """Causal grouped-query attention. q [B, S, Hq, 128], k/v [B, S, Hkv, 128] bf16 ->
    (o [B, S, Hq, 128] bf16, lse [B, Hq, S] fp32)."""
    for t, nm in ((q, "q"), (k, "k"), (v, "v")):
        _need(t, nm, torch.bfloat16, 4)
    B, S, Hq, D = q.shape
    Hkv = k.shape[2]
    if tuple(k.shape) != (B, S, Hkv, D) or tuple(v.shape) != (B, S, Hkv, D):
        raise ValueError("q / k / v shape mismatch")
    scale = D ** -0.5 if scale is None else float(scale)
    o = torch.empty_like(q)
    lse = torch.empty((B, Hq, S), dtype=torch.float32, device=q.device)
    call("plz_attn_fwd", _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse), B, S, Hq, Hkv, D, scale,
         _stream(q))
    return o, lse


def attn_bwd(q, k, v, o, lse, grad_o, scale=None):
    """Backward of attn_fwd: (grad_q, grad_k, grad_v), bf16 in the shapes of q, k, v."""
    for t, nm in ((q, "q"), (k, "k"), (v, "v"), (o, "o"), (grad_o, "grad_o")):
        _need(t, nm, torch.bfloat16, 4)
    _need(lse, "lse", torch.float32, 3)
    B, S, Hq, D = q.shape
    Hkv = k.shape[2]
    if (tuple(k.shape) != (B, S, Hkv, D) or tuple(v.shape) != (B, S, Hkv, D)
            or o.shape != q.shape or grad_o.shape != q.shape or tuple(lse.shape) != (B, Hq, S)):
        raise ValueError("attention backward shape mismatch")
    scale = D ** -0.5 if scale is None else float(scale)
    gq, gk, gv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ws = _opt_workspace(query("plz_attn_bwd_workspace", B, S, Hq), q.device)
    call("plz_attn_bwd", _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(grad_o), _ptr(lse), _ptr(gq),
         _ptr(gk), _ptr(gv), _ptr(ws), _numel(ws), B, S, Hq, Hkv, D, scale, _stream(q))
    return gq, gk, gv


# ---- decoding over a paged key-value cache -----------------------------------------------------
def _on(dev, name, *args):
    """call() on device `dev`, with its current stream as the last argument."""
    args += (torch._C._cuda_getCurrentRawStream(dev),)
    if torch._C._cuda_getDevice() == dev:
        call(name, *args)
    else:
        with torch.cuda.device(dev):
            call(name, *args)


def _one_device(name, *tensors):
    """The device of the first tensor, which all others (or None) are on."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{name}: the tensors are on different devices")
    return dev


def _dense_int32(tensors):
    """The device that dense int32 GPU tensors share; -1 where they are not that (the checks that say
    what is wrong come after)."""
    dev = tensors[0].get_device() if isinstance(tensors[0], torch.Tensor) else -1
    for t in tensors:
        if not (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.get_device() == dev
                and t.is_contiguous()):
            return -1
    return dev


def _ints(t, name, *shape):
    """An int32 GPU tensor of that shape."""
    _need(t, name, torch.int32, len(shape))
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    return t


def _no_backward(name, *tensors):
    """Refuses tensors (or None) that need a gradient, where gradients are on."""
    # one call of torch for all of them: 0.3 us, a loop over the properties 1.1
    if torch.is_grad_enabled() and torch._C._any_requires_grad(*tensors):
        raise RuntimeError(f"{name} has no backward: call it under torch.no_grad()")


def paged_cache(num_pages, page_size, kv_heads, head_dim, device):
    """(k_cache, v_cache) of one layer, zeros: bf16 [num_pages, kv_heads, head_dim / 8, page_size, 8]
    and [num_pages, kv_heads, page_size, head_dim]."""
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two of 16 to 1024, got {page_size}")
    if head_dim not in (64, 128, 256):
        raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
    kw = dict(dtype=torch.bfloat16, device=device)
    return (torch.zeros(num_pages, kv_heads, head_dim // 8, page_size, 8, **kw),
            torch.zeros(num_pages, kv_heads, page_size, head_dim, **kw))


_BF16 = torch.bfloat16


def _paged_caches(k_cache, v_cache):
    """(num_pages, kv_heads, page_size, head_dim) of a layer's cache."""
    if (isinstance(v_cache, torch.Tensor) and isinstance(k_cache, torch.Tensor) and v_cache.dim() == 4
            and v_cache.is_cuda and v_cache.dtype is _BF16 and k_cache.dtype is _BF16
            and v_cache.is_contiguous() and k_cache.is_contiguous() and k_cache.is_cuda):
        n, hkv, P, D = shape = v_cache.shape
        if k_cache.shape == (n, hkv, D >> 3, P, 8) and D & 7 == 0:
            return shape
    _need(k_cache, "k_cache", torch.bfloat16, 5)
    _need(v_cache, "v_cache", torch.bfloat16, 4)
    n, hkv, P, D = v_cache.shape
    if k_cache.shape != (n, hkv, D // 8, P, 8) or D % 8:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} and v_cache {tuple(v_cache.shape)} must be "
                         "[pages, kv_heads, head_dim / 8, page_size, 8] and "
                         "[pages, kv_heads, page_size, head_dim]")
    return n, hkv, P, D


def _token_rows(t, name, heads=None, dim=None):
    """The pitch of bf16 rows [tokens, heads, head_dim] whose heads are dense (a slice of a
    projection's output is fine)."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is torch.bfloat16 and t.dim() == 3):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
        if not _on_gpu(t):
            raise RuntimeError(f"{name} must be a GPU tensor (palettize_hip has no CPU path)")
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be {torch.bfloat16}, got {t.dtype}")
        if t.dim() != 3:
            raise ValueError(f"{name} must be 3-D, got shape {tuple(t.shape)}")
    T, H, D = t.shape
    if (heads is not None and H != heads) or (dim is not None and D != dim):
        raise ValueError(f"{name} {tuple(t.shape)} does not match {heads or H} heads of {dim or D}")
    st, sh, sd = t.stride()
    if (sd != 1 and D > 1) or (sh != D and H > 1):
        raise ValueError(f"the heads of {name} must be dense")
    return st if T > 1 else H * D


def paged_step(lens, new_tokens, block_table, free_pages, free_count, page_size, keep=None,
               rows=None, rows_each=0, lens_out=None, free_count_out=None):
    """One scheduler step of a paged cache: pages handed back and taken, and where the step's
    tokens go (plz_paged_step).

    lens, new_tokens, keep (optional) int32 [B]: the tokens each request has, adds and keeps of what
    it has (None: all; 0 ends a request and frees its row). block_table int32 [B, W] and free_pages
    int32 [num_pages], the stack of the pages that nobody holds, are updated in place; free_count
    int32 [1] of them are valid. rows: the size of the token buffer (default B: one token each), in
    which the requests' tokens follow each other; with rows_each every request owns that many rows of
    it and adds at most that many tokens (rows is B rows_each: 1 for a batch whose row b is request b).
    Returns (slots [rows], positions [rows], starts [B + 1], lens [B], free_count [1]); lens_out and
    free_count_out receive the last two (lens and free_count themselves may be given). A request
    that finds no page keeps the tokens that have room, and the others get slot -1."""
    ints = (lens, new_tokens, block_table, free_pages, free_count)
    if keep is not None or lens_out is not None or free_count_out is not None:
        ints += tuple(t for t in (keep, lens_out, free_count_out) if t is not None)
    dev = _dense_int32(ints)
    B = lens.shape[0] if dev >= 0 else -1
    if not (dev >= 0 and lens.dim() == 1 and new_tokens.shape == lens.shape and block_table.dim() == 2
            and block_table.shape[0] == B and free_pages.dim() == 1 and free_count.shape == (1,)
            and (keep is None or keep.shape == lens.shape)
            and (lens_out is None or lens_out.shape == lens.shape)
            and (free_count_out is None or free_count_out.shape == (1,))):
        _need(lens, "lens", torch.int32, 1)
        B = lens.shape[0]
        _ints(new_tokens, "new_tokens", B)
        _need(block_table, "block_table", torch.int32, 2)
        if block_table.shape[0] != B:
            raise ValueError(f"block_table has {block_table.shape[0]} rows for {B} requests")
        _need(free_pages, "free_pages", torch.int32, 1)
        _ints(free_count, "free_count", 1)
        for t, nm, n in ((keep, "keep", B), (lens_out, "lens_out", B),
                         (free_count_out, "free_count_out", 1)):
            if t is not None:
                _ints(t, nm, n)
        dev = _one_device("plz_paged_step", *ints)
    rows = B * (rows_each or 1) if rows is None else int(rows)
    if rows < 0 or rows_each < 0 or (rows_each and rows != B * rows_each):
        raise ValueError(f"rows ({rows}) must be at least 0, and B rows_each with rows_each "
                         f"({rows_each})")
    # the five outputs in one allocation
    buf = lens.new_empty(2 * (rows + B + 1))
    slots, positions, starts, own_lens, own_count = buf.split_with_sizes((rows, rows, B + 1, B, 1))
    if lens_out is None:
        lens_out = own_lens
    if free_count_out is None:
        free_count_out = own_count
    at = buf.data_ptr()
    _on(dev, "plz_paged_step", lens.data_ptr(), _ptr(keep), new_tokens.data_ptr(),
        block_table.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(), at, at + 4 * rows,
        at + 8 * rows, lens_out.data_ptr(), free_count_out.data_ptr(), B, block_table.shape[1],
        free_pages.shape[0], rows, rows_each, int(page_size))
    return slots, positions, starts, lens_out, free_count_out


def paged_rope_write(q, k, v, cos, sin, positions, slots, k_cache, v_cache, q_weight=None,
                     k_weight=None, eps=1e-6):
    """q [T, H, D], k, v [T, Hkv, D] (bf16, dense heads, any row pitch that is a multiple of 8)
    through per-head RMSNorm (q_weight, k_weight bf16 [D], or neither) and the rotation at each
    token's position (cos, sin fp32 [max_positions, D]): returns q [T, H, D]; k and v go into
    slots [T] of the cache in place (plz_paged_rope_write). Tokens with slot -1 are stored nowhere; two
    tokens must not share a slot. There is no backward: tensors that need a gradient are refused."""
    n, hkv, P, D = _paged_caches(k_cache, v_cache)
    ldq = _token_rows(q, "q", None, D)
    T, H = q.shape[0], q.shape[1]
    ldk, ldv = _token_rows(k, "k", hkv, D), _token_rows(v, "v", hkv, D)
    normed = q_weight is not None and k_weight is not None
    if not (k.shape[0] == T and v.shape[0] == T and isinstance(cos, torch.Tensor)
            and isinstance(sin, torch.Tensor) and cos.dim() == 2 and cos.shape[1] == D
            and sin.shape == cos.shape and cos.dtype is torch.float32 and sin.dtype is torch.float32
            and cos.is_cuda and sin.is_cuda and cos.is_contiguous() and sin.is_contiguous()
            and _dense_int32((positions, slots)) >= 0 and positions.shape == (T,) == slots.shape
            and (normed or (q_weight is None and k_weight is None))):
        if k.shape[0] != T or v.shape[0] != T:
            raise ValueError("q / k / v have different numbers of tokens")
        for t, nm in ((cos, "cos"), (sin, "sin")):
            _need(t, nm, torch.float32, 2)
        if cos.shape != sin.shape or cos.shape[1] != D:
            raise ValueError(f"cos and sin must be [positions, {D}]")
        _ints(positions, "positions", T)
        _ints(slots, "slots", T)
        if (q_weight is None) != (k_weight is None):
            raise ValueError("q_weight and k_weight must be given together")
    dev = q.get_device()
    if normed:
        if not (isinstance(q_weight, torch.Tensor) and isinstance(k_weight, torch.Tensor)
                and q_weight.dtype is _BF16 and k_weight.dtype is _BF16
                and q_weight.shape == (D,) == k_weight.shape
                and q_weight.is_contiguous() and k_weight.is_contiguous()
                and q_weight.get_device() == dev == k_weight.get_device()):
            _norm_weight(q_weight, D)
            _norm_weight(k_weight, D)
            _one_device("plz_paged_rope_write", q, q_weight, k_weight)
    if not (k.get_device() == dev == v.get_device() and cos.get_device() == dev == sin.get_device()
            and positions.get_device() == dev == slots.get_device()
            and k_cache.get_device() == dev == v_cache.get_device()):
        _one_device("plz_paged_rope_write", q, k, v, cos, sin, positions, slots, k_cache, v_cache)
    _no_backward("plz_paged_rope_write", q, k, v, q_weight, k_weight, cos, sin, k_cache, v_cache)
    out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((T, H, D))
    _on(dev, "plz_paged_rope_write", q.data_ptr(), k.data_ptr(), v.data_ptr(), ldq, ldk, ldv,
        _ptr(q_weight), _ptr(k_weight), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(),
        slots.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), T, H, hkv, D,
        cos.shape[0], n, P, float(eps))
    return out


@functools.lru_cache(maxsize=256)
def _paged_attn_workspace(*sizes):
    return query("plz_paged_attn_workspace", *sizes)


def paged_attn(q, k_cache, v_cache, block_table, lens, scale=None):
    """Attention of one new token a request over its cached tokens: q [B, H, D] (bf16, dense heads),
    block_table int32 [B, W], lens int32 [B] (the new token's own included) -> (o [B, H, D] bf16,
    lse [B, H] fp32) (plz_paged_attn). Requests without tokens give 0 and -inf. There is no backward:
    tensors that need a gradient are refused."""
    n, hkv, P, D = _paged_caches(k_cache, v_cache)
    ldq = _token_rows(q, "q", None, D)
    B, H = q.shape[0], q.shape[1]
    if not (_dense_int32((block_table, lens)) >= 0 and block_table.dim() == 2
            and block_table.shape[0] == B and lens.shape == (B,)):
        _need(block_table, "block_table", torch.int32, 2)
        if block_table.shape[0] != B:
            raise ValueError(f"block_table has {block_table.shape[0]} rows for {B} requests")
        _ints(lens, "lens", B)
    scale = D ** -0.5 if scale is None else float(scale)
    dev = q.get_device()
    if not (k_cache.get_device() == dev == v_cache.get_device()
            and block_table.get_device() == dev == lens.get_device()):
        _one_device("plz_paged_attn", q, k_cache, v_cache, block_table, lens)
    _no_backward("plz_paged_attn", q, k_cache, v_cache)
    o = torch.empty_like(q) if q.is_contiguous() else q.new_empty((B, H, D))
    lse = q.new_empty((B, H), dtype=torch.float32)
    W = block_table.shape[1]
    nbytes = _paged_attn_workspace(B, W, P, H, hkv, D)
    ws = lens.new_empty((nbytes + 3) // 4) if nbytes else None
    _on(dev, "plz_paged_attn", q.data_ptr(), ldq, k_cache.data_ptr(), v_cache.data_ptr(),
        block_table.data_ptr(), lens.data_ptr(), o.data_ptr(), lse.data_ptr(), _ptr(ws), nbytes, B,
        W, H, hkv, D, n, P, scale)
    return o, lse
