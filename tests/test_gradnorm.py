"""CPU checks of the gradient norm's entry points: what they refuse, and their workspace."""
import ctypes as C
import os

import pytest


@pytest.fixture(scope="module")
def lib():
    from palettize_hip import _lib
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return _lib.lib()


def arrays(ptrs, sizes, kinds):
    n = len(ptrs)
    return (C.c_void_p * n)(*ptrs), (C.c_int64 * n)(*sizes), (C.c_int32 * n)(*kinds), n


A = C.c_void_p(4096)  # an address on 16 bytes that no refused call reads


@pytest.mark.parametrize("ptrs,sizes,kinds,word", [
    ([None], [4], [0], b"null"), ([4096], [-1], [0], b"large"), ([4096], [1 << 40], [2], b"large"),
    ([4096], [4], [3], b"type"), ([4097], [4], [0], b"aligned"), ([4098], [4], [2], b"aligned")])
def test_refusals(lib, ptrs, sizes, kinds, word):
    p, s, k, n = arrays(ptrs, sizes, kinds)
    assert lib.plz_grad_norm(p, s, k, n, A, A, 1 << 40, None) == 1 and word in lib.plz_last_error()
    g, _, f, _ = arrays([8192], [4], [0])
    assert lib.plz_clip_grads(p, s, k, g, f, n, 1.0, A, A, 1 << 40, None) == 1
    if sizes[0] == 4:
        assert lib.plz_clip_grads(g, s, f, p, k, n, 1.0, A, A, 1 << 40, None) == 1
        assert word in lib.plz_last_error()


def test_other_refusals(lib):
    p, s, k, n = arrays([4096, 8192], [4, 4], [0, 2])
    _, _, other, _ = arrays([4096, 8192], [4, 4], [0, 0])
    assert lib.plz_grad_norm(p, s, k, n, None, A, 1 << 40, None) == 1
    assert lib.plz_grad_norm(None, s, k, n, A, A, 1 << 40, None) == 1
    assert lib.plz_grad_norm(p, s, k, -1, A, A, 1 << 40, None) == 1
    assert lib.plz_grad_norm(p, s, k, n, A, None, 0, None) == 4
    assert lib.plz_grad_norm(p, s, k, n, A, A, 300, None) == 4 and b"workspace" in lib.plz_last_error()
    assert lib.plz_grad_norm(p, s, k, n, A, C.c_void_p(4104), 1 << 40, None) == 1
    for bad in (-1.0, float("nan")):
        assert lib.plz_clip_grads(p, s, k, p, k, n, bad, A, A, 1 << 40, None) == 1
        assert b"max_norm" in lib.plz_last_error()
    assert lib.plz_clip_grads(p, s, k, p, other, n, 1.0, A, A, 1 << 40, None) == 1
    assert b"in place" in lib.plz_last_error()


def test_workspace(lib):
    _, s, _, n = arrays([None] * 3, [0, 1, 10 ** 9], [0] * 3)
    # eight bytes for every 32768 values of a tensor
    assert 8 * (10 ** 9 // 32768) < lib.plz_grad_norm_workspace(s, n) < 8 * (10 ** 9 // 32768) + 1024
    assert lib.plz_grad_norm_workspace(None, 0) >= 256
    assert lib.plz_grad_norm_workspace(None, 2) == 0


def test_a_gradient_read_beside_its_own_clipping_is_refused(monkeypatch):
    """Tensors given twice, once or both times in place: refused before anything is launched. (The table's
    addresses are of the CPU's memory, and no call gets past the checks.)"""
    import torch
    from palettize_hip import ops
    launched = []
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(ops, "_on", lambda dev, name, *args: launched.append(name))
    monkeypatch.setattr(ops, "query", lambda *args: 256)
    g, h, b, c = (torch.ones(64) for _ in range(4))
    for grads, out in (([g, g], [g, b]), ([g, g], [b, g]), ([g, h, g], [b, h, g]), ([g, h], [h, b]),
                       ([g, g, h], [c, b, g])):
        with pytest.raises(ValueError, match="another gradient"):
            ops.clip_grads(grads, 1.0, out=out)
    assert not launched
    for grads, out in (([g, g], [b, c]), ([g, h], [g, b]), ([g, h], [g, h]), ([g, h], [b, c])):
        ops.clip_grads(grads, 1.0, out=out)
    assert launched == ["plz_clip_grads"] * 4
