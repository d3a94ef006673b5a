"""CPU checks of the losses over a vocabulary: what the C entry points refuse, and their workspaces."""
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


A = C.c_void_p(4096)  # an address on 16 bytes that no refused call reads


def ce_fwd(lib, x=A, w=A, labels=A, size=8, loss=A, lse=A, ws=A, ws_bytes=1 << 40, N=4, V=100, H=64):
    return lib.plz_linear_ce_fwd(x, w, labels, size, -100, loss, lse, None, ws, ws_bytes, N, V, H, None)


def kl_fwd(lib, tx=A, tw=A, inv=1.0, N=4, V=100, H=64, Ht=64, ws=A, ws_bytes=1 << 40):
    return lib.plz_linear_kl_fwd(A, A, tx, tw, None, inv, A, A, None, ws, ws_bytes, N, V, H, Ht, None)


@pytest.mark.parametrize("kw,status,word", [
    (dict(size=2), 1, b"bytes"), (dict(x=None), 1, b"null"), (dict(w=None), 1, b"null"),
    (dict(labels=None), 1, b"null"), (dict(loss=None), 1, b"null"), (dict(lse=None), 1, b"null"),
    (dict(H=60), 1, b"multiples of 8"), (dict(H=0), 1, b"shape"), (dict(V=0), 1, b"shape"),
    (dict(N=-1), 1, b"shape"), (dict(x=C.c_void_p(4098)), 1, b"aligned"),
    (dict(ws=None), 4, b"workspace"), (dict(ws_bytes=1000), 4, b"workspace"),
    (dict(ws=C.c_void_p(4098)), 1, b"aligned"),
    (dict(N=1 << 22), 3, b"2^22"), (dict(N=1 << 20, H=4096), 3, b"2^31"),
    (dict(V=(1 << 31) - 1), 3, b"2^31")])
def test_ce_forward_refuses(lib, kw, status, word):
    assert ce_fwd(lib, **kw) == status and word in lib.plz_last_error()


@pytest.mark.parametrize("kw,status,word", [
    (dict(tx=None), 1, b"null"), (dict(tw=None), 1, b"null"), (dict(inv=0.0), 1, b"temperature"),
    (dict(inv=-1.0), 1, b"temperature"), (dict(inv=float("nan")), 1, b"temperature"),
    (dict(inv=float("inf")), 1, b"temperature"), (dict(Ht=0), 1, b"shape"), (dict(Ht=12), 1, b"multiples"),
    (dict(tw=C.c_void_p(4104)), 1, b"aligned"), (dict(ws_bytes=64), 4, b"workspace")])
def test_kl_forward_refuses(lib, kw, status, word):
    assert kl_fwd(lib, **kw) == status and word in lib.plz_last_error()


def test_backward_refuses(lib):
    def bwd(lse=A, grad=A, mode=2, gx=A, gw=A, ws=A, ws_bytes=1 << 40, size=8):
        return lib.plz_linear_ce_bwd(A, A, A, size, -100, lse, grad, mode, gx, gw, ws, ws_bytes, 4, 100, 64,
                                     None)
    for kw, status, word in ((dict(lse=None), 1, b"null"), (dict(grad=None), 1, b"null"),
                             (dict(mode=3), 1, b"reduction"), (dict(gx=C.c_void_p(8)), 1, b"aligned"),
                             (dict(gw=C.c_void_p(8)), 1, b"aligned"), (dict(ws=None), 4, b"workspace"),
                             (dict(ws_bytes=10), 4, b"workspace"), (dict(size=1), 1, b"bytes")):
        assert bwd(**kw) == status and word in lib.plz_last_error(), kw
    assert bwd(gx=None, gw=None) == 0  # nothing wanted, nothing done


def test_workspaces(lib):
    fwd, bwd = lib.plz_vocab_loss_workspace, lib.plz_vocab_loss_bwd_workspace
    N, V, H = 4096, 151936, 2560
    # the packed rows and the tiles' statistics: far less than the logits (2.5 GB)
    assert N * H * 2 < fwd(N, V, H, 0) < 64 << 20
    # at most a piece of bf16 gradients of logits (1 GiB), the packed rows and dx in fp32 parts
    assert bwd(N, V, H, 0, 1) < (1 << 30) + (1 << 29)
    assert bwd(N, V, H, 0, 0) < bwd(N, V, H, 0, 1) < bwd(N, V, H, 2560, 1)
    assert bwd(1 << 17, V, 2560, 0, 0) < (1 << 30) + (1 << 30)
    assert fwd(0, 1, 8, 0) > 0 and fwd(0, 1, 8, 8) > 0
    assert fwd(-1, 100, 64, 0) == 0 and bwd(0, 100, 64, 0, 1) == 0


def test_steps_that_fit(lib):
    step = lib.plz_vocab_loss_step_workspace
    # 2 bytes a logit of whole tiles, under 4 GiB; 10 of a distillation, under 8 GiB
    assert (1 << 30) < step(4096, 151936, 2560, 0, 1) < (2 << 30)
    assert step(14080, 151936, 2560, 0, 1) > 0 and step(14337, 151936, 2560, 0, 1) == 0
    assert step(5632, 151936, 2560, 2560, 1) > 0 and step(5889, 151936, 2560, 2560, 1) == 0
    assert step(0, 1000, 64, 0, 1) == 0 and step(16, 1 << 20, 2048, 0, 1) == 0

    def call(N, mode=2, gx=A, gw=A):
        return lib.plz_linear_ce_step(A, A, A, 8, -100, mode, A, A, None, gx, gw, A, 1 << 44, N, 151936,
                                      2560, None)
    assert call(14337) == 3 and b"logits" in lib.plz_last_error()
    assert call(0) == 3
    for kw, word in ((dict(mode=0), b"reduction"), (dict(mode=7), b"reduction"),
                     (dict(gx=C.c_void_p(8)), b"aligned"), (dict(gw=C.c_void_p(2)), b"aligned")):
        assert call(64, **kw) == 1 and word in lib.plz_last_error()


def test_a_workspace_is_sized_on_the_device_of_its_call(monkeypatch):
    """Devices of other CU counts need other workspaces for the same sizes; whether a step fits does not go
    by the device, and is not asked of one."""
    import functools

    import torch
    from palettize_hip import ops
    now = [0]
    # a cache of its own: what is looked up here is not the library's
    monkeypatch.setattr(ops, "_vocab_workspace", functools.lru_cache(ops._vocab_workspace.__wrapped__))

    class On:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.before, now[0] = now[0], self.dev

        def __exit__(self, *_):
            now[0] = self.before

    class Sized(Exception):
        pass

    def workspace(nbytes, device):
        raise Sized(nbytes)

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(ops, "query", lambda which, *sizes: 1000 * (now[0] + 1))
    monkeypatch.setattr(ops, "_need", lambda t, *_: t)
    monkeypatch.setattr(ops, "_workspace", workspace)
    x, w, labels = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    lse = torch.zeros(2, 3)
    calls = (lambda: ops.linear_ce_fwd(x, w, labels), lambda: ops.linear_ce_step(x, w, labels),
             lambda: ops.linear_ce_bwd(x, w, labels, lse, torch.ones(1)),
             lambda: ops.linear_kl_fwd(x, w, x, w), lambda: ops.linear_kl_step(x, w, x, w),
             lambda: ops.linear_kl_bwd(x, w, x, w, torch.zeros(4, 3), torch.ones(1)))
    for current in (0, 1):
        now[0] = current
        for dev in (1, 0, 2, 1):
            monkeypatch.setattr(ops, "_one_device", lambda *_: dev)
            for call in calls:
                with pytest.raises(Sized) as got:
                    call()
                assert got.value.args == (1000 * (dev + 1),) and now[0] == current
