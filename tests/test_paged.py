"""CPU checks of the paged-cache operators: refusals of the C entry points and of their wrappers (no
call reaches a GPU), and the references that the GPU tests use against each other."""
import importlib.util
import os
import random
import subprocess

import pytest
import torch

import paged_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FAKE = 4096  # an aligned address that is never read: a check fails first


@pytest.fixture(scope="module")
def lib():
    from palettize_hip import _lib
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return _lib.lib()


def _step_args(**kw):
    a = dict(lens=FAKE, keep=FAKE, new=FAKE, table=FAKE, free=FAKE, count=FAKE, slots=FAKE, pos=FAKE,
             starts=FAKE, lens_out=2 * FAKE, count_out=FAKE, batch=4, width=8, pages=32, rows=4, each=0,
             page=16, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("kw,word", [
    (dict(page=8), b"power of two"), (dict(page=48), b"power of two"), (dict(page=2048), b"power"),
    (dict(batch=-1), b"negative"), (dict(rows=-1), b"negative"), (dict(width=-1), b"negative"),
    (dict(pages=-1), b"negative"), (dict(rows=(1 << 30) + 1), b"2^30"),
    (dict(batch=1 << 20, width=1 << 11), b"2^30"), (dict(width=1 << 28), b"2^30"),
    (dict(pages=1 << 27), b"2^30"), (dict(lens=None), b"null"), (dict(new=None), b"null"),
    (dict(table=None), b"null"), (dict(free=None), b"null"), (dict(count=None), b"null"),
    (dict(slots=None), b"null"), (dict(pos=None), b"null"), (dict(starts=None), b"null"),
    (dict(lens_out=None), b"null"), (dict(count_out=None), b"null"), (dict(each=2), b"rows_each"),
    (dict(each=-1), b"rows_each"), (dict(each=1, rows=3), b"rows_each"),
    (dict(new=FAKE + 64, lens_out=FAKE + 64, keep=None), b"new_tokens or keep"),
    (dict(lens_out=FAKE), b"new_tokens or keep")])
def test_step_refusals(lib, kw, word):
    assert lib.plz_paged_step(*_step_args(**kw)) == 1
    assert word in lib.plz_last_error()


def _write_args(**kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, ldq=1024, ldk=256, ldv=256, qw=FAKE, kw=FAKE, cos=FAKE, sin=FAKE,
             pos=FAKE, slots=FAKE, out=FAKE, kc=FAKE, vc=FAKE, tokens=3, heads=8, kv=2, dim=128,
             max_pos=64, pages=4, page=16, eps=1e-6, stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("kw,code,word", [
    (dict(dim=96), 3, b"head_dim"), (dict(tokens=-1), 1, b"tokens"), (dict(heads=0), 1, b"heads"),
    (dict(kv=0), 1, b"heads"), (dict(max_pos=0), 1, b"positions"), (dict(pages=0), 1, b"pages"),
    (dict(page=24), 1, b"power of two"), (dict(tokens=1 << 31), 1, b"2^30"),
    (dict(pages=1 << 28), 1, b"2^30"), (dict(heads=20000), 1, b"16384"),
    (dict(ldq=1016), 1, b"pitch"), (dict(ldk=264 - 4), 1, b"pitch"), (dict(ldv=0), 1, b"pitch"),
    (dict(qw=None), 1, b"together"), (dict(kw=None), 1, b"together"), (dict(q=None), 1, b"null"),
    (dict(pos=None), 1, b"null"), (dict(slots=None), 1, b"null"), (dict(vc=None), 1, b"null"),
    (dict(k=FAKE + 8), 1, b"aligned"), (dict(kc=FAKE + 2), 1, b"aligned"),
    (dict(cos=FAKE + 4), 1, b"aligned"),
    (dict(tokens=1 << 30, heads=16384, ldq=1 << 21), 1, b"too many"),
    (dict(tokens=1 << 28, heads=1, kv=1), 1, b"too many")])
def test_write_refusals(lib, kw, code, word):
    if word == b"together":
        word = b"go together"
    assert lib.plz_paged_rope_write(*_write_args(**kw)) == code
    assert word in lib.plz_last_error()


def _attn_args(lib, **kw):
    a = dict(q=FAKE, ldq=1024, kc=FAKE, vc=FAKE, table=FAKE, lens=FAKE, o=FAKE, lse=FAKE, ws=FAKE,
             nws=1 << 40, batch=3, width=40, heads=8, kv=2, dim=128, pages=16, page=16, scale=0.1,
             stream=None)
    assert set(kw) <= set(a)
    return list({**a, **kw}.values())


@pytest.mark.parametrize("kw,code,word", [
    (dict(dim=80), 3, b"head_dim"), (dict(batch=-1), 1, b"batch"), (dict(width=-1), 1, b"width"),
    (dict(heads=0), 1, b"heads"), (dict(kv=0), 1, b"heads"), (dict(heads=9), 1, b"multiple"),
    (dict(pages=0), 1, b"pages"), (dict(page=17), 1, b"power of two"), (dict(page=8), 1, b"power"),
    (dict(batch=65537), 1, b"65536"), (dict(width=1 << 27), 1, b"2^30"),
    (dict(pages=1 << 27), 1, b"2^30"), (dict(batch=1 << 16, width=1 << 16), 1, b"2^35"),
    (dict(scale=0.0), 1, b"scale"),
    (dict(scale=float("nan")), 1, b"scale"), (dict(ldq=1000), 1, b"pitch"),
    (dict(ldq=1028), 1, b"pitch"), (dict(q=None), 1, b"null"), (dict(lens=None), 1, b"null"),
    (dict(table=None), 1, b"null"), (dict(o=None), 1, b"null"), (dict(lse=None), 1, b"null"),
    (dict(q=FAKE + 8), 1, b"aligned"), (dict(vc=FAKE + 8), 1, b"aligned"),
    (dict(o=FAKE + 2), 1, b"aligned")])
def test_attn_refusals(lib, kw, code, word):
    assert lib.plz_paged_attn(*_attn_args(lib, **kw)) == code
    assert word in lib.plz_last_error()


def test_empty_calls_need_no_pointers(lib):
    null = dict.fromkeys(("q", "k", "v", "qw", "kw", "cos", "sin", "pos", "slots", "out", "kc", "vc"))
    assert lib.plz_paged_rope_write(*_write_args(tokens=0, **null)) == 0
    null = dict.fromkeys(("q", "kc", "vc", "table", "lens", "o", "lse", "ws"))
    assert lib.plz_paged_attn(*_attn_args(lib, batch=0, nws=0, **null)) == 0


# ---- the wrappers (every check that needs no GPU) ------------------------------------------------
def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


@pytest.fixture()
def ops(monkeypatch):
    """ops with its device check answering yes, so that CPU tensors reach the checks behind it, and no
    call let through."""
    from palettize_hip import ops as o

    def stop(*args):
        raise AssertionError("a refused call went through")

    monkeypatch.setattr(o, "_on_gpu", lambda t: True)
    monkeypatch.setattr(o, "_on", stop)
    return o


def test_wrappers_refuse_cpu_tensors():
    from palettize_hip import ops as o
    with pytest.raises(RuntimeError, match="GPU tensor"):
        o.paged_step(_i32(2), _i32(2), _i32(2, 4), _i32(8), _i32(1), 16)
    kc, vc = o.paged_cache(4, 16, 2, 64, "cpu")
    with pytest.raises(RuntimeError, match="GPU tensor"):
        o.paged_attn(_bf(2, 4, 64), kc, vc, _i32(2, 2), _i32(2))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        o.paged_rope_write(_bf(2, 4, 64), _bf(2, 2, 64), _bf(2, 2, 64), torch.zeros(8, 64),
                           torch.zeros(8, 64), _i32(2), _i32(2), kc, vc)


def test_step_wrapper_refusals(ops):
    ok = dict(lens=_i32(2), new_tokens=_i32(2), block_table=_i32(2, 4), free_pages=_i32(8),
              free_count=_i32(1), page_size=16)
    for bad, err in ((dict(lens=_i32(2).long()), TypeError), (dict(new_tokens=_i32(3)), ValueError),
                     (dict(block_table=_i32(3, 4)), ValueError),
                     (dict(block_table=_i32(4, 2).t()), ValueError),
                     (dict(free_pages=_i32(2, 4)), ValueError), (dict(free_count=_i32(2)), ValueError),
                     (dict(keep=_i32(3)), ValueError), (dict(rows=-1), ValueError),
                     (dict(rows_each=-1), ValueError), (dict(rows_each=2, rows=3), ValueError),
                     (dict(lens_out=_i32(3)), ValueError), (dict(free_count_out=_i32(2)), ValueError),
                     (dict(lens=[1, 2]), TypeError)):
        with pytest.raises(err):
            ops.paged_step(**{**ok, **bad})


def test_write_wrapper_refusals(ops):
    kc, vc = ops.paged_cache(4, 16, 2, 64, "cpu")
    ok = dict(q=_bf(3, 4, 64), k=_bf(3, 2, 64), v=_bf(3, 2, 64), cos=torch.zeros(8, 64),
              sin=torch.zeros(8, 64), positions=_i32(3), slots=_i32(3), k_cache=kc, v_cache=vc)
    for bad, err in ((dict(q=_bf(3, 4, 64).float()), TypeError), (dict(q=_bf(3, 256)), ValueError),
                     (dict(q=_bf(4, 4, 64)), ValueError), (dict(k=_bf(3, 3, 64)), ValueError),
                     (dict(v=_bf(2, 2, 64)), ValueError), (dict(q=_bf(3, 4, 128)), ValueError),
                     (dict(q=_bf(4, 3, 64).transpose(0, 1)), ValueError),
                     (dict(k=_bf(3, 2, 128)[..., ::2]), ValueError),
                     (dict(cos=torch.zeros(8, 32)), ValueError),
                     (dict(sin=torch.zeros(9, 64)), ValueError),
                     (dict(cos=torch.zeros(8, 64).double()), TypeError),
                     (dict(positions=_i32(4)), ValueError), (dict(slots=_i32(3).long()), TypeError),
                     (dict(q_weight=_bf(64)), ValueError),
                     (dict(q_weight=_bf(32), k_weight=_bf(64)), ValueError),
                     (dict(q_weight=torch.zeros(64), k_weight=torch.zeros(64)), TypeError),
                     (dict(k_cache=_bf(4, 2, 8, 32, 8)), ValueError),
                     (dict(v_cache=_bf(4, 2, 16, 60)), ValueError),
                     (dict(v_cache=vc.transpose(0, 1)), ValueError), (dict(q=None), TypeError)):
        with pytest.raises(err):
            ops.paged_rope_write(**{**ok, **bad})


def test_attn_wrapper_refusals(ops):
    kc, vc = ops.paged_cache(4, 16, 2, 64, "cpu")
    ok = dict(q=_bf(3, 4, 64), k_cache=kc, v_cache=vc, block_table=_i32(3, 2), lens=_i32(3))
    for bad, err in ((dict(q=_bf(3, 4, 128)), ValueError), (dict(q=_bf(4, 3, 64).transpose(0, 1)),
                                                            ValueError),
                     (dict(block_table=_i32(2, 2)), ValueError), (dict(lens=_i32(2)), ValueError),
                     (dict(lens=_i32(3).long()), TypeError), (dict(lens=_i32(3, 1)), ValueError),
                     (dict(block_table=_i32(3, 4)[:, ::2]), ValueError),
                     (dict(k_cache=kc.float()), TypeError), (dict(v_cache=_bf(4, 2, 32, 64)), ValueError)):
        with pytest.raises(err):
            ops.paged_attn(**{**ok, **bad})


def test_cache_refusals(ops):
    for page, dim in ((8, 64), (24, 64), (2048, 64), (16, 96)):
        with pytest.raises(ValueError):
            ops.paged_cache(4, page, 2, dim, "cpu")


def test_tensors_of_two_devices_are_refused():
    from types import SimpleNamespace
    from palettize_hip import ops as o
    a, b = SimpleNamespace(get_device=lambda: 0), SimpleNamespace(get_device=lambda: 1)
    with pytest.raises(ValueError, match="different devices"):
        o._one_device("plz_paged_step", a, None, b)
    assert o._one_device("plz_paged_step", b, None, b) == 1


def test_calls_run_on_their_tensors_device(monkeypatch):
    """The device of the tensors is current during the call, whatever was before, and so is its
    stream."""
    from palettize_hip import ops as o
    log, current = [], [0]

    class Guard:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.before, current[0] = current[0], self.dev

        def __exit__(self, *exc):
            current[0] = self.before

    monkeypatch.setattr(o, "call", lambda *a: log.append((a, current[0])))
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 100 + d, raising=False)
    for dev in (0, 1):
        o._on(dev, "plz_paged_attn", 7)
    assert log == [(("plz_paged_attn", 7, 100), 0), (("plz_paged_attn", 7, 101), 1)]
    assert current == [0]


def test_attn_needs_its_workspace(lib):
    need = lib.plz_paged_attn_workspace(3, 40, 16, 8, 2, 128)
    assert need > 0
    for kw in (dict(ws=None), dict(nws=need - 1), dict(ws=FAKE + 8)):
        assert lib.plz_paged_attn(*_attn_args(lib, **kw)) == 4
        assert b"workspace" in lib.plz_last_error()
    for args in ((0, 40, 16, 8, 2, 128), (3, 0, 16, 8, 2, 128), (3, 40, 0, 8, 2, 128),
                 (3, 40, 16, 0, 2, 128), (3, 40, 16, 8, 0, 128), (3, 40, 16, 9, 2, 128),
                 (3, 40, 16, 8, 2, 0), (-1, 40, 16, 8, 2, 128), (3, -40, 16, 8, 2, 128)):
        assert lib.plz_paged_attn_workspace(*args) == 0
    # tables of up to 512 tokens whose requests have waves of their own share nothing: up to 1024 of them
    # (batch x kv heads x tiles of 16 heads; 1536 and 512 for heads of 64 and 256), any number up to 320
    # tokens, and 2^22 at most
    assert lib.plz_paged_attn_workspace(1, 8, 64, 8, 2, 128) == 0
    for batch, heads, hkv, dim in ((512, 8, 2, 128), (256, 40, 2, 128), (64, 16, 16, 128),
                                   (768, 8, 2, 64), (256, 8, 2, 256)):
        for width in (21, 32):
            assert lib.plz_paged_attn_workspace(batch, width, 16, heads, hkv, dim) == 0
            assert lib.plz_paged_attn_workspace(batch + 1, width, 16, heads, hkv, dim) > 0
        assert lib.plz_paged_attn_workspace(batch + 1, 20, 16, heads, hkv, dim) == 0
    for width in (0, 20):
        assert lib.plz_paged_attn_workspace(65536, width, 16, 128, 64, 128) == 0
        assert lib.plz_paged_attn_workspace(65536, width, 16, 130, 65, 128) > 0
        assert lib.plz_paged_attn_workspace(1 << 40, width, 16, 1 << 30, 1 << 30, 128) > 0
    assert lib.plz_paged_attn_workspace(1, 9, 64, 8, 2, 128) > 0
    assert lib.plz_paged_attn_workspace(5, 33, 16, 8, 2, 128) > 0
    assert lib.plz_paged_attn_workspace(1 << 40, 1 << 20, 1024, 8, 2, 128) > 0


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
def test_tokens_are_dealt_once(tmp_path):
    exe = tmp_path / "paged_check"
    cmd = [HIPCC, "--offload-arch=gfx950", "-O1", "-g", "-std=c++17",
           "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "qwen-palettize_amd", "csrc"),
           os.path.join(ROOT, "tests", "native", "paged_check.hip"), "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
    assert "checks passed" in r.stdout


# ---- the references against each other -------------------------------------------------------------
def random_step(rng, short=False):
    """Lists of a random step: rows that keep all, some or nothing, odd lengths, and pools that run out
    where `short`."""
    B, W, P = rng.choice((1, 2, 7, 33)), rng.choice((1, 3, 16)), rng.choice((16, 32, 128))
    lens = [rng.choice((0, 1, P - 1, P, P + 1, W * P, rng.randint(0, W * P))) for _ in range(B)]
    lens = [min(n, W * P) for n in lens]
    keep = [rng.choice((n, n, 0, rng.randint(0, n), max(0, n - 2))) for n in lens]
    new = [rng.choice((0, 1, 1, 5, rng.randint(0, 3 * P))) for _ in range(B)]
    held = sum(paged_ref.pages(n, P) for n in lens)
    extra = sum(paged_ref.pages(k + n, P) for k, n in zip(keep, new))
    F = held + (rng.randint(0, max(1, extra // 2)) if short else extra + rng.randint(0, 3))
    ids = list(range(F))
    rng.shuffle(ids)
    table = [[-7] * W for _ in range(B)]
    for b, n in enumerate(lens):
        for w in range(paged_ref.pages(n, P)):
            table[b][w] = ids.pop()
    count = len(ids)
    free = ids + [-9] * (F - count)
    total = sum(new)
    rows = total + rng.choice((0, 0, 1, 70)) if rng.random() < 0.9 else rng.randint(0, total + 1)
    return dict(lens=lens, keep=keep, new=new, table=table, free=free, count=count, P=P, rows=rows)


@pytest.fixture(scope="module")
def plain_step():
    spec = importlib.util.spec_from_file_location("paged_operators",
                                                  os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m._step


@pytest.mark.parametrize("short", [False, True])
def test_step_references_agree(plain_step, short):
    rng = random.Random(5 + short)
    for _ in range(60):
        c = random_step(rng, short)
        t = {k: torch.tensor(v, dtype=torch.int32) for k, v in c.items() if k not in ("P", "rows")}
        got = plain_step(dict(lens=t["lens"], keep=t["keep"], new=t["new"], table=t["table"],
                              free=t["free"], count=t["count"].reshape(1), page=c["P"],
                              rows=c["rows"]))
        want = paged_ref.step(**c)
        for g, w, nm in zip(got, want, ("slots", "positions", "starts", "lens", "count", "table",
                                        "free")):
            assert g.flatten().tolist() == torch.tensor(w).flatten().tolist(), (nm, c)


def test_step_reference_conserves_pages():
    """Every page is held by one row or free, before and after."""
    rng = random.Random(9)
    for _ in range(60):
        c = random_step(rng, short=rng.random() < 0.5)
        F = len(c["free"])
        _, _, _, lens, count, table, free = paged_ref.step(**c)
        held = [p for b, n in enumerate(lens) for p in table[b][:paged_ref.pages(n, c["P"])]]
        assert sorted(held + free[:count]) == list(range(F))


def test_cache_and_layer_refusals():
    from palettize_hip import decode
    for kw in (dict(batch=0), dict(layers=0), dict(max_tokens=0), dict(num_pages=0), dict(page_size=24),
               dict(head_dim=100)):
        with pytest.raises(ValueError):
            decode.PagedKVCache(**{**dict(layers=1, batch=2, max_tokens=64, kv_heads=2, head_dim=64,
                                          device="cpu"), **kw})
    c = decode.PagedKVCache(2, 3, 100, 2, 64, page_size=16, device="cpu")
    assert c.num_pages == 3 * 7 and c.block_table.shape == (3, 7) and len(c.k) == len(c.v) == 2
    with pytest.raises(RuntimeError, match="GPU tensor"):
        c.step([1, 1, 1])
    for request, n in ((3, 1), (-1, 1), (0, 113), (0, -1)):
        with pytest.raises(ValueError, match="tokens of request"):
            c.tokens(0, request, n)
    assert c.tokens(1, 2, 112)[0].shape == (112, 2, 64) == c.tokens(1, 2, 112)[1].shape
    q = _bf(3, 4, 64).requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        c.attend(0, q)
    with pytest.raises(RuntimeError, match="no backward"):
        c.write(0, q, _bf(3, 2, 64), _bf(3, 2, 64), None, None, None)
    with pytest.raises(ValueError, match="rows"):
        decode.HardDecoderLayer.prefill.__wrapped__(
            type("L", (), {"cfg": None})(), torch.zeros(5, 8), c, 0, None, [2, 2], None, None)


def test_cache_tokens_that_a_request_does_not_have():
    """tokens() reads a request's own pages only: rows past its length are zeros, whatever its table's
    unused entries name."""
    from palettize_hip import decode
    c = decode.PagedKVCache(1, 3, 64, 2, 64, page_size=16, num_pages=4, device="cpu")
    for t in (c.k[0], c.v[0]):
        t.copy_(torch.arange(1, 5).view(4, 1, 1, 1, *[1] * (t.dim() - 4)))  # a page's number + 1
    c.v[0][0, :, 5:] = float("nan")
    c.lens.copy_(torch.tensor([5, 16, 0]))
    c.block_table[1, 0], c.block_table[1, 1], c.block_table[2, 0] = 3, 2 ** 31 - 1, -1
    for request, has, page in ((0, 5, 1), (1, 16, 4), (2, 0, None)):
        for x in c.tokens(0, request, 20):
            assert x.shape == (20, 2, 64)
            assert bool((x[has:] == 0).all())
            assert page is None or bool((x[:has] == page).all())


def test_operators_refuse_gradients(ops):
    """The operators have no backward: each tensor of values that needs a gradient is refused where
    gradients are on, and taken under no_grad (here: up to the call itself)."""
    kc, vc = ops.paged_cache(4, 16, 2, 64, "cpu")
    write = dict(q=_bf(3, 4, 64), k=_bf(3, 2, 64), v=_bf(3, 2, 64), cos=torch.zeros(8, 64),
                 sin=torch.zeros(8, 64), positions=_i32(3), slots=_i32(3), k_cache=kc, v_cache=vc,
                 q_weight=_bf(64), k_weight=_bf(64))
    attn = dict(q=_bf(3, 4, 64), k_cache=kc, v_cache=vc, block_table=_i32(3, 2), lens=_i32(3))
    for fn, ok in ((ops.paged_rope_write, write), (ops.paged_attn, attn)):
        for name, t in ok.items():
            if t.is_floating_point():
                needs = {**ok, name: t.clone().requires_grad_()}
                with pytest.raises(RuntimeError, match="no backward"):
                    fn(**needs)
                with torch.no_grad(), pytest.raises(Exception) as e:
                    fn(**needs)
                assert "no backward" not in str(e.value)
