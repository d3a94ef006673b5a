"""GPU parity of the paged-cache operators (scheduler step, cache write, attention of one token)
against tests/paged_ref.py, each by itself and as a decoding batch runs them together."""
import math
import random

import pytest
import torch

import paged_ref
from test_paged import random_step

pytestmark = pytest.mark.gpu
ops = pytest.importorskip("palettize_hip.ops")


def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# ---- scheduler step ---------------------------------------------------------------------------
def _run_step(c, dev, keep=True, **kw):
    t = {k: _ints(v, dev) for k, v in c.items() if k not in ("P", "rows", "each")}
    out = ops.paged_step(t["lens"], t["new"], t["table"].reshape(len(c["lens"]), -1), t["free"],
                         t["count"].reshape(1), c["P"], keep=t["keep"] if keep else None,
                         rows=c["rows"], rows_each=c.get("each", 0), **kw)
    return (*out, t["table"], t["free"])


def _same_step(got, want, what):
    for g, w, nm in zip(got, want, ("slots", "positions", "starts", "lens", "count", "table", "free")):
        assert g.flatten().tolist() == torch.tensor(w).flatten().tolist(), (nm, what)


@pytest.mark.parametrize("short", [False, True], ids=["pages", "pages-run-out"])
def test_step_against_lists(dev, short):
    rng = random.Random(21 + short)
    for _ in range(40):
        c = random_step(rng, short)
        _same_step(_run_step(c, dev), paged_ref.step(**c), c)


@pytest.mark.parametrize("B", [1, 1023, 1024, 1025, 2500, 9000])
def test_step_of_many_requests(dev, B):
    """Batches around and over the workgroup's chunk: sums carried from chunk to chunk, every kind of
    row among them."""
    rng = random.Random(B)
    P, W = 16, 6
    lens = [rng.randint(0, W * P) for _ in range(B)]
    keep = [rng.choice((n, n, 0, n // 2)) for n in lens]
    new = [rng.choice((0, 1, 1, 40)) for _ in range(B)]
    F = sum(paged_ref.pages(n, P) for n in lens) + 2 * B
    ids = list(range(F))
    rng.shuffle(ids)
    table = [[-1] * W for _ in range(B)]
    for b, n in enumerate(lens):
        for w in range(paged_ref.pages(n, P)):
            table[b][w] = ids.pop()
    c = dict(lens=lens, keep=keep, new=new, table=table, count=len(ids), free=ids + [0] * (F - len(ids)),
             P=P, rows=sum(new) + 5)
    _same_step(_run_step(c, dev), paged_ref.step(**c), B)


@pytest.mark.parametrize("each", [1, 4, 200])
def test_step_with_rows_of_their_own(dev, each):
    """Every request owns `each` rows, in one launch and in two: row b each is request b's first token,
    also where others have none, more than they own, or no room."""
    rng = random.Random(30 + each)
    for i in range(12):
        c = random_step(rng, short=i % 3 == 0)
        _same_step(_run_step(dict(c, rows=len(c["lens"]) * each, each=each), dev),
                   paged_ref.step(**dict(c, rows=len(c["lens"]) * each, each=each)), c)
    B, P, W = 3000, 16, 20
    new = [rng.choice((0, 0, 1, each, each + 3, -2)) for _ in range(B)]
    c = dict(lens=[rng.randint(0, 30) for _ in range(B)], keep=[0] * B, new=new,
             table=[[7] * W for _ in range(B)], free=list(range(4000)) + [0] * 6000, count=4000, P=P,
             rows=B * each, each=each)
    _same_step(_run_step(c, dev), paged_ref.step(**c), each)


@pytest.mark.parametrize("rows_more", [0, 3])
def test_step_of_long_prompts(dev, rows_more):
    """Hundreds of thousands of token rows, thousands of pages a row."""
    P, W, B = 16, 6000, 5
    new = [96000, 1, 0, 70001, 33]
    F = sum(paged_ref.pages(n, P) for n in new) + 2
    c = dict(lens=[0] * B, keep=[0] * B, new=new, table=[[0] * W for _ in range(B)], count=F,
             free=list(range(F)), P=P, rows=sum(new) + rows_more)
    got = _run_step(c, dev)
    _same_step(got, paged_ref.step(**c), "prompts")
    # and all of it handed back
    c = dict(c, lens=got[3].tolist(), new=[0, 0, 2, 0, 0], table=got[5].tolist(), count=int(got[4]),
             free=got[6].tolist(), rows=4)
    _same_step(_run_step(c, dev), paged_ref.step(**c), "handed back")


def test_step_values_out_of_range_are_clamped(dev):
    """Lengths past the table, negative ones, kept counts past the length, counts past the pool, page
    numbers that no pool has: the result of the clamped values, nothing outside the buffers."""
    c = dict(lens=[1000, -5, 20, 7], keep=[2000, -1, -3, 90], new=[3, -2, 17, 2 ** 31 - 1],
             table=[[3, 4], [0, 0], [-8, 99], [5, 6]], free=[0, 1, 2, 9, 9, 9, 9], count=900, P=16,
             rows=40)
    _same_step(_run_step(c, dev), paged_ref.step(**c), "clamped")
    c = dict(c, count=-4)
    _same_step(_run_step(c, dev), paged_ref.step(**c), "negative count")


def test_step_without_keep_rows_or_requests(dev):
    c = dict(lens=[3, 0, 31], keep=[3, 0, 31], new=[1, 1, 1], table=[[0, 0], [0, 0], [2, 3]],
             free=[1, 4, 5, 0, 0, 0], count=3, P=16, rows=3)
    _same_step(_run_step(c, dev, keep=False), paged_ref.step(**c), "all kept")
    t = {k: _ints(c[k], dev) for k in ("lens", "new", "table", "free")}
    slots, pos, starts, lens, count = ops.paged_step(t["lens"], t["new"], t["table"], t["free"],
                                                     _ints([3], dev), 16)
    assert slots.tolist() == paged_ref.step(**c)[0]  # a row for each request by default
    c = dict(c, rows=0)
    _same_step(_run_step(c, dev), paged_ref.step(**c), "no rows")
    out = ops.paged_step(_ints([], dev), _ints([], dev), _ints([], dev).reshape(0, 4),
                         _ints([1, 2], dev), _ints([2], dev), 16, rows=3)
    assert [x.tolist() for x in out] == [[-1] * 3, [0] * 3, [0], [], [2]]
    no_width = dict(lens=[4, 0], keep=[4, 0], new=[1, 2], table=[[], []], free=[0], count=1, P=16, rows=3)
    _same_step(_run_step(no_width, dev), paged_ref.step(**no_width), "no width")


def test_step_in_place_many_times(dev):
    """lens and free_count updated in place over a hundred steps, as a decoding loop keeps them, with
    rows that end, roll back and start; no page is lost or held twice."""
    rng = random.Random(3)
    B, W, P, F = 6, 8, 16, 30
    lens, count = _ints([0] * B, dev), _ints([F], dev)
    table, free = torch.full((B, W), -1, dtype=torch.int32, device=dev), _ints(list(range(F)), dev)
    state = dict(lens=[0] * B, table=table.tolist(), free=list(range(F)), count=F)
    for _ in range(100):
        keep = [rng.choice((n, n, n, max(0, n - 3), 0)) for n in state["lens"]]
        new = [rng.choice((1, 1, 4, 0, 50)) for _ in range(B)]
        rows = sum(new)
        out = ops.paged_step(lens, _ints(new, dev), table, free, count, P, keep=_ints(keep, dev),
                             rows=rows, lens_out=lens, free_count_out=count)
        assert out[3] is lens and out[4] is count
        want = paged_ref.step(state["lens"], keep, new, state["table"], state["free"], state["count"], P,
                              rows)
        _same_step((*out, table, free), want, (keep, new))
        state = dict(lens=want[3], count=want[4], table=want[5], free=want[6])
        held = [p for b, n in enumerate(state["lens"])
                for p in state["table"][b][:paged_ref.pages(n, P)]]
        assert sorted(held + state["free"][:state["count"]]) == list(range(F))


# ---- cache write --------------------------------------------------------------------------------
def _tables(n, dim, dev):
    inv = 1e4 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    a = torch.outer(torch.arange(n, dtype=torch.float64), inv)
    a = torch.cat([a, a], -1)
    return a.cos().float().to(dev), a.sin().float().to(dev)


def _write_case(T, H, Hkv, D, P, seed, dev, norm=True, fused=False, std=1.0):
    g = torch.Generator().manual_seed(seed)
    width = (H + 2 * Hkv) * D
    qkv = (torch.randn(T, width, generator=g) * std).to(torch.bfloat16).to(dev)
    parts = [x.unflatten(1, (-1, D)) for x in qkv.split([H * D, Hkv * D, Hkv * D], 1)]
    if not fused:
        parts = [x.contiguous() for x in parts]
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(torch.bfloat16).to(dev) if norm else None
              for _ in range(2))
    pages = paged_ref.pages(T, P) + 2
    slots = torch.randperm(pages * P, generator=g)[:T].to(torch.int32)
    pos = torch.randint(0, 300, (T,), generator=g).to(torch.int32)
    cos, sin = _tables(300, D, "cpu")
    sin = sin * 0.9  # tables of any values: no identity between the two is used
    cos[:, D // 2:] *= 1.1
    return (*parts, cos.to(dev), sin.to(dev), pos.to(dev), slots.to(dev), qw, kw)


def _check_write(q, k, v, cos, sin, pos, slots, qw, kw, P, eps=1e-6):
    T, H, D = q.shape
    Hkv = k.shape[1]
    pages = paged_ref.pages(T, P) + 2
    kc, vc = ops.paged_cache(pages, P, Hkv, D, q.device)
    kc.fill_(7.0), vc.fill_(-3.0)
    out = ops.paged_rope_write(q, k, v, cos, sin, pos, slots, kc, vc, qw, kw, eps)
    c, s = cos[pos.clamp(0, cos.shape[0] - 1).long()], sin[pos.clamp(0, cos.shape[0] - 1).long()]
    outside = (pos < 0) | (pos >= cos.shape[0])
    want, bound, _ = paged_ref.rope(q, qw, eps, c, s)
    assert torch.isnan(out[outside]).all()
    assert ((out.double() - want).abs() <= bound)[~outside].all()
    want, bound, _ = paged_ref.rope(k, kw, eps, c, s)
    live = (slots >= 0) & (slots < pages * P) & ~outside
    page, at = slots[live].long() // P, slots[live].long() % P
    got = kc[page, :, :, at].reshape(-1, Hkv, D)
    assert ((got.double() - want[live]).abs() <= bound[live]).all()
    assert torch.equal(vc[page, :, at], v[live])
    # nothing else is written
    kc[page, :, :, at], vc[page, :, at] = 7.0, -3.0
    assert bool((kc == 7.0).all()) and bool((vc == -3.0).all())
    return out


@pytest.mark.parametrize("T,H,Hkv,D,P,norm,fused", [
    (1, 32, 8, 128, 64, True, False), (5, 32, 8, 128, 16, True, True), (48, 6, 3, 128, 32, False, True),
    (333, 4, 2, 64, 16, True, False), (17, 14, 2, 64, 128, False, True), (70, 5, 1, 256, 64, True, True),
    (1000, 1, 1, 256, 1024, True, False), (2049, 8, 4, 128, 64, True, True)])
def test_write_against_64_bits(dev, T, H, Hkv, D, P, norm, fused):
    c = _write_case(T, H, Hkv, D, P, T + D, dev, norm, fused)
    _check_write(*c, P)


def test_write_skips_dead_rows_and_bad_places(dev):
    """Rows without a slot, slots past the cache, positions outside the tables: stored nowhere."""
    c = list(_write_case(40, 4, 2, 128, 16, 3, dev))
    slots, pos = c[6], c[5]
    slots[3:9] = -1
    slots[12], slots[13], slots[14] = 5 * 16, 2 ** 31 - 1, -2 ** 31
    pos[20], pos[21], pos[22] = -1, 300, 2 ** 31 - 1
    _check_write(*c, 16)


@pytest.mark.parametrize("std", [1e-3, 30.0])
def test_write_scales(dev, std):
    _check_write(*_write_case(20, 4, 2, 128, 16, 8, dev, std=std), 16)


def test_write_zero_and_nonfinite_rows(dev):
    """A row of zeros stays zero (eps); NaN and infinity stay in their head's row."""
    q, k, v, cos, sin, pos, slots, qw, kw = _write_case(8, 4, 2, 128, 16, 5, dev)
    q[0], k[0] = 0, 0
    q[2, 1, 5], q[3, 0, 9], v[4, 1, 3] = math.nan, math.inf, math.nan
    kc, vc = ops.paged_cache(3, 16, 2, 128, dev)
    out = ops.paged_rope_write(q, k, v, cos, sin, pos, slots, kc, vc, qw, kw)
    assert bool((out[0] == 0).all())
    assert bool(torch.isnan(out[2, 1]).all())  # the norm spreads it over its row
    bad = torch.isnan(out).any(-1)
    bad[2, 1] = bad[3, 0] = False
    assert not bool(bad.any())
    assert bool(torch.isnan(vc).sum() == 1)


def test_write_same_as_the_training_kernels(dev):
    """Against head_norm_rope_fwd, the training layers' pass: it rounds the normalised and the weighted
    value to bf16 before the rotation, 2^-8 each of both products (1.01: and their own product)."""
    T, H, D = 64, 8, 128
    q, k, v, cos, sin, pos, slots, qw, kw = _write_case(T, H, 2, D, 16, 6, dev)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    kc, vc = ops.paged_cache(8, 16, 2, D, dev)
    got = ops.paged_rope_write(q, k, v, cos, sin, pos, slots, kc, vc, qw, kw)
    want, _ = ops.head_norm_rope_fwd(q[None], qw, cos[:T].contiguous(), sin[:T].contiguous(), 1e-6)
    _, bound, size = paged_ref.rope(q, qw, 1e-6, cos[pos.long()], sin[pos.long()])
    assert ((got.double() - want[0].double()).abs() <= 2 * bound + 1.01 * 2.0 ** -7 * size).all()


def test_write_of_no_tokens(dev):
    kc, vc = ops.paged_cache(2, 16, 2, 64, dev)
    cos, sin = _tables(4, 64, dev)
    e = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=dev)
    out = ops.paged_rope_write(e, e[:, :2].contiguous(), e[:, :2].contiguous(), cos, sin,
                               _ints([], dev), _ints([], dev), kc, vc)
    assert tuple(out.shape) == (0, 4, 64)


# ---- attention ------------------------------------------------------------------------------------
def _attn_case(lens, H, Hkv, D, P, seed, dev, std=1.5, more=2, width=None, poison=True):
    """q, caches, table: pages in random order; what is behind a row's last token (and every page and
    table entry that nobody uses) is NaN or out of range."""
    g = torch.Generator().manual_seed(seed)
    n = sum(paged_ref.pages(max(x, 0), P) for x in lens) + more
    W = max([paged_ref.pages(max(x, 0), P) for x in lens] + [1]) + 1 if width is None else width
    kc = torch.randn(n, Hkv, D // 8, P, 8, generator=g).to(torch.bfloat16)
    vc = torch.randn(n, Hkv, P, D, generator=g).to(torch.bfloat16)
    ids = torch.randperm(n, generator=g).tolist()
    table = torch.full((len(lens), W), 2 ** 31 - 1, dtype=torch.int32)
    used = torch.zeros(n, P, dtype=torch.bool)
    for b, x in enumerate(lens):
        for w in range(paged_ref.pages(max(x, 0), P)):
            table[b, w] = ids.pop()
            used[table[b, w], :min(P, x - w * P)] = True
    if poison:
        kc.masked_fill_(~used[:, None, None, :, None], math.nan)
        vc.masked_fill_(~used[:, None, :, None], math.nan)
    q = (torch.randn(len(lens), H, D, generator=g) * std).to(torch.bfloat16)
    return q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), _ints(lens, dev)


def _check_attn(q, kc, vc, table, lens, scale=None, rows=None):
    o, lse = ops.paged_attn(q, kc, vc, table, lens, scale)
    assert o.shape == q.shape and lse.shape == q.shape[:2]
    scale = q.shape[2] ** -0.5 if scale is None else scale
    for b in range(q.shape[0]) if rows is None else rows:
        k, v = paged_ref.rows_of(kc, vc, table[b], max(int(lens[b]), 0))
        wo, wl, bo, bl = paged_ref.attend(q[b], k, v, scale)
        err = (o[b].double() - wo).abs()
        assert (err <= bo).all(), (b, int(lens[b]), float((err - bo).max()))
        if lens[b] > 0:
            assert ((lse[b].double() - wl).abs() <= bl).all(), (b, int(lens[b]))
        else:
            assert bool((lse[b] == -math.inf).all())
    return o, lse


@pytest.mark.parametrize("H,Hkv,D,P", [(32, 8, 128, 64), (32, 8, 128, 16), (14, 2, 64, 32),
                                       (8, 8, 128, 32), (5, 1, 128, 128), (16, 1, 64, 16),
                                       (20, 1, 128, 64), (34, 2, 64, 256), (6, 3, 256, 64),
                                       (40, 2, 256, 1024)])
def test_attn_lengths_and_heads(dev, H, Hkv, D, P):
    """Every edge of tiles and pages, an empty row at both ends and in the middle."""
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 0, 63, 64, 65, 127, 128, 129, 300, 511, 1024, 1500, -3, 0]
    _check_attn(*_attn_case(lens, H, Hkv, D, P, H + D + P, dev))


@pytest.mark.parametrize("lens", [[1], [37], [4097], [20000], [0], [0, 0, 0], [5000, 1], [1, 5000],
                                  [3] * 300, [130] * 70, [0] * 200 + [700]],
                         ids=lambda v: f"{len(v)}x{max(v)}")
def test_attn_batches(dev, lens):
    _check_attn(*_attn_case(lens, 8, 2, 128, 64, 11, dev),
                rows=None if len(lens) < 80 else list(range(0, len(lens), 7)) + [len(lens) - 1])


def test_attn_many_ragged_requests(dev):
    rng = random.Random(4)
    lens = [rng.choice((0, 1, rng.randint(1, 60), rng.randint(1, 400))) for _ in range(1500)]
    lens[700], lens[1400] = 6000, 2500
    _check_attn(*_attn_case(lens, 4, 2, 64, 16, 12, dev), rows=[0, 1, 2, 3, 699, 700, 701, 1400, 1499]
                + rng.sample(range(1500), 30))


# four waves a request, two, one, one over several rounds
@pytest.mark.parametrize("H,Hkv,D,P,width,many", [(8, 2, 128, 64, 8, 1), (20, 1, 64, 16, 32, 1),
                                                  (3, 3, 256, 512, 1, 1), (16, 8, 128, 16, 32, 7),
                                                  (40, 8, 256, 64, 4, 4), (80, 4, 64, 32, 16, 9),
                                                  (16, 8, 128, 16, 8, 9), (4, 2, 256, 16, 20, 30),
                                                  (40, 8, 128, 32, 10, 13)])
def test_attn_small_tables_without_a_workspace(dev, H, Hkv, D, P, width, many):
    """Tables of up to 512 tokens: waves of their own for every request, no second launch; empty rows,
    every number of tiles a wave, one length past its table; and the same rows through a wider table's
    equal runs."""
    most = width * P
    lens = [min(n, most) for n in [37, 0, 512, 1, 128, 129, 300, 511, 0, 480, 33, 200, 0]] * many
    q, kc, vc, table, n = _attn_case(lens, H, Hkv, D, P, 14, dev, width=width)
    assert ops.query("plz_paged_attn_workspace", len(lens), width, P, H, Hkv, D) == 0
    o, lse = _check_attn(q, kc, vc, table, n)
    long = n.clone()
    long[3] = most + 1
    o2, lse2 = ops.paged_attn(q, kc, vc, table, long)
    assert bool(torch.isnan(o2[3]).all()) and bool(torch.isnan(lse2[3]).all())
    rest = [b for b in range(len(lens)) if b != 3]
    assert torch.equal(o2[rest], o[rest]) and torch.equal(lse2[rest], lse[rest])
    wide = torch.cat([table] * (512 // most + 1), 1).contiguous()
    assert ops.query("plz_paged_attn_workspace", len(lens), wide.shape[1], P, H, Hkv, D) > 0
    _check_attn(q, kc, vc, wide, n)


def test_attn_many_requests_of_small_tables(dev):
    """More (request, kv head) pairs than a grid's second dimension takes."""
    B = 9000
    g = torch.Generator(device=dev).manual_seed(2)
    kc = torch.randn(64, 8, 8, 16, 8, generator=g, device=dev).to(torch.bfloat16)
    vc = torch.randn(64, 8, 16, 64, generator=g, device=dev).to(torch.bfloat16)
    q = torch.randn(B, 8, 64, generator=g, device=dev).to(torch.bfloat16)
    table = torch.randint(0, 64, (B, 3), generator=g, device=dev, dtype=torch.int32)
    lens = torch.randint(0, 49, (B,), generator=g, device=dev, dtype=torch.int32)
    _check_attn(q, kc, vc, table, lens, rows=[0, 1, 8191, 8192, 8999] + list(range(5, B, 700)))


def test_attn_largest_batch(dev):
    """65536 requests, 1024 a lane of the waves that deal them out; and a wave each."""
    B = 65536
    g = torch.Generator(device=dev).manual_seed(3)
    kc = torch.randn(32, 1, 8, 16, 8, generator=g, device=dev).to(torch.bfloat16)
    vc = torch.randn(32, 1, 16, 64, generator=g, device=dev).to(torch.bfloat16)
    q = torch.randn(B, 2, 64, generator=g, device=dev).to(torch.bfloat16)
    table = torch.randint(0, 32, (B, 33), generator=g, device=dev, dtype=torch.int32)
    lens = torch.randint(-8, 66, (B,), generator=g, device=dev, dtype=torch.int32).clamp_(0, 64)
    lens[:3000] = 0
    lens[-1] = 64
    for t in (table, table[:, :4].contiguous()):
        _check_attn(q, kc, vc, t, lens, rows=[0, 2999, 3000, 65535] + list(range(3001, B, 1500)))


@pytest.mark.parametrize("B", [3, 3000])
def test_attn_table_without_columns(dev, B):
    kc, vc = ops.paged_cache(2, 16, 2, 128, dev)
    q = torch.randn(B, 4, 128, device=dev, dtype=torch.bfloat16)
    lens = torch.zeros(B, dtype=torch.int32, device=dev)
    lens[1] = 5  # more than the table holds
    o, lse = ops.paged_attn(q, kc, vc, lens.new_empty(B, 0), lens)
    rest = [0] + list(range(2, B))
    assert bool((o[rest] == 0).all()) and bool((lse[rest] == float("-inf")).all())
    assert bool(torch.isnan(o[1]).all()) and bool(torch.isnan(lse[1]).all())


@pytest.mark.parametrize("std", [0.05, 12.0])
def test_attn_flat_and_peaked(dev, std):
    _check_attn(*_attn_case([700, 90, 1, 2100], 8, 2, 128, 64, 5, dev, std=std))


def test_attn_rising_and_falling_scores(dev):
    """Key norms that grow or shrink along the sequence: the running maximum moves in every tile, or
    never after the first."""
    q, kc, vc, table, lens = _attn_case([1000, 1000], 8, 2, 128, 64, 6, dev)
    for b, growth in ((0, 1.0), (1, -1.0)):
        for w in range(16):
            ramp = torch.exp(growth * (torch.arange(64, device=dev) + 64 * w - 500) / 250)
            page = int(table[b, w])
            kc[page] = (kc[page].float() * ramp[:, None]).to(torch.bfloat16)
    _check_attn(q, kc, vc, table, lens)


def test_attn_scale(dev):
    _check_attn(*_attn_case([300, 17], 8, 2, 128, 16, 7, dev), scale=0.3)


def test_attn_pitched_queries(dev):
    q, kc, vc, table, lens = _attn_case([300, 17, 0, 90], 8, 2, 128, 16, 8, dev)
    wide = torch.full((4, 12, 128), math.nan, dtype=torch.bfloat16, device=dev)
    wide[:, 2:10] = q
    o, lse = _check_attn(wide[:, 2:10], kc, vc, table, lens)
    o2, lse2 = ops.paged_attn(q, kc, vc, table, lens)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_attn_bad_tables_give_nan_in_their_rows_only(dev):
    """A page number outside the cache (both signs) among those that a row needs, and a length past its
    table: NaN there, the other rows as they are."""
    lens = [200, 200, 700, 64, 5]
    q, kc, vc, table, n = _attn_case(lens, 8, 2, 128, 64, 9, dev)
    want, want_lse = ops.paged_attn(q, kc, vc, table, n)
    bad = table.clone()
    bad[0, 3], bad[2, 9] = kc.shape[0], -1
    long = n.clone()
    long[4] = table.shape[1] * 64 + 1
    o, lse = ops.paged_attn(q, kc, vc, bad, long)
    for b in (0, 2, 4):
        assert bool(torch.isnan(o[b]).all()) and bool(torch.isnan(lse[b]).all())
    for b in (1, 3):
        assert torch.equal(o[b], want[b]) and torch.equal(lse[b], want_lse[b])
    none = ops.paged_attn(q, kc, vc, table[:, :0].contiguous(), n)
    assert bool(torch.isnan(none[0]).all())
    none = ops.paged_attn(q, kc, vc, table[:, :0].contiguous(), n * 0)
    assert bool((none[0] == 0).all()) and bool((none[1] == -math.inf).all())


def test_attn_nonfinite_values(dev):
    """Infinite and NaN entries of the tokens themselves act as in the formula: in the heads and
    columns that they reach, nowhere else."""
    q, kc, vc, table, lens = _attn_case([100, 100, 100], 8, 2, 128, 16, 10, dev)
    page = table[1, 2].item()
    vc[page, 0, 5, 7] = math.inf
    kc[table[2, 1].item(), 1, 3, 4, 2] = math.nan
    o, lse = ops.paged_attn(q, kc, vc, table, lens)
    assert bool((o[1, :4, 7] == math.inf).all())
    o2 = o.clone()
    o2[1, :4, 7] = 0
    assert bool(torch.isfinite(o2[:2]).all()) and bool(torch.isfinite(o2[2, :4]).all())
    assert bool(torch.isnan(o2[2, 4:]).all()) and bool(torch.isnan(lse[2, 4:]).all())
    # a key that gives -inf (weight 0) among finite ones
    q, kc, vc, table, lens = _attn_case([400], 2, 2, 128, 16, 10, dev)
    q[0, :, 0] = 1.0
    want_k = kc.clone()
    for t in range(0, 300):
        kc[table[0, t // 16].item(), :, 0, t % 16, 0] = -math.inf
    o, lse = ops.paged_attn(q, kc, vc, table, lens)
    k, v = paged_ref.rows_of(want_k, vc, table[0], 400)
    wo, wl, bo, bl = paged_ref.attend(q[0], k[300:], v[300:], 128 ** -0.5)
    assert ((o[0].double() - wo).abs() <= bo).all() and ((lse[0].double() - wl).abs() <= bl).all()


# waves a request (many requests of 8 kv heads): four, two, one, one over several rounds, equal runs
@pytest.mark.parametrize("many,width", [(1, 16), (17, 32), (20, 8), (60, 20), (60, 40)])
def test_attn_bad_and_nonfinite_rows_among_many(dev, many, width):
    """Rows with a page outside the cache, an infinite value and a NaN key, each among good ones, through
    every way of dealing requests to waves: only what they reach differs."""
    lens = [100, 90, 128, 1, 0, 77]
    q, kc, vc, table, n = _attn_case(lens, 16, 8, 128, 16, 17, dev, width=width)
    again = dict(k_cache=kc, v_cache=vc, block_table=table.repeat(many, 1), lens=n.repeat(many))
    qs = q.repeat(many, 1, 1)
    want, want_lse = ops.paged_attn(qs, **again)
    # row 0 needs a page that is not there, in its last tile; the first value of row 1's token 40 and of
    # row 2's token 70 in kv head 3 are infinite and NaN
    again["block_table"][:, 6].masked_fill_(again["lens"] == 100, kc.shape[0])
    vc[table[1, 2], 3, 8, 0] = math.inf
    kc[table[2, 4], 3, 0, 6, 0] = math.nan
    o, lse = ops.paged_attn(qs, **again)
    kind = torch.arange(len(lens) * many, device=dev) % len(lens)
    assert bool(torch.isnan(o[kind == 0]).all()) and bool(torch.isnan(lse[kind == 0]).all())
    assert bool((o[kind == 1][:, 6:8, 0] == math.inf).all())
    assert bool(torch.isnan(o[kind == 2][:, 6:8]).all()) and bool(torch.isnan(lse[kind == 2][:, 6:8]).all())
    same = (kind != 0)[:, None, None].expand_as(o).clone()
    same[kind == 1, 6:8, 0] = False
    same[kind == 2, 6:8] = False
    assert torch.equal(o[same], want[same])
    assert torch.equal(lse[kind == 1], want_lse[kind == 1]) and torch.equal(lse[kind > 2], want_lse[kind > 2])


def test_attn_twice_gives_the_same_bits(dev):
    c = _attn_case([3000, 1, 77, 0, 900], 32, 8, 128, 64, 13, dev)
    o, lse = ops.paged_attn(*c)
    for _ in range(3):
        o2, lse2 = ops.paged_attn(*c)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_attn_cache_past_32_bit_offsets(dev):
    """A cache of 5 GB for each of K and V: pages at its end, past 2^32 bytes and 2^31 values."""
    Hkv, D, P, n = 8, 128, 64, 40000
    kc = torch.empty(n, Hkv, D // 8, P, 8, dtype=torch.bfloat16, device=dev)
    vc = torch.empty(n, Hkv, P, D, dtype=torch.bfloat16, device=dev)
    table = _ints([[n - 1, 3, n - 2], [39000, 38999, 7]], dev)
    g = torch.Generator(device=dev).manual_seed(1)
    for page in table.flatten().tolist():
        kc[page] = torch.randn(kc.shape[1:], generator=g, device=dev).to(torch.bfloat16)
        vc[page] = torch.randn(vc.shape[1:], generator=g, device=dev).to(torch.bfloat16)
    q = torch.randn(2, 32, D, generator=g, device=dev).to(torch.bfloat16)
    _check_attn(q, kc, vc, table, _ints([190, 129], dev))
    # and a write there
    x = torch.randn(3, Hkv, D, generator=g, device=dev).to(torch.bfloat16)
    cos, sin = torch.ones(4, D, device=dev), torch.zeros(4, D, device=dev)
    slots = _ints([(n - 1) * P + 63, (n - 2) * P, 39000 * P + 1], dev)
    ops.paged_rope_write(x, x, x, cos, sin, _ints([0, 1, 2], dev), slots, kc, vc)
    page, at = slots.long() // P, slots.long() % P
    assert torch.equal(kc[page, :, :, at].reshape(3, Hkv, D), x) and torch.equal(vc[page, :, at], x)


# ---- streams, graphs, a decoding batch ------------------------------------------------------------------
class _Loop:
    """A batch that decodes through the three operators with static buffers, one layer."""

    def __init__(self, dev, B=3, H=8, Hkv=2, D=128, P=16, W=8, pages=20, seed=0):
        self.P, self.dev = P, dev
        self.lens, self.count = _ints([0] * B, dev), _ints([pages], dev)
        self.table = torch.zeros(B, W, dtype=torch.int32, device=dev)
        self.free = torch.arange(pages, dtype=torch.int32, device=dev)
        self.kc, self.vc = ops.paged_cache(pages, P, Hkv, D, dev)
        self.new = _ints([1] * B, dev)
        self.cos, self.sin = _tables(W * P, D, dev)
        self.qkv = torch.zeros(B, (H + 2 * Hkv) * D, dtype=torch.bfloat16, device=dev)
        self.q, self.k, self.v = (x.unflatten(1, (-1, D)) for x in
                                  self.qkv.split([H * D, Hkv * D, Hkv * D], 1))
        self.g = torch.Generator().manual_seed(seed)

    def feed(self):
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=self.g).to(torch.bfloat16))

    def pass_(self):
        slots, pos, _, _, _ = ops.paged_step(self.lens, self.new, self.table, self.free, self.count,
                                             self.P, lens_out=self.lens, free_count_out=self.count)
        q = ops.paged_rope_write(self.q, self.k, self.v, self.cos, self.sin, pos, slots, self.kc, self.vc)
        return ops.paged_attn(q, self.kc, self.vc, self.table, self.lens)


def test_decoding_batch_against_whole_sequences(dev):
    """Seventy tokens of three requests, one row without a token in every third step: each step's
    output is the last row of attention over the whole sequence so far, in 64 bits from the bf16 q, k
    and v that the operators' own roundings give."""
    loop = _Loop(dev)
    ks, vs = [[] for _ in range(3)], [[] for _ in range(3)]
    for step in range(70):
        loop.feed()
        live = [0, 1, 2] if step % 3 else [0, 2]
        loop.new.copy_(torch.tensor([1 if b in live else 0 for b in range(3)]))
        # rows follow each other: the token rows of the live requests come first
        slots, pos, starts, _, _ = ops.paged_step(
            loop.lens, loop.new, loop.table, loop.free, loop.count, loop.P, lens_out=loop.lens,
            free_count_out=loop.count)
        q = ops.paged_rope_write(loop.q, loop.k, loop.v, loop.cos, loop.sin, pos, slots, loop.kc,
                                 loop.vc)
        per_request = torch.zeros_like(q)
        for row, b in enumerate(live):
            per_request[b] = q[row]
            c, s = loop.cos[len(ks[b])][None], loop.sin[len(ks[b])][None]
            want, bound, _ = paged_ref.rope(loop.k[row:row + 1], None, 0, c, s)
            got = paged_ref.rows_of(loop.kc, loop.vc, loop.table[b], len(ks[b]) + 1)[0][-1]
            assert ((got.double() - want[0]).abs() <= bound[0]).all()
            ks[b].append(got.clone()), vs[b].append(loop.v[row].clone())
        o, lse = ops.paged_attn(per_request, loop.kc, loop.vc, loop.table, loop.lens)
        assert loop.lens.tolist() == [len(x) for x in ks]
        for b in range(3):
            if ks[b]:
                wo, wl, bo, bl = paged_ref.attend(per_request[b], torch.stack(ks[b]), torch.stack(vs[b]),
                                                  128 ** -0.5)
                assert ((o[b].double() - wo).abs() <= bo).all()
                assert ((lse[b].double() - wl).abs() <= bl).all()


def test_decoding_on_another_stream(dev):
    a, b = _Loop(dev, seed=1), _Loop(dev, seed=1)
    side = torch.cuda.Stream()
    for _ in range(5):
        a.feed(), b.feed()
        want = a.pass_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = b.pass_()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_decoding_in_a_graph(dev):
    """One captured step, replayed forty times with eager work of its own kind and synchronisations
    between the replays, against the same steps run eagerly, bit for bit."""
    a, b = _Loop(dev, seed=2, pages=30), _Loop(dev, seed=2, pages=30)
    b.feed()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.pass_()
    torch.cuda.current_stream().wait_stream(side)
    # back to the start
    fresh = _Loop(dev, seed=2, pages=30)
    for nm in ("lens", "count", "table", "free", "kc", "vc"):
        getattr(b, nm).copy_(getattr(fresh, nm))
    b.g = torch.Generator().manual_seed(2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.pass_()
    other = _Loop(dev, seed=5, B=7, pages=60)
    for i in range(40):
        a.feed(), b.feed()
        want = a.pass_()
        graph.replay()
        if i % 3 == 0:
            other.feed()
            other.pass_()
        if i % 4 == 0:
            torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want)), i
        assert torch.equal(a.table, b.table) and torch.equal(a.lens, b.lens)


def test_two_calls_at_once(dev):
    """Eager attentions of two batches on two streams without a wait between them, again and again."""
    cases = [_attn_case([2500, 5, 700, 1200], 8, 2, 128, 64, 40 + i, dev) for i in range(2)]
    want = [ops.paged_attn(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_attn(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, y) for g in got[i] for x, y in zip(g, want[i]))


def test_two_graphs_of_attention_side_by_side(dev):
    """Two captured attentions replayed on two streams at once, each against its eager result."""
    cases = [_attn_case([3000, 5, 700], 8, 2, 128, 64, 30 + i, dev) for i in range(2)]
    want = [ops.paged_attn(*c) for c in cases]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_attn(*c))
        graphs.append(g)
    for _ in range(10):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(got, ref))
            for x in got:
                x.zero_()


# ---- what the sizes above do not reach ------------------------------------------------------------------
def _each(T, H, Hkv, D):
    """Heads a workgroup of the cache write."""
    tb, heads = 4 * (64 // (D // 8)), H + 2 * Hkv
    each = 1
    while each < 8 and -(-T // tb) * heads >= 2048 * each:
        each *= 2
    return each


# groups of 4 and 8 heads: across q | k and k | v, the last one ragged, tokens that fill no block
@pytest.mark.parametrize("T,H,Hkv,D,P,norm,fused,each", [
    (4001, 14, 2, 128, 64, True, True, 4), (9403, 5, 1, 128, 16, False, False, 4),
    (8191, 14, 2, 128, 32, True, False, 8), (18811, 5, 1, 128, 64, True, True, 8),
    (8007, 14, 2, 64, 16, True, False, 4), (37501, 5, 1, 64, 64, True, True, 8),
    (17503, 9, 3, 64, 128, False, True, 8), (2201, 14, 2, 256, 64, False, True, 4),
    (4771, 5, 1, 256, 16, True, True, 4), (4409, 9, 3, 256, 32, True, False, 8)])
def test_write_of_many_heads_a_workgroup(dev, T, H, Hkv, D, P, norm, fused, each):
    assert _each(T, H, Hkv, D) == each
    c = list(_write_case(T, H, Hkv, D, P, T + D, dev, norm, fused))
    pos, slots = c[5], c[6]
    dead = torch.randperm(T, generator=torch.Generator().manual_seed(T))[:200].to(dev)
    slots[dead[:100]] = -1
    pos[dead[100:120]] = 300
    slots[-3:] = -1
    _check_write(*c, P)


def _waves(batch, width, P, H, Hkv, D):
    """Waves a (kv head, 16 query heads) that the equal runs are dealt to, from the workspace's size."""
    G = H // Hkv
    tiles = -(-G // 16)
    need = ops.query("plz_paged_attn_workspace", batch, width, P, H, Hkv, D)
    part = Hkv * tiles * 2 * min(G, 16) * D * 4 + H * 16 + 8
    assert need > 0 and need % part == 0
    return 4 * need // part


# What tile i (32 tokens) of a request adds to its scores, in log2 units
RAMPS = {"rising": lambda i: 10.0 * i, "falling": lambda i: -10.0 * i, "slow": lambda i: 3.0 * i,
         "sawtooth": lambda i: (0.0, 9.0, 20.0, 4.0, 31.0)[i % 5] + i, "flat": lambda i: 0.0 * i}


def _ramped(lens, H, Hkv, D, P, seed, dev, width=None):
    """_attn_case whose request b's scores follow ramp b % 5, tile by tile: value 0 of a key is what its
    tile adds, value 0 of a query 16, the others are noise of standard deviation about 1 in log2 units."""
    q, kc, vc, table, n = _attn_case(lens, H, Hkv, D, P, seed, dev, std=0.7, width=width)
    scale = D ** -0.5
    unit = 16 * scale / math.log(2)
    q[:, :, 0] = 16
    ramps = list(RAMPS.values())
    for b, x in enumerate(lens):
        t = torch.arange(x, device=dev)
        add = torch.tensor([ramps[b % len(ramps)](i) for i in range(-(-x // 32))], device=dev) / unit
        page, at = table[b].long()[t // P], t % P
        kc[page, :, 0, at, 0] = add[t // 32].to(torch.bfloat16)[:, None]
    return q, kc, vc, table, n


def _check_heads(c, heads, got=None, rows=None):
    """paged_attn on c, these query heads of it (of one kv head each) against 64 bits."""
    q, kc, vc, table, lens = c
    o, lse = ops.paged_attn(*c) if got is None else got
    G = q.shape[1] // vc.shape[1]
    for b in range(q.shape[0]) if rows is None else rows:
        k, v = paged_ref.rows_of(kc, vc, table[b], int(lens[b]))
        for h in heads:
            wo, wl, bo, bl = paged_ref.attend(q[b, h:h + 1], k[:, h // G, None], v[:, h // G, None],
                                              q.shape[2] ** -0.5)
            assert ((o[b, h].double() - wo[0]).abs() <= bo[0]).all(), (b, h)
            assert ((lse[b, h].double() - wl[0]).abs() <= bl[0]).all(), (b, h)
    return o, lse


@pytest.mark.parametrize("H,Hkv,D,P", [(32, 32, 128, 64), (96, 48, 64, 16), (30, 15, 256, 32)])
def test_attn_ramps_in_one_wave(dev, H, Hkv, D, P):
    """Tables of 320 tokens and more pairs of requests and kv heads than have a place at once: one wave for
    all ten tiles of a request, whose maximum moves at every tile, at some, or never."""
    width = 320 // P
    lens = [320, 320, 320, 320, 320, 311, 289, 300, 320, 257, 33, 64] * 4
    resident = {64: 768, 128: 512, 256: 256}[D]
    assert len(lens) * Hkv > 2 * resident
    assert ops.query("plz_paged_attn_workspace", len(lens), width, P, H, Hkv, D) == 0
    _check_heads(_ramped(lens, H, Hkv, D, P, 18, dev, width=width), [0, H // 2, H - 1],
                 rows=list(range(12)) + [47])


# (heads, kv heads, head dim, page, lengths, tiles a wave at least): 8 workgroups a (kv head, 16 heads) in
# the first four, 1 and 32
LONG = [(1024, 1, 64, 16, [40000, 40001], 70), (1024, 4, 64, 64, [30000, 20, 50007], 70),
        (1024, 2, 64, 1024, [45000, 36001], 70), (512, 1, 128, 64, [40000, 36003], 70),
        (8192, 1, 64, 32, [5000, 0, 5003, 65], 70), (8, 8, 256, 16, [21000, 1, 21500, 9], 8)]


@pytest.mark.parametrize("H,Hkv,D,P,lens,tiles", LONG)
def test_attn_many_tiles_a_wave(dev, H, Hkv, D, P, lens, tiles):
    """Runs of more tiles of one request than a wave looks up pages for at once (32), a page that is not
    there behind the first 32 tiles of a run, which makes its request NaN and leaves the others as they are,
    and requests of every ramp, of about as many tiles as a run."""
    heads = [0, 1, H // 2 + 1, H - 1]
    q, kc, vc, table, n = c = _attn_case(lens, H, Hkv, D, P, 19, dev)
    waves = _waves(len(lens), table.shape[1], P, H, Hkv, D)
    total = sum(-(-x // 32) for x in lens)
    assert total // waves >= tiles
    o, lse = _check_heads(c, heads, rows=[b for b, x in enumerate(lens) if x])
    for b, x in enumerate(lens):
        if x == 0:
            assert bool((o[b] == 0).all()) and bool((lse[b] == -math.inf).all())
    run = total // waves
    bad = table.clone()
    bad[0, (min(run, 50) - 5) * 32 // P] = kc.shape[0]
    o2, lse2 = ops.paged_attn(q, kc, vc, bad, n)
    assert bool(torch.isnan(o2[0]).all()) and bool(torch.isnan(lse2[0]).all())
    assert torch.equal(o2[1:], o[1:]) and torch.equal(lse2[1:], lse[1:])
    if run < 32:
        return
    lens = [32 * 70, 32 * 71 - 5, 32 * 68 + 1, 32 * 70, 32 * 64] * (2 * waves // 5 + 1)
    c = _ramped(lens, H, Hkv, D, P, 20, dev)
    assert sum(-(-x // 32) for x in lens) // _waves(len(lens), c[3].shape[1], P, H, Hkv, D) >= 70
    _check_heads(c, heads[1:3], rows=list(range(5)) + [len(lens) - 1])


def test_attn_of_one_workgroup_a_head(dev):
    """As many (kv head, 16 heads) pairs as workgroups: each has one, which joins nothing with others, for
    several requests, empty ones among them."""
    for H, Hkv, D in ((8192, 1, 64), (512, 512, 64), (512, 256, 256)):
        lens = [700, 0, 2000, 1, 0, 515]
        c = _attn_case(lens, H, Hkv, D, 16, 21, dev)
        assert _waves(len(lens), c[3].shape[1], 16, H, Hkv, D) == 4
        o, lse = _check_heads(c, [0, H // 2, H - 1], rows=[0, 2, 3, 5])
        assert bool((o[[1, 4]] == 0).all()) and bool((lse[[1, 4]] == -math.inf).all())
