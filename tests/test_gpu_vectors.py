"""GPU suite: the document-vector operators (include/mdd.h, "Document vectors") against their definitions in 64 bits.

Tolerances are bounds, not measurements: an output rounded once is off by half a step of its value (R.half), and a float sum of n
terms by at most n * 2^-24 of the sum of their magnitudes, whatever its order; products and factors add a 2^-24 each."""
import numpy as np
import pytest
import torch

import os
import sys

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import vec_ref as R  # noqa: E402
from map_neo_amd.lib import MddError

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _close(got, want, tol, what=""):
    got = got.double().cpu()
    off = (got - want).abs()
    worst = (off - tol).max().item() if off.numel() else 0.0
    assert got.shape == want.shape and worst <= 0, f"{what}: off by {off.max().item():.3g}, {worst:.3g} beyond the bound"


def _ragged(lens, dev):
    o = np.zeros(len(lens) + 1, np.int64)
    o[1:] = np.cumsum(lens)
    return torch.from_numpy(o).to(dev)


def _ids(n, v, g, dtype=torch.int32, hot=0):
    ids = torch.randint(-1, v + 1, (n,), generator=g)          # -1 and v are padding
    if hot:
        ids[torch.rand(n, generator=g) < 0.3] = hot
    return ids.to(dtype)


# ---------------------------------------------------------------------------------------------------- embedding lookup
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,n,idt", [(1, 1, torch.int32), (8, 33, torch.int64), (31, 100, torch.int32), (64, 257, torch.int64),
                                       (129, 65, torch.int32), (256, 16, torch.int32), (513, 70, torch.int64), (1100, 9, torch.int32)])
def test_embed_rows(engine, dtype, dim, n, idt):
    g = torch.Generator().manual_seed(dim * 7 + n)
    table, ids = torch.randn(50, dim, generator=g).to(dtype), _ids(n, 50, g, idt)
    got = engine.embed(table.cuda(), ids.cuda(), scale=1.7)
    want, mag, _ = R.embed(table, ids, None, float(np.float32(1.7)), "sum")
    assert got.dtype == dtype
    _close(got, want, R.half(dtype, mag) + 2 * R.U32 * mag)
    assert (got[(ids < 0) | (ids >= 50)] == 0).all()


@pytest.mark.parametrize("mode", ["mean", "sum"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,lens", [(1, [0, 1, 2]), (24, [5, 0, 0, 64, 65, 1]), (64, [100, 0, 3000, 7, 129]), (200, [31, 33, 0, 1]),
                                      (256, [1]), (300, [0, 0, 0]), (520, [9, 2000, 40]), (1024, [32, 33, 31, 64, 1, 500])])
def test_embed_documents(engine, dtype, mode, dim, lens):
    """ragged documents, empty ones, ones longer than a piece of the id axis (32 ids at these sizes), odd widths"""
    g = torch.Generator().manual_seed(dim + len(lens))
    n = sum(lens)
    table, ids = torch.randn(97, dim, generator=g).to(dtype), _ids(n, 97, g)
    offs = _ragged(lens, "cuda")
    got = engine.embed(table.cuda(), ids.cuda(), offs, scale=0.5, mode=mode)
    want, mag, cnt = R.embed(table, ids, offs, 0.5, mode)
    assert got.shape == (len(lens), dim) and got.dtype == dtype
    _close(got, want, R.half(dtype, want.abs()) + (cnt[:, None].double() + 4) * R.U32 * mag)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [512, 768, 1000])
def test_embed_documents_of_a_large_table(engine, dtype, dim):
    """a table beyond an L2 whose rows are named again: columns in slabs of 256, the last one short; one document longer than a
    piece, empty ones, infinities and a NaN in single columns; and from rows further apart than their width"""
    g = torch.Generator().manual_seed(dim)
    lens = [0, 4000] + torch.randint(0, 90, (200,), generator=g).tolist() + [0, 1]
    v = sum(lens) // 2
    wide = torch.randn(v, dim + 8, generator=g).to(dtype)
    wide[7, 3], wide[8, 259], wide[9, dim - 1] = float("inf"), float("nan"), -float("inf")
    table, ids = wide[:, :dim], _ids(sum(lens), v, g)
    assert v * dim * wide.element_size() > 4 << 20 and ids.numel() >= 32 * len(lens)
    offs = _ragged(lens, "cuda")
    got = engine.embed(table.contiguous().cuda(), ids.cuda(), offs, scale=0.5)
    want, mag, cnt = R.embed(table, ids, offs, 0.5, "mean")
    odd = ~want.isfinite()
    g64 = got.double().cpu()
    assert odd.any() and (g64[odd].isnan() == want[odd].isnan()).all() and (g64[odd & ~want.isnan()] == want[odd & ~want.isnan()]).all()
    tol = R.half(dtype, want.abs()) + (cnt[:, None].double() + 4) * R.U32 * mag
    _close(got.cpu().masked_fill(odd, 0), want.masked_fill(odd, 0), tol.masked_fill(odd, 0))
    assert torch.equal(engine.embed(wide.cuda()[:, :dim], ids.cuda(), offs, scale=0.5).view(torch.uint8), got.view(torch.uint8))


def test_calls_beyond_the_last_level_cache(engine):
    """results of more than 256 MiB go past the caches: the same numbers as in two halves, which do not"""
    g = torch.Generator(device="cuda").manual_seed(1)
    n, dim = 70002, 1000
    table = torch.randn(500, dim, generator=g, device="cuda")
    ids = torch.randint(-1, 501, (n,), generator=g, device="cuda", dtype=torch.int32)
    got = engine.embed(table, ids)
    assert got.numel() * 4 > 1 << 28 and torch.equal(got, torch.cat([engine.embed(table, ids[: n // 2]), engine.embed(table, ids[n // 2:])]))
    # every position a document of its own is the same gradient in the same order, read through the caches
    each = torch.arange(n + 1, device="cuda")
    assert torch.equal(engine.embed_backward(got, ids, 500), engine.embed_backward(got, ids, 500, each, mode="sum"))
    x, r, w = got[: n // 2], got[n // 2:], torch.randn(dim, generator=g, device="cuda")
    whole, parts = engine.rms_norm(x, w, r), [engine.rms_norm(a, w, b) for a, b in zip(x.chunk(3), r.chunk(3))]
    assert all(torch.equal(whole[k], torch.cat([q[k] for q in parts])) for k in range(3))
    for kind in ("int8", "e4m3"):
        whole, parts = engine.rms_norm_q8(x, w, r, kind=kind), [engine.rms_norm_q8(a, w, b, kind=kind) for a, b in zip(x.chunk(4), r.chunk(4))]
        assert all(torch.equal(whole[k].view(torch.uint8), torch.cat([q[k].view(torch.uint8) for q in parts])) for k in range(3))


def test_embed_one_long_document_and_many_short(engine):
    """pieces of 32 to 1024 ids: one document of 300000 ids among short ones, a document of padding only"""
    g = torch.Generator().manual_seed(5)
    lens = [3, 300000, 0, 40, 1, 700]
    table, ids = torch.randn(500, 40, generator=g), _ids(sum(lens), 500, g, torch.int64)
    ids[300003:300043] = -1
    offs = _ragged(lens, "cuda")
    for mode in ("mean", "sum"):
        got = engine.embed(table.cuda(), ids.cuda(), offs, mode=mode)
        want, mag, cnt = R.embed(table, ids, offs, 1.0, mode)
        _close(got, want, (cnt[:, None].double() + 4) * R.U32 * mag)
        assert (got[3] == 0).all() and (got[2] == 0).all()
        assert torch.equal(got, engine.embed(table.cuda(), ids.cuda(), offs, mode=mode))


def test_embed_views_nan_in_unused_rows_and_offsets_out_of_range(engine):
    g = torch.Generator().manual_seed(6)
    wide = torch.randn(60, 50, generator=g)
    wide[0] = float("nan")                                      # row 0 is what padding lanes read: it must not leak
    ids = torch.tensor([-1, 5, 59, -7, 60, 2 ** 31 - 1, 8], dtype=torch.int32)
    offs = torch.tensor([0, 2, 2, 7])
    table = wide.cuda()[:, 3:40]                                # row stride 50, odd start
    want, mag, cnt = R.embed(wide[:, 3:40], ids, offs, 1.0, "sum")
    got = engine.embed(table, ids.cuda(), offs.cuda(), mode="sum")
    _close(got, want, (cnt[:, None].double() + 4) * R.U32 * mag)
    _close(engine.embed(table, ids.cuda()), R.embed(wide[:, 3:40], ids, None, 1.0, "sum")[0], 0.0)
    bad = torch.tensor([0, 2, 10 ** 15, 7, 3], dtype=torch.int64).cuda()   # clamped: no access outside ids
    assert engine.embed(table, ids.cuda(), bad, mode="sum").shape == (4, 37)
    assert (engine.embed(table[:0], ids.cuda(), offs.cuda()) == 0).all()   # an empty table: all padding
    assert engine.embed(table, ids[:0].cuda()).shape == (0, 37)
    assert (engine.embed(table, ids[:0].cuda(), torch.zeros(4, dtype=torch.int64).cuda()) == 0).all()
    assert engine.embed(table, ids.cuda(), torch.zeros(1, dtype=torch.int64).cuda()).shape == (0, 37)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,n,v,docs", [(1, 1, 1, 0), (16, 40, 9, 0), (37, 300, 64, 5), (64, 9000, 300, 0), (130, 20000, 70000, 40),
                                          (512, 700, 40, 3), (1030, 100, 5, 0)])
def test_embed_backward(engine, dtype, dim, n, v, docs):
    """one-block sort (<= 8192 ids) and the passes beyond, a hot id, ids that nothing names, shared documents"""
    g = torch.Generator().manual_seed(dim + n)
    ids = _ids(n, v, g, torch.int64 if n % 2 else torch.int32, hot=v // 2)
    offs = None
    if docs:
        cut = torch.sort(torch.randint(0, n + 1, (docs - 1,), generator=g)).values
        offs = torch.cat([torch.tensor([0]), cut, torch.tensor([n - n // 10])]).sort().values      # ids behind the last document
    grad = torch.randn(docs or n, dim, generator=g).to(dtype)
    for mode in ("mean", "sum") if docs else ("sum",):
        dev = None if offs is None else offs.cuda()
        got = engine.embed_backward(grad.cuda(), ids.cuda(), v, dev, scale=1.25, mode=mode)
        want, mag, cnt = R.embed_backward(grad, ids, v, offs, 1.25, mode)
        assert got.dtype == torch.float32 and got.shape == (v, dim)
        _close(got, want, (cnt + 5) * R.U32 * mag, mode)
        assert torch.equal(got, engine.embed_backward(grad.cuda(), ids.cuda(), v, dev, scale=1.25, mode=mode))
        low = engine.embed_backward(grad.cuda(), ids.cuda(), v, dev, scale=1.25, mode=mode, dtype=dtype)
        assert torch.equal(low, got.to(dtype))


@pytest.mark.parametrize("mode", ["mean", "sum"])
@pytest.mark.parametrize("long", [200, 1500, 9000])
def test_embed_backward_many_empty_documents(engine, long, mode):
    """more documents begin within 64 positions than a wave holds, and fewer; positions before the first and behind the last one"""
    g = torch.Generator().manual_seed(long)
    lens = [0] * 100 + [3] + [0] * 70 + [1] * 80 + [long] + [0] * 65 + [5, 62, 64, 1, 0, 63]
    n = sum(lens) + 150
    ids, offs = _ids(n, 40, g), _ragged(lens, "cuda") + 100
    grad = torch.randn(len(lens), 9, generator=g)
    got = engine.embed_backward(grad.cuda(), ids.cuda(), 40, offs, scale=1.5, mode=mode)
    want, mag, cnt = R.embed_backward(grad, ids, 40, offs, 1.5, mode)
    _close(got, want, R.half(torch.float32, want.abs()) + (cnt + 4) * R.U32 * mag)


def test_embed_gradient_against_differences(engine):
    """d loss / d table by central differences of the forward pass (linear: any step is exact up to rounding)"""
    g = torch.Generator().manual_seed(11)
    table, ids = torch.randn(12, 5, generator=g).cuda(), torch.tensor([3, 3, -1, 7, 0, 11, 3], dtype=torch.int32).cuda()
    offs, w = torch.tensor([0, 4, 4, 7]).cuda(), torch.randn(3, 5, generator=g).cuda()
    grad = engine.embed_backward(w, ids, 12, offs, scale=2.0)
    for r, c in ((3, 0), (7, 4), (0, 2), (1, 1), (11, 3)):
        up, dn = table.clone(), table.clone()
        up[r, c] += 0.5
        dn[r, c] -= 0.5
        d = ((engine.embed(up, ids, offs, scale=2.0).double() - engine.embed(dn, ids, offs, scale=2.0).double()) * w.double()).sum()
        assert abs(d.item() - grad[r, c].item()) < 2e-5      # 30 roundings of 2^-24 of values below 8


def test_embed_backward_empty(engine):
    e32, none = torch.zeros(0, dtype=torch.int32).cuda(), torch.zeros(0, 7).cuda()
    assert (engine.embed_backward(none, e32, 5) == 0).all()
    assert engine.embed_backward(none, e32, 0).shape == (0, 7)
    assert (engine.embed_backward(torch.ones(3, 7).cuda(), e32, 5, torch.zeros(4, dtype=torch.int64).cuda()) == 0).all()
    ids = torch.tensor([1, 1, 4], dtype=torch.int32).cuda()
    assert (engine.embed_backward(none, ids, 5, torch.zeros(1, dtype=torch.int64).cuda()) == 0).all()      # ids in no document


# ---------------------------------------------------------------------------------------------------- norm
DIMS = [(1, 3), (7, 5), (8, 33), (9, 70), (64, 1), (100, 37), (129, 18), (250, 9), (257, 9), (384, 11), (390, 21), (515, 9), (512, 4), (768, 130), (1200, 6), (1536, 9), (1000, 3), (2048, 2), (2049, 5), (5000, 3), (8192, 2), (10001, 2), (32768, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,n", DIMS)
def test_rms_norm_forward_backward(engine, dtype, dim, n):
    g = torch.Generator().manual_seed(dim)
    wide = torch.randn(n, dim + 3, generator=g).to(dtype)
    x, res = wide[:, 1: dim + 1], torch.randn(n, dim, generator=g).to(dtype)
    w, gy, gs = (torch.randn(s, generator=g).to(dtype) for s in ((dim,), (n, dim), (n, dim)))
    for residual, weight, gsum in ((None, None, None), (res, w, gs), (None, w, None), (res, None, gs)):
        c = lambda t: None if t is None else t.cuda()
        y, total, rstd = engine.rms_norm(wide.cuda()[:, 1: dim + 1], c(weight), c(residual), eps=1e-5)
        wy, wh, wr = R.rms_norm(x, weight, residual, float(np.float32(1e-5)))
        rel = (dim + 12) * R.U32
        _close(rstd, wr, rel * wr)
        # the sum h is rounded to 32 bits before it is scaled
        hm = x.double().abs() + (0 if residual is None else residual.double().abs())
        _close(y, wy, R.half(dtype, wy.abs()) + rel * (hm * wr[:, None] * (1 if weight is None else weight.double().abs())) * 1.01)
        if residual is not None:
            _close(total, wh, R.half(dtype, hm) + R.U32 * 1.01 * hm)
        # backward: h as stored
        h = total.double().cpu()
        dx, dw = engine.rms_norm_backward(gy.cuda(), total, rstd, c(weight), c(gsum))
        wd = torch.ones(dim, dtype=torch.float64) if weight is None else weight.double()
        r = rstd.double().cpu()[:, None]
        nx, gw = h * r, gy.double() * wd
        mean = (gw * nx).mean(1, keepdim=True)
        want = r * (gw - nx * mean) + (0 if gsum is None else gsum.double())
        bound = R.half(dtype, want.abs()) + R.U32 * (8 * (r * gw).abs() + (dim + 12) * (r * nx).abs() * (gw * nx).abs().mean(1, keepdim=True) +
                                                      (0 if gsum is None else 2 * gsum.double().abs()))
        _close(dx, want, bound * 1.01, "dx")
        if weight is None:
            assert dw is None
        else:
            _close(dw, (gy.double() * nx).sum(0), (n + 8) * R.U32 * (gy.double() * nx).abs().sum(0), "dw")
            dx2, dw2 = engine.rms_norm_backward(gy.cuda(), total, rstd, c(weight), c(gsum))
            assert torch.equal(dw, dw2) and torch.equal(dx, dx2)


def test_rms_norm_backward_many_rows(engine):
    """more rows than blocks: the weight's gradient over several rounds of every block"""
    g = torch.Generator().manual_seed(3)
    for n, dim in ((5003, 96), (700, 2100)):
        h, gy, w = torch.randn(n, dim, generator=g), torch.randn(n, dim, generator=g), torch.randn(dim, generator=g)
        _, _, rstd = engine.rms_norm(h.cuda(), w.cuda())
        _, dw = engine.rms_norm_backward(gy.cuda(), h.cuda(), rstd, w.cuda())
        t = gy.double() * h.double() * rstd.double().cpu()[:, None]
        _close(dw, t.sum(0), (n + 8) * R.U32 * t.abs().sum(0))


def test_rms_norm_gradient_against_differences(engine):
    g = torch.Generator().manual_seed(4)
    x, res, w, c = torch.randn(2, 6, generator=g), torch.randn(2, 6, generator=g), torch.randn(6, generator=g), torch.randn(2, 6, generator=g)
    f = lambda a, ww: (R.rms_norm(a, ww, res, 1e-6)[0] * c.double()).sum().item()
    y, total, rstd = engine.rms_norm(x.cuda(), w.cuda(), res.cuda())
    dx, dw = engine.rms_norm_backward(c.cuda(), total, rstd, w.cuda())
    e = 1e-5
    for i in range(2):
        for j in range(6):
            up, dn = x.double().clone(), x.double().clone()
            up[i, j] += e
            dn[i, j] -= e
            assert abs((f(up, w) - f(dn, w)) / (2 * e) - dx[i, j].item()) < 1e-5      # step^2 and 2^-24 of values below 30
    for j in range(6):
        up, dn = w.double().clone(), w.double().clone()
        up[j] += e
        dn[j] -= e
        assert abs((f(x, up) - f(x, dn)) / (2 * e) - dw[j].item()) < 1e-5


@pytest.mark.parametrize("kind,top", [("int8", 127), ("e4m3", 448)])
def test_q8_scale_of_products_above_32_bits(engine, kind, top):
    """h * weight leaves the range of float, its quotient by the row's norm and the largest code does not"""
    x = torch.zeros(2, 64)
    x[0, 3], x[1] = 4, 4
    w = torch.full((64,), 3e38)
    codes, scales, _ = engine.rms_norm_q8(x.cuda(), w.cuda(), eps=0.0, kind=kind)
    r = 1 / (x.double() ** 2).mean(1).sqrt()
    want = 4 * w[0].double() * r / top                           # rstd: a sum of 64 squares, root, quotient; two roundings here
    assert ((scales.double().cpu() - want).abs() <= want * 2.0 ** -24 * 16).all()
    assert (codes.float().cpu() == torch.where(x > 0, float(top), 0.0)).all()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,n", DIMS)
def test_rms_norm_q8(engine, kind, dtype, dim, n):
    """codes equal to exact arithmetic, ties included (bf16 rows tie often); scales to the norm's rounding"""
    g = torch.Generator().manual_seed(dim + 1)
    x, res, w = torch.randn(n, dim, generator=g).to(dtype), torch.randn(n, dim, generator=g).to(dtype), torch.randn(dim, generator=g).to(dtype)
    for residual, weight in ((None, None), (res, w), (None, w)):
        c = lambda t: None if t is None else t.cuda()
        codes, scales, total = engine.rms_norm_q8(x.cuda(), c(weight), c(residual), kind=kind)
        q, s = R.q8(x, weight, residual, float(np.float32(1e-6)), kind)
        assert torch.equal(codes.float().double().cpu(), q)
        _close(scales, s, (dim + 16) * R.U32 * s.abs())
        if residual is None:
            assert total is None
        else:
            assert torch.equal(total.cpu(), (x.float() + residual.float()).to(dtype))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_rms_norm_q8_special_rows(engine, kind):
    x = torch.randn(8, 100, generator=torch.Generator().manual_seed(9))
    x[1] = 0
    x[2, 50] = float("nan")
    x[3, 99] = float("inf")
    x[4] = 1e-30
    x[5] = 0
    x[5, 0] = -3
    x[6] *= 2.0 ** torch.arange(100) / 2.0 ** 60                  # most codes zero or subnormal
    codes, scales, _ = engine.rms_norm_q8(x.cuda(), kind=kind)
    q, s = R.q8(x, None, None, float(np.float32(1e-6)), kind)
    assert torch.equal(codes.float().double().cpu(), q)
    assert torch.isnan(scales[2:4]).all() and scales[1] == 0 and (codes[1:4].float() == 0).all()
    zero, s0, _ = engine.rms_norm_q8(x[1:2].cuda(), kind=kind, eps=0.0)
    assert (zero.float() == 0).all() and s0.item() == 0
    ok = [0, 1, 4, 5, 6, 7]
    _close(scales[ok], s[ok], 120 * R.U32 * s[ok].abs())


# ---------------------------------------------------------------------------------------------------- edges
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [1, 15, 16, 17, 31, 64, 65, 100, 128, 129, 255, 256, 257, 768, 1000, 1025, 2000])
def test_edge_cosines(engine, kind, dim):
    g = torch.Generator().manual_seed(dim)
    n, e = 40, 333
    v = torch.randn(n, dim, generator=g)
    v[3] = 0
    v[9] = v[8]
    rows = (v * 30).clamp(-127, 127).round().to(torch.int8) if kind == "int8" else (v * 30).to(torch.float8_e4m3fn)
    eu, ev = torch.randint(0, n + 2, (e,), generator=g).int(), torch.randint(0, n, (e,), generator=g).int()
    eu[0], ev[0] = 9, 8
    eu[1] = -1                                                   # 2^32 - 1 as an index: no such row
    got = engine.edge_cosines(rows.cuda(), eu.cuda(), ev.cuda())
    a = torch.zeros(n + 2, dim, dtype=torch.float64)
    a[:n] = rows.float().double()
    want = R.cosines(a[torch.where(eu < 0, torch.tensor(n), eu).long()], a[ev.long()])
    # int8: exact sums, three roundings; e4m3: dim terms each.  By Cauchy-Schwarz the magnitudes' sum is at most 1.
    _close(got, want, 6 * R.U32 if kind == "int8" else (2 * dim + 6) * R.U32)
    wide = torch.zeros(n, dim + 5, dtype=rows.dtype)
    wide.view(torch.int8)[:, 2: dim + 2] = rows.view(torch.int8)
    assert torch.equal(engine.edge_cosines(wide.cuda()[:, 2: dim + 2], eu.cuda(), ev.cuda()), got)
    assert engine.edge_cosines(rows.cuda(), eu[:0].cuda(), ev[:0].cuda()).numel() == 0
    assert (engine.edge_cosines(rows[:0].cuda(), eu.cuda(), ev.cuda()) == 0).all()       # no rows at all


@pytest.mark.parametrize("n,docs", [(0, 5), (1, 5), (2, 2), (63, 7), (65, 2 ** 32 - 1), (1025, 40), (4000, 3), (8191, 90), (8192, 70000), (8193, 300), (50001, 256), (100000, 2 ** 20), (30000, 2 ** 31)])
def test_sort_edges(engine, n, docs):
    """one block and many; an odd and an even number of passes; equal edges"""
    g = np.random.default_rng(n)
    u, v = (g.integers(0, docs, n).astype(np.uint32) for _ in range(2))
    eu, ev = engine.to_device(u), engine.to_device(v)
    engine.sort_edges(eu, ev, docs)
    order = np.lexsort((v, u))
    assert (eu.cpu().numpy().view(np.uint32) == u[order]).all() and (ev.cpu().numpy().view(np.uint32) == v[order]).all()


# ---------------------------------------------------------------------------------------------------- microscaled 4 bits
def _vectors(n, dim, g, spread=4.0):
    return torch.randn(n, dim, generator=g) * torch.exp2(torch.randint(0, int(spread) + 1, (n, (dim + 31) // 32), generator=g).float()).repeat_interleave(32, 1)[:, :dim]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,dim", [(1, 1), (1, 32), (5, 33), (31, 127), (32, 128), (33, 129), (70, 500), (3, 1024)])
def test_mx_quantize(engine, dtype, n, dim):
    g = torch.Generator().manual_seed(n + dim)
    x = _vectors(n, dim, g).to(dtype)
    x[0, : min(dim, 32)] = 0                                     # a block of zeros
    if dim > 64:
        x[n // 2, 32: 64] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9]).repeat(4).to(dtype)      # every midpoint, and beyond 6
        x[n - 1, 64] = float("inf")
        x[n - 1, 33] = float("nan")
    if dtype != torch.float16 and dim >= 32:                     # near and below the smallest normal number: the scale stops at 2^-127
        x[n - 1, :32] = (2.0 ** torch.linspace(-128, -123, 32)).to(dtype) * torch.tensor([1.0, -1.0]).repeat(16).to(dtype)
        x[n // 3, :32] = 2.0 ** -130
    m = engine.mx_quantize(x.cuda())
    codes, sb = R.mx_unpack(m.codes, m.scales, n, dim)
    want, wb = R.mx_codes(x)
    assert (sb[:n, : wb.shape[1]] == wb).all()
    assert (codes[:n, :dim] == want).all()
    assert (codes[n:] == 0).all() and (codes[:, dim:] == 0).all() and (sb[n:] == 127).all() and (sb[:, wb.shape[1]:] == 127).all()
    wide = torch.zeros(n, dim + 7, dtype=dtype)
    wide[:, 3: dim + 3] = x
    m2 = engine.mx_quantize(wide.cuda()[:, 3: dim + 3])
    assert torch.equal(m.codes, m2.codes) and torch.equal(m.scales, m2.scales)


SHAPES = [(1, 1, 1), (1, 1000, 300), (3, 33, 129), (32, 40000, 64), (33, 100, 200), (64, 31, 1500), (65, 1000, 257), (128, 70, 128), (129, 65, 96), (300, 520, 1000),
          (130, 40000, 130), (4100, 4200, 260), (100, 20000, 300), (1100, 1300, 520), (1500, 1600, 130), (2000, 2, 260), (2001, 3, 100), (70000, 3, 40), (33000, 1, 300), (30001, 64, 200),
          (40000, 33, 130)]


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,dim", SHAPES)
def test_mx_matmul(engine, out, m, n, dim):
    """streaming, split, groups of 128 rows, tiles; rows and columns that end inside a tile"""
    g = torch.Generator().manual_seed(m + n)
    a, b = _vectors(m, dim, g), _vectors(n, dim, g)
    qa, qb = engine.mx_quantize(a.cuda()), engine.mx_quantize(b.cuda())
    va = torch.from_numpy(R.mx_values(*R.mx_unpack(qa.codes, qa.scales, m, dim))[:m, :dim])
    vb = torch.from_numpy(R.mx_values(*R.mx_unpack(qb.codes, qb.scales, n, dim))[:n, :dim])
    got = engine.mx_matmul(qa, qb, dtype=out, alpha=0.75)
    want, mag = 0.75 * va @ vb.T, 0.75 * va.abs() @ vb.abs().T
    assert got.dtype == out
    _close(got, want, R.half(out, want.abs()) + (dim + 4) * R.U32 * mag)


def test_mx_matmul_nan_blocks_and_padding(engine):
    """a block without numbers reaches its own row of the product and no other"""
    g = torch.Generator().manual_seed(1)
    a, b = torch.randn(200, 160, generator=g), torch.randn(150, 160, generator=g)
    a[7, 40] = float("nan")
    b[149, 159] = float("inf")
    for rows in (200, 20):
        c = engine.mx_matmul(engine.mx_quantize(a[:rows].cuda()), engine.mx_quantize(b.cuda()))
        bad = torch.isnan(c).cpu()
        want = torch.zeros_like(bad)
        want[7], want[:, 149] = True, True
        assert torch.equal(bad, want) and torch.isfinite(c[~bad]).all()
    e = engine.mx_quantize(a[:0].cuda())
    assert engine.mx_matmul(e, engine.mx_quantize(b.cuda())).shape == (0, 150)
    assert engine.mx_matmul(engine.mx_quantize(b.cuda()), e).shape == (150, 0)


@pytest.mark.parametrize("n,dim", [(0, 64), (1, 64), (2, 100), (127, 300), (700, 256), (2999, 384), (6000, 200)])
def test_mx_pairs(engine, n, dim):
    """duplicates well above the threshold, unrelated rows well below: one tile and many, diagonal ones, ragged ends"""
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, dim, generator=g)
    if n > 1:
        k = max(1, n // 20)
        p = torch.randperm(n, generator=g)
        x[p[:k]] = x[p[k: 2 * k]] + 0.05 * torch.randn(k, dim, generator=g)
        x[p[0]] = 0                                              # a row of zeros pairs with nothing
        x[p[-1], 3] = float("nan")                                # nor does one with a NaN
    m = engine.mx_quantize(x.cuda())
    eu, ev = engine.mx_pairs(m, 0.9)
    v = np.nan_to_num(R.mx_values(*R.mx_unpack(m.codes, m.scales, n, dim))[:n, :dim], nan=0.0) if n else np.zeros((0, dim))
    if n > 1:
        v[p[-1].item()] = 0
    ln = np.sqrt((v * v).sum(1))
    c = (v @ v.T) / np.where(ln > 0, ln, np.inf)[:, None] / np.where(ln > 0, ln, np.inf)[None]
    assert n < 2 or np.abs(c[np.tril_indices(n, -1)] - 0.9).min() > 1e-4      # the data leaves no pair at the threshold
    wu, wv = np.nonzero(np.tril(c >= 0.9, -1))
    assert (eu.cpu().numpy() == wu).all() and (ev.cpu().numpy() == wv).all() and (n < 100 or len(wu) > 0)


@pytest.mark.parametrize("n", [2, 3, 64, 91, 92, 128, 129])
def test_mx_pairs_order(engine, n):
    """few enough pairs to come out in order, in the first pass or (91 rows: 4095 pairs) the second, and one more row"""
    m = engine.mx_quantize(torch.ones(n, 40).cuda())
    eu, ev = engine.mx_pairs(m, 0.5)
    wu, wv = np.nonzero(np.tril(np.ones((n, n)), -1))
    assert (eu.cpu().numpy() == wu).all() and (ev.cpu().numpy() == wv).all()


@pytest.mark.parametrize("power", [-120, -75, -61, -56, 56, 61, 75, 120])
def test_mx_pairs_long_and_short_rows(engine, power):
    """32 equal rows of `power` and 32 rows each along an axis of its own, where a product of lengths may leave the range of
    a 32-bit number: pairs among the equal rows only, and none where the length is outside [2^-60, 2^60]"""
    x = torch.zeros(96, 64)
    x[:32, :4] = 2.0 ** (power - 1)                              # length 2^power
    x[torch.arange(32, 64), torch.arange(4, 36)] = 2.0 ** power
    x[64:, 40:44] = 0.5                                          # length 1
    eu, ev = engine.mx_pairs(engine.mx_quantize(x.cuda()), 0.9)
    wu, wv = np.nonzero(np.tril(np.ones((32, 32)), -1))
    mid = wu + 64, wv + 64
    if -60 <= power <= 60:
        mid = np.concatenate([wu, mid[0]]), np.concatenate([wv, mid[1]])
    assert (eu.cpu().numpy() == mid[0]).all() and (ev.cpu().numpy() == mid[1]).all()


def test_mx_pairs_all_alike(engine):
    """every pair is near: more pairs than the first pass has room for, then more than allowed"""
    n = 500
    x = torch.randn(1, 96, generator=torch.Generator().manual_seed(2)).expand(n, -1).contiguous()
    m = engine.mx_quantize(x.cuda())
    eu, ev = engine.mx_pairs(m, 1.0 - 1e-6)
    wu, wv = np.nonzero(np.tril(np.ones((n, n)), -1))
    assert (eu.cpu().numpy() == wu).all() and (ev.cpu().numpy() == wv).all()
    with pytest.raises(MddError, match="more than max_pairs"):
        engine.mx_pairs(m, 0.9, max_pairs=100)
    with pytest.raises(MddError, match="more than max_pairs"):
        engine.mx_pairs(m, 0.9, max_pairs=0)
    assert all(t.numel() == 0 for t in engine.mx_pairs(engine.mx_quantize(x[:1].cuda()), 0.9, max_pairs=0))
