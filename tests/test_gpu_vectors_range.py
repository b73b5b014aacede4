"""GPU suite: the document-vector operators at the ends of the 32-bit range.  Bounds as in test_gpu_vectors.py."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import vec_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu


def _close(got, want, tol, what=""):
    got = got.double().cpu()
    off = (got - want).abs()
    worst = (off - tol).max().item()
    assert got.shape == want.shape and worst <= 0, f"{what}: off by {off.max().item():.3g}, {worst:.3g} beyond the bound"


# sizes of rows: with eps = 0 the squares of all but those near 1 leave the 32-bit numbers or their normal range
SIZES = [1.0, 1e-17, 1e-19, 1e-21, 1.0, 1e-25, 1e-30, 3e-38, 2e-42, 1e18, 1e19, 1e25, 3e37, 1.0]


def _rows(dim, dtype, g):
    x = torch.randn(len(SIZES), dim, generator=g, dtype=torch.float64) * torch.tensor(SIZES, dtype=torch.float64)[:, None]
    return x.to(dtype)


@pytest.mark.parametrize("eps", [0.0, 1e-35, 1e-6])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [1, 5, 100, 129, 384, 500, 768, 1000, 1300, 2048, 3001, 5000, 10001, 20000])
def test_norms_of_very_small_and_large_rows(engine, dim, dtype, eps):
    g = torch.Generator().manual_seed(dim)
    x, res = _rows(dim, dtype, g), _rows(dim, dtype, g)
    w, gy = torch.randn(dim, generator=g).to(dtype), torch.randn(len(SIZES), dim, generator=g).to(dtype)
    e = float(np.float32(eps))
    for residual, weight in ((None, None), (res, w)):
        c = lambda t: None if t is None else t.cuda()
        h = x.float() if residual is None else x.float() + residual.float()      # h is a 32-bit number
        wy, _, wr = R.rms_norm(h, weight, None, e)
        live = h.abs().amax(1) > 0                                # (a row may round to zeros, whose r without eps is infinite)
        y, total, rstd = engine.rms_norm(x.cuda(), c(weight), c(residual), eps=eps)
        rel = (dim + 12) * R.U32
        fits = live & (wr < 2.0 ** 127)
        _close(rstd[fits], wr[fits], rel * wr[fits] + 2.0 ** -149, "rstd")
        assert torch.isinf(rstd.cpu()[live & (wr > 2.0 ** 129)]).all()
        _close(y[live], wy[live], (R.half(dtype, wy.abs()) + 1.01 * rel * wy.abs())[live], "y")
        codes, scales, _ = engine.rms_norm_q8(x.cuda(), c(weight), c(residual), eps=eps)
        q, s = R.q8(x, weight, residual, e, "int8")
        assert torch.equal(codes.float().double().cpu(), q)
        _close(scales[live], s[live], (dim + 16) * R.U32 * s[live].abs() + 2.0 ** -149, "scales")
        # backward, from what the forward pass stored, where a gradient of about r is a number of the type
        ok = [k for k in range(len(SIZES)) if fits[k] and wr[k] < 1e34 and wr[k] > 1e-37]
        r, hh = rstd.double().cpu()[ok][:, None], total.double().cpu()[ok]
        dx, dw = engine.rms_norm_backward(gy.cuda()[ok], total[ok], rstd[ok], c(weight))
        nx, gw = hh * r, gy.double()[ok] * (1 if weight is None else weight.double())
        want = r * (gw - nx * (gw * nx).mean(1, keepdim=True))
        bound = R.half(dtype, want.abs()) + 1.01 * R.U32 * (8 * (r * gw).abs() + (dim + 12) * (r * nx).abs() * (gw * nx).abs().mean(1, keepdim=True))
        _close(dx, want, bound, "dx")


def test_norms_of_zeros_infinities_and_nan(engine):
    """what they gave before: a row of zeros y = 0 * inf without eps and 0 with it; an infinity or a NaN reaches its row and no other"""
    x = torch.randn(6, 200, generator=torch.Generator().manual_seed(1)) * 1e-25
    x[1] = 0
    x[2, 150], x[3, 7] = float("nan"), float("inf")
    y, _, rstd = engine.rms_norm(x.cuda(), eps=0.0)
    assert torch.isnan(y[1]).all() and torch.isinf(rstd[1]) and torch.isnan(y[2]).all() and torch.isnan(rstd[2])
    assert rstd[3] == 0 and torch.isnan(y[3, 7]) and (y[3, :7] == 0).all()
    ok = [0, 4, 5]
    _close(y[ok], R.rms_norm(x, None, None, 0.0)[0][ok], 220 * R.U32 * R.rms_norm(x, None, None, 0.0)[0][ok].abs())
    assert (engine.rms_norm(x[1:2].cuda())[0] == 0).all()
    codes, scales, _ = engine.rms_norm_q8(x.cuda(), eps=0.0)
    assert scales[1] == 0 and torch.isnan(scales[2:4]).all() and (codes[1:4] == 0).all()


# ------------------------------------------------------------------------------------------------ pairs next to the threshold
@pytest.mark.parametrize("dim", [96, 4096, 8192, 32768])
@pytest.mark.parametrize("n", [2, 33, 300])
def test_equal_rows_of_any_width(engine, n, dim):
    """one large block and many small ones: sums of squares depend on their order, and equal rows have to be near at 1 - 2^-20 anyhow"""
    x = torch.zeros(1, dim)
    x[0, 0] = 4096
    x[0, 32::32], x[0, 33::32] = 0.5, 0.5
    eu, ev = engine.mx_pairs(engine.mx_quantize(x.expand(n, -1).contiguous().cuda()), 1 - 2.0 ** -20)
    wu, wv = np.nonzero(np.tril(np.ones((n, n)), -1))
    assert eu.tolist() == wu.tolist() and ev.tolist() == wv.tolist()           # (arrays of 0 and 1 entries would compare as equal)


@pytest.mark.parametrize("dim", [128, 2048, 32768])
def test_products_and_lengths_within_the_bound(engine, dim):
    """rows whose sums lose the most: a block of 2^12 and small ones of one sign behind it.  The cosine by which a pair is chosen, from the
    same sums, against 64 bits: within (dim / 16 + 16) * 2^-24, as mdd.h says"""
    g = torch.Generator().manual_seed(dim)
    x = torch.rand(64, dim, generator=g) * 0.7 + 0.1
    x[:, 0] = torch.randint(2 ** 10, 2 ** 13, (64,), generator=g).float()
    x[::2, 32:] *= torch.exp2(torch.randint(0, 3, (32, (dim - 32) // 32), generator=g).float()).repeat_interleave(32, 1)
    m = engine.mx_quantize(x.cuda())
    v = torch.from_numpy(R.mx_values(*R.mx_unpack(m.codes, m.scales, 64, dim))[:64, :dim])
    ln = v.norm(dim=1)
    want = (v @ v.T) / ln[:, None] / ln[None]
    c = engine.mx_matmul(m, m).double().cpu()
    got = c / c.diagonal().sqrt()[:, None] / c.diagonal().sqrt()[None]
    bound = (dim / 16 + 16) * 2.0 ** -24
    assert ((got - want).abs() <= bound).all()
    for t in (0.3, 0.6, 0.9, 0.99, 0.9999):
        eu, ev = engine.mx_pairs(m, t)
        found = torch.zeros(64, 64, dtype=torch.bool)
        found[eu.cpu().long(), ev.cpu().long()] = True
        low = torch.ones(64, 64, dtype=torch.bool).tril(-1)
        assert found[low & (want > t + bound)].all() and not found[want < t - bound].any()


# ------------------------------------------------------------------------------------------------ subnormal numbers in sums
@pytest.mark.parametrize("dtype,least", [(torch.bfloat16, -133), (torch.float16, -24), (torch.float32, -149)])
@pytest.mark.parametrize("dim,lens", [(8, [1, 2, 3, 16, 0, 65]), (256, [7, 64, 100, 3000]), (520, [9, 40, 128])])
def test_sums_of_subnormal_rows(engine, dim, lens, dtype, least):
    """rows of a few of the type's smallest steps, alone and beside the smallest normal numbers: lookups, sums and gradients keep them"""
    g = torch.Generator().manual_seed(dim)
    step = 2.0 ** least
    table = (torch.randint(-7, 8, (40, dim), generator=g).double() * step).to(dtype)
    table[30:] = (torch.randn(10, dim, generator=g).double() * step * 2 ** 10).to(dtype)
    assert (table.double() % step == 0).all() and (table[:30] != 0).any()
    ids = torch.randint(0, 40, (sum(lens),), generator=g, dtype=torch.int32)
    ids[: lens[0] + lens[1]] %= 30                               # documents of such rows only
    offs = torch.tensor([0] + lens).cumsum(0)
    assert torch.equal(engine.embed(table.cuda(), ids.cuda()).cpu(), table[ids.long()])
    for mode in ("sum", "mean"):
        want, mag, cnt = R.embed(table, ids, offs, 1.0, mode)
        got = engine.embed(table.cuda(), ids.cuda(), offs.cuda(), mode=mode)
        # sums in 32 bits of whole steps of 2^-149 and above; a mean is rounded once more there
        _close(got, want, R.half(dtype, want.abs()) + (cnt[:, None].double() + 4) * R.U32 * mag + 2.0 ** -149, mode)
        assert (got[0] != 0).any()
    grad = table[torch.randint(0, 40, (len(lens),), generator=g)]
    want, mag, cnt = R.embed_backward(grad, ids, 40, offs, 1.0, "sum")
    _close(engine.embed_backward(grad.cuda(), ids.cuda(), 40, offs.cuda(), mode="sum"), want, (cnt + 4) * R.U32 * mag, "gradient")
    rows = table[torch.randint(0, 40, (sum(lens),), generator=g)]
    want, mag, cnt = R.embed_backward(rows, ids, 40, None, 1.0, "sum")
    for out in {torch.float32, dtype}:
        _close(engine.embed_backward(rows.cuda(), ids.cuda(), 40, dtype=out), want, R.half(out, want.abs()) + (cnt + 4) * R.U32 * mag, "gradient of rows")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_sums_with_infinities_and_large_numbers(engine, dtype):
    """infinities and NaN by column, as in 64 bits; the largest finite numbers of either sign beside each other"""
    big = torch.finfo(dtype).max
    table = torch.zeros(6, 16, dtype=dtype)
    table[0, 0], table[1, 0], table[2, 1], table[3, 1], table[4, 2] = float("inf"), -float("inf"), float("inf"), 3.0, float("nan")
    table[0, 3], table[1, 3], table[0, 4], table[1, 4], table[5] = big, -big, big, 0, 1
    ids = torch.arange(6, device="cuda")
    for n in (2, 4, 6):
        got = engine.embed(table.cuda(), ids[:n], torch.tensor([0, n], device="cuda"), mode="sum").double().cpu()
        want = table[:n].double().sum(0, keepdim=True)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~want.isnan()].isinf(), want[~want.isnan()].isinf())
        fin = want.isfinite()
        # the result is rounded to the type: 65504 + 1 lies between 65504 and 65536, the next in float16, and is off by 1 <= half a step, 16
        assert ((got - want)[fin].abs() <= 2.0 ** -24 * 6 * big + R.half(dtype, want[fin].abs())).all() and (got[:, 5:] == want[:, 5:]).all()


# ------------------------------------------------------------------------------------------------ 8-bit codes next to a midpoint
@pytest.mark.parametrize("kind,top", [("int8", 127), ("e4m3", 448)])
@pytest.mark.parametrize("dtype,gap,lost", [(torch.bfloat16, -36, -60), (torch.float16, -24, None), (torch.float32, -28, -60)])
def test_codes_of_sums_of_numbers_far_apart(engine, dtype, gap, lost, kind, top):
    """a residual that lifts or lowers a midpoint by 2^gap decides it; one below the 64 bits that h is held in does not (the tie
    goes to the even code), as mdd.h says"""
    mids = [2.5, 3.5, -2.5, -7.5, 0.5] if kind == "int8" else [17.0, 19.0, -17.0, -23.0, 17.0]
    up = [3, 4, -3, -8, 1] if kind == "int8" else [18, 20, -18, -24, 18]
    down = [2, 3, -2, -7, 0] if kind == "int8" else [16, 18, -16, -22, 16]
    even = [2, 4, -2, -8, 0] if kind == "int8" else [16, 20, -16, -24, 16]
    x = torch.tensor([[top] + mids]).to(dtype).cuda()
    sign = torch.tensor([[0] + mids]).sign()
    for power, want in ((gap, up), (gap, down), (lost, even)):
        if power is None:
            continue
        res = (sign * 2.0 ** power * (-1 if want is down else 1)).to(dtype)
        codes, _, _ = engine.rms_norm_q8(x, None, res.cuda(), kind=kind)
        assert codes.float().cpu().tolist() == [[top] + want]
