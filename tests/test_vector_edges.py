"""dedup.vector_edges where 4 and 8 bits say little about a vector: the pairs it keeps have to be those of the vectors themselves.
On the CPU (the operators from their definitions) and, marked gpu, on the engine."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from map_neo_amd import dedup as D  # noqa: E402
from map_neo_amd.lib import MddError  # noqa: E402
from map_neo_amd.vectors import TooManyPairs  # noqa: E402
from test_vectors_path import VectorBackend  # noqa: E402


@pytest.fixture(params=["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])
def backend(request):
    return VectorBackend() if request.param == "cpu" else request.getfixturevalue("engine")


def _true_cosines(x):
    x = x.double()
    n = x / x.norm(dim=1, keepdim=True)
    c = n @ n.T
    return c[np.tril_indices(len(x), -1)].numpy(), np.tril_indices(len(x), -1)


def _pairs(backend, x, t):
    u, v = D.vector_edges(backend, x.to(backend.device), t)
    return list(zip(u.cpu().tolist(), v.cpu().tolist()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,big", [(1024, 130), (4096, 250), (4096, 260)])
def test_one_column_that_outweighs_the_others(backend, dim, big, dtype):
    """rows of +-1 but for a common column that sets the step of the 8-bit codes: the others become 0 or a whole step"""
    x = torch.randint(0, 2, (8, dim), generator=torch.Generator().manual_seed(0)).float() * 2 - 1
    x[:, 0] = big
    x = x.to(dtype)
    c, (u, v) = _true_cosines(x)
    assert c.max() < 0.97 and c.min() > 0.9
    assert _pairs(backend, x, 0.98) == []
    assert _pairs(backend, x, c.min() - 0.005) == list(zip(u, v))
    cut = np.sort(c)[13:15].mean()                               # between two pairs
    assert np.abs(c - cut).min() > 1e-9 and 0 < (c > cut).sum() < 28
    assert _pairs(backend, x, cut) == list(zip(u[c > cut], v[c > cut]))


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_pairs_on_both_sides_of_the_threshold(backend, dtype, many):
    """cosines closer together than 8 bits can tell: 0.9 +- 10^-3 .. 10^-5, evenly sized columns; beside few other pairs, and
    beside a group of equal rows (more pairs than rows), one of them above and one below the threshold to all others"""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(60, 512, generator=g, dtype=torch.float64)
    x /= x.norm(dim=1, keepdim=True)
    for k in range(30):
        c = 0.9 + (-1) ** k * 10.0 ** (-3 - 2 * k / 29)
        e = torch.randn(512, generator=g, dtype=torch.float64)
        e -= (e @ x[k]) * x[k]
        x[30 + k] = c * x[k] + np.sqrt(1 - c * c) * e / e.norm()
    if many:
        y = x[:1].repeat(20, 1)
        y[3], y[4] = x[30 + 4], x[30 + 5]
        x = torch.cat([y, x])
    x = (x * 3.7).to(dtype)
    c, (u, v) = _true_cosines(x)
    assert np.abs(c - 0.9).min() > 1e-9 and ((c >= 0.9).sum() > len(x)) == many
    assert _pairs(backend, x, 0.9) == list(zip(u[c >= 0.9], v[c >= 0.9]))


def _columns(kind, dim, g):
    scale = torch.ones(dim, dtype=torch.float64)
    if kind == "lognormal":
        scale = torch.randn(dim, generator=g, dtype=torch.float64).exp()
    elif kind == "one in 32":
        scale[::32] = 20
    elif kind == "first":
        scale[0] = dim ** 0.5
    return scale


@pytest.mark.parametrize("t", [0.8, 0.9, 0.95])
@pytest.mark.parametrize("dim,kind", [(2, "even"), (4, "even"), (16, "even"), (32, "even"), (64, "one in 32"), (64, "lognormal"), (256, "lognormal"),
                                      (256, "one in 32"), (768, "one in 32"), (768, "first"), (512, "even")])
def test_screen_keeps_pairs_at_the_threshold(dim, kind, t):
    """the 4-bit cosines of pairs 0.002 above the threshold, noise like the rows or alike in all columns, against the margin that is
    measured on other rows of that kind.  Less than one in a thousand may fall below it: of n pairs at most n / 1000 + 4 sqrt(n / 1000)"""
    n = 4000 if dim > 256 else 12000
    g = torch.Generator().manual_seed(dim)
    scale = _columns(kind, dim, g)
    draw = lambda k: torch.randn(k, dim, generator=g, dtype=torch.float64) * scale
    margin = D.screen_margin(draw(3000).float(), t)
    assert D.SCREEN_MARGIN <= margin < 0.3
    be, x = VectorBackend(), draw(n)
    x /= x.norm(dim=1, keepdim=True)
    missed = 0
    for z in (draw(n // 2), torch.randn(n - n // 2, dim, generator=g, dtype=torch.float64)):
        o = x[:len(z)] if missed == 0 else x[-len(z):]
        z -= (z * o).sum(1, keepdim=True) * o
        z /= z.norm(dim=1, keepdim=True)
        y = (t + 0.002) * o + np.sqrt(1 - (t + 0.002) ** 2) * z
        a, b = be.mx_quantize(o.float()), be.mx_quantize(y.float())
        missed += int(((a * b).sum(1) / (a.norm(dim=1) * b.norm(dim=1)) < t - margin).sum())
    assert missed <= n / 1000 + 4 * (n / 1000) ** 0.5


@pytest.mark.parametrize("dim,kind", [(4, "even"), (16, "even"), (256, "one in 32"), (768, "first")])
def test_narrow_and_uneven_vectors(backend, dim, kind):
    """all pairs at 0.8, those just above it included: 300 planted ones at 0.8 + 10^-3"""
    g = torch.Generator().manual_seed(dim + 1)
    x = torch.randn(600, dim, generator=g, dtype=torch.float64) * _columns(kind, dim, g)
    x /= x.norm(dim=1, keepdim=True)
    z = x[torch.randperm(600, generator=g)[:300]]
    z = torch.where((z - x[:300]).abs().amax(1, keepdim=True) == 0, x[300:], z)
    z = z - (z * x[:300]).sum(1, keepdim=True) * x[:300]
    x[300:] = 0.801 * x[:300] + np.sqrt(1 - 0.801 ** 2) * z / z.norm(dim=1, keepdim=True)
    x = x.float()
    c, (u, v) = _true_cosines(x)
    assert np.abs(c - 0.8).min() > 1e-9
    got, want = set(_pairs(backend, x, 0.8)), set(zip(u[c >= 0.8].tolist(), v[c >= 0.8].tolist()))
    assert got <= want and {(300 + k, k) for k in range(300)} <= want
    assert len(want - got) <= len(want) / 1000
    narrow = D.vector_edges(backend, x.to(backend.device), 0.8, margin=0.05)[0].numel()
    assert len(want) - narrow > 10                               # what a fixed margin of 0.05 misses


def test_four_bits_are_the_operators():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(50, 100, generator=g) * torch.randn(100, generator=g).exp()
    x[3, :32], x[4, 40], x[6, 96:] = 0, 2.0 ** -100, 2.0 ** -90
    x[5, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9])
    assert torch.equal(D._four_bits(x)[:, :100].double(), VectorBackend().mx_quantize(x))
    x[7, :32] = 2.0 ** -140
    assert D._four_bits(x).isfinite().all()
    x[8, 50], x[9, 7] = float("inf"), float("nan")
    assert 0.05 <= D.screen_margin(x, 0.9) < 0.3
    assert D.screen_margin(torch.zeros(5, 8), 0.9) == D.screen_margin(x[:1], 0.9) == D.SCREEN_MARGIN


# ------------------------------------------------------------------------------------------------ more pairs or rows than a search takes
def _limited(backend, monkeypatch, pairs=None, rows=None):
    """the backend with a search that returns at most `pairs` pairs; ranges of at most `rows` rows"""
    if rows is not None:
        monkeypatch.setattr(D, "MAX_PAIR_ROWS", rows)
    calls, search = [], backend.mx_pairs

    def limited(m, t):
        calls.append(m)
        if isinstance(backend, VectorBackend):
            u, v = search(m, t)
            if pairs is not None and u.numel() > pairs:
                raise TooManyPairs(u.numel(), pairs, t)
            return u, v
        return search(m, t) if pairs is None else search(m, t, max_pairs=pairs)

    monkeypatch.setattr(backend, "mx_pairs", limited, raising=False)
    return calls


def _groups(n, dim, groups, noise, g):
    """random rows; the rows of each group are one vector, but for noise"""
    x = torch.randn(n, dim, generator=g)
    for rows in groups:
        x[rows] = x[rows[0]] + noise * torch.randn(len(rows), dim, generator=g)
    return x


@pytest.mark.parametrize("rows,pairs", [(64, None), (33, None), (None, 40), (50, 40), (2, None), (3, 1)])
def test_edges_do_not_depend_on_the_search(backend, monkeypatch, rows, pairs):
    """in ranges of few rows, and of few pairs: the same edges in the same order"""
    g = torch.Generator().manual_seed(8)
    n = 21 if rows in (2, 3) else 150
    p = torch.randperm(n, generator=g).tolist()
    x = _groups(n, 256, [p[:n // 10], p[n // 5: n // 5 + 2], p[n // 2: n // 2 + 7]], 0.05, g)
    x[p[0]] = 0
    want = _pairs(backend, x, 0.95)
    assert len(want) > 20 and want == sorted(want)
    calls = _limited(backend, monkeypatch, pairs, rows)
    assert _pairs(backend, x, 0.95) == want and len(calls) > 3
    with pytest.raises(TooManyPairs, match="max_pairs=20"):
        D.vector_edges(backend, x.to(backend.device), 0.95, max_pairs=20)


@pytest.mark.parametrize("rows,pairs", [(None, 500), (100, None), (None, 50), (1000, 10 ** 9)])
def test_clusters_of_many_alike_vectors(backend, monkeypatch, rows, pairs):
    """200 equal rows (19900 pairs), 60 nearly equal ones, a row near to the equal ones; rows of zeros and of NaN, which are as
    equal as can be and pair with nothing; a shingle duplicate"""
    g = torch.Generator().manual_seed(9)
    n = 400
    p = torch.randperm(n, generator=g).tolist()
    same, alike, zero, nan = sorted(p[:200]), sorted(p[200:260]), p[260:280], p[280:300]
    x = _groups(n, 128, [same], 0.0, g)
    x[alike] = x[alike[0]] + 0.02 * torch.randn(60, 128, generator=g)
    x[p[300]] = x[same[0]] + 0.02 * torch.randn(128, generator=g)
    x[zero], x[nan] = 0, float("nan")
    sig = np.random.default_rng(0).integers(0, 2 ** 32, (n, 128), dtype=np.uint64).astype(np.uint32)
    sig[p[302]] = sig[p[301]]
    want = np.arange(n)
    for c in (same + [p[300]], alike, [p[301], p[302]]):
        want[c] = min(c)
    calls = _limited(backend, monkeypatch, pairs, rows)
    out = D.cluster_local(backend, backend.to_device(sig), vectors=x.to(backend.device), min_cosine=0.95)
    assert (out["labels"].cpu().numpy() == want).all() and (len(calls) == 1) == (pairs == 10 ** 9)
    assert out["removed"].cpu().numpy().astype(bool).tolist() == (want != np.arange(n)).tolist()
    # the edges that come back join the same components
    labels = backend.components_init(n)
    backend.components_union(labels, out["edge_u"], out["edge_v"])
    backend.components_finish(labels)
    assert (labels.cpu().numpy() == want).all()
    if len(calls) > 1:
        assert out["edge_u"].numel() == (want != np.arange(n)).sum()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_first_equal_row(dtype):
    x = torch.randn(9, 40, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[4], x[8], x[5] = x[2], x[2], x[3]
    x[6:8] = 0
    x[5, 39] += 1                                                # all but equal
    assert D._first_equal(x).tolist() == [0, 1, 2, 3, 2, 5, 6, 7, 2]
    assert D._first_equal(x[:, ::2].contiguous()[:, 1:]).tolist() == [0, 1, 2, 3, 2, 3, 6, 7, 2]
    assert D._first_equal(x[:0]).tolist() == []


def test_token_ids_in_several_lookups(monkeypatch, tmp_path):
    """more ids than one lookup takes: whole rows at a time, empty ones among them; a row that alone is too long is refused"""
    from map_neo_amd.cli import dedup as stage
    rng = np.random.default_rng(3)
    table, lens = rng.standard_normal((50, 12)).astype(np.float32), [3, 0, 7, 9, 0, 0, 1, 4, 9, 0]
    ids = rng.integers(0, 50, sum(lens) + 5).astype(np.int32)
    offs = np.concatenate([[2], 2 + np.cumsum(lens)]).astype(np.int64)
    for name, a in (("t", table), ("i", ids), ("o", offs)):
        np.save(tmp_path / (name + ".npy"), a)
    args = stage.build_parser().parse_args(["--input_dir", "x", "--output_dir", "y", "--min_cosine", "0.9", "--embedding_table", str(tmp_path / "t.npy"),
                                            "--token_ids", str(tmp_path / "i.npy"), "--token_offsets", str(tmp_path / "o.npy")])
    rows = np.array([0, 1, 3, 7, 8, 9])
    want = stage.document_vectors(VectorBackend(), args, rows, 10)
    assert want.shape == (6, 12) and (want[1] == 0).all() and (want[2] != 0).any()
    for limit in (9, 10, 12, 33):
        monkeypatch.setattr(stage, "MAX_IDS", limit)
        assert torch.equal(stage.document_vectors(VectorBackend(), args, rows, 10), want)
    monkeypatch.setattr(stage, "MAX_IDS", 8)
    with pytest.raises(SystemExit, match="row 3 has 9 token ids"):
        stage.document_vectors(VectorBackend(), args, rows, 10)


@pytest.mark.gpu
def test_more_rows_than_one_search_takes(engine):
    """2^22 + 5000 documents: pairs within the first half, within the second and across, and 30000 equal rows (4.5 * 10^8 pairs)"""
    n, dim = (1 << 22) + 5000, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(n, dim, device="cuda", generator=g)
    p = torch.randperm(n, device="cuda", generator=g)[:40000]
    a, b = p[:4000], p[4000: 8000]
    x[b] = x[a] + 0.05 * torch.randn(4000, dim, device="cuda", generator=g)
    x[p[8000: 38000]] = x[p[8000]].clone()
    labels = engine.components_init(n)
    D._join_near(engine, labels, x.half(), 0.97)
    engine.components_finish(labels)
    want = torch.arange(n, device="cuda")
    want[torch.maximum(a, b)] = torch.minimum(a, b)
    want[p[8000: 38000]] = p[8000: 38000].min()
    assert torch.equal(labels.long(), want)


@pytest.mark.gpu
def test_too_many_pairs_says_how_many(engine):
    m = engine.mx_quantize(torch.ones(300, 40).cuda())
    with pytest.raises(TooManyPairs, match="44850 pairs reach 0.5: more than max_pairs=1000") as e:
        engine.mx_pairs(m, 0.5, max_pairs=1000)
    assert (e.value.count, e.value.limit) == (44850, 1000)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [None, 3])
def test_refusals_of_the_engine(engine, monkeypatch, rows):
    """the same for one search and for more rows than one takes: before anything is measured or searched"""
    if rows:
        monkeypatch.setattr(D, "MAX_PAIR_ROWS", rows)
    x = torch.randn(20, 16, device="cuda")
    sig = torch.zeros(20, 128, dtype=torch.int32, device="cuda")
    for bad, what in ((x.double(), "type torch.float64"), (x[0], "matrix"), (x[:, :0], "0 columns"), (x.t().contiguous().t(), "unit stride"), (x.cpu(), "tensor on"),
                      (x.to(torch.int32), "type torch.int32"), (x.clone().requires_grad_(), "requires a gradient")):
        with pytest.raises(MddError, match=what):
            D.vector_edges(engine, bad, 0.9)
        if bad.shape[0] == 20:
            with pytest.raises(MddError, match=what):
                D.cluster_local(engine, sig, vectors=bad, min_cosine=0.9)
    assert D.vector_edges(engine, x[:1], 0.9)[0].numel() == 0 and D.vector_edges(engine, x[:, :1], 0.9)[0].numel() > 20


@pytest.mark.gpu
def test_many_pairs_of_narrow_vectors(engine):
    """4 columns: (a - sin a cos a) / pi = 5.2 % of all pairs, a = acos(0.8), reach 0.8, 936000 of 18 million, far more candidates than rows; all pairs but those next to the threshold, in 64 bits"""
    x = torch.randn(6000, 4, generator=torch.Generator().manual_seed(3)).half()
    c, (u, v) = _true_cosines(x)
    got = torch.zeros(6000, 6000, dtype=torch.bool)
    eu, ev = D.vector_edges(engine, x.cuda(), 0.8)
    got[eu.cpu().long(), ev.cpu().long()] = True
    got = got.numpy()[u, v]
    assert not got[c < 0.8 - 1e-9].any() and eu.numel() == got.sum() > 900000
    assert (~got[c > 0.8 + 1e-9]).sum() <= (c > 0.8).sum() / 10 ** 5
