"""GPU suite: the document-vector operators as a program uses them -- one after the other, captured into a graph and replayed,
on other streams, side by side, and past 2^32 elements.  Bounds as in test_gpu_vectors.py."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import vec_ref as R  # noqa: E402
from map_neo_amd.minhash import Engine  # noqa: E402

pytestmark = pytest.mark.gpu


def _within(got, want, tol):
    off = (got.double().cpu() - want).abs()
    assert got.shape == want.shape and bool((off <= tol).all()), f"{(off - tol).max().item():.3g} beyond the bound"


def _corpus(seed, docs=300, vocab=2000, dim=320):
    """token ids of documents of which every tenth repeats another's with a few tokens changed"""
    g = torch.Generator().manual_seed(seed)
    table = torch.randn(vocab, dim, generator=g)
    lens = torch.randint(40, 120, (docs,), generator=g)
    ids = [torch.randint(0, vocab, (int(n),), generator=g) for n in lens]
    for d in range(10, docs, 10):
        ids[d] = ids[d - 7].clone()
        ids[d][:2] = torch.randint(0, vocab, (2,), generator=g)
    offs = torch.zeros(docs + 1, dtype=torch.int64)
    offs[1:] = torch.cumsum(torch.tensor([len(i) for i in ids]), 0)
    return table, torch.cat(ids).int(), offs


def test_from_token_ids_to_near_duplicates(engine):
    """ids -> document vectors -> norm, 8 and 4 bits -> near pairs -> checked pairs -> labels"""
    table, ids, offs = _corpus(1)
    x = engine.embed(table.cuda(), ids.cuda(), offs.cuda())
    y, total, rstd = engine.rms_norm(x)
    assert total is x
    codes, scales, _ = engine.rms_norm_q8(x)
    # the 8-bit rows stand for the normalised ones: half a step of the largest / 127, and the norm's rounding
    _within(codes.float() * scales[:, None], y.double().cpu(), scales.double().cpu()[:, None] * 0.5 + 400 * R.U32 * y.double().cpu().abs())
    m = engine.mx_quantize(y)
    u, v = engine.mx_pairs(m, 0.85)
    cos = engine.edge_cosines(codes, u, v)
    keep = cos >= 0.92
    want = {(d, d - 7) for d in range(10, 300, 10)}
    assert set(zip(u[keep].tolist(), v[keep].tolist())) == want
    # the product of the 4-bit rows over their lengths is the cosine that the pairs were chosen by
    c = engine.mx_matmul(m, m)
    ln = c.diagonal().sqrt()
    near = torch.nonzero(torch.tril(c / ln[:, None] / ln[None] >= 0.85, -1))
    assert torch.equal(near[:, 0].int(), u) and torch.equal(near[:, 1].int(), v)
    labels = engine.components_init(300)
    engine.components_union(labels, u[keep], v[keep])
    engine.components_finish(labels)
    exp = np.arange(300)
    exp[10::10] -= 7
    assert (labels.cpu().numpy() == exp).all()


def test_a_table_is_fitted(engine):
    """two steps of gradient descent through embed and rms_norm: gradients against the same in 64 bits"""
    table, ids, offs = _corpus(2, docs=40, vocab=120, dim=48)
    target = torch.randn(40, 48, generator=torch.Generator().manual_seed(0))
    t = table.cuda()
    for _ in range(2):
        x = engine.embed(t, ids.cuda(), offs.cuda())
        y, total, rstd = engine.rms_norm(x)
        dx, _ = engine.rms_norm_backward(y - target.cuda(), total, rstd)
        grad = engine.embed_backward(dx, ids.cuda(), 120, offs.cuda())
        ref = t.double().cpu().requires_grad_(True)
        w = torch.zeros(40, 120, dtype=torch.float64)
        w.index_put_((torch.repeat_interleave(torch.arange(40), offs.diff()), ids.long()), torch.ones(len(ids), dtype=torch.float64), accumulate=True)
        h = w @ ref / offs.diff()[:, None]
        z = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6)
        (0.5 * ((z - target.double()) ** 2).sum()).backward()
        # norm's and sums' roundings: (120 + 2 * 48 + 40) * 2^-24 of magnitudes that stay below 300
        _within(grad, ref.grad, 300 * 256 * R.U32)
        t = t - 0.05 * grad


def test_captured_and_replayed():
    """every call that enqueues only, in one graph on the engine's own stream, replayed on changed inputs with eager work between"""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        eng = Engine(0)
        table, ids, offs = (t.cuda() for t in _corpus(3, docs=200, dim=264))
        res, w, g = torch.randn(200, 264, device="cuda"), torch.randn(264, device="cuda"), torch.randn(200, 264, device="cuda")
        eu, ev = (torch.randint(0, 200, (9000,), device="cuda", dtype=torch.int32) for _ in range(2))
        cnt = torch.zeros(1, dtype=torch.int64, device="cuda")
        pu, pv = torch.zeros(4096, dtype=torch.int32, device="cuda"), torch.zeros(4096, dtype=torch.int32, device="cuda")
        ws = torch.empty(eng.L.mdd_mx_pairs_ws_bytes(200), dtype=torch.uint8, device="cuda")

        def work():
            x = eng.embed(table, ids, offs)
            rows = eng.embed(table, ids, scale=3.0)
            y, total, rstd = eng.rms_norm(x, w, res)
            dx, dw = eng.rms_norm_backward(g, total, rstd, w, grad_sum=y)
            grad = eng.embed_backward(dx, ids, 2000, offs)
            codes, scales, _ = eng.rms_norm_q8(x, w, res)
            m = eng.mx_quantize(y)
            c = eng.mx_matmul(m, m)
            few = eng.mx_matmul(eng.mx_quantize(y[:5]), m)
            assert eng.L.mdd_mx_pairs(eng.ctx, m.codes.data_ptr(), m.scales.data_ptr(), 200, 264, 0.9, pu.data_ptr(), pv.data_ptr(), 4096, cnt.data_ptr(), ws.data_ptr(),
                                      ws.numel()) == 0
            cos = eng.edge_cosines(codes, eu, ev)
            su, sv = eng.sort_edges(eu.clone(), ev.clone(), 200)
            return [x, rows, y, total, rstd, dx, dw, grad, codes, scales, m.codes, m.scales, c, few, cnt, cos, su, sv]

        work()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            captured = work()
        for k in range(4):
            table.copy_(torch.randn_like(table) + 0.1 * k)
            ids.copy_(torch.randint(-1, 2001, ids.shape, device="cuda", dtype=torch.int32))
            g.normal_()
            eu.copy_(torch.randint(0, 201, eu.shape, device="cuda", dtype=torch.int32))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in captured]
            for a, b in zip(got, work()):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_two_graphs_share_nothing():
    """two captured graphs of the same engine, replayed in turn and interleaved"""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        eng = Engine(0)
        a, b = ([t.cuda() for t in _corpus(k, docs=100, dim=64)] for k in (4, 5))
        want = [(eng.embed(*x), eng.embed_backward(eng.embed(*x), x[1], 2000, x[2])) for x in (a, b)]
        torch.cuda.synchronize()
        graphs, outs = [], []
        for x in (a, b):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=s):
                y = eng.embed(*x)
                outs.append((y, eng.embed_backward(y, x[1], 2000, x[2])))
            graphs.append(gr)
        for order in ((0, 1), (1, 0), (0, 0, 1, 1)):
            for k in order:
                graphs[k].replay()
            torch.cuda.synchronize()
            for got, exp in zip(outs, want):
                assert torch.equal(got[0], exp[0]) and torch.equal(got[1], exp[1])


def test_under_another_stream_than_the_engines(engine):
    """inputs made and results used on the caller's stream, without a synchronisation in between"""
    table, ids, offs = (t.cuda() for t in _corpus(6, docs=400, dim=512))
    want = engine.embed(table * 2, ids, offs) + 1
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-4                                   # keeps the stream busy while the call is enqueued
        t2 = table * 2 + 0 * big[0, 0].nan_to_num()
        got = engine.embed(t2, ids, offs) + 1
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_two_engines_side_by_side():
    """two streams at once, each with its own engine and workspaces"""
    table, ids, offs = (t.cuda() for t in _corpus(7, docs=500, dim=256))
    streams, engines = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            engines.append(Engine(0))
    outs = []
    for _ in range(3):
        for s, e in zip(streams, engines):
            with torch.cuda.stream(s):
                x = e.embed(table, ids, offs)
                outs.append((x, e.embed_backward(x, ids, 2000, offs), e.mx_matmul(e.mx_quantize(x), e.mx_quantize(x))))
    torch.cuda.synchronize()
    for o in outs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(o, outs[0]))


def test_past_four_gibibytes(engine):
    """a table of 6 GB, vectors of 5 GB into 4 bits, a product of 4.9 * 10^9 numbers: offsets need 64 bits"""
    n, d = 3_000_000, 1024
    table = torch.empty(n, d, dtype=torch.float16, device="cuda")
    for k in range(0, n, 500_000):
        table[k: k + 500_000] = (torch.arange(k, k + 500_000, device="cuda") % 1009).to(torch.float16)[:, None]
    ids = torch.tensor([0, n - 1, 2_500_000, 2_097_152, 2_097_151, n], device="cuda")
    want = torch.tensor([k % 1009 for k in (0, n - 1, 2_500_000, 2_097_152, 2_097_151)] + [0]).half()
    assert torch.equal(engine.embed(table, ids)[:, 17].cpu(), want)
    offs = torch.tensor([0, 2, 6], device="cuda")
    assert torch.equal(engine.embed(table, ids, offs, mode="sum")[:, 1023].cpu(), torch.stack([want[:2].sum(), want[2:].sum()]))
    grad = engine.embed_backward(torch.ones(6, d, dtype=torch.float16, device="cuda"), ids, n, dtype=torch.float16)
    assert grad.sum(1, dtype=torch.float32).nonzero().flatten().cpu().tolist() == [0, 2_097_151, 2_097_152, 2_500_000, n - 1]
    del grad
    m = engine.mx_quantize(table[:2_700_000])
    tail = engine.mx_quantize(table[2_699_968:2_700_000])                # a row tile: the last one of m
    assert torch.equal(m.codes[-1], tail.codes[0]) and torch.equal(m.scales[-1], tail.scales[0])
    del m, table
    torch.cuda.empty_cache()
    x = torch.randn(70001, 32, device="cuda")
    q = engine.mx_quantize(x)
    c = engine.mx_matmul(q, q, dtype=torch.bfloat16)
    v = torch.from_numpy(R.mx_values(*R.mx_codes(x.cpu())))
    for r in (0, 30678, 61356, 61357, 70000):                            # 61356 * 70001 crosses 2^32
        want = v @ v[r]
        _within(c[r], want, R.half(torch.bfloat16, want.abs()) + 40 * R.U32 * (v.abs() @ v[r].abs()))


def test_current_device_and_errors_leave_no_trace(engine):
    table, ids, _ = _corpus(8, docs=5, dim=16)
    assert torch.cuda.current_device() == 0
    engine.embed(table.cuda(), ids.cuda())
    assert torch.cuda.current_device() == 0
    rc = engine.L.mdd_embed(engine.ctx, None, 0, 5, 16, 16, None, 4, 5, None, 0, 0, 1.0, None, None, 0)
    assert rc == -1 and b"out is NULL" in engine.L.mdd_last_error()
    engine.sync()
