"""The document-vector methods make no autograd node: a tensor that requires a gradient is refused while gradients are recorded, not
answered with a result that has lost it."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from map_neo_amd.lib import MddError  # noqa: E402
from test_vectors_refusals import E  # noqa: E402

M, W, I32 = torch.zeros(4, 8), torch.zeros(8), torch.zeros(4, dtype=torch.int32)
G, GW = torch.zeros(4, 8, requires_grad=True), torch.zeros(8, requires_grad=True)
CALLS = {"table": lambda t: E.embed(t, I32), "grad": lambda t: E.embed_backward(t, I32, 5), "x": lambda t: E.rms_norm(t), "residual": lambda t: E.rms_norm(M, W, t),
         "total": lambda t: E.rms_norm_backward(M, t, W[:4]), "grad_sum": lambda t: E.rms_norm_backward(M, M, W[:4], W, t)}


@pytest.mark.parametrize("name", CALLS)
def test_matrices(name):
    with pytest.raises(MddError, match=f"{name} requires a gradient.*{name}.detach"):
        CALLS[name](G)


@pytest.mark.parametrize("call", [lambda: E.rms_norm(M, GW), lambda: E.rms_norm_q8(M, GW), lambda: E.rms_norm_backward(M, M, W[:4], GW)])
def test_weight(call):
    with pytest.raises(MddError, match="weight requires a gradient"):
        call()


def test_others():
    for call in (lambda: E.rms_norm_q8(G), lambda: E.mx_quantize(G)):
        with pytest.raises(MddError, match="x requires a gradient"):
            call()


@pytest.mark.gpu
def test_without_recording_it_is_answered(engine):
    table = torch.nn.Parameter(torch.randn(50, 16, generator=torch.Generator().manual_seed(0)).cuda())
    ids = torch.tensor([3, 49, -1, 7], device="cuda")
    with pytest.raises(MddError, match="table requires a gradient"):
        engine.embed(table, ids)
    with torch.no_grad():
        got = engine.embed(table, ids)
        assert not got.requires_grad
    assert torch.equal(got, engine.embed(table.detach(), ids)) and torch.equal(got[0], table[3].detach())
    x = torch.randn(3, 16, device="cuda", requires_grad=True)
    with torch.inference_mode():
        assert torch.equal(engine.rms_norm(x)[0], engine.rms_norm(x.detach())[0])


@pytest.mark.gpu
def test_in_a_node_of_the_callers(engine):
    """what the refusal asks for: the backward methods inside a torch.autograd.Function, against torch's own gradients"""

    class Mean(torch.autograd.Function):
        @staticmethod
        def forward(ctx, table, ids, offs, weight):
            h = engine.embed(table.detach(), ids, offs)
            y, total, rstd = engine.rms_norm(h, weight.detach())
            ctx.save_for_backward(ids, offs, total, rstd, weight)
            ctx.rows = table.shape[0]
            return y

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, dy):
            ids, offs, total, rstd, weight = ctx.saved_tensors
            dx, dw = engine.rms_norm_backward(dy.contiguous(), total, rstd, weight)
            return engine.embed_backward(dx, ids, ctx.rows, offs), None, None, dw

    g = torch.Generator().manual_seed(1)
    table, weight, dy = (torch.randn(s, generator=g) for s in ((40, 24), (24,), (3, 24)))
    ids, offs = torch.tensor([3, 3, 7, 39, -1, 12, 0]), torch.tensor([0, 3, 5, 7])
    t, w = table.cuda().requires_grad_(), weight.cuda().requires_grad_()
    (Mean.apply(t, ids.cuda(), offs.cuda(), w) * dy.cuda()).sum().backward()
    td, wd = table.double().requires_grad_(), weight.double().requires_grad_()
    h = torch.stack([td[[3, 3, 7]].mean(0), td[[39]].mean(0), td[[12, 0]].mean(0)])
    (h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * wd * dy.double()).sum().backward()
    # 60 roundings of 2^-24 of numbers below 20
    assert (t.grad.double().cpu() - td.grad).abs().max() < 60 * 2.0 ** -24 * 20 and (w.grad.double().cpu() - wd.grad).abs().max() < 60 * 2.0 ** -24 * 20
