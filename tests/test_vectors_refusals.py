"""CPU suite: what the document-vector entry points refuse.  Every check of arguments comes before the first HIP call, so a
zeroed block of memory may stand for the context and made-up addresses for buffers: nothing is dereferenced."""
import ctypes as C
import os
import re
import shutil
import subprocess
from types import SimpleNamespace

import pytest
import torch

from map_neo_amd import lib as mlib
from map_neo_amd import vectors as V

L = mlib.load()
CTX = C.create_string_buffer(4096)
P, ODD, BIG = 1 << 20, (1 << 20) + 1, 1 << 40
F32, BF16, I8 = 0, 1, 3


def _refused(rc, needle):
    assert rc == -1, rc
    assert needle in L.mdd_last_error().decode(), L.mdd_last_error()


def _call(fn, defaults, **change):
    args = dict(defaults)
    args.update(change)
    return getattr(L, fn)(*args.values())


EMBED = dict(ctx=CTX, table=P, type=F32, n_rows=10, stride=64, dim=64, ids=P, id_bytes=4, n_ids=100000, offsets=P, n_docs=3, mean=1, scale=1.0, out=P,
             ws=P, ws_bytes=BIG)


@pytest.mark.parametrize("change,needle", [
    (dict(ctx=None), "ctx is NULL"), (dict(dim=0), "dim=0"), (dict(dim=32769), "dim=32769"), (dict(type=3), "element type"), (dict(id_bytes=2), "id_bytes"),
    (dict(n_ids=2 ** 31), "2^31"), (dict(n_rows=2 ** 32 - 1), "2^32"), (dict(out=None), "out is NULL"), (dict(out=ODD), "aligned"), (dict(ids=None), "ids"),
    (dict(ids=P + 2), "ids"), (dict(table=None), "table is NULL"), (dict(table=ODD), "aligned"), (dict(stride=63), "stride"), (dict(stride=2 ** 30), "2^30"), (dict(ws=None), "workspace"),
    (dict(ws=P + 128), "workspace"), (dict(ws_bytes=100), "workspace")])
def test_embed(change, needle):
    _refused(_call("mdd_embed", EMBED, **change), needle)


BACK = dict(ctx=CTX, grad=P, type=BF16, stride=64, dim=64, ids=P, id_bytes=8, n_ids=1000, offsets=P, n_docs=3, mean=1, scale=1.0, out=P, out_type=F32, n_rows=10,
            ws=P, ws_bytes=BIG)


@pytest.mark.parametrize("change,needle", [
    (dict(ctx=None), "ctx is NULL"), (dict(dim=0), "dim=0"), (dict(type=9), "element type"), (dict(out_type=2), "out_type"), (dict(id_bytes=1), "id_bytes"),
    (dict(n_ids=2 ** 31), "2^31"), (dict(n_docs=2 ** 31), "2^31"), (dict(n_rows=2 ** 31), "2^31"), (dict(out=None), "table_grad"), (dict(out=P + 2), "table_grad"),
    (dict(ids=P + 4), "ids"), (dict(grad=None), "grad is NULL"), (dict(stride=1), "stride"), (dict(stride=2 ** 31), "2^30"), (dict(ws=None), "workspace"), (dict(ws_bytes=8), "workspace")])
def test_embed_backward(change, needle):
    _refused(_call("mdd_embed_backward", BACK, **change), needle)


NORM = dict(ctx=CTX, x=P, type=F32, xs=64, res=P, rs=64, weight=P, eps=1e-6, n=5, dim=64, y=P, sum=P, rstd=P)
Q8 = dict(ctx=CTX, x=P, type=F32, xs=64, res=P, rs=64, weight=P, eps=1e-6, n=5, dim=64, kind=I8, codes=P, scales=P, sum=P)
NBACK = dict(ctx=CTX, g=P, type=F32, gs=64, h=P, hs=64, gsum=P, gss=64, weight=P, rstd=P, n=5, dim=64, dx=P, dw=P, ws=P, ws_bytes=BIG)
COMMON = [(dict(ctx=None), "ctx is NULL"), (dict(dim=0), "dim=0"), (dict(dim=40000), "dim=40000"), (dict(type=7), "element type")]


@pytest.mark.parametrize("change,needle", COMMON + [
    (dict(x=None), "x is NULL"), (dict(x=ODD), "aligned"), (dict(xs=63), "stride"), (dict(rs=2), "stride"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(y=None), "y is NULL")])
def test_rms_norm(change, needle):
    _refused(_call("mdd_rms_norm", NORM, **change), needle)


@pytest.mark.parametrize("change,needle", COMMON + [
    (dict(x=None), "x is NULL"), (dict(xs=63), "stride"), (dict(res=ODD), "aligned"), (dict(eps=-1.0), "eps"), (dict(kind=0), "8-bit kind"), (dict(codes=None), "NULL"),
    (dict(scales=None), "NULL")])
def test_rms_norm_q8(change, needle):
    _refused(_call("mdd_rms_norm_q8", Q8, **change), needle)


@pytest.mark.parametrize("change,needle", [c for c in COMMON] + [
    (dict(g=None), "grad is NULL"), (dict(h=None), "h is NULL"), (dict(hs=1), "stride"), (dict(gsum=ODD), "aligned"), (dict(dx=None), "x_grad"), (dict(rstd=None), "rstd"),
    (dict(ws=None), "workspace"), (dict(ws_bytes=10), "workspace")])
def test_rms_norm_backward(change, needle):
    _refused(_call("mdd_rms_norm_backward", NBACK, **change), needle)


COS = dict(ctx=CTX, codes=P, kind=I8, stride=64, n=5, dim=64, u=P, v=P, e=7, out=P)
SORT = dict(ctx=CTX, u=P, v=P, e=10000, docs=100, ws=P, ws_bytes=BIG)


@pytest.mark.parametrize("change,needle", [
    (dict(ctx=None), "ctx is NULL"), (dict(kind=1), "8-bit kind"), (dict(dim=0), "dim=0"), (dict(stride=63), "stride"), (dict(codes=None), "NULL"), (dict(u=None), "NULL"),
    (dict(out=None), "NULL")])
def test_edge_cosines(change, needle):
    _refused(_call("mdd_edge_cosines", COS, **change), needle)


@pytest.mark.parametrize("change,needle", [
    (dict(ctx=None), "ctx is NULL"), (dict(e=2 ** 31), "2^31"), (dict(docs=2 ** 32), "2^32"), (dict(u=None), "NULL"), (dict(ws=None), "workspace"),
    (dict(ws_bytes=1000), "workspace")])
def test_sort_edges(change, needle):
    _refused(_call("mdd_sort_edges", SORT, **change), needle)


QUANT = dict(ctx=CTX, x=P, type=F32, xs=64, n=5, dim=64, codes=P, scales=P)
MUL = dict(ctx=CTX, ac=P, as_=P, m=5, bc=P, bs=P, n=6, dim=64, alpha=1.0, c=P, c_type=F32, cs=6)
PAIRS = dict(ctx=CTX, codes=P, scales=P, m=100, dim=64, t=0.9, u=P, v=P, cap=10, count=P, ws=P, ws_bytes=BIG)


@pytest.mark.parametrize("change,needle", [
    (dict(ctx=None), "ctx is NULL"), (dict(dim=0), "dim=0"), (dict(type=4), "element type"), (dict(n=2 ** 31), "2^31"), (dict(x=None), "x is NULL"), (dict(xs=63), "stride"),
    (dict(codes=None), "NULL"), (dict(codes=P + 8), "16-byte"), (dict(scales=P + 4), "16-byte")])
def test_mx_quantize(change, needle):
    _refused(_call("mdd_mx_quantize", QUANT, **change), needle)


@pytest.mark.parametrize("change,needle", [
    (dict(ctx=None), "ctx is NULL"), (dict(dim=0), "dim=0"), (dict(c_type=2), "c_type"), (dict(m=2 ** 31 - 255), "2^31"), (dict(n=2 ** 31), "2^31"), (dict(ac=None), "A is NULL"),
    (dict(bs=P + 2), "16-byte"), (dict(c=None), "c is NULL"), (dict(c=P + 2), "aligned"), (dict(cs=5), "c_stride"), (dict(m=2 ** 30, n=2 ** 30, cs=2 ** 30), "2^31 tiles")])
def test_mx_matmul(change, needle):
    _refused(_call("mdd_mx_matmul", MUL, **change), needle)


@pytest.mark.parametrize("change,needle", [
    (dict(ctx=None), "NULL"), (dict(count=None), "NULL"), (dict(dim=0), "dim=0"), (dict(t=0.0), "min_cosine"), (dict(t=1.5), "min_cosine"), (dict(t=float("nan")), "min_cosine"),
    (dict(m=2 ** 22 + 1), "2^22"), (dict(u=None), "NULL"), (dict(codes=None), "NULL"), (dict(ws=None), "workspace"), (dict(ws_bytes=4), "workspace")])
def test_mx_pairs(change, needle):
    _refused(_call("mdd_mx_pairs", PAIRS, **change), needle)


def test_workspace_sizes():
    assert L.mdd_embed_ws_bytes(32, 256) == 0                                  # one piece: nothing to share
    assert L.mdd_embed_ws_bytes(33, 256) >= 2 * 2 * 256 * 4
    assert L.mdd_embed_backward_ws_bytes(100, 0, 1000, 8) >= 2 * 400 + 1001 * 8
    assert L.mdd_sort_edges_ws_bytes(8192) == 0 and L.mdd_sort_edges_ws_bytes(8193) >= 2 * 8193 * 4
    assert L.mdd_mx_pairs_ws_bytes(33) >= 64 * 4
    assert L.mdd_rms_norm_backward_ws_bytes(10 ** 6, 100) >= 512 * 400


def test_library_holds_no_packed_float_instructions(tmp_path):
    """v_pk_add_f32, v_pk_mul_f32 and v_pk_fma_f32 have given wrong results on this hardware: none in any kernel"""
    tool = "/opt/rocm/llvm/bin/llvm-objdump"
    if not os.path.exists(tool):
        pytest.skip("no llvm-objdump")
    shutil.copy(mlib.SO_PATH, tmp_path / "lib.so")
    subprocess.run([tool, "--offloading", "lib.so"], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    objects = [f for f in os.listdir(tmp_path) if "gfx950" in f]
    assert objects
    for f in objects:
        asm = subprocess.run([tool, "-d", f], cwd=tmp_path, check=True, stdout=subprocess.PIPE).stdout
        assert b"s_endpgm" in asm
        assert not re.search(rb"v_pk_(add|mul|fma)_f32", asm), f


# ------------------------------------------------------------------------------------------------ the Python methods
class _Engine(V.VectorOps):
    """the method bodies without their stream ordering; a library call would be an error"""
    device = torch.device("cpu")
    L = SimpleNamespace()
    ctx = None

    def __getattribute__(self, name):
        f = getattr(V.VectorOps, name, None)
        if f is not None and hasattr(f, "__wrapped__"):
            return f.__wrapped__.__get__(self)
        return super().__getattribute__(name)


E = _Engine()
M, I32 = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int32)


@pytest.mark.parametrize("call,needle", [
    (lambda: E.embed(M.double(), I32), "type"), (lambda: E.embed(M[0], I32), "matrix"), (lambda: E.embed(M.t(), I32), "unit stride"), (lambda: E.embed(M, I32.float()), "type"),
    (lambda: E.embed(M, I32, mode="max"), "mode"), (lambda: E.embed(M, I32, I32), "offsets"), (lambda: E.embed(M, I32, torch.zeros(0, dtype=torch.int64)), "n_docs"),
    (lambda: E.embed(M.to("meta"), I32), "tensor on"), (lambda: E.embed(M, torch.zeros(6, dtype=torch.int32)[::2]), "contiguous"),
    (lambda: E.embed(M.expand(4, 8)[:, :0], I32), "columns"), (lambda: E.embed(M[:1].expand(4, 8), I32), "unit stride"),
    (lambda: E.embed_backward(M, I32, 5), "rows"), (lambda: E.embed_backward(M[:3], I32, 5, dtype=torch.float16), "dtype"), (lambda: E.embed_backward(M[:3], I32, -1), "negative"),
    (lambda: E.rms_norm(M, M[0, :7]), "entries"), (lambda: E.rms_norm(M, None, M[:3]), "rows"), (lambda: E.rms_norm(M, M[0].half()), "type"),
    (lambda: E.rms_norm_q8(M, kind="int4"), "kind"), (lambda: E.rms_norm_backward(M, M, M[0]), "entries"), (lambda: E.rms_norm_backward(M.half(), M, M[:, 0].clone()), "type"),
    (lambda: E.edge_cosines(M, I32, I32), "int8"), (lambda: E.edge_cosines(M.to(torch.int8), I32, I32[:2]), "entries"), (lambda: E.sort_edges(I32, I32.long(), 5), "type"),
    (lambda: E.mx_matmul(M, M), "MxMatrix"), (lambda: E.mx_matmul(V.MxMatrix(M, M, 4, 8), None), "contiguous uint8"),
    (lambda: E.mx_pairs(V.MxMatrix(I32, I32, 1, 0), 0.9), "columns are supported"),
    (lambda: E.mx_pairs(V.MxMatrix(I32[:0].byte(), I32[:0].byte(), 0, 4), 0.9, max_pairs=-1), "max_pairs is negative")])
def test_python_refusals(call, needle):
    with pytest.raises(mlib.MddError, match=needle):
        call()


def test_python_refuses_products_that_do_not_fit():
    mx = lambda n, d: V.MxMatrix(torch.zeros(2048 * ((n + 31) // 32) * ((d + 127) // 128), dtype=torch.uint8),
                                 torch.zeros(128 * ((n + 31) // 32) * ((d + 127) // 128), dtype=torch.uint8), n, d)
    with pytest.raises(mlib.MddError, match="columns and b"):
        E.mx_matmul(mx(3, 8), mx(3, 9))
    with pytest.raises(mlib.MddError, match="dtype"):
        E.mx_matmul(mx(3, 8), mx(3, 8), dtype=torch.float16)
