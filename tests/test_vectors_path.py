"""Document vectors on the dedup path: dedup.vector_edges, cluster_local with vectors, and the --min_cosine options of cli/dedup.
The same tests run on the CPU (a backend that computes the operators from their definitions) and, marked gpu, on the engine."""
import json
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import vec_ref as R  # noqa: E402
from cpu_backend import OracleBackend  # noqa: E402
from map_neo_amd import dedup as D  # noqa: E402
from map_neo_amd.cli import dedup as stage  # noqa: E402


class VectorBackend(OracleBackend):
    def bucket_edges(self, key, meta, tuple_base, *rest):
        return super().bucket_edges(key, meta, tuple_base.reshape(-1), *rest)      # (addresses tuples in a flat array)

    def embed(self, table, ids, offsets=None, scale=1.0, mode="mean"):
        return R.embed(table, ids, offsets, scale, mode)[0].to(table.dtype)

    def rms_norm_q8(self, x, weight=None, residual=None, eps=1e-6, kind="int8"):
        q, s = R.q8(x, weight, residual, eps, kind)
        return q.to(torch.int8), s.float(), None

    def mx_quantize(self, x):
        v = R.mx_values(*R.mx_codes(x))
        return torch.from_numpy(v)

    def mx_pairs(self, v, min_cosine):
        ln = v.norm(dim=1)
        c = (v @ v.t()) / torch.where(ln > 0, ln, torch.full_like(ln, float("inf")))[:, None] / torch.where(ln > 0, ln, torch.full_like(ln, float("inf")))
        u, w = torch.nonzero(torch.tril(c >= min_cosine, -1), as_tuple=True)
        return u.int(), w.int()

    def edge_cosines(self, codes, eu, ev):
        return R.cosines(codes[eu.long()], codes[ev.long()]).float()


@pytest.fixture(params=["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])
def backend(request):
    return VectorBackend() if request.param == "cpu" else request.getfixturevalue("engine")


def _clustered(n, dim, near, g):
    """unit-scale vectors; `near` lists (copy, original, cosine)"""
    x = torch.randn(n, dim, generator=g, dtype=torch.float64)
    x /= x.norm(dim=1, keepdim=True)
    for c, o, cos in near:
        e = torch.randn(dim, generator=g, dtype=torch.float64)
        e -= (e @ x[o]) * x[o]
        x[c] = cos * x[o] + np.sqrt(1 - cos * cos) * e / e.norm()
    return x * 3.7


NEAR = [(10, 2, 0.99), (11, 2, 0.97), (40, 30, 0.93), (41, 31, 0.87), (50, 33, 0.8)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_vector_edges_keeps_what_reaches_the_threshold(backend, dtype):
    """0.93 and above stay at 0.9; 0.87 passes the 4-bit screen and fails the 8-bit check; order (u, v)"""
    g = torch.Generator().manual_seed(3)
    x = _clustered(120, 512, NEAR, g).to(dtype)
    x[100] = 0
    x[101, 5] = float("nan")
    u, v = D.vector_edges(backend, x.to(backend.device), 0.9)
    got = list(zip(u.cpu().tolist(), v.cpu().tolist()))
    # 11 and 10 are both near 2: cos(10, 11) is 0.99 * 0.97 plus or minus sin * sin / sqrt(512), above 0.9
    assert got == [(10, 2), (11, 2), (11, 10), (40, 30)]
    u, v = D.vector_edges(backend, x.to(backend.device), 0.85)
    assert (41, 31) in list(zip(u.cpu().tolist(), v.cpu().tolist()))
    assert D.vector_edges(backend, x[:0].to(backend.device), 0.9)[0].numel() == 0
    x[60:63] = x[59]
    u, v = D.vector_edges(backend, x.to(backend.device), 1.0)
    assert list(zip(u.cpu().tolist(), v.cpu().tolist())) == [(60, 59), (61, 59), (61, 60), (62, 59), (62, 60), (62, 61)]
    for bad in (0.0, 1.1, float("nan")):
        with pytest.raises(ValueError):
            D.vector_edges(backend, x.to(backend.device), bad)


def test_cluster_local_joins_both_kinds_of_edges(backend):
    """a shingle duplicate, a vector duplicate, and a chain of one of each; without vectors nothing changes"""
    sig = np.random.default_rng(0).integers(0, 2 ** 32, (60, 128), dtype=np.uint64).astype(np.uint32)
    sig[20] = sig[5]
    sig[31] = sig[30]
    x = _clustered(60, 256, [(45, 7, 0.99), (50, 31, 0.98)], torch.Generator().manual_seed(1)).float().to(backend.device)
    s = backend.to_device(sig)
    plain = D.cluster_local(backend, s)["labels"].cpu().numpy()
    both = D.cluster_local(backend, s, vectors=x, min_cosine=0.95)
    want = np.arange(60)
    want[20], want[31] = 5, 30
    assert (plain == want).all()
    want[45], want[50] = 7, 30
    assert (both["labels"].cpu().numpy() == want).all()
    assert both["removed"].cpu().numpy().nonzero()[0].tolist() == [20, 31, 45, 50]
    with pytest.raises(ValueError, match="go together"):
        D.cluster_local(backend, s, vectors=x)
    with pytest.raises(ValueError, match="59 rows"):
        D.cluster_local(backend, s, vectors=x[:59], min_cosine=0.9)


def _shards(tmp_path, texts):
    """two shards; the rows 3 and 8 have no content and are never hashed"""
    inp = tmp_path / "in"
    inp.mkdir()
    for name, lo, hi in (("a.jsonl", 0, 7), ("b.jsonl", 7, len(texts))):
        with open(inp / name, "w") as f:
            for i in range(lo, hi):
                f.write(json.dumps({"doc_id": "d%02d" % i, "raw_content": None if i in (3, 8) else texts[i]}) + "\n")
    return inp


def _texts():
    rng = np.random.default_rng(7)
    words = ["".join(chr(97 + c) for c in rng.integers(0, 26, 6)) for _ in range(400)]
    t = [" ".join(words[j] for j in rng.integers(0, 400, 60)) for _ in range(15)]
    t[4] = t[1]                                            # a duplicate by its text
    return t


@pytest.mark.parametrize("kind", ["embeddings", "table"])
def test_stage_command(backend, tmp_path, kind):
    inp, n = _shards(tmp_path, _texts()), 15
    g = torch.Generator().manual_seed(2)
    if kind == "embeddings":
        x = _clustered(n, 300, [(12, 6, 0.98), (9, 4, 0.98), (8, 2, 0.999)], g)      # row 8 is not hashed: its pair does not count
        np.save(tmp_path / "e.npy", x.numpy().astype(np.float16))
        extra = ["--embeddings", str(tmp_path / "e.npy")]
    else:
        table = torch.randn(500, 300, generator=g).numpy()
        ids = [np.random.default_rng(k).integers(0, 500, 20 + k) for k in range(n)]
        ids[12] = np.concatenate([ids[6], [-1, 10 ** 6]])   # the same tokens and two of padding
        ids[9] = np.concatenate([ids[4], ids[4][:2]])
        ids[8] = ids[2]
        np.save(tmp_path / "t.npy", table)
        np.save(tmp_path / "i.npy", np.concatenate(ids).astype(np.int64))
        np.save(tmp_path / "o.npy", np.concatenate([[0], np.cumsum([len(i) for i in ids])]).astype(np.int64))
        extra = ["--embedding_table", str(tmp_path / "t.npy"), "--token_ids", str(tmp_path / "i.npy"), "--token_offsets", str(tmp_path / "o.npy")]
    base = ["--input_dir", str(inp), "--workers", "1", "--normalize", "none"]
    run = lambda out, more: stage.run(stage.build_parser().parse_args(base + ["--output_dir", str(tmp_path / out)] + more), engine_factory=lambda d: backend)
    assert run("plain", [])["n_removed_ids"] == 1
    s = run("both", extra + ["--min_cosine", "0.9"])
    assert open(tmp_path / "both" / "removed_ids.txt").read().split() == ["d04", "d09", "d12"]
    clusters = {r["doc_id"]: r["cluster"] for r in map(json.loads, open(tmp_path / "both" / "clusters.jsonl"))}
    assert clusters == {"d01": "d01", "d04": "d01", "d09": "d01", "d06": "d06", "d12": "d06"} and s["n_clusters"] == 2


def test_stage_command_refusals(tmp_path):
    inp = _shards(tmp_path, _texts())
    x = np.random.default_rng(0).standard_normal((15, 40)).astype(np.float32)
    np.save(tmp_path / "e.npy", x)
    np.save(tmp_path / "short.npy", x[:14])
    np.save(tmp_path / "f64.npy", x.astype(np.float64))
    np.save(tmp_path / "i.npy", np.arange(10, dtype=np.int32))
    np.save(tmp_path / "o.npy", np.full(16, 11, dtype=np.int64))
    np.save(tmp_path / "o2.npy", np.zeros(15, dtype=np.int64))
    e, t = ["--embeddings", str(tmp_path / "e.npy")], ["--embedding_table", str(tmp_path / "e.npy"), "--token_ids", str(tmp_path / "i.npy")]
    c = ["--min_cosine", "0.9"]
    for more, what in ((c, "needs either"), (e, "needs either"), (e + ["--min_cosine", "1.5"], "0, 1"), (t + c, "go together"),
                       (e + t + ["--token_offsets", str(tmp_path / "o.npy")] + c, "needs either"), (e + c + ["--checkpoint_dir", str(tmp_path / "ck")], "without --checkpoint"),
                       (e + c + ["--distributed"], "single-process"), (["--embeddings", str(tmp_path / "short.npy")] + c, "14 rows"),
                       (["--embeddings", str(tmp_path / "f64.npy")] + c, "float64"), (t + ["--token_offsets", str(tmp_path / "o.npy")] + c, "does not ascend"),
                       (t + ["--token_offsets", str(tmp_path / "o2.npy")] + c, "15 entries")):
        args = stage.build_parser().parse_args(["--input_dir", str(inp), "--workers", "1", "--output_dir", str(tmp_path / "o")] + more)
        with pytest.raises(SystemExit, match=what):
            stage.run(args, engine_factory=lambda d: VectorBackend())
