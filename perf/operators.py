"""The document-vector operators of map_neo_amd as measurable cases: what each is given, its plain form in elementary
torch operations, and the call a user of minhash.Engine makes.

The path they come from is near-duplicate detection by document vectors: token ids are looked up in an embedding table
and averaged per document (embed), the vectors are normalised and held in 8 bits (rms_norm_q8) or in microscaled 4 bits
(mx_quantize), compared with an index (mx_matmul) or among themselves (mx_pairs), and the pairs found are checked on the
8-bit rows (edge_cosines).  A table is fitted to a corpus with the two backward passes.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_handle = None


# ---------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # a single short text embedded on its own, as a lookup service does: latency
        {"name": "embed_query", "op": "embed", "docs": 1, "mean_len": 24, "vocab": 64000, "dim": 256, "type": "bf16", "mode": "mean"},
        # the documents of one ingest block (ragged, some empty, padding ids among them) averaged over a static table
        {"name": "embed_corpus", "op": "embed", "docs": 40000, "mean_len": 480, "vocab": 64000, "dim": 256, "type": "bf16", "mode": "mean"},
        # a training step's token-level lookup and its gradient: 262144 tokens, frequent tokens many times over
        {"name": "embed_train", "op": "embed_train", "docs": 0, "tokens": 262144, "vocab": 64000, "dim": 1024, "type": "bf16", "mode": "sum"},
        # one vector normalised and put into 8 bits: latency
        {"name": "norm_query", "op": "rms_norm_q8", "rows": 1, "dim": 768, "type": "bf16", "kind": "int8", "residual": False},
        # the last layer's outputs of an encoder with their residual stream, a block of documents
        {"name": "norm_corpus", "op": "rms_norm_q8", "rows": 262144, "dim": 768, "type": "bf16", "kind": "int8", "residual": True},
        # a training step's norm, forward and backward, at an odd width, with the gradient that reaches the residual stream
        {"name": "norm_train", "op": "rms_norm_train", "rows": 20001, "dim": 1000, "type": "fp16", "residual": True},
        # one query against an index held in 4 bits: the single-token product, bound by reading the index
        {"name": "mx_query", "op": "mx_matmul", "rows": 1, "index": 262144, "dim": 1024, "type": "bf16", "out": "fp32"},
        # a block of documents against an index: the large product
        {"name": "mx_block", "op": "mx_matmul", "rows": 8192, "index": 32768, "dim": 2048, "type": "bf16", "out": "bf16"},
        # near pairs of a small shard, odd sizes
        {"name": "pairs_small", "op": "mx_pairs", "docs": 2999, "dim": 384, "type": "fp32"},
        # near pairs of a block of documents
        {"name": "pairs_block", "op": "mx_pairs", "docs": 45000, "dim": 768, "type": "bf16"},
        # candidate pairs of a small shard checked on 8-bit floating rows
        {"name": "cosines_small", "op": "edge_cosines", "rows": 5000, "dim": 257, "edges": 1500, "kind": "e4m3"},
        # candidate pairs of a whole corpus checked on 8-bit integer rows
        {"name": "cosines_corpus", "op": "edge_cosines", "rows": 262144, "dim": 768, "edges": 2000000, "kind": "int8"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "embed_train", "rms_norm_q8", "rms_norm_train", "mx_matmul", "mx_pairs", "edge_cosines"])
    typ = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "embed":
        dim, mean_len = _log_int(rng, 32, 1024), _log_int(rng, 4, 2000)
        docs = _log_int(rng, 1, max(1, min(60000, 2400000000 // (dim * mean_len))))
        return {"op": op, "docs": docs, "mean_len": mean_len, "vocab": _log_int(rng, 1000, 128000), "dim": dim, "type": typ,
                "mode": rng.choice(["mean", "sum"])}
    if op == "embed_train":
        dim, tokens = _log_int(rng, 32, 1024), _log_int(rng, 16, 262144)
        return {"op": op, "docs": rng.choice([0, max(1, tokens // 100)]), "tokens": tokens, "vocab": _log_int(rng, 1000, 64000),
                "dim": dim, "type": typ, "mode": rng.choice(["mean", "sum"])}
    if op in ("rms_norm_q8", "rms_norm_train"):
        dim = _log_int(rng, 64, 8192)
        rows = _log_int(rng, 1, min(200000, (50000000 if typ != "fp32" else 25000000) // dim))
        c = {"op": op, "rows": rows, "dim": dim, "type": typ, "residual": rng.random() < 0.5}
        if op == "rms_norm_q8":
            c["kind"] = rng.choice(["int8", "e4m3"])
        return c
    if op == "mx_matmul":
        return {"op": op, "rows": _log_int(rng, 1, 6000), "index": _log_int(rng, 100, 32768), "dim": _log_int(rng, 64, 2048),
                "type": typ, "out": rng.choice(["fp32", "bf16"])}
    if op == "mx_pairs":
        return {"op": op, "docs": _log_int(rng, 200, 40000), "dim": rng.randint(256, 1024), "type": typ}
    return {"op": op, "rows": _log_int(rng, 100, 200000), "dim": _log_int(rng, 64, 1024), "edges": _log_int(rng, 1, 1000000),
            "kind": rng.choice(["int8", "e4m3"])}


# ------------------------------------------------------------------------------------------------------------ the work
def work(case):
    op = case["op"]
    if op == "embed":
        tokens, d, e = case["docs"] * case["mean_len"], case["dim"], BYTES[case["type"]]
        touched = min(case["vocab"], tokens)
        return {"bytes": 4 * tokens + 8 * (case["docs"] + 1) + touched * d * e + case["docs"] * d * e, "flops": tokens * d}
    if op == "embed_train":
        tokens, d, e = case["tokens"], case["dim"], BYTES[case["type"]]
        rows = case["docs"] or tokens
        return {"bytes": 4 * tokens + 8 * (case["docs"] + 1) + min(case["vocab"], tokens) * d * e + 2 * rows * d * e + case["vocab"] * d * 4,
                "flops": 2 * tokens * d}
    if op == "rms_norm_q8":
        n, e = case["rows"] * case["dim"], BYTES[case["type"]]
        return {"bytes": n * e * (3 if case["residual"] else 1) + n + 4 * case["rows"] + case["dim"] * e, "flops": 6 * n}
    if op == "rms_norm_train":
        n, e = case["rows"] * case["dim"], BYTES[case["type"]]
        return {"bytes": n * e * (7 if case["residual"] else 4) + case["dim"] * (e + 4), "flops": 14 * n}
    if op == "mx_matmul":
        m, n, k = case["rows"], case["index"], case["dim"]
        packed = n * (k / 2 + k / 32)
        return {"bytes": int(m * k * BYTES[case["type"]] + packed + m * n * BYTES[case["out"]]), "flops": 2 * m * n * k}
    if op == "mx_pairs":
        n, k = case["docs"], case["dim"]
        return {"bytes": int(n * k * BYTES[case["type"]]), "flops": n * (n - 1) * k}
    return {"bytes": min(case["rows"], 2 * case["edges"]) * case["dim"] + 12 * case["edges"], "flops": 6 * case["edges"] * case["dim"]}


# ----------------------------------------------------------------------------------------------------------- the inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _zipf_ids(n, vocab, g):
    """token ids as text has them: frequency about 1 / rank; 1 in 64 is padding (-1)"""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    rank = torch.exp(u * math.log(vocab + 1.0)).long() - 1
    rank = (rank.clamp_(0, vocab - 1) * 7919) % vocab
    pad = torch.rand(n, generator=g, device="cuda") < 1.0 / 64
    return torch.where(pad, torch.full_like(rank, -1), rank).to(torch.int32)


def _offsets(docs, total, g):
    """`docs` ragged documents over `total` tokens; about 1 in 50 is empty (never the only one)"""
    w = torch.exp(torch.randn(docs, generator=g, device="cuda", dtype=torch.float64))
    if docs > 1:
        w = torch.where(torch.rand(docs, generator=g, device="cuda") < 0.02, torch.zeros_like(w), w)
        w[0] += 0.01
    cut = torch.cumsum(w, 0) / w.sum()
    offs = torch.zeros(docs + 1, device="cuda", dtype=torch.int64)
    offs[1:] = (cut * total).round().long()
    offs[-1] = total
    return torch.cummax(offs, 0).values


def _vectors(n, dim, typ, g):
    """document vectors: a common direction and a topic of their own; one document in 40 has three copies with noise, anywhere"""
    x = torch.randn(n, dim, generator=g, device="cuda") + 0.3 * torch.randn(1, dim, generator=g, device="cuda")
    place, m = torch.randperm(n, generator=g, device="cuda"), n // 40
    x[place[m: 4 * m]] = x[place[:m]].repeat(3, 1) + 0.1 * torch.randn(3 * m, dim, generator=g, device="cuda")
    return x.to(typ)


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    st = dict(case)
    if op in ("embed", "embed_train"):
        tokens = case["docs"] * case["mean_len"] if op == "embed" else case["tokens"]
        st["ids"] = _zipf_ids(tokens, case["vocab"], g)
        st["offsets"] = _offsets(case["docs"], tokens, g) if case["docs"] else None
        st["scale"] = 1.0 if case["docs"] else math.sqrt(case["dim"])
        st["table"] = (torch.randn(case["vocab"], case["dim"], generator=g, device="cuda") * 0.1).to(TYPES[case["type"]])
        if op == "embed_train":
            st["grad"] = (torch.randn(case["docs"] or tokens, case["dim"], generator=g, device="cuda") * 0.01).to(TYPES[case["type"]])
    elif op in ("rms_norm_q8", "rms_norm_train"):
        t, shape = TYPES[case["type"]], (case["rows"], case["dim"])
        st["x"] = (torch.randn(shape, generator=g, device="cuda") * 2).to(t)
        st["weight"] = (1 + 0.2 * torch.randn(case["dim"], generator=g, device="cuda")).to(t)
        st["res"] = torch.randn(shape, generator=g, device="cuda").to(t) if case["residual"] else None
        if op == "rms_norm_train":
            st["grad"] = (torch.randn(shape, generator=g, device="cuda") * 0.1).to(t)
            st["grad_sum"] = (torch.randn(shape, generator=g, device="cuda") * 0.1).to(t) if case["residual"] else None
    elif op == "mx_matmul":
        st["x"] = _vectors(case["rows"], case["dim"], TYPES[case["type"]], g)
        st["codes"], st["scales"] = _mx_pack(_vectors(case["index"], case["dim"], torch.bfloat16, g))
    elif op == "mx_pairs":
        st["x"] = _vectors(case["docs"], case["dim"], TYPES[case["type"]], g)
        st["min_cosine"] = 0.9
    else:
        v = _vectors(case["rows"], case["dim"], torch.float32, g)
        v = v / v.abs().amax(1, keepdim=True)
        st["rows8"] = (v * 127).round().to(torch.int8) if case["kind"] == "int8" else (v * 448).to(torch.float8_e4m3fn)
        st["eu"] = torch.randint(0, case["rows"], (case["edges"],), generator=g, device="cuda").to(torch.int32)
        st["ev"] = torch.randint(0, case["rows"], (case["edges"],), generator=g, device="cuda").to(torch.int32)
    return st


# ------------------------------------------------------------------------- microscaled 4-bit numbers, in plain operations
def _mx_split(x):
    """x [n, k] -> (values on the 4-bit grid [n, k32, 32], exponents [n, k32]): per 32 columns one power of two,
    2^(floor(log2(largest)) - 2), elements rounded to the nearest of 0 .5 1 1.5 2 3 4 6, ties to even, larger ones to 6"""
    n, k = x.shape
    kb = (k + 31) // 32
    b = torch.nn.functional.pad(x.float(), (0, kb * 32 - k)).view(n, kb, 32)
    e = (torch.frexp(b.abs().amax(2)).exponent - 3).clamp(-127, 127)
    a = torch.ldexp(b, -e[:, :, None].float())
    m = a.abs()
    q = torch.where(m < 2, (m * 2).round() / 2, torch.where(m < 4, m.round(), (m / 2).round() * 2)).clamp_(max=6)
    return torch.copysign(q, a), e


def _mx_values(x):
    """the values that the 4-bit form of x stands for, float32 [n, k]"""
    q, e = _mx_split(x)
    return torch.ldexp(q, e[:, :, None].float()).reshape(x.shape[0], -1)[:, : x.shape[1]]


def _mx_pack(x):
    """the packed form: 32-row by 128-column tiles, codes [row tile, column tile, block of 32 columns, row, 16 bytes],
    scales [row tile, column tile, half of the block (block & 1), row, block >> 1] as the matrix instruction reads them"""
    n, k = x.shape
    rt, ct = (n + 31) // 32, (k + 127) // 128
    q, e = _mx_split(x)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=x.device)
    c = torch.bucketize(q.abs(), grid).to(torch.uint8) | (torch.signbit(q).to(torch.uint8) << 3)
    full = torch.zeros(rt * 32, ct * 4, 32, dtype=torch.uint8, device=x.device)
    full[:n, : c.shape[1]] = c
    byte = full[..., 0::2] | (full[..., 1::2] << 4)
    codes = byte.view(rt, 32, ct, 4, 16).permute(0, 2, 3, 1, 4).contiguous()
    s = torch.full((rt * 32, ct * 4), 127, dtype=torch.uint8, device=x.device)
    s[:n, : e.shape[1]] = (e + 127).to(torch.uint8)
    scales = s.view(rt, 32, ct, 2, 2).permute(0, 2, 4, 1, 3).contiguous()
    return codes, scales


def _mx_unpack(codes, scales, n, k):
    rt, ct = codes.shape[:2]
    byte = codes.permute(0, 3, 1, 2, 4).reshape(rt * 32, ct * 4, 16)
    lut = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = lut[torch.stack([byte & 15, byte >> 4], -1).int()].view(rt * 32, ct * 4, 32)
    e = scales.permute(0, 3, 1, 4, 2).reshape(rt * 32, ct * 4).float() - 127
    return torch.ldexp(v, e[:, :, None]).view(rt * 32, ct * 128)[:n, :k]


# -------------------------------------------------------------------------------------------------------------- one pass
def _nearest(z, kind):
    """the nearest 8-bit value, ties to even: whole numbers, or 3 bits behind the leading one (steps of 2^-9 below 2^-6)"""
    if kind == "int8":
        return z.round()
    step = torch.ldexp(torch.ones_like(z), torch.frexp(z.abs().clamp(min=2.0 ** -6)).exponent - 4)
    return (z / step).round() * step


def _doc_of(st):
    offs = st["offsets"]
    return torch.repeat_interleave(torch.arange(st["docs"], device="cuda"), offs[1:] - offs[:-1], output_size=st["ids"].numel())


def _plain(st):
    op = st["op"]
    if op in ("embed", "embed_train"):
        ids = st["ids"].long()
        ok = (ids >= 0) & (ids < st["vocab"])
        safe = torch.where(ok, ids, torch.zeros_like(ids))
        if st["offsets"] is not None:
            doc = _doc_of(st)
            n = torch.zeros(st["docs"], device="cuda").index_add_(0, doc, ok.float())
            per_doc = st["scale"] / n.clamp(min=1) if st["mode"] == "mean" else torch.full_like(n, st["scale"])
        out = st["table"].float()[safe] * ok[:, None]
        if st["offsets"] is not None:
            out = torch.zeros(st["docs"], st["dim"], device="cuda").index_add_(0, doc, out) * per_doc[:, None]
        else:
            out = out * st["scale"]
        out = {"vectors": out.to(st["table"].dtype)}
        if op == "embed":
            return out
        g = st["grad"].float()
        g = (g * per_doc[:, None])[doc] if st["offsets"] is not None else g * st["scale"]
        out["table_grad"] = torch.zeros(st["vocab"], st["dim"], device="cuda").index_add_(0, safe, g * ok[:, None])
        return out
    if op == "rms_norm_q8":
        h = st["x"].float() + st["res"].float() if st["res"] is not None else st["x"].float()
        # the norm's factor is common to a row: it goes into the row's scale alone, and a code depends on h * weight only --
        # in 64 bits, since the codes next to a rounding border are lost in 32
        y = st["x"].double() * st["weight"].double()
        if st["res"] is not None:
            y = y + st["res"].double() * st["weight"].double()
        top = 127.0 if st["kind"] == "int8" else 448.0
        big = y.abs().amax(1)
        s = big.float() * torch.rsqrt(h.square().mean(1) + 1e-6) / top
        q = _nearest(y * top / big[:, None], st["kind"]).float()
        out = {"values": q * s[:, None], "scales": s}
        if st["res"] is not None:
            out["sum"] = h.to(st["x"].dtype)
        return out
    if op == "rms_norm_train":
        h = st["x"].float() + st["res"].float() if st["res"] is not None else st["x"].float()
        g, w, r = st["grad"].float(), st["weight"].float(), torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-6)
        y, x = (h * r * w).to(st["x"].dtype), h.to(st["x"].dtype).float()       # the backward pass has the sum as it was stored
        gw = g * w
        dx = r * gw - x * (r ** 3) * (gw * x).mean(1, keepdim=True)
        if st["grad_sum"] is not None:
            dx = dx + st["grad_sum"].float()
        return {"normed": y, "sum": x.to(st["x"].dtype), "x_grad": dx.to(st["x"].dtype), "weight_grad": (g * x * r).sum(0)}
    if op == "mx_matmul":
        b = _mx_unpack(st["codes"], st["scales"], st["index"], st["dim"])
        return {"product": (_mx_values(st["x"]) @ b.t()).to(TYPES[st["out"]])}
    if op == "mx_pairs":
        v = _mx_values(st["x"])
        v = v / v.square().sum(1, keepdim=True).sqrt().clamp(min=1e-30)
        near = torch.tril(v @ v.t() >= st["min_cosine"], -1).nonzero()
        return {"u": near[:, 0].int(), "v": near[:, 1].int()}
    a, b = st["rows8"].float()[st["eu"].long()], st["rows8"].float()[st["ev"].long()]
    return {"cosines": (a * b).sum(1) / (a.square().sum(1) * b.square().sum(1)).sqrt()}


def run(state):
    if not own:
        return _plain(state)
    from map_neo_amd.minhash import Engine, MxMatrix
    global _handle
    if _handle is None:
        _handle = Engine(torch.cuda.current_device())
    eng, st, op = _handle, state, state["op"]
    if op in ("embed", "embed_train"):
        out = {"vectors": eng.embed(st["table"], st["ids"], st["offsets"], scale=st["scale"], mode=st["mode"])}
        if op == "embed_train":
            out["table_grad"] = eng.embed_backward(st["grad"], st["ids"], st["vocab"], st["offsets"], scale=st["scale"], mode=st["mode"])
        return out
    if op == "rms_norm_q8":
        codes, scales, total = eng.rms_norm_q8(st["x"], st["weight"], st["res"], kind=st["kind"])
        values = codes * scales[:, None] if st["kind"] == "int8" else codes.float().mul_(scales[:, None])
        return {"values": values, "scales": scales} if total is None else {"values": values, "scales": scales, "sum": total}
    if op == "rms_norm_train":
        y, total, rstd = eng.rms_norm(st["x"], st["weight"], st["res"])
        dx, dw = eng.rms_norm_backward(st["grad"], total, rstd, st["weight"], grad_sum=st["grad_sum"])
        return {"normed": y, "sum": total, "x_grad": dx, "weight_grad": dw}
    if op == "mx_matmul":
        index = MxMatrix(st["codes"], st["scales"], st["index"], st["dim"])
        return {"product": eng.mx_matmul(eng.mx_quantize(st["x"]), index, dtype=TYPES[st["out"]])}
    if op == "mx_pairs":
        u, v = eng.mx_pairs(eng.mx_quantize(st["x"]), st["min_cosine"])
        return {"u": u, "v": v}
    return {"cosines": eng.edge_cosines(st["rows8"], st["eu"], st["ev"])}


# --------------------------------------------------------------------------------------- the definitions, in 64 bits
def _exact_mx(x):
    """the 4-bit values of x from the definition: every element compared with the seven midpoints of the grid (an element on
    a midpoint takes the neighbour with the even code)"""
    n, k = x.shape
    kb = -(-k // 32)
    b = torch.zeros(n, kb * 32, dtype=torch.float64, device=x.device)
    b[:, :k] = x.double()
    b = b.view(n, kb, 32)
    top = b.abs().amax(2, keepdim=True)
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    e = torch.where(top > 0, e, torch.full_like(e, -125.0)) - 2
    unit = torch.exp2(e.clamp(-127, 127))
    m = (b.abs() / unit)
    v = torch.zeros_like(m)
    for mid, step, even_above in ((0.25, 0.5, False), (0.75, 0.5, True), (1.25, 0.5, False), (1.75, 0.5, True), (2.5, 1.0, False),
                                  (3.5, 1.0, True), (5.0, 2.0, False)):
        v += step * ((m >= mid) if even_above else (m > mid))
    return (torch.sign(b) * v * unit).view(n, -1)[:, :k]


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op in ("embed", "embed_train"):
        ids, v = st["ids"].long(), case["vocab"]
        ok = (ids >= 0) & (ids < v)
        offs = st["offsets"] if st["offsets"] is not None else torch.arange(ids.numel() + 1, device="cuda")
        run_ok = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), torch.cumsum(ok.long(), 0)])
        n_ok = run_ok[offs[1:]] - run_ok[offs[:-1]]
        scale = torch.full((offs.numel() - 1,), float(st["scale"]), dtype=torch.float64, device="cuda")
        if st["offsets"] is not None and case["mode"] == "mean":
            scale = scale / n_ok.clamp(min=1)
        if op == "embed":
            out = torch.empty(case["docs"], case["dim"], dtype=torch.float64, device="cuda")
            ends = offs.tolist()
            step = max(1, 20000000 // case["dim"])
            d0 = 0
            while d0 < case["docs"]:
                d1 = d0 + 1
                while d1 < case["docs"] and ends[d1 + 1] - ends[d0] <= step:
                    d1 += 1
                part, good = ids[ends[d0]: ends[d1]], ok[ends[d0]: ends[d1]]
                rows = st["table"][part.clamp(0, v - 1)].double() * good[:, None]
                total = torch.cat([torch.zeros(1, case["dim"], dtype=torch.float64, device="cuda"), torch.cumsum(rows, 0)])
                out[d0:d1] = total[offs[d0 + 1: d1 + 1] - ends[d0]] - total[offs[d0:d1] - ends[d0]]
                d0 = d1
            return {"vectors": out * scale[:, None]}
        if st["offsets"] is None:
            vectors = torch.where(ok[:, None], st["table"].double()[ids.clamp(0, v - 1)], 0.0) * scale[:, None]
        else:
            which = torch.searchsorted(offs, torch.arange(ids.numel(), device="cuda"), right=True) - 1
            vectors = torch.stack([torch.zeros(case["docs"], dtype=torch.float64, device="cuda").index_put_(
                (which,), st["table"][:, c].double()[ids.clamp(0, v - 1)] * ok, accumulate=True) for c in range(case["dim"])], 1) * scale[:, None]
        order = torch.argsort(torch.where(ok, ids, torch.full_like(ids, v)), stable=True)
        row = torch.searchsorted(offs, order, right=True) - 1 if st["offsets"] is not None else order
        first = torch.searchsorted(torch.where(ok, ids, torch.full_like(ids, v))[order].contiguous(), torch.arange(v + 1, device="cuda"))
        out = torch.empty(v, case["dim"], dtype=torch.float64, device="cuda")
        for c in range(0, case["dim"], 128):
            rows = st["grad"][:, c: c + 128].double()[row] * scale[row][:, None]
            total = torch.cat([torch.zeros(1, rows.shape[1], dtype=torch.float64, device="cuda"), torch.cumsum(rows, 0)])
            out[:, c: c + 128] = total[first[1:]] - total[first[:-1]]
        return {"vectors": vectors, "table_grad": out}
    if op == "rms_norm_q8":
        h = st["x"].double()
        if st["res"] is not None:
            h = h + st["res"].double()
        y = h * st["weight"].double()
        top = 127.0 if case["kind"] == "int8" else 448.0
        big = y.abs().max(1).values
        s = big / (h.pow(2).sum(1) / case["dim"] + 1e-6).sqrt() / top
        z = y * top / big[:, None]
        if case["kind"] == "int8":
            q = torch.round(z)
        else:                                        # 3 bits behind the leading one, steps of 2^-9 below 2^-6
            unit = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
            q = torch.round(z / unit) * unit
        out = {"values": q * s[:, None], "scales": s}
        if st["res"] is not None:
            out["sum"] = h
        return out
    if op == "rms_norm_train":
        h = st["x"].double()
        if st["res"] is not None:
            h = h + st["res"].double()
        g, w, r = st["grad"].double(), st["weight"].double(), 1 / (h.pow(2).sum(1, keepdim=True) / case["dim"] + 1e-6).sqrt()
        x = h.to(st["x"].dtype).double()
        n = x * r
        dx = r * (g * w - n * ((g * w * n).sum(1, keepdim=True) / case["dim"]))
        if st["grad_sum"] is not None:
            dx = dx + st["grad_sum"].double()
        return {"normed": h * r * w, "sum": h, "x_grad": dx, "weight_grad": (g * n).sum(0)}
    if op == "mx_matmul":
        a = _exact_mx(st["x"])
        b = _mx_unpack(st["codes"], st["scales"], case["index"], case["dim"]).double()
        return {"product": a.mm(b.t().contiguous())}
    if op == "mx_pairs":
        v = _exact_mx(st["x"])
        v = v / v.pow(2).sum(1).clamp(min=1e-60).sqrt()[:, None]
        us, vs = [], []
        for r in range(0, case["docs"], 4096):
            hit = v[r: r + 4096].mm(v[: r + 4096].t().contiguous()) >= st["min_cosine"]
            i, j = hit.nonzero(as_tuple=True)
            i = i + r
            us.append(i[j < i])
            vs.append(j[j < i])
        return {"u": torch.cat(us).int(), "v": torch.cat(vs).int()}
    out = torch.empty(case["edges"], dtype=torch.float64, device="cuda")
    for k in range(0, case["edges"], 1 << 18):
        a = st["rows8"][st["eu"][k: k + (1 << 18)].long()].to(torch.float64)
        b = st["rows8"].float()[st["ev"][k: k + (1 << 18)].long()].to(torch.float64)
        out[k: k + (1 << 18)] = (a * b).sum(1) / a.norm(dim=1) / b.norm(dim=1)
    return {"cosines": out}
