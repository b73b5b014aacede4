"""Whole-path drivers: signatures -> band records -> buckets/edges -> components -> removed.

`dedup_local`       one GPU, everything stays in HBM.
`dedup_distributed` one process per GPU (torch.distributed; backend "nccl" = RCCL over xGMI):
                    documents are sharded by contiguous global index range, band records are
                    routed to their owner rank with an all-to-all so that every (band, tuple)
                    bucket lives on ONE GPU (EN:136's groupBy shuffle, ZH-1:58-61's per-band
                    directories), the edges every rank finds are all-gathered and every rank
                    runs the same union-find, so labels are identical on all ranks and equal
                    to the one-GPU result.

Both take a `backend` object implementing the stage methods of minhash.Engine.  The product
backend is Engine (HIP); tests may inject another backend to exercise the sharding / exchange
logic on CPU with gloo.  Nothing in this module computes a hash or a signature itself.
"""
from __future__ import annotations

import math
from typing import Optional

import numpy as np
import torch

from .minhash import BANDS, NUM_PERM, ROWS, SEED, WIDTH
from .vectors import MAX_PAIR_ROWS, TooManyPairs


class StageTimer:
    """Optional per-stage timing with events on the current stream (bench only)."""

    def __init__(self):
        self.marks = []

    def mark(self, name: str):
        ev = torch.cuda.Event(enable_timing=True)
        ev.record()
        self.marks.append((name, ev))

    def result_ms(self) -> dict:
        torch.cuda.synchronize()
        out = {}
        for (_, e0), (name, e1) in zip(self.marks[:-1], self.marks[1:]):
            out[name] = out.get(name, 0.0) + e0.elapsed_time(e1)
        return out


def verified_edges(be, sig: torch.Tensor, eu: torch.Tensor, ev: torch.Tensor, min_jaccard: float):
    """The edges whose two documents agree on at least ceil(min_jaccard * K) signature components (datasketch's
    MinHash.jaccard() >= min_jaccard).  An extension: the reference has no such step (EN:136-145 unions every pair)."""
    need = int(math.ceil(float(min_jaccard) * sig.shape[1] - 1e-9))
    keep = be.signature_matches(sig, eu, ev) >= need
    return eu[keep], ev[keep]


def _four_bits(x: torch.Tensor) -> torch.Tensor:
    """x rounded as mx_quantize does (include/mdd.h), in float32, columns filled up to whole blocks; blocks below 2^-100, which
    do not count beside a row's length of 1, to zeros"""
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).view(x.shape[0], -1, 32)
    e = torch.frexp(x.abs().amax(2, keepdim=True))[1].clamp(min=-100) - 3
    x = torch.ldexp(x, -e)
    step = torch.where(x.abs() < 2, 0.5, torch.where(x.abs() < 4, 1.0, 2.0))
    return torch.ldexp((torch.round(x / step) * step).clamp(-6.0, 6.0), e).view(x.shape[0], -1)


# The 4-bit screen of vector_edges looks this far below the threshold, at least
SCREEN_MARGIN = 0.05


def screen_margin(vectors: torch.Tensor, min_cosine: float) -> float:
    """How far below min_cosine the 4-bit rows of two such vectors may fall.  Their rounding takes 0.01 off the cosine on average; how
    much it scatters depends on how many columns carry a row: at 0.9 up to 0.02 with 768 even ones, 0.08 with one in 32 twenty times
    the others, 0.12 with 4 columns.  So it is measured: up to 8192 rows, each with a vector at exactly that cosine which
    leaves it in the direction of another row -- of every second, with its columns in other places.  A quarter more than the worst of
    them, and 0.01: of pairs right at the threshold fewer than one in a thousand is missed, in any of these sets."""
    n, dim = vectors.shape
    if n < 2:
        return SCREEN_MARGIN
    m = max(256, min(8192, (1 << 21) // dim))
    k = torch.arange(m, device=vectors.device)
    row = k * n // m if n > m else k % n
    other = (row + 1 + (k * 31 + k // n * 7) % (n - 1)) % n                      # never the row itself
    x, z = vectors[row].float(), vectors[other].float()
    z[1::2] = torch.roll(z[1::2], dim // 2 + 1, 1)
    x, z = (t / t.norm(dim=1, keepdim=True) for t in (x, z))
    z = torch.nn.functional.normalize(z - (z * x).sum(1, keepdim=True) * x)
    a, b = _four_bits(x), _four_bits(min_cosine * x + math.sqrt(max(0.0, 1.0 - min_cosine ** 2)) * z)
    loss = min_cosine - (a * b).sum(1) / torch.sqrt((a * a).sum(1) * (b * b).sum(1))
    return max(SCREEN_MARGIN, 1.25 * float(torch.nan_to_num(loss, nan=0.0, posinf=0.0).max()) + 0.01)


def _blocks(n: int, dim: int):
    """ranges of rows that hold about 2^25 numbers each: what the checks below take into 64 bits at a time"""
    step = max(1, (1 << 25) // max(1, dim))
    return [(k, min(n, k + step)) for k in range(0, n, step)]


def _cosines64(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    a, b = a.double(), b.double()
    return (a * b).sum(1) / torch.sqrt((a * a).sum(1) * (b * b).sum(1))


def _angles(cosines: torch.Tensor) -> torch.Tensor:
    return torch.acos(cosines.double().clamp(-1.0, 1.0))


def _reach(be, vectors, eu, ev, min_cosine: float) -> torch.Tensor:
    """which pairs have vectors with a cosine >= min_cosine, decided in 64 bits by the vectors themselves; of many pairs only those
    that their 8-bit rows leave open.  Angles on a sphere add up like distances: the angle of two vectors is that of their 8-bit
    rows, give or take the angles between each and its own.  Open are cosines within 0.007 of 0.9 for 768 evenly sized columns,
    far more where one column sets the step of all codes."""
    n, dim = vectors.shape
    keep = torch.zeros(eu.numel(), dtype=torch.bool, device=eu.device)
    open_ = None
    if eu.numel() > n:                                           # a row's angle to its 8-bit form costs what a pair's cosine does
        limit = math.acos(min(1.0, min_cosine))
        codes, _, _ = be.rms_norm_q8(vectors)
        off = torch.empty(n, dtype=torch.float64, device=vectors.device)
        for a, b in _blocks(n, dim):
            off[a:b] = _angles(_cosines64(vectors[a:b], codes[a:b]) - 2.0 ** -40)
        open_ = []
        for a, b in _blocks(eu.numel(), 2):
            cos, slack = be.edge_cosines(codes, eu[a:b], ev[a:b]).double(), off[eu[a:b].long()] + off[ev[a:b].long()]
            keep[a:b] = _angles(cos - 2.0 ** -20) + slack <= limit               # 2^-20: the roundings of a cosine in 32 bits
            open_.append(torch.nonzero(~keep[a:b] & (_angles(cos + 2.0 ** -20) - slack <= limit)).flatten() + a)
        open_ = torch.cat(open_)
    for a, b in _blocks(eu.numel() if open_ is None else open_.numel(), dim):
        k = slice(a, b) if open_ is None else open_[a:b]
        keep[k] = _cosines64(vectors[eu[k].long()], vectors[ev[k].long()]) >= min_cosine - 2.0 ** -40             # (equal rows: 1 but for roundings)
    return keep


def _near_pairs(be, vectors, min_cosine: float, margin: Optional[float] = None, split: bool = True):
    """yields (u, v), u > v: every pair of vector_edges once, in one piece and ordered where one search takes them all.  Rows
    beyond MAX_PAIR_ROWS, and sets with more candidates than mx_pairs returns, are cut into ranges: each is searched by itself,
    and each two of them as one matrix, of which the pairs across count (twice the products of a single search)."""
    if not 0.0 < float(min_cosine) <= 1.0:
        raise ValueError("min_cosine must be in (0, 1]")
    be.mx_quantize(vectors[:0])                                  # refuses what is no matrix of vectors
    n = vectors.shape[0]
    if margin is None:
        margin = screen_margin(vectors, float(min_cosine))
    todo = [((0, n), None)]
    while todo:
        one, two = todo.pop()
        first, size = one[1] - one[0], sum(r[1] - r[0] for r in (one, two) if r)
        cuts = 2
        if size <= MAX_PAIR_ROWS:
            x = vectors[one[0]: one[1]] if two is None else torch.cat([vectors[r[0]: r[1]] for r in (one, two)])
            try:
                u, v = be.mx_pairs(be.mx_quantize(x), max(float(min_cosine) - margin, 0.01))
            except TooManyPairs as e:
                if not split or size <= 2:
                    raise
                cuts = min(size, 64, max(2, math.ceil(2 * math.sqrt(e.count / max(1, e.limit)))))
            else:
                if two is not None:
                    across = (u >= first) & (v < first)
                    u, v = u[across], v[across]
                keep = _reach(be, x, u, v, float(min_cosine))
                u, v = u[keep], v[keep]
                yield (u if one[0] == 0 and two is None else u + (one[0] if two is None else two[0] - first)), (v if one[0] == 0 else v + one[0])
                continue
        elif not split:
            raise TooManyPairs(size, MAX_PAIR_ROWS, min_cosine)
        pieces = [[p for p in zip(c[:-1], c[1:]) if p[0] < p[1]] for c in ([r[0] + (r[1] - r[0]) * k // cuts for k in range(cuts + 1)] for r in (one, two) if r)]
        if two is None:
            todo += [(p, None) for p in pieces[0]] + [(p, q) for k, q in enumerate(pieces[0]) for p in pieces[0][:k]]
        else:
            todo += [(p, q) for p in pieces[0] for q in pieces[1]]


def vector_edges(be, vectors: torch.Tensor, min_cosine: float, margin: Optional[float] = None, max_pairs: int = 1 << 28):
    """Near-duplicate pairs by document vectors [n, dim]: of the pairs whose 4-bit rows reach min_cosine - margin (default: by
    screen_margin), those whose vectors have a cosine >= min_cosine.  Returns (u, v), u > v, ordered; more than max_pairs raise
    TooManyPairs.  Every pair returned reaches min_cosine; the screen may miss a few, fewer than one in a thousand, of those
    that barely reach it.  An extension: the reference compares documents by their shingles only.  Vectors of zeros, with a
    NaN, or of a length outside [2^-60, 2^60] pair with nothing."""
    parts, count = [], 0
    for u, v in _near_pairs(be, vectors, min_cosine, margin):
        count += u.numel()
        if count > max_pairs:
            raise TooManyPairs(count, max_pairs, float(min_cosine))
        parts.append((u, v))
    if len(parts) == 1:
        return parts[0]
    key = torch.sort(torch.cat([u.long() << 32 | v.long() for u, v in parts])).values
    return (key >> 32).int(), (key & 0xFFFFFFFF).int()


def _first_equal(vectors: torch.Tensor) -> torch.Tensor:
    """int64 [n]: the first row that holds the same bits as this one; the row itself where it pairs with nothing"""
    n, dim = vectors.shape
    dev, me = vectors.device, torch.arange(n, device=vectors.device)
    mul = torch.randint(-2 ** 63, 2 ** 63 - 1, (dim,), generator=torch.Generator().manual_seed(0)).to(dev)
    bits = {4: torch.int32, 2: torch.int16}[vectors.element_size()]
    h, live = torch.empty(n, dtype=torch.int64, device=dev), torch.empty(n, dtype=torch.bool, device=dev)
    for a, b in _blocks(n, dim):
        x = vectors[a:b].contiguous()
        h[a:b] = (x.view(bits).long() * mul).sum(1)
        length = x.double().norm(dim=1)
        live[a:b] = (length >= 2.0 ** -60) & (length <= 2.0 ** 60)
    values, inverse = torch.unique(h, return_inverse=True)
    first = torch.full((values.numel(),), n, dtype=torch.int64, device=dev).scatter_reduce_(0, inverse, me, "amin")[inverse]
    for a, b in _blocks(n, dim):                                 # equal sums are not yet equal rows
        live[a:b] &= (vectors[a:b] == vectors[first[a:b]]).all(1)
    return torch.where(live, first, me)


def _join_near(be, labels, vectors, min_cosine: float):
    """unions the near pairs of `vectors` into labels without holding all of them: equal rows, of which a corpus may have any
    number (empty pages, error pages), are joined to the first one and searched once"""
    first = _first_equal(vectors)
    me = torch.arange(first.numel(), device=first.device)
    again, row = torch.nonzero(first != me).flatten(), torch.nonzero(first == me).flatten()
    be.components_union(labels, again.int(), first[again].int())
    for u, v in _near_pairs(be, vectors[row] if again.numel() else vectors, min_cosine):
        be.components_union(labels, row[u.long()].int(), row[v.long()].int())


def cluster_local(be, sig: torch.Tensor, bands: int = BANDS, rows: int = ROWS, key_bits: int = 64,
                  want_buckets: bool = False, timer: Optional[StageTimer] = None, min_jaccard: Optional[float] = None,
                  vectors: Optional[torch.Tensor] = None, min_cosine: Optional[float] = None):
    """Band records -> buckets/edges -> union-find -> removed mask for signatures already in HBM
    (EN:133-145 / ZH-2..ZH-4).  Document index = row of `sig`.  min_jaccard (default None = the reference's behaviour)
    drops candidate edges (document, smallest document of its bucket) whose estimated Jaccard similarity is lower.  vectors
    [n, dim] with min_cosine (default None) add the pairs of vector_edges; where one search does not take them all (more than
    MAX_PAIR_ROWS documents, or 2^28 candidate pairs), they are joined piece by piece and edge_u / edge_v are one edge
    for every document that is not the smallest of its component, to that one."""
    n, num_perm = sig.shape
    if (vectors is None) != (min_cosine is None):
        raise ValueError("vectors and min_cosine go together")
    if vectors is not None and vectors.shape[0] != n:
        raise ValueError("vectors has %d rows for %d documents" % (vectors.shape[0], n))
    mark = timer.mark if timer is not None else (lambda name: None)
    key, meta = be.band_keys(sig, bands, rows, 0, key_bits)
    mark("band_keys")
    eu, ev, n_coll, rb = be.bucket_edges(key, meta, sig, bands, num_perm, rows, rows, want_buckets)
    mark("bucket_edges")
    if min_jaccard is not None:
        eu, ev = verified_edges(be, sig, eu, ev, min_jaccard)
        mark("verify")
    joined = False
    if vectors is not None:
        try:
            for vu, vv in _near_pairs(be, vectors, min_cosine, split=False):
                eu, ev = torch.cat([eu, vu]), torch.cat([ev, vv])
            joined = True
        except TooManyPairs:
            pass
        mark("vector_edges")
    labels = be.components_init(n)
    be.components_union(labels, eu, ev)
    if vectors is not None and not joined:
        _join_near(be, labels, vectors, min_cosine)
    be.components_finish(labels)
    if vectors is not None and not joined:
        eu, ev = be.forest_edges(labels, n)
    removed, n_removed = be.removed_mask(labels, 0, n)
    mark("components")
    return {"sig": sig, "key": key, "meta": meta, "edge_u": eu, "edge_v": ev, "labels": labels,
            "removed": removed, "n_removed": n_removed, "n_collisions": int(n_coll),
            "rec_bucket": rb}


def dedup_local(be, text: torch.Tensor, offsets: torch.Tensor, num_perm: int = NUM_PERM, width: int = WIDTH,
                unit: str = "char", bands: int = BANDS, rows: int = ROWS, seed: int = SEED,
                text_bytes: Optional[int] = None, key_bits: int = 64, want_buckets: bool = False,
                timer: Optional[StageTimer] = None, min_jaccard: Optional[float] = None,
                vectors: Optional[torch.Tensor] = None, min_cosine: Optional[float] = None):
    """One-GPU path.  Returns a dict of device tensors: sig [n,K], edge_u/edge_v, labels [n]
    (label = smallest doc index of the component), removed [n] uint8, n_removed (device
    int64[1]), n_collisions (host int)."""
    mark = timer.mark if timer is not None else (lambda name: None)
    mark("start")
    sig = be.signatures(text, offsets, num_perm, width, unit, seed, text_bytes=text_bytes)
    mark("signatures")
    return cluster_local(be, sig, bands, rows, key_bits, want_buckets, timer, min_jaccard, vectors, min_cosine)


def signatures_streamed(be, blocks, n_docs: int, num_perm=NUM_PERM, width: int = WIDTH, unit: str = "char", seed: int = SEED,
                        on_block=None):
    """Signatures of a corpus that does not (have to) fit in HBM as text: `blocks` yields (text, offsets, text_bytes) of
    consecutive document ranges (packed device tensors, as for Engine.signatures); every block is hashed into its rows of
    ONE resident signature matrix and may then be dropped -- at 100 M documents the text is ~220 GB, the signatures 51 GB.
    num_perm may be a tuple: several matrices from one pass over the text (band sweeps with different K).
    on_block(first_doc, text, offsets, text_bytes, ms) is called after each block (ms: kernel time by events).
    Returns the int32 matrix [n_docs, K] (a dict K -> matrix when num_perm is a tuple)."""
    many = isinstance(num_perm, (tuple, list))
    Ks = list(num_perm) if many else [num_perm]
    sigs = {K: torch.empty((n_docs, K), dtype=torch.int32, device=be.device) for K in Ks}
    d0 = 0
    for text, offs, nbytes in blocks:
        nd = offs.numel() - 1
        if d0 + nd > n_docs:
            raise ValueError("signatures_streamed: the blocks hold more than n_docs documents")
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        for K in Ks:
            be.signatures(text, offs, K, width, unit, seed, text_bytes=nbytes, out=sigs[K][d0:d0 + nd])
        e1.record()
        if on_block is not None:
            e1.synchronize()
            on_block(d0, text, offs, nbytes, e0.elapsed_time(e1))
        d0 += nd
    if d0 != n_docs:
        raise ValueError("signatures_streamed: the blocks hold %d documents, expected %d" % (d0, n_docs))
    return sigs if many else sigs[Ks[0]]


# RCCL on this stack silently drops the tail of an all_to_all_single message beyond 1 GiB (measured with one rank:
# everything past the first half of a 1 GiB + 8 KiB message arrives untouched, tools/diag_a2a.py), so no single
# collective call here moves more than COLLECTIVE_BYTES (half the observed limit) in total; larger exchanges run in rounds.
COLLECTIVE_BYTES = 512 << 20


def _host_staged(t: torch.Tensor, group=None) -> bool:
    """gloo carries CUDA tensors through the host anyway and was seen to dead-lock with several ranks on one GPU
    (rehearsals of the multi-rank path on a one-GPU box): with that backend the exchanges below are staged
    explicitly through host memory.  RCCL (backend "nccl") always works on the device buffers."""
    import os
    import torch.distributed as dist
    if os.environ.get("MDD_GLOO_DEVICE_TENSORS") == "1":      # diagnosis only (tools/gloo_probe.py)
        return False
    return t.is_cuda and dist.get_backend(group) == "gloo"


def _all_to_all_v(t: torch.Tensor, send_counts, recv_counts, width: int, group=None, limit_bytes: Optional[int] = None):
    """Variable all-to-all of records of `width` elements: t holds the records for peer 0, peer 1, ... back to back
    (send_counts records each); returns what the peers sent here, grouped by peer (recv_counts)."""
    import torch.distributed as dist
    if _host_staged(t, group):
        return _all_to_all_v(t.cpu(), send_counts, recv_counts, width, group, limit_bytes).to(t.device)
    world = len(send_counts)
    send_counts = [int(c) for c in send_counts]
    recv_counts = [int(c) for c in recv_counts]
    out = torch.empty(sum(recv_counts) * width, dtype=t.dtype, device=t.device)
    per_peer = max(1, (limit_bytes or COLLECTIVE_BYTES) // (t.element_size() * width * world))   # records per peer per round
    mx = torch.tensor([max(send_counts + recv_counts + [0])], dtype=torch.int64, device=t.device)
    dist.all_reduce(mx, op=dist.ReduceOp.MAX, group=group)       # every rank must run the same number of rounds
    rounds = max(1, -(-int(mx.item()) // per_peer))
    if rounds == 1:
        dist.all_to_all_single(out, t, [c * width for c in recv_counts], [c * width for c in send_counts], group=group)
        return out
    s_off = [0] * world
    r_off = [0] * world
    for p in range(1, world):
        s_off[p] = s_off[p - 1] + send_counts[p - 1]
        r_off[p] = r_off[p - 1] + recv_counts[p - 1]
    for k in range(rounds):
        s_cnt = [min(max(c - k * per_peer, 0), per_peer) for c in send_counts]
        r_cnt = [min(max(c - k * per_peer, 0), per_peer) for c in recv_counts]
        sbuf = torch.cat([t[(s_off[p] + k * per_peer) * width: (s_off[p] + k * per_peer + s_cnt[p]) * width] for p in range(world)])
        rbuf = torch.empty(sum(r_cnt) * width, dtype=t.dtype, device=t.device)
        dist.all_to_all_single(rbuf, sbuf, [c * width for c in r_cnt], [c * width for c in s_cnt], group=group)
        pos = 0
        for p in range(world):
            out[(r_off[p] + k * per_peer) * width: (r_off[p] + k * per_peer + r_cnt[p]) * width] = rbuf[pos: pos + r_cnt[p] * width]
            pos += r_cnt[p] * width
    return out


def _all_gather_v(t: torch.Tensor, group=None, limit_bytes: Optional[int] = None):
    """All-gather of variable-length 1-D tensors (sizes exchanged first), in rounds of bounded size."""
    import torch.distributed as dist
    if _host_staged(t, group):
        return _all_gather_v(t.cpu(), group, limit_bytes).to(t.device)
    world = dist.get_world_size(group)
    n = torch.tensor([t.numel()], dtype=torch.int64, device=t.device)
    sizes = [torch.zeros_like(n) for _ in range(world)]
    dist.all_gather(sizes, n, group=group)
    sizes = [int(s.item()) for s in sizes]
    per_rank = max(1, (limit_bytes or COLLECTIVE_BYTES) // (t.element_size() * world))
    parts = [[] for _ in range(world)]
    for lo in range(0, max(max(sizes), 1), per_rank):
        cnt = [min(max(s - lo, 0), per_rank) for s in sizes]
        mx = max(max(cnt), 1)
        pad = torch.zeros(mx, dtype=t.dtype, device=t.device)
        mine = t[lo: lo + per_rank]
        pad[: mine.numel()] = mine
        outs = [torch.empty_like(pad) for _ in range(world)]
        dist.all_gather(outs, pad, group=group)
        for p in range(world):
            parts[p].append(outs[p][: cnt[p]])
    return torch.cat([x for p in range(world) for x in parts[p]])


class TorchComm:
    """The exchanges of the multi-GPU path over torch.distributed.  This is the TEST / rehearsal transport: gloo on CPU
    tensors (tests/test_distributed_cpu.py) and gloo with every rank on one GPU (rehearsals on a one-GPU box).  The
    product transport is NativeComm (collectives issued by libmdd_hip.so against RCCL)."""

    name = "torch.distributed"

    def __init__(self, group=None):
        self.group = group

    def exchange(self, tuples_s: torch.Tensor, meta_s: torch.Tensor, send_counts: torch.Tensor, rows: int):
        import torch.distributed as dist
        send = [int(c) for c in send_counts.tolist()]
        sc = torch.tensor(send, dtype=torch.int64, device=meta_s.device)
        rc = torch.empty_like(sc)
        if _host_staged(sc, self.group):
            sc_h, rc_h = sc.cpu(), rc.cpu()
            dist.all_to_all_single(rc_h, sc_h, group=self.group)
            rc = rc_h
        else:
            dist.all_to_all_single(rc, sc, group=self.group)
        recv = [int(c) for c in rc.tolist()]
        tuples_r = _all_to_all_v(tuples_s, send, recv, rows, self.group)
        meta_r = _all_to_all_v(meta_s, send, recv, 1, self.group)
        return tuples_r, meta_r, send, recv

    def allgather_edges(self, eu: torch.Tensor, ev: torch.Tensor):
        return _all_gather_v(eu, self.group), _all_gather_v(ev, self.group)


class CommInitError(RuntimeError):
    """mdd_comm_init did not succeed on every rank"""


class NativeComm:
    """The exchanges issued by libmdd_hip.so itself (include/mdd.h: mdd_comm_init, mdd_exchange_counts / _bands,
    mdd_allgather_counts / _edges) against RCCL, on the engine's stream; torch only owns the buffers.  The
    communicator's id travels from rank 0 to the others through the torch.distributed process group that launched
    the job (object broadcast: plumbing).  One host synchronisation per exchange (the counts), inside the library."""

    name = "libmdd_hip + RCCL"

    def __init__(self, engine, group=None):
        import torch.distributed as dist
        self.eng = engine
        self.rank, self.world = dist.get_rank(group), dist.get_world_size(group)
        box = [engine.comm_unique_id() if self.rank == 0 else None]
        if self.world > 1:
            dist.broadcast_object_list(box, src=dist.get_global_rank(group, 0) if group is not None else 0, group=group)
        # mdd_comm_init is collective, but a rank can still fail on its own after ncclCommInitRank (staging allocation):
        # agree on the outcome, so that either every rank uses the native transport or none does
        ok, why = 1, ""
        try:
            engine.comm_init(box[0], self.rank, self.world)
        except Exception as e:      # noqa: BLE001 -- the other ranks must hear of it whatever it was
            ok, why = 0, repr(e)
        if self.world > 1:
            flag = torch.tensor([ok], dtype=torch.int32, device=engine.device)
            dist.all_reduce(flag, op=dist.ReduceOp.MIN, group=group)
            all_ok = int(flag.item()) == 1
        else:
            all_ok = ok == 1
        if not all_ok:
            if ok:
                engine.comm_destroy()
            raise CommInitError(why or "mdd_comm_init failed on another rank")

    @classmethod
    def from_unique_id(cls, engine, unique_id: bytes, rank: int, world: int):
        """For launchers without torch.distributed (one thread or process per GPU that hands rank 0's
        Engine.comm_unique_id() to the others by its own means): collective, every rank calls it."""
        self = cls.__new__(cls)
        self.eng, self.rank, self.world = engine, int(rank), int(world)
        engine.comm_init(unique_id, self.rank, self.world)
        return self

    def exchange(self, tuples_s, meta_s, send_counts, rows):
        return self.eng.exchange_bands(tuples_s, meta_s, send_counts, rows)

    def allgather_edges(self, eu, ev):
        return self.eng.allgather_edges(eu, ev)


def default_comm(be, group=None):
    """NativeComm for the HIP engine under the RCCL ("nccl") backend, TorchComm otherwise (gloo: CPU tests, one-GPU
    rehearsals; MDD_COMM=torch forces it).  Cached on the engine: a context has one communicator."""
    import os
    import torch.distributed as dist
    native = (hasattr(be, "comm_init") and dist.get_backend(group) == "nccl" and os.environ.get("MDD_COMM", "native") != "torch")
    if not native:
        return TorchComm(group)
    comm = getattr(be, "_native_comm", None)
    if comm is None:
        # RCCL must be loadable on EVERY rank before any rank enters ncclCommInitRank (a rank that cannot load it would
        # leave the others waiting there for ever): probe locally, agree, and only then initialise.  Without agreement
        # all ranks take torch.distributed's RCCL communicator instead -- loudly; it is the same library and the same
        # wire traffic, issued from Python.
        ok, why = 1, ""
        try:
            be.comm_unique_id()
        except Exception as e:      # noqa: BLE001 -- whatever went wrong, the other ranks must hear of it
            ok, why = 0, repr(e)
        flag = torch.tensor([ok], dtype=torch.int32, device=be.device)
        dist.all_reduce(flag, op=dist.ReduceOp.MIN, group=group)
        if int(flag.item()) == 0:
            import sys
            print("map_neo_amd: libmdd_hip could not bind RCCL on every rank (%s): the exchanges go through "
                  "torch.distributed on this run" % (why or "another rank failed"), file=sys.stderr, flush=True)
            comm = TorchComm(group)
        else:
            try:
                comm = NativeComm(be, group)
            except CommInitError as e:
                import sys
                print("map_neo_amd: mdd_comm_init did not succeed on every rank (%s): the exchanges go through "
                      "torch.distributed on this run" % e, file=sys.stderr, flush=True)
                comm = TorchComm(group)
        be._native_comm = comm
    return comm


def dedup_distributed(be, text: torch.Tensor, offsets: torch.Tensor, doc_base: int, n_global: int,
                      num_perm: int = NUM_PERM, width: int = WIDTH, unit: str = "char", bands: int = BANDS,
                      rows: int = ROWS, seed: int = SEED, text_bytes: Optional[int] = None, key_bits: int = 64,
                      group=None, timings: Optional[dict] = None, timer: Optional[StageTimer] = None, comm=None):
    """Multi-GPU path; every rank calls it with its own shard (documents doc_base ..
    doc_base+n_local of n_global).  Returns the same dict as dedup_local; labels cover all
    n_global documents (replicated), removed covers the local shard."""
    if timer is not None:
        timer.mark("start")
    sig = be.signatures(text, offsets, num_perm, width, unit, seed, text_bytes=text_bytes)
    if timer is not None:
        timer.mark("signatures")
    return cluster_distributed(be, sig, doc_base, n_global, bands, rows, key_bits, group, timings, timer, comm)


def cluster_distributed(be, sig: torch.Tensor, doc_base: int, n_global: int, bands: int = BANDS, rows: int = ROWS,
                        key_bits: int = 64, group=None, timings: Optional[dict] = None, timer: Optional[StageTimer] = None,
                        comm=None):
    """Multi-GPU clustering of signatures already in HBM (row i of `sig` = global document doc_base + i):
    band records -> all-to-all by bucket owner -> local buckets -> spanning forest -> all-gather ->
    replicated union-find.  Same return value as dedup_distributed.  `comm` carries the two exchanges
    (default_comm: libmdd_hip + RCCL for the HIP engine, torch.distributed for tests)."""
    if comm is None:
        comm = default_comm(be, group)
    if getattr(comm, "world", None) is not None:      # NativeComm knows its communicator (and may run without torch.distributed)
        world, rank = comm.world, comm.rank
    else:
        import torch.distributed as dist
        world, rank = dist.get_world_size(group), dist.get_rank(group)
    n_local = sig.shape[0]
    mark = timer.mark if timer is not None else (lambda name: None)
    key, meta = be.band_keys(sig, bands, rows, doc_base, key_bits)
    mark("band_keys")
    # --- route band records to their owner rank (all-to-all over xGMI); the counts stay on the device
    tuples_s, meta_s, send_counts = be.route(sig, key, meta, bands, rows, world)
    mark("route")
    tuples_r, meta_r, send_list, recv_list = comm.exchange(tuples_s, meta_s, send_counts, rows)
    mark("all_to_all")
    del tuples_s, meta_s
    # --- local buckets over the records this rank owns
    key_r = be.packed_keys(tuples_r, meta_r, rows, key_bits)
    eu, ev, n_coll, _ = be.bucket_edges(key_r, meta_r, tuples_r, 1, rows, 0, rows, False)
    mark("bucket_edges")
    # --- merge: reduce this rank's edges to a spanning forest (at most one edge per touched
    # document), all-gather the forests, identical union-find everywhere
    n_local_edges = int(eu.numel())
    if world > 1 and n_local_edges:
        lab_local = be.components_init(n_global)
        be.components_union(lab_local, eu, ev)
        be.components_finish(lab_local)
        eu, ev = be.forest_edges(lab_local, n_local_edges)
        del lab_local
    mark("forest")
    eu_all, ev_all = comm.allgather_edges(eu, ev)
    mark("all_gather")
    labels = be.components_init(n_global)
    be.components_union(labels, eu_all, ev_all)
    be.components_finish(labels)
    removed, n_removed = be.removed_mask(labels, doc_base, n_local)
    mark("components")
    if timings is not None:
        rec_bytes = 4 * rows + 8
        timings["transport"] = comm.name
        timings["records_sent"] = int(sum(send_list))
        timings["records_received"] = int(sum(recv_list))
        timings["records_sent_to_other_ranks"] = int(sum(send_list) - send_list[rank])
        timings["all_to_all_bytes_sent"] = int(sum(send_list)) * rec_bytes
        timings["all_to_all_bytes_received"] = int(sum(recv_list)) * rec_bytes
        timings["record_bytes"] = rec_bytes
        timings["edges_local"] = n_local_edges
        timings["forest_edges_local"] = int(eu.numel())
        timings["edges_global"] = int(eu_all.numel())
        timings["all_gather_bytes_received"] = int(eu_all.numel()) * 8
    return {"sig": sig, "edge_u": eu_all, "edge_v": ev_all, "labels": labels, "removed": removed,
            "n_removed": n_removed, "n_collisions": int(n_coll)}
