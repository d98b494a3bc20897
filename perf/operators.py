"""Measured cases of the local side of the memory: a paged cache of local keys and values, the attention of new
tokens over it, and the local attention with score terms (cap, distance bias, document and prefix masks) with its
backward.

``run`` computes a case in plain torch operations (``own = False``) or with the package's kernels (``own = True``);
``exact`` computes it from the definition in 64 bits.  A case's lengths, documents and page tables follow from its
``pattern`` number; the values in them follow from the seed."""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EMPTY_LSE = torch.finfo(torch.float32).min
META = 16  # words in front of a cache's bookkeeping


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step of 64 sequences writes its new rows (512 local keys each: the decode batch of the benchmark)
        dict(name="append-decode-64", op="append", dtype="bf16", H=8, d=128, page=16, pages=4096, rows=64, width=64,
             length=512, new=1, pattern=1),
        # prompts of a batch enter the cache: ragged chunks that begin and end inside pages
        dict(name="append-prompts", op="append", dtype="fp16", H=8, d=128, page=64, pages=1024, rows=8, width=96,
             length=700, new=2048, pattern=2),
        # a step of a beam search: the beams that lost leave, the ones that won are forked into their rows
        dict(name="fork-beams", op="fork", dtype="bf16", H=8, d=128, page=64, pages=4096, rows=128, width=64,
             length=2048, pattern=3),
        # a pool after many requests came and went is packed to its front, so that its tail can be given away
        dict(name="compact-pool", op="compact", dtype="bf16", H=8, d=128, page=64, pages=8192, rows=96, width=96,
             length=3500, pattern=4),
        # the smallest call: one token of one sequence, where latency is all
        dict(name="chunk-one-token", op="chunk", dtype="bf16", H=8, G=4, d=128, page=16, rows=1, new=1, length=512,
             cap=0.0, slopes=False, prefix=0, pattern=5),
        # a decode step of the benchmark's 64 sequences over their 512 local keys
        dict(name="chunk-decode-64", op="chunk", dtype="bf16", H=8, G=4, d=128, page=16, rows=64, new=1, length=512,
             cap=0.0, slopes=False, prefix=0, pattern=6),
        # decode over long local windows with a distance bias: all bytes of the cache are read once
        dict(name="chunk-decode-long", op="chunk", dtype="fp16", H=8, G=8, d=128, page=64, rows=32, new=1,
             length=32768, cap=0.0, slopes=True, prefix=0, pattern=7),
        # chunked prefill: ragged chunks of new tokens behind what is cached, capped scores
        dict(name="chunk-prefill", op="chunk", dtype="bf16", H=8, G=4, d=128, page=64, rows=4, new=1024, length=16384,
             cap=30.0, slopes=False, prefix=0, pattern=8),
        # a toy training step in fp32 (the benchmark's smallest configuration)
        dict(name="train-toy-fp32", op="train", dtype="fp32", H=1, G=1, d=64, S=512, L=512, causal=True, cap=20.0,
             slopes=True, docs=1, prefix=0, pattern=9),
        # packed documents under a cap, at the heads and tokens of the benchmark's prefill chunk
        dict(name="train-documents", op="train", dtype="bf16", H=8, G=4, d=128, S=2048, L=2048, causal=True, cap=30.0,
             slopes=False, docs=5, prefix=0, pattern=10),
        # the local attention of the benchmark's largest configuration, with a distance bias and a prefix
        dict(name="train-64-heads", op="train", dtype="bf16", H=8, G=8, d=128, S=4096, L=4096, causal=True, cap=0.0,
             slopes=True, docs=1, prefix=300, pattern=11),
        # odd extents, more keys than queries, every term at once, fp16 at the smaller head dimension
        dict(name="train-ragged-fp16", op="train", dtype="fp16", H=4, G=2, d=64, S=1501, L=2011, causal=True, cap=25.0,
             slopes=True, docs=3, prefix=40, pattern=12),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    top = {}
    for c in listed():
        top[c["op"]] = max(top.get(c["op"], 0.0), _cost(c))
    while True:
        op = rng.choice(["append", "fork", "compact", "chunk", "chunk", "train", "train"])
        c = dict(op=op, dtype=rng.choice(["bf16", "fp16", "bf16", "fp32"]), d=rng.choice([64, 128, 128, 256]),
                 H=rng.choice([1, 2, 4, 8]), pattern=rng.randrange(1 << 20))
        if op == "train":
            S = _spread(rng, 16, 4096)
            L = S + rng.choice([0, 0, _spread(rng, 1, 2048)])
            c.update(G=rng.choice([1, 2, 3, 4, 8]), S=S, L=L, causal=rng.random() < 0.8,
                     cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.5,
                     docs=min(L, rng.choice([1, 1, 2, 7])), prefix=rng.choice([0, 0, _spread(rng, 1, 500)]))
            if c["H"] * c["G"] * S * L > 1.1e9:
                continue
        elif op == "chunk":
            c.update(G=rng.choice([1, 2, 3, 4, 8]), page=rng.choice([16, 32, 64, 128]), rows=_spread(rng, 1, 64),
                     new=rng.choice([1, 1, _spread(rng, 2, 1024)]), length=_spread(rng, 1, 16384),
                     cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.4,
                     prefix=rng.choice([0, 0, _spread(rng, 1, 300)]))
            if c["rows"] * c["H"] * c["G"] * c["new"] * c["length"] > 2.2e9:
                continue
        else:
            page = rng.choice([16, 32, 64])
            rows, length = _spread(rng, 1, 256), _spread(rng, 1, 4096)
            width = length // page + 2 + (_spread(rng, 1, 2048) // page + 1 if op == "append" else 0)
            c.update(page=page, rows=rows, length=length, width=width, pages=rows * width + _spread(rng, 16, 2048))
            if op == "append":
                c["new"] = rng.choice([1, 1, min(2048, (width - length // page - 1) * page)])
            if 2 * c["pages"] * c["H"] * page * c["d"] * _size(c) > 2.2e9:
                continue
        if _cost(c) <= top[op]:
            return c


def _size(case):
    return 4 if case["dtype"] == "fp32" else 2


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


# ------------------------------------------------------------------------------------- what a pattern stands for
def _pool(case):
    """Bookkeeping of a cache in use: lengths, tables and reference counts, and what the case asks of it."""
    rng = np.random.RandomState(case["pattern"])
    R, P, n, M = case["rows"], case["page"], case["pages"], case["width"]
    most = max(1, case["length"])
    length = rng.randint(max(1, most // 2), most + 1, R).astype(np.int64)
    if case["op"] == "fork":
        length[R // 2 + R % 2:] = 0  # the rows that the winning beams are forked into
    refs, table = np.zeros(n, np.int64), np.full((R, M), -1, np.int64)
    order, at = rng.permutation(n), 0
    for r in range(R):
        count = -(-int(length[r]) // P)
        shared = 0
        if r % 4 == 3:  # a row that was forked from its neighbour earlier: its whole first pages are shared
            shared = min(int(length[r - 1]) // P, int(length[r]) // P) // 2
            table[r, :shared] = table[r - 1, :shared]
            refs[table[r, :shared]] += 1
        table[r, shared:count] = order[at:at + count - shared]
        refs[table[r, shared:count]] += 1
        at += count - shared
    asked = {}
    if case["op"] == "append":
        new = np.minimum(rng.randint(max(1, case["new"] // 2), case["new"] + 1, R), M * P - length)
        asked["cu"] = np.concatenate([[0], np.cumsum(np.maximum(new, 0))])
    if case["op"] == "fork":
        half = R // 2 + R % 2
        drop = np.zeros(R, np.int64)
        lost = rng.permutation(half)[:half // 4]
        drop[lost] = 1 << 20
        left = np.setdiff1d(np.arange(half), lost)
        src = np.full(R, -1, np.int64)
        src[half:] = left[rng.randint(0, len(left), R - half)]
        asked.update(drop=drop, src=src)
    return length, refs, table, asked


def _chunk(case):
    """Lengths (new tokens among them) and new tokens of every row of a batch, and its pages."""
    rng = np.random.RandomState(case["pattern"])
    R, P = case["rows"], case["page"]
    new = rng.randint(max(1, case["new"] * 3 // 4), case["new"] + 1, R)
    length = np.maximum(new, rng.randint(max(1, case["length"] // 2), case["length"] + 1, R))
    M = -(-int(length.max()) // P)
    n = int(sum(-(-int(x) // P) for x in length)) + 8
    order, at = rng.permutation(n), 0
    table = np.full((R, M), -1, np.int64)
    for r in range(R):
        count = -(-int(length[r]) // P)
        table[r, :count] = order[at:at + count]
        at += count
    return length, np.concatenate([[0], np.cumsum(new)]), table, n


def _documents(case):
    """Document of every key, its first key, and how many keys each query sees as far as order goes."""
    rng = np.random.RandomState(case["pattern"])
    S, L = case["S"], case["L"]
    cuts = np.sort(rng.choice(np.arange(1, L), case["docs"] - 1, replace=False)) if case["docs"] > 1 else np.zeros(0, int)
    doc = np.searchsorted(cuts, np.arange(L), side="right")
    first = np.concatenate([[0], cuts])[doc]
    prefix = np.zeros(S, np.int64)
    if case["prefix"]:
        at = np.clip(np.arange(S) + L - S, 0, L - 1)
        prefix = np.minimum(first[at] + case["prefix"], L)
    order = np.clip(np.arange(S) + L - S + 1, 0, L) if case["causal"] else np.full(S, L)
    return doc, first, prefix, np.minimum(L, np.maximum(order, prefix))


def work(case):
    e = _size(case)
    if case["op"] == "train":
        doc, first, _, seen = _documents(case)
        S, L, HG = case["S"], case["L"], case["H"] * case["G"]
        at = np.clip(np.arange(S) + L - S, 0, L - 1)
        last = np.searchsorted(doc, doc[at], side="right")
        pairs = float(np.maximum(0, np.minimum(seen, last) - first[at]).sum()) * HG
        rows = HG * S * case["d"] * e * 4.0 + HG * S * 8.0  # q, out, dout, dq; lse, dlse
        return dict(bytes=rows + case["H"] * L * case["d"] * e * 4.0, flops=14.0 * case["d"] * pairs)
    if case["op"] == "chunk":
        length, cu, table, _ = _chunk(case)
        HG, T = case["H"] * case["G"], int(cu[-1])
        new = np.diff(cu)
        pairs = sum(float(n) * (x - n) + n * (n + 1) / 2.0 for n, x in zip(new, length)) * HG
        return dict(bytes=float(length.sum()) * case["H"] * case["d"] * e * 2 + T * HG * (2.0 * case["d"] * e + 4) + table.size * 4,
                    flops=4.0 * case["d"] * pairs)
    length, refs, table, asked = _pool(case)
    row = 2.0 * case["H"] * case["d"] * e  # one token's keys and values
    book = 8.0 * (case["rows"] + 1)
    if case["op"] == "append":
        moved = 2 * row * int(asked["cu"][-1])
    elif case["op"] == "fork":
        src = asked["src"][asked["src"] >= 0]
        moved = 2 * row * float((length[src] % case["page"]).sum())
        book += 16.0 * float((-(-length[src] // case["page"])).sum())
    else:
        used = int((refs > 0).sum())
        moved = 2 * row * case["page"] * float((refs[used:] > 0).sum())
        book += 8.0 * (refs.size + float((-(-length // case["page"])).sum()))
    return dict(bytes=moved + book, flops=0.0)


# -------------------------------------------------------------------------------------------------- the inputs
def _randn(g, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype) * scale


def _ints(a):
    return torch.tensor(np.ascontiguousarray(a), dtype=torch.int32, device="cuda")


def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, H, d = DTYPES[case["dtype"]], case["H"], case["d"]
    s = dict(case=case, scale=d ** -0.5, slopes=_slopes(H * case["G"]) if case.get("slopes") else None)
    if case["op"] == "train":
        doc, _, prefix, _ = _documents(case)
        S, L, HG = case["S"], case["L"], H * case["G"]
        s.update(q=_randn(g, (HG, S, d), dt, 1.5), k=_randn(g, (H, L, d), dt), v=_randn(g, (H, L, d), dt),
                 dout=_randn(g, (HG, S, d), dt), dlse=_randn(g, (HG, S), torch.float32, 0.1),
                 doc_k=_ints(doc) if case["docs"] > 1 else None,
                 doc_q=_ints(doc[np.clip(np.arange(S) + L - S, 0, L - 1)]) if case["docs"] > 1 else None,
                 prefix=_ints(prefix) if case["prefix"] else None)
        if own:
            from fast_memory_amd import ScoreTerms
            s["terms"] = ScoreTerms(case["cap"], s["slopes"], s["doc_q"], s["doc_k"], s["prefix"])
        return s
    if case["op"] == "chunk":
        length, cu, table, n = _chunk(case)
        refs = np.zeros(n, np.int64)
        refs[table[table >= 0]] = 1
        s.update(q=_randn(g, (int(cu[-1]), H * case["G"], d), dt, 1.5), cu=_ints(cu), max_new=int(np.diff(cu).max()),
                 prefix=_ints(np.full(case["rows"], case["prefix"])) if case["prefix"] else None)
    else:
        length, refs, table, asked = _pool(case)
        n = case["pages"]
        s.update({k: _ints(v) for k, v in asked.items()})
        if case["op"] == "append":
            s.update(k_new=_randn(g, (int(asked["cu"][-1]), H, d), dt), v_new=_randn(g, (int(asked["cu"][-1]), H, d), dt))
    s.update(k=_randn(g, (n, H, case["page"], d), dt), v=_randn(g, (n, H, case["page"], d), dt),
             book=_ints(np.concatenate([np.zeros(META, np.int64), length, refs, table.reshape(-1)])))
    R = case["rows"]
    s.update(length=s["book"][META:META + R], refs=s["book"][META + R:META + R + n],
             table=s["book"][META + R + n:].view(R, -1), saved=s["book"].clone())
    if own:
        from fast_memory_amd import PagedCache, ScoreTerms
        s["cache"] = PagedCache.over(s["k"], s["v"], s["book"], R)
        s["terms"] = ScoreTerms(case.get("cap", 0.0), s["slopes"], prefix=s.get("prefix"))
    return s


# ------------------------------------------------------------------------------------------------------ a pass
def run(s):
    op = s["case"]["op"]
    if op == "train":
        return _train_own(s) if own else _train(s)
    if op == "chunk":
        return _attend_own(s) if own else _attend(s)
    s["book"].copy_(s["saved"])  # as a program does that takes a step back: every pass starts from the same bookkeeping
    if own:
        if op == "append":
            s["cache"].append(s["k_new"], s["v_new"], s["cu"])
        elif op == "fork":
            s["cache"].drop(s["drop"])
            s["cache"].fork(s["src"])
        else:
            s["cache"].compact()
    else:
        {"append": _append, "fork": _fork, "compact": _compact}[op](s)
    return dict(k=s["k"], v=s["v"], length=s["length"], refs=s["refs"], table=s["table"])


def _train_own(s):
    from fast_memory_amd import local_attention_backward, ops
    out, lse = ops.local_attn_terms_fwd(s["q"], s["k"], s["v"], s["scale"], s["case"]["causal"], s["terms"])
    dq, dk, dv = local_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, s["scale"], s["case"]["causal"],
                                          terms=s["terms"], dlse=s["dlse"])
    return dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv)


def _attend_own(s):
    out, lse = s["cache"].attend(s["q"], s["cu"], s["scale"], terms=s["terms"], max_new=s["max_new"])
    return dict(out=out, lse=lse)


def _softmax(x):
    """Rows of probabilities and their log-sum-exp; a row of nothing but -inf gives zeros and the empty marker."""
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(x.sub_(m))
    z = p.sum(-1, keepdim=True)
    lse = torch.where(z > 0, m + torch.log(z), torch.full_like(m, EMPTY_LSE)).squeeze(-1)
    return p.div_(torch.where(z > 0, z, torch.ones_like(z))), lse


def _train(s):
    c = s["case"]
    H, G, S, L, d, cap = c["H"], c["G"], c["S"], c["L"], c["d"], c["cap"]
    dev, dt = s["q"].device, s["q"].dtype
    q, k, v, do = (s[n].float() for n in ("q", "k", "v", "dout"))
    q, do = q.view(H, G * S, d), do.view(H, G * S, d)
    at, j = torch.arange(S, device=dev) + (L - S), torch.arange(L, device=dev)
    seen = (at + 1).clamp(0, L) if c["causal"] else torch.full((S,), L, device=dev)
    if s["prefix"] is not None:
        seen = torch.maximum(seen, s["prefix"])
    ok = j[None, :] < seen[:, None]
    if s["doc_q"] is not None:
        ok = ok & (s["doc_q"][:, None] == s["doc_k"][None, :])
    x = torch.matmul(q, k.transpose(1, 2)).mul_(s["scale"])
    t = None
    if cap > 0:
        t = torch.tanh(x / cap)
        x = cap * t
    x = x.view(H, G, S, L)
    if s["slopes"] is not None:
        x = x - s["slopes"].view(H, G, 1, 1) * (at[:, None] - j[None, :]).abs().float()
    x = x.masked_fill(~ok, -math.inf)
    p, lse = _softmax(x)
    p = p.view(H, G * S, L)
    out = torch.matmul(p, v)
    dv = torch.matmul(p.transpose(1, 2), do)
    D = (do * out).sum(-1) - s["dlse"].view(H, G * S)
    ds = torch.matmul(do, v.transpose(1, 2)).sub_(D[..., None]).mul_(p)
    if cap > 0:
        ds.mul_(1 - t * t)
    ds.mul_(s["scale"])
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(1, 2), q)
    shape = (H * G, S, d)
    return dict(out=out.view(shape).to(dt), lse=lse.view(H * G, S), dq=dq.view(shape).to(dt), dk=dk.to(dt), dv=dv.to(dt))


def _attend(s):
    c = s["case"]
    H, G, d, P, R, cap = c["H"], c["G"], c["d"], c["page"], c["rows"], c["cap"]
    dev, dt = s["q"].device, s["q"].dtype
    T, N, M = s["q"].shape[0], s["max_new"], s["table"].shape[1]
    page = s["table"].long().clamp(min=0)
    k, v = (x[page].float().permute(0, 2, 1, 3, 4).reshape(R, H, M * P, d) for x in (s["k"], s["v"]))
    start, new, length = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long(), s["length"].long()
    i, j = torch.arange(N, device=dev), torch.arange(M * P, device=dev)
    q = s["q"].float()[(start[:, None] + i).clamp(max=T - 1)].view(R, N, H, G, d).permute(0, 2, 3, 1, 4)
    at = (length - new)[:, None] + i  # R, N: the position of a row's i-th new token
    seen = at + 1
    if s["prefix"] is not None:
        seen = torch.maximum(seen, s["prefix"][:, None].long())
    ok = (j < torch.minimum(seen, length[:, None])[..., None])[:, None, None]
    x = torch.matmul(q.reshape(R, H, G * N, d), k.transpose(2, 3)).mul_(s["scale"]).view(R, H, G, N, M * P)
    if cap > 0:
        x = torch.tanh(x.div_(cap)).mul_(cap)
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, H, G, 1, 1) * (at[:, :, None] - j).abs().float()[:, None, None]
    p, lse = _softmax(x.masked_fill(~ok, -math.inf))
    v = v * (j < length[:, None])[:, None, :, None]  # what lies behind a row's end is nobody's
    out = torch.matmul(p.view(R, H, G * N, M * P), v).view(R, H, G, N, d).permute(0, 3, 1, 2, 4).reshape(R, N, H * G, d)
    lse = lse.permute(0, 3, 1, 2).reshape(R, N, H * G)
    row = torch.searchsorted(s["cu"][1:].contiguous(), torch.arange(T, device=dev, dtype=torch.int32), right=True)
    col = torch.arange(T, device=dev) - start[row]
    return dict(out=out[row, col].to(dt), lse=lse[row, col])


def _free_pages(refs):
    """Page numbers, the free ones first, each part ascending."""
    return torch.sort((refs != 0).to(torch.uint8), stable=True)[1]


def _append(s):
    P, R, dev = s["case"]["page"], s["case"]["rows"], s["k"].device
    length, refs, table, cu = s["length"], s["refs"], s["table"], s["cu"]
    T, M = s["k_new"].shape[0], table.shape[1]
    after = length + (cu[1:] - cu[:-1])
    m = torch.arange(M, device=dev)
    fresh = (m >= ((length + P - 1) // P)[:, None]) & (m < ((after + P - 1) // P)[:, None])
    rank = (fresh.view(-1).cumsum(0) - 1).clamp(min=0, max=refs.numel() - 1)
    page = _free_pages(refs)[rank].view(R, M)
    refs.scatter_add_(0, page.view(-1), fresh.view(-1).to(refs.dtype))
    table.copy_(torch.where(fresh, page.to(table.dtype), table))
    t = torch.arange(T, device=dev, dtype=torch.int32)
    row = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    at = length[row] + t - cu[row]
    to = table[row, (at // P).long()].long()
    slot = (at % P).long()
    s["k"][to, :, slot] = s["k_new"]
    s["v"][to, :, slot] = s["v_new"]
    length.copy_(after)


def _fork(s):
    P, R, dev = s["case"]["page"], s["case"]["rows"], s["k"].device
    length, refs, table = s["length"], s["refs"], s["table"]
    M = table.shape[1]
    # drop: the first pages of a row leave it
    have = (length + P - 1) // P
    n = torch.minimum(s["drop"].clamp(min=0), have)
    m = torch.arange(M, device=dev)
    gone = m < n[:, None]
    refs.scatter_add_(0, table.clamp(min=0).long().view(-1), -gone.view(-1).to(refs.dtype))
    at = m + n[:, None]
    moved = table.gather(1, at.clamp(max=M - 1).long())
    table.copy_(torch.where(at < have[:, None], moved, torch.full_like(table, -1)))
    length.copy_((length - n * P).clamp(min=0))
    # fork: whole pages are shared, a last partial one is copied
    src = s["src"].long()
    takes, of = src >= 0, src.clamp(min=0)
    part = takes & (length[of] % P != 0)
    rank = (part.cumsum(0) - 1).clamp(min=0)
    to = _free_pages(refs)[rank]
    full = length[of] // P
    shared = takes[:, None] & (m < full[:, None])
    refs.scatter_add_(0, table[of].clamp(min=0).long().view(-1), shared.view(-1).to(refs.dtype))
    refs.scatter_add_(0, to, part.to(refs.dtype))
    own_page = (part[:, None] & (m == full[:, None]))
    old = table[of].gather(1, full.long().clamp(max=M - 1)[:, None]).clamp(min=0).view(-1).long()
    table.copy_(torch.where(shared, table[of], torch.where(own_page, to[:, None].to(table.dtype), table)))
    slot = torch.arange(P, device=dev)
    row, slot = (part[:, None] & (slot < (length[of] % P)[:, None])).nonzero(as_tuple=True)  # the rows to copy
    for x in (s["k"], s["v"]):
        x[to[row], :, slot] = x[old[row], :, slot]
    length.copy_(torch.where(takes, length[of], length))


def _compact(s):
    dev, refs, table = s["k"].device, s["refs"], s["table"]
    n = refs.numel()
    used = refs > 0
    count = used.sum()
    at = torch.arange(n, device=dev)
    hole, mover = ~used & (at < count), used & (at >= count)
    holes, movers = (torch.sort((~x).to(torch.uint8), stable=True)[1] for x in (hole, mover))
    moves = int(mover.sum())  # the copies need a shape
    to, of = holes[:moves], movers[:moves]
    new = at.clone()
    new[of] = to
    for x in (s["k"], s["v"]):
        x[to] = x[of]
    refs[to] = refs[of]
    refs[of] = 0
    table.copy_(torch.where(table >= 0, new[table.clamp(min=0).long()].to(table.dtype), table))


# ------------------------------------------------------------------------- the same from the definition, 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"train": _exact_train, "chunk": _exact_chunk}.get(case["op"], _exact_pool)(s)


def _exact_scores(q, k, scale, cap, slope, at, seen):
    """Scores [n, L] of the queries at positions `at`, -inf where not seen, and the derivative of the cap."""
    x = (q @ k.T) * scale
    slack = torch.ones_like(x)
    if cap > 0:
        y = torch.tanh(x / cap)
        x, slack = cap * y, 1 - y * y
    x = x - slope * (at[:, None] - torch.arange(k.shape[0], device=k.device)).abs()
    return torch.where(seen, x, torch.full_like(x, -math.inf)), slack


def _exact_train(s):
    c = s["case"]
    G, S, L, d = c["G"], c["S"], c["L"], c["d"]
    doc, _, _, lim = _documents(c)
    dev = s["q"].device
    at = torch.arange(S, device=dev) + (L - S)
    doc = torch.tensor(doc, device=dev)
    seen = torch.arange(L, device=dev)[None] < torch.tensor(lim, device=dev)[:, None]
    seen &= doc[at.clamp(0, L - 1)][:, None] == doc[None]
    res = {n: [] for n in ("out", "lse", "dq")}
    dk, dv = (torch.zeros((c["H"], L, d), dtype=torch.float64, device=dev) for _ in range(2))
    for h in range(c["H"] * G):
        q, do, k, v = s["q"][h].double(), s["dout"][h].double(), s["k"][h // G].double(), s["v"][h // G].double()
        slope = float(s["slopes"][h]) if s["slopes"] is not None else 0.0
        x, slack = _exact_scores(q, k, s["scale"], c["cap"], slope, at, seen)
        lse = torch.logsumexp(x, 1)
        some = lse > -math.inf
        p = torch.where(seen, torch.exp(x - torch.where(some, lse, torch.zeros_like(lse))[:, None]), torch.zeros_like(x))
        out = p @ v
        g = p * (do @ v.T - (do * out).sum(1, keepdim=True) + s["dlse"][h].double()[:, None]) * slack * s["scale"]
        res["out"].append(out)
        res["lse"].append(torch.where(some, lse, torch.full_like(lse, EMPTY_LSE)))
        res["dq"].append(g @ k)
        dk[h // G] += g.T @ q
        dv[h // G] += p.T @ do
    return dict({n: torch.stack(v) for n, v in res.items()}, dk=dk, dv=dv)


def _exact_chunk(s):
    c = s["case"]
    G, dev = c["G"], s["q"].device
    cu, length, table = s["cu"].tolist(), s["length"].tolist(), s["table"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=dev)
    for r, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        n = length[r]
        pages = torch.tensor([p for p in table[r] if p >= 0], device=dev)
        k, v = (x[pages].transpose(0, 1).reshape(c["H"], -1, c["d"])[:, :n].double() for x in (s["k"], s["v"]))
        at = torch.arange(n - (b - a), n, device=dev)
        seen = torch.arange(n, device=dev)[None] < torch.clamp(at + 1, min=c["prefix"])[:, None]
        for h in range(c["H"] * G):
            slope = float(s["slopes"][h]) if s["slopes"] is not None else 0.0
            x, _ = _exact_scores(s["q"][a:b, h].double(), k[h // G], s["scale"], c["cap"], slope, at, seen)
            z = torch.logsumexp(x, 1)
            lse[a:b, h] = z
            out[a:b, h] = torch.exp(x - z[:, None]) @ v[h // G]
    return dict(out=out, lse=lse)


def _exact_pool(s):
    c = s["case"]
    P = c["page"]
    length, refs, table = s["length"].tolist(), s["refs"].tolist(), s["table"].tolist()
    rows = [[p for p in t if p >= 0] for t in table]
    writes = []  # ((page, slots), source pool or None, (page, slots) or token range)
    if c["op"] == "append":
        cu = s["cu"].tolist()
        for r in range(c["rows"]):
            for t in range(cu[r], cu[r + 1]):
                if length[r] % P == 0:
                    page = refs.index(0)
                    refs[page] = 1
                    rows[r].append(page)
                writes.append((rows[r][length[r] // P], length[r] % P, t))
                length[r] += 1
        if writes:
            page, slot, t = (torch.tensor(x, device=s["k"].device) for x in zip(*writes))
            for x, y in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
                x[page, :, slot] = y[t]
    elif c["op"] == "fork":
        for r, n in enumerate(s["drop"].tolist()):
            for _ in range(min(max(n, 0), len(rows[r]))):
                refs[rows[r].pop(0)] -= 1
                length[r] = max(0, length[r] - P)
        src = s["src"].tolist()
        for r in range(c["rows"]):
            if src[r] >= 0:
                length[r] = length[src[r]]
                whole = length[r] // P
                rows[r] = rows[src[r]][:whole]
                if length[r] % P:
                    page = refs.index(0)
                    refs[page] = 1
                    rows[r].append(page)
                    writes.append((page, rows[src[r]][whole], length[r] % P))
        for r in range(c["rows"]):
            if src[r] >= 0:
                for page in rows[r][:length[r] // P]:
                    refs[page] += 1
        for to, of, n in writes:
            for x in (s["k"], s["v"]):
                x[to, :, :n] = x[of, :, :n]
    else:
        used = [p for p in range(len(refs)) if refs[p]]
        holes = [p for p in range(len(used)) if not refs[p]]
        moved = dict(zip([p for p in used if p >= len(used)], holes))
        rows = [[moved.get(p, p) for p in t] for t in rows]
        for of, to in moved.items():
            refs[to], refs[of] = refs[of], 0
        if moved:
            of, to = (torch.tensor(list(x), device=s["k"].device) for x in (moved.keys(), moved.values()))
            for x in (s["k"], s["v"]):
                x[to] = x[of]
    dev = s["k"].device
    table = [t + [-1] * (s["table"].shape[1] - len(t)) for t in rows]
    return dict(k=s["k"], v=s["v"], **{n: torch.tensor(x, dtype=torch.int32, device=dev)
                                       for n, x in (("length", length), ("refs", refs), ("table", table))})
