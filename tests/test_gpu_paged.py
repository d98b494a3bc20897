"""The paged cache of local keys: its bookkeeping against lists of pages, its rows against the tokens that went in, and
the attention over it against the plain 64-bit form (bounds derived in oracle/local_side.py)."""
import random

import pytest
import torch

from fast_memory_amd import Memory, MemoryBatch, PagedCache, ScoreTerms, fit_projection, ops
from oracle import local_side as O
from tests.test_gpu_local_terms import close
from tests.util import gen

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def cu_of(counts):
    c = [0]
    for n in counts:
        c.append(c[-1] + n)
    return i32(c)


def same_book(cache, model, what):
    torch.cuda.synchronize()
    assert cache.length.tolist() == model.length, f"{what}: length"
    assert cache.refs.tolist() == model.refs, f"{what}: refs"
    assert cache.table.tolist() == model.table(), f"{what}: table"


class Both:
    """A cache on the GPU beside its model; `rows[r]` = the tokens row r should hold, as numbers."""

    def __init__(self, R, n_pages, P, H, d, dtype, width, seed):
        self.cache = PagedCache(R, n_pages, P, H, d, dtype, max_tokens=width * P)
        self.model = O.Cache(R, n_pages, P, width)
        self.H, self.d, self.dtype, self.g, self.tokens = H, d, dtype, gen(seed), []
        self.rows = [[] for _ in range(R)]

    def append(self, counts):
        T = sum(counts)
        k, v = (torch.randn(T, self.H, self.d, generator=self.g).to(self.dtype) for _ in range(2))
        self.cache.append(k.cuda(), v.cuda(), cu_of(counts))
        if self.model.append(counts) is None:
            return False
        at = 0
        for r, n in enumerate(counts):
            self.rows[r] += range(len(self.tokens) + at, len(self.tokens) + at + n)
            at += n
        self.tokens += list(zip(k, v))
        return True

    def fork(self, src):
        self.cache.fork(i32(src))
        if self.model.fork(src) is None:
            return False
        before = [list(r) for r in self.rows]
        for r, s in enumerate(src):
            if s >= 0:
                self.rows[r] = before[s]
        return True

    def drop(self, pages):
        self.cache.drop(i32(pages))
        self.model.drop(pages)
        for r, n in enumerate(pages):
            if n > 0:
                self.rows[r] = self.rows[r][n * self.model.P:]

    def compact(self):
        self.cache.compact()
        self.model.compact()

    def kv(self, r):
        """What row r should hold, [H, length, d]."""
        if not self.rows[r]:
            return torch.zeros(2, self.H, 0, self.d, dtype=self.dtype)
        return torch.stack([torch.stack([self.tokens[t][i] for t in self.rows[r]], 1) for i in range(2)])

    def same_rows(self, what):
        same_book(self.cache, self.model, what)
        for r in range(len(self.rows)):
            n = self.model.length[r]
            pages = torch.tensor(self.model.rows[r], dtype=torch.long)
            want = self.kv(r)
            for x, w in zip((self.cache.k_pages, self.cache.v_pages), want):
                got = x.cpu()[pages].transpose(0, 1).reshape(self.H, -1, self.d)[:, :n]
                assert torch.equal(got, w), f"{what}: row {r}"


@pytest.mark.parametrize("dtype,P,H,d", [(torch.bfloat16, 16, 2, 128), (torch.float16, 4, 1, 6), (torch.float32, 1, 2, 5),
                                         (torch.bfloat16, 8, 3, 64), (torch.bfloat16, 2, 1, 1)])
def test_a_life_of_requests(dtype, P, H, d):
    rng = random.Random(int(P * 100 + d))
    R, width, n_pages = 6, 7, 23
    b = Both(R, n_pages, P, H, d, dtype, width, 5)
    refused = 0
    for step in range(60):
        do = rng.choice(["append", "append", "append", "fork", "drop", "compact"])
        if do == "append":
            refused += not b.append([rng.choice([0, 0, 1, 1, P, rng.randrange(3 * P + 1)]) for _ in range(R)])
        elif do == "fork":
            full = [r for r in range(R) if b.model.length[r]]
            src = [-1] * R
            for r in range(R):
                if not b.model.length[r] and full and rng.random() < 0.7:
                    src[r] = rng.choice(full)
            refused += not b.fork(src)
        elif do == "drop":
            b.drop([rng.choice([0, 0, -3, 1, 2, 1 << 30]) for _ in range(R)])
        else:
            b.compact()
        same_book(b.cache, b.model, f"step {step} {do}")
    b.same_rows("at the end")
    assert int(b.cache.book[0]) == refused
    if refused:
        with pytest.raises(RuntimeError, match="refused"):
            b.cache.check()
    b.cache.check()


def test_many_rows_and_pages():
    """More rows than a workgroup has threads, more pages than a round of its search looks at."""
    R, n_pages, P, width = 1500, 20011, 4, 24
    b = Both(R, n_pages, P, 1, 8, torch.bfloat16, width, 7)
    rng = random.Random(3)
    assert b.append([rng.randrange(0, 50) for _ in range(R)])
    same_book(b.cache, b.model, "append")
    b.drop([1 << 30 if r % 3 == 0 else r % 5 for r in range(R)])
    same_book(b.cache, b.model, "drop")
    assert b.fork([r - 1 if r % 3 == 0 and r else -1 for r in range(R)])
    same_book(b.cache, b.model, "fork")
    assert b.append([rng.randrange(0, 40) for _ in range(R)])
    same_book(b.cache, b.model, "append 2")
    b.compact()
    b.same_rows("compact")


def test_refused_calls_change_nothing():
    b = Both(3, 5, 4, 1, 8, torch.float32, 4, 9)
    assert b.append([7, 0, 6])                                  # 2 + 2 pages of 5
    before = b.cache.book.clone()
    pages = b.cache.k_pages.clone()
    c = b.cache
    k = torch.randn(16, 1, 8, device="cuda")
    wrong = [lambda: c.append(k, k, cu_of([0, 8, 0])),            # two pages, one is free
             lambda: c.append(k, k, cu_of([10, 0, 0])),           # five pages for a row of four
             lambda: c.append(k, k, i32([0, 5, 3, 5])),           # not ascending
             lambda: c.append(k, k, i32([1, 5, 6, 7])),           # not from 0
             lambda: c.append(k, k, i32([0, 1, 1, 17])),          # beyond the tokens given
             lambda: c.append(k, k, i32([0, -5, 0, 1])),
             lambda: c.fork(i32([-1, 3, -1])),                    # no such row
             lambda: c.fork(i32([2, -1, -1])),                    # into a row that holds tokens
             lambda: c.fork(i32([-1, 1, -1]))]                    # from itself
    for i, f in enumerate(wrong):
        f()
        torch.cuda.synchronize()
        assert int(c.book[0]) == i + 1, i
        assert torch.equal(c.book[16:], before[16:]) and torch.equal(c.k_pages, pages), i
    assert int(c.book[1]) == 1
    with pytest.raises(RuntimeError, match="9 call"):
        c.check()
    assert b.append([1, 0, 2])
    assert b.fork([-1, 0, -1])
    same_book(c, b.model, "after")
    # a copy of a partial page needs a page, and there is none; a fork from a row that is forked into is refused
    b.drop([0, 1 << 30, 0])
    assert b.append([0, 0, 3])                                  # 8 and 11 tokens: pages 2 + 0 + 3
    assert not b.fork([-1, 2, -1])
    with pytest.raises(RuntimeError, match="fewer free pages"):
        c.check()
    b.drop([1 << 30, 0, 0])
    assert not b.fork([1, 2, -1])
    with pytest.raises(RuntimeError, match="forked into"):
        c.check()
    same_book(c, b.model, "at the end")


def test_strided_tokens_and_rows_behind_the_last():
    H, d, P = 3, 64, 16
    both = torch.randn(40, 2, H, d, device="cuda").to(torch.bfloat16)      # keys and values of a token side by side
    c = PagedCache(2, 8, P, H, d)
    c.k_pages.fill_(7.0)
    c.append(both[:, 0], both[:, 1], i32([0, 5, 21]))                      # tokens 21 .. 39 are nobody's
    c.check()
    t = c.table.tolist()
    assert c.length.tolist() == [5, 16] and t[0][0] == 0 and t[1][0] == 1
    assert torch.equal(c.k_pages[0, :, :5].transpose(0, 1), both[:5, 0])
    assert torch.equal(c.v_pages[1].transpose(0, 1), both[5:21, 1])
    assert (c.k_pages[0, :, 5:] == 7).all() and (c.k_pages[2:] == 7).all()
    heads_first = both[:, 0].transpose(0, 1).contiguous().transpose(0, 1)
    c.append(heads_first, heads_first, cu_of([0, 3]))
    assert torch.equal(c.k_pages[2, :, :3].transpose(0, 1), both[:3, 0])


# ------------------------------------------------------------------------------------------- attention
def attend_case(seed, lengths, new, H, G, d, P, dtype, t, perm=True, heads_first=False, max_new=0, scale_q=1.0, dirty=None):
    R = len(lengths)
    M = max(1, max(-(-n // P) for n in lengths))
    n_pages = sum(-(-n // P) for n in lengths) + 3
    g = gen(seed)
    order = torch.randperm(n_pages, generator=g).tolist() if perm else list(range(n_pages))
    k, v = (torch.randn(n_pages, H, P, d, generator=g).to(dtype) for _ in range(2))
    rows, at = [], 0
    for n in lengths:
        rows.append(order[at:at + -(-n // P)])
        at += len(rows[-1])
    if dirty is not None:                                   # what lies behind a row's end, and in free pages
        for x in (k, v):
            for r, n in zip(rows, lengths):
                if n % P:
                    x[r[-1], :, n % P:] = dirty
            x[order[at:]] = dirty
    book = torch.zeros(16 + R + n_pages + R * M, dtype=torch.int32)
    book[16:16 + R] = torch.tensor(lengths)
    for p in order[:at]:
        book[16 + R + p] = 1
    table = torch.full((R, M), -1, dtype=torch.int32)
    for r, pages in enumerate(rows):
        table[r, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
    book[16 + R + n_pages:] = table.view(-1)
    T = sum(new)
    q = (torch.randn(T, H * G, d, generator=g) * scale_q).to(dtype)
    cache = PagedCache.over(k.cuda(), v.cuda(), book.cuda(), R)
    gq = q.cuda()
    if heads_first:
        gq = gq.transpose(0, 1).contiguous().transpose(0, 1)
    terms = ScoreTerms(**{n: x.cuda() if torch.is_tensor(x) else x for n, x in t.items()})
    cu = cu_of(new)
    out, lse = cache.attend(gq, cu, d ** -0.5, terms, max_new)
    start = 0
    for r, (n, m) in enumerate(zip(lengths, new)):
        if m == 0:
            continue
        kr, vr = (x[torch.tensor(rows[r], dtype=torch.long)].transpose(0, 1).reshape(H, -1, d)[:, :n] for x in (k, v))
        pre = None if "prefix" not in t else t["prefix"][r].expand(m)
        for h in range(H * G):
            slope = float(t["slopes"][h]) if "slopes" in t else 0.0
            if n == 0:
                assert (out[start:start + m, h] == 0).all() and (lse[start:start + m, h] == O.EMPTY).all()
                continue
            f = O.attention(q[start:start + m, h], kr[h // G], vr[h // G], d ** -0.5, O.seen_mask(m, n, True, pre),
                            t.get("softcap", 0.0), slope, t=dtype)
            close(out[start:start + m, h], f["out"], f["out_tol"], f"row {r} head {h} out")
            close(lse[start:start + m, h], f["lse"], f["lse_tol"], f"row {r} head {h} lse")
        start += m
    return cache, gq, cu, terms, out, lse


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("H,G,d,P", [(2, 4, 128, 16), (1, 8, 64, 32), (2, 1, 256, 16), (1, 3, 128, 128), (2, 2, 128, 4), (1, 5, 72, 8)])
def test_single_tokens(dtype, H, G, d, P):
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 130, 333]
    attend_case(21, lengths, [1] * len(lengths), H, G, d, P, dtype, {}, max_new=1)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lengths,new", [([5], [5]), ([64], [64]), ([100, 200], [37, 1]), ([300, 1, 0, 257], [129, 1, 0, 200]),
                                         ([40, 500], [0, 17]), ([3], [8]), ([700], [2])])
@pytest.mark.parametrize("d,P,G", [(128, 16, 4), (64, 64, 2), (128, 32, 1)])
def test_chunks(dtype, lengths, new, d, P, G):
    attend_case(22, lengths, new, 2, G, d, P, dtype, {}, max_new=max(new))
    attend_case(23, lengths, new, 1, G, d, P, dtype, {}, heads_first=True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 40], [150, 9, 1]])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_paged_terms(dtype, new, d):
    g = gen(31)
    lengths = [150, 77, 401]
    for cap, slopes, prefix in ((8.0, False, False), (0.0, True, False), (0.0, False, True), (20.0, True, True)):
        t = dict(softcap=cap)
        if slopes:
            t["slopes"] = torch.rand(8, generator=g) * 0.3
        if prefix:
            t["prefix"] = torch.tensor([120, 500, 0], dtype=torch.int32)
        attend_case(24, lengths, new, 2, 4, d, 16, dtype, t, scale_q=3.0)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dirty", [float("nan"), float("inf")])
@pytest.mark.parametrize("new", [[1, 1, 1], [20, 1, 90]])
def test_what_lies_behind_a_row_is_nobodys(dtype, dirty, new):
    attend_case(25, [133, 9, 250], new, 1, 4, 128, 32, dtype, {}, dirty=dirty)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("new", [[5], [70]])
def test_a_later_token_does_not_reach_an_earlier_one(dtype, new):
    cache, q, cu, terms, out, lse = attend_case(26, [200], new, 1, 2, 128, 16, dtype, {})
    page, slot = int(cache.table[0, 199 // 16]), 199 % 16
    cache.v_pages[page, :, slot] = float("nan")
    out2, lse2 = cache.attend(q, cu, 128 ** -0.5, terms)
    # (that tile goes another way: equal up to the rounding of its result and of its probabilities)
    a, b = out[:-1].float(), out2[:-1].float()
    assert torch.isfinite(b).all() and (a - b).abs().max() <= 4 * torch.finfo(dtype).eps * a.abs().max()
    assert torch.isnan(out2[-1]).all()


def test_long_rows_are_split_and_joined():
    # one sequence, few rows: the keys are split over many workgroups
    for dtype, n, m, t in ((torch.bfloat16, 9000, 1, {}), (torch.float16, 7001, 3, dict(softcap=20.0)),
                           (torch.bfloat16, 5000, 20, dict(slopes=torch.tensor([0.5, 0.01])))):
        attend_case(27, [n], [m], 1, 2, 128, 64, dtype, t, max_new=m)
    attend_case(28, [6000, 3], [1, 1], 1, 2, 128, 16, torch.float32, {})


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 2, 33, 50]])
def test_short_rows_beside_a_long_one(dtype, new):
    # the pieces are cut by the widest row: a short row has fewer tiles of keys than pieces, some of its pieces have none
    attend_case(32, [5200, 2, 130, 300], new, 1, 2, 64, 16, dtype, {}, max_new=max(new))
    attend_case(33, [5200, 70, 1025, 65], new, 1, 1, 128, 32, dtype, dict(softcap=20.0))


def test_a_single_token_beside_a_long_prompt():
    """The prompt's blocks fill the card and stay whole, the single token's long row is cut into pieces."""
    H, G, d, P, dtype = 64, 1, 64, 64, torch.bfloat16
    lengths, new = [2100, 5200, 0], [2100, 1, 0]
    g = gen(35)
    k, v = (torch.randn(120, H, P, d, generator=g).to(dtype) for _ in range(2))
    cache = PagedCache(3, 120, P, H, d, dtype)
    cache.k_pages.copy_(k), cache.v_pages.copy_(v)
    pages = torch.randperm(120, generator=g)
    rows = [pages[:33], pages[33:115], pages[:0]]
    for r, at in enumerate(rows):
        cache.table[r, :len(at)] = at.int().cuda()
    cache.length.copy_(i32(lengths))
    q = torch.randn(sum(new), H, d, generator=g).to(dtype)
    out, lse = cache.attend(q.cuda(), cu_of(new), d ** -0.5)
    for r, start, tokens in ((0, 0, [0, 1, 127, 128, 1500, 2099]), (1, 2100, [0])):
        n, m = lengths[r], new[r]
        kr, vr = (x[rows[r]].transpose(0, 1).reshape(H, -1, d)[:, :n] for x in (k, v))
        seen = O.seen_mask(m, n, True, None)[tokens]
        at = torch.tensor(tokens) + start
        for h in range(0, H, 7):
            f = O.attention(q[at, h], kr[h], vr[h], d ** -0.5, seen, 0.0, 0.0, t=dtype)
            close(out[at.cuda(), h], f["out"], f["out_tol"], f"row {r} head {h} out")
            close(lse[at.cuda(), h], f["lse"], f["lse_tol"], f"row {r} head {h} lse")


def test_bad_page_numbers_stay_inside_the_pool():
    cache, q, cu, terms, out, lse = attend_case(29, [100, 70], [1, 30], 1, 2, 128, 16, torch.bfloat16, {})
    cache.table[0, 2] = 1 << 30
    cache.table[1, 0] = -7
    cache.length[1] = 1 << 30
    out, lse = cache.attend(q, cu, 0.1, terms)
    torch.cuda.synchronize()
    assert torch.isfinite(out.float()).all()


def test_tokens_of_no_row():
    cache, q, cu, terms, out, lse = attend_case(30, [40, 50], [3, 4], 1, 2, 64, 16, torch.bfloat16, {})
    more = torch.cat([q, q])
    o, l = cache.attend(more, cu, 64 ** -0.5, terms)
    assert torch.equal(o[:7], out) and torch.equal(l[:7], lse)
    assert (o[7:] == 0).all() and (l[7:] == O.EMPTY).all()
    o, l = cache.attend(q[:0], i32([0, 0, 0]), 1.0)
    assert o.shape == (0, 2, 64) and l.shape == (0, 2)


def test_tokens_in_front_of_the_first_row():
    cache, q, cu, terms, out, lse = attend_case(34, [40, 50], [3, 4], 1, 2, 64, 16, torch.bfloat16, {})
    o, l = cache.attend(torch.cat([q[:2], q]), cu + 2, 64 ** -0.5, terms)
    assert torch.equal(o[2:], out) and torch.equal(l[2:], lse)
    assert (o[:2] == 0).all() and (l[:2] == O.EMPTY).all()


def test_a_decoding_run_over_a_forked_cache_and_a_memory():
    """Prompt, fork, decode, drop what the memory takes over, compact: every step against the plain form, merged with the
    memory's attention; the batch of memories takes the same path."""
    H, G, d, P, dtype = 2, 4, 128, 16, torch.bfloat16
    b = Both(4, 64, P, H, d, dtype, 16, 41)
    g = gen(42)
    keys, vals = (torch.randn(4, H, 300, d, generator=g).to(dtype).cuda() for _ in range(2))
    mems = [Memory.build(keys[i], vals[i], fit_projection(keys[i], 8), 64) for i in range(4)]
    batch = MemoryBatch(mems)
    assert b.append([50, 0, 33, 0])
    assert b.fork([-1, 0, -1, 2])
    for step in range(5):
        if step == 2:
            b.drop([1, 0, 2, 0])
        if step == 3:
            b.compact()
        assert b.append([1, 1, 1, 1])
        q = torch.randn(4, H, G, d, generator=g).to(dtype).cuda()
        out, lse = batch.attend_with_cache(q, b.cache, d ** -0.5)
        one, one_lse = mems[1].attend_with_cache(q[1].clone(), b.cache, 1, d ** -0.5, G)
        assert torch.allclose(out[1], one, atol=2e-2, rtol=1e-2) and torch.allclose(lse[1], one_lse, atol=1e-3)
        kl, vl = (torch.zeros(4, H, 64, d, dtype=dtype) for _ in range(2))
        for r in range(4):
            kv = b.kv(r)
            n = kv.shape[2]
            o, l = mems[r].attend_with_local(q[r], kv[0].cuda(), kv[1].cuda(), d ** -0.5, G)
            # the merged result in fp32 from two parts rounded to bf16 each way: two half steps of each and of p
            assert (o - out[r]).abs().max() <= 4 * 2.0 ** -8 * max(1.0, o.abs().max()) and (l - lse[r]).abs().max() < 1e-3
    b.same_rows("after the run")


def test_replays_of_a_captured_decode_step():
    """append and attend recorded once: every replay writes the next token and sees one key more."""
    H, G, d, P, dtype, R = 2, 4, 128, 16, torch.bfloat16, 3
    g = gen(51)
    make = lambda: PagedCache(R, 40, P, H, d, dtype, max_tokens=160)
    prompt = torch.randn(60, H, d, generator=g).to(dtype).cuda()
    steps = [(torch.randn(R, H * G, d, generator=g).to(dtype).cuda(), torch.randn(R, H, d, generator=g).to(dtype).cuda()) for _ in range(20)]
    a, e = make(), make()
    for c in (a, e):
        c.append(prompt, prompt, i32([0, 15, 31, 60]))
    cu = i32([0, 1, 2, 3])
    q, k = steps[0][0].clone(), steps[0][1].clone()

    def step(c, q, k):
        c.append(k, k, cu)
        return c.attend(q, cu, d ** -0.5, max_new=1)
    saved = a.snapshot()
    step(a, q, k)
    a.restore(saved)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step(a, q, k)
    for sq, sk in steps:
        q.copy_(sq)
        k.copy_(sk)
        graph.replay()
        torch.cuda.synchronize()
        o, l = step(e, sq, sk)
        assert torch.equal(out, o) and torch.equal(lse, l)
        assert torch.equal(a.book, e.book) and torch.equal(a.k_pages, e.k_pages)
    a.check()


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 elements: the pages at its end are written, forked, moved and read."""
    H, d, P, n_pages = 8, 128, 64, 70000                                     # 4.6e9 elements a pool, 9.2 GB
    c = PagedCache(2, n_pages, P, H, d, torch.bfloat16, max_tokens=4 * P)
    c.refs[:n_pages - 6] = 1                                                 # only the last pages are free
    k = torch.randn(150, H, d, device="cuda").to(torch.bfloat16)
    c.append(k, k, i32([0, 150, 150]))
    c.fork(i32([-1, 0]))
    c.check()
    assert c.table.tolist() == [[n_pages - 6, n_pages - 5, n_pages - 4, -1], [n_pages - 6, n_pages - 5, n_pages - 3, -1]]
    q = torch.randn(2, H * 2, d, device="cuda").to(torch.bfloat16)
    out, lse = c.attend(q, i32([0, 1, 2]), d ** -0.5, max_new=1)
    for r in range(2):
        for h in (0, 15):
            f = O.attention(q[r:r + 1, h].cpu(), k[:, h // 2].cpu(), k[:, h // 2].cpu(), d ** -0.5, torch.ones(1, 150, dtype=torch.bool),
                            t=torch.bfloat16)
            close(out[r:r + 1, h], f["out"], f["out_tol"], "out")
    c.refs[:n_pages - 6] = 0
    c.compact()
    assert c.table[:, :3].tolist() == [[0, 1, 2], [0, 1, 3]]
    again, _ = c.attend(q, i32([0, 1, 2]), d ** -0.5, max_new=1)
    assert torch.equal(out, again)
