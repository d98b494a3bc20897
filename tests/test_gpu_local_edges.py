"""The local side at its edges: what lies far below the largest score, tokens that a caller did not announce, infinities in
the last key, refusals around a snapshot, integers beyond 32 bits (bounds derived in oracle/local_side.py)."""
import pytest
import torch

from fast_memory_amd import PagedCache, ScoreTerms, ops
from oracle import local_side as O
from tests.test_gpu_local_terms import check, close, inputs, on_gpu, terms_of
from tests.test_gpu_paged import attend_case, cu_of, i32
from tests.util import gen

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


# ------------------------------------------------------------------ keys far below the largest score
def tail(seed, L, d, dtype, below, dominant=0):
    """One key at score 0 whose value is 0, and L - 1 keys `below` under it with values in [1/2, 1): their weights are small one by
    one and not together.  The query is the first unit vector times sqrt(d), so that the scale d^-1/2 leaves k's first element."""
    q = torch.zeros(d)
    q[0] = d ** 0.5
    k = torch.zeros(L, d)
    k[:, 0] = -below
    k[dominant] = 0
    v = 0.5 + 0.5 * torch.rand(L, d, generator=gen(seed)) * (1 - 2 ** -7)
    v[dominant] = 0
    return q.to(dtype), k.to(dtype), v.to(dtype)


def sum_tol(f, L):
    """The oracle's bound of the log-sum-exp leaves out the rounding of the sum itself.  A tile of at least 16 of a lane's keys is
    summed first (one of 32 keys, 8 of them a lane's, in the kernel for few rows, whose four waves take every fourth), then added:
    at most L / 32 + 32 additions of positive numbers follow one another, each off by 2^-24 of a sum that is at most the whole, and
    at most 64 pieces are joined.  The logarithm is off by the sum's relative error."""
    return f["lse_tol"] + (L / 32 + 96) * O.W


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("S,L,dominant", [(1, 65536, 0), (33000, 32768, 0), (33000, 32768, 20000)])
def test_a_long_tail_under_one_key(dtype, d, S, L, dominant):
    if dtype == torch.float32 and S > 1:
        S = 300
    q, k, v = tail(3, L, d, dtype, 17.5, dominant)
    out, lse = ops.local_attn_terms_fwd(q.expand(1, S, d).contiguous().cuda(), k[None].cuda(), v[None].cuda(), d ** -0.5, False)
    f = O.attention(q[None], k, v, d ** -0.5, torch.ones(1, L, dtype=torch.bool), t=dtype)
    assert f["out"].min() > 2 ** -11                        # (the tail is most of the answer)
    close(out[0], f["out"].expand(S, d), f["out_tol"].expand(S, d), "out")
    close(lse[0], f["lse"].expand(S), sum_tol(f, L).expand(S), "lse")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows,new,G", [(128, 1, 1), (128, 3, 4), (16, 80, 8)])
def test_a_long_tail_in_a_cache(dtype, d, rows, new, G):
    # all rows name the same pages; as many rows as it takes that a row's keys stay in one piece
    H, P, L = 8, 16, 32768
    if dtype == torch.float32:
        rows, new = 4, min(new, 4)
    q, k, v = tail(5, L, d, dtype, 17.5)
    pages = lambda x: x.view(L // P, 1, P, d).expand(L // P, H, P, d).contiguous().cuda()
    book = torch.zeros(16 + rows + L // P + rows * (L // P), dtype=torch.int32)
    book[16:16 + rows] = L
    book[16 + rows:16 + rows + L // P] = rows
    book[16 + rows + L // P:] = torch.arange(L // P, dtype=torch.int32).repeat(rows)
    c = PagedCache.over(pages(k), pages(v), book.cuda(), rows)
    out, lse = c.attend(q.expand(rows * new, H * G, d).contiguous().cuda(), cu_of([new] * rows), d ** -0.5, max_new=new)
    f = O.attention(q[None].expand(new, d), k, v, d ** -0.5, O.seen_mask(new, L, True), t=dtype)
    whole = lambda x: x.unsqueeze(1).expand(new, H * G, *x.shape[1:]).repeat(rows, *[1] * x.dim())
    close(out, whole(f["out"]), whole(f["out_tol"]), "out")
    close(lse, whole(f["lse"]), whole(sum_tol(f, L)), "lse")


# ------------------------------------------------------------------ values that are not finite
def one_row(seed, n, new, H, G, d, P, dtype):
    """A cache of one row of n tokens in order, and queries of its last `new`."""
    g = gen(seed)
    k, v = (torch.randn(n, H, d, generator=g).to(dtype) for _ in range(2))
    c = PagedCache(1, -(-n // P), P, H, d, dtype)
    q = torch.randn(new, H * G, d, generator=g).to(dtype)
    return c, k, v, q


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("G,new,max_new", [(16, 2, 1), (32, 2, 1), (16, 3, 2), (8, 5, 1), (1, 40, 3), (16, 2, 2), (16, 2, 0), (32, 4, 0)])
@pytest.mark.parametrize("n", [100, 128, 1100])
def test_more_new_tokens_than_announced(dtype, G, new, max_new, n):
    """max_new shapes the launch only: with too small a one the results are right, and a later token's NaN stays out of earlier ones."""
    H, d, P = 2, 64, 16
    c, k, v, q = one_row(11, n, new, H, G, d, P, dtype)
    v[-1] = float("nan")
    c.append(k.cuda(), v.cuda(), i32([0, n]))
    out, lse = c.attend(q.cuda(), i32([0, new]), d ** -0.5, max_new=max_new)
    for h in range(H * G):
        f = O.attention(q[:, h], k[:, h // G], v[:, h // G], d ** -0.5, O.seen_mask(new, n, True), t=dtype)
        f["out_tol"] = f["out_tol"].nan_to_num(0)
        close(out[:-1, h], f["out"][:-1], f["out_tol"][:-1], f"head {h} out")
        close(lse[:, h], f["lse"], f["lse_tol"], f"head {h} lse")
    assert torch.isnan(out[-1]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,new,G", [(1, 1, 4), (33, 1, 4), (97, 1, 1), (100, 3, 4), (100, 60, 2), (1500, 1, 8)])
def test_an_infinite_value_in_the_last_key(dtype, d, n, new, G):
    # the last token sees it and comes out infinite, where its probability is not zero: no NaN from the places behind it
    H, P = 1, 16
    c, k, v, q = one_row(13, n, new, H, G, d, P, dtype)
    v[-1, :, ::2] = float("inf")
    v[-1, :, 1::4] = -float("inf")
    c.append(k.cuda(), v.cuda(), i32([0, n]))
    out, _ = c.attend(q.cuda(), i32([0, new]), d ** -0.5, max_new=new)
    assert torch.equal(out[-1], v[-1].cuda().expand(G, d)) if n == 1 else \
        torch.equal(out[-1][:, ~torch.isfinite(v[-1, 0])].cpu(), v[-1][:, ~torch.isfinite(v[-1, 0])].expand(G, -1))
    finite = torch.isfinite(v[-1, 0])
    assert torch.isfinite(out[-1][:, finite]).all() and torch.isfinite(out[:-1]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_gradient_that_is_not_finite_is_not_lost(dtype, d):
    """Key 7 weighs nothing (its score is 1e4 under the others'), and D of every query that sees it is not finite: its gradient is 0
    times that, in a tile with masked places as in one without.  Queries that see no such value keep theirs."""
    S = 40
    g = gen(17)
    q, k, v, do = (torch.randn(1, S, d, generator=g).to(dtype) for _ in range(4))
    q[..., 0] = d ** 0.5
    k[..., 0] = 0
    k[:, 7, 0] = -1e4
    v[:, 7:9] = float("inf")
    q, k, v, do = (x.cuda() for x in (q, k, v, do))
    out, lse = ops.local_attn_terms_fwd(q, k, v, d ** -0.5, True)
    dq, dk, dv = ops.local_attn_terms_bwd(do, q, k, v, out, lse, d ** -0.5, True)
    assert not torch.isfinite(dk[0, 7]).any() and torch.isfinite(dq[0, :7]).all() and not torch.isfinite(dq[0, 8:]).any()


# ------------------------------------------------------------------ the cache
def test_a_refusal_outlives_a_restore():
    c = PagedCache(2, 3, 4, 1, 8, torch.float32)
    k = torch.randn(16, 1, 8, device="cuda")
    c.append(k, k, i32([0, 4, 5]))
    saved = c.snapshot()
    c.append(k, k, i32([0, 9, 9]))                           # a fourth page for a row of three
    c.restore(saved)
    assert c.length.tolist() == [4, 1]
    with pytest.raises(RuntimeError, match="1 call.*outgrow its table"):
        c.check()
    # and one that was told about is not told again
    c.append(k, k, i32([0, 9, 9]))
    saved = c.snapshot()
    with pytest.raises(RuntimeError, match="1 call"):
        c.check()
    c.append(k, k, i32([0, 1, 2]))
    c.restore(saved)
    c.check()
    assert c.length.tolist() == [4, 1] and c.table.tolist() == [[0, -1, -1], [1, -1, -1]] and c.refs.tolist() == [1, 1, 0]
    c.append(k, k, i32([0, 2, 3]))                           # the page that came back is found again
    c.check()
    assert c.table.tolist() == [[0, 2, -1], [1, -1, -1]]
    with pytest.raises(ValueError, match="no snapshot"):
        c.restore(saved[:1])


def test_integers_beyond_32_bits():
    """int64 arguments: what does not fit 32 bits does not come back as another number."""
    i64 = lambda x: torch.tensor(x, dtype=torch.int64, device="cuda")
    H, d, P = 1, 64, 4
    c = PagedCache(2, 8, P, H, d, torch.float32)
    k, v = (torch.randn(6, H, d, generator=gen(21)).cuda() for _ in range(2))
    c.append(k, v, i64([0, (1 << 32) + 1, 1 << 33]))          # (as 32 bits: 0, 1, 0 and 0, 1, ..)
    c.fork(i64([1 << 32, -1]))                               # (from row 0)
    with pytest.raises(RuntimeError, match="2 call"):
        c.check()
    assert c.length.tolist() == [0, 0] and c.refs.sum() == 0
    c.append(k, v, i64([0, 6, 6]))
    q = torch.randn(2, H, d, generator=gen(22)).cuda()
    want = c.attend(q, i32([0, 2, 2]), 0.1, ScoreTerms(prefix=i32([6, 0])))
    got = c.attend(q, i64([0, 2, 2]), 0.1, ScoreTerms(prefix=i64([1 << 40, -(1 << 40)])))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    c.drop(i64([1 << 40, -(1 << 32) + 1]))
    c.check()
    assert c.length.tolist() == [0, 0] and c.refs.sum() == 0
    x = torch.randn(1, 5, d, generator=gen(23)).cuda()
    doc = [0, 0, -(1 << 32), 0, 0]                             # (as 32 bits: 0, no padding)
    a = ops.local_attn_terms_fwd(x, x, x, 0.1, True, ScoreTerms(doc_q=i64(doc), doc_k=i64(doc)))
    b = ops.local_attn_terms_fwd(x, x, x, 0.1, True, ScoreTerms(doc_q=i32([0, 0, -1, 0, 0]), doc_k=i32([0, 0, -1, 0, 0])))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_a_row_near_2_to_the_31_tokens():
    """The page count of a row whose last page ends behind 2^31 - 1."""
    P, width = 4096, 1 << 19
    c = PagedCache(1, 4, P, 1, 8, torch.bfloat16, max_tokens=width * P)
    c.length.fill_((width - 1) * P)                           # all but one page of the table, as if they were held
    k = torch.randn(3, 1, 8, generator=gen(25)).to(torch.bfloat16).cuda()
    c.append(k[:1], k[:1], i32([0, 1]))
    c.append(k[1:], k[1:], i32([0, 2]))
    c.check()
    assert c.length.tolist() == [(width - 1) * P + 3] and c.table[0, -2:].tolist() == [-1, 0] and c.refs.tolist() == [1, 0, 0, 0]
    assert torch.equal(c.k_pages[0, 0, :3], k[:, 0])
    c.append(k[:1].expand(P - 4, 1, 8), k[:1].expand(P - 4, 1, 8), i32([0, P - 4]))
    c.check()
    c.append(k[:1], k[:1], i32([0, 1]))                       # 2^31
    with pytest.raises(RuntimeError, match="outgrow"):
        c.check()
    c.drop(i32([width - 1]))
    assert c.length.tolist() == [P - 1] and c.table[0, :2].tolist() == [0, -1]
    c.drop(i32([1]))
    assert c.length.tolist() == [0] and c.refs.tolist() == [0, 0, 0, 0]


def test_no_gradient_is_dropped_in_silence():
    c = PagedCache(1, 2, 16, 1, 64)
    k = torch.randn(3, 1, 64, device="cuda").to(torch.bfloat16)
    c.append(k, k, i32([0, 3]))
    q = k[:1].clone().requires_grad_()
    with pytest.raises(ValueError, match="no backward"):
        c.attend(q, i32([0, 1]), 0.1)
    with torch.no_grad():
        a = c.attend(q, i32([0, 1]), 0.1)
    b = c.attend(q.detach(), i32([0, 1]), 0.1)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------ rows without new tokens
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("G,active", [(1, {37: 1}), (4, {69: 1}), (4, {0: 1, 1: 1, 64: 2, 69: 1}), (2, {5: 40, 6: 1, 66: 1}), (8, {3: 3, 12: 20, 68: 1}),
                                      (1, {i: 1 for i in range(0, 70, 2)}), (2, {10: 70}), (1, {20: 33, 64: 33, 65: 1, 66: 3}), (1, {1: 66, 69: 5})])
def test_few_rows_with_tokens_among_many(dtype, G, active):
    """70 rows of which a few have new tokens, long and short ones: fewer tokens than rows, as many, more."""
    lengths = [(37 * r) % 90 for r in range(70)]
    for at, r in enumerate(active):
        lengths[r] = max(active[r], (5200, 33, 700, 64)[at % 4])
    new = [active.get(r, 0) for r in range(70)]
    attend_case(37, lengths, new, 2, G, 64, 16, dtype, {}, max_new=max(new))
    attend_case(38, lengths, new, 1, G, 64, 16, dtype, dict(softcap=20.0), heads_first=True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_offsets_that_do_not_fit_stay_inside(dtype):
    """cu that does not ascend, or leaves the tokens there are: some result, and nothing outside of it is touched."""
    cache, q, cu, terms, out, lse = attend_case(39, [40] * 9, [0, 0, 3, 0, 0, 0, 1, 0, 0], 1, 2, 64, 16, dtype, {})
    for bad in ([9, 8, 7, 6, 5, 4, 3, 2, 1, 0], [0, 1 << 30, -5, 4, 1 << 30, 0, 0, 2, 4, 1 << 30], [4] * 10, [-3] * 10, [0] * 9 + [1 << 30]):
        whole = torch.full((8, 2, 64), 7.0, dtype=q.dtype, device="cuda")
        whole[2:6] = q
        o, l = cache.attend(whole[2:6], i32(bad), 0.1)
        torch.cuda.synchronize()
        assert o.shape == (4, 2, 64) and (whole[:2] == 7).all() and (whole[6:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("front,back", [(0, 700), (300, 0), (257, 1000), (0, 0), (1, 1)])
def test_a_padded_batch(dtype, heads_first, front, back):
    """Tokens of no row on both sides: empty, whatever lay there, and the rows' results as without them."""
    cache, q, cu, terms, out, lse = attend_case(40, [40, 50, 0], [3, 40, 0], 2, 3, 64, 16, dtype, {}, heads_first=heads_first)
    pad = lambda n: torch.full((n, 6, 64), float("nan"), dtype=dtype, device="cuda")
    more = torch.cat([pad(front), q, pad(back)])
    if heads_first:
        more = more.transpose(0, 1).contiguous().transpose(0, 1)
    torch.empty(1 << 24, device="cuda").fill_(float("nan"))    # (what the results' memory holds beforehand)
    o, l = cache.attend(more, cu + front, 64 ** -0.5)
    mine = slice(front, front + 43)
    # (the number of pieces follows the number of tokens: equal up to the rounding of the result and of the probabilities)
    assert (o[mine].float() - out.float()).abs().max() <= 4 * torch.finfo(dtype).eps * out.float().abs().max()
    assert (l[mine] - lse).abs().max() < 1e-5
    for part in (slice(0, front), slice(front + 43, None)):
        assert (o[part] == 0).all() and (l[part] == O.EMPTY).all()


# ------------------------------------------------------------------ fp32 products in pieces
FP32_PRODUCTS = [(torch.float32, 64), (torch.float32, 128), (torch.float32, 256), (torch.bfloat16, 96), (torch.float16, 80), (torch.float32, 37)]


@pytest.mark.parametrize("dtype,d", FP32_PRODUCTS, ids=str)
@pytest.mark.parametrize("H,G,S,L,cap,slopes,docs,prefix,causal", [
    (1, 8, 300, 300, 0.0, False, 0, 0, True), (1, 8, 301, 450, 20.0, True, 0, 0, True), (2, 5, 270, 270, 0.0, False, 4, 0, True),
    (1, 3, 333, 200, 0.0, True, 0, 150, True), (1, 6, 257, 511, 15.0, False, 3, 40, False), (1, 1, 1500, 40, 0.0, False, 0, 0, False),
    (1, 16, 33, 33, 5.0, True, 2, 9, True), (1, 40, 3, 700, 0.0, False, 0, 0, True)])
def test_few_blocks_in_pieces(dtype, d, H, G, S, L, cap, slopes, docs, prefix, causal):
    """Too few blocks of queries, or of keys, for the card: the others' tiles are cut into pieces, across heads as well."""
    check(121, H, G, S, L, d, dtype, causal, terms_of(14, H, G, S, L, cap, slopes, docs, prefix, pad=7 if docs else 0))


@pytest.mark.parametrize("dtype,d", FP32_PRODUCTS, ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_pieces_of_queries_with_masked_places_that_are_not_finite(dtype, d, bad):
    H, G, S, L = 1, 7, 290, 150
    q, k, v, do, dl = inputs(123, H, G, S, L, d, dtype)
    doc_q, doc_k = torch.zeros(S, dtype=torch.int32), torch.zeros(L, dtype=torch.int32)
    doc_q[20:40], doc_q[200:230], doc_q[280:] = 1, 2, -1
    doc_k[40:50], doc_k[149:] = 1, -1
    t = dict(doc_q=doc_q, doc_k=doc_k, softcap=10.0)
    scale = d ** -0.5
    want, tol = O.local(q, k, v, scale, False, dout=do, dlse=dl, **t)
    for x in (q, do):                                       # document 2 has no keys, document 1's rows are finite
        x[:, 200:230], x[:, 280:] = bad, bad
    dl[:, 200:230], dl[:, 280:] = bad, bad
    for x in (k, v):
        x[:, 149:] = bad
    gq, gk, gv, gdo, gdl = (x.cuda() for x in (q, k, v, do, dl))
    out, lse = ops.local_attn_terms_fwd(gq, gk, gv, scale, False, on_gpu(t))
    got = ops.local_attn_terms_bwd(gdo, gq, gk, gv, out, lse, scale, False, on_gpu(t), gdl)
    for n, x in zip(("out", "lse", "dq", "dk", "dv"), (out, lse) + got):
        close(x, want[n], tol[n], n)
    again = ops.local_attn_terms_bwd(gdo, gq, gk, gv, out, lse, scale, False, on_gpu(t), gdl)
    for x, y in zip(got, again):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("S,L,t", [(9000, 40, {}), (6000, 129, dict(softcap=20.0)), (1, 40000, {}), (3, 33000, dict(softcap=20.0))])
def test_a_single_block_in_many_pieces(dtype, d, S, L, t):
    """One block of keys under many queries, and of queries over many keys: up to 64 pieces."""
    check(131, 1, 1, S, L, d, dtype, S < L, t)


# ------------------------------------------------------------------ replays
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_replays_follow_which_rows_have_tokens(dtype):
    """attend recorded once over a cache of 70 rows: every replay finds the rows that have tokens then, and the padding."""
    R, H, G, d, P, T = 70, 2, 4, 64, 16, 40
    g = gen(141)
    n = 40
    k, v = (torch.randn(n, H, P, d, generator=g).to(dtype).cuda() for _ in range(2))
    c = PagedCache.over(k, v, torch.zeros(16 + R + n + R * 30, dtype=torch.int32, device="cuda"), R)
    c.length.copy_(i32([(53 * r) % 480 + 1 for r in range(R)]))
    c.table.copy_(torch.randint(0, n, (R, 30), generator=g).int())
    q = torch.randn(T, H * G, d, generator=g).to(dtype).cuda()
    new = [{3: 1, 69: 2}, {0: 40}, {r: 1 for r in range(0, 40)}, {10: 9, 11: 1, 50: 20, 68: 3}, {}, {69: 1}]
    cus = [cu_of([x.get(r, 0) for r in range(R)]) for x in new]
    cu = cus[0].clone()
    c.attend(q, cu, 0.125)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = c.attend(q, cu, 0.125)
    for at in (1, 2, 3, 4, 5, 0, 3):
        cu.copy_(cus[at])
        graph.replay()
        torch.cuda.synchronize()
        o, l = c.attend(q, cus[at], 0.125)
        assert torch.equal(out, o) and torch.equal(lse, l), at
        # a token sees something if it is some row's and lies at a position of 0 or more (row 0 holds one key under 40 new tokens)
        sees = [p >= 0 for r in range(R) for p in range((53 * r) % 480 + 1 - new[at].get(r, 0), (53 * r) % 480 + 1)]
        sees = torch.tensor(sees + [False] * (T - len(sees)), device="cuda")
        assert (out[~sees] == 0).all() and (lse[~sees] == O.EMPTY).all() and (lse[sees] > -1e30).all(), at
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.float32, 256), (torch.bfloat16, 96), (torch.float16, 64)], ids=str)
def test_replays_of_a_step_in_pieces(dtype, d):
    H, G, S, L = 1, 4, 300, 420
    data = [tuple(x.cuda() for x in inputs(151 + i, H, G, S, L, d, dtype)) for i in range(3)]
    terms = on_gpu(terms_of(16, H, G, S, L, 15.0, True, 3, 30))

    def step(q, k, v, do, dl):
        out, lse = ops.local_attn_terms_fwd(q, k, v, 0.09, True, terms)
        return (out, lse) + ops.local_attn_terms_bwd(do, q, k, v, out, lse, 0.09, True, terms, dl)
    held = tuple(x.clone() for x in data[0])
    step(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held)
    for i in (1, 2, 0, 1):
        for h, x in zip(held, data[i]):
            h.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, step(*data[i])):
            assert torch.equal(x, y)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("size", [1e-3, 3e-2])
def test_the_log_sum_exp_of_small_scores(dtype, d, size):
    """Scores near 0 over one key: the log-sum-exp is the score.  Beside its bound an exponent against the maximum is rounded once, which
    fp16 holds 12 off (half a step of 12 is 2^-21), and the logarithm of the sum by as much again."""
    S = 64
    g = gen(161)
    q, k, v = ((torch.randn(1, n, d, generator=g) * s).to(dtype) for n, s in ((S, size), (1, 1.0), (1, 1.0)))
    f = O.attention(q[0], k[0], v[0], d ** -0.5, torch.ones(S, 1, dtype=torch.bool), t=dtype)
    more = 2 * 2.0 ** -21 if dtype == torch.float16 else 0.0
    out, lse = ops.local_attn_terms_fwd(q.cuda(), k.cuda(), v.cuda(), d ** -0.5, False)
    close(lse[0], f["lse"], f["lse_tol"] + more, "lse")
    close(out[0], f["out"], f["out_tol"], "out")
    c = PagedCache(S, S, 16, 1, d, dtype)
    c.append(k[0, 0].expand(S, 1, d).contiguous().cuda(), v[0, 0].expand(S, 1, d).contiguous().cuda(), i32(list(range(S + 1))))
    out, lse = c.attend(q[0][:, None].cuda(), i32(list(range(S + 1))), d ** -0.5, max_new=1)
    close(lse[:, 0], f["lse"], f["lse_tol"] + more, "lse")
    close(out[:, 0], f["out"], f["out_tol"], "out")
