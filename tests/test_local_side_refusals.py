"""Refusals of the paged cache, the attention over it and the local attention with score terms: by status code before
anything is launched, and by the Python layer."""
import pytest
import torch

from fast_memory_amd import _lib

p = 4096  # never dereferenced


def test_cache_status_codes():
    lib = _lib.load()
    ws = lib.fm_cache_workspace(8, 2)
    assert lib.fm_cache_book_ints(8, 2, 4) == 16 + 2 + 8 + 8 and lib.fm_cache_book_ints(0, 2, 4) == 0
    ok = (p, p, p, 8, 2, 4, 16, 1, 64, p, p, 64, 64, 64, 64, p, 3, 1, p, ws, None)
    for at, bad, rc in ((0, None, 1), (2, None, 1), (3, 0, 1), (4, 0, 1), (5, 0, 1), (6, 3, 1), (6, 0, 1), (6, 8192, 1), (7, 0, 1),
                        (8, 0, 1), (8, 257, 1), (9, None, 1), (15, None, 1), (16, -1, 1), (17, 5, 1), (18, None, 1), (19, ws - 1, 3)):
        a = list(ok)
        a[at] = bad
        assert lib.fm_cache_append(*a) == rc, at
        assert b"fm_cache_append" in lib.fm_last_error()
    ok = (p, p, p, 8, 2, 4, 16, 1, 64, p, 1, p, ws, None)
    for at, bad, rc in ((1, None, 1), (6, 5, 1), (9, None, 1), (10, 3, 1), (11, None, 1), (12, ws - 1, 3)):
        a = list(ok)
        a[at] = bad
        assert lib.fm_cache_fork(*a) == rc, at
    assert lib.fm_cache_drop(None, 8, 2, 4, 16, p, None) == 1 and lib.fm_cache_drop(p, 8, 2, 4, 16, None, None) == 1
    assert lib.fm_cache_drop(p, 8, 2, 4, 7, p, None) == 1
    assert lib.fm_cache_compact(p, p, p, 8, 2, 4, 16, 1, 64, 1, None, ws, None) == 1
    assert lib.fm_cache_compact(p, p, p, 8, 2, 4, 16, 1, 64, 1, p, ws - 1, None) == 3


def test_attention_status_codes():
    lib = _lib.load()
    nan, inf = float("nan"), float("inf")
    # q k v out lse | cap slopes doc_q doc_k prefix | H G S L d | scale causal dtype ws bytes stream
    fws = lib.fm_local_attn_terms_fwd_workspace(2, 2, 10, 10, 64, 1)
    ok = (p, p, p, p, p, 0.0, None, None, None, None, 2, 2, 10, 10, 64, 0.1, 1, 1, p, fws, None)
    for at, bad, rc in ((0, None, 1), (4, None, 1), (5, -1.0, 1), (5, nan, 1), (5, inf, 1), (5, 1e-40, 1), (7, p, 1), (8, p, 1),
                        (10, 0, 1), (11, 0, 1), (12, 0, 1), (13, 0, 1), (14, 0, 1), (14, 300, 1), (15, 0.0, 1), (15, -1.0, 1),
                        (15, nan, 1), (17, 9, 1), (18, None, 1), (10, 40000, 2), (12, (1 << 24) + 1, 2), (13, (1 << 24) + 1, 2)):
        a = list(ok)
        a[at] = bad
        assert lib.fm_local_attn_terms_fwd(*a) == rc, (at, bad)
        assert b"fm_local_attn_terms_fwd" in lib.fm_last_error()
    bws = lib.fm_local_attn_terms_bwd_workspace(2, 2, 10, 10, 64, 1)
    assert bws >= 2 * 2 * 10 * 4
    ok = (p,) * 6 + (None, p, p, p, 0.0, None, None, None, None, 2, 2, 10, 10, 64, 0.1, 1, 1, p, bws, None)
    for at, bad, rc in ((0, None, 1), (5, None, 1), (7, None, 1), (9, None, 1), (10, -2.0, 1), (12, p, 1), (19, 0, 1), (20, inf, 1),
                        (23, None, 1), (24, bws - 1, 3)):
        a = list(ok)
        a[at] = bad
        assert lib.fm_local_attn_terms_bwd(*a) == rc, (at, bad)
    # q st sh k v book | n_pages rows width page | cu out st sh lse st sh | T max_new H G d | scale cap slopes prefix dtype ws ..
    pws = lib.fm_paged_attn_fwd_workspace(2, 3, 1, 2, 2, 64, 4, 16, 1)
    ok = (p, 256, 64, p, p, p, 8, 2, 4, 16, p, p, 256, 64, p, 4, 1, 3, 1, 2, 2, 64, 0.1, 0.0, None, None, 1, p, pws, None)
    for at, bad, rc in ((0, None, 1), (5, None, 1), (6, 0, 1), (7, 0, 1), (8, 0, 1), (9, 12, 1), (9, 8192, 1), (10, None, 1), (17, -1, 1),
                        (18, -1, 1), (19, 0, 1), (20, 0, 1), (21, 0, 1), (21, 257, 1), (22, nan, 1), (23, -1.0, 1), (26, 4, 1),
                        (27, None, 1), (8, 1 << 21, 2), (19, 40000, 2)):
        a = list(ok)
        a[at] = bad
        assert lib.fm_paged_attn_fwd(*a) == rc, (at, bad)
        assert b"fm_paged_attn_fwd" in lib.fm_last_error()
    a = list(ok)
    a[17] = 0
    assert lib.fm_paged_attn_fwd(*a) == 0          # no token: nothing to do


def test_python_refusals():
    from fast_memory_amd import PagedCache, ScoreTerms, ops
    x = torch.zeros(2, 4, 64)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        ops.local_attn_terms_fwd(x, x, x, 1.0)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        PagedCache(1, 4, 16, 1, 64, device="cpu")
    with pytest.raises(ValueError):
        PagedCache(0, 4, 16, 1, 64, device="cpu")
    assert ScoreTerms() == (0.0, None, None, None, None)


@pytest.mark.gpu
def test_python_refusals_on_the_gpu():
    from fast_memory_amd import PagedCache, ScoreTerms, local_attention, local_attention_backward, ops
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    q, k = bf(4, 10, 64), bf(2, 12, 64)
    fwd = lambda *a, **t: ops.local_attn_terms_fwd(*a, 0.1, True, ScoreTerms(**t))
    ints = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")
    for bad in (lambda: fwd(q[0], k, k), lambda: fwd(bf(3, 10, 64), k, k), lambda: fwd(q, k, k.half()), lambda: fwd(q, k, bf(2, 11, 64)),
                lambda: fwd(q, k, k, slopes=torch.zeros(3, device="cuda")), lambda: fwd(q, k, k, slopes=torch.zeros(4, device="cuda").half()),
                lambda: fwd(q, k, k, slopes=torch.zeros(4)), lambda: fwd(q, k, k, doc_q=ints(10)), lambda: fwd(q, k, k, prefix=ints(12)),
                lambda: fwd(q, k, k, doc_q=ints(10), doc_k=ints(10)), lambda: fwd(q, k, k, doc_q=ints(10).float(), doc_k=ints(12)),
                lambda: fwd(q, k, k, softcap=-1.0), lambda: ops.local_attn_terms_fwd(q, k, k, 0.0),
                lambda: local_attention(q, k, k, 0.1, True, ScoreTerms(slopes=torch.zeros(4, device="cuda", requires_grad=True))),
                lambda: local_attention_backward(q, q, k, k, q, torch.zeros(4, 10, device="cuda"), 0.1, True, staged=True, terms=ScoreTerms()),
                lambda: ops.local_attn_terms_bwd(bf(4, 9, 64), q, k, k, q, torch.zeros(4, 10, device="cuda"), 0.1)):
        with pytest.raises(ValueError):
            bad()
    c = PagedCache(2, 4, 16, 2, 64)
    t, cu = bf(3, 2, 64), ints(3)
    for bad in (lambda: c.append(t, t, ints(2)), lambda: c.append(t, t[:2], cu), lambda: c.append(t.half(), t.half(), cu),
                lambda: c.append(bf(3, 1, 64), bf(3, 1, 64), cu), lambda: c.append(t, t, cu.float()), lambda: c.append(t.cpu(), t.cpu(), cu),
                lambda: c.fork(ints(3)), lambda: c.drop(ints(1)), lambda: c.free(torch.zeros(3, dtype=torch.bool, device="cuda")),
                lambda: c.attend(bf(3, 3, 64), cu, 0.1), lambda: c.attend(bf(3, 4, 32), cu, 0.1), lambda: c.attend(bf(3, 4, 64), ints(2), 0.1),
                lambda: c.attend(bf(3, 4, 64), cu, 0.1, ScoreTerms(doc_q=ints(3), doc_k=ints(3))), lambda: c.attend(bf(3, 4, 64), cu, -1.0),
                lambda: c.attend(bf(3, 4, 64), cu, 0.1, ScoreTerms(prefix=ints(3))), lambda: c.attend(bf(3, 4, 64), cu, 0.1, max_new=-1),
                lambda: PagedCache(2, 4, 12, 2, 64), lambda: PagedCache.over(c.k_pages, c.v_pages, c.book[:-1], 2),
                lambda: PagedCache.over(c.k_pages, c.v_pages.half(), c.book, 2)):
        with pytest.raises(ValueError):
            bad()
    c.check()


def test_a_long_prompt_beside_single_tokens_needs_no_large_workspace():
    lib = _lib.load()
    for dt in (_lib.FM_BF16, _lib.FM_F32):
        for rows, T, max_new in ((2, 8192, 0), (64, 8192, 0), (1, 8192, 1), (1, 8192, 8192), (2048, 2048, 1)):
            assert 0 < lib.fm_paged_attn_fwd_workspace(rows, T, max_new, 8, 8, 128, 4096, 16, dt) <= 100 << 20, (rows, T, max_new)
