"""Local attention with score terms (cap, distance bias, document and prefix masks), forward and backward, against the
plain 64-bit form; how far a kernel may be from it is derived in oracle/local_side.py."""
import math

import pytest
import torch

from fast_memory_amd import ScoreTerms, local_attention, local_attention_backward, ops
from oracle import local_side as O
from tests.util import gen

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def inputs(seed, H, G, S, L, d, dtype, scale_q=1.0):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    return ((r(H * G, S, d) * scale_q).to(dtype), r(H, L, d).to(dtype), r(H, L, d).to(dtype), r(H * G, S, d).to(dtype),
            r(H * G, S) * 0.3)


def terms_of(seed, H, G, S, L, cap, slopes, docs, prefix, pad=0):
    g = gen(seed)
    t = dict(softcap=cap)
    if slopes:
        t["slopes"] = torch.rand(H * G, generator=g) * 0.4
    if docs:
        cuts = torch.randint(0, max(L, 1), (docs - 1,), generator=g).sort()[0]
        doc = torch.searchsorted(cuts, torch.arange(L), right=True).int()
        if pad:
            doc[L - pad:] = -1
        at = (torch.arange(S) + L - S)
        t.update(doc_k=doc, doc_q=torch.where(at >= 0, doc[at.clamp(min=0)], torch.full((S,), -1, dtype=torch.int32)))
    if prefix:
        t["prefix"] = torch.randint(0, prefix + 1, (S,), generator=g).int()
    return t


def on_gpu(t):
    return ScoreTerms(**{k: v.cuda() if torch.is_tensor(v) else v for k, v in t.items()})


def close(got, want, tol, what):
    got = got.double().cpu()
    assert not torch.isnan(got).any(), f"{what}: NaN"
    over = (got - want).abs() - tol
    assert (over <= 0).all(), f"{what}: off by {(got - want).abs().flatten()[over.argmax()].item():.3e}, allowed " \
                              f"{tol.flatten()[over.argmax()].item():.3e}, {int((over > 0).sum())} of {over.numel()} values"


def check(seed, H, G, S, L, d, dtype, causal, t, backward=True, scale_q=1.0, data=None):
    q, k, v, do, dl = inputs(seed, H, G, S, L, d, dtype, scale_q) if data is None else data
    scale = d ** -0.5
    want, tol = O.local(q, k, v, scale, causal, dout=do if backward else None, dlse=dl, **t)
    gq, gk, gv, gdo, gdl = (x.cuda() for x in (q, k, v, do, dl))
    terms = on_gpu(t)
    out, lse = ops.local_attn_terms_fwd(gq, gk, gv, scale, causal, terms)
    close(out, want["out"], tol["out"], "out")
    close(lse, want["lse"], tol["lse"], "lse")
    if backward:
        got = ops.local_attn_terms_bwd(gdo, gq, gk, gv, out, lse, scale, causal, terms, gdl)
        for n, x in zip(("dq", "dk", "dv"), got):
            assert x.dtype == dtype
            close(x, want[n], tol[n], n)
    return out, lse


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("S,L", [(1, 1), (1, 77), (33, 33), (64, 200), (129, 129), (257, 300), (300, 140)])
@pytest.mark.parametrize("d", [64, 128])
def test_causal_extents(dtype, S, L, d):
    check(11 + S, 2, 2, S, L, d, dtype, True, {})


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [8, 40, 72, 96, 192, 256])
def test_head_dimensions(dtype, d):
    check(21 + d, 1, 3, 130, 150, d, dtype, True, terms_of(d, 1, 3, 130, 150, 15.0, True, 0, 0))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("cap,slopes,docs,prefix,causal", [
    (20.0, False, 0, 0, True), (0.0, True, 0, 0, True), (0.0, False, 4, 0, True), (0.0, False, 0, 90, True),
    (5.0, True, 3, 120, True), (8.0, True, 0, 0, False), (0.0, False, 5, 0, False), (30.0, True, 9, 40, True)])
@pytest.mark.parametrize("d", [64, 128])
def test_terms(dtype, cap, slopes, docs, prefix, causal, d):
    H, G, S, L = 2, 3, 205, 270
    check(31, H, G, S, L, d, dtype, causal, terms_of(5, H, G, S, L, cap, slopes, docs, prefix), scale_q=3.0)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_longer_rows(dtype):
    H, G, S, L = 1, 2, 700, 1100
    check(41, H, G, S, L, 128, dtype, True, terms_of(6, H, G, S, L, 30.0, True, 3, 200))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d,cap,slopes,docs,prefix,causal", [
    (64, 0.0, False, 0, 0, True), (128, 20.0, True, 3, 60, True), (256, 0.0, False, 5, 0, False), (64, 25.0, True, 0, 1900, True)])
def test_few_rows_over_many_keys(dtype, d, cap, slopes, docs, prefix, causal):
    # too few blocks of queries for the card: their keys are cut into pieces and joined
    H, G, S, L = 1, 2, 201, 2100
    check(43, H, G, S, L, d, dtype, causal, terms_of(12, H, G, S, L, cap, slopes, docs, prefix, pad=11 if docs else 0))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_pieces_with_masked_places_that_are_not_finite(dtype, d, bad):
    H, G, S, L = 1, 1, 70, 1300
    q, k, v, do, dl = inputs(44, H, G, S, L, d, dtype)
    doc_k = torch.zeros(L, dtype=torch.int32)
    doc_k[40:50], doc_k[600:640], doc_k[1299:] = 1, 1, -1
    t = dict(doc_q=torch.zeros(S, dtype=torch.int32), doc_k=doc_k, softcap=10.0)
    t["doc_q"][5] = -1
    scale = d ** -0.5
    want, tol = O.local(q, k, v, scale, False, dout=do, dlse=dl, **t)
    for x in (k, v):
        x[:, 40:50] = bad
        x[:, 600:640] = bad
        x[:, 1299:] = bad
    q[:, 5], do[:, 5], dl[:, 5] = bad, bad, bad
    gq, gk, gv, gdo, gdl = (x.cuda() for x in (q, k, v, do, dl))
    out, lse = ops.local_attn_terms_fwd(gq, gk, gv, scale, False, on_gpu(t))
    dq, dk, dv = ops.local_attn_terms_bwd(gdo, gq, gk, gv, out, lse, scale, False, on_gpu(t), gdl)
    seen = doc_k == 0
    for n, x, rows in (("out", out, slice(None)), ("lse", lse, slice(None)), ("dq", dq, slice(None)), ("dk", dk, seen), ("dv", dv, seen)):
        close(x[:, rows], want[n][:, rows], tol[n][:, rows], n)
    assert (dk[:, ~seen] == 0).all() and (dv[:, ~seen] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("cap", [1e-3, 0.05, 1.0, 300.0, 1e5, 1e20])
def test_caps_of_every_size(dtype, cap):
    # small caps bind every score, large ones none; both ends leave the range of the small-argument polynomial's coefficients
    check(46, 1, 2, 80, 100, 64, dtype, True, dict(softcap=cap))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_that_see_nothing_and_padding(dtype, d):
    # more queries than keys (the first see nothing), padding behind the last document, a document without keys
    H, G, S, L = 2, 2, 190, 150
    t = terms_of(7, H, G, S, L, 0.0, True, 3, 0, pad=37)
    t["doc_q"][60:70] = 77
    out, lse = check(51, H, G, S, L, d, dtype, True, t)
    nothing = ~O.seen_mask(S, L, True, None, t["doc_q"], t["doc_k"]).any(1)
    assert nothing[:40].all() and nothing[60:70].all()
    assert (out[:, nothing.cuda()] == 0).all() and (lse[:, nothing.cuda()] == O.EMPTY).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_masked_touches_nothing(dtype, d, bad):
    """NaN and infinities in padding, and in the rows of one document: nobody else's results may change."""
    H, G, S = 1, 2, 200
    q, k, v, do, dl = inputs(61, H, G, S, S, d, dtype)
    doc = torch.zeros(S, dtype=torch.int32)
    doc[90:120] = 1
    doc[170:] = -1
    t = dict(doc_q=doc, doc_k=doc)
    gt, scale = on_gpu(t), d ** -0.5

    def run(q, k, v, do, dl):
        q, k, v, do, dl = (x.cuda() for x in (q, k, v, do, dl))
        out, lse = ops.local_attn_terms_fwd(q, k, v, scale, True, gt)
        return (out, lse) + ops.local_attn_terms_bwd(do, q, k, v, out, lse, scale, True, gt, dl)
    clean = run(q, k, v, do, dl)
    want, tol = O.local(q, k, v, scale, True, dout=do, dlse=dl, **t)
    q2, k2, v2, do2, dl2 = (x.clone() for x in (q, k, v, do, dl))
    for x in (q2, k2, v2, do2):
        x[:, 95:118] = bad
        x[:, 180:] = bad
    dl2[:, 95:118] = bad
    dl2[:, 180:] = bad
    dirty = run(q2, k2, v2, do2, dl2)
    other = doc == 0
    for n, x, y in zip(("out", "lse", "dq", "dk", "dv"), dirty, clean):
        close(x[:, other], want[n][:, other], tol[n][:, other], n)
        pad = x[:, 170:]
        assert (pad == (O.EMPTY if n == "lse" else 0)).all(), f"{n}: padding"


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_later_key_does_not_reach_an_earlier_query(dtype):
    d, S = 128, 150
    q, k, v, do, dl = inputs(63, 1, 1, S, S, d, dtype)
    v2, k2 = v.clone(), k.clone()
    v2[:, 100], k2[:, 101] = float("nan"), float("inf")
    a = ops.local_attn_terms_fwd(q.cuda(), k.cuda(), v.cuda(), d ** -0.5, True)
    b = ops.local_attn_terms_fwd(q.cuda(), k2.cuda(), v2.cuda(), d ** -0.5, True)
    want, tol = O.local(q, k, v, d ** -0.5, True)
    close(b[0][:, :100], want["out"][:, :100], tol["out"][:, :100], "out")
    assert torch.isnan(b[0][:, 100:]).any(-1).all()
    close(a[0], want["out"], tol["out"], "out")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_large_and_small_scores(dtype, d):
    """Scores beyond the range of a naive exponential, with and without a cap; a lone far key under a steep bias."""
    check(71, 1, 2, 100, 180, d, dtype, True, {}, scale_q=40.0)
    check(72, 1, 2, 100, 180, d, dtype, True, dict(softcap=50.0), scale_q=40.0)
    doc_k = torch.zeros(900, dtype=torch.int32)
    doc_k[0] = 3
    doc_q = torch.full((64,), 3, dtype=torch.int32)
    check(73, 1, 1, 64, 900, d, dtype, True, dict(slopes=torch.tensor([2.0]), doc_q=doc_q, doc_k=doc_k))


@pytest.mark.parametrize("grad", [1e-7, 1.0, 3e4])
def test_fp16_gradients_keep_their_precision_at_any_scale(grad):
    H, G, S, d = 1, 2, 260, 64
    q, k, v, do, dl = inputs(81, H, G, S, S, d, torch.float16)
    do = do * (grad / 8)  # (the product with 3e4 first would be infinite)
    v = (v * 0.25).to(torch.float16)
    scale = d ** -0.5
    out, lse = ops.local_attn_terms_fwd(q.cuda(), k.cuda(), v.cuda(), scale, True)
    got = ops.local_attn_terms_bwd(do.cuda(), q.cuda(), k.cuda(), v.cuda(), out, lse, scale, True, None, None)
    want, tol = O.local(q, k, v, scale, True, dout=do)
    for n, x in zip(("dq", "dk", "dv"), got):
        # results below fp16's normal numbers are off by half its smallest step, 2^-25; above its largest they overflow
        t = tol[n] + 2.0 ** -25
        fits = want[n].abs() < 6.0e4
        close(torch.where(fits.cuda(), x, torch.zeros_like(x)), torch.where(fits, want[n], torch.zeros_like(want[n])), t, n)


def test_gradients_against_differences():
    H, G, S, L, d = 1, 2, 20, 27, 16
    q, k, v, do, dl = (x.double() for x in inputs(91, H, G, S, L, d, torch.float32))
    t = terms_of(8, H, G, S, L, 3.0, True, 2, 9)
    scale = d ** -0.5
    value = lambda q, k, v: sum(((w["out"] * do).sum() + (torch.where(w["lse"] > -1e30, w["lse"], torch.zeros_like(w["lse"])) * dl).sum())
                                for w in [O.local(q, k, v, scale, True, **t)[0]])
    g = lambda x: x.float().cuda().requires_grad_()
    gq, gk, gv = g(q), g(k), g(v)
    out, lse = local_attention(gq, gk, gv, scale, True, on_gpu(t))
    torch.autograd.backward((out, lse), (do.float().cuda(), dl.float().cuda()))
    eps = 1e-6
    rng = gen(92)
    for x, grad, at in ((q, gq.grad, 0), (k, gk.grad, 1), (v, gv.grad, 2)):
        for _ in range(12):
            i = int(torch.randint(0, x.numel(), (1,), generator=rng))
            args = [q, k, v]
            args[at] = x.clone()
            args[at].view(-1)[i] += eps
            hi = value(*args)
            args[at].view(-1)[i] -= 2 * eps
            lo = value(*args)
            # central difference: error ~ eps^2 and 2^-52 |value| / eps ~ 1e-8; the kernel's, fp32 sums of ~30 terms
            assert abs((hi - lo) / (2 * eps) - grad.view(-1)[i].item()) < 5e-5, (at, i)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_same_bits_every_time_and_on_another_stream(dtype):
    H, G, S, L, d = 2, 4, 333, 450, 128
    q, k, v, do, dl = (x.cuda() for x in inputs(95, H, G, S, L, d, dtype))
    terms = on_gpu(terms_of(9, H, G, S, L, 20.0, True, 3, 50))

    def run():
        out, lse = ops.local_attn_terms_fwd(q, k, v, 0.1, True, terms)
        return (out, lse) + ops.local_attn_terms_bwd(do, q, k, v, out, lse, 0.1, True, terms, dl)
    a = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = run()
    side.synchronize()
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_merged_with_a_memory_the_gradients_are_the_local_share():
    """out and lse merged with other keys: the gradients are those of the local keys inside the whole softmax."""
    H, G, S, L, d, dtype = 1, 2, 70, 90, 64, torch.float32
    q, k, v, do, _ = inputs(97, H, G, S, L + 40, d, dtype)
    scale = d ** -0.5
    t = dict(softcap=10.0)
    # the first 40 keys are the other part, seen by all queries; the rest is local and causal
    ok = O.seen_mask(S, L + 40, True)
    whole = [O.attention(q[h], k[0], v[0], scale, ok, 10.0, t=dtype) for h in range(G)]
    out = torch.stack([w["out"] for w in whole])
    lse = torch.stack([w["lse"] for w in whole])
    g = lambda x: x.float().cuda()
    dq, dk, dv = local_attention_backward(g(do), g(q), g(k[:, 40:]).contiguous(), g(v[:, 40:]).contiguous(), g(out), g(lse), scale,
                                          True, terms=ScoreTerms(**t))
    lok = O.seen_mask(S, L, True)
    for h in range(G):
        f = O.attention(q[h], k[0, 40:], v[0, 40:], scale, lok, 10.0, t=dtype)
        b = O.attention_backward(q[h], k[0, 40:], v[0, 40:], do[h], f, scale, lok, t=dtype, lse=lse[h], out=out[h])
        # (lse and out come rounded to fp32: p is off by another 2^-24 |lse| + .., within the four times of its bound)
        close(dq[h], b["dq"], b["dq_tol"], "dq")
        want, tol = (b, {n: b[n + "_tol"] for n in ("dk", "dv")}) if h == 0 else (
            {n: want[n] + b[n] for n in ("dk", "dv")}, {n: tol[n] + b[n + "_tol"] for n in ("dk", "dv")})
    for n, x in (("dk", dk), ("dv", dv)):
        close(x[0], want[n], tol[n] + O.W * want[n].abs(), n)


def test_terms_reach_the_module_forward_and_the_memory():
    from fast_memory_amd import Memory, fit_projection, merge, ring_cross_attention_approx
    H, G, S, N, C, Z, d, dtype = 2, 2, 96, 512, 8, 64, 128, torch.bfloat16
    g = gen(99)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    keys, vals, q, kl, vl = r(H, N, d), r(H, N, d), r(H, G * S, d), r(H, S, d), r(H, S, d)
    terms = on_gpu(terms_of(3, H, G, S, S, 20.0, True, 2, 0))
    mem = Memory.build(keys, vals, fit_projection(keys, C), Z)
    out, lse = mem.attend_with_local(q, kl, vl, d ** -0.5, G, terms=terms)
    lo, ll = ops.local_attn_terms_fwd(q.view(H * G, S, d), kl, vl, d ** -0.5, True, terms)
    want = merge(lo.reshape(H, G * S, d), ll.reshape(H, G * S), *mem.attend(q, d ** -0.5))
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    # the module forward: with the terms of nothing it gives the plain one's result to rounding, with terms another one
    q1, ks, vs = (x.reshape(1, -1, S, d).requires_grad_() for x in (q, kl, vl))
    k1, v1 = keys[None].clone().requires_grad_(), vals[None].clone().requires_grad_()
    kq = r(1, H * G, N, d)
    cent = torch.randn(C, d, generator=g).to(dtype).cuda()
    run = lambda **kw: ring_cross_attention_approx(q1, kq, ks, vs, k1, v1, cent, d ** -0.5, C, Z, centroid_topk=16, **kw)
    plain, none, some = run(), run(local_terms=ScoreTerms()), run(local_terms=terms)
    assert (plain - none).abs().max() <= 2 ** -6 * plain.abs().max()
    assert (plain - some).abs().max() > 2 ** -5 * plain.abs().max()
    do = torch.randn_like(plain)
    a = torch.autograd.grad(plain, (q1, ks, vs, k1, v1), do)
    b = torch.autograd.grad(none, (q1, ks, vs, k1, v1), do)
    for x, y in zip(a, b):
        assert (x.float() - y.float()).norm() <= 0.02 * x.float().norm()
    assert all(torch.isfinite(x).all() for x in torch.autograd.grad(some, (q1, ks, vs, k1, v1), do))


def test_saved_inputs_changed_in_place_are_caught():
    q, k, v, do, _ = (x.cuda() for x in inputs(101, 1, 1, 40, 40, 64, torch.bfloat16))
    doc = torch.zeros(40, dtype=torch.int32, device="cuda")
    q.requires_grad_()
    out, _ = local_attention(q, k, v, 0.125, True, ScoreTerms(doc_q=doc, doc_k=doc))
    doc.fill_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(do)


def test_replays_of_a_captured_step_follow_their_inputs():
    H, G, S, L, d, dtype = 2, 2, 150, 210, 128, torch.bfloat16
    data = [tuple(x.cuda() for x in inputs(111 + i, H, G, S, L, d, dtype)) for i in range(3)]
    terms = on_gpu(terms_of(4, H, G, S, L, 15.0, True, 3, 30))

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
