"""Plain 64-bit forms of the local side of the memory: attention with score terms and its gradients, attention over a
paged cache, and the cache's bookkeeping in lists.  Test infrastructure, CPU only.

Every form comes with how far a kernel may be from it.  The kernels hold scores, maxima, sums and accumulators in fp32
and round, besides each result, two things to the inputs' type t: the probabilities p in front of the product with the
values (and, in the backward, with dout), and g = p (dP - D) slack in front of the products with the keys and queries.
With u = finfo(t).eps / 2 a rounding is off by at most u |value|, so with w = 2^-24 (a rounding in fp32)

    x is off by       dx  = sm_scale (d + 2) w sum|q||k| + 8 w |x| (scaling, cap, bias) + c 2^-22 (the cap's tanh)
    p is off by       dp  = p (2 dx' + 4 w |x| ..) <= 4 max(dx) p         (its own x, the sum's, the exponentials)
    out is off by     u |out| + (u + 4 max(dx)) sum p |v| + (L + 4) w sum p |v|
    lse is off by     2 max(dx) + 8 w |lse|
    D is off by       u sum|do||out| + (d + 4) w sum|do||out| + w |dlse|   (it is formed from the rounded out)
    dP is off by      (d + 2) w sum|do||v|
    g is off by       u |g| + 4 max(dx) |g| + p slack (d(D) + d(dP)) + |p (dP - D)| d(slack)
    dq = sum g k      u |dq| + sum d(g) |k| + (L + 4) w sum|g||k|, and dk, dv likewise.
fp16 holds p and g times powers of two that keep its smallest normal number 2^-20 below the largest |p| = 1 and
2^-20 below the bound max|do| (max|v| + max|out|) of |g| or better: what falls below is off by at most 2^-30 of that.
A result below fp16's smallest normal number 2^-14 is a multiple of 2^-24: rounding it is off by at most 2^-25, whatever
u |value| says.  (First written without this; a dv of 2^-17 was then 2.07e-8 < 2^-25 = 2.98e-8 off.)
The hardware's exponential gives 0 for what is below fp32's smallest normal number, 2^-126: p is off by that much more, and
a result by that times the at most 2^14 terms of its sum and the at most 2^12 that |dP - D| |k| or |v| comes to in the
tests: 2^-100.  (First written without this; a dk of 5e-38 = 2^-124 was then missing.)"""
import torch

EMPTY = torch.finfo(torch.float32).min
W = 2.0 ** -24


def rounding(x, t):
    """How far the rounding of results x to type t is off."""
    u = torch.finfo(t).eps / 2 if t != torch.float32 else W
    return u * x.abs() + (2.0 ** -25 if t == torch.float16 else 2.0 ** -100)


def seen_mask(S, L, causal, prefix=None, doc_q=None, doc_k=None):
    at, j = torch.arange(S) + (L - S), torch.arange(L)
    lim = (at + 1).clamp(0, L) if causal else torch.full((S,), L)
    if prefix is not None:
        lim = torch.maximum(lim, prefix.long())
    ok = j[None] < lim.clamp(max=L)[:, None]
    if doc_q is not None:
        ok = ok & (doc_q[:, None] == doc_k[None]) & (doc_q[:, None] >= 0)
    return ok


def scores(q, k, scale, softcap, slope, at):
    raw = q @ k.T * scale
    x, slack = raw, torch.ones_like(raw)
    if softcap > 0:
        t = torch.tanh(raw / softcap)
        x, slack = softcap * t, 1 - t * t
    dist = (at[:, None] - torch.arange(k.shape[0])[None]).abs().double()
    x = x - slope * dist
    dx = scale * (q.shape[1] + 2) * W * (q.abs() @ k.abs().T) + 8 * W * (raw.abs() + slope * dist)
    if softcap > 0:
        dx = dx + softcap * 2.0 ** -22
    return x, slack, dx


def attention(q, k, v, scale, ok, softcap=0.0, slope=0.0, at=None, t=torch.float32):
    """One head: q [S,d], k,v [L,d] of any type, ok [S,L] -> out, lse in 64 bits and the bounds of a kernel's."""
    q, k, v = q.double(), k.double(), v.double()
    S, L = ok.shape
    at = torch.arange(S) + (L - S) if at is None else at
    any_ = ok.any(1)
    # what is masked touches nothing, NaN included: only what some query sees enters the products
    k = torch.where(ok.any(0)[:, None], k, torch.zeros_like(k))
    x, slack, dx = scores(q, k, scale, softcap, slope, at)
    x = torch.where(ok, x, torch.full_like(x, -float("inf")))
    dxm = torch.where(ok, dx, torch.zeros_like(dx)).amax(1)
    lse = torch.logsumexp(x, 1)
    p = torch.where(ok, torch.exp(x - torch.where(any_, lse, torch.zeros_like(lse))[:, None]), torch.zeros_like(x))
    out = masked_product(p, v, ok)
    mag = masked_product(p, v.abs(), ok)
    u = torch.finfo(t).eps / 2 if t != torch.float32 else W
    up = u if t != torch.float32 else 0.0
    out_tol = rounding(out, t) + (up + 4 * dxm[:, None] + (L + 4) * W) * mag
    if t == torch.float16:
        out_tol = out_tol + 2.0 ** -30 * L * v.abs().nan_to_num(0, 0, 0).max()
    lse_tol = 2 * dxm + 8 * W * lse.abs() + 4 * W
    lse = torch.where(any_, lse, torch.full_like(lse, EMPTY))
    return dict(out=out, lse=lse, out_tol=out_tol, lse_tol=torch.where(any_, lse_tol, torch.zeros_like(lse_tol)), p=p,
                slack=slack, dxm=dxm)


def masked_product(p, v, ok):
    """sum over the seen of p v: a NaN or an infinity that is not seen does not enter."""
    if torch.isfinite(v).all():
        return p @ v
    res = p @ torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    for j in (~torch.isfinite(v)).any(1).nonzero().flatten().tolist():
        bad = ~torch.isfinite(v[j])
        rows = ok[:, j]
        part = res[rows]
        part[:, bad] += p[rows, j][:, None] * v[j][bad]
        res[rows] = part
    return res


def attention_backward(q, k, v, do, f, scale, ok, dlse=None, t=torch.float32, lse=None, out=None):
    """Gradients of one head from its forward `f` (or a merged lse / out): dq, and this head's share of dk, dv."""
    q, k, v, do = q.double(), k.double(), v.double(), do.double()
    d, (S, L) = q.shape[1], ok.shape
    p, o = f["p"], f["out"] if out is None else out.double()
    if lse is not None:
        p = p * torch.exp(torch.where(f["lse"] > -1e30, f["lse"] - lse.double(), torch.zeros_like(f["lse"])))[:, None]
    some_q, some_k = ok.any(1)[:, None], ok.any(0)[:, None]
    q, do, o = (torch.where(some_q, a, torch.zeros_like(a)) for a in (q, do, o))
    k, v = (torch.where(some_k, a, torch.zeros_like(a)) for a in (k, v))
    dl = torch.zeros(S, dtype=torch.float64) if dlse is None else dlse.double()
    dl = torch.where(some_q[:, 0], dl, torch.zeros_like(dl))
    D = (do * o).sum(1) - dl
    dP = torch.where(ok, do @ v.T, torch.zeros_like(p))
    g = torch.where(ok, p * (dP - D[:, None]) * f["slack"], torch.zeros_like(p))
    u = torch.finfo(t).eps / 2 if t != torch.float32 else W
    ug = u if t != torch.float32 else 4 * W
    doo, dov = (do.abs() * o.abs()).sum(1), do.abs() @ v.abs().T
    e = torch.exp(torch.clamp(f["dxm"], max=1.0))[:, None]
    dD = (u * doo + (d + 4) * W * doo + 2 * W * dl.abs())[:, None]
    dslack = 4 * (f["dxm"][:, None] + 2.0 ** -22)
    dg = (ug + 4 * f["dxm"][:, None]) * g.abs() + e * p * f["slack"] * (dD + (d + 2) * W * dov) + (p * (dP - D[:, None])).abs() * torch.where(
        f["slack"] < 1, dslack.expand_as(p), torch.zeros_like(p))
    if t == torch.float16:
        dg = dg + torch.where(ok, torch.full_like(p, 2.0 ** -30 * float(do.abs().sum(1).max() * (v.abs().max() + o.abs().max()) + dl.abs().max())), torch.zeros_like(p))
    dg = torch.where(ok, dg, torch.zeros_like(dg))
    up = (u if t != torch.float32 else 0.0) + 4 * f["dxm"][:, None]
    dp = up * p + (2.0 ** -30 * ok if t == torch.float16 else 0.0)
    n = S + 4
    return dict(dq=g @ k * scale, dk=g.T @ q * scale, dv=p.T @ do,
                dq_tol=rounding(g @ k * scale, t) + scale * (dg @ k.abs() + (L + 4) * W * (g.abs() @ k.abs())),
                dk_tol=scale * (dg.T @ q.abs() + n * W * (g.abs().T @ q.abs())), dv_tol=dp.T @ do.abs() + n * W * (p.T @ do.abs()))


def local(q, k, v, scale, causal, softcap=0.0, slopes=None, doc_q=None, doc_k=None, prefix=None, dout=None, dlse=None):
    """All heads: q [H*G,S,d], k,v [H,L,d].  Returns a dict of results and a dict of bounds."""
    HG, S, d = q.shape
    H, L, _ = k.shape
    G, t = HG // H, q.dtype
    ok = seen_mask(S, L, causal, prefix, doc_q, doc_k)
    names = ["out", "lse"] + (["dq"] if dout is not None else [])
    res, tol = {n: [] for n in names}, {n: [] for n in names}
    dk, dv = torch.zeros(H, L, d, dtype=torch.float64), torch.zeros(H, L, d, dtype=torch.float64)
    dk_tol, dv_tol = torch.zeros_like(dk), torch.zeros_like(dv)
    for h in range(HG):
        f = attention(q[h], k[h // G], v[h // G], scale, ok, softcap, 0.0 if slopes is None else float(slopes[h]), t=t)
        if dout is not None:
            b = attention_backward(q[h], k[h // G], v[h // G], dout[h], f, scale, ok, None if dlse is None else dlse[h], t)
            f.update(dq=b["dq"], dq_tol=b["dq_tol"])
            dk[h // G] += b["dk"]
            dv[h // G] += b["dv"]
            dk_tol[h // G] += b["dk_tol"]
            dv_tol[h // G] += b["dv_tol"]
        for n in names:
            res[n].append(f[n])
            tol[n].append(f[n + "_tol"])
    res, tol = {n: torch.stack(x) for n, x in res.items()}, {n: torch.stack(x) for n, x in tol.items()}
    if dout is not None:
        res.update(dk=dk, dv=dv)
        tol.update(dk=dk_tol + rounding(dk, t), dv=dv_tol + rounding(dv, t))
    return res, tol


class Cache:
    """The bookkeeping of a paged cache in lists, a token at a time."""

    def __init__(self, n_rows, n_pages, page, width):
        self.P, self.width = page, width
        self.refs, self.rows, self.length = [0] * n_pages, [[] for _ in range(n_rows)], [0] * n_rows

    def copy(self):
        c = Cache(len(self.rows), len(self.refs), self.P, self.width)
        c.refs, c.rows, c.length = list(self.refs), [list(r) for r in self.rows], list(self.length)
        return c

    def take(self, other):
        self.refs, self.rows, self.length = other.refs, other.rows, other.length

    def append(self, counts):
        """(page, slot) of every new token in order, or None where the call is refused."""
        c, at = self.copy(), []
        for r, n in enumerate(counts):
            for _ in range(n):
                if c.length[r] % c.P == 0:
                    if 0 not in c.refs or len(c.rows[r]) == c.width:
                        return None
                    page = c.refs.index(0)
                    c.refs[page] = 1
                    c.rows[r].append(page)
                at.append((c.rows[r][c.length[r] // c.P], c.length[r] % c.P))
                c.length[r] += 1
        self.take(c)
        return at

    def fork(self, src):
        """(to, from, tokens) of every page that is copied, or None where the call is refused."""
        c, copies = self.copy(), []
        for r, s in enumerate(src):
            if s < 0:
                continue
            if s >= len(src) or s == r or self.length[r] or src[s] >= 0:
                return None
            whole, part = divmod(self.length[s], c.P)
            c.rows[r], c.length[r] = self.rows[s][:whole], self.length[s]
            if part:
                if 0 not in c.refs:
                    return None
                page = c.refs.index(0)
                c.refs[page] = 1
                c.rows[r].append(page)
                copies.append((page, self.rows[s][whole], part))
        for r, s in enumerate(src):
            if s >= 0:
                for page in self.rows[s][:self.length[s] // c.P]:
                    c.refs[page] += 1
        self.take(c)
        return copies

    def drop(self, counts):
        for r, n in enumerate(counts):
            for _ in range(min(max(n, 0), len(self.rows[r]))):
                self.refs[self.rows[r].pop(0)] -= 1
                self.length[r] = max(0, self.length[r] - self.P)

    def compact(self):
        """{from: to} of the pages that move."""
        used = [p for p, n in enumerate(self.refs) if n]
        moved = dict(zip([p for p in used if p >= len(used)], [p for p in range(len(used)) if not self.refs[p]]))
        for a, b in moved.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.rows = [[moved.get(p, p) for p in r] for r in self.rows]
        return moved

    def table(self):
        return [r + [-1] * (self.width - len(r)) for r in self.rows]
