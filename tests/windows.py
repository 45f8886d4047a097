"""Ring windows for the tests of drafts, masks and kept weights, and their 64-bit forms.

A Window holds ragged streams' caches with every slot outside the windows set to
NaN, so that a kernel that lets one through shows it.  attend64 is attention from
its definition in 64 bits on one stream's ordered rows; its bound is an upper bound
of the rounding of an f32 evaluation.
"""
import numpy as np
import torch

U = 2.0 ** -24  # half a step of f32, relative


class Window:
    def __init__(self, seed, B, KH, M, D, lens, dtype=torch.float32, starts=None):
        rng = np.random.default_rng(seed)
        self.rng, self.B, self.KH, self.M, self.D = rng, B, KH, M, D
        self.lens = np.asarray(lens, np.int32)
        self.starts = rng.integers(0, M, B).astype(np.int32) if starts is None else np.asarray(starts, np.int32)
        self.dtype = dtype
        k = torch.full((B, KH, M, D), float("nan"), dtype=dtype)
        v = torch.full((B, KH, M, D), float("nan"), dtype=dtype)
        for b in range(B):
            s = torch.from_numpy(self.slots(b))
            k[b, :, s] = torch.from_numpy(rng.standard_normal((KH, len(s), D))).to(dtype)
            v[b, :, s] = torch.from_numpy(rng.standard_normal((KH, len(s), D))).to(dtype)
        self.k, self.v = k, v

    def slots(self, b):
        return (int(self.starts[b]) + np.arange(int(self.lens[b]))) % self.M

    def rows(self, b, t):
        """Stream b's ordered rows of a cache, [KH, L, D] in 64 bits."""
        return t[b][:, torch.from_numpy(self.slots(b))].double().numpy()

    def dev(self, *names):
        out = []
        for n in names:
            x = getattr(self, n)
            out.append((torch.from_numpy(x) if isinstance(x, np.ndarray) else x).cuda())
        return out


def queries(rng, *shape):
    """f32 queries, some heads broad and some sharp."""
    return (rng.standard_normal(shape) * rng.uniform(0.5, 3.0, (shape[-2], 1))).astype(np.float32)


def attend64(q, k, v, seen, scale, softcap=0.0, slopes=None, w=None):
    """q [n,H,D], k/v [KH,L,D], seen [n,L] -> (out [n,H,D], p [n,H,L], bound [n,H]).

    bound: of an evaluation whose products are f32's or those of two f16 parts (off
    by 4 u of the element, or of its row's largest where the second part is below
    f16's normal range, and by 4 u of the product for the parts left out).  A score, a
    sum of D products with two scalings, is then off by at most
    scale ((D + 16) u sum |q k| + 4 u sum |q| max |k| + 4 u sum |k| max |q|) with the
    maxima of its own rows.  The cap's tanh, within 3 u relative, and the bias add 8 u
    of their size.  A score off by e turns its weight by the factor 1 +- (e + 3u) (the
    base-2 exponential of the hardware within 2 u), the normalised sum by twice that;
    the weights' and values' own parts add 16 u, and adding up L weighted rows (L + 8)
    u, all of the largest |v|."""
    n, H, D = q.shape
    g = H // k.shape[0]
    L = k.shape[1]
    out, p, bound = np.zeros((n, H, D)), np.zeros((n, H, L)), np.zeros((n, H))
    for h in range(H):
        kk, vv = k[h // g], v[h // g]
        x = np.full((n, L), -np.inf)
        size = np.zeros((n, L))
        for i in range(n):
            at = np.flatnonzero(seen[i])
            if not len(at):
                continue
            qi = q[i, h].astype(np.float64)
            s = kk[at] @ qi * scale
            ka, qa = np.abs(kk[at]), np.abs(qi)
            big = (ka @ qa * (D + 16) + 4 * qa.sum() * ka.max(1) + 4 * ka.sum(1) * qa.max()) * abs(scale) * U
            if softcap > 0:
                s = softcap * np.tanh(s / softcap)
                big = big + 8 * U * np.abs(s)
            if slopes is not None:
                away = slopes[h] * np.abs(w[i] - at)
                s = s - away
                big = big + 8 * U * (np.abs(away) + np.abs(s))
            # The exponent's own scaling by log2 e and the subtraction of the maximum.
            big = big + 4 * U * np.abs(s).max()
            e = np.exp(s - s.max())
            p[i, h, at] = e / e.sum()
            out[i, h] = p[i, h, at] @ vv[at]
            bound[i, h] = (2 * (big.max() + 3 * U) + (L + 24) * U) * np.abs(vv[at]).max()
    return out, p, bound


def ancestors(parents, n):
    """[n, n] truth: j is i or above it; a parent outside 0..i-1 is the committed row."""
    a = np.eye(n, dtype=bool)
    for i in range(n):
        if 0 <= parents[i] < i:
            a[i] |= a[parents[i]]
    return a


def depths(parents, n):
    d = np.zeros(n, np.int64)
    for i in range(n):
        if 0 <= parents[i] < i:
            d[i] = d[parents[i]] + 1
    return d


def tree_seen(parents, n, L):
    seen = np.ones((n, L), bool)
    seen[:, L - n:] = ancestors(parents, n)
    return seen


def random_tree(rng, n, T):
    p = np.full(T, -1, np.int32)
    for i in range(1, n):
        p[i] = rng.integers(-1, i)
    return p


def evict64(w, keep, recent):
    """The rows kept of one head's ordered weights, by sorting."""
    L = len(w)
    if L <= keep:
        return np.arange(L)
    old = np.where(np.isnan(w[:L - recent]), np.inf, w[:L - recent])  # NaN: the largest
    nan = np.isnan(w[:L - recent])
    order = np.lexsort((np.arange(len(old)), -old, ~nan))
    return np.concatenate([np.sort(order[:keep - recent]), np.arange(L - recent, L)])


def attend64_channels(q, k, v, seen, scale, softcap=0.0, slopes=None, w=None):
    """attend64 with a bound for every output channel: (out [n,H,D], bound [n,H,D]).

    The bound of an evaluation whose every operand keeps f32's 24 bits at any size:
    f32 products, or the six larger products of three bf16 parts each.  (Parts rounded
    to nearest stand for the value exactly; the three products left out are below
    2^-26 of it together, u/4.)  A score adds up 6 D products of |q k| at most and is
    scaled twice: off by e = scale (6 D + 16) u sum |q k|, and 8 u of its size for cap
    and bias each, 4 u of the largest for the exponent.  A weight is off by the factor
    e of its own row, the sum of the weights by their mean e, 3 u each for the
    exponentials.  A channel adds up 6 L terms p |v| at most, and 24 u covers the
    weights' parts, merge and division.  Weights below 2^-110 of the largest may be
    lost whole.  Every term is a share of that channel's own sum of p |v|."""
    n, H, D = q.shape
    g = H // k.shape[0]
    out, bound = np.zeros((n, H, D)), np.zeros((n, H, D))
    for h in range(H):
        kk, vv = k[h // g], v[h // g]
        for i in range(n):
            at = np.flatnonzero(seen[i])
            if not len(at):
                continue
            qi = q[i, h].astype(np.float64)
            s = kk[at] @ qi * scale
            e = np.abs(kk[at]) @ np.abs(qi) * (6 * D + 16) * abs(scale) * U
            if softcap > 0:
                s = softcap * np.tanh(s / softcap)
                e = e + 8 * U * np.abs(s)
            if slopes is not None:
                away = slopes[h] * np.abs(w[i] - at)
                s = s - away
                e = e + 8 * U * (np.abs(away) + np.abs(s))
            e = e + 4 * U * np.abs(s).max()
            p = np.exp(s - s.max())
            p = p / p.sum()
            va = np.abs(vv[at])
            off = e + p @ e + (6 * len(at) + 24) * U
            out[i, h] = p @ vv[at]
            bound[i, h] = (p * off) @ va + 2.0 ** -110 * va.sum(0)
    return out, bound
