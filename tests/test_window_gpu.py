"""Drafts, masks and kept attention weights over ring windows, against 64 bits.

Every slot outside the windows holds NaN; outputs start as NaN.
"""
import numpy as np
import pytest
import torch

import sts_attn
from conftest import scale_for
from windows import Window, ancestors, attend64, evict64, queries, random_tree, tree_seen

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def close(got, want, bound, what):
    err = np.abs(got - want)
    assert np.isfinite(got).all(), what
    worst = (err - bound[..., None]).max()
    assert worst <= 0, f"{what}: off by {err.max():.3e}, bound {bound.max():.3e}"


def same(got, clean, bound, what):
    """Two evaluations of one value, each within its bound of it (the values that a
    query does not see may decide how its tile is multiplied, not what comes out)."""
    assert np.isfinite(got).all(), what
    assert (np.abs(got - clean) <= 2 * bound[..., None]).all(), what


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int32)).cuda()


# ---- drafts ---------------------------------------------------------------------

def run_tree(w, q, parents, counts, scale, out=None):
    k, v, lens, starts = w.dev("k", "v", "lens", "starts")
    if out is None:
        out = torch.full(q.shape, float("nan"), device="cuda")
    sts_attn.tree_attention(torch.from_numpy(q).cuda(), k, v, i32(parents), lens, starts, scale,
                            counts=None if counts is None else i32(counts), out=out)
    return out.cpu().numpy()


TREES = [
    # B, T, H, KH, D, M, lens, counts, dtype
    (1, 1, 2, 2, 128, 40, [33], None, F32),             # one token
    (1, 1, 2, 2, 64, 1, [1], None, F32),                # a window of the token alone
    (4, 5, 4, 4, 128, 64, [64, 5, 17, 0], [5, 5, 3, 2], F32),  # full ring, draft alone, none
    (3, 16, 4, 2, 64, 300, [300, 100, 16], [16, 0, 16], F32),
    (2, 17, 6, 2, 96, 260, [259, 31], [17, 11], F32),   # padded head dim, three heads a group
    (2, 33, 2, 2, 128, 700, [693, 40], [33, 33], BF16),
    (2, 24, 8, 1, 64, 513, [513, 512], [24, 23], BF16), # all heads on one K/V head
    (1, 64, 4, 4, 128, 900, [897], [64], F32),
    (2, 100, 2, 1, 4, 500, [500, 333], [100, 99], F32), # the smallest head dim
    (1, 256, 2, 2, 128, 1000, [999], [256], F32),       # the largest draft
    (1, 200, 3, 1, 120, 450, [450], [129], BF16),
    (2, 40, 72, 1, 64, 200, [200, 128], [2, 40], F32),  # 72 heads a group: a query's rows span blocks
    (3, 12, 32, 32, 128, 3000, [2999, 1, 700], [12, 1, 7], F32),  # several splits
    (1, 8, 4, 1, 8, 4000, [4000], [8], BF16),           # long, narrow
]


@pytest.mark.parametrize("case", TREES, ids=lambda c: "-".join(str(x) for x in c[:6]))
def test_tree_attention(gpu, case):
    B, T, H, KH, D, M, lens, counts, dtype = case
    w = Window(hash(case[:6]) % 1000, B, KH, M, D, lens, dtype)
    q = queries(w.rng, B, T, H, D)
    n = [min(T, L) for L in lens] if counts is None else [min(c, T, L) for c, L in zip(counts, lens)]
    parents = np.stack([random_tree(w.rng, c, T) for c in n])
    got = run_tree(w, q, parents, counts, scale_for(D))
    again = run_tree(w, q, parents, counts, scale_for(D))
    np.testing.assert_array_equal(got, again)
    for b in range(B):
        assert not got[b, n[b]:].any(), "rows behind the draft are zeros"
        if n[b]:
            seen = tree_seen(parents[b], n[b], lens[b])
            want, _, bound = attend64(q[b, :n[b]], w.rows(b, w.k), w.rows(b, w.v), seen, scale_for(D))
            close(got[b, :n[b]], want, bound, f"stream {b}")


@pytest.mark.parametrize("shape", ["chain", "star", "comb"])
@pytest.mark.parametrize("T", [2, 32, 65, 256])
def test_tree_shapes(gpu, shape, T):
    """A chain (a causal chunk), a star (every node sees itself alone), a comb."""
    i = np.arange(T)
    parents = {"chain": i - 1, "star": np.full(T, -1), "comb": np.where(i % 2, i - 1, i - 2)}[shape].astype(np.int32)
    parents[0] = -1
    w = Window(T, 1, 2, 400, 64, [T + 77])
    q = queries(w.rng, 1, T, 2, 64)
    got = run_tree(w, q, parents[None], None, 0.125)
    want, _, bound = attend64(q[0], w.rows(0, w.k), w.rows(0, w.v), tree_seen(parents, T, T + 77), 0.125)
    close(got[0], want, bound, shape)
    if shape == "chain":
        assert ancestors(parents, T).sum() == T * (T + 1) // 2


def test_tree_parents_out_of_range(gpu):
    """A parent that is not an earlier node is the last committed row."""
    T = 9
    w = Window(3, 1, 2, 60, 64, [50])
    q = queries(w.rng, 1, T, 2, 64)
    bad = np.array([[5, 1, -7, 3, 900, -(2 ** 31), 2 ** 31 - 1, 8, 2]], np.int32)
    fixed = np.array([[-1, -1, -1, -1, -1, -1, -1, -1, 2]], np.int32)
    np.testing.assert_array_equal(run_tree(w, q, bad, None, 0.125), run_tree(w, q, fixed, None, 0.125))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 100, 128])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), float("-inf"), 3e38])
def test_tree_hidden_values(gpu, poison, D, dtype):
    """What a node does not see has no influence, whatever is there: the siblings of
    a node with such K and V rows get what they get without them, and only the
    nodes that see it do not."""
    if dtype == BF16 and D % 8:
        D = 104
    T, L = 21, 90
    w = Window(5, 1, 2, 128, D, [L], dtype)
    q = queries(w.rng, 1, T, 4, D)
    parents = random_tree(w.rng, T, T)
    parents[4] = -1
    clean = run_tree(w, q, parents[None], None, scale_for(D))
    bound = attend64(q[0], w.rows(0, w.k), w.rows(0, w.v), tree_seen(parents, T, L), scale_for(D))[2]
    slot = int(w.slots(0)[L - T + 4])
    w.k[0, :, slot] = poison
    w.v[0, :, slot, ::3] = poison
    got = run_tree(w, q, parents[None], None, scale_for(D))
    below = ancestors(parents, T)[:, 4]
    assert 1 <= below.sum() < T
    same(got[0, ~below], clean[0, ~below], bound[~below], "nodes that do not see it")
    assert (got[0, below] != clean[0, below]).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["tiny", "huge", "steps", "zeros first", "one row", "zeros"])
@pytest.mark.parametrize("T", [8, 30, 64])
def test_tree_magnitudes(gpu, T, kind, dtype):
    """Rows of any size: all tiny or huge, from step to step, zeros before others,
    one row far above the rest."""
    L, D = 500, 128
    w = Window(7, 1, 1, 600, D, [L], dtype)
    size = {"tiny": np.full(L, 1e-20), "huge": np.full(L, 1e20), "steps": 10.0 ** (np.arange(L) // 40 - 6),
            "zeros first": np.where(np.arange(L) < 300, 0, 1e-3), "one row": np.where(np.arange(L) == 137, 1e6, 1.0),
            "zeros": np.zeros(L)}[kind]
    f = torch.from_numpy(size).to(F32)[None, :, None]
    slots = torch.from_numpy(w.slots(0))
    w.v[0][:, slots] = (w.v[0][:, slots].float() * f).to(dtype)
    for which in ("values", "rows"):
        if which == "rows":  # keys too, with queries that keep the scores moderate
            w.k[0][:, slots] = (w.k[0][:, slots].float() * f).to(dtype)
        q = queries(w.rng, 1, T, 2, D) / (np.float32(size.max() or 1) if which == "rows" else np.float32(1))
        parents = random_tree(w.rng, T, T)
        got = run_tree(w, q, parents[None], None, scale_for(D))
        want, _, bound = attend64(q[0], w.rows(0, w.k), w.rows(0, w.v), tree_seen(parents, T, L), scale_for(D))
        close(got[0], want, bound, which)


@pytest.mark.parametrize("size", [1e30, 1e22, 1e-30])
@pytest.mark.parametrize("T", [8, 30])
def test_tree_query_magnitudes(gpu, T, size):
    """Queries of any size against keys that keep the scores moderate."""
    L, D = 200, 64
    w = Window(17, 1, 1, 200, D, [L])
    w.k = w.k / np.float32(size)
    q = queries(w.rng, 1, T, 2, D) * np.float32(size)
    parents = random_tree(w.rng, T, T)
    got = run_tree(w, q, parents[None], None, scale_for(D))
    want, _, bound = attend64(q[0], w.rows(0, w.k), w.rows(0, w.v), tree_seen(parents, T, L), scale_for(D))
    close(got[0], want, bound, "queries")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,H,KH,T", [(64, 4, 2, 3), (65, 4, 2, 3), (2, 12, 1, 6), (130, 2, 2, 1)])
def test_streams_of_very_different_lengths(gpu, B, H, KH, T, dtype):
    """One long window among short and empty ones: splits by the rows of all of them
    (up to 64 streams) or the same for each; drafts, kept weights, single tokens."""
    M, D = 3000, 64
    rng = np.random.default_rng(B)
    lens = rng.integers(0, 40, B)
    lens[B // 2], lens[0] = M, 0
    w = Window(B, B, KH, M, D, lens, dtype)
    q = queries(w.rng, B, T, H, D)
    n = np.minimum(lens, T)
    parents = np.stack([random_tree(w.rng, c, T) for c in n])
    got = run_tree(w, q, parents, None, 0.125)
    one = run_masked(w, q[:, :1].copy(), 0.125, lo=np.maximum(lens - 1500, 0)[:, None])
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    acc = torch.zeros((B, KH, M), device="cuda")
    dec = sts_attn.decode_ring_weights(torch.from_numpy(q[:, 0].copy()).cuda(), k, v, acc, dl, ds, 0.125)
    dec, acc = dec.cpu().numpy(), acc.cpu().numpy()
    for b in range(B):
        L = int(lens[b])
        if L == 0:
            assert not got[b].any() and not one[b].any() and not dec[b].any() and not acc[b].any()
            continue
        kk, vv = w.rows(b, w.k), w.rows(b, w.v)
        want, _, bound = attend64(q[b, :n[b]], kk, vv, tree_seen(parents[b], n[b], L), 0.125)
        close(got[b, :n[b]], want, bound, f"draft {b}")
        want, p, bound = attend64(q[b, :1], kk, vv, np.ones((1, L), bool), 0.125)
        close(dec[b], want[0], bound[0], f"decode {b}")
        assert np.allclose(acc[b].sum(-1), H // KH, rtol=1e-4)
        want, _, bound = attend64(q[b, :1], kk, vv, (np.arange(L) >= L - 1500)[None], 0.125)
        close(one[b], want, bound, f"window {b}")


def test_tree_visible_infinite_value(gpu):
    """An infinite V element reaches exactly the nodes and dims that see it."""
    T, L, D = 10, 40, 64
    w = Window(6, 1, 1, 64, D, [L])
    q = queries(w.rng, 1, T, 2, D)
    parents = random_tree(w.rng, T, T)
    parents[2] = -1
    clean = run_tree(w, q, parents[None], None, scale_for(D))
    bound = attend64(q[0], w.rows(0, w.k), w.rows(0, w.v), tree_seen(parents, T, L), scale_for(D))[2]
    w.v[0, 0, int(w.slots(0)[L - T + 2]), 7] = float("inf")
    got = run_tree(w, q, parents[None], None, scale_for(D))
    below = ancestors(parents, T)[:, 2]
    assert (got[0, below][..., 7] == np.inf).all()
    same(np.delete(got[0, below], 7, -1), np.delete(clean[0, below], 7, -1), bound[below], "its other dims")
    same(got[0, ~below], clean[0, ~below], bound[~below], "nodes that do not see it")


def test_tree_of_the_whole_batch_range(gpu):
    """Many streams, one after another in length, drafts longer than their windows."""
    B, T, M = 70, 8, 70
    lens = np.arange(B) + 1
    w = Window(8, B, 1, M, 64, lens)
    q = queries(w.rng, B, T, 2, 64)
    n = np.minimum(lens, T)
    parents = np.stack([random_tree(w.rng, c, T) for c in n])
    got = run_tree(w, q, parents, np.full(B, 1000), 0.125)
    for b in range(B):
        want, _, bound = attend64(q[b, :n[b]], w.rows(b, w.k), w.rows(b, w.v),
                                  tree_seen(parents[b], n[b], int(lens[b])), 0.125)
        close(got[b, :n[b]], want, bound, f"stream {b}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128, 8])
def test_tree_commit(gpu, D, dtype):
    B, T, KH, M = 5, 40, 3, 64
    lens, counts = np.array([64, 50, 40, 3, 0]), np.array([40, 17, 40, 40, 2])
    n = np.minimum(counts, lens)
    w = Window(9, B, KH, M, D, lens, dtype)
    path = np.zeros((B, T), np.int32)
    accepted = np.array([11, 17, 1, 2, 1], np.int32)
    path[0, :11] = np.sort(w.rng.choice(40, 11, replace=False))
    path[1] = np.arange(T)         # everything accepted: nothing moves
    path[2, 0] = 39
    path[3, :2] = [2, 1]           # not ascending: still row by row from the old draft
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    sts_attn.tree_commit(k, v, i32(path), i32(accepted), dl, ds, counts=i32(counts))
    for t, got in ((w.k, k.cpu()), (w.v, v.cpu())):
        want = t.clone()
        for b in range(B):
            slots = w.slots(b)
            for j in range(min(accepted[b], n[b])):
                want[b, :, slots[lens[b] - n[b] + j]] = t[b][:, slots[lens[b] - n[b] + path[b, j]]]
        assert torch.equal(got.nan_to_num(9e9), want.nan_to_num(9e9))


def test_tree_commit_ignores_what_is_out_of_range(gpu):
    w = Window(10, 1, 2, 32, 64, [20])
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    path = i32([[-3, 0, 6, 2 ** 31 - 1, 5, 1, 0, 0]])
    sts_attn.tree_commit(k, v, path, i32([6]), dl, ds, counts=i32([6]))
    want = w.k.clone()
    s = w.slots(0)
    want[0, :, s[14 + 4]] = w.k[0][:, s[14 + 5]]
    assert torch.equal(k.cpu().nan_to_num(9e9), want.nan_to_num(9e9))


# ---- masks ------------------------------------------------------------------------

def run_masked(w, q, scale, lo=None, hi=None, counts=None, slopes=None, softcap=0.0):
    k, v, lens, starts = w.dev("k", "v", "lens", "starts")
    out = torch.full(q.shape, float("nan"), device="cuda")
    sts_attn.masked_attention(torch.from_numpy(q).cuda(), k, v, lens, starts, scale,
                              lo=None if lo is None else i32(lo), hi=None if hi is None else i32(hi),
                              counts=None if counts is None else i32(counts),
                              slopes=None if slopes is None else torch.from_numpy(slopes).cuda(), softcap=softcap,
                              out=out)
    return out.cpu().numpy()


def check_masked(w, q, scale, lo=None, hi=None, counts=None, slopes=None, softcap=0.0):
    B, S = q.shape[:2]
    got = run_masked(w, q, scale, lo, hi, counts, slopes, softcap)
    for b in range(B):
        L = int(w.lens[b])
        n = min(S if counts is None else max(int(counts[b]), 0), S, L)
        assert not got[b, n:].any()
        if not n:
            continue
        rows, at = np.arange(L), np.arange(L - n, L)
        first = np.zeros(n) if lo is None else lo[b, :n]
        last = at + 1 if hi is None else hi[b, :n]
        seen = (rows >= np.asarray(first)[:, None]) & (rows < np.asarray(last)[:, None])
        want, _, bound = attend64(q[b, :n], w.rows(b, w.k), w.rows(b, w.v), seen, scale, softcap, slopes, at)
        close(got[b, :n], want, bound, f"stream {b}")
        assert not got[b, :n][~seen.any(1)].any(), "a query that sees nothing gets zeros"
    return got


MASKED = [
    # B, S, H, KH, D, M, lens, counts, dtype
    (1, 1, 4, 4, 128, 50, [50], None, F32),
    (3, 1, 8, 2, 64, 3000, [3000, 1, 0], None, F32),       # single tokens, splits
    (2, 7, 4, 4, 128, 129, [129, 7], None, F32),
    (2, 60, 4, 2, 64, 257, [257, 99], [60, 41], BF16),
    (1, 130, 3, 1, 100, 300, [290], None, F32),
    (1, 200, 2, 2, 128, 1100, [1099], None, BF16),
    (2, 33, 5, 5, 36, 120, [33, 20], None, F32),           # chunks at the window's start
    (1, 513, 2, 1, 128, 600, [600], None, F32),
]


@pytest.mark.parametrize("feature", ["causal", "cap", "bias", "both"])
@pytest.mark.parametrize("case", MASKED, ids=lambda c: "-".join(str(x) for x in c[:6]))
def test_masked_causal(gpu, case, feature):
    B, S, H, KH, D, M, lens, counts, dtype = case
    w = Window(sum(case[:6]), B, KH, M, D, lens, dtype)
    q = queries(w.rng, B, S, H, D)
    slopes = (2.0 ** -w.rng.uniform(0, 8, H)).astype(np.float32) if feature in ("bias", "both") else None
    cap = 5.0 if feature in ("cap", "both") else 0.0
    check_masked(w, q, scale_for(D), counts=counts, slopes=slopes, softcap=cap)


@pytest.mark.parametrize("case", MASKED, ids=lambda c: "-".join(str(x) for x in c[:6]))
@pytest.mark.parametrize("mask", ["documents", "prefix", "window", "random"])
def test_masked_ranges(gpu, case, mask):
    B, S, H, KH, D, M, lens, counts, dtype = case
    w = Window(sum(case[:6]) + 1, B, KH, M, D, lens, dtype)
    q = queries(w.rng, B, S, H, D)
    lo, hi = np.zeros((B, S), np.int64), np.zeros((B, S), np.int64)
    for b in range(B):
        n = min(S if counts is None else counts[b], lens[b])
        at = np.arange(lens[b] - n, lens[b])
        if not n:
            continue
        hi[b, :n] = at + 1
        if mask == "documents":
            edges = np.unique(np.concatenate([[0], w.rng.integers(0, lens[b], 4)]))
            lo[b, :n] = edges[np.searchsorted(edges, at, side="right") - 1]
        elif mask == "prefix":
            hi[b, :n] = np.maximum(at + 1, w.rng.integers(0, lens[b] + 1))
        elif mask == "window":
            lo[b, :n] = at + 1 - w.rng.integers(1, 20)  # reaches below 0 at the start
        else:
            # Any ranges, some of them empty, turned round, or past both ends.
            lo[b, :n] = w.rng.integers(-10, lens[b] + 10, n)
            hi[b, :n] = w.rng.integers(-10, lens[b] + 10, n)
            lo[b, ::5] = hi[b, ::5]
            if n > 2:
                lo[b, 1], hi[b, 1] = -(2 ** 31), 2 ** 31 - 1
                lo[b, 2], hi[b, 2] = 2 ** 31 - 1, -(2 ** 31)
    check_masked(w, q, scale_for(D), lo, hi, counts)


SINGLE = [
    # B, H, D, M, lens (f32 rows, every head its own)
    (4, 3, 128, 64, [64, 1, 0, 33]),                        # one wave a head
    (3, 2, 40, 50, [50, 20, 7]),
    (5, 2, 64, 1500, [1500, 1, 700, 1499, 0]),              # several splits
    (2, 3, 100, 9001, [9000, 513]),
    (1, 1, 4, 20000, [20000]),
    (37, 8, 128, 1100, [(97 * i) % 1101 for i in range(37)]),  # more heads than CUs: longer splits
    (70, 4, 12, 2100, [(331 * i) % 2101 for i in range(70)]),
]


@pytest.mark.parametrize("feature", ["plain", "cap", "bias", "both"])
@pytest.mark.parametrize("case", SINGLE, ids=lambda c: "-".join(str(x) for x in c[:4]))
def test_masked_single_tokens(gpu, case, feature):
    """A token a stream under any range: none, one row, the ring's seam, past both ends,
    a stream without a token."""
    B, H, D, M, lens = case
    w = Window(sum(case[:4]), B, H, M, D, lens, F32)
    q = queries(w.rng, B, 1, H, D)
    slopes = (2.0 ** -w.rng.uniform(0, 8, H)).astype(np.float32) if feature in ("bias", "both") else None
    cap = 5.0 if feature in ("cap", "both") else 0.0
    lo = np.stack([w.rng.integers(-3, max(L, 1), 1) for L in lens])
    hi = np.stack([w.rng.integers(-1, L + 3, 1) for L in lens])
    hi[::3] = lo[::3] + 1
    hi[1::3] = 2 ** 31 - 1
    lo[3::7] = 2 ** 31 - 1
    counts = np.ones(B, np.int64)
    counts[2::9] = 0
    check_masked(w, q, scale_for(D), lo, hi, counts, slopes, cap)
    check_masked(w, q, scale_for(D), lo, None, None, slopes, cap)
    check_masked(w, q, scale_for(D), None, hi, None, slopes, cap)


def test_masked_nothing_seen(gpu):
    """All ranges empty, of a block or of the whole call: zeros."""
    w = Window(4, 2, 2, 200, 64, [200, 150])
    q = queries(w.rng, 2, 100, 4, 64)
    lo = np.full((2, 100), 5)
    hi = np.full((2, 100), 5)
    assert not run_masked(w, q, 0.125, lo, hi).any()
    hi[1, 90:] = 100
    check_masked(w, q, 0.125, lo, hi)


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), float("-inf")])
def test_masked_hidden_values(gpu, poison):
    """Rows of another document may hold anything."""
    L, S = 160, 100
    w = Window(11, 1, 2, 200, 128, [L])
    q = queries(w.rng, 1, S, 4, 128)
    at = np.arange(L - S, L)
    lo = np.where(at >= 101, 101, 0)[None]
    clean = run_masked(w, q, 0.09, lo)
    rows = np.arange(L)
    seen = (rows >= lo[0][:, None]) & (rows <= at[:, None])
    bound = attend64(q[0], w.rows(0, w.k), w.rows(0, w.v), seen, 0.09)[2]
    hidden = torch.from_numpy(w.slots(0)[:101])
    w.k[0][:, hidden] = poison
    w.v[0][:, hidden[::2]] = poison
    got = run_masked(w, q, 0.09, lo)
    same(got[0, at >= 101], clean[0, at >= 101], bound[at >= 101], "the other document")
    # And a poisoned row of the same document, for the queries before it.
    clean = got
    w.v[0][:, int(w.slots(0)[133])] = poison
    w.k[0][:, int(w.slots(0)[133])] = poison
    got = run_masked(w, q, 0.09, lo)
    early = (at >= 101) & (at < 133)
    same(got[0, early], clean[0, early], bound[early], "the queries before it")


def test_masked_large_scores(gpu):
    """Scores of thousands and the cap's far ends: no overflow on the way."""
    w = Window(12, 1, 2, 100, 64, [100])
    q = queries(w.rng, 1, 20, 2, 64) * 500
    check_masked(w, q, 1.0, softcap=30.0)
    got = run_masked(w, q, 1.0)
    assert np.isfinite(got).all()


def test_masked_equals_prefill_and_decode(gpu):
    """The causal chunk and the single token of the calls that were there."""
    H, D, M, L, S = 8, 128, 500, 470, 60
    w = Window(13, 1, H, M, D, [L])
    w.k, w.v = w.k.nan_to_num(0.0), w.v.nan_to_num(0.0)
    q = queries(w.rng, 1, S, H, D)
    got = run_masked(w, q, scale_for(D))
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    want = sts_attn.prefill_attention(torch.from_numpy(q[0]).cuda(), k, v, int(w.starts[0]), L, scale_for(D)).cpu()
    ref = attend64(q[0], w.rows(0, w.k), w.rows(0, w.v), np.tri(S, L, L - S, bool), scale_for(D))
    assert (np.abs(got[0] - want.numpy()) <= 2 * ref[2][..., None]).all()
    one = run_masked(w, q[:, -1:].copy(), scale_for(D))
    dec = sts_attn.decode_ring(torch.from_numpy(q[:, -1].copy()).cuda(), k, v, dl, ds, scale_for(D)).cpu().numpy()
    assert (np.abs(one[0, 0] - dec[0]) <= 2 * ref[2][-1][:, None]).all()


# ---- kept weights and eviction ---------------------------------------------------------

WEIGHTS = [
    # B, H, KH, D, M, lens, dtype
    (1, 4, 4, 128, 30, [30], F32),
    (3, 8, 8, 64, 100, [1, 0, 99], F32),
    (2, 8, 2, 128, 3000, [3000, 1234], F32),
    (2, 24, 8, 64, 5003, [5003, 64], BF16),
    (1, 72, 1, 128, 150, [149], F32),     # more heads than a block's rows
    (2, 20, 1, 80, 333, [332, 16], BF16),
    (1, 6, 3, 12, 77, [70], F32),
    # every head its own rows: head dims between, long windows in many parts
    (3, 5, 5, 40, 700, [700, 1, 33], F32),
    (1, 2, 2, 100, 4100, [4099], F32),
    (1, 1, 1, 128, 20001, [20000], F32),
    (2, 2, 2, 64, 9000, [8999, 17], F32),
    (70, 1, 1, 4, 65, [(7 * i) % 66 for i in range(70)], F32),
]


@pytest.mark.parametrize("case", WEIGHTS, ids=lambda c: "-".join(str(x) for x in c[:5]))
def test_decode_weights(gpu, case):
    B, H, KH, D, M, lens, dtype = case
    w = Window(sum(case[:5]), B, KH, M, D, lens, dtype)
    q = queries(w.rng, B, H, D)
    before = w.rng.uniform(0, 3, (B, KH, M)).astype(np.float32)
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    acc = torch.from_numpy(before).cuda()
    out = torch.full((B, H, D), float("nan"), device="cuda")
    dq = torch.from_numpy(q).cuda()
    sts_attn.decode_ring_weights(dq, k, v, acc, dl, ds, scale_for(D), out=out)
    got, kept = out.cpu().numpy(), acc.cpu().numpy()
    again = torch.from_numpy(before).cuda()
    sts_attn.decode_ring_weights(dq, k, v, again, dl, ds, scale_for(D))
    assert torch.equal(acc, again)
    g = H // KH
    for b in range(B):
        L = lens[b]
        outside = np.setdiff1d(np.arange(M), w.slots(b))
        np.testing.assert_array_equal(kept[b][:, outside], before[b][:, outside])
        if L == 0:
            assert not got[b].any()
            continue
        want, p, bound = attend64(q[b][None], w.rows(b, w.k), w.rows(b, w.v), np.ones((1, L), bool), scale_for(D))
        close(got[b], want[0], bound[0], f"stream {b}")
        given = p[0].reshape(KH, g, L).sum(1)
        # Each weight within twice the scores' error of itself, the sums of the group
        # and with what was there rounded once per term.
        size = attend64(q[b][None], w.rows(b, w.k), np.ones((KH, L, D)), np.ones((1, L), bool), scale_for(D))[2][0]
        tol = given * size.max() + (g + 2) * 2.0 ** -24 * (before[b][:, w.slots(b)] + given)
        assert (np.abs(kept[b][:, w.slots(b)] - (before[b][:, w.slots(b)] + given)) <= tol).all()


EVICT = [
    # B, KH, D, M, lens, keep, recent, dtype, weights
    (1, 2, 128, 64, [64], 20, 5, F32, "random"),
    (4, 2, 64, 100, [100, 20, 21, 0], 20, 0, F32, "random"),
    (2, 3, 64, 300, [300, 150], 120, 120, F32, "random"),     # only the newest stay
    (1, 4, 128, 3000, [2999], 1500, 200, F32, "few values"),  # ties
    (2, 2, 64, 2500, [2500, 2049], 1, 0, BF16, "equal"),
    (1, 1, 4, 5000, [5000], 4999, 7, F32, "random"),
    (2, 2, 72, 90, [80, 90], 33, 1, BF16, "special"),
    (1, 2, 100, 90, [88], 40, 3, F32, "special"),
    (1, 1, 8, 20011, [20011], 9000, 100, BF16, "random"),
    (3, 8, 128, 1000, [1000, 900, 511], 511, 64, F32, "few values"),
]


@pytest.mark.parametrize("case", EVICT, ids=lambda c: "-".join(str(x) for x in c[:4]) + c[8])
def test_evict(gpu, case):
    B, KH, D, M, lens, keep, recent, dtype, kind = case
    w = Window(keep + M, B, KH, M, D, lens, dtype)
    acc = {"random": w.rng.exponential(1.0, (B, KH, M)), "few values": w.rng.integers(0, 4, (B, KH, M)) / 8,
           "equal": np.full((B, KH, M), 0.25),
           "special": w.rng.choice([0.0, -0.0, -1.5, np.nan, np.inf, -np.inf, 1e-42, 2.0], (B, KH, M))}[kind]
    acc = acc.astype(np.float32)
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    dw = torch.from_numpy(acc).cuda()
    kept = torch.full((B, KH, keep), 77, dtype=torch.int32, device="cuda")
    sts_attn.evict_ring(k, v, dw, dl, ds, keep, recent, kept=kept)
    kept = kept.cpu().numpy()
    want_k, want_v, want_w = w.k.clone(), w.v.clone(), acc.copy()
    for b in range(B):
        slots, L = w.slots(b), lens[b]
        for h in range(KH):
            rows = evict64(acc[b, h, slots], keep, recent)
            np.testing.assert_array_equal(kept[b, h, :len(rows)], rows)
            assert (kept[b, h, len(rows):] == -1).all()
            if L > keep:
                to = slots[L - keep:]
                want_k[b, h, to] = w.k[b, h, slots[rows]]
                want_v[b, h, to] = w.v[b, h, slots[rows]]
                want_w[b, h, to] = acc[b, h, slots[rows]]
    assert torch.equal(k.cpu().nan_to_num(9e9), want_k.nan_to_num(9e9))
    assert torch.equal(v.cpu().nan_to_num(9e9), want_v.nan_to_num(9e9))
    np.testing.assert_array_equal(dw.cpu().numpy(), want_w)


# ---- streams, graphs, refusals on the GPU --------------------------------------------------

def calls(seed, stream=None):
    """One call of each kind on its own tensors, as functions that return what they write."""
    w = Window(seed, 3, 4, 2000, 64, [2000, 1999, 300])
    w.k, w.v = w.k.nan_to_num(0.0), w.v.nan_to_num(0.0)
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    T = 20
    q = torch.from_numpy(queries(w.rng, 3, T, 8, 64)).cuda()
    parents = i32(np.stack([random_tree(w.rng, T, T) for _ in range(3)]))
    out = [torch.zeros_like(q), torch.zeros_like(q), torch.zeros((3, 8, 64), device="cuda")]
    acc = torch.rand((3, 4, 2000), device="cuda", generator=torch.Generator("cuda").manual_seed(seed))
    q1 = q[:, 0].contiguous()
    kept = torch.zeros((3, 4, 900), dtype=torch.int32, device="cuda")
    keep = (k.clone(), v.clone(), acc.clone())

    def tree():
        return [sts_attn.tree_attention(q, k, v, parents, dl, ds, 0.125, out=out[0], stream=stream)]

    def masked():
        return [sts_attn.masked_attention(q, k, v, dl, ds, 0.125, softcap=9.0, out=out[1], stream=stream)]

    def weights():
        return [sts_attn.decode_ring_weights(q1, k, v, acc, dl, ds, 0.125, out=out[2], stream=stream), acc]

    def evict():
        return [sts_attn.evict_ring(k, v, acc, dl, ds, 900, 50, kept=kept, stream=stream), k, v, acc]

    def restore():
        for a, z in zip((k, v, acc), keep):
            a.copy_(z)
        for o in out:
            o.fill_(float("nan"))

    return [tree, masked, weights, evict], restore


def test_calls_replay_from_a_graph(gpu):
    """All four captured together on a side stream, with eager work between replays."""
    side = torch.cuda.Stream()
    fns, restore = calls(21, side)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        want = [t.clone() for f in fns for t in f()]
    torch.cuda.synchronize()
    restore()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = [t for f in fns for t in f()]
    # acc appears in two of the lists, in its last state.
    for rep in range(4):
        restore()
        junk = torch.randn(1 << 20, device="cuda") * 2.0
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, (a, b) in enumerate(zip(got, want)):
            if x != 3:  # the weights before the eviction
                assert torch.equal(a, b), (rep, x)
        restore()
        with torch.cuda.stream(side):
            eager = [t.clone() for f in fns for t in f()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, want))
        del junk


def test_calls_on_two_streams_at_once(gpu):
    """Different streams use different workspaces: results as alone."""
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    fa, ra = calls(22, a)
    fb, rb = calls(23, b)
    torch.cuda.synchronize()
    wants = []
    for fns, restore, s in ((fa, ra, a), (fb, rb, b)):
        with torch.cuda.stream(s):
            wants.append([t.clone() for f in fns[:2] for t in f()])
        torch.cuda.synchronize()
        restore()
    torch.cuda.synchronize()
    for _ in range(20):
        for f, g in zip(fa[:2], fb[:2]):
            x, y = f(), g()
    torch.cuda.synchronize()
    for fns, want in ((fa, wants[0]), (fb, wants[1])):
        got = [t for f in fns[:2] for t in f()]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_stream_argument_without_its_context(gpu):
    """A stream that is not the current one, results allocated by the call."""
    w = Window(24, 2, 2, 900, 64, [900, 400])
    q = torch.from_numpy(queries(w.rng, 2, 8, 2, 64)).cuda()
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    parents = i32(np.stack([random_tree(w.rng, 8, 8) for _ in range(2)]))
    acc = [torch.zeros((2, 2, 900), device="cuda") for _ in range(2)]
    want = sts_attn.tree_attention(q, k, v, parents, dl, ds, 0.125)
    one = sts_attn.decode_ring_weights(q[:, 0].contiguous(), k, v, acc[0], dl, ds, 0.125)
    side = torch.cuda.Stream()
    for s in (side, side.cuda_stream):
        acc[1].zero_()
        torch.cuda.synchronize()
        got = sts_attn.tree_attention(q, k, v, parents, dl, ds, 0.125, stream=s)
        two = sts_attn.decode_ring_weights(q[:, 0].contiguous(), k, v, acc[1], dl, ds, 0.125, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(one, two) and torch.equal(acc[0], acc[1])


def test_binding_refuses_on_the_gpu(gpu):
    w = Window(25, 2, 2, 50, 64, [50, 40])
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    q = torch.zeros((2, 4, 2, 64), device="cuda")
    p = i32(np.zeros((2, 4)))
    with pytest.raises(ValueError, match="parents"):
        sts_attn.tree_attention(q, k, v, p[:, :3].contiguous(), dl, ds, 0.1)
    with pytest.raises(ValueError, match="contiguous"):
        sts_attn.tree_attention(q, k.transpose(0, 1), v.transpose(0, 1), p, dl, ds, 0.1)
    with pytest.raises(ValueError, match="lens"):
        sts_attn.tree_attention(q, k, v, p, dl[:1], ds, 0.1)
    with pytest.raises(TypeError, match="starts"):
        sts_attn.tree_attention(q, k, v, p, dl, ds.long(), 0.1)
    with pytest.raises(ValueError, match="lens must be on"):
        sts_attn.tree_attention(q, k, v, p, dl.cpu(), ds, 0.1)
    with pytest.raises(ValueError, match="q must be"):
        sts_attn.masked_attention(q[..., :32].contiguous(), k, v, dl, ds, 0.1)
    with pytest.raises(sts_attn.StsError, match="query heads"):
        sts_attn.masked_attention(torch.zeros((2, 4, 3, 64), device="cuda"), k, v, dl, ds, 0.1)
    with pytest.raises(ValueError, match="weights"):
        sts_attn.decode_ring_weights(q[:, 0].contiguous(), k, v, torch.zeros((2, 2, 49), device="cuda"), dl, ds, 0.1)
    for keep, recent in ((0, 0), (51, 0), (10, 11), (10, -1)):
        with pytest.raises(sts_attn.StsError):
            sts_attn.evict_ring(k, v, torch.zeros((2, 2, 50), device="cuda"), dl, ds, keep, recent)
    with pytest.raises(sts_attn.StsError, match="aligned"):
        sts_attn.tree_attention(torch.zeros(2 * 4 * 2 * 64 + 1, device="cuda")[1:].view(2, 4, 2, 64), k, v, p, dl, ds, 0.1)


def test_rows_of_all_streams_past_32_bits(gpu):
    """33 streams whose windows hold more than 2^32 rows together, 4 dims each: the
    splits cover every row (69 GB, K and V the same, of ones: the mean is one)."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB")
    B, M = 33, 0x7FFFFFF0 // 16
    lens = torch.full((B,), M, dtype=torch.int32, device="cuda")
    starts = torch.arange(B, dtype=torch.int32, device="cuda") * 1000
    assert B * M > 2 ** 32
    k = torch.ones((B, 1, M, 4), device="cuda")
    q = torch.randn((B, 1, 1, 4), device="cuda")
    parents = torch.full((B, 1), -1, dtype=torch.int32, device="cuda")
    for run in (lambda out: sts_attn.tree_attention(q, k, k, parents, lens, starts, 0.5, out=out),
                lambda out: sts_attn.masked_attention(q, k, k, lens, starts, 0.5, out=out)):
        out = torch.full((B, 1, 1, 4), float("nan"), device="cuda")
        run(out)
        # Every weight is the same: sums of equal terms, in chains of at most 2^17.
        assert (out - 1).abs().max().item() <= 2.0 ** 17 * 2.0 ** -24
    del k
    torch.cuda.empty_cache()
