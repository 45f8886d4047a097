"""Drafts and masked chunks over rows, elements and channels of very different size.

Every wave gets several tiles: 512 heads without splits, five tiles of 32 rows a wave.
Outputs are held to f32's grade channel by channel.
"""
import numpy as np
import pytest
import torch

from conftest import scale_for
from test_window_gpu import BF16, F32, run_masked, run_tree
from windows import Window, attend64_channels, queries, random_tree, tree_seen

pytestmark = pytest.mark.gpu

KH, L = 512, 700  # 22 tiles of 32 rows, dealt to the four waves of a workgroup


def window(seed, D, dtype=F32, lens=(L,), M=L + 5):
    return Window(seed, len(lens), KH, M, D, lens, dtype)


def resize(w, which, factor):
    """Multiplies stream 0's rows r of a cache by factor[r] (or factor[r][d])."""
    t = getattr(w, which)
    slots = torch.from_numpy(w.slots(0))
    f = torch.from_numpy(np.asarray(factor, np.float32))
    f = f[None, :, None] if f.dim() == 1 else f[None]
    t[0][:, slots] = (t[0][:, slots].float() * f).to(t.dtype)


HEADS = [0, 1, 255, 511]  # compared with 64 bits; the others run the same code


def check_tree(w, q, parents, what):
    T, D = q.shape[1], q.shape[3]
    got = run_tree(w, q, parents[None], None, scale_for(D))[0]
    assert np.isfinite(got).all(), what
    seen = tree_seen(parents, T, int(w.lens[0]))
    want, bound = attend64_channels(q[0][:, HEADS], w.rows(0, w.k)[HEADS], w.rows(0, w.v)[HEADS], seen, scale_for(D))
    over = np.abs(got[:, HEADS] - want) - bound
    assert (over <= 0).all(), f"{what}: {(np.abs(got[:, HEADS] - want) / bound).max():.3g} times the bound"


def check_masked(w, q, lo, what, softcap=0.0):
    S, D = q.shape[1], q.shape[3]
    n = int(w.lens[0])
    got = run_masked(w, q, scale_for(D), lo[None], softcap=softcap)[0]
    assert np.isfinite(got).all(), what
    at, rows = np.arange(n - S, n), np.arange(n)
    seen = (rows >= lo[:, None]) & (rows <= at[:, None])
    want, bound = attend64_channels(q[0][:, HEADS], w.rows(0, w.k)[HEADS], w.rows(0, w.v)[HEADS], seen, scale_for(D),
                                    softcap)
    over = np.abs(got[:, HEADS] - want) - bound
    assert (over <= 0).all(), f"{what}: {(np.abs(got[:, HEADS] - want) / bound).max():.3g} times the bound"


# Row sizes of V; a wave's first tile is one of the first 128 rows.
ROW_SIZES = {
    "1e-30 then 1e4": np.where(np.arange(L) < 128, 1e-30, 1e4),
    "1e-5 then 1e29": np.where(np.arange(L) < 128, 1e-5, 1e29),
    "1e29 then 1e-5": np.where(np.arange(L) < 128, 1e29, 1e-5),
    "zeros then 1e-20 then 1e20": np.where(np.arange(L) < 128, 0, np.where(np.arange(L) < 400, 1e-20, 1e20)),
    "one row of 1e29": np.where(np.arange(L) == 333, 1e29, 1e-3),
    "every row its own": 10.0 ** np.random.default_rng(1).uniform(-20, 20, L),
    "as they are": np.ones(L),
}


@pytest.mark.parametrize("kind", ROW_SIZES)
@pytest.mark.parametrize("D,dtype", [(64, F32), (100, F32), (128, F32), (64, BF16)])
def test_value_rows_of_any_size(gpu, D, dtype, kind):
    w = window(31, D, dtype)
    resize(w, "v", ROW_SIZES[kind])
    q = queries(w.rng, 1, 20, KH, D)
    check_tree(w, q, random_tree(w.rng, 20, 20), kind)
    check_masked(w, q, np.zeros(20, int), kind)


@pytest.mark.parametrize("D,dtype", [(64, F32), (128, F32), (64, BF16)])
@pytest.mark.parametrize("spread", [4, 12, 24])
def test_channels_of_any_size(gpu, D, spread, dtype):
    """V's channels from 1 down to 10^-spread, K's elements up and down with the
    queries' the other way: no channel is held by another's measure."""
    w = window(32, D, dtype)
    size = 10.0 ** -np.linspace(0, spread, D)
    resize(w, "v", np.tile(w.rng.permutation(size), (L, 1)))
    tilt = w.rng.permutation(size ** 0.5)
    resize(w, "k", np.tile(tilt, (L, 1)))
    q = (queries(w.rng, 1, 20, KH, D) / tilt).astype(np.float32)
    check_tree(w, q, random_tree(w.rng, 20, 20), "draft")
    check_masked(w, q, np.zeros(20, int), "chunk", softcap=20.0)


@pytest.mark.parametrize("D,dtype", [(64, F32), (128, F32), (64, BF16)])
@pytest.mark.parametrize("hidden", [8192.0, 1e30])
def test_hidden_rows_set_no_measure(gpu, hidden, D, dtype):
    """Large rows of another document, in every wave's first tile and beside seen rows:
    the queries that do not see them keep f32's grade in every channel."""
    w = window(33, D, dtype)
    size = 10.0 ** -np.linspace(0, 8, D)
    resize(w, "v", np.tile(size, (L, 1)))
    edge = 330
    slots = torch.from_numpy(w.slots(0)[:edge])
    w.v[0][:, slots] = hidden
    w.k[0][:, slots] = hidden
    q = queries(w.rng, 1, 40, KH, D)
    check_masked(w, q, np.full(40, edge), "chunk")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_small_weights_of_large_rows(gpu, dtype):
    """Rows that get e^-30 to e^-5 of the weight and are as much larger: each gives
    its share of the output to f32's grade."""
    D = 64
    w = window(34, D, dtype)
    # Dim 0 of K alone makes the scores: x_r = q_0 k_r0 scale, from 0 to -30.
    x = np.where(np.arange(L) % 3 == 0, 0.0, -np.random.default_rng(5).uniform(5, 30, L))
    k = torch.zeros((L, D), dtype=F32)
    k[:, 0] = torch.from_numpy(x / scale_for(D)).to(F32)
    w.k[0][:, torch.from_numpy(w.slots(0))] = k.to(dtype)[None]
    resize(w, "v", np.exp(-x) * 10.0 ** np.random.default_rng(6).uniform(-2, 2, L))
    q = np.zeros((1, 20, KH, D), np.float32)
    q[..., 0] = 1
    check_tree(w, q, random_tree(w.rng, 20, 20), "draft")
    check_masked(w, q, np.zeros(20, int), "chunk")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), 3.4e38])
def test_tiles_that_are_not_finite_between_others(gpu, poison, dtype):
    """A wave goes from products of parts to f32 and back: hidden values that are not
    finite in its second, third and fifth tiles, K and V apart and together."""
    D = 128 if dtype == F32 else 64
    w = window(35, D, dtype)
    q = queries(w.rng, 1, 24, KH, D)
    # Query i sees every row but those before lo; the poisoned rows are the first and
    # one of each tile that the first twelve queries do not see.
    S, n = 24, L
    lo = np.where(np.arange(S) % 2 == 0, 560, 0)
    want_hidden = [140, 300, 301, 555]
    for which, rows in (("v", want_hidden[:2]), ("k", want_hidden[1:3]), ("v", want_hidden[3:]), ("k", want_hidden[3:])):
        getattr(w, which)[0][:, torch.from_numpy(w.slots(0)[rows])] = poison
    got = run_masked(w, q, scale_for(D), lo[None])[0]
    rows, at = np.arange(n), np.arange(n - S, n)
    even = lo == 560
    seen = (rows >= lo[:, None]) & (rows <= at[:, None])
    want, bound = attend64_channels(q[0][even][:, HEADS], w.rows(0, w.k)[HEADS], w.rows(0, w.v)[HEADS], seen[even],
                                    scale_for(D))
    assert np.isfinite(got[even]).all()
    assert (np.abs(got[even][:, HEADS] - want) <= bound).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T", [4, 20])
def test_many_rows_of_the_largest_values(gpu, T, dtype):
    """60000 rows of values near 1e30 whose scores lie above those of every wave's
    first tile, by e^5.47 = 2^7.9: the sums stay in f32's range on the way."""
    import sts_attn
    D, n = 8, 60000
    at = np.arange(n)
    x = np.where(at < 128, 0.0, 5.46875).astype(np.float32)  # exact in bf16
    k1 = torch.zeros((n, D))
    k1[:, 0] = torch.from_numpy(x)
    v1 = torch.from_numpy((1e30 * (0.9 + 0.1 * at / n)).astype(np.float32))[:, None].expand(n, D)
    k = k1.to(dtype).cuda()[None, None].expand(1, KH, n, D).contiguous()
    v = v1.to(dtype).cuda()[None, None].expand(1, KH, n, D).contiguous()
    q = torch.zeros((1, T, KH, D), device="cuda")
    q[..., 0] = 1
    lens, starts = (torch.tensor([y], dtype=torch.int32, device="cuda") for y in (n, 0))
    parents = torch.full((1, T), -1, dtype=torch.int32, device="cuda")
    q64, k64, v64 = np.zeros((T, 1, D)), k1.double().numpy()[None], v1.to(dtype).double().numpy()[None]
    q64[..., 0] = 1
    causal = at[None, :] <= np.arange(n - T, n)[:, None]
    runs = [(tree_seen(np.full(T, -1), T, n), sts_attn.tree_attention(q, k, v, parents, lens, starts, 1.0)),
            (causal, sts_attn.masked_attention(q, k, v, lens, starts, 1.0))]
    for seen, got in runs:
        want, bound = attend64_channels(q64, k64, v64, seen, 1.0)
        got = got[0].cpu().numpy()
        assert np.isfinite(got).all()
        assert (np.abs(got - want) <= bound).all()
    acc = torch.zeros((1, KH, n), device="cuda")
    pair = torch.zeros((1, 2 * KH, D), device="cuda")
    pair[..., 0] = 1
    got = sts_attn.decode_ring_weights(pair, k, v, acc, lens, starts, 1.0)[0].cpu().numpy()
    want, bound = attend64_channels(q64[:1], k64, v64, np.ones((1, n), bool), 1.0)
    assert np.isfinite(got).all() and (np.abs(got - want[0]) <= bound[0]).all()


def test_every_row_counts_past_32_bits(gpu):
    """33 streams whose windows hold more than 2^32 rows together (69 GB), two query
    heads a K/V head.  Some thousand rows of each, the window's ends, the ring's seam
    and others, share the whole weight, and each has values of its own: a row that is
    missed or met twice shows in the mean."""
    import sts_attn
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB")
    B, M = 33, 0x7FFFFFF0 // 16
    assert B * M > 2 ** 32
    rng = np.random.default_rng(44)
    t = torch.zeros((B, 1, M, 4), device="cuda")  # K and V: dim 0 makes the scores, all four are values
    lens = np.full(B, M, np.int32)
    lens[1], lens[2] = M - 12345, 1000
    starts = rng.integers(0, M, B).astype(np.int32)
    lo = np.where(np.arange(B) % 3 == 0, lens // 3, 0).astype(np.int32)
    marked = []
    for b in range(B):
        n, first = int(lens[b]), int(lo[b])
        seam = (M - int(starts[b])) % M
        at = np.unique(np.concatenate([[first, first + 1, first - 1, n - 1, n - 2, seam, seam - 1],
                                       rng.integers(0, n, 1000)]))
        at = at[(at >= 0) & (at < n)]
        x = rng.uniform(-100, 100, (len(at), 4)).astype(np.float32)
        x[:, 0] = 80  # score 40: a row of zeros gets e^-40 of a marked one's weight
        slots = torch.from_numpy((int(starts[b]) + at) % M).cuda()
        t[b, 0, slots] = torch.from_numpy(x).cuda()
        marked.append((at, x.astype(np.float64)))
    q = torch.zeros((B, 1, 2, 4), device="cuda")
    q[..., 0] = 1
    dl, ds, dlo = (torch.from_numpy(x).cuda() for x in (lens, starts, lo[:, None].copy()))
    parents = torch.full((B, 1), -1, dtype=torch.int32, device="cuda")
    got = [sts_attn.tree_attention(q, t, t, parents, dl, ds, 0.5), sts_attn.masked_attention(q, t, t, dl, ds, 0.5, lo=dlo)]
    got = [x.cpu().numpy()[:, 0] for x in got]
    del t
    torch.cuda.empty_cache()
    for b in range(B):
        at, x = marked[b]
        for y, seen in ((got[0][b], at >= 0), (got[1][b], at >= lo[b])):
            # Equal weights: only the sums of the marked rows are rounded, and the
            # zero rows' weights, M e^-40 = 6e-10 of one row's, lost or kept.
            tol = (seen.sum() + 16) * 2.0 ** -24 * np.abs(x[seen]).mean(0) + 1e-6
            assert (np.abs(y - x[seen].mean(0)) <= tol).all(), b


def test_scores_are_short_sums(gpu):
    """Up to 16 query rows over f32 rows: the outputs' error in the norm.

    A score of standard deviation 3 is the sum of 128 products of variance
    9 (log2 e)^2 / 128 = v.  An addition in f32 that reaches x is off by a variance of
    (u x)^2 / 3 at most, and x^2 after k products is k v: one sum of all is off by
    u sqrt(8256 v / 3) = 20 u, four sums of 32 and their sums by
    u sqrt((4 * 528 + 256) v / 3) = 10.7 u, and q's rounding adds 2.5 u.  The weights,
    and with them the outputs, are off by ln 2 times that: 8.3e-7 and 4.5e-7."""
    import sts_attn
    B, G, D, n = 4, 8, 128, 1000
    w = Window(36, B, 4, n, D, [n, 800, 600, 400])
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    q = 3 * w.rng.standard_normal((B, 1, 4 * G, D)).astype(np.float32)
    dq = torch.from_numpy(q).cuda()
    acc = torch.zeros((B, 4, n), device="cuda")
    parents = torch.full((B, 1), -1, dtype=torch.int32, device="cuda")
    got = {"tree": sts_attn.tree_attention(dq, k, v, parents, dl, ds, scale_for(D)),
           "masked": sts_attn.masked_attention(dq, k, v, dl, ds, scale_for(D)),
           "weights": sts_attn.decode_ring_weights(dq[:, 0].contiguous(), k, v, acc, dl, ds, scale_for(D))[:, None]}
    want = np.stack([attend64_channels(q[b], w.rows(b, w.k), w.rows(b, w.v), np.ones((1, int(w.lens[b])), bool),
                                       scale_for(D))[0] for b in range(B)])
    for name, x in got.items():
        err = np.linalg.norm(x.cpu().numpy() - want) / np.linalg.norm(want)
        assert err <= 6e-7, f"{name}: {err:.2e}"
