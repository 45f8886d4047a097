"""K/V rows in pages on the GPU: append, gather and decode against 64-bit forms."""
import numpy as np
import pytest
import torch

import oracle
import sts_attn
from conftest import scale_for
from pages import DTYPES, Pool, stored, value64
from windows import attend64_channels, queries

pytestmark = pytest.mark.gpu


def bits(t):
    return t.view({4: torch.int32, 2: torch.int16, 1: torch.int8}[t.element_size()])


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------

def appended(pool, k_new, v_new, counts):
    """The pool's tensors after the append, from the definition."""
    want = {k: v if v is None else v.clone() for k, v in pool.data.items()}
    pages = len(want["k"])
    T = k_new.shape[1]
    for b in range(pool.B):
        L = max(0, int(pool.lens[b]))
        n = min(max(int(counts[b]), 0), T, L)
        for i in range(n):
            r = L - n + i
            page = int(pool.table[b, r // pool.R])
            if not 0 <= page < pages:
                continue
            for name, new in (("k", k_new), ("v", v_new)):
                x, s = stored(new[b, i], pool.rows)
                want[name][page, :, r % pool.R] = x
                if s is not None:
                    want[name + "_scale"][page, :, r % pool.R] = s
    return want


@pytest.mark.parametrize("rows,D,KH,R", [("f32", 128, 3, 16), ("f32", 4, 5, 32), ("f32", 100, 1, 64), ("bf16", 128, 2, 256),
                                         ("bf16", 8, 4, 16), ("bf16", 72, 3, 16), ("int8", 128, 2, 16), ("int8", 64, 5, 128),
                                         ("int8", 16, 1, 16), ("int8", 80, 3, 32)])
def test_append(gpu, rows, D, KH, R):
    """Rows of ragged streams land rounded in their places, bit for bit; every other byte stays."""
    lens = [0, 1, 7, R, R + 1, 2 * R + 3, -5, 40]
    pool = Pool(1, lens, KH, D, R, rows, bad=((5, 1),))
    T = 9
    counts = np.array([3, 9, 2, 9, 9, 9, 4, -1], np.int32)
    k_new, v_new = (pool.rng.standard_normal((len(lens), T, KH, D)).astype(np.float32) for _ in range(2))
    want = appended(pool, k_new, v_new, counts)
    cache, table, lens_ = pool.gpu()
    cache.append(torch.from_numpy(k_new).cuda(), torch.from_numpy(v_new).cuda(), table, lens_,
                 counts=torch.from_numpy(counts).cuda())
    for name in ("k", "v", "k_scale", "v_scale"):
        if want[name] is not None:
            assert torch.equal(bits(getattr(cache, name).cpu()), bits(want[name])), name


def edge_rows(D):
    """Rows at which rounding to 8 bits can go wrong."""
    rng = np.random.default_rng(5)
    e = np.zeros((14, D), np.float32)
    e[1, 0] = 127.0  # scale 1: codes halfway between two steps go to the even one
    e[1, 1:] = (np.arange(D - 1) % 60) - 29.5
    e[2, :2] = 127 * 2.0 ** -70, 1e-30  # below 2^-64: zeros
    e[3] = 2.0 ** -64
    e[4] = 3.4e38 * np.where(np.arange(D) % 2, 1, -0.5)
    e[5, D - 1] = np.inf
    e[6, 3] = np.nan
    e[7, :2] = -np.inf, np.nan
    e[8] = -1.0
    for i in range(9, 14):  # quotients within a rounding of halfway
        s = np.float32(rng.uniform(0.5, 2.0))
        e[i, 0] = np.float32(s * 127)
        scale = np.float32(float(e[i, 0]) / 127.0)
        x = ((np.arange(D - 1) % 100 + 0.5) * np.float64(scale)).astype(np.float32)
        e[i, 1:] = np.nextafter(x, np.float32([0, np.inf, x.mean()][i % 3]))
    return e


def test_append_8_bit_edges(gpu):
    D = 128
    rows = edge_rows(D)
    n = len(rows)
    pool = Pool(2, [n], 1, D, 16, "int8")
    new = rows[None, :, None, :]
    want = appended(pool, new, new[:, ::-1], [n])
    cache, table, lens = pool.gpu()
    cache.append(torch.from_numpy(new.copy()).cuda(), torch.from_numpy(new[:, ::-1].copy()).cuda(), table, lens)
    for name in ("k", "v"):
        assert torch.equal(getattr(cache, name).cpu(), want[name]), name
        s, t = getattr(cache, name + "_scale").cpu(), want[name + "_scale"]
        assert torch.equal(torch.isnan(s), torch.isnan(t)) and torch.equal(torch.nan_to_num(s), torch.nan_to_num(t))
    k, v = (torch.zeros((1, 1, n, D), device="cuda") for _ in range(2))
    cache.gather(table, lens, k, v)
    bad = torch.from_numpy(~np.isfinite(rows).all(1))
    assert torch.isnan(k[0, 0].cpu()[bad]).all()
    assert torch.isfinite(k[0, 0].cpu()[~bad]).all()


@pytest.mark.parametrize("rows,D", [("f32", 128), ("int8", 64), ("bf16", 40)])
def test_append_rotates_at_the_row_index(gpu, rows, D):
    R, KH, T = 16, 2, 5
    lens = [70, 5, 33]
    pool = Pool(3, lens, KH, D, R, rows)
    k_new, v_new = (pool.rng.standard_normal((3, T, KH, D)).astype(np.float32) for _ in range(2))
    tabs = oracle.rope_tables(D, 80)
    turned = np.concatenate([oracle.rope_apply(k_new[b:b + 1], lens[b] - T, tabs) for b in range(3)])
    want = appended(pool, turned, v_new, [T] * 3)
    cache, table, lens_ = pool.gpu()
    cache.append(torch.from_numpy(k_new).cuda(), torch.from_numpy(v_new).cuda(), table, lens_,
                 rope=sts_attn.RoPE(D, 80))
    for name in ("k", "v"):
        assert torch.equal(bits(getattr(cache, name).cpu()), bits(want[name])), name


def test_append_of_packed_rows(gpu):
    """Tokens of a packed qkv, no copy made."""
    B, T, H, KH, D, R = 3, 4, 6, 2, 64, 16
    pool = Pool(4, [20, 4, 9], KH, D, R, "int8")
    qkv = pool.rng.standard_normal((B, T, H + 2 * KH, D)).astype(np.float32)
    want = appended(pool, qkv[:, :, H:H + KH], qkv[:, :, H + KH:], [T] * B)
    cache, table, lens = pool.gpu()
    x = torch.from_numpy(qkv).cuda()
    cache.append(x[:, :, H:H + KH], x[:, :, H + KH:], table, lens)
    assert torch.equal(cache.k.cpu(), want["k"]) and torch.equal(cache.v.cpu(), want["v"])


# ---------------------------------------------------------------------------
# Gather
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("rows,D,KH,R,out", [("f32", 128, 2, 16, "f32"), ("f32", 20, 3, 64, "bf16"), ("bf16", 128, 2, 32, "f32"),
                                             ("bf16", 64, 1, 128, "bf16"), ("int8", 128, 3, 16, "f32"),
                                             ("int8", 48, 2, 4096, "bf16")])
def test_gather(gpu, rows, D, KH, R, out):
    """Rows from `first` on, to the bit; rows behind and other streams' stay; no page: zeros."""
    lens = [0, 1, 50, 2 * R + 5, 77, -3]
    first = np.array([0, 0, 13, R - 1, 90, 2], np.int32)
    M = 45
    pool = Pool(6, lens, KH, D, R, rows, bad=((3, 1),))
    cache, table, lens_ = pool.gpu()
    k, v = (torch.full((len(lens), KH, M, D), 7.5, dtype=DTYPES[out], device="cuda") for _ in range(2))
    for starts in (None, first):
        cache.gather(table, lens_, k, v, first=None if starts is None else torch.from_numpy(starts).cuda())
        for name, got in (("k", k.cpu()), ("v", v.cpu())):
            for b in range(len(lens)):
                x, there = pool.stream(b, name)
                x = np.where(there[None, :, None], x, 0.0)[:, 0 if starts is None else starts[b]:][:, :M]
                # One product in f32, then the caches' type.
                want = torch.from_numpy(x).float().to(DTYPES[out])
                assert torch.equal(got[b, :, :x.shape[1]], want), (name, b)
                assert (got[b, :, x.shape[1]:] == 7.5).all()
        k.fill_(7.5), v.fill_(7.5)


# ---------------------------------------------------------------------------
# Decode
# ---------------------------------------------------------------------------

def check_decode(pool, H, q=None, scale=None, got=None, **kw):
    D = pool.D
    scale = scale_for(D) if scale is None else scale
    if q is None:
        q = queries(pool.rng, pool.B, H, D)
    if got is None:
        cache, table, lens = pool.gpu()
        got = cache.decode(torch.from_numpy(q).cuda(), table, lens, scale, **kw).cpu().numpy()
    for b in range(pool.B):
        k, there = pool.stream(b, "k")
        v, _ = pool.stream(b, "v")
        if not there.any():
            assert (got[b] == 0).all(), b
            continue
        out, bound = attend64_channels(q[b:b + 1], k, v, there[None], scale)
        off = np.abs(got[b] - out[0])
        assert (off <= bound[0] + 1e-300).all(), (b, float((off / bound[0]).max()))
    return got


SHAPES = [("f32", 128, 4, 4, 16), ("f32", 64, 8, 2, 64), ("f32", 20, 3, 3, 16), ("f32", 100, 6, 2, 32),
          ("bf16", 128, 4, 4, 16), ("bf16", 64, 12, 4, 128), ("bf16", 8, 2, 2, 16), ("bf16", 72, 10, 2, 32),
          ("int8", 128, 4, 4, 16), ("int8", 64, 9, 3, 256), ("int8", 16, 2, 1, 16), ("int8", 80, 5, 1, 32),
          ("int8", 48, 4, 2, 64), ("f32", 4, 2, 2, 16), ("f32", 4, 6, 2, 16)]


@pytest.mark.parametrize("rows,D,H,KH,R", SHAPES)
def test_decode_lengths(gpu, rows, D, H, KH, R):
    """From no row at all to more than every split takes, on both sides of tiles and pages."""
    pool = Pool(7, [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 257, 511, 700, -1], KH, D, R, rows)
    check_decode(pool, H)


@pytest.mark.parametrize("rows", ["f32", "bf16", "int8"])
@pytest.mark.parametrize("group", [1, 2, 7, 8, 15, 16, 17, 33])
def test_decode_groups(gpu, rows, group):
    pool = Pool(8, [301, 1500], 2, 64, 32, rows)
    check_decode(pool, 2 * group)


@pytest.mark.parametrize("rows", ["f32", "bf16", "int8"])
@pytest.mark.parametrize("D", [80, 128])
@pytest.mark.parametrize("group", [9, 11, 12, 13, 16, 17, 33])
def test_decode_wide_groups(gpu, rows, D, group):
    """Groups whose outputs are more columns than a workgroup has threads, in splits that are merged
    at once and, for the longer streams, in clusters."""
    check_decode(Pool(27, [301, 1500, 5], 2, D, 32, rows), 2 * group)
    check_decode(Pool(28, [3003], 1, D, 64, rows), group)


@pytest.mark.parametrize("rows", ["f32", "bf16", "int8"])
@pytest.mark.parametrize("H,KH", [(12, 1), (16, 1), (29, 1), (80, 4)])
def test_decode_wide_groups_long(gpu, rows, H, KH):
    """The most splits there are, of up to sixteen heads a block."""
    check_decode(Pool(29, [18001], KH, 128, 256, rows), H)
    check_decode(Pool(30, [9000, 700, 0, 2001], KH, 128, 16, rows), H)


@pytest.mark.parametrize("rows", ["f32", "bf16", "int8"])
def test_decode_wide_groups_that_append(gpu, rows):
    """Blocks of sixteen heads all see the row that the first of them stores."""
    B, H, KH, D = 4, 50, 2, 128
    lens = [2000, 1, 33, 700]
    pool = Pool(31, lens, KH, D, 16, rows)
    qkv = torch.from_numpy(queries(pool.rng, B, H + 2 * KH, D)).cuda()
    q, k_new, v_new = qkv[:, :H], qkv[:, H:H + KH], qkv[:, H + KH:]
    one, table, lens_ = pool.gpu()
    got = one.decode(q, table, lens_, scale_for(D), k_new=k_new, v_new=v_new).cpu().numpy()
    want = appended(pool, k_new[:, None].cpu().numpy(), v_new[:, None].cpu().numpy(), [1] * B)
    for name in ("k", "v", "k_scale", "v_scale"):
        if want[name] is not None:
            assert torch.equal(bits(getattr(one, name).cpu()), bits(want[name])), name
    pool.data = want
    check_decode(pool, H, q=q.cpu().numpy(), got=got)


@pytest.mark.parametrize("rows", ["f32", "bf16", "int8"])
def test_decode_long(gpu, rows):
    """One stream whose splits are merged many at once, and one head of many rows."""
    check_decode(Pool(9, [20011], 1, 64, 256, rows), 3)
    check_decode(Pool(10, [9000, 3], 1, 128, 16, rows), 1)


@pytest.mark.parametrize("rows", ["f32", "bf16", "int8"])
def test_decode_many_streams(gpu, rows):
    """More streams than a wave looks at."""
    lens = np.random.default_rng(11).integers(0, 90, 131)
    check_decode(Pool(12, lens, 2, 64, 16, rows), 4)


@pytest.mark.parametrize("rows,H", [("f32", 1), ("bf16", 2), ("int8", 3), ("int8", 1)])
def test_decode_many_streams_in_splits(gpu, rows, H):
    """More streams than a wave looks at, with few heads, so that each is split."""
    lens = np.r_[np.random.default_rng(24).integers(0, 700, 68), 900, 1]
    check_decode(Pool(25, lens, 1, 64, 32, rows), H)


@pytest.mark.parametrize("D", [64, 128])
def test_decode_many_heads_over_long_rows(gpu, D):
    """8-bit rows of more than a thousand heads, one stream long: fewer workgroups a CU."""
    lens = np.r_[np.random.default_rng(36).integers(0, 40, 65), 2050]
    check_decode(Pool(37, lens, 16, D, 64, "int8"), 16)


@pytest.mark.parametrize("rows", ["f32", "bf16", "int8"])
def test_decode_missing_pages(gpu, rows):
    """Rows of an entry that is no page have no part: in the middle, first, last, all of them."""
    bad = [(0, 0), (0, 5), (1, 1), (2, 3), (3, 0), (3, 1)]
    pool = Pool(13, [100, 64, 55, 20, 300], 2, 128, 16, rows, bad=bad)
    check_decode(pool, 4)


@pytest.mark.parametrize("rows", ["f32", "bf16", "int8"])
def test_decode_unequal_rows_and_channels(gpu, rows):
    """Rows, channels and queries of very different sizes: every output channel is held to its own."""
    def values(rng, shape):
        x = rng.standard_normal(shape) * np.exp(rng.uniform(-9, 3, (shape[0], 1, 1)))
        if rows != "int8":
            x = x * np.exp2(rng.integers(-12, 12, (1, 1, shape[2])))
        return x
    pool = Pool(14, [600, 47], 2, 128, 64, rows, values=values)
    q = queries(pool.rng, 2, 8, 128) * np.exp2(-np.arange(128) % 5).astype(np.float32)
    check_decode(pool, 8, q=q, scale=0.02)


@pytest.mark.parametrize("rows", ["f32", "bf16", "int8"])
def test_decode_sharp(gpu, rows):
    """Scores of hundreds: the weights of all rows but a few vanish."""
    pool = Pool(15, [500, 80], 2, 64, 16, rows)
    check_decode(pool, 4, scale=20.0)


def test_decode_small_and_large_values(gpu):
    for rows, size in (("f32", 1e30), ("bf16", 1e30), ("int8", 1e30), ("f32", 1e-18), ("int8", 1e-18)):
        pool = Pool(16, [300], 1, 64, 16, rows, values=lambda rng, s: rng.standard_normal(s) * size)
        check_decode(pool, 2, scale=0.1 / size)


def test_decode_not_a_number(gpu):
    """A row that is NaN shows in the heads that see it and in no other stream."""
    for rows in ("f32", "int8"):
        pool = Pool(17, [40, 40], 2, 64, 16, rows)
        pg, ro = int(pool.table[0, 1]), 3
        if rows == "int8":
            pool.data["k_scale"][pg, 1, ro] = float("nan")
        else:
            pool.data["k"][pg, 1, ro] = float("nan")
        cache, table, lens = pool.gpu()
        q = torch.from_numpy(queries(pool.rng, 2, 4, 64)).cuda()
        out = cache.decode(q, table, lens, 0.1).cpu()
        assert torch.isnan(out[0, 2:]).all()
        assert torch.isfinite(out[0, :2]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("H", [2, 6])
def test_decode_infinite_scores(gpu, H):
    """Rows whose score is -infinity have no part, and a stream of such rows alone gets zeros."""
    pool = Pool(18, [40, 5, 300], 2, 64, 16)
    cache, table, lens = pool.gpu()
    q = queries(pool.rng, 3, H, 64)
    q[:, :, 3] = np.abs(q[:, :, 3]) + 0.5
    seen = [np.ones(n, bool) for n in (40, 5, 300)]
    seen[0][[7, 39]] = False
    seen[1][:] = False
    seen[2][64:] = False
    for b, on in enumerate(seen):
        for r in np.flatnonzero(~on):
            cache.k[int(pool.table[b, r // 16]), :, r % 16, 3] = float("-inf")
    got = cache.decode(torch.from_numpy(q).cuda(), table, lens, 0.1).cpu().numpy()
    for b in (0, 2):
        out, bound = attend64_channels(q[b:b + 1], pool.stream(b, "k")[0], pool.stream(b, "v")[0], seen[b][None], 0.1)
        assert (np.abs(got[b] - out[0]) <= bound[0]).all()
    assert (got[1] == 0).all()


@pytest.mark.parametrize("rows,D,H,KH", [("f32", 128, 4, 4), ("bf16", 64, 6, 2), ("int8", 128, 4, 4), ("int8", 32, 40, 2),
                                         ("f32", 36, 34, 2), ("bf16", 128, 8, 8)])
@pytest.mark.parametrize("rope", [False, True])
def test_decode_that_appends(gpu, rows, D, H, KH, rope):
    """The step leaves what append leaves and gives what decode after it gives, to the bit."""
    lens = [1, 16, 17, 0, 65, 300, 129]
    B = len(lens)
    pool = Pool(18, lens, KH, D, 16, rows, bad=((4, 4),))
    qkv = torch.from_numpy(queries(pool.rng, B, H + 2 * KH, D)).cuda()
    q, k_new, v_new = qkv[:, :H], qkv[:, H:H + KH], qkv[:, H + KH:]
    r = sts_attn.RoPE(D, 400) if rope else None
    one, table, lens_ = pool.gpu()
    two, _, _ = pool.gpu()
    one.append(k_new[:, None], v_new[:, None], table, lens_, rope=r)
    a = one.decode(q, table, lens_, scale_for(D), rope=r)
    b = two.decode(q, table, lens_, scale_for(D), k_new=k_new, v_new=v_new, rope=r)
    for name in ("k", "v", "k_scale", "v_scale"):
        if getattr(one, name) is not None:
            assert torch.equal(bits(getattr(one, name)), bits(getattr(two, name))), name
    assert torch.equal(a, b)
    # The queries turned at the newest row's index, against 64 bits.
    qn = q.cpu().numpy().copy()
    if rope:
        tabs = oracle.rope_tables(D, 400)
        for i, n in enumerate(lens):
            if n:
                qn[i] = oracle.rope_apply(qn[i][None, None], n - 1, tabs)[0, 0]
    for name in ("k", "v", "k_scale", "v_scale"):
        pool.data[name] = None if getattr(two, name) is None else getattr(two, name).cpu()
    check_decode(pool, H, q=qn, got=b.cpu().numpy())


def test_decode_max_rows(gpu):
    """lens above max_rows are taken as max_rows."""
    pool = Pool(19, [200, 90, 100], 2, 64, 16, "bf16")
    q = queries(pool.rng, 3, 4, 64)
    cache, table, lens = pool.gpu()
    got = cache.decode(torch.from_numpy(q).cuda(), table, lens, 0.125, max_rows=100).cpu().numpy()
    pool.lens = np.minimum(pool.lens, 100)
    check_decode(pool, 4, q=q, scale=0.125, got=got)


def test_pool_past_4_gb(gpu):
    """Rows beyond 2^32 bytes and 2^31 rows' worth of them, in and out."""
    pages, KH, R, D = 2300, 4, 4096, 128  # 4.8 GB of codes
    cache = sts_attn.PagedKV.empty(pages, R, KH, D, torch.int8)
    table = torch.tensor([[pages - 1, 0], [1, pages - 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([4100, 4099], dtype=torch.int32, device="cuda")
    rng = np.random.default_rng(20)
    x = rng.standard_normal((2, 4100, KH, D)).astype(np.float32)
    new = torch.from_numpy(x).cuda()
    counts = lens.clone()
    cache.append(new, new, table, lens, counts=counts)
    q = queries(rng, 2, 8, D)
    got = cache.decode(torch.from_numpy(q).cuda(), table, lens, scale_for(D)).cpu().numpy()
    k, v = (torch.zeros((2, KH, 4100, D), device="cuda") for _ in range(2))
    cache.gather(table, lens, k, v)
    for b in range(2):
        n = int(lens[b])
        rows = value64(*stored(x[b, :n], "int8")).transpose(0, 1)
        assert torch.equal(k[b, :, :n].cpu(), rows.float()) and torch.equal(v[b, :, :n].cpu(), rows.float())
        out, bound = attend64_channels(q[b:b + 1], rows.numpy(), rows.numpy(), np.ones((1, n), bool), scale_for(D))
        assert (np.abs(got[b] - out[0]) <= bound[0]).all()


@pytest.mark.parametrize("H", [1, 3])
def test_rows_past_2_32(gpu, H):
    """Row numbers past 2^32, of codes and of scales, in and out.  (K and V are one memory, to which
    append gives the same rows twice: 86 GB instead of 172.)"""
    KH, R, D = 1, 4096, 16
    pages = 2 ** 32 // R + 3
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB of GPU memory")
    x = torch.empty((pages, KH, R, D), dtype=torch.int8, device="cuda")
    s = torch.empty((pages, KH, R), device="cuda")
    cache = sts_attn.PagedKV(x, x, s, s)
    half = 2 ** 31 // R
    t = np.array([[pages - 1, half - 1, pages - 2], [0, half, pages - 3]], np.int32)
    table = torch.from_numpy(t).cuda()
    n = [2 * R + 70, 2 * R + 9]
    lens = torch.tensor(n, dtype=torch.int32, device="cuda")
    rng = np.random.default_rng(32)
    new = rng.standard_normal((2, n[0], KH, D)).astype(np.float32)
    dev = torch.from_numpy(new).cuda()
    cache.append(dev, dev, table, lens, counts=lens)
    k, v = (torch.zeros((2, KH, n[0], D), device="cuda") for _ in range(2))
    cache.gather(table, lens, k, v)
    q = queries(rng, 2, H, D)
    got = cache.decode(torch.from_numpy(q).cuda(), table, lens, scale_for(D)).cpu().numpy()
    row = torch.from_numpy(queries(rng, 2, KH, D)).cuda()
    step = cache.decode(torch.from_numpy(q).cuda(), table, lens, scale_for(D), k_new=row, v_new=row).cpu().numpy()
    for b in range(2):
        codes, scales = stored(new[b, :n[b]], "int8")
        for i in range(3):  # where the definition puts them
            at = slice(i * R, min((i + 1) * R, n[b]))
            m = min(R, n[b] - i * R) - (i == 2)  # (the step has written over the last)
            assert torch.equal(x[t[b, i], 0, :m].cpu(), codes[at][:m, 0])
            assert torch.equal(s[t[b, i], 0, :m].cpu(), scales[at][:m, 0])
        rows = value64(codes, scales).transpose(0, 1)
        assert torch.equal(k[b, :, :n[b]].cpu(), rows.float()) and torch.equal(v[b], k[b])
        last = value64(*stored(row[b].cpu().numpy(), "int8"))
        other = rows.clone()
        other[:, -1] = last
        for out, r in ((got[b], rows), (step[b], other)):
            want, bound = attend64_channels(q[b:b + 1], r.numpy(), r.numpy(), np.ones((1, n[b]), bool), scale_for(D))
            assert (np.abs(out - want[0]) <= bound[0]).all()
    del cache, x, s
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------
# Streams, graphs, together
# ---------------------------------------------------------------------------

def test_decode_in_a_graph(gpu):
    """Replayed with other rows, lens and queries, beside eager calls."""
    pool = Pool(21, [400, 37, 1000], 4, 128, 64, "int8")
    cache, table, lens = pool.gpu()
    q = torch.from_numpy(queries(pool.rng, 3, 4, 128)).cuda()
    k_new, v_new = (torch.randn((3, 4, 128), device="cuda") for _ in range(2))
    s = torch.cuda.Stream()
    out = torch.empty((3, 4, 128), device="cuda")
    with torch.cuda.stream(s):
        cache.decode(q, table, lens, 0.1, k_new=k_new, v_new=v_new, out=out)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        cache.decode(q, table, lens, 0.1, k_new=k_new, v_new=v_new, out=out)
    for turn in range(4):
        q.copy_(torch.randn_like(q))
        k_new.copy_(torch.randn_like(q))
        lens.sub_(3 * turn)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, cache.decode(q, table, lens, 0.1))


def test_calls_on_another_stream(gpu):
    """Results of a call on a stream that is busy come from that stream's memory."""
    pool = Pool(22, [900, 64], 2, 64, 16, "bf16")
    cache, table, lens = pool.gpu()
    q = torch.from_numpy(queries(pool.rng, 2, 4, 64)).cuda()
    want = cache.decode(q, table, lens, 0.1)
    k, v = (torch.zeros((2, 2, 900, 64), device="cuda") for _ in range(2))
    cache.gather(table, lens, k, v)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.randn((4000, 4000), device="cuda") @ torch.randn((4000, 4000), device="cuda")
    outs = [cache.decode(q, table, lens, 0.1, stream=s) for _ in range(3)]
    k2, v2 = (torch.zeros_like(k) for _ in range(2))
    s.wait_stream(torch.cuda.current_stream())
    cache.gather(table, lens, k2, v2, stream=s)
    s.synchronize()
    for o in outs:
        assert torch.equal(o, want)
    assert torch.equal(k, k2) and torch.equal(v, v2)


def test_two_streams_at_once(gpu):
    """Split decodes that run side by side on two streams keep to their own workspaces."""
    pools = [Pool(26 + i, [3000 - 500 * i, 800], 2, 128, 32, rows) for i, rows in enumerate(("int8", "f32"))]
    calls = []
    for pool, H in zip(pools, (2, 6)):
        cache, table, lens = pool.gpu()
        calls.append((cache, torch.from_numpy(queries(pool.rng, 2, H, 128)).cuda(), table, lens))
    want = [c.decode(q, t, n, 0.1) for c, q, t, n in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(20):
        for i, (c, q, t, n) in enumerate(calls):
            got[i].append(c.decode(q, t, n, 0.1, stream=streams[i]))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


@pytest.mark.parametrize("rows", ["f32", "bf16", "int8"])
def test_prompt_then_tokens(gpu, rows):
    """A prompt's rows appended and read back for its chunk's attention, then tokens one by one:
    together as a server uses them, every step against 64 bits over what the pages stand for."""
    B, H, KH, D, R, S = 2, 4, 2, 64, 16, 37
    scale = scale_for(D)
    rng = np.random.default_rng(23)
    cache = sts_attn.PagedKV.empty(8, R, KH, D, DTYPES[rows])
    table = torch.tensor([[5, 0, 3], [1, 7, 2]], dtype=torch.int32, device="cuda")
    lens = torch.full((B,), S, dtype=torch.int32, device="cuda")
    rope = sts_attn.RoPE(D, 48)
    tabs = oracle.rope_tables(D, 48)
    k_new, v_new = (rng.standard_normal((B, S, KH, D)).astype(np.float32) for _ in range(2))
    cache.append(torch.from_numpy(k_new).cuda(), torch.from_numpy(v_new).cuda(), table, lens, rope=rope, max_rows=48)
    kept = {"k": [oracle.rope_apply(k_new[b:b + 1], 0, tabs)[0] for b in range(B)], "v": [v_new[b] for b in range(B)]}

    def rows64(name, b):
        return value64(*stored(kept[name][b], rows)).transpose(0, 1).numpy()

    k, v = (torch.zeros((B, KH, 48, D), device="cuda") for _ in range(2))
    cache.gather(table, lens, k, v)
    q = queries(rng, B, S, H, D)
    starts = torch.zeros(B, dtype=torch.int32, device="cuda")
    got = sts_attn.masked_attention(torch.from_numpy(q).cuda(), k, v, lens, starts, scale).cpu().numpy()
    for b in range(B):
        out, bound = attend64_channels(q[b], rows64("k", b), rows64("v", b), np.tril(np.ones((S, S), bool)), scale)
        assert (np.abs(got[b] - out) <= bound).all()
    for step in range(6):
        lens += 1
        qkv = queries(rng, B, H + 2 * KH, D)
        x = torch.from_numpy(qkv).cuda()
        got = cache.decode(x[:, :H], table, lens, scale, k_new=x[:, H:H + KH], v_new=x[:, H + KH:], rope=rope,
                           max_rows=48).cpu().numpy()
        turned = oracle.rope_apply(qkv[:, None], S + step, tabs)[:, 0]
        for b in range(B):
            kept["k"][b] = np.concatenate([kept["k"][b], turned[b][None, H:H + KH]])
            kept["v"][b] = np.concatenate([kept["v"][b], qkv[b][None, H + KH:]])
            n = S + step + 1
            out, bound = attend64_channels(turned[b:b + 1, :H], rows64("k", b), rows64("v", b), np.ones((1, n), bool), scale)
            assert (np.abs(got[b] - out[0]) <= bound[0]).all(), (step, b)
