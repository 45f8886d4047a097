"""Paged K/V rows for the tests, what they stand for in 64 bits, and the verdict on a
draft in exact fractions.

A Pool holds ragged streams' rows anywhere in its pages; every row that is no stream's
is NaN, so that a kernel that lets one through shows it.
"""
from fractions import Fraction

import numpy as np
import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "int8": torch.int8}


def stored(x, rows):
    """(what the pages hold of f32 rows x [..., D], its scales or None): from the definition."""
    x = np.asarray(x, np.float32)
    if rows != "int8":
        return torch.from_numpy(x).to(DTYPES[rows]), None
    top = np.abs(x).max(-1).astype(np.float64)
    bad = ~np.isfinite(x).all(-1)
    scale = np.where(top < 2.0 ** -64, 0.0, top / 127.0).astype(np.float32)
    scale[bad] = np.nan
    by = np.where(scale > 0, scale, 1.0).astype(np.float64)[..., None]
    codes = np.where((scale > 0)[..., None], np.rint(np.where(bad[..., None], 0, x).astype(np.float64) / by), 0)
    return torch.from_numpy(codes.astype(np.int8)), torch.from_numpy(scale)


def value64(t, scale):
    """What stored rows stand for, in 64 bits."""
    x = t.double()
    return x if scale is None else x * scale.double()[..., None]


class Pool:
    def __init__(self, seed, lens, KH, D, R, rows="f32", spare=3, bad=(), values=None):
        """bad: (stream, page index) pairs whose table entry names no page."""
        rng = self.rng = np.random.default_rng(seed)
        self.lens = np.asarray(lens, np.int32)
        B = len(self.lens)
        self.B, self.KH, self.D, self.R, self.rows = B, KH, D, R, rows
        L = np.maximum(self.lens, 0)
        used = -(-L // R)
        pages = int(used.sum()) + spare
        where = rng.permutation(pages)
        self.table = np.full((B, max(1, int(used.max()))), -1, np.int32)
        for b, at in enumerate(np.cumsum(used) - used):
            self.table[b, :used[b]] = where[at:at + used[b]]
        shape = (pages, KH, R, D)
        self.data = {}
        for name in ("k", "v"):
            if rows == "int8":
                t = torch.full(shape, 99, dtype=torch.int8)
                s = torch.full(shape[:3], float("nan"))
            else:
                t, s = torch.full(shape, float("nan"), dtype=DTYPES[rows]), None
            for b in range(B):
                r = np.arange(L[b])
                x = rng.standard_normal((L[b], KH, D)) if values is None else values(rng, (L[b], KH, D))
                x, sx = stored(x, rows)
                pg, ro = torch.from_numpy(self.table[b][r // R].astype(np.int64)), torch.from_numpy(r % R)
                t[pg, :, ro] = x
                if s is not None:
                    s[pg, :, ro] = sx
            self.data[name], self.data[name + "_scale"] = t, s
        for b, page in bad:
            self.table[b, page] = [-1, pages, -2 ** 31, 2 ** 31 - 1][(b + page) % 4]

    def gpu(self):
        """A sts_attn.PagedKV of the pool's rows, table and lens."""
        import sts_attn
        d = {k: v if v is None else v.cuda() for k, v in self.data.items()}
        return (sts_attn.PagedKV(d["k"], d["v"], d["k_scale"], d["v_scale"]), torch.from_numpy(self.table).cuda(),
                torch.from_numpy(self.lens).cuda())

    def stream(self, b, name):
        """(stream b's rows [KH, L, D] in 64 bits, which of them there are [L])."""
        r = np.arange(max(0, int(self.lens[b])))
        pg = self.table[b][r // self.R].astype(np.int64)
        there = (pg >= 0) & (pg < len(self.data[name]))
        pg, ro = torch.from_numpy(np.where(there, pg, 0)), torch.from_numpy(r % self.R)
        x, s = self.data[name][pg, :, ro], self.data[name + "_scale"]
        x = value64(x, None if s is None else s[pg, :, ro])
        return x.transpose(0, 1).numpy(), there


def verdict(target, draft, tokens, parents, n, rand):
    """(path, next) of one stream, from the definition in exact fractions."""
    T, V = target.shape

    def weights(row):
        return [Fraction(float(x)) if x > 0 else Fraction(0) for x in row]

    if n == 0:
        return [], -1
    cur, path = 0, [0]
    r, m, q = weights(target[0]), Fraction(1), None if draft is None else weights(draft[0])
    for i in range(1, n):
        if parents[i] != cur or not 0 <= parents[i] < i:
            continue
        x = int(tokens[i])
        known = 0 <= x < V
        qx = Fraction(1) if q is None else q[x] if known else Fraction(0)
        if known and Fraction(float(rand[i])) * qx * m < r[x]:
            cur = i
            path.append(i)
            r, m, q = weights(target[i]), Fraction(1), None if draft is None else weights(draft[i])
            continue
        rest = ([Fraction(0) if y == x else r[y] for y in range(V)] if q is None
                else [max(Fraction(0), a / m - z) for a, z in zip(r, q)])
        total = sum(rest)
        if total > 0:
            r, m = rest, total
    point, run = Fraction(float(rand[0])) * sum(r), Fraction(0)
    for y in range(V):
        run += r[y]
        if run > point:
            return path, y
    return path, -1
