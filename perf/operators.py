"""Operators over the K/V ring beside plain decode and prefill, as a program that serves with them calls them.

    tree      tree_attention: drafted nodes of each stream against its window, every node seeing
              the committed rows, its ancestors and itself
    masked    masked_attention: a chunk (or one token) of each stream under a row range per query
              (causal, documents, prefix, sliding window), with capped scores and a distance bias
    weights   decode_ring_weights: one token of each stream, and what each cached row got of the
              attention added to its account
    evict     evict_ring: each stream's window cut down to the rows that got most, and the newest

Windows are ring windows: row r of stream b is slot (starts[b] + r) % ring of its caches
[batch][kv_heads][ring][dim]; K and V are float32 or bfloat16, queries and results float32.

listed() holds the fixed cases, draw() more of the same ranges, prepare() makes inputs from a seed,
run() makes one pass (plain torch operations, or with `own` the framework's entry points), exact()
says in 64 bits what run() returns, work() what a pass cannot do without.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
KV = {"f32": torch.float32, "bf16": torch.bfloat16}
# The temporal transformer: 32 heads x 128, a ring of 3000 rows.
TEMPORAL = dict(heads=32, kv_heads=32, dim=128, ring=3000)


def _framework():
    if "sts_attn" not in sys.modules:
        sys.path.insert(0, os.path.join(ROOT, "sts-web_amd"))
    import sts_attn
    return sts_attn


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    tree = dict(TEMPORAL, kind="tree", kv="f32")
    masked = dict(TEMPORAL, kind="masked", kv="f32", batch=1, mask="causal", docs=0, softcap=0.0, bias=False)
    weights = dict(TEMPORAL, kind="weights", kv="f32")
    evict = dict(TEMPORAL, kind="evict", kv="f32")
    return [
        # A short draft early in one conversation: a few microseconds, latency counts.
        dict(tree, name="tree_8_early", batch=1, nodes=8, depth=4, shortest=257, longest=257),
        # A wide draft late in one conversation: the whole ring is read.
        dict(tree, name="tree_60_full_ring", batch=1, nodes=60, depth=7, shortest=3000, longest=3000),
        # A server's 16 conversations of their own ages and drafts, shared K/V heads, bf16 caches.
        dict(tree, name="tree_16_streams_bf16", batch=16, nodes=16, depth=5, kv_heads=8, kv="bf16", shortest=130,
             longest=2999),
        # 24 conversations with deep drafts and shared K/V heads: many query rows on every K/V row.
        dict(tree, name="tree_24_streams_wide", batch=24, nodes=40, depth=12, kv_heads=8, shortest=900, longest=3000),
        # One token of 9 streams that look back a while with a distance bias.
        dict(masked, name="masked_1_token_window", batch=9, seq=1, mask="window", docs=700, bias=True, shortest=31,
             longest=2777),
        # A prompt chunk of packed documents behind an earlier one, capped scores.
        dict(masked, name="masked_512_documents", seq=512, mask="documents", docs=5, softcap=30.0, shortest=768,
             longest=768),
        # A long prompt whose first part sees itself in both directions, shared K/V heads, bf16 caches.
        dict(masked, name="masked_1000_prefix_bf16", seq=1000, mask="prefix", docs=601, kv_heads=8, kv="bf16",
             shortest=2600, longest=2600),
        # One token late in one conversation, every row's share of the attention kept.
        dict(weights, name="weights_full_ring", batch=1, shortest=3000, longest=3000),
        # A server's 64 conversations, of their own ages.
        dict(weights, name="weights_64_streams", batch=64, shortest=128, longest=3000),
        # Small heads in groups, bf16 caches, a longer ring.
        dict(weights, name="weights_7_streams_bf16", batch=7, heads=24, kv_heads=8, dim=64, ring=20011, kv="bf16",
             shortest=5, longest=20011),
        # One conversation's ring halved.
        dict(evict, name="evict_full_ring", batch=1, shortest=3000, longest=3000, keep=1500, recent=256),
        # 20 conversations trimmed at once, some of which need no trimming.
        dict(evict, name="evict_20_streams", batch=20, kv_heads=8, shortest=700, longest=2963, keep=1111, recent=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "masked", "masked", "weights", "weights", "evict"])
    heads, group, dim = rng.choice([(32, 1, 128), (32, 4, 128), (16, 1, 64), (24, 3, 64), (32, 8, 128), (12, 2, 96),
                                    (20, 5, 80)])
    ring = rng.randint(1400, 3000)
    longest = _log(rng, 40, ring)
    case = dict(kind=kind, heads=heads, kv_heads=heads // group, dim=dim, ring=ring, kv=rng.choice(["f32", "f32", "bf16"]),
                batch=_log(rng, 1, 24), longest=longest, shortest=rng.randint(1, longest))
    if kind == "tree":
        nodes = _log(rng, 1, 40)
        return dict(case, nodes=nodes, depth=rng.randint(1, min(nodes, 12)))
    if kind == "masked":
        seq = _log(rng, 1, 300)
        mask = rng.choice(["causal", "documents", "prefix", "window"])
        batch = max(1, min(case["batch"], 600 // seq))
        docs = {"causal": 0, "documents": rng.randint(1, 9), "prefix": rng.randint(0, longest),
                "window": _log(rng, 1, longest)}[mask]
        return dict(case, batch=batch, seq=seq, mask=mask, docs=docs, softcap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                    bias=rng.random() < 0.4)
    if kind == "weights":
        return case
    keep = rng.randint(1, longest)
    return dict(case, keep=keep, recent=rng.randint(0, keep))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _lengths(case):
    """The streams' window lengths: spread evenly from the shortest to the longest."""
    n = case["batch"]
    return np.linspace(case["longest"], case["shortest"], n).round().astype(np.int64)


def _counts(case, lens):
    """How many nodes or queries each stream has: all of them in the longest, fewer in others; a window may be shorter."""
    full = case["nodes"] if case["kind"] == "tree" else case["seq"]
    part = np.array([full - (full * (i % 4)) // 5 for i in range(len(lens))], np.int64)
    return np.minimum(part, lens)


def _spans(case, length, count):
    """(lo, hi) of a stream's `count` queries, its last rows, in a window of `length` rows."""
    row = np.arange(length - count, length)
    lo, hi = np.zeros(count, np.int64), row + 1
    if case["mask"] == "documents":  # documents of unequal lengths, the first one the longest
        edges = np.unique((length * (np.arange(case["docs"]) / case["docs"]) ** 0.8).astype(np.int64))
        lo = edges[np.searchsorted(edges, row, side="right") - 1]
    elif case["mask"] == "prefix":
        hi = np.maximum(hi, min(case["docs"], length))
    elif case["mask"] == "window":
        lo = np.maximum(row + 1 - case["docs"], 0)
    return lo, hi


def _tree(rs, count, nodes, depth):
    """Parents of a draft: each node hangs on an earlier one (or on the last committed row, -1) above the depth limit."""
    parents, level = np.full(nodes, -1, np.int32), np.zeros(nodes, np.int64)
    for i in range(1, count):
        p = rs.randint(-1, i)
        if p >= 0 and level[p] + 1 < depth:
            parents[i], level[i] = p, level[p] + 1
    return parents


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 2654435761 % (1 << 62))
    rs = np.random.RandomState(int(seed) * 2654435761 % (1 << 32))
    B, H, KH, D, M = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "ring"))
    kind = case["kind"]

    def put(a, dtype=torch.int32):
        return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).to(DEV)

    order = rs.permutation(B)
    lens = _lengths(case)[order]
    s = dict(case=case, kind=kind, lens=put(lens), starts=put(rs.randint(0, M, B)), scale=float(np.float32(D) ** np.float32(-0.5)))
    s["k"] = torch.randn((B, KH, M, D), generator=g, device=DEV).to(KV[case["kv"]])
    s["v"] = torch.randn((B, KH, M, D), generator=g, device=DEV).to(KV[case["kv"]])
    if kind in ("weights", "evict"):
        # Few rows hold most of what was given so far; many have next to nothing, some nothing at all.
        w = torch.rand((B, KH, M), generator=g, device=DEV)
        s["weights"] = torch.where(w > 0.2, 40.0 * w ** 9, torch.zeros_like(w))
    if kind == "evict":
        return s
    n = {"tree": case.get("nodes"), "masked": case.get("seq"), "weights": 1}[kind]
    # Heads look sharply or broadly: scores of standard deviation 0.5 to 3.
    sharp = 0.5 + 2.5 * torch.rand((H, 1), generator=g, device=DEV)
    s["q"] = torch.randn((B, n, H, D), generator=g, device=DEV) * sharp
    if kind == "weights":
        s["q"] = s["q"].reshape(B, H, D)
        return s
    counts = _counts(case, _lengths(case))[order]
    s["counts"] = put(counts)
    if kind == "tree":
        s["parents"] = put(np.stack([_tree(rs, c, n, case["depth"]) for c in counts]))
        return s
    lo, hi = np.zeros((B, n), np.int64), np.zeros((B, n), np.int64)
    for b in range(B):
        lo[b, :counts[b]], hi[b, :counts[b]] = _spans(case, int(lens[b]), int(counts[b]))
    s["lo"], s["hi"] = put(lo), put(hi)
    s["slopes"] = put(2.0 ** (-8.0 * (np.arange(H) + 1) / H), torch.float32) if case["bias"] else None
    return s


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------

def _window_rows(s):
    """The window row that each slot holds, [batch][ring]; at or past the length: none."""
    M = s["k"].shape[2]
    return (torch.arange(M, device=DEV) - s["starts"][:, None].long()) % M


def _attend(scores, seen, v, shape):
    """softmax over the seen slots times V: scores [B][KH][group][n][M], seen broadcast over them."""
    B, KH, G, n, M = scores.shape
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.matmul(p.reshape(B, KH, G * n, M), v.float())
    return out.reshape(B, KH, G, n, -1).permute(0, 3, 1, 2, 4).reshape(shape), p


def _scores(s, q):
    """scale * q.k of every query with every slot, [B][KH][group][n][M]."""
    B, n, H, D = q.shape
    KH, M = s["k"].shape[1:3]
    rows = q.reshape(B, n, KH, H // KH, D).permute(0, 2, 3, 1, 4).reshape(B, KH, -1, D)
    x = torch.matmul(rows * s["scale"], s["k"].float().transpose(-1, -2))
    return x.reshape(B, KH, H // KH, n, M)


def _plain_tree(s):
    q = s["q"]
    B, n = q.shape[:2]
    row, lens, counts = _window_rows(s), s["lens"].long()[:, None], s["counts"].long()[:, None]
    # Ancestors: powers of (1 + the parent relation), entry (i, j) > 0 where j is i or above it.
    node = torch.arange(n, device=DEV)
    step = (s["parents"].long()[:, :, None] == node).double() + torch.eye(n, device=DEV, dtype=torch.float64)
    above = torch.linalg.matrix_power(step, s["case"]["depth"]) > 0.5  # [B][i][j]
    j = row - (lens - counts)
    drafted = torch.gather(above, 2, j.clamp(0, n - 1)[:, None, :].expand(-1, n, -1))
    seen = (row < lens)[:, None] & ((j < 0)[:, None] | drafted) & (node < counts)[:, :, None]
    return _attend(_scores(s, q), seen[:, None, None], s["v"], q.shape)[0]


def _plain_masked(s):
    q, case = s["q"], s["case"]
    n = q.shape[1]
    row, lens, counts = _window_rows(s)[:, None], s["lens"].long()[:, None, None], s["counts"].long()[:, None, None]
    x = _scores(s, q)
    if case["softcap"] > 0:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    if s["slopes"] is not None:
        at = lens - counts + torch.arange(n, device=DEV)[:, None]
        slopes = s["slopes"].reshape(1, x.shape[1], x.shape[2], 1, 1)
        x = x - slopes * (at - row).abs().float()[:, None, None]
    seen = (row >= s["lo"].long()[..., None]) & (row < s["hi"].long()[..., None]) & (row < lens)
    return _attend(x, seen[:, None, None], s["v"], q.shape)[0]


def _plain_weights(s):
    q = s["q"][:, None]
    seen = _window_rows(s) < s["lens"].long()[:, None]
    out, p = _attend(_scores(s, q), seen[:, None, None, None], s["v"], q.shape)
    s["weights"] += p.sum((2, 3))
    return {"out": out[:, 0], "weights": s["weights"]}


def _plain_evict(s):
    k, v, w, case = s["k"], s["v"], s["weights"], s["case"]
    B, KH, M, D = k.shape
    keep, recent = case["keep"], case["recent"]
    lens, starts = s["lens"].long()[:, None, None], s["starts"].long()[:, None, None]
    r = torch.arange(M, device=DEV)
    ordered = torch.gather(w, 2, ((starts + r) % M).expand(B, KH, M))
    # The newest rows first of all, rows outside the window last; among equals the oldest first.
    rank = torch.where(r < lens - recent, ordered, torch.full_like(ordered, math.inf))
    rank = torch.where(r < lens, rank, torch.full_like(rank, -math.inf))
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    j = torch.arange(keep, device=DEV)
    whole = lens <= keep  # nothing to evict: every row stays where it is
    kept = torch.where(whole, torch.minimum(j, lens - 1), kept)
    src = (starts + kept) % M
    dst = (starts + torch.where(whole, kept, lens - keep + j)) % M
    dst = dst.expand(B, KH, keep)
    for_rows = src[..., None].expand(-1, -1, -1, D)
    to_rows = dst[..., None].expand(-1, -1, -1, D)
    k.scatter_(2, to_rows, torch.gather(k, 2, for_rows))
    v.scatter_(2, to_rows, torch.gather(v, 2, for_rows))
    w.scatter_(2, dst, torch.gather(w, 2, src))
    kept = torch.where(whole & (j >= lens), torch.full_like(kept, -1), kept)
    return {"k": k, "v": v, "weights": w, "kept": kept.int()}


def run(state):
    s = state
    kind = s["kind"]
    if not own:
        return {"tree": _plain_tree, "masked": _plain_masked, "weights": _plain_weights, "evict": _plain_evict}[kind](s)
    sts = _framework()
    if kind == "tree":
        return sts.tree_attention(s["q"], s["k"], s["v"], s["parents"], s["lens"], s["starts"], s["scale"],
                                  counts=s["counts"])
    if kind == "masked":
        return sts.masked_attention(s["q"], s["k"], s["v"], s["lens"], s["starts"], s["scale"], counts=s["counts"],
                                    lo=s["lo"], hi=s["hi"], slopes=s["slopes"], softcap=s["case"]["softcap"])
    if kind == "weights":
        out = sts.decode_ring_weights(s["q"], s["k"], s["v"], s["weights"], s["lens"], s["starts"], s["scale"])
        return {"out": out, "weights": s["weights"]}
    kept = sts.evict_ring(s["k"], s["v"], s["weights"], s["lens"], s["starts"], s["case"]["keep"], s["case"]["recent"])
    return {"k": s["k"], "v": s["v"], "weights": s["weights"], "kept": kept}


# ---------------------------------------------------------------------------
# In 64 bits, stream by stream on the ordered window
# ---------------------------------------------------------------------------

def _exact_stream(case, s, b, out):
    H, KH, D, M, kind = case["heads"], case["kv_heads"], case["dim"], case["ring"], case["kind"]
    L, at = int(s["lens"][b]), int(s["starts"][b])
    slots = (at + torch.arange(L, device=DEV)) % M
    n = 1 if kind == "weights" else int(s["counts"][b])
    q = (s["q"][b][None] if kind == "weights" else s["q"][b, :n]).double()
    seen = np.ones((n, L), bool)
    where = np.arange(L)
    if kind == "tree":
        parents = s["parents"][b].cpu().numpy()
        seen[:, L - n:] = False
        for i in range(n):
            j = i
            while j >= 0:
                seen[i, L - n + j] = True
                j = int(parents[j])
    elif kind == "masked":
        lo, hi = s["lo"][b].cpu().numpy(), s["hi"][b].cpu().numpy()
        seen = (where >= lo[:n, None]) & (where < hi[:n, None])
    seen = torch.from_numpy(seen).to(DEV)
    given = torch.zeros((KH, L), dtype=torch.float64, device=DEV)
    for h in range(H):
        kh = h // (H // KH)
        x = (q[:, h] @ s["k"][b, kh, slots].double().T) * s["scale"]
        if kind == "masked" and case["softcap"] > 0:
            x = case["softcap"] * torch.tanh(x / case["softcap"])
        if kind == "masked" and s["slopes"] is not None:
            away = np.abs(np.arange(L - n, L)[:, None] - where)
            x = x - s["slopes"][h].double() * torch.from_numpy(away).to(DEV).double()
        e = torch.where(seen, x, torch.full_like(x, -math.inf))
        e = torch.where(seen, torch.exp(e - e.amax(1, keepdim=True)), torch.zeros_like(e))
        e = e / e.sum(1, keepdim=True).clamp_min(1e-300)
        out[b, :n, h] = e @ s["v"][b, kh, slots].double()
        given[kh] += e.sum(0)
    return slots, given


def _exact_evict(case, s):
    k, v, w = (s[x].double() for x in ("k", "v", "weights"))
    B, KH, M, D = k.shape
    kept = np.full((B, KH, case["keep"]), -1, np.int32)
    lens, starts, given = s["lens"].cpu().numpy(), s["starts"].cpu().numpy(), s["weights"].cpu().numpy()
    for b in range(B):
        L, K = int(lens[b]), case["keep"]
        if L <= K:
            kept[b, :, :L] = np.arange(L)
            continue
        to = (starts[b] + np.arange(L - K, L)) % M
        for h in range(KH):
            old = given[b, h, (starts[b] + np.arange(L - case["recent"])) % M]
            best = np.lexsort((np.arange(len(old)), -old))[:K - case["recent"]]
            rows = np.concatenate([np.sort(best), np.arange(L - case["recent"], L)])
            kept[b, h] = rows
            a, z = (torch.from_numpy(i).to(DEV) for i in ((starts[b] + rows) % M, to))
            for t in (k, v, w):
                t[b, h, z] = t[b, h, a]
    return {"k": k, "v": v, "weights": w, "kept": torch.from_numpy(kept)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "evict":
        return _exact_evict(case, s)
    shape = s["q"].shape
    out = torch.zeros((shape[0], 1) + tuple(shape[1:]) if case["kind"] == "weights" else shape, dtype=torch.float64, device=DEV)
    total = s["weights"].double() if case["kind"] == "weights" else None
    for b in range(case["batch"]):
        slots, given = _exact_stream(case, s, b, out)
        if total is not None:
            total[b][:, slots] += given
    return out if total is None else {"out": out[:, 0], "weights": total}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    H, KH, D, kind = case["heads"], case["kv_heads"], case["dim"], case["kind"]
    size = 2 if case["kv"] == "bf16" else 4
    lens = _lengths(case)
    if kind == "evict":
        cut = lens[lens > case["keep"]]
        moved = KH * len(cut) * (case["keep"] - case["recent"])
        return {"bytes": float(4 * KH * cut.sum() + moved * (4 * D * size + 8) + 4 * KH * case["keep"] * len(lens)),
                "flops": float(KH * cut.sum())}
    rows, pairs, queries = 0, 0, 0
    counts = np.ones_like(lens) if kind == "weights" else _counts(case, lens)
    for L, n in zip(lens.tolist(), counts.tolist()):
        queries += n
        if kind == "masked":
            lo, hi = _spans(case, L, n)
            rows += int(np.max(hi)) - int(np.min(lo))
            pairs += int(np.sum(hi - lo))
        else:
            rows += L
            pairs += n * L if kind == "weights" else n * (L - n) + n * min(n, case["depth"])
    full = {"tree": case.get("nodes"), "masked": case.get("seq"), "weights": 1}[kind] * case["batch"]
    data = 2 * KH * D * size * rows + 4 * H * D * (queries + full) + (8 * KH * rows if kind == "weights" else 0)
    return {"bytes": float(data), "flops": float(4 * H * D * pairs)}
