"""The verdict on a draft on the GPU, against exact fractions."""
from fractions import Fraction

import numpy as np
import pytest
import torch

import sts_attn
from conftest import scale_for
from pages import verdict
from windows import Window, attend64_channels, queries, tree_seen

pytestmark = pytest.mark.gpu


def soft(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def tree(rng, T):
    parents = np.full(T, -1, np.int32)
    for i in range(1, T):
        parents[i] = i - 1 if rng.random() < 0.3 else rng.integers(0, i)
    return parents


def check(target, draft, tokens, parents, rand, counts=None):
    B, T, V = target.shape
    dev = [None if x is None else torch.from_numpy(np.array(x, order="C")).cuda()
           for x in (target, tokens.astype(np.int32), parents.astype(np.int32), rand.astype(np.float32), draft,
                     None if counts is None else np.asarray(counts, np.int32))]
    path, accepted, following = (x.cpu().numpy() for x in sts_attn.verify_draft(*dev[:4], draft=dev[4], counts=dev[5]))
    taken = 0
    for b in range(B):
        n = T if counts is None else min(max(int(counts[b]), 0), T)
        want, word = verdict(target[b], None if draft is None else draft[b], tokens[b], parents[b], n, rand[b])
        assert list(path[b][:len(want)]) == want and (path[b][len(want):] == -1).all(), (b, path[b], want)
        assert accepted[b] == len(want) and following[b] == word, (b, following[b], word)
        taken += max(len(want) - 1, 0)
    return taken


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V", [1, 2, 3, 5, 255, 257, 1000, 4097])
def test_trees(gpu, V, drawn):
    """Random trees, some nodes kept and some not, some streams with fewer nodes."""
    rng = np.random.default_rng(V + drawn)
    B, T = 12, 14
    x = rng.standard_normal((B, T, V)) * 2
    target, draft = soft(x), soft(0.7 * x + 0.5 * rng.standard_normal((B, T, V)))
    parents = np.stack([tree(rng, T) for _ in range(B)])
    tokens = np.zeros((B, T), np.int32)
    for b in range(B):
        for i in range(1, T):
            q = draft[b, parents[b, i]].astype(np.float64)
            tokens[b, i] = rng.choice(V, p=q / q.sum()) if drawn else np.argsort(-q)[min(i % 3, V - 1)]
    counts = rng.integers(0, T + 2, B)
    taken = check(target, draft if drawn else None, tokens, parents, rng.random((B, T), np.float32), counts)
    assert taken > 0 or V > 1000  # (of thousands of words none is likely)


@pytest.mark.parametrize("drawn", [False, True])
def test_large_vocabulary(gpu, drawn):
    rng = np.random.default_rng(30)
    B, T, V = 2, 5, 70001
    x = rng.standard_normal((B, T, V)) * 3
    target, draft = soft(x), soft(x + 0.8 * rng.standard_normal((B, T, V)))
    parents = np.array([[-1, 0, 0, 0, 1], [-1, 0, 1, 2, 3]])
    tokens = rng.integers(0, V, (B, T))
    tokens[1, 1] = target[1, 0].argmax()
    check(target, draft if drawn else None, tokens, parents, rng.random((B, T), np.float32))


def test_most_nodes(gpu):
    rng = np.random.default_rng(31)
    B, T, V = 2, 256, 40
    target = soft(rng.standard_normal((B, T, V)))
    parents = np.stack([tree(rng, T), np.r_[-1, np.zeros(T - 1, int)]])  # a tree, and 255 children of one node
    check(target, None, rng.integers(0, V, (B, T)), parents, rng.random((B, T), np.float32))
    check(target, soft(rng.standard_normal((B, T, V))), rng.integers(0, V, (B, T)), parents,
          rng.random((B, T), np.float32))


@pytest.mark.parametrize("drawn", [False, True])
def test_many_children(gpu, drawn):
    """Hundreds of children of one node, words among them more than once."""
    rng = np.random.default_rng(11)
    B, T, V = 6, 200, 300
    x = rng.standard_normal((B, T, V)) * 0.3
    target, draft = soft(x), soft(x + 0.1 * rng.standard_normal((B, T, V)))
    parents = np.zeros((B, T), np.int32)
    parents[:, 0] = -1
    parents[3:, 150:] = 70  # (below one that few streams keep)
    tokens = rng.integers(0, V // 2, (B, T))
    check(target, draft if drawn else None, tokens, parents, rng.random((B, T), np.float32))


def test_chosen_cases(gpu):
    """Dyadic probabilities, whose sums are exact: borders, siblings of one token, nothing left."""
    p = np.array([0.5, 0.25, 0.125, 0.125], np.float32)
    one = np.array([0, 1, 0, 0], np.float32)
    half = np.array([0.5, 0.5, 0, 0], np.float32)
    none = np.zeros(4, np.float32)

    def run(target, tokens, parents, rand, draft=None):
        T = len(tokens)
        check(np.broadcast_to(target, (1, T, 4)) if target.ndim == 1 else target[None], draft if draft is None else
              np.broadcast_to(draft, (1, T, 4)), np.array([tokens]), np.array([parents]), np.array([rand], np.float32))

    for u in (0.0, 0.25, 0.5, 0.75, 0.874, 0.875, 0.999):
        run(p, [0], [-1], [u])
        for w in (0.0, 0.249, 0.25, 0.5, 0.75):
            run(p, [0, 1], [-1, 0], [u, w])
            run(p, [0, 1], [-1, 0], [u, w], draft=half)
            run(p, [0, 1, 1, 2], [-1, 0, 0, 0], [u, w, w, w])           # two siblings of one token
            run(p, [0, 0, 1, 2, 3], [-1, 0, 0, 0, 0], [u, .9, .9, .9, .9])  # every word tried
            run(p, [0, 1, 0], [-1, 0, 0], [u, w, w], draft=p)            # r = 0 once it is cut: stays as it was
            run(one, [0, 1, 0], [-1, 0, 0], [u, w, w])
            run(one, [0, 0, 1], [-1, 0, 0], [u, w, w], draft=half)
            run(p, [0, 3, 3], [-1, 0, 1], [u, w, w], draft=one)          # a token its draft could not give
    run(none, [0, 1, 2], [-1, 0, 0], [0.3, 0.0, 0.0])
    run(none, [0], [-1], [0.0], draft=half)
    # Tokens and parents that are none.
    run(p, [0, -1, 4, 2 ** 31 - 1, 1], [-1, 0, 0, 0, 0], [0.6, 0.0, 0.0, 0.0, 0.1])
    run(p, [0, -7, 0], [-1, 0, 0], [0.6, 0.0, 0.3], draft=half)
    run(p, [0, 0, 0, 0], [0, 1, 3, -2], [0.6, 0.0, 0.0, 0.0])
    # Negative probabilities and NaN count as nothing.
    odd = np.array([np.nan, -0.5, 0.25, 0.75], np.float32)
    run(odd, [0, 0, 1, 2], [-1, 0, 0, 0], [0.9, 0.0, 0.0, 0.7])
    run(odd, [0, 2, 3], [-1, 0, 0], [0.9, 0.8, 0.9], draft=np.array([np.nan, 0.25, 0.5, -1], np.float32))


def test_rows_that_do_not_sum_to_one(gpu):
    """Rows cut to a few words and not normalised, dyadic so that every sum is exact: where the first
    rejected child has all that is left of its row, it stays, and later rejections take its mass."""
    def run(target, tokens, rand):
        T = len(tokens)
        check(np.broadcast_to(np.float32(target), (1, T, 4)), None, np.array([tokens]),
              np.array([[-1] + [0] * (T - 1)]), np.array([rand], np.float32))

    half = [0, 0.5, 0, 0]
    run(half, [0, 1, 2, 1], [0.3, 0.9, 0.9, 0.9])        # kept at last: 0.9 * 0.5 < 0.5
    run(half, [0, 1, 2], [0.3, 0.9, 0.9])                # no child kept: the word is drawn
    run(half, [0, 1, -1, 1], [0.3, 0.9, 0.9, 0.9])       # the second child's token is none
    run(half, [0, 2, 1, 1], [0.3, 0.9, 0.9, 0.9])        # a word without mass goes first
    run(half, [0, -1, 1], [0.3, 0.9, 0.9])
    run(half, [0, 1, 1, 2, 3, 1], [0.3, 0.9, 0.9, 0.9, 0.9, 0.9])
    run([0.25, 0.25, 0, 0], [0, 0, 1], [0.3, 0.9, 0.9])  # the second word takes all that is left
    run([0.25, 0.25, 0, 0], [0, 0, 0, 2, 1], [0.3, 0.9, 0.9, 0.9, 0.9])
    run([0, 0, 0, 0], [0, 1, 2, 1], [0.3, 0.9, 0.9, 0.9])

    rng = np.random.default_rng(40)
    for V, T, B in ((2, 7, 300), (4, 9, 300), (6, 80, 100)):
        target = np.zeros((B, T, V), np.float32)
        for _ in range(2):
            at = rng.integers(0, V, (B, T, 1))
            np.put_along_axis(target, at, (rng.integers(0, 12, (B, T, 1)) / 16).astype(np.float32), 2)
        tokens = rng.integers(-1, V + 1, (B, T))
        parents = np.where(rng.random((B, T)) < 0.8, 0, np.stack([tree(rng, T) for _ in range(B)]))
        parents[:, 0] = -1
        rand = ((rng.integers(8, 16, (B, T)) * 2 + 1) / 32).astype(np.float32)
        check(target, None, tokens, parents, rand)


def cut_to(p, share):
    """p's likeliest words, `share` of it together, as probabilities."""
    by = np.argsort(-p)
    few = by[:int(np.searchsorted(np.cumsum(p[by].astype(np.float64)), share)) + 1]
    y = np.zeros_like(p)
    y[few] = p[few]
    return (y / y.sum(dtype=np.float64)).astype(np.float32)


def left_after(p, q, k):
    """What k rejections leave of p, exactly: (whole numbers, one for each word, in proportion; the
    distance from a border within which a verdict is open)."""
    one = 2 ** 160
    p, q = ([int(Fraction(float(x)) * one) for x in a] for a in (p, q))
    r, unit, near = p, one, Fraction(1, 2 ** 45)  # r[x] / unit is what q[x] is taken off
    for j in range(k):
        r = [max(0, a * one - unit * b) for a, b in zip(r, q)]
        if j > 0:
            near *= 4 / Fraction(sum(r), unit * one)
        unit = sum(r)
    return r, near


def beside(border, near):
    """The float32 numbers next to a border on both sides that are `near` away at least."""
    lo = np.float32(float(border - near))
    while Fraction(float(lo)) > border - near:
        lo = np.nextafter(lo, np.float32(-1))
    hi = np.float32(float(border + near))
    while Fraction(float(hi)) < border + near:
        hi = np.nextafter(hi, np.float32(2))
    return lo, hi


@pytest.mark.parametrize("noise", [0.02, 0.3, 1.0])
@pytest.mark.parametrize("k", [1, 2, 3, 4])
def test_next_to_borders(gpu, k, noise):
    """After k rejections at one place, of words that the target's row leaves out, random numbers as
    near to a child's border and to those of the draw as the verdict is exact there."""
    rng = np.random.default_rng(41 + k)
    V, T = 150, k + 2
    trees = []  # (p, q, tokens, rand, nodes, whether the last child is kept)
    while len(trees) < 48:
        x = rng.standard_normal(V) * 2
        q, p = soft(x), cut_to(soft(x + noise * rng.standard_normal(V)), 0.999)
        r, near = left_after(p, q, k)
        total = sum(r)
        out = np.flatnonzero(p == 0)
        below, child, draw = 0, [], []  # (distance, word, number, whether it is below the border)
        for x in range(V):
            below += r[x]
            for sides, border in ((child, Fraction(r[x], total) / Fraction(float(q[x]))), (draw, Fraction(below, total))):
                if r[x] and near < border < 1 - near:
                    sides += [(abs(Fraction(float(u)) - border), x, u, u < border) for u in beside(border, near)]
        for _, x, u, kept in sorted(child)[:2]:
            trees.append((p, q, np.r_[0, rng.choice(out, k), x], np.r_[0.5, np.ones(k) * 0.5, u], T, kept))
        for _, x, u, _ in sorted(draw)[:2]:
            trees.append((p, q, np.r_[0, rng.choice(out, k), 0], np.r_[u, np.ones(k) * 0.5, 0.5], T - 1, False))
    p, q, tokens, rand, n, kept = (np.array(x) for x in zip(*trees))
    B = len(n)
    parents = np.tile(np.r_[-1, np.zeros(T - 1, int)], (B, 1))
    rows = [np.repeat(x[:, None], T, 1) for x in (p, q)]
    assert check(rows[0], rows[1], tokens, parents, rand, counts=n) == kept.sum() > 0


@pytest.mark.parametrize("V", [3, 700, 5000, 270001])
def test_the_end_of_the_vocabulary(gpu, V):
    """A share of all that is left (a number past the range, as rounding may give) takes the last
    word with anything left; no share the first."""
    p = np.zeros((2, 2, V), np.float32)
    first, last = V // 3, V - 1 - V // 4
    p[:, :, first:last + 1:2] = 2.0 ** -20
    last -= (last - first) % 2
    i = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    rand = torch.tensor([[1.0, 0.5], [0.0, 0.5]], device="cuda")
    path, accepted, following = sts_attn.verify_draft(torch.from_numpy(p).cuda(), i, i - 1, rand)
    assert path.tolist() == [[0, -1], [0, -1]] and accepted.tolist() == [1, 1]
    assert following.tolist() == [last, first]


def test_tokens_follow_the_target(gpu):
    """The first token after node 0, kept or drawn, comes as often as the target says: within five
    standard deviations of a binomial count."""
    rng = np.random.default_rng(33)
    B, V = 60000, 5
    p, q = soft(rng.standard_normal(V)), soft(rng.standard_normal(V))
    tokens = np.zeros((B, 3), np.int32)
    tokens[:, 1:] = rng.choice(V, (B, 2), p=q.astype(np.float64) / q.astype(np.float64).sum())
    target = np.broadcast_to(p, (B, 3, V)).copy()
    draft = np.broadcast_to(q, (B, 3, V)).copy()
    parents = np.tile(np.array([-1, 0, 0], np.int32), (B, 1))
    args = [torch.from_numpy(x).cuda() for x in (target, tokens, parents, rng.random((B, 3), np.float32), draft)]
    path, accepted, following = (x.cpu().numpy() for x in sts_attn.verify_draft(*args[:4], draft=args[4]))
    first = np.where(accepted > 1, tokens[np.arange(B), np.maximum(path[:, 1], 0)], following)
    assert (accepted > 1).mean() > 0.3
    for v in range(V):
        want = float(p[v])
        assert abs((first == v).mean() - want) < 5 * np.sqrt(want * (1 - want) / B), v


def test_siblings_drawn_without_replacement(gpu):
    """Children drawn one from what the other leaves, judged as chosen without chance: the first token
    comes as often as the target says (with their probabilities it would not: .4, .4, .2 for
    .5, .3, .2 under .2, .2, .6), within five standard deviations of a binomial count."""
    rng = np.random.default_rng(35)
    B, V = 60000, 3
    p, q = np.float32([0.5, 0.3, 0.2]), np.array([0.2, 0.2, 0.6])
    tokens = np.zeros((B, 3), np.int32)
    tokens[:, 1:] = np.argsort(-(np.log(q) + rng.gumbel(size=(B, V))), 1)[:, :2]
    target = np.broadcast_to(p, (B, 3, V)).copy()
    parents = np.tile(np.array([-1, 0, 0], np.int32), (B, 1))
    args = [torch.from_numpy(x).cuda() for x in (target, tokens, parents, rng.random((B, 3), np.float32))]
    path, accepted, following = (x.cpu().numpy() for x in sts_attn.verify_draft(*args))
    first = np.where(accepted > 1, tokens[np.arange(B), np.maximum(path[:, 1], 0)], following)
    for v in range(V):
        want = float(p[v])
        assert abs((first == v).mean() - want) < 5 * np.sqrt(want * (1 - want) / B), v


def test_refusals(gpu):
    p = torch.zeros((2, 3, 5), device="cuda")
    i = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    u = torch.zeros((2, 3), device="cuda")
    with pytest.raises(ValueError, match="target"):
        sts_attn.verify_draft(p[0], i, i, u)
    with pytest.raises(ValueError, match="tokens"):
        sts_attn.verify_draft(p, i[:, :2].contiguous(), i, u)
    with pytest.raises(TypeError, match="tokens"):
        sts_attn.verify_draft(p, i.long(), i, u)
    with pytest.raises(ValueError, match="draft"):
        sts_attn.verify_draft(p, i, i, u, draft=p[:, :2].contiguous())
    with pytest.raises(ValueError, match="contiguous"):
        sts_attn.verify_draft(p.transpose(0, 1).contiguous().transpose(0, 1), i, i, u)


def test_in_a_graph(gpu):
    rng = np.random.default_rng(34)
    B, T, V = 4, 6, 3001
    target = torch.from_numpy(soft(rng.standard_normal((B, T, V)))).cuda()
    parents = torch.from_numpy(np.stack([tree(rng, T) for _ in range(B)])).cuda()
    tokens = target.argmax(-1).int()
    rand = torch.rand((B, T), device="cuda")
    sts_attn.verify_draft(target, tokens, parents, rand)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sts_attn.verify_draft(target, tokens, parents, rand)
    for _ in range(4):
        rand.copy_(torch.rand_like(rand) ** 3)
        tokens.copy_(torch.randint(0, 9, tokens.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, sts_attn.verify_draft(target, tokens, parents, rand)):
            assert torch.equal(a, b)


def test_draft_attended_judged_committed(gpu):
    """A draft's round as a server runs it: its attention, the verdict, the commit, and the next
    token's attention over the rows that stayed, against 64 bits."""
    B, H, KH, M, D, T, V = 5, 4, 2, 90, 64, 8, 300
    scale = scale_for(D)
    lens = [60, 33, 89, 8, 20]
    w = Window(35, B, KH, M, D, lens)
    parents = np.stack([tree(w.rng, T) for _ in range(B)])
    counts = np.array([8, 5, 8, 8, 1], np.int32)
    k, v, lens_, starts = w.dev("k", "v", "lens", "starts")
    par, cnt = torch.from_numpy(parents).cuda(), torch.from_numpy(counts).cuda()
    q = queries(w.rng, B, T, H, D)
    hidden = sts_attn.tree_attention(torch.from_numpy(q).cuda(), k, v, par, lens_, starts, scale, counts=cnt)
    for b in range(B):
        n = counts[b]
        out, bound = attend64_channels(q[b, :n], w.rows(b, w.k), w.rows(b, w.v), tree_seen(parents[b], n, lens[b]), scale)
        assert (np.abs(hidden[b, :n].cpu().numpy() - out) <= bound).all()
    # Probabilities after each node, from its hidden state.
    head = torch.randn((H * D, V), generator=torch.Generator().manual_seed(1)).cuda()
    target = torch.softmax(hidden.reshape(B, T, H * D) @ head, -1)
    tokens = target.argmax(-1).int()
    at = par.clamp_min(0).long()
    tokens = torch.gather(tokens, 1, at).int()  # each child its parent's likeliest word
    rand = torch.rand((B, T), generator=torch.Generator().manual_seed(2)).cuda()
    path, accepted, following = sts_attn.verify_draft(target, tokens, par, rand, counts=cnt)
    for b in range(B):
        want, word = verdict(target[b].cpu().numpy(), None, tokens[b].cpu().numpy(), parents[b], counts[b],
                             rand[b].cpu().numpy())
        assert path[b, :len(want)].tolist() == want and int(accepted[b]) == len(want) and int(following[b]) == word
    assert int(accepted.max()) > 1
    sts_attn.tree_commit(k, v, path, accepted, lens_, starts, counts=cnt)
    left = lens_ - cnt + accepted
    q1 = queries(w.rng, B, H, D)
    got = sts_attn.masked_attention(torch.from_numpy(q1[:, None]).cuda(), k, v, left, starts, scale).cpu().numpy()
    for b in range(B):
        rows = np.r_[np.arange(lens[b] - counts[b]), lens[b] - counts[b] + path[b, :int(accepted[b])].cpu().numpy()]
        kk, vv = (w.rows(b, x)[:, rows] for x in (w.k, w.v))
        out, bound = attend64_channels(q1[b:b + 1], kk, vv, np.ones((1, len(rows)), bool), scale)
        assert (np.abs(got[b] - out) <= bound).all()
