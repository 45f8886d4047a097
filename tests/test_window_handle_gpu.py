"""Drafts, kept weights and eviction on the K/V handle, as a serving loop runs them."""
import numpy as np
import pytest
import torch

import oracle
import sts_attn
from conftest import scale_for
from windows import ancestors, attend64, depths, evict64, queries, random_tree

pytestmark = pytest.mark.gpu


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Model:
    """The handle's window in 64-bit form: ordered rows per K/V head, their weights."""

    def __init__(self, KH, D, M, tabs):
        self.k, self.v = np.zeros((KH, 0, D), np.float32), np.zeros((KH, 0, D), np.float32)
        self.w = np.zeros((KH, 0))
        self.M, self.tabs, self.offset = M, tabs, 0

    def rope(self, x, pos):
        """x [n, heads, D] rotated at pos[n], as the library rotates (f32)."""
        return np.concatenate([oracle.rope_apply(np.ascontiguousarray(x[i][None, None]), int(p), self.tabs)[0]
                               for i, p in enumerate(pos)])

    def append(self, k, v, pos=None):
        n = len(k)
        k = self.rope(k, self.offset + np.arange(n) if pos is None else pos)
        self.k = np.concatenate([self.k, k.transpose(1, 0, 2)], 1)[:, -self.M:]
        self.v = np.concatenate([self.v, v.transpose(1, 0, 2)], 1)[:, -self.M:]
        self.w = np.concatenate([self.w, np.zeros((len(self.w), n))], 1)[:, -self.M:]
        self.offset += n

    def attend(self, q, seen, scale, count=False):
        out, p, bound = attend64(q, self.k.astype(np.float64), self.v.astype(np.float64), seen, scale)
        if count:
            self.w = self.w + p[0].reshape(len(self.k), -1, p.shape[-1]).sum(1)
        return out, bound


@pytest.mark.parametrize("mirror", [False, True])
@pytest.mark.parametrize("H,KH,D,M", [(8, 8, 128, 96), (8, 2, 64, 300), (6, 3, 40, 64)])
def test_serving_loop(gpu, H, KH, D, M, mirror):
    """Prefill, then rounds of: a draft, its path kept, decodes that keep the weights,
    an eviction; past the ring's end.  Outputs, rows and weights against 64 bits."""
    rng = np.random.default_rng(H * D)
    scale = scale_for(D)
    cache = sts_attn.KVCache(M, KH, D, bf16_mirror=mirror, n_heads=H, keep_weights=True)
    rope = sts_attn.RoPE(D, 600)
    m = Model(KH, D, M, oracle.rope_tables(D, 600, 10000.0))

    def rows(n):
        return (queries(rng, n, H, D), rng.standard_normal((n, KH, D)).astype(np.float32),
                rng.standard_normal((n, KH, D)).astype(np.float32))

    def check(got, want, bound, what):
        err = np.abs(got.cpu().numpy() - want)
        assert (err <= bound[..., None]).all(), f"{what}: {err.max():.3e} over {bound.max():.3e}"

    q, k, v = rows(37)
    got = cache.prefill(dev(q), dev(k), dev(v), scale, rope=rope)
    qr = m.rope(q, np.arange(37))
    m.append(k, v)
    check(got, *m.attend(qr, np.tri(37, 37, dtype=bool), scale), "prefill")

    for turn in range(9):
        T = int(rng.integers(1, 24))
        parents = random_tree(rng, T, T)
        q, k, v = rows(T)
        pos = m.offset + depths(parents, T)
        got = cache.tree_step(dev(q), dev(k), dev(v), dev(parents), scale, rope=rope)
        before = (m.k, m.v, m.w, m.offset)
        m.append(k, v, pos)
        L = m.k.shape[1]
        seen = np.ones((T, L), bool)
        seen[:, L - T:] = ancestors(parents, T)
        check(got, *m.attend(m.rope(q, pos), seen, scale), f"draft {turn}")
        leaf = int(rng.integers(-1, T))
        path = np.flatnonzero(ancestors(parents, T)[leaf]) if leaf >= 0 else np.zeros(0, int)
        cache.tree_commit(T, [int(x) for x in path])
        at = np.concatenate([np.arange(L - T), L - T + path]).astype(int)
        m.k, m.v, m.w = m.k[:, at], m.v[:, at], m.w[:, at]
        m.offset = before[3] + len(path)
        assert (cache.offset(), cache.seq_len()) == (m.offset, m.k.shape[1])

        for _ in range(3):
            q, k, v = rows(1)
            got = cache.decode_step(dev(q), dev(k), dev(v), scale, rope=rope)
            qr = m.rope(q, [m.offset])
            m.append(k, v)
            check(got, *m.attend(qr, np.ones((1, m.k.shape[1]), bool), scale, count=True), f"decode {turn}")
        if turn % 3 == 2:
            L = m.k.shape[1]
            keep, recent = L // 2 + 1, 5
            # The library's own weights decide: they differ from 64 bits in the last place.
            start, ln = cache.window()
            w = cache.read_weights()[0].cpu().numpy()[:, (start + np.arange(ln)) % M]
            np.testing.assert_allclose(w, m.w, rtol=2e-4, atol=1e-6)
            kept = torch.zeros((1, KH, keep), dtype=torch.int32, device="cuda")
            cache.evict(keep, recent, kept=kept if turn == 2 else None)
            chosen = [evict64(w[h], keep, recent) for h in range(KH)]
            if turn == 2:
                np.testing.assert_array_equal(kept[0].cpu().numpy(), chosen)
            m.k = np.stack([m.k[h, c] for h, c in enumerate(chosen)])
            m.v = np.stack([m.v[h, c] for h, c in enumerate(chosen)])
            m.w = np.stack([m.w[h, c] for h, c in enumerate(chosen)])
        start, ln = cache.window()
        slots = (start + np.arange(ln)) % M
        kb, vb = cache.read_buffers()
        np.testing.assert_array_equal(kb[0].cpu().numpy()[:, slots], m.k)
        np.testing.assert_array_equal(vb[0].cpu().numpy()[:, slots], m.v)
        if mirror:
            k16, _ = cache.mirror_buffers()
            assert torch.equal(k16[0][:, dev(slots)].view(torch.bfloat16), dev(m.k).bfloat16())
    assert m.offset > 37


def test_draft_equals_the_steps_it_stands_for(gpu):
    """A chain draft, all of it accepted, leaves what as many decode steps leave."""
    H, D, M, T = 4, 64, 50, 7
    rng = np.random.default_rng(2)
    a, b = sts_attn.KVCache(M, H, D), sts_attn.KVCache(M, H, D)
    rope = sts_attn.RoPE(D, 100)
    first = [dev(rng.standard_normal((1, 45, H, D)).astype(np.float32)) for _ in range(2)]
    a.update(*first)
    b.update(*first)
    q, k, v = (dev(rng.standard_normal((T, H, D)).astype(np.float32)) for _ in range(3))
    a.tree_step(q, k, v, torch.arange(-1, T - 1, dtype=torch.int32, device="cuda"), 0.125, rope=rope)
    a.tree_commit(T, range(T))
    for i in range(T):
        b.decode_step(q[i:i + 1], k[i:i + 1], v[i:i + 1], 0.125, rope=rope)
    assert (a.offset(), a.window()) == (b.offset(), b.window())
    for x, y in zip(a.read_buffers(), b.read_buffers()):
        assert torch.equal(x, y)


def test_weights_cache_batch_and_attend(gpu):
    """A batch of streams: attend counts, decode_step counts and clears the slot that
    it takes, update and prefill clear theirs, rollback lets the next row start anew."""
    B, H, D, M = 3, 2, 64, 10
    g = torch.Generator(device="cuda").manual_seed(5)

    def r(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    c = sts_attn.KVCache(M, H, D, keep_weights=True)
    plain = sts_attn.KVCache(M, H, D)
    k, v = r(B, 8, H, D), r(B, 8, H, D)
    c.update(k, v)
    plain.update(k, v)
    assert not c.read_weights().any()
    q = r(B, H, D)
    x, y = c.attend(q, 0.125), plain.attend(q, 0.125)
    assert (x - y).abs().max() < 1e-5  # two f32 evaluations of 8 rows
    w = c.read_weights()
    assert (w.sum(-1) - 1).abs().max() < 1e-5 and not w[..., 8:].any()
    for _ in range(5):  # past the ring's end
        q, k, v = r(B, H, D), r(B, H, D), r(B, H, D)
        slot, old = c.write_pos(), c.read_weights()
        x, y = c.decode_step(q, k, v, 0.125), plain.decode_step(q, k, v, 0.125)
        assert (x - y).abs().max() < 1e-5
        added = c.read_weights() - old
        added[..., slot] += old[..., slot]  # it started at zero
        assert (added.sum(-1) - 1).abs().max() < 1e-5 and (added > -1e-6).all()
    pos = c.write_pos()
    c.rollback(2)
    c.update(r(B, 2, H, D), r(B, 2, H, D))
    assert c.write_pos() == pos
    w = c.read_weights()
    assert not w[..., [(pos - 1) % M, (pos - 2) % M]].any() and (w > 0).sum() == B * H * (M - 2)
    c.reset_keep_buffers()
    assert not c.read_weights().any()
    c.reset()
    assert c.read_weights() is None
    one = sts_attn.KVCache(M, H, D, keep_weights=True)
    one.prefill(r(4, H, D), r(4, H, D), r(4, H, D), 0.125)
    assert not one.read_weights().any()
    with pytest.raises(sts_attn.StsError, match="query heads"):
        sts_attn._check(sts_attn.load().sts_kv_set_query_heads(one.handle, 4))


def test_evict_then_decode_from_a_graph(gpu):
    """A captured decode of a cache that keeps weights replays as eager ones."""
    H, D, M = 4, 128, 2000
    g = torch.Generator(device="cuda").manual_seed(6)
    c = sts_attn.KVCache(M, H, D, keep_weights=True)
    c.update(torch.randn((1, M, H, D), generator=g, device="cuda"), torch.randn((1, M, H, D), generator=g, device="cuda"))
    q = torch.randn((1, H, D), generator=g, device="cuda")
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        c.attend(q, 0.09, out=out)
    torch.cuda.synchronize()
    want, w1 = out.clone(), c.read_weights()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.attend(q, 0.09, out=out)
    for rep in range(2, 5):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        w = c.read_weights()
        # rep times the same weight, added one after another.
        assert (w - rep * w1).abs().max() <= rep * 2.0 ** -24 * (rep * w1).max()
    c.evict(700, 10)
    assert c.seq_len() == 700
    c.attend(q, 0.09)
    torch.cuda.synchronize()


def test_batch_caches_refuse_drafts(gpu):
    c = sts_attn.KVCache(20, 2, 64)
    x = torch.zeros((2, 4, 2, 64), device="cuda")
    c.update(x, x)
    q = torch.zeros((3, 2, 64), device="cuda")
    p = torch.full((3,), -1, dtype=torch.int32, device="cuda")
    with pytest.raises(sts_attn.StsError, match="batch-1"):
        c.tree_step(q, q, q, p, 0.1)
    with pytest.raises(sts_attn.StsError, match="batch-1"):
        c.tree_commit(2, [0])
    one = sts_attn.KVCache(20, 2, 64)
    with pytest.raises(ValueError, match="k_new"):
        one.tree_step(q, q[:2], q, p, 0.1)
    rope = sts_attn.RoPE(64, 2)
    with pytest.raises(sts_attn.StsError, match="RoPE"):
        one.tree_step(q, q, q, p, 0.1, rope=rope)
    assert one.state().allocated == 0 and one.offset() == 0
