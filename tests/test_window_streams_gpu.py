"""Drafts, masks, kept weights and eviction on streams other than the current one."""
import numpy as np
import pytest
import torch

import sts_attn
from test_window_gpu import calls, i32
from windows import Window, queries, random_tree

pytestmark = pytest.mark.gpu

SLEEP = 20_000_000  # clocks: some milliseconds at least, a fraction of a second at most


@pytest.mark.parametrize("as_handle", [False, True])
@pytest.mark.parametrize("what", ["tree", "masked", "weights", "scratch", "evict", "step"])
def test_new_memory_is_not_the_current_streams(gpu, what, as_handle):
    """A block that the current stream has freed, but is still working on, is not
    taken for the results or the scratch of a call on another stream."""
    B, H, M, D, T = 2, 4, 1000, 64, 8
    w = Window(41, B, H, M, D, [M, 700])
    w.k, w.v = w.k.nan_to_num(0.0), w.v.nan_to_num(0.0)
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    q = torch.from_numpy(queries(w.rng, B, T, H, D)).cuda()
    parents = i32(np.stack([random_tree(w.rng, T, T) for _ in range(B)]))
    acc = torch.rand((B, H, M), device="cuda")
    side = torch.cuda.Stream()
    s = side.cuda_stream if as_handle else side
    cache = sts_attn.KVCache(M, H, D)
    q1, o1 = q[:, 0].contiguous(), torch.zeros((B, H, D), device="cuda")
    scratch = sts_attn.load().sts_decode_ring_weights_scratch(B, H, M)
    run, words = {
        "tree": (lambda: sts_attn.tree_attention(q, k, v, parents, dl, ds, 0.125, stream=s), q.numel()),
        "masked": (lambda: sts_attn.masked_attention(q, k, v, dl, ds, 0.125, stream=s), q.numel()),
        "weights": (lambda: sts_attn.decode_ring_weights(q1, k, v, acc, dl, ds, 0.125, stream=s), q1.numel()),
        "scratch": (lambda: sts_attn.decode_ring_weights(q1, k, v, acc, dl, ds, 0.125, out=o1, stream=s), scratch),
        "evict": (lambda: sts_attn.evict_ring(k, v, acc, dl, ds, 300, 20, stream=s), B * H * 300),
        "step": (lambda: cache.tree_step(q[0], q[0], q[0], parents[0], 0.125, stream=s), q[0].numel()),
    }[what]
    run()  # the workspaces
    torch.cuda.synchronize()
    block = torch.full((words,), 7.0, device="cuda")
    torch.cuda._sleep(SLEEP)
    copy = block.clone()
    del block
    run()
    torch.cuda.synchronize()
    assert (copy == 7.0).all()


def test_new_memory_for_the_null_stream(gpu):
    """The same with another stream current and the null stream's handle given."""
    w = Window(46, 1, 4, 900, 64, [900])
    w.k, w.v = w.k.nan_to_num(0.0), w.v.nan_to_num(0.0)
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    q = torch.from_numpy(queries(w.rng, 1, 4, 64)).cuda()
    out = torch.zeros_like(q)
    acc = [torch.zeros((1, 4, 900), device="cuda") for _ in range(2)]
    words = sts_attn.load().sts_decode_ring_weights_scratch(1, 4, 900)
    sts_attn.decode_ring_weights(q, k, v, acc[0], dl, ds, 0.125, out=out)  # allocates, and frees, on the null stream
    torch.cuda.synchronize()
    block = torch.full((words,), 7.0, device="cuda")
    where = block.data_ptr()
    torch.cuda.synchronize()
    del block  # free for work on the null stream, and for it alone
    seen = []
    real = sts_attn._empty
    with pytest.MonkeyPatch.context() as m, torch.cuda.stream(torch.cuda.Stream()):
        m.setattr(sts_attn, "_empty", lambda *a: seen.append(real(*a)) or seen[-1])
        sts_attn.decode_ring_weights(q, k, v, acc[1], dl, ds, 0.125, out=out, stream=0)
        assert [t.data_ptr() for t in seen] == [where]
    torch.cuda.synchronize()
    assert torch.equal(acc[0], acc[1])


def test_results_of_another_stream_outlive_it(gpu):
    """A result that the current stream still reads is not overwritten by the next
    call on the stream that made it."""
    w = Window(42, 2, 4, 500, 64, [500, 400])
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    q = torch.from_numpy(queries(w.rng, 2, 8, 4, 64)).cuda()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    want, other = sts_attn.masked_attention(q, k, v, dl, ds, 0.125), q * 2
    torch.cuda.synchronize()
    got = sts_attn.masked_attention(q, k, v, dl, ds, 0.125, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda._sleep(SLEEP)
    copy = got.clone()
    del got
    for _ in range(3):
        sts_attn.masked_attention(other, k, v, dl, ds, 0.125, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(copy, want)


def test_results_made_at_the_same_time(gpu):
    """All four calls on two streams at once, what each wrote while the other ran kept
    on its own stream and compared with what it writes alone."""
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    work = [calls(43 + i, s) for i, s in enumerate(sides)]
    torch.cuda.synchronize()

    def once(i):
        fns, restore = work[i]
        with torch.cuda.stream(sides[i]):
            restore()
            return [t.clone() for f in fns for t in f()]

    alone = []
    for i in range(2):
        alone.append(once(i))
        torch.cuda.synchronize()
    rounds = [[once(i) for i in range(2)] for _ in range(12)]
    torch.cuda.synchronize()
    for got in rounds:
        for i in range(2):
            assert len(got[i]) == len(alone[i]) == 8
            assert all(torch.equal(a, b) for a, b in zip(got[i], alone[i]))
    assert not torch.equal(alone[0][0], alone[1][0])


def test_a_cap_that_is_zero_in_float32(gpu):
    """Not taken for no cap."""
    w = Window(45, 1, 1, 20, 64, [20])
    k, v, dl, ds = w.dev("k", "v", "lens", "starts")
    q = torch.zeros((1, 3, 1, 64), device="cuda")
    with pytest.raises(ValueError, match="softcap"):
        sts_attn.masked_attention(q, k, v, dl, ds, 0.125, softcap=1e-50)
    with pytest.raises(sts_attn.StsError, match="softcap"):
        sts_attn.masked_attention(q, k, v, dl, ds, 0.125, softcap=-1e-50 * 1e20)


@pytest.mark.parametrize("keep_weights", [False, True])
def test_a_refused_allocation_is_reported_once(gpu, keep_weights):
    """A cache too large for any memory is refused (no memory is taken); the calls
    after it are not refused for it."""
    big = sts_attn.KVCache(2 ** 31 - 1, 65535, 128, keep_weights=keep_weights)
    x = torch.ones((1, 3, 2, 64), device="cuda")
    c = sts_attn.KVCache(16, 2, 64, keep_weights=keep_weights)
    for _ in range(2):
        with pytest.raises(sts_attn.StsError, match="allocation"):
            sts_attn._check(sts_attn.load().sts_kv_ensure_allocated(big.handle, 1, None, None, None, None))
        c.update(x, x)
        assert c.attend(x[:, 0].contiguous(), 0.125).eq(1).all()
    assert big.state().allocated == 0 and c.seq_len() == 6
