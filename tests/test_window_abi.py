"""Refusals of the calls over drafts, masks and kept weights (no GPU needed).

Argument errors come before any device work: fake pointers, never dereferenced.
"""
import ctypes
import re

import pytest
import torch

import sts_attn
from test_abi import FAKE, HEADER, _err


def tree(q=FAKE, k=FAKE, v=FAKE, out=FAKE, parents=FAKE, counts=None, lens=FAKE, starts=FAKE, batch=2, nodes=8,
         heads=8, kv_heads=4, dim=128, max_len=100, scale=0.1, rows=0):
    return sts_attn.load().sts_tree_attention(q, k, v, out, parents, counts, lens, starts, batch, nodes, heads,
                                              kv_heads, dim, max_len, scale, rows, None)


def masked(q=FAKE, k=FAKE, v=FAKE, out=FAKE, lens=FAKE, starts=FAKE, batch=2, seq=8, heads=8, kv_heads=4, dim=128,
           max_len=100, scale=0.1, cap=0.0, rows=0):
    return sts_attn.load().sts_masked_attention(q, k, v, out, None, None, None, None, lens, starts, batch, seq,
                                                heads, kv_heads, dim, max_len, scale, cap, rows, None)


def weights(q=FAKE, k=FAKE, v=FAKE, out=FAKE, w=FAKE, scratch=FAKE, lens=FAKE, starts=FAKE, batch=2, heads=8,
            kv_heads=4, dim=128, max_len=100, scale=0.1, rows=0):
    return sts_attn.load().sts_decode_ring_weights(q, k, v, out, w, scratch, lens, starts, batch, heads, kv_heads,
                                                   dim, max_len, scale, rows, None)


def evict(k=FAKE, v=FAKE, w=FAKE, kept=FAKE, lens=FAKE, starts=FAKE, batch=2, kv_heads=4, dim=128, max_len=100,
          keep=10, recent=4, rows=0):
    return sts_attn.load().sts_evict_ring(k, v, w, kept, lens, starts, batch, kv_heads, dim, max_len, keep, recent,
                                          rows, None)


def commit(k=FAKE, v=FAKE, path=FAKE, accepted=FAKE, counts=None, lens=FAKE, starts=FAKE, batch=2, nodes=8,
           kv_heads=4, dim=128, max_len=100, rows=0):
    return sts_attn.load().sts_tree_commit(k, v, path, accepted, counts, lens, starts, batch, nodes, kv_heads, dim,
                                           max_len, rows, None)


@pytest.mark.parametrize("call", [tree, masked, weights])
def test_attention_refusals(call):
    for name in ("q", "k", "v", "out", "lens", "starts"):
        assert "null" in _err(call(**{name: None}))
    for name in ("q", "k", "v", "out"):
        assert "aligned" in _err(call(**{name: FAKE + 8}))
    for dim in (0, 2, 102, 132, 256):
        assert "head_dim" in _err(call(dim=dim))
    assert "multiple of 8" in _err(call(dim=100, rows=1))
    assert "query heads" in _err(call(heads=6))
    assert "empty" in _err(call(heads=0, kv_heads=4))
    assert "empty" in _err(call(kv_heads=0))
    assert "empty" in _err(call(batch=0))
    assert "empty" in _err(call(max_len=0))
    assert "65535" in _err(call(batch=65536))
    assert "65535" in _err(call(heads=70000, kv_heads=70000))
    assert "row type" in _err(call(rows=2))
    assert "scale" in _err(call(scale=float("nan")))
    assert "scale" in _err(call(scale=float("inf")))
    # A head's rows stay below 2 GiB: 4194304 rows of 128 floats are that much.
    assert "max_len" in _err(call(max_len=4194304))


def test_tree_refusals():
    assert "null" in _err(tree(parents=None))
    assert "nodes" in _err(tree(nodes=0))
    assert "nodes" in _err(tree(nodes=257))


def test_masked_refusals():
    assert "softcap" in _err(masked(cap=-1.0))
    assert "softcap" in _err(masked(cap=float("nan")))
    assert "softcap" in _err(masked(cap=float("inf")))
    assert "softcap" in _err(masked(cap=1e-44, scale=1.0))  # scale / softcap is not finite
    assert "softcap" in _err(masked(cap=2e30, scale=1.0))  # scale / softcap below 2^-100
    assert "softcap" in _err(masked(cap=-1.0, scale=0.0))
    assert "empty" in _err(masked(seq=0))
    assert "too many" in _err(masked(seq=1 << 28, heads=8, kv_heads=8))


def test_weights_refusals():
    assert "null" in _err(weights(w=None))
    assert "null" in _err(weights(scratch=None))
    assert "aligned" in _err(weights(scratch=FAKE + 4))
    # Whole tiles of 16 scores and two statistics for each head of each stream.
    assert sts_attn.load().sts_decode_ring_weights_scratch(3, 5, 33) == 3 * 5 * (48 + 2)
    assert sts_attn.load().sts_decode_ring_weights_scratch(65535, 65535, 2 ** 31) == 65535 ** 2 * (2 ** 31 + 2)


def test_evict_refusals():
    for name in ("k", "v", "w", "kept", "lens", "starts"):
        assert "null" in _err(evict(**{name: None}))
    assert "aligned" in _err(evict(k=FAKE + 8))
    assert "keep" in _err(evict(keep=0))
    assert "keep" in _err(evict(keep=101))
    assert "recent" in _err(evict(recent=11))
    assert "row type" in _err(evict(rows=-1))
    assert "head_dim" in _err(evict(dim=130))


def test_commit_refusals():
    for name in ("k", "v", "path", "accepted", "lens", "starts"):
        assert "null" in _err(commit(**{name: None}))
    assert "nodes" in _err(commit(nodes=0))
    assert "nodes" in _err(commit(nodes=300))
    assert "head_dim" in _err(commit(dim=6))
    assert "batch" in _err(commit(batch=30000))


def test_handle_refusals_leave_the_cache():
    lib = sts_attn.load()
    c = sts_attn.KVCache(64, 4, 128)
    step = lib.sts_kv_tree_step
    for word, args in [("null", (None, FAKE, FAKE, None, FAKE, FAKE, 5, 0.1)),
                       ("null", (None, FAKE, FAKE, FAKE, None, FAKE, 5, 0.1)),
                       ("nodes", (None, FAKE, FAKE, FAKE, FAKE, FAKE, 0, 0.1)),
                       ("nodes", (None, FAKE, FAKE, FAKE, FAKE, FAKE, 65, 0.1)),
                       ("aligned", (None, FAKE, FAKE + 4, FAKE, FAKE, FAKE, 5, 0.1)),
                       ("scale", (None, FAKE, FAKE, FAKE, FAKE, FAKE, 5, float("inf")))]:
        assert word in _err(step(c.handle, *args, None))
    assert "null" in _err(step(None, None, FAKE, FAKE, FAKE, FAKE, FAKE, 5, 0.1, None))
    s = c.state()
    assert (s.offset, s.len, s.write_pos, s.allocated) == (0, 0, 0, 0)
    c.advance(20)
    with pytest.raises(sts_attn.StsError, match="nodes"):
        c.tree_commit(21, [0])
    with pytest.raises(sts_attn.StsError, match="ascending"):
        c.tree_commit(5, [1, 1])
    with pytest.raises(sts_attn.StsError, match="ascending"):
        c.tree_commit(5, [5])
    with pytest.raises(sts_attn.StsError, match="accepted"):
        c.tree_commit(2, [0, 1, 2])
    with pytest.raises(sts_attn.StsError, match="weights"):
        c.evict(10, 2)
    assert (c.offset(), c.seq_len()) == (20, 20)


def test_commit_counters():
    """Accepted rows stay, the others are rolled back; no buffers, nothing moves."""
    c = sts_attn.KVCache(64, 4, 128)
    c.advance(30)
    c.tree_commit(8, [0, 3, 4])
    assert (c.offset(), c.seq_len(), c.write_pos()) == (25, 25, 25)
    c.tree_commit(4, [])
    assert (c.offset(), c.seq_len(), c.write_pos()) == (21, 21, 21)


def test_weight_cache_flags():
    lib = sts_attn.load()
    h = ctypes.c_void_p()
    assert "flags" in _err(lib.sts_kv_create_ex(10, 2, 64, 4, ctypes.byref(h)))
    c = sts_attn.KVCache(16, 2, 64, keep_weights=True, bf16_mirror=True)
    assert c.state().flags == sts_attn.KV_WEIGHTS | sts_attn.KV_BF16_MIRROR
    assert c.read_weights() is None
    with pytest.raises(sts_attn.StsError, match="no buffers"):
        c.evict(4, 2)
    with pytest.raises(sts_attn.StsError, match="recent"):
        c.evict(4, 5)
    with pytest.raises(sts_attn.StsError, match="keep"):
        c.evict(17, 5)


def test_constants_match_header():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    found = dict(re.findall(r"\b(STS_(?:ROWS_\w+|TREE_MAX_NODES|KV_WEIGHTS|KV_BF16_MIRROR))\s*=?\s*(\d+)", text))
    assert {k: int(v) for k, v in found.items()} == {
        "STS_ROWS_F32": sts_attn.ROWS_F32, "STS_ROWS_BF16": sts_attn.ROWS_BF16,
        "STS_TREE_MAX_NODES": sts_attn.TREE_MAX_NODES, "STS_KV_WEIGHTS": sts_attn.KV_WEIGHTS,
        "STS_KV_BF16_MIRROR": sts_attn.KV_BF16_MIRROR}


def test_tensors_of_the_wrong_place_type_or_shape():
    """The binding refuses what would be read out of bounds: here tensors on the CPU."""
    k = torch.zeros((2, 4, 16, 64))
    q = torch.zeros((2, 3, 8, 64))
    i = torch.zeros(2, dtype=torch.int32)
    p = torch.zeros((2, 3), dtype=torch.int32)
    with pytest.raises((ValueError, RuntimeError)):
        sts_attn.tree_attention(q, k, k, p, i, i, 0.1)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        sts_attn.tree_attention(q, k.double(), k.double(), p, i, i, 0.1)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        sts_attn.masked_attention(q, k, k.bfloat16(), i, i, 0.1)
    with pytest.raises(ValueError, match="KVH, M, D"):
        sts_attn.decode_ring_weights(q[:, 0], k, k[:, :2], k[..., 0], i, i, 0.1)
    with pytest.raises(ValueError, match="shape"):
        sts_attn._arg(q, "q", torch.float32, (2, 3, 8, 32), q.device)
    with pytest.raises(TypeError, match="parents"):
        sts_attn._arg(p.long(), "parents", torch.int32, (2, 3), q.device)
    with pytest.raises(ValueError, match="contiguous"):
        sts_attn._arg(q.transpose(0, 1), "q", torch.float32, (3, 2, 8, 64), q.device)
    with pytest.raises(ValueError, match="must be on"):
        sts_attn._arg(q, "q", torch.float32, q.shape, torch.device("meta"))


def test_values_that_c_types_would_change():
    """A path entry past 32 bits is refused, not taken modulo 2^32."""
    c = sts_attn.KVCache(64, 4, 128)
    c.advance(20)
    for path in ([2 ** 32], [0, 2 ** 32 + 1], [-1], [-(2 ** 32)]):
        with pytest.raises(sts_attn.StsError, match="ascending"):
            c.tree_commit(3, path)
    assert (c.offset(), c.seq_len()) == (20, 20)


@pytest.mark.parametrize("index", [None, 1])
def test_kept_rows_on_another_device(monkeypatch, index):
    """Only a tensor on the current GPU may receive the kept rows."""
    c = sts_attn.KVCache(16, 2, 64, keep_weights=True)

    class Kept:
        dtype, shape = torch.int32, (0, 2, 4)
        device = torch.device("cpu") if index is None else torch.device("cuda", index)

        def is_contiguous(self):
            return True

        def data_ptr(self):
            raise AssertionError("its address is not taken")

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="current GPU"):
        c.evict(4, 2, kept=Kept())
