"""Refusals of the calls over paged K/V rows and drafts' verdicts (no GPU needed).

Argument errors come before any device work: fake pointers, never dereferenced.
"""
import ctypes
import re

import pytest
import torch

import sts_attn
from test_abi import FAKE, HEADER, _err


def pool(k=FAKE, v=FAKE, ks=None, vs=None, pages=9, page_rows=16, kv_heads=4, dim=128, rows=0):
    return ctypes.byref(sts_attn.Pages(k, v, ks, vs, pages, page_rows, kv_heads, dim, rows))


def append(pages=pool, rope=None, k=FAKE, v=FAKE, stride=512, table=FAKE, counts=None, lens=FAKE, batch=2, seq=3,
           max_pages=5, max_rows=80, **kw):
    return sts_attn.load().sts_paged_append(pages(**kw) if pages else None, rope, k, v, stride, table, counts, lens,
                                            batch, seq, max_pages, max_rows, None)


def decode(pages=pool, rope=None, q=FAKE, q_stride=1024, k_new=None, v_new=None, stride=512, out=FAKE, table=FAKE,
           lens=FAKE, batch=2, heads=8, max_pages=5, max_rows=80, scale=0.1, **kw):
    return sts_attn.load().sts_paged_decode(pages(**kw) if pages else None, rope, q, q_stride, k_new, v_new, stride,
                                            out, table, lens, batch, heads, max_pages, max_rows, scale, None)


def gather(pages=pool, rope=None, k_out=FAKE, v_out=FAKE, table=FAKE, first=None, lens=FAKE, batch=2, max_pages=5,
           max_rows=80, max_len=80, out_type=0, **kw):
    return sts_attn.load().sts_paged_gather(pages(**kw) if pages else None, k_out, v_out, table, first, lens, batch,
                                            max_pages, max_rows, max_len, out_type, None)


def verify(target=FAKE, draft=None, tokens=FAKE, parents=FAKE, counts=None, rand=FAKE, path=FAKE, accepted=FAKE,
           following=FAKE, batch=2, nodes=8, vocab=100):
    return sts_attn.load().sts_verify_draft(target, draft, tokens, parents, counts, rand, path, accepted, following,
                                            batch, nodes, vocab, None)


@pytest.mark.parametrize("call", [append, decode, gather])
def test_refusals_of_every_paged_call(call):
    assert "null" in _err(call(pages=None))
    for name in ("k", "v"):
        if call is not append:  # (append's own k and v are the new rows)
            assert "null" in _err(call(**{name: None}))
            assert "aligned" in _err(call(**{name: FAKE + 8}))
    for name in ("table", "lens"):
        assert "null" in _err(call(**{name: None}))
    assert "row type" in _err(call(rows=3))
    assert "row type" in _err(call(rows=-1))
    assert "k_scale" in _err(call(rows=2))
    assert "k_scale" in _err(call(rows=2, ks=FAKE))
    assert "aligned" in _err(call(rows=2, ks=FAKE + 4, vs=FAKE))
    for dim in (0, 2, 66, 132, 256):
        assert "head_dim" in _err(call(dim=dim))
    assert "multiple of 8" in _err(call(dim=100, rows=1))
    assert "multiple of 16" in _err(call(dim=72, rows=2, ks=FAKE, vs=FAKE))
    for rows in (0, 8, 24, 48, 8192):
        assert "page_rows" in _err(call(page_rows=rows))
    for name in ("batch", "pages_", "kv_heads", "max_pages", "max_rows"):
        kw = {"pages": lambda **k: pool(pages=0, **k)} if name == "pages_" else {name: 0}
        assert "empty" in _err(call(**kw))
    assert "65535" in _err(call(batch=65536))
    assert "65535" in _err(call(kv_heads=65536))
    assert "max_rows" in _err(call(max_rows=81))
    assert "too many pages" in _err(call(max_pages=1 << 27))
    assert "too many pages" in _err(call(pages=lambda **k: pool(pages=1 << 31, **k)))


def test_append_refusals():
    for name in ("k", "v"):
        assert "null" in _err(append(**{name: None}))
        assert "aligned" in _err(append(**{name: FAKE + 4}))
    assert "new_stride" in _err(append(stride=508))
    assert "new_stride" in _err(append(stride=514))
    assert "seq" in _err(append(seq=0))
    assert "seq" in _err(append(seq=81))
    assert "too many" in _err(append(seq=1 << 20, batch=64, max_pages=1 << 17, max_rows=1 << 21))


def test_decode_refusals():
    for name in ("q", "out"):
        assert "null" in _err(decode(**{name: None}))
        assert "aligned" in _err(decode(**{name: FAKE + 8}))
    assert "both" in _err(decode(k_new=FAKE))
    assert "both" in _err(decode(v_new=FAKE))
    assert "query heads" in _err(decode(heads=6))
    assert "query heads" in _err(decode(heads=0))
    assert "q_stride" in _err(decode(q_stride=1020))
    assert "q_stride" in _err(decode(q_stride=1026))
    assert "new_stride" in _err(decode(k_new=FAKE, v_new=FAKE, stride=508))
    assert "aligned" in _err(decode(k_new=FAKE + 4, v_new=FAKE))
    assert "scale" in _err(decode(scale=float("nan")))
    assert "scale" in _err(decode(scale=float("inf")))
    assert "too many" in _err(decode(batch=60000, kv_heads=100, heads=100, q_stride=12800))


def test_gather_refusals():
    for name in ("k_out", "v_out"):
        assert "null" in _err(gather(**{name: None}))
        assert "aligned" in _err(gather(**{name: FAKE + 8}))
    assert "row type" in _err(gather(out_type=2))
    assert "max_len" in _err(gather(max_len=0))
    assert "max_len" in _err(gather(max_len=1 << 31))
    assert "too many" in _err(gather(batch=60000, kv_heads=1000))


def test_verify_refusals():
    for name in ("target", "tokens", "parents", "rand", "path", "accepted", "following"):
        assert "null" in _err(verify(**{name: None}))
    for nodes in (0, 257):
        assert "nodes" in _err(verify(nodes=nodes))
    assert "empty" in _err(verify(batch=0))
    assert "empty" in _err(verify(vocab=0))
    assert "65535" in _err(verify(batch=65536))
    assert "vocab" in _err(verify(vocab=(1 << 28) + 1))


def test_pages_layout_matches_header():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct sts_pages \{(.*?)\} sts_pages;", text, re.S).group(1)
    fields = re.findall(r"(void\*|float\*|u?int32_t)\s+(\w+);", body)
    of = {"void*": ctypes.c_void_p, "float*": ctypes.c_void_p, "uint32_t": ctypes.c_uint32, "int32_t": ctypes.c_int32}
    assert [(n, of[t]) for t, n in fields] == list(sts_attn.Pages._fields_)
    enum = dict(re.findall(r"\b(STS_PAGES_\w+)\s*=\s*(\d+)", text))
    assert {k: int(v) for k, v in enum.items()} == {"STS_PAGES_F32": sts_attn.PAGES_F32,
                                                    "STS_PAGES_BF16": sts_attn.PAGES_BF16,
                                                    "STS_PAGES_INT8": sts_attn.PAGES_INT8}


def test_pools_of_the_wrong_type_or_shape():
    k = torch.zeros((3, 2, 16, 64))
    s = torch.zeros((3, 2, 16))
    with pytest.raises(TypeError, match="int8"):
        sts_attn.PagedKV(k.half(), k.half())
    with pytest.raises(TypeError, match="int8"):
        sts_attn.PagedKV(k, k.bfloat16())
    with pytest.raises(ValueError, match="KVH, page_rows"):
        sts_attn.PagedKV(k, k[:2])
    with pytest.raises(ValueError, match="contiguous"):
        sts_attn.PagedKV(k.transpose(0, 1), k.transpose(0, 1))
    with pytest.raises(ValueError, match="need k_scale"):
        sts_attn.PagedKV(k.to(torch.int8), k.to(torch.int8), s)
    with pytest.raises(ValueError, match="no scales"):
        sts_attn.PagedKV(k, k, s, s)
    with pytest.raises(ValueError, match="k_scale"):
        sts_attn.PagedKV(k.to(torch.int8), k.to(torch.int8), s[:2], s)
    with pytest.raises(ValueError, match="current GPU"):
        sts_attn.PagedKV(k, k).gather(torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), k, k)
    with pytest.raises(ValueError, match="current GPU"):
        sts_attn.verify_draft(torch.zeros((1, 2, 5)), None, None, None)


def test_strides_of_new_rows():
    cpu = torch.device("cpu")

    def at(t, lead, heads=2):
        return sts_attn._heads_stride(t, "k_new", lead, heads, 8, cpu)[1]

    qkv = torch.zeros((3, 5, 6, 8))  # tokens of packed heads
    assert at(qkv[:, :, 2:4], (3, 5)) == 48
    assert at(qkv[:, :1, 2:4], (3, 1)) == 240
    assert at(qkv[:1, :, 2:4], (1, 5)) == 48
    assert at(qkv[0, :, 2:4], (5,)) == 48
    assert at(qkv[:1, :1, 2:4], (1, 1)) == 16
    one = torch.zeros((1, 1, 2, 8))
    for wrong in (qkv[:, :4, 2:4], qkv.transpose(0, 1)[:, :, 2:4], one.expand(3, 1, 2, 8), one.expand(1, 5, 2, 8),
                  one.expand(3, 5, 2, 8), qkv[:1, :, 2:4].expand(3, 5, 2, 8), qkv.as_strided((3, 5, 2, 8), (60, 12, 8, 1))):
        with pytest.raises(ValueError, match="equally far"):
            at(wrong, tuple(wrong.shape[:2]))
    for wrong in (one[0].expand(3, 2, 8), qkv.as_strided((3, 2, 8), (8, 8, 1))):
        with pytest.raises(ValueError, match="overlap"):
            at(wrong, (3,))
    assert at(one.expand(3, 5, 2, 8)[:1, :1], (1, 1)) == 16
    with pytest.raises(ValueError, match="heads must be contiguous"):
        at(qkv[:, :, ::3], (3, 5))
    with pytest.raises(TypeError, match="float32"):
        at(qkv.double()[:, :, :2], (3, 5))
    with pytest.raises(ValueError, match="must be"):
        at(qkv[:, :, :3], (3, 5))


def test_a_pool_keeps_its_tensors():
    """Another tensor in their place would leave the calls with the old ones' addresses, freed perhaps."""
    k, s = torch.zeros((3, 2, 16, 64), dtype=torch.int8), torch.zeros((3, 2, 16))
    pool = sts_attn.PagedKV(k, k.clone(), s, s.clone())
    for name in ("k", "v", "k_scale", "v_scale"):
        t = getattr(pool, name)
        with pytest.raises(AttributeError):
            setattr(pool, name, t.clone())
        assert getattr(pool, name) is t and getattr(pool._c, name) == t.data_ptr()
