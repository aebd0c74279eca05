"""Refusals of the decode operators that need no GPU: everything the host can see is refused before a CUDA call."""
import ctypes as C

import pytest
import torch

from pcp_b200 import BackendError
from pcp_b200 import backend as bk
from pcp_b200 import decode_ops as ops


def _cache(dtype=torch.bfloat16, hd=64, heads=2, page=16, pages=4, batch=2, width=2, scales=True):
    k = torch.zeros(pages, heads, page, hd, dtype=dtype)
    s = torch.zeros(pages, heads, page) if dtype != torch.bfloat16 and scales else None
    return ops.KvCache(k, k.clone(), torch.zeros(batch, width, dtype=torch.int32), s, None if s is None else s.clone())


def _refused(code, fn, *a, **kw):
    with pytest.raises(BackendError) as ei:
        fn(*a, **kw)
    assert ei.value.code == code, ei.value
    return str(ei.value)


I32 = torch.int32


def test_cache_descriptions(lib_built):
    z = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    bt = torch.zeros(2, 2, dtype=I32)
    _refused(bk.E_INVALID, ops.KvCache, z, z.float(), bt)                        # two types
    _refused(bk.E_INVALID, ops.KvCache, z.float(), z.float(), bt)                # a type no cache has
    _refused(bk.E_INVALID, ops.KvCache, z.transpose(1, 2), z.transpose(1, 2), bt)
    _refused(bk.E_INVALID, ops.KvCache, z, z, bt.long())
    _refused(bk.E_INVALID, ops.KvCache, z, z, bt[0])
    _refused(bk.E_INVALID, _cache, torch.int8, scales=False)
    assert _cache(torch.float8_e4m3fn).c.dtype == ops.E4M3


def _kv(cache, n=3, dtype=torch.bfloat16, **kw):
    hd, h = cache.head_dim, cache.n_kv_head
    k = kw.pop("k", torch.zeros(n, h, hd, dtype=dtype))
    v = kw.pop("v", torch.zeros(n, h, hd, dtype=dtype))
    return (cache, k, v, kw.pop("cu", torch.tensor([0, 1, n], dtype=I32)), kw.pop("pos0", torch.zeros(2, dtype=I32)), kw.pop("n_entries", n))


@pytest.mark.parametrize("fn", [ops.kv_write, ops.kv_read])
def test_kv_refusals(lib_built, fn):
    c = _cache()
    _refused(bk.E_INVALID, fn, *_kv(c, k=torch.zeros(3, 2, 32, dtype=torch.bfloat16)))
    _refused(bk.E_INVALID, fn, *_kv(c, k=torch.zeros(3, 1, 64, dtype=torch.bfloat16)))
    _refused(bk.E_INVALID, fn, *_kv(c, dtype=torch.float16))
    _refused(bk.E_INVALID, fn, *_kv(c, k=torch.zeros(3, 2, 64)))                 # k and v of different types
    _refused(bk.E_INVALID, fn, *_kv(c, cu=torch.zeros(2, dtype=I32)))            # too short
    _refused(bk.E_INVALID, fn, *_kv(c, pos0=torch.zeros(2, dtype=torch.int64)))
    _refused(bk.E_INVALID, fn, *_kv(c, n_entries=-1))
    _refused(bk.E_INVALID, fn, *_kv(c), index=torch.zeros(2, dtype=I32))
    odd = torch.zeros(3, 2, 68, dtype=torch.bfloat16)[..., :64]                  # heads 136 bytes apart
    assert "16-byte" in _refused(bk.E_INVALID, fn, *_kv(c, k=odd, v=odd))
    shifted = torch.zeros(3 * 128 + 1, dtype=torch.bfloat16)[1:].view(3, 2, 64)
    assert "16-byte" in _refused(bk.E_INVALID, fn, *_kv(c, k=shifted, v=shifted))
    _refused(bk.E_INVALID, fn, *_kv(_cache(hd=48)))
    fn(*_kv(c, n_entries=0))                                                     # nothing to do: no device is needed
    for field, bad in (("page_stride", 64), ("n_pages", 0), ("page_tokens", 0), ("dtype", bk.F16), ("batch", 0), ("block_table", None), ("v", None)):
        c = _cache()
        setattr(c.c, field, bad)
        _refused(bk.E_INVALID, fn, *_kv(c, cu=torch.tensor([0, 1, 3], dtype=I32)))
    c = _cache()
    c.c.max_pages = 2 ** 31 - 1
    _refused(bk.E_TOO_LARGE, fn, *_kv(c))


def _attn(cache, n=3, heads=4, max_nodes=3, ws=None, **kw):
    hd, h = cache.head_dim, cache.n_kv_head
    bf = torch.bfloat16
    q = kw.get("q", torch.zeros(n, heads, hd, dtype=bf))
    k = kw.get("k", torch.zeros(n, h, hd, dtype=bf))
    ws = torch.zeros(ops.tree_attention_workspace(_cache(), 4, 256), dtype=torch.uint8) if ws is None else ws
    return (cache, q, k, kw.get("v", k.clone()), kw.get("out", torch.zeros(n, q.shape[1], hd, dtype=bf)), kw.get("cu", torch.tensor([0, 1, n], dtype=I32)),
            kw.get("parent"), kw.get("ctx", torch.zeros(2, dtype=I32)), max_nodes, ws)


def test_attention_refusals(lib_built):
    c = _cache()
    f = ops.tree_attention
    _refused(bk.E_INVALID, f, *_attn(c, heads=3))                                # not a multiple of the kv heads
    _refused(bk.E_INVALID, f, *_attn(c, max_nodes=0))
    _refused(bk.E_TOO_LARGE, f, *_attn(c, max_nodes=257))
    _refused(bk.E_TOO_LARGE, f, *_attn(_cache(batch=1025), cu=torch.zeros(1026, dtype=I32), ctx=torch.zeros(1025, dtype=I32)))
    _refused(bk.E_INVALID, f, *_attn(c, q=torch.zeros(3, 4, 64)))                # f32
    _refused(bk.E_INVALID, f, *_attn(c, k=torch.zeros(2, 2, 64, dtype=torch.bfloat16)))
    _refused(bk.E_INVALID, f, *_attn(c, parent=torch.zeros(3, dtype=torch.int64)))
    _refused(bk.E_INVALID, f, *_attn(c, ctx=torch.zeros(1, dtype=I32)))
    _refused(bk.E_INVALID, f, *_attn(c), lse=torch.zeros(3, 3))
    ws = torch.zeros(1 << 20, dtype=torch.uint8)
    _refused(bk.E_INVALID, f, *_attn(c, ws=ws[1:]))
    f(*_attn(c, n=0, cu=torch.zeros(3, dtype=I32)))                              # no rows: nothing to do
    with pytest.raises(BackendError):
        ops.tree_attention_workspace(c, 5, 4)


def _ver(n=4, V=100, B=2, D=3, **kw):
    return dict(logits=kw.get("logits", torch.zeros(n, V, dtype=torch.bfloat16)), token=kw.get("token", torch.zeros(n, dtype=torch.int64)),
                cu_nodes=kw.get("cu", torch.tensor([0, 2, n], dtype=I32)), parent=kw.get("parent"), u_accept=kw.get("ua", torch.zeros(n)),
                u_sample=kw.get("us", torch.zeros(B)), tokens_out=torch.zeros(B, D, dtype=torch.int64), path_out=kw.get("path", torch.zeros(B, D, dtype=I32)),
                n_out=torch.zeros(B, dtype=I32), max_nodes=kw.get("max_nodes", 3), temperature=kw.get("T", 1.0), draft_probs=kw.get("draft"))


def test_verify_refusals(lib_built):
    f = ops.verify_drafts
    _refused(bk.E_INVALID, f, **_ver(logits=torch.zeros(4, 100, dtype=torch.float16)))
    _refused(bk.E_INVALID, f, **_ver(logits=torch.zeros(100, 4).T))
    _refused(bk.E_INVALID, f, **_ver(token=torch.zeros(4, dtype=I32)))
    _refused(bk.E_INVALID, f, **_ver(draft=torch.zeros(4, 99)))
    _refused(bk.E_INVALID, f, **_ver(path=torch.zeros(2, 4, dtype=I32)))
    _refused(bk.E_INVALID, f, **_ver(T=-1.0))
    _refused(bk.E_INVALID, f, **_ver(T=float("nan")))
    _refused(bk.E_INVALID, f, **_ver(T=float("inf")))
    _refused(bk.E_INVALID, f, **_ver(ua=torch.zeros(3)))
    a = _ver()
    a["u_sample"] = None
    _refused(bk.E_INVALID, f, **a)                                               # sampling needs its numbers
    _refused(bk.E_TOO_LARGE, f, **_ver(max_nodes=257))
    _refused(bk.E_INVALID, f, **_ver(max_nodes=0))


def test_null_arguments_through_the_c_entry(lib_built):
    lib = ops._library()
    err = C.create_string_buffer(256)
    for fn in (lib.pcpb_op_kv_write, lib.pcpb_op_kv_read, lib.pcpb_op_tree_attention):
        assert fn(None, None, None, None, err, 256) == bk.E_INVALID and err.value
        assert fn(None, _cache()._ref, None, None, err, 256) == bk.E_INVALID and err.value
    assert lib.pcpb_op_verify_drafts(None, None, None, err, 256) == bk.E_INVALID and err.value
    assert lib.pcpb_op_verify_drafts(None, None, None, None, 0) == bk.E_INVALID          # no room for the reason


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the error without a device")
def test_without_a_device_the_calls_fail(lib_built):
    c = _cache()
    _refused(bk.E_CUDA, ops.kv_write, *_kv(c))
    _refused(bk.E_CUDA, ops.tree_attention, *_attn(c))
    _refused(bk.E_CUDA, ops.verify_drafts, **_ver())
