"""Decode operators on caller-owned device memory: a quantised paged KV cache (kv_write, kv_read), attention of a tree of
drafted tokens over it (tree_attention), and the choice of the accepted ones (verify_drafts).  Declarations, definitions
and rules: include/pcp_b200.h, "decode operators".

Tensors are anything with data_ptr(), shape, stride() and dtype (torch tensors): types, shapes and strides are checked here,
the rest (device, alignment, sizes) in the library.  `stream` is a cudaStream_t value or None for the default stream; a
call enqueues and returns.  A decoding step with drafts:

    cache = KvCache(k_pages, v_pages, block_table, k_scale, v_scale)
    ws = torch.empty(tree_attention_workspace(cache, n_head, max_nodes), dtype=torch.uint8, device="cuda")
    tree_attention(cache, q, k, v, out, cu_nodes, parent, ctx_len, max_nodes, ws)          # every layer
    verify_drafts(logits, token, cu_nodes, parent, u_accept, u_sample, tokens, path, n, max_nodes, temperature)
    kv_write(cache, k, v, cu_path, ctx_len, path.numel(), index=path)                      # every layer: the accepted rows
"""
from __future__ import annotations

import ctypes as C
import threading

from .backend import BF16, F32, BackendError, E_INVALID, load_library

I8, E4M3 = 16, 17
OPS_BAD_PAGE, OPS_BAD_LENGTH, OPS_BAD_TREE, OPS_NO_CHOICE, OPS_STUCK = 1, 2, 4, 8, 16
TREE_MAX_NODES, TREE_MAX_BATCH = 256, 1024
_ERR_CAP = 256


class CKvCache(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("block_table", C.c_void_p),
                ("page_stride", C.c_longlong), ("scale_stride", C.c_longlong), ("dtype", C.c_int), ("n_pages", C.c_int), ("n_kv_head", C.c_int),
                ("head_dim", C.c_int), ("page_tokens", C.c_int), ("batch", C.c_int), ("max_pages", C.c_int)]


class CKvRows(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_row", C.c_longlong), ("k_head", C.c_longlong), ("v_row", C.c_longlong),
                ("v_head", C.c_longlong), ("cu_rows", C.c_void_p), ("pos0", C.c_void_p), ("index", C.c_void_p), ("dtype", C.c_int),
                ("n_rows", C.c_int), ("n_entries", C.c_int)]


class CTreeAttn(C.Structure):
    _fields_ = [("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("out", C.c_void_p), ("lse", C.c_void_p), ("q_row", C.c_longlong),
                ("q_head", C.c_longlong), ("k_row", C.c_longlong), ("k_head", C.c_longlong), ("v_row", C.c_longlong), ("v_head", C.c_longlong),
                ("out_row", C.c_longlong), ("out_head", C.c_longlong), ("cu_nodes", C.c_void_p), ("parent", C.c_void_p), ("ctx_len", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t), ("n_rows", C.c_int), ("n_head", C.c_int), ("max_nodes", C.c_int),
                ("null_self", C.c_int), ("scale", C.c_float)]


class CVerify(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("draft_probs", C.c_void_p), ("logits_row", C.c_longlong), ("draft_row", C.c_longlong),
                ("cu_nodes", C.c_void_p), ("parent", C.c_void_p), ("token", C.c_void_p), ("u_accept", C.c_void_p), ("u_sample", C.c_void_p),
                ("tokens_out", C.c_void_p), ("path_out", C.c_void_p), ("n_out", C.c_void_p), ("temperature", C.c_double), ("dtype", C.c_int),
                ("vocab", C.c_int), ("n_rows", C.c_int), ("batch", C.c_int), ("max_nodes", C.c_int), ("max_out", C.c_int)]


_lib = None


def _library():
    global _lib
    if _lib is None:
        lib = load_library()
        vp, sz = C.c_void_p, C.c_size_t
        lib.pcpb_op_kv_write.argtypes = lib.pcpb_op_kv_read.argtypes = [vp, vp, vp, vp, C.c_char_p, sz]
        lib.pcpb_op_tree_attention.argtypes = [vp, vp, vp, vp, C.c_char_p, sz]
        lib.pcpb_op_tree_attention_workspace.argtypes = [C.c_int, vp, C.c_int, C.c_int, C.c_char_p, sz]
        lib.pcpb_op_tree_attention_workspace.restype = sz
        lib.pcpb_op_verify_drafts.argtypes = [vp, vp, vp, C.c_char_p, sz]
        _lib = lib
    return _lib


def _refuse(msg):
    raise BackendError(E_INVALID, msg)


_DTYPES: dict = {}


def _dtype(t):
    """Name of a tensor's element type without the framework's prefix ("bfloat16"); looked up once per type."""
    d = t.dtype
    name = _DTYPES.get(d)
    if name is None:
        name = _DTYPES[d] = str(d).rsplit(".", 1)[-1]
    return name


def _vector(t, what, dtype, n=0):
    """Address of a contiguous tensor of one type with at least n values (None stays None)."""
    if t is None:
        return None
    d = t.dtype
    if (_DTYPES.get(d) or _dtype(t)) != dtype:
        _refuse(f"{what} must be {dtype}, not {_dtype(t)}")
    if not t.is_contiguous():
        _refuse(f"{what} must be contiguous")
    if t.numel() < n:
        _refuse(f"{what} holds {t.numel()} values, {n} are needed")
    return t.data_ptr()


def _rows(t, what, dtypes, heads, width):
    """(address, row stride, head stride) of a tensor [rows][heads][width] whose last dimension is dense."""
    shape, stride = t.shape, t.stride()
    d = t.dtype
    if (_DTYPES.get(d) or _dtype(t)) not in dtypes:
        _refuse(f"{what} must be {' or '.join(dtypes)}, not {_dtype(t)}")
    if len(shape) != 3 or shape[2] != width or (heads is not None and shape[1] != heads):
        _refuse(f"{what} must be [rows][{'heads' if heads is None else heads}][{width}], not {tuple(shape)}")
    r, h, e = stride
    if e != 1:
        _refuse(f"the last dimension of {what} must be dense")
    return t.data_ptr(), r if shape[0] > 1 else 0, h if shape[1] > 1 else 0


_CODES = {"bfloat16": BF16, "int8": I8, "float8_e4m3fn": E4M3}
_ROWS = {"bfloat16": BF16, "float32": F32}


class KvCache:
    """One layer's paged cache in tensors of the caller's: k, v [pages][n_kv_head][page_tokens][head_dim] in bfloat16, int8 or
    float8_e4m3fn, the 8-bit ones with k_scale, v_scale [pages][n_kv_head][page_tokens] float32; block_table [batch][max_pages] int32.
    Pages may lie apart (stride of the first dimension); what is inside a page is dense.  The tensors are kept alive."""

    def __init__(self, k, v, block_table, k_scale=None, v_scale=None):
        if len(k.shape) != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            _refuse("k and v must be tensors [pages][n_kv_head][page_tokens][head_dim] of one type, shape and layout")
        if _dtype(k) not in _CODES:
            _refuse(f"cache tensors must be bfloat16, int8 or float8_e4m3fn, not {_dtype(k)}")
        n, h, p, d = k.shape
        if n * h * p == 0 or not k[0].is_contiguous() or not v[0].is_contiguous():
            _refuse("what is inside a page must be dense, and there must be a page")
        c = CKvCache(k=k.data_ptr(), v=v.data_ptr(), dtype=_CODES[_dtype(k)], n_pages=n, n_kv_head=h, head_dim=d, page_tokens=p,
                     page_stride=k.stride(0) if n > 1 else 0)
        if c.dtype != BF16:
            if k_scale is None or v_scale is None or tuple(k_scale.shape) != (n, h, p) or k_scale.shape != v_scale.shape or \
                    k_scale.stride() != v_scale.stride() or not k_scale[0].is_contiguous() or not v_scale[0].is_contiguous() or \
                    {_dtype(k_scale), _dtype(v_scale)} != {"float32"}:
                _refuse("an 8-bit cache needs float32 k_scale and v_scale [pages][n_kv_head][page_tokens] of one layout")
            c.k_scale, c.v_scale, c.scale_stride = k_scale.data_ptr(), v_scale.data_ptr(), k_scale.stride(0) if n > 1 else 0
        if len(block_table.shape) != 2:
            _refuse("block_table must be [batch][max_pages]")
        c.block_table = _vector(block_table, "block_table", "int32")
        c.batch, c.max_pages = block_table.shape
        self.c, self._ref = c, C.addressof(c)
        self.head_dim, self.n_kv_head, self.batch = d, h, c.batch
        self._keep = (k, v, k_scale, v_scale, block_table)


class _Err(threading.local):
    """Room for the reason of a refusal, one per thread."""

    def __init__(self):
        self.buf = C.create_string_buffer(_ERR_CAP)


_err = _Err()


def _call(fn, stream, *args):
    buf = _err.buf
    rc = fn(stream, *args, buf, _ERR_CAP)
    if rc:
        raise BackendError(rc, buf.value.decode())


def _kv_rows(fn, cache, k, v, cu_rows, pos0, n_entries, index, status, stream):
    kp, kr, kh = _rows(k, "k", _ROWS, cache.n_kv_head, cache.head_dim)
    vp, vr, vh = _rows(v, "v", _ROWS, cache.n_kv_head, cache.head_dim)
    if k.dtype != v.dtype or k.shape[0] != v.shape[0]:
        _refuse("k and v must have one type and one number of rows")
    r = CKvRows(kp, vp, kr, kh, vr, vh, _vector(cu_rows, "cu_rows", "int32", cache.batch + 1), _vector(pos0, "pos0", "int32", cache.batch),
                _vector(index, "index", "int32", n_entries), _ROWS[_dtype(k)], k.shape[0], n_entries)
    _call(fn, stream, cache._ref, C.addressof(r), _vector(status, "status", "int32", 1))


def kv_write(cache: KvCache, k, v, cu_rows, pos0, n_entries: int, index=None, status=None, stream=None):
    """Writes rows k, v [rows][n_kv_head][head_dim] (bfloat16 or float32) into the cache: sequence b's entries cu_rows[b] ..
    cu_rows[b + 1] go to positions pos0[b] and on; entry e takes row index[e] (None: row e; negative: nothing is written)."""
    _kv_rows(_library().pcpb_op_kv_write, cache, k, v, cu_rows, pos0, n_entries, index, status, stream)


def kv_read(cache: KvCache, k, v, cu_rows, pos0, n_entries: int, index=None, status=None, stream=None):
    """The reverse of kv_write: rows of the cache as values into k, v."""
    _kv_rows(_library().pcpb_op_kv_read, cache, k, v, cu_rows, pos0, n_entries, index, status, stream)


def tree_attention_workspace(cache: KvCache, n_head: int, max_nodes: int, device: int = 0) -> int:
    """Bytes of device memory tree_attention needs for this cache, n_head query heads and trees of up to max_nodes."""
    err = C.create_string_buffer(_ERR_CAP)
    n = _library().pcpb_op_tree_attention_workspace(device, cache._ref, n_head, max_nodes, err, _ERR_CAP)
    if not n:
        raise BackendError(E_INVALID, err.value.decode())
    return int(n)


def tree_attention(cache: KvCache, q, k, v, out, cu_nodes, parent, ctx_len, max_nodes: int, workspace, scale: float | None = None,
                   null_self: bool = False, lse=None, status=None, stream=None):
    """Attention of the nodes of drafted trees: q, out [rows][n_head][head_dim], k, v [rows][n_kv_head][head_dim], all bfloat16;
    sequence b has the rows cu_nodes[b] .. cu_nodes[b + 1] and ctx_len[b] cached positions; parent [rows] int32 (None: chains).
    scale None: head_dim ** -0.5."""
    d, bf = cache.head_dim, ("bfloat16",)
    qp, qr, qh = _rows(q, "q", bf, None, d)
    n, heads = q.shape[0], q.shape[1]
    kp, kr, kh = _rows(k, "k", bf, cache.n_kv_head, d)
    vp, vr, vh = _rows(v, "v", bf, cache.n_kv_head, d)
    op, orow, oh = _rows(out, "out", bf, heads, d)
    if k.shape[0] != n or v.shape[0] != n or out.shape[0] != n:
        _refuse("q, k, v and out must have one number of rows")
    a = CTreeAttn(qp, kp, vp, op, _vector(lse, "lse", "float32", n * heads), qr, qh, kr, kh, vr, vh, orow, oh,
                  _vector(cu_nodes, "cu_nodes", "int32", cache.batch + 1), _vector(parent, "parent", "int32", n),
                  _vector(ctx_len, "ctx_len", "int32", cache.batch), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                  n, heads, max_nodes, 1 if null_self else 0, d ** -0.5 if scale is None else scale)
    _call(_library().pcpb_op_tree_attention, stream, cache._ref, C.addressof(a), _vector(status, "status", "int32", 1))


def verify_drafts(logits, token, cu_nodes, parent, u_accept, u_sample, tokens_out, path_out, n_out, max_nodes: int, temperature: float = 1.0,
                  draft_probs=None, status=None, stream=None):
    """Walks every sequence's tree from node 0 along the accepted children.  logits [rows][vocab] bfloat16 or float32, token [rows]
    int64, u_accept [rows] and u_sample [batch] float32 in [0, 1) (None when temperature is 0), draft_probs [rows][vocab] float32 or None;
    tokens_out [batch][max_out] int64, path_out [batch][max_out] int32, n_out [batch] int32 receive the result."""
    if len(logits.shape) != 2 or _dtype(logits) not in _ROWS or logits.stride(1) != 1:
        _refuse("logits must be [rows][vocab] bfloat16 or float32 with dense rows")
    n, V = logits.shape
    qp, qr = None, 0
    if draft_probs is not None:
        if tuple(draft_probs.shape) != (n, V) or _dtype(draft_probs) != "float32" or draft_probs.stride(1) != 1:
            _refuse("draft_probs must be float32 [rows][vocab] with dense rows")
        qp, qr = draft_probs.data_ptr(), draft_probs.stride(0)
    if len(tokens_out.shape) != 2 or tokens_out.shape != path_out.shape:
        _refuse("tokens_out and path_out must be [batch][max_out]")
    B, D = tokens_out.shape
    a = CVerify(logits.data_ptr(), qp, logits.stride(0), qr, _vector(cu_nodes, "cu_nodes", "int32", B + 1), _vector(parent, "parent", "int32", n),
                _vector(token, "token", "int64", n), _vector(u_accept, "u_accept", "float32", n), _vector(u_sample, "u_sample", "float32", B),
                _vector(tokens_out, "tokens_out", "int64"), _vector(path_out, "path_out", "int32"), _vector(n_out, "n_out", "int32", B),
                temperature, _ROWS[_dtype(logits)], V, n, B, max_nodes, D)
    _call(_library().pcpb_op_verify_drafts, stream, C.addressof(a), _vector(status, "status", "int32", 1))
