"""The decode operators on the GPU against their 64-bit restatement (oracle/decode.py): quantised cache rows bit for bit, tree attention
within a bound made of its roundings, verification token for token; bad pages, lengths and trees; a decoding loop of all three.

Bound of the attention (eps = 2^-8 is half a bf16 step): out = sum w v.  Every weight is rounded to bf16 once (eps), the result once
(eps |out|).  The f32 part: a score is a sum of head_dim products, off by at most head_dim 2^-23 sum |q k| scale (truncating
accumulation), and shifts its weight by twice that; exp2 and the factors' roundings are below 2^-20; the sums over n keys add n 2^-23.
So |error| <= eps |out| + (eps + 2 head_dim 2^-23 slack + 2^-20 + n 2^-23) sum w |v|."""
import math
import random

import pytest
import torch

from oracle import decode as ref
from pcp_b200 import BackendError
from pcp_b200 import backend as bk
from pcp_b200 import decode_ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I32 = torch.int32


def _i32(x):
    return torch.tensor(list(x), dtype=I32, device=DEV)


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return _i32(out)


def _table(lens, page, g, spare=3):
    need = [(n + page - 1) // page for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g).tolist()
    bt = torch.zeros(len(lens), max(max(need), 1), dtype=I32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = torch.tensor(order[at:at + n], dtype=I32)
        at += n
    return bt, total


def _cache(kind, total, heads, page, hd, gap=0):
    """Tensors of a cache; gap: elements between pages (strided pages)."""
    def pages():
        t = torch.zeros(total, heads * page * hd + gap, dtype=torch.uint8 if kind != "bf16" else torch.bfloat16, device=DEV)
        t[:, heads * page * hd:] = 77
        return t, t[:, :heads * page * hd].unflatten(1, (heads, page, hd)).view(ref.TORCH[kind])
    kb, k = pages()
    vb, v = pages()
    s = [torch.full((total, heads, page), -5.0, device=DEV) for _ in range(2)] if kind != "bf16" else [None, None]
    return k, v, s[0], s[1], kb, vb


def _raw(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


# ---------------------------------------------------------------------------------------------------------- cache rows
@pytest.mark.parametrize("kind", ["bf16", "e4m3", "i8"])
@pytest.mark.parametrize("hd,heads,page,lens,src", [
    (128, 8, 16, [1, 1, 1], "bf16"), (64, 3, 24, [33, 0, 7, 1], "bf16"), (32, 1, 5, [40, 2], "f32"), (128, 2, 16, [130], "f32"),
    (64, 16, 8, [3] * 40, "bf16"), (32, 20, 64, [65, 64, 63], "f32")])
def test_rows_are_written_and_read_back_bit_for_bit(kind, hd, heads, page, lens, src):
    g = torch.Generator().manual_seed(hd + heads)
    before = [(7 * i + 3) % (2 * page) for i in range(len(lens))]
    bt, total = _table([a + b for a, b in zip(lens, before)], page, g)
    k, v, ks, vs, kb, vb = _cache(kind, total, heads, page, hd, gap=64)
    dt = torch.bfloat16 if src == "bf16" else torch.float32
    N = sum(lens)
    fused = (torch.randn(N + 2, 3 * heads, hd, generator=g) * torch.exp(3 * torch.randn(N + 2, 3 * heads, 1, generator=g))).to(dt)
    fused[0, heads] = 0.0                                        # a row of zeros
    fused[0, heads + heads - 1, 0] = 1e-38                       # below the smallest scale's reach
    fused[-3, 2 * heads, 3] = 3e38 if src == "f32" else 1e38
    x = fused.to(DEV)
    kr, vr = x[:, heads:2 * heads], x[:, 2 * heads:]             # strided rows, two behind the last sequence
    cache = ops.KvCache(k, v, bt.to(DEV), ks, vs)
    status = torch.zeros(1, dtype=I32, device=DEV)
    ops.kv_write(cache, kr, vr, _starts(lens), _i32(before), N + 2, status=status)
    out = [torch.full((N + 2, heads, hd), 9.0, dtype=dt, device=DEV) for _ in range(2)]
    ops.kv_read(cache, out[0], out[1], _starts(lens), _i32(before), N + 2, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    assert (kb[:, heads * page * hd:] == 77).all() and (vb[:, heads * page * hd:] == 77).all()      # between the pages
    for which, pages, scales, got in ((kr, k, ks, out[0]), (vr, v, vs, out[1])):
        want = torch.zeros(pages.shape, dtype=pages.dtype)
        wscale = torch.full(pages.shape[:3], -5.0)
        codes, a = (which.cpu().to(torch.bfloat16), None) if kind == "bf16" else ref.quantise(which.cpu(), kind)
        e = 0
        for b, n in enumerate(lens):
            for t in range(before[b], before[b] + n):
                p, o = int(bt[b, t // page]), t % page
                _raw(want)[p, :, o] = _raw(codes)[e]
                if a is not None:
                    wscale[p, :, o] = a[e]
                e += 1
        assert torch.equal(_raw(pages).cpu(), _raw(want))
        if a is not None:
            assert torch.equal(scales.cpu(), wscale)
        val = codes[:N].float() if a is None else codes[:N].float() * a[:N, :, None]
        assert torch.equal(got[:N].cpu(), val.to(dt)) and (got[N:] == 9.0).all()


@pytest.mark.parametrize("kind", ["e4m3", "i8"])
def test_a_row_with_an_infinity_or_nan_reads_back_as_nan(kind):
    k, v, ks, vs, _, _ = _cache(kind, 1, 2, 8, 64)
    cache = ops.KvCache(k, v, torch.zeros(1, 1, dtype=I32, device=DEV), ks, vs)
    x = torch.randn(4, 2, 64, device=DEV)
    x[1, 0, 5], x[2, 1, 63], x[3, 0, 0] = math.nan, math.inf, -math.inf
    ops.kv_write(cache, x, x, _i32([0, 4]), _i32([0]), 4)
    out = torch.zeros(4, 2, 64, device=DEV)
    ops.kv_read(cache, out, out.clone(), _i32([0, 4]), _i32([0]), 4)
    bad = torch.zeros(4, 2, dtype=torch.bool, device=DEV)
    bad[1, 0] = bad[2, 1] = bad[3, 0] = True
    assert torch.equal(out.isnan(), bad[..., None].expand_as(out))


@pytest.mark.parametrize("kind", ["e4m3", "i8"])
def test_codes_of_rows_of_every_size(kind):
    """f32 rows from 2^-140 to 2^120, on both sides of every switch in the quotient, with elements across 40 powers of two: codes and scales bit
    for bit those of f32 divisions."""
    g = torch.Generator().manual_seed(11)
    n, page, hd = 261, 16, 64
    x = torch.randn(n, 2, hd, generator=g).double() * torch.exp2(-40 * torch.rand(n, 2, hd, generator=g).double())
    x = (x * torch.exp2(torch.arange(n).double() - 140)[:, None, None]).float()
    k, v, ks, vs, _, _ = _cache(kind, 17, 1, page, hd)
    cache = ops.KvCache(k, v, torch.arange(17, dtype=I32, device=DEV)[None], ks, vs)
    d = x.to(DEV)
    ops.kv_write(cache, d[:, :1], d[:, 1:], _i32([0, n]), _i32([0]), n)
    for i, (pages, scales) in enumerate(((k, ks), (v, vs))):
        c, a = ref.quantise(x[:, i], kind)
        assert torch.equal(scales.cpu().flatten()[:n], a)
        assert torch.equal(_raw(pages).cpu().reshape(-1, hd)[:n], _raw(c))


def test_index_lists_bad_pages_and_bad_positions():
    """index picks source rows and leaves entries out; entries of pages outside the cache or positions outside the table are left out (written)
    or zero (read), and say so."""
    page, heads, hd = 4, 2, 32
    k, v, _, _, _, _ = _cache("bf16", 3, heads, page, hd)
    bt = torch.tensor([[2, 99, -1], [0, 1, 1 << 30]], dtype=I32)
    cache = ops.KvCache(k, v, bt.to(DEV))
    x = torch.arange(10, device=DEV, dtype=torch.float32)[:, None, None].expand(10, heads, hd).contiguous() + 1
    status = torch.zeros(1, dtype=I32, device=DEV)
    # sequence 0: positions 2 .. 5 from rows 7, -, 3, 4 (position 4, 5 are on page 99); sequence 1: positions 0, 1 from rows 9, 0
    ops.kv_write(cache, x, -x, _i32([0, 4, 6]), _i32([2, 0]), 6, index=_i32([7, -1, 3, 4, 9, 0]), status=status)
    want = torch.zeros(3, heads, page, hd)
    want[2, :, 2], want[0, :, 0], want[0, :, 1] = 8.0, 10.0, 1.0
    assert int(status) == ops.OPS_BAD_PAGE
    assert torch.equal(k.float().cpu(), want) and torch.equal(v.float().cpu(), -want)
    # reading: rows go where index says; bad pages give zeros, the rest of the output stays
    out = torch.full((10, heads, hd), 5.0, device=DEV)
    out2 = out.clone()
    status.zero_()
    ops.kv_read(cache, out, out2, _i32([0, 4, 6]), _i32([2, 0]), 6, index=_i32([6, 5, -1, 1, 0, -7]), status=status)
    w = torch.full((10, heads, hd), 5.0)
    w[6], w[5], w[1], w[0] = 8.0, 0.0, 0.0, 10.0
    assert torch.equal(out.cpu(), w) and int(status) == ops.OPS_BAD_PAGE
    # positions before the start and behind the table, source rows outside, cu_rows out of order
    for cu, pos, idx in (([0, 2, 2], [-3, 0], None), ([0, 2, 2], [12, 0], None), ([0, 2, 2], [2 ** 31 - 1, 0], None), ([0, 2, 2], [0, 0], [10, 2 ** 31 - 1])):
        status.zero_()
        before = k.clone()
        ops.kv_write(cache, x, x, _i32(cu), _i32(pos), 2, index=None if idx is None else _i32(idx), status=status)
        assert int(status) == ops.OPS_BAD_LENGTH and torch.equal(k, before), (cu, pos, idx)
    ops.kv_write(cache, x, x, _i32([-5, -9, -20]), _i32([0, 0]), 10, status=status)


# ----------------------------------------------------------------------------------------------------------- attention
def _tree(n, kind, r):
    if kind == "chain":
        return None
    if kind == "star":
        return ([-1] + [0] * (n - 1))[:n]
    if kind == "roots":                                          # several roots: branches that share nothing but the cache
        return [-1 if i % 3 == 0 else i - 1 for i in range(n)]
    return ([-1] + [max(0, i - 1 - r.randrange(0, 4)) for i in range(1, n)])[:n]


def _attention_case(hd, kind, G, Hkv, page, nodes, ctx, tree, seed=0, null_self=False, lse=True, gain=1.0, edit=None, gap=0, scale=None):
    g = torch.Generator().manual_seed(seed)
    r = random.Random(seed)
    bt, total = _table(ctx, page, g)
    k, v, ks, vs, _, _ = _cache(kind, total, Hkv, page, hd, gap)
    for pages, scales in ((k, ks), (v, vs)):
        x = torch.randn(pages.shape, generator=g)
        if kind == "bf16":
            pages.copy_(x.to(torch.bfloat16))
        else:
            c, a = ref.quantise(x, kind)
            _raw(pages).copy_(_raw(c))
            scales.copy_(a)
    N, H = sum(nodes), G * Hkv
    fused = (torch.randn(N + 3, H + 2 * Hkv, hd, generator=g) * gain).to(torch.bfloat16)
    parents = [_tree(n, tree, r) for n in nodes]
    s = dict(bt=bt, k=k, v=v, ks=ks, vs=vs, fused=fused, parents=parents, nodes=nodes, ctx=list(ctx), page=page, hd=hd, H=H, Hkv=Hkv)
    if edit:
        edit(s)
    x = s["fused"].to(DEV)
    q, kn, vn = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    par = None if tree == "chain" else _i32(sum((p for p in parents), []) + [7, 7, 7])
    cache = ops.KvCache(k, v, s["bt"].to(DEV), ks, vs)
    out = torch.full((N + 3, H, hd), 3.0, dtype=torch.bfloat16, device=DEV)
    l = torch.full((N + 3, H), 3.0, device=DEV) if lse else None
    status = torch.zeros(1, dtype=I32, device=DEV)
    most = max(max(nodes), 1)
    ws = torch.full((ops.tree_attention_workspace(cache, H, most),), 255, dtype=torch.uint8, device=DEV)
    args = (cache, q, kn, vn, out, _starts(nodes), par, _i32(s["ctx"]), most, ws)
    kw = dict(null_self=null_self, lse=l, status=status, scale=scale)
    ops.tree_attention(*args, **kw)
    torch.cuda.synchronize()
    s.update(args=args, kw=kw, out=out, lse=l, status=int(status), null_self=null_self, scale=hd ** -0.5 if scale is None else scale)
    return s


def _check_attention(s):
    at, H, Hkv, hd = 0, s["H"], s["Hkv"], s["hd"]
    for b, n in enumerate(s["nodes"]):
        ctx = min(max(s["ctx"][b], 0), s["bt"].shape[1] * s["page"])
        ko, there = ref.cached_rows(s["k"], s["ks"], s["bt"][b], s["page"], ctx)
        vo, _ = ref.cached_rows(s["v"], s["vs"], s["bt"][b], s["page"], ctx)
        f = s["fused"][at:at + n]
        par = s["parents"][b] if s["parents"][b] is not None else [i - 1 for i in range(n)]
        o, l, spread, slack = ref.tree_attention(f[:, :H], f[:, H:H + Hkv], f[:, H + Hkv:], ko, vo, there, par, s["scale"], s["null_self"])
        got = s["out"][at:at + n].double().cpu()
        keys = ctx + n
        eps, f32 = 2.0 ** -8, 2.0 ** -23
        score = hd * f32 * slack
        bound = eps * o.abs() + (eps + (2 * score + 2.0 ** -20 + keys * f32)[..., None]) * spread + 1e-30
        same = (got == o) | (got.isnan() & o.isnan())
        err = torch.where(same, 0.0, (got - o).abs())
        assert not (err > bound).any() and not (err.isnan() & ~same).any(), (b, float((err / bound).nan_to_num(1e9).max()))
        if s["lse"] is not None:
            gl = s["lse"][at:at + n].double().cpu()
            lb = score + 2.0 ** -20 + keys * f32 + l.abs() * 2.0 ** -22
            same = (gl == l) | (gl.isnan() & l.isnan())
            assert not (torch.where(same, 0.0, (gl - l).abs()) > lb).any(), (b, float((gl - l).abs().max()))
        at += n
    assert (s["out"][at:] == 3.0).all() and (s["lse"] is None or (s["lse"][at:] == 3.0).all())


CASES = [
    # hd, cache, G, Hkv, page, nodes, ctx, tree
    (128, "bf16", 4, 2, 16, [1], [1], "chain"),
    (128, "bf16", 4, 2, 16, [1, 1, 1], [0, 127, 129], "chain"),
    (128, "bf16", 8, 1, 16, [7, 0, 2], [128, 50, 300], "tree"),
    (128, "bf16", 1, 3, 24, [17], [515], "tree"),
    (128, "e4m3", 4, 2, 16, [1, 1], [700, 33], "chain"),
    (128, "e4m3", 2, 2, 7, [24, 13], [260, 1], "tree"),
    (128, "i8", 4, 2, 16, [1, 3], [390, 255], "chain"),
    (128, "i8", 4, 1, 64, [64], [1000], "tree"),
    (64, "bf16", 1, 4, 8, [40, 1], [140, 600], "tree"),
    (64, "bf16", 1, 2, 24, [130], [77], "chain"),
    (64, "e4m3", 8, 2, 32, [5, 6], [513, 512], "star"),
    (64, "i8", 2, 2, 1, [9], [37], "roots"),
    (32, "bf16", 4, 2, 16, [12, 1], [200, 0], "tree"),
    (32, "e4m3", 1, 2, 16, [20], [129], "roots"),
    (32, "i8", 3, 1, 16, [6, 6], [64, 300], "tree"),
    (128, "bf16", 1, 1, 128, [256], [0], "chain"),
    (128, "bf16", 2, 1, 16, [256], [90], "tree"),
    (128, "e4m3", 5, 1, 16, [33], [3000], "tree"),
    (128, "e4m3", 16, 1, 16, [1], [600], "chain"),
    (128, "i8", 8, 1, 16, [1, 1], [2000, 31], "chain"),
    (64, "i8", 2, 3, 16, [65, 64, 63], [128, 64, 192], "tree"),
    (128, "bf16", 1, 2, 16, [129], [64], "roots"),
    (64, "bf16", 4, 1, 16, [2] * 50, [(37 * i) % 400 for i in range(50)], "chain"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"hd{c[0]}-{c[1]}-G{c[2]}x{c[3]}-p{c[4]}-n{max(c[5])}-c{max(c[6])}-{c[7]}")
def test_tree_attention_against_64_bits(case):
    s = _attention_case(*case)
    assert s["status"] == 0
    _check_attention(s)
    first = s["out"].clone()
    s["args"][-1].random_(0, 256)                                # the workspace's contents do not matter, nor what the last call left
    s["out"].fill_(3.0)
    ops.tree_attention(*s["args"], **s["kw"])
    assert torch.equal(s["out"], first)                          # the same bits every time


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "i8"])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_own_slot_as_a_zero_key_and_value(kind, hd):
    s = _attention_case(hd, kind, 2, 2, 16, [1, 6, 20, 1], [0, 40, 150, 129], "tree", null_self=True)
    _check_attention(s)
    assert (s["out"][0] == 0).all() and (s["lse"][0] == 0).all()          # nothing but the zero slot


@pytest.mark.parametrize("hd,G,nodes", [(128, 4, [3, 2]), (64, 2, [40, 9])])
def test_bad_pages_lengths_and_trees_are_left_out(hd, G, nodes):
    def pages(s):
        s["bt"][0, 1], s["bt"][0, 3], s["bt"][1, 0] = 10 ** 6, -1, 2 ** 31 - 1
    s = _attention_case(hd, "e4m3", G, 2, 16, nodes, [70, 16], "tree", edit=pages)
    assert s["status"] == ops.OPS_BAD_PAGE
    _check_attention(s)

    def lengths(s):
        s["ctx"][0], s["ctx"][1] = 10 ** 6, -4
    s = _attention_case(hd, "bf16", G, 2, 16, nodes, [64, 20], "tree", edit=lengths)
    assert s["status"] == ops.OPS_BAD_LENGTH
    _check_attention(s)

    def trees(s):
        s["parents"][1][1] = 1
        s["parents"][0][2] = 2 ** 31 - 1
        s["parents"][0][1] = -2 ** 31
    s = _attention_case(hd, "bf16", G, 2, 16, nodes, [64, 20], "tree", edit=trees)
    assert s["status"] == ops.OPS_BAD_TREE
    _check_attention(s)


@pytest.mark.parametrize("kind", ["bf16", "i8"])
@pytest.mark.parametrize("hd,G,n", [(128, 1, 10), (64, 4, 40)])
def test_infinities_and_nan_in_masked_places_stay_out(kind, hd, G, n):
    """Rows of the cache behind ctx_len and of pages of nobody are NaN; one branch of the tree has NaN keys, infinite or NaN values: only its own
    nodes may show them."""
    def edit(s):
        used = torch.zeros(s["k"].shape[0], s["page"], dtype=torch.bool)
        for t in range(s["ctx"][0]):
            used[int(s["bt"][0, t // s["page"]]), t % s["page"]] = True
        for pages, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])):
            t = pages if scales is None else scales
            m = ~used.to(DEV)
            t.transpose(1, 2)[m] = math.nan
        s["parents"][0] = [-1, 0, 0] + [1 + (i + 1) % 2 if i < 5 else i - 2 for i in range(3, n)]
        H, Hkv = s["H"], s["Hkv"]
        s["fused"][2, H + Hkv:, 5] = math.inf                    # values of node 2 (and of what hangs below it)
        s["fused"][4, H:H + Hkv] = math.nan                      # keys of node 4
        s["fused"][4, H + Hkv:, 0] = math.nan
        s["fused"][n:] = math.nan                                # rows of nobody
    s = _attention_case(hd, kind, G, 2, 16, [n], [150], "tree", edit=edit)
    _check_attention(s)
    clean = ~ref.ancestors(s["parents"][0])[:, [2, 4]].any(1)
    assert int(clean.sum()) >= 3 and s["out"][:n].cpu()[clean].isfinite().all()


def test_scores_of_any_size():
    """Large scores (a softmax that is nearly one-hot), large negative ones, scale 0 and a negative scale; strided pages."""
    for gain, scale in ((12.0, None), (30.0, 1.0), (1.0, 0.0), (2.0, -0.3)):
        _check_attention(_attention_case(128, "bf16", 4, 1, 16, [6], [333], "tree", gain=gain, scale=scale, gap=64, lse=gain < 20))


# -------------------------------------------------------------------------------------------------------- verification
def _verify_case(nodes, V, T, tree, draft, dtype=torch.bfloat16, seed=0, max_out=None, edit=None):
    g = torch.Generator().manual_seed(seed)
    r = random.Random(seed)
    N, B = sum(nodes), len(nodes)
    z = torch.randn(N, V, generator=g) * 2.0
    parents = [_tree(n, tree, r) for n in nodes]
    lists = [p if p is not None else [i - 1 for i in range(n)] for p, n in zip(parents, nodes)]
    probs = torch.softmax(z + 0.5 * torch.randn(N, V, generator=g), -1) if draft else None
    token, at = torch.zeros(N, dtype=torch.int64), 0
    for p in lists:
        for i, u in enumerate(p):
            if u >= 0:
                if draft:
                    token[at + i] = int(torch.multinomial(probs[at + u], 1, generator=g))
                else:
                    token[at + i] = r.randrange(V)
                    z[at + u, token[at + i]] = z[at + u].max() + (r.randrange(0, 3) if T < 1e-6 else 2.0 * r.randrange(0, 4))
        at += len(p)
    s = dict(z=z.to(dtype), token=token, lists=lists, probs=probs, ua=torch.rand(N, generator=g), us=torch.rand(B, generator=g))
    if edit:
        edit(s)
    D = max_out or max(max(nodes), 1)
    big = torch.full((N, V + 5), 99.0, dtype=dtype)
    big[:, :V] = s["z"]
    big = big.to(DEV)
    out = [torch.full((B, D), -9, dtype=torch.int64, device=DEV), torch.full((B, D), -9, dtype=I32, device=DEV), torch.full((B,), -9, dtype=I32, device=DEV)]
    status = torch.zeros(1, dtype=I32, device=DEV)
    par = None if tree == "chain" else _i32(sum(s["lists"], []))
    args = (big[:, :V], s["token"].to(DEV), _starts(nodes), par, s["ua"].to(DEV), s["us"].to(DEV), *out, max(max(nodes), 1), T)
    kw = dict(draft_probs=None if s["probs"] is None else s["probs"].to(DEV), status=status)
    ops.verify_drafts(*args, **kw)
    at, accepted = 0, 0
    for b, n in enumerate(nodes):
        sl = slice(at, at + n)
        tok, path = ref.verify(s["z"][sl], s["token"][sl].tolist(), s["lists"][b], s["ua"][sl].tolist(), float(s["us"][b]), T,
                               None if s["probs"] is None else s["probs"][sl], D)
        assert int(out[2][b]) == len(tok), b
        assert out[0][b].tolist() == tok + [0] * (D - len(tok)), b
        assert out[1][b].tolist() == [at + i for i in path] + [-1] * (D - len(tok)), b
        accepted += max(len(tok) - 1, 0)
        at += n
    return dict(accepted=accepted, status=int(status), args=args, kw=kw, out=out)


@pytest.mark.parametrize("T", [0.0, 0.7, 1.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes,V,tree,draft", [
    ([1], 65, "chain", False), ([6, 1, 0, 9], 1000, "chain", False), ([6, 1, 0, 9] + [7] * 8, 1003, "chain", True), ([24] * 7, 50304, "tree", False),
    ([12] * 9, 513, "tree", True), ([9] * 5, 2000, "star", True), ([30] * 4, 31, "star", False), ([256, 100], 4099, "tree", False)])
def test_verification_token_for_token(T, dtype, nodes, V, tree, draft):
    r = _verify_case(nodes, V, T, tree, draft, dtype)
    assert r["status"] == 0
    if max(nodes) > 5 and V > 100 and not (draft and T == 0.0):      # a greedy target rarely takes sampled drafts
        assert r["accepted"] > 0


def test_verification_of_equal_siblings_ties_and_the_ends():
    def same(s):                                                 # siblings with one token: the second has nothing left
        s["token"][1:] = s["token"][1]
    for draft in (False, True):
        for seed in range(6):
            _verify_case([8], 50, 1.0, "star", draft, seed=seed, edit=same)

    def ties(s):
        s["z"][:] = 1.0
        s["token"][:] = 0
    r = _verify_case([5], 300, 0.0, "chain", False, edit=ties)   # the first of equal maxima is token 0
    assert r["accepted"] == 4
    for u in (0.0, 1.0 - 2.0 ** -24):                            # both ends of the interval
        def ends(s):
            s["ua"][:], s["us"][:] = u, u
        _verify_case([7, 7], 501, 1.0, "tree", False, edit=ends)
        _verify_case([7, 7], 501, 1.0, "tree", True, edit=ends)
    r = _verify_case([9, 9], 400, 0.0, "chain", False, max_out=2)        # the walk ends when the places are full
    assert int(r["out"][2].max()) <= 2


def test_verification_without_a_choice_and_masked_tokens():
    def masked(s):                                               # tokens ruled out by -inf, NaN that must not win
        s["z"][:, 3:] = -math.inf
        s["z"][1, 0] = math.nan
    for T in (0.0, 1.0):
        _verify_case([4, 4], 200, T, "tree", False, edit=masked)

    def none(s):
        s["z"][0] = -math.inf
        s["z"][5, 7] = math.inf
        s["z"][8] = math.nan
    for T in (0.0, 1.0):
        r = _verify_case([4, 4, 4], 200, T, "chain", False, edit=none)
        assert r["status"] & ops.OPS_NO_CHOICE and int(r["out"][0][0, 0]) == -1

    def outside(s):
        s["token"][1], s["token"][2] = -1, 200
    for T in (0.0, 1.0):
        assert _verify_case([4], 200, T, "star", False, edit=outside)["status"] == ops.OPS_NO_CHOICE

    def trees(s):
        s["lists"][0][3] = 3
    assert _verify_case([5], 100, 1.0, "tree", False, edit=trees)["status"] == ops.OPS_BAD_TREE


# --------------------------------------------------------------------------------------------------- streams, graphs, refusals
def test_side_stream_and_graph_replay():
    """The three operators captured once on a side stream and replayed on new inputs: the same bits as eager calls."""
    s = _attention_case(128, "e4m3", 4, 2, 16, [5, 9], [300, 40], "tree", lse=False)
    v = _verify_case([6, 7], 700, 1.0, "tree", False)
    cache, q, kn, vn, out, cu, par, ctx, most, ws = s["args"]
    rows = [torch.zeros(14, 2, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    def step(stream):
        ops.tree_attention(*s["args"], **s["kw"], stream=stream)
        ops.kv_read(cache, rows[0], rows[1], _cu14, _pos0, 14, stream=stream)
        ops.verify_drafts(*v["args"], **v["kw"], stream=stream)
    _cu14, _pos0 = _i32([0, 7, 14]), _i32([20, 3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step(side.cuda_stream)
    side.synchronize()
    want = [t.clone() for t in (out[:14], *rows, *v["out"])]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(side.cuda_stream)
    for t in (out[:14], *rows, *v["out"]):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, (out[:14], *rows, *v["out"])))
    q.copy_(torch.randn_like(q.float()))                         # new inputs in the same places
    s["fused"] = torch.cat([q, kn, vn], 1).cpu()
    graph.replay()
    torch.cuda.synchronize()
    out_r = out.clone()
    ops.tree_attention(*s["args"], **s["kw"])
    assert torch.equal(out[:14], out_r[:14])
    del graph


def test_first_call_inside_a_capture_and_calls_without_nodes():
    """A process whose first use of a kernel is a captured one; sequences that are all empty leave everything as it is."""
    s = _attention_case(32, "i8", 3, 1, 8, [2, 3], [40, 9], "tree", lse=False)
    want = s["out"].clone()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    v = _verify_case([3], 40, 0.0, "chain", False, dtype=torch.float32)
    with torch.cuda.graph(graph, stream=side):
        ops.tree_attention(*s["args"], **s["kw"], stream=side.cuda_stream)
        ops.verify_drafts(*v["args"], **v["kw"], stream=side.cuda_stream)
    s["out"][:5].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(s["out"], want)
    del graph
    none = list(s["args"])
    none[5] = _i32([0, 0, 0])
    for hd in (32, 128):
        e = _attention_case(hd, "bf16", 4, 2, 16, [0, 0], [40, 9], "tree", lse=False)
        assert e["status"] == 0 and (e["out"] == 3.0).all()
    ops.tree_attention(*none, **s["kw"])
    assert torch.equal(s["out"], want)


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "i8"])
@pytest.mark.parametrize("hd,G,nodes,tree", [(128, 4, 24, "tree"), (128, 4, 64, "tree"), (64, 1, 130, "chain"), (128, 4, 1, "chain")])
def test_the_same_bits_over_many_runs(kind, hd, G, nodes, tree):
    """Many tiles a block and several blocks an item, run a hundred times: a race between the roles of a block would show as another result
    now and then."""
    s = _attention_case(hd, kind, G, 4, 16, [nodes] * 6, [3000, 2900, 1700, 2500, 40, 2222], tree, lse=False)
    want = s["out"].clone()
    for _ in range(100):
        s["out"].fill_(3.0)
        ops.tree_attention(*s["args"], **s["kw"])
        assert torch.equal(s["out"], want)
    s["nodes"], s["ctx"], s["parents"] = s["nodes"][:1], s["ctx"][:1], s["parents"][:1]          # and the first sequence against 64 bits
    s["out"] = torch.cat([s["out"][:nodes], s["out"][-3:]])
    _check_attention(s)


def test_two_calls_at_once_share_the_inputs():
    """Two streams, one cache and one set of inputs, two outputs and workspaces."""
    for case in ((128, "e4m3", 4, 2, 16, [1, 1, 1], [3000, 2000, 50], "chain"), (128, "bf16", 4, 2, 16, [24, 9, 17], [900, 2000, 50], "tree")):
        s = _attention_case(*case, lse=False)
        cache, q, kn, vn, out, cu, par, ctx, most, ws = s["args"]
        outs, spaces = [torch.full_like(out, 3.0) for _ in range(2)], [torch.empty_like(ws) for _ in range(2)]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(20):
            for i in range(2):
                ops.tree_attention(cache, q, kn, vn, outs[i], cu, par, ctx, most, spaces[i], stream=streams[i].cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], out) and torch.equal(outs[1], out)


@pytest.mark.parametrize("nodes", [[1], [40]])
def test_offsets_pass_32_bits(nodes):
    """Two pages more than 2^31 elements apart: the second one is written, attended and read back."""
    hd, page, stride = 64, 16, (1 << 31) + 4096
    big = [torch.zeros(stride + hd * page, dtype=torch.int8, device=DEV) for _ in range(2)]
    k, v = (t.as_strided((2, 1, page, hd), (stride, page * hd, hd, 1)) for t in big)
    ks, vs = (torch.zeros(2, 1, page, device=DEV) for _ in range(2))
    bt = torch.tensor([[1, 0]], dtype=I32)
    cache = ops.KvCache(k, v, bt.to(DEV), ks, vs)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(24, 2, hd, generator=g).to(torch.bfloat16).to(DEV)
    ops.kv_write(cache, x[:, :1], x[:, 1:], _i32([0, 24]), _i32([0]), 24)
    back = [torch.zeros(24, 1, hd, device=DEV) for _ in range(2)]
    ops.kv_read(cache, back[0], back[1], _i32([0, 24]), _i32([0]), 24)
    for i in range(2):
        assert torch.equal(back[i].cpu(), ref.values(*ref.quantise(x[:, i:i + 1], "i8")).float())
    n = nodes[0]
    f = torch.randn(n, 3, hd, generator=g).to(torch.bfloat16)
    out = torch.empty(n, 1, hd, dtype=torch.bfloat16, device=DEV)
    ws = torch.empty(ops.tree_attention_workspace(cache, 1, n), dtype=torch.uint8, device=DEV)
    y = f.to(DEV)
    ops.tree_attention(cache, y[:, :1], y[:, 1:2], y[:, 2:], out, _i32([0, n]), None, _i32([24]), n, ws)
    _check_attention(dict(H=1, Hkv=1, hd=hd, nodes=nodes, ctx=[24], bt=bt, page=page, k=k, v=v, ks=ks, vs=vs, fused=f, parents=[None], scale=hd ** -0.5,
                          null_self=False, out=out, lse=None))


def test_host_memory_is_refused():
    k, v, _, _, _, _ = _cache("bf16", 2, 1, 16, 64)
    bt = torch.zeros(1, 2, dtype=I32, device=DEV)
    cache = ops.KvCache(k, v, bt)
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16, device=DEV)
    for bad in range(4):
        a = [x, x, _i32([0, 2]), _i32([0])]
        a[bad] = a[bad].cpu()
        with pytest.raises(BackendError) as ei:
            ops.kv_write(cache, *a, 2)
        assert ei.value.code == bk.E_INVALID and "not device memory" in str(ei.value)
    small = torch.zeros(64, dtype=torch.uint8, device=DEV)
    with pytest.raises(BackendError) as ei:
        ops.tree_attention(cache, x, x, x, x.clone(), _i32([0, 2]), None, _i32([3]), 2, small)
    assert ei.value.code == bk.E_INVALID and "workspace" in str(ei.value)


# ------------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("kind", ["bf16", "e4m3", "i8"])
def test_a_decoding_loop_with_drafts_writes_what_one_token_at_a_time_would(kind):
    """Three steps of draft, attend, verify, write for three sequences; the model is a fixed table from the attention's output to logits.  The
    cache afterwards holds, bit for bit, the rows of the accepted tokens in order, and the attention of a new token over it equals the attention
    of the 64-bit restatement over those rows."""
    hd, Hkv, G, page, B, V = 64, 2, 2, 8, 3, 300
    g = torch.Generator().manual_seed(5)
    H = G * Hkv
    emb = torch.randn(V, H + 2 * Hkv, hd, generator=g).to(torch.bfloat16).to(DEV)
    head = (torch.randn(H * hd, V, generator=g) * 0.4).to(DEV)
    bt = torch.randperm(B * 6, generator=g).to(I32).view(B, 6)
    k, v, ks, vs, _, _ = _cache(kind, B * 6, Hkv, page, hd)
    cache = ops.KvCache(k, v, bt.to(DEV), ks, vs)
    ctx = [11, 0, 25]
    prompt = [torch.randint(0, V, (n,), generator=g).tolist() for n in ctx]
    flat = emb[sum(prompt, [])]
    ops.kv_write(cache, flat[:, H:H + Hkv], flat[:, H + Hkv:], _starts(ctx), _i32([0] * B), sum(ctx))
    last = [int(t) for t in torch.randint(0, V, (B,), generator=g)]
    held = [list(p) for p in prompt]
    r = random.Random(1)
    ctx_len = _i32(ctx)
    nodes, most = [6, 5, 7], 7
    ws = torch.empty(ops.tree_attention_workspace(cache, H, most), dtype=torch.uint8, device=DEV)
    total_accepted = 0
    for step in range(3):
        parents = [[-1] + [max(0, i - 1 - r.randrange(2)) for i in range(1, n)] for n in nodes]
        token = torch.randint(0, V, (sum(nodes),), generator=g)
        at = 0
        for b, n in enumerate(nodes):
            token[at] = last[b]
            at += n
        token = token.to(DEV)
        cu, par = _starts(nodes), _i32(sum(parents, []))
        out = torch.empty(sum(nodes), H, hd, dtype=torch.bfloat16, device=DEV)
        for _ in range(2):                                       # second pass: the drafts become the target's favourites of their parents
            x = emb[token]
            ops.tree_attention(cache, x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], out, cu, par, ctx_len, most, ws)
            logits = out.reshape(sum(nodes), -1).float() @ head
            fav, at = logits.argmax(-1), 0
            for b, n in enumerate(nodes):
                for i in range(1, n if step < 2 else 2):
                    token[at + i] = fav[at + parents[b][i]]
                at += n
        x = emb[token]
        ops.tree_attention(cache, x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], out, cu, par, ctx_len, most, ws)
        logits = out.reshape(sum(nodes), -1).float() @ head
        toks, path, n_out = torch.empty(B, most, dtype=torch.int64, device=DEV), torch.empty(B, most, dtype=I32, device=DEV), torch.empty(B, dtype=I32, device=DEV)
        ops.verify_drafts(logits, token, cu, par, None, None, toks, path, n_out, most, 0.0)
        ops.kv_write(cache, x[:, H:H + Hkv], x[:, H + Hkv:], _i32(range(0, B * most + 1, most)), ctx_len, B * most, index=path)
        ctx_len = ctx_len + n_out
        for b in range(B):
            n = int(n_out[b])
            assert n >= 1
            held[b] += [int(token[int(p)]) for p in path[b][:n]]
            last[b] = int(toks[b][n - 1])
            total_accepted += n - 1
    assert total_accepted >= B
    assert ctx_len.tolist() == [len(h) for h in held]
    got = [torch.empty(sum(map(len, held)), Hkv, hd, device=DEV) for _ in range(2)]
    ops.kv_read(cache, got[0], got[1], _starts(map(len, held)), _i32([0] * B), sum(map(len, held)))
    rows = emb[sum(held, [])].cpu()
    for part, have in ((rows[:, H:H + Hkv], got[0]), (rows[:, H + Hkv:], got[1])):
        want = part.float() if kind == "bf16" else ref.values(*ref.quantise(part, kind)).float()
        assert torch.equal(have.cpu(), want)
    x = emb[torch.tensor(last)]
    out = torch.empty(B, H, hd, dtype=torch.bfloat16, device=DEV)
    ops.tree_attention(cache, x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], out, _starts([1] * B), None, ctx_len, 1, ws)
    s = dict(H=H, Hkv=Hkv, hd=hd, nodes=[1] * B, ctx=ctx_len.tolist(), bt=bt, page=page, k=k, v=v, ks=ks, vs=vs, fused=x.cpu(), parents=[[-1]] * B,
             scale=hd ** -0.5, null_self=False, out=out, lse=None)
    _check_attention(s)
