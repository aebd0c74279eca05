"""Measured cases of the decode-side operators: the quantised paged KV cache (written and read back), attention of a tree
of drafted tokens over it, and the verification of drafted tokens against the target's probabilities.

    run(state) with own = False   elementary torch operations in 32 bits (64 for the verification, whose decisions hang on values next to a border)
    run(state) with own = True    pcp_b200.decode_ops, as a decoding loop calls it

Definitions (the kernels, the plain forms and exact() compute these):

  kv     a row x of head_dim values is held as codes c with one f32 scale a: a = max(amax |x| / Q, 2^-126), Q = 448 (e4m3) or 127 (i8),
         c = round(x / a) in the code's type, value a * c.  bf16 caches hold the row itself.
  attn   node i of a sequence (rows of q, k, v) attends the first ctx positions of its sequence's cache, its ancestors and itself:
         out_i = sum_j softmax_j(scale q_i . k_j) v_j; query head h reads kv head h // (n_head / n_kv_head).
  verify walk from node 0; p = softmax(logits of the node / T).  The node's children are tried in index order: child c (token t, number u)
         is taken if u q_t D < max(p_t - a q_t, 0), where q is the distribution that the children were drawn from, a = 0 and D = 1 at
         first, and after each refusal a += D, D = sum max(p - a q, 0) (the residual of repeated rejection).  Without q the children
         count as certain: taken if u D < p_t, after each refusal p_t = 0 and D -= p_t.  When no child is left, the last token is the
         first index whose running sum of the remaining weights passes u_sample times their total.  T = 0: children and the last
         token are compared with the first maximum of the logits.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
QMAX = {"e4m3": 448.0, "i8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "i8": torch.int8, "bf16": torch.bfloat16}
TINY = 2.0 ** -126


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of each of the engine's 16 sequences goes into an e4m3 cache and is read back: the smallest call, latency
        dict(name="kv_token_e4m3", op="kv", cache="e4m3", batch=16, rows=1, kv_heads=8, head_dim=128, page=16, src="bf16", out="bf16"),
        # a batch of prompts of ragged lengths into an i8 cache, read back for the next chunk's attention
        dict(name="kv_prompts_i8", op="kv", cache="i8", batch=16, rows=2048, kv_heads=8, head_dim=128, page=16, src="bf16", out="bf16"),
        # f32 rows (an f32 model's keys) of odd page size and 64-wide heads into an e4m3 cache and back to f32
        dict(name="kv_rows_f32_e4m3", op="kv", cache="e4m3", batch=5, rows=1000, kv_heads=16, head_dim=64, page=24, src="f32", out="f32"),
        # single tokens: one sequence with a short context, bf16 cache: latency
        dict(name="attn_token_bf16_b1", op="attn", cache="bf16", batch=1, nodes=1, ctx=576, heads=32, kv_heads=8, head_dim=128, page=16, tree=False),
        # single tokens: sixteen ragged contexts, e4m3 cache: bandwidth
        dict(name="attn_token_e4m3_b16", op="attn", cache="e4m3", batch=16, nodes=1, ctx=8192, heads=32, kv_heads=8, head_dim=128, page=16, tree=False),
        # trees of 24 drafted tokens over ordinary contexts, bf16 cache
        dict(name="attn_tree_bf16", op="attn", cache="bf16", batch=16, nodes=24, ctx=2048, heads=32, kv_heads=8, head_dim=128, page=16, tree=True),
        # wide trees over long contexts, i8 cache: 256 query rows share every key
        dict(name="attn_tree_i8_long", op="attn", cache="i8", batch=4, nodes=64, ctx=40960, heads=32, kv_heads=8, head_dim=128, page=64, tree=True),
        # a chain of 130 tokens (the next chunk of a prompt) with 64-wide heads, one query head per kv head, odd page size
        dict(name="attn_chain_hd64", op="attn", cache="bf16", batch=8, nodes=130, ctx=1000, heads=16, kv_heads=16, head_dim=64, page=24, tree=False),
        # greedy check of a short chain of one sequence: the smallest verification, latency
        dict(name="verify_greedy_b1", op="verify", batch=1, nodes=6, vocab=50304, logits="bf16", T=0.0, tree=False, draft=False),
        # chains sampled from a drafter whose distributions are at hand, f32 logits
        dict(name="verify_drafter_f32", op="verify", batch=16, nodes=8, vocab=65536, logits="f32", T=0.8, tree=False, draft=True),
        # trees of 24 tokens without a drafter's distribution, the largest vocabulary
        dict(name="verify_tree_bf16", op="verify", batch=32, nodes=24, vocab=151936, logits="bf16", T=1.0, tree=True, draft=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["kv", "attn", "attn", "verify"])
    if op == "kv":
        while True:
            c = dict(op="kv", cache=rng.choice(["bf16", "e4m3", "i8"]), batch=_log(rng, 1, 64), rows=_log(rng, 1, 4096), kv_heads=rng.choice([1, 2, 4, 8, 10, 16]),
                     head_dim=rng.choice([64, 128]), page=rng.choice([8, 16, 24, 32, 64, 128]), src=rng.choice(["bf16", "f32"]), out=rng.choice(["bf16", "f32"]))
            if c["batch"] * c["rows"] * c["kv_heads"] * c["head_dim"] <= 16 * 2048 * 8 * 128 // 2:
                return c
    if op == "attn":
        while True:
            kv = rng.choice([1, 2, 4, 8, 16])
            c = dict(op="attn", cache=rng.choice(["bf16", "e4m3", "i8"]), batch=_log(rng, 1, 64), nodes=_log(rng, 1, 200), ctx=_log(rng, 1, 40000), heads=kv * rng.choice([1, 2, 4, 8]),
                     kv_heads=kv, head_dim=rng.choice([64, 128]), page=rng.choice([8, 16, 24, 32, 64, 128]), tree=rng.random() < 0.6)
            if c["heads"] <= 64 and work(c)["flops"] <= work(listed()[6])["flops"] and work(c)["bytes"] <= work(listed()[6])["bytes"]:
                return c
    while True:
        c = dict(op="verify", batch=_log(rng, 1, 64), nodes=_log(rng, 1, 40), vocab=rng.choice([_log(rng, 65, 160000), 50304, 65536, 151936]),
                 logits=rng.choice(["bf16", "f32"]), T=rng.choice([0.0, 0.6, 1.0, round(rng.uniform(0.3, 1.5), 3)]), tree=rng.random() < 0.5, draft=rng.random() < 0.5)
        if c["batch"] * c["nodes"] * c["vocab"] <= 32 * 24 * 151936 // 2 and c["vocab"] > c["nodes"] + 8:
            return c


# the lengths of a case's sequences: ragged, a function of the case alone
def _lens(case, key):
    top, B = case[key], case["batch"]
    return [max(1 if key != "ctx" else 0, top - (b * 7919 % (top // 2 + 1) if b else 0)) for b in range(B)]


def _nodes(case):
    n = case["nodes"]
    return [max(1, n - (b % 3 if b and n > 4 else 0)) for b in range(case["batch"])]


def work(case):
    if case["op"] == "kv":
        n = sum(_lens(case, "rows")) * case["kv_heads"] * 2                    # rows of K and V
        src, out = (2 if case["src"] == "bf16" else 4), (2 if case["out"] == "bf16" else 4)
        held = case["head_dim"] * (2 if case["cache"] == "bf16" else 1) + (0 if case["cache"] == "bf16" else 4)
        # written (source read, codes written) and read back (codes read, values written)
        return {"bytes": n * (case["head_dim"] * (src + out) + 2 * held), "flops": n * case["head_dim"] * 4}
    if case["op"] == "attn":
        hd, H, Hkv = case["head_dim"], case["heads"], case["kv_heads"]
        held = hd * (2 if case["cache"] == "bf16" else 1) + (0 if case["cache"] == "bf16" else 4)
        by = fl = 0
        for c, n in zip(_lens(case, "ctx"), _nodes(case)):
            by += 2 * Hkv * (c * held + n * hd * 2) + 2 * n * H * hd * 2
            fl += 4 * H * hd * (n * c + (n if case["tree"] else n * (n + 1) // 2))
        return {"bytes": by, "flops": fl}
    # only the rows of the nodes on the accepted path have to be read: one a sequence at least, and about one more for each
    # accepted token (0.7 of the tried levels; trees are about log2 levels deep)
    depth = case["nodes"] - 1 if not case["tree"] else math.log2(case["nodes"] + 1)
    rows = case["batch"] * (1 + sum(0.7 ** (k + 1) for k in range(int(depth))))
    return {"bytes": rows * case["vocab"] * ((2 if case["logits"] == "bf16" else 4) + (4 if case["draft"] else 0)), "flops": rows * case["vocab"] * 4}


# -------------------------------------------------------------------------------------------------------------- prepare
def _pages(lens, page, g):
    """Block table of sequences of these lengths: pages in a shuffled order, a few spare ones among them."""
    need = [(n + page - 1) // page for n in lens]
    width, total = max(max(need), 1), sum(need) + 3
    order = torch.randperm(total, generator=g).tolist()
    bt, at = torch.zeros(len(lens), width, dtype=torch.int32), 0
    for b, n in enumerate(need):
        bt[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return bt.to(DEV), total


def _empty_cache(case, total):
    shape = (total, case["kv_heads"], case["page"], case["head_dim"])
    k, v = (torch.zeros(shape, dtype=CODE[case["cache"]], device=DEV) for _ in range(2))
    if case["cache"] == "bf16":
        return k, v, None, None
    return k, v, torch.zeros(shape[:3], dtype=torch.float32, device=DEV), torch.zeros(shape[:3], dtype=torch.float32, device=DEV)


def _quantise(x, kind):
    """Codes and scales of rows x [..., head_dim], in 32 bits."""
    x = x.float()
    top = x.abs().amax(-1)
    a = (top / torch.full_like(top, QMAX[kind])).clamp_min(TINY)               # a division: by a plain number it would be a product with the inverse
    y = x / a[..., None]
    return (y.to(CODE[kind]) if kind == "e4m3" else y.round().to(torch.int8)), a


def _starts(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)


def _tree(n, tree, r):
    """Parent of each node (index within the sequence, -1 for the root): a chain, or each node under a recent one."""
    if not tree:
        return [i - 1 for i in range(n)]
    return [-1] + [max(0, int(i - 1 - r.randrange(0, max(1, (i + 1) // 2 + 1)))) for i in range(1, n)]


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device=DEV).manual_seed(seed)
    r = random.Random(seed)
    s = {"case": case}
    if case["op"] == "kv":
        lens = _lens(case, "rows")
        before = [r.randrange(0, 3 * case["page"]) for _ in lens]               # rows that are in the cache already
        s["bt"], total = _pages([a + b for a, b in zip(lens, before)], case["page"], g)
        s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"] = _empty_cache(case, total)
        dt = torch.bfloat16 if case["src"] == "bf16" else torch.float32
        N = sum(lens)
        # keys and values as a projection leaves them: one buffer of q | k | v rows, read with its stride; heads of different size
        qkv = torch.randn(N, 3 * case["kv_heads"], case["head_dim"], generator=gd, device=DEV)
        qkv *= torch.rand(3 * case["kv_heads"], case["head_dim"], generator=gd, device=DEV) * 3 + 0.1
        s["qkv"] = qkv.to(dt)
        s["k"], s["v"] = s["qkv"][:, case["kv_heads"]:2 * case["kv_heads"]], s["qkv"][:, 2 * case["kv_heads"]:]
        s["cu"], s["pos0"], s["lens"], s["before"] = _starts(lens), torch.tensor(before, dtype=torch.int32, device=DEV), lens, before
        odt = torch.bfloat16 if case["out"] == "bf16" else torch.float32
        s["k_out"], s["v_out"] = (torch.empty(N, case["kv_heads"], case["head_dim"], dtype=odt, device=DEV) for _ in range(2))
    elif case["op"] == "attn":
        ctx, nodes = _lens(case, "ctx"), _nodes(case)
        s["bt"], total = _pages(ctx, case["page"], g)
        s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"] = _empty_cache(case, total)
        shape = s["k_pages"].shape
        # keys with a few large channels, as trained models have them
        gain = torch.ones(case["kv_heads"], 1, case["head_dim"], device=DEV)
        gain[:, :, ::37] = 3.0
        for p in range(0, total, 4096):
            for name, w in (("k", gain), ("v", 1.0)):
                x = torch.randn((min(4096, total - p),) + tuple(shape[1:]), generator=gd, device=DEV) * w
                if case["cache"] == "bf16":
                    s[name + "_pages"][p:p + 4096] = x.to(torch.bfloat16)
                else:
                    s[name + "_pages"][p:p + 4096], s[name + "_scale"][p:p + 4096] = _quantise(x, case["cache"])
        N, H, Hkv, hd = sum(nodes), case["heads"], case["kv_heads"], case["head_dim"]
        s["qkv"] = torch.randn(N, H + 2 * Hkv, hd, generator=gd, device=DEV).to(torch.bfloat16)
        s["q"], s["k"], s["v"] = s["qkv"][:, :H], s["qkv"][:, H:H + Hkv], s["qkv"][:, H + Hkv:]
        s["cu"], s["ctx_len"] = _starts(nodes), torch.tensor(ctx, dtype=torch.int32, device=DEV)
        s["parents"] = [_tree(n, case["tree"], r) for n in nodes]
        s["parent"] = torch.tensor(sum(s["parents"], []), dtype=torch.int32, device=DEV) if case["tree"] else None
        s["ctx"], s["nodes"], s["out"] = ctx, nodes, torch.empty(N, H, hd, dtype=torch.bfloat16, device=DEV)
    else:
        nodes, V, T = _nodes(case), case["vocab"], case["T"]
        N = sum(nodes)
        s["parents"] = [_tree(n, case["tree"], r) for n in nodes]
        s["parent"] = torch.tensor(sum(s["parents"], []), dtype=torch.int32, device=DEV) if case["tree"] else None
        z = torch.randn(N, V, generator=gd, device=DEV) * 2.5
        tok = torch.zeros(N, dtype=torch.int64)
        s["draft"] = None
        first = np.cumsum([0] + nodes)
        if case["draft"]:                                                        # a drafter near the target; children drawn from it
            s["draft"] = torch.softmax((z + 0.6 * torch.randn(N, V, generator=gd, device=DEV)) / (T or 1.0), -1)
            drawn = torch.multinomial(s["draft"], max(nodes), replacement=True, generator=gd).cpu()
        else:                                                                    # the nodes' favourites: children share about 0.7 of a node's mass
            drawn = torch.randint(0, V - 64, (N, 1), generator=g) + torch.randperm(64, generator=g)[None, :max(nodes)]
        for b, par in enumerate(s["parents"]):
            kids = {}
            for i, p in enumerate(par):
                if p >= 0:
                    kids.setdefault(p, []).append(i)
            for p, ks in kids.items():
                u = int(first[b]) + p
                for j, c in enumerate(ks):
                    tok[int(first[b]) + c] = drawn[u, j]
                if not case["draft"]:
                    t = tok[[int(first[b]) + c for c in ks]].to(DEV)
                    lse = torch.logsumexp(z[u] / (T or 1.0), 0)
                    share = torch.rand(len(ks), generator=gd, device=DEV) + 0.2
                    z[u, t] = (T or 1.0) * (lse + math.log(0.7 / 0.3) + torch.log(share / share.sum()))
                    if T == 0.0 and r.random() < 0.7:
                        z[u, t[r.randrange(len(ks))]] = z[u].amax() + 1.0
        s["logits"] = z.to(torch.bfloat16) if case["logits"] == "bf16" else z
        s["token"], s["cu"], s["nodes"] = tok.to(DEV), _starts(nodes), nodes
        s["u_accept"] = torch.rand(N, generator=gd, device=DEV)
        s["u_sample"] = torch.rand(case["batch"], generator=gd, device=DEV)
        B, D = case["batch"], max(nodes)
        s["tokens_out"], s["path_out"] = torch.empty(B, D, dtype=torch.int64, device=DEV), torch.empty(B, D, dtype=torch.int32, device=DEV)
        s["n_out"] = torch.empty(B, dtype=torch.int32, device=DEV)
    if own and case["op"] != "verify":
        from pcp_b200 import decode_ops as ops
        s["handle"] = ops.KvCache(s["k_pages"], s["v_pages"], s["bt"], s["k_scale"], s["v_scale"])
        if case["op"] == "attn":
            s["ws"] = torch.empty(ops.tree_attention_workspace(s["handle"], case["heads"], max(s["nodes"]), 0), dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------------------------------------------------------------------ run
def run(state):
    s, case = state, state["case"]
    if own:
        from pcp_b200 import decode_ops as ops
        st = torch.cuda.current_stream().cuda_stream
        if case["op"] == "kv":
            n = s["k"].shape[0]
            ops.kv_write(s["handle"], s["k"], s["v"], s["cu"], s["pos0"], n, stream=st)
            ops.kv_read(s["handle"], s["k_out"], s["v_out"], s["cu"], s["pos0"], n, stream=st)
            return s["k_out"], s["v_out"]
        if case["op"] == "attn":
            ops.tree_attention(s["handle"], s["q"], s["k"], s["v"], s["out"], s["cu"], s["parent"], s["ctx_len"], case["nodes"], s["ws"], stream=st)
            return s["out"]
        ops.verify_drafts(s["logits"], s["token"], s["cu"], s["parent"], s["u_accept"], s["u_sample"], s["tokens_out"], s["path_out"], s["n_out"],
                          case["nodes"], case["T"], draft_probs=s["draft"], stream=st)
        return s["tokens_out"], s["path_out"], s["n_out"]
    if case["op"] == "kv":
        return _plain_kv(s, case)
    return _plain_attn(s, case) if case["op"] == "attn" else _plain_verify(s, case)


def _entry_slots(s, case):
    """Physical page and offset of every entry: entry e of sequence b is position pos0[b] + e - cu[b]."""
    N = s["k"].shape[0]
    e = torch.arange(N, dtype=torch.int32, device=DEV)
    b = torch.searchsorted(s["cu"], e, right=True) - 1
    pos = s["pos0"][b] + e - s["cu"][b]
    return s["bt"][b, (pos // case["page"]).long()].long(), (pos % case["page"]).long()


def _plain_kv(s, case):
    pg, off = _entry_slots(s, case)
    for name in ("k", "v"):
        pages, scale = s[name + "_pages"], s[name + "_scale"]
        if scale is None:
            pages[pg, :, off] = s[name].to(torch.bfloat16)
            s[name + "_out"].copy_(pages[pg, :, off])
        else:
            c, a = _quantise(s[name], case["cache"])
            pages.view(torch.uint8)[pg, :, off] = c.view(torch.uint8)
            scale[pg, :, off] = a
            s[name + "_out"].copy_(pages.view(torch.uint8)[pg, :, off].view(pages.dtype).float() * scale[pg, :, off][..., None])
    return s["k_out"], s["v_out"]


def _cached(s, case, name, b, n):
    """The first n rows [n, kv_heads, head_dim] of sequence b in the cache, in 32 bits."""
    pages, scale, page = s[name + "_pages"], s[name + "_scale"], case["page"]
    if n == 0:
        return torch.zeros(0, case["kv_heads"], case["head_dim"], device=DEV)
    at = s["bt"][b, :(n + page - 1) // page].long()
    x = pages.view(torch.uint8)[at].view(pages.dtype).float() if scale is not None else pages[at].float()
    if scale is not None:
        x = x * scale[at][..., None]
    return x.transpose(1, 2).reshape(-1, case["kv_heads"], case["head_dim"])[:n]


def _ancestors(par):
    """[n, n] truth: node j is node i or above it."""
    m = np.eye(len(par), dtype=bool)
    for i, p in enumerate(par):
        if p >= 0:
            m[i] |= m[p]
    return torch.from_numpy(m).to(DEV)


def _plain_attn(s, case):
    H, Hkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    G, at = H // Hkv, 0
    for b, (ctx, n) in enumerate(zip(s["ctx"], s["nodes"])):
        q = s["q"][at:at + n].float().reshape(n, Hkv, G, hd).permute(1, 2, 0, 3).reshape(Hkv, G * n, hd)
        k = torch.cat([_cached(s, case, "k", b, ctx), s["k"][at:at + n].float()]).permute(1, 2, 0)
        v = torch.cat([_cached(s, case, "v", b, ctx), s["v"][at:at + n].float()]).transpose(0, 1)
        z = torch.matmul(q, k) * (1.0 / math.sqrt(hd))
        z.view(Hkv, G, n, ctx + n)[..., ctx:].masked_fill_(~_ancestors(s["parents"][b]), -math.inf)
        e = torch.exp(z - z.amax(-1, keepdim=True))
        o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
        s["out"][at:at + n] = o.reshape(Hkv, G, n, hd).permute(2, 0, 1, 3).reshape(n, H, hd).to(torch.bfloat16)
        at += n
    return s["out"]


def _plain_verify(s, case):
    """All sequences step by step: at every level the rows of the current nodes, then their children in turn."""
    B, D, T = case["batch"], s["tokens_out"].shape[1], case["T"]
    cu = s["cu"].long()
    first, count = cu[:-1], cu[1:] - cu[:-1]
    slot = torch.arange(D, device=DEV)
    there = slot[None, :] < count[:, None]                                       # [B, D] nodes of each sequence
    row = first[:, None] + torch.where(there, slot[None, :], 0)
    par = torch.where(there, s["parent"][row].long() if s["parent"] is not None else slot[None, :] - 1, -2)
    node = torch.zeros(B, dtype=torch.long, device=DEV)
    alive = torch.ones(B, dtype=torch.bool, device=DEV)
    tokens, path, n_out = s["tokens_out"], s["path_out"], s["n_out"]
    tokens.zero_(); path.fill_(-1); n_out.zero_()
    pick = torch.arange(B, device=DEV)
    deepest = max(_depth(p) for p in s["parents"])
    widest = max(max((p.count(u) for u in set(p) if u >= 0), default=0) for p in s["parents"])
    for level in range(deepest):
        here = row[pick, node]
        z = s["logits"][here].double()
        path[:, level] = torch.where(alive, here.int(), path[:, level])
        kid = par == node[:, None]
        rank = torch.cumsum(kid, 1)
        taken = torch.full((B,), -1, dtype=torch.long, device=DEV)
        if T == 0.0:
            best = torch.argmax(z, -1)
        else:
            z = (z - z.amax(-1, keepdim=True)) / T
            p = torch.exp(z)
            p = p / p.sum(-1, keepdim=True)
            w = p.clone()
            q = s["draft"][here].double() if s["draft"] is not None else None
            a, d = torch.zeros(B, dtype=torch.double, device=DEV), torch.ones(B, dtype=torch.double, device=DEV)
        for j in range(widest):
            is_j = kid & (rank == j + 1)
            has = is_j.any(1)
            c = torch.where(has, is_j.int().argmax(1), 0)
            t = s["token"][row[pick, c]]
            if T == 0.0:
                ok = has & (t == best)
            else:
                u = s["u_accept"][row[pick, c]].double()
                qt = q[pick, t] if q is not None else 1.0
                ok = has & (u * qt * d < w[pick, t])
            ok = ok & (taken < 0)
            taken = torch.where(ok, c, taken)
            if T != 0.0:                                                         # the residual after a refusal
                no = has & (taken < 0)
                if q is not None:
                    a2 = a + d
                    w2 = (p - a2[:, None] * q).clamp_min(0.0)
                    d2 = w2.sum(-1)
                    keep = no & (d2 > 0)
                    a, d, w = torch.where(keep, a2, a), torch.where(keep, d2, d), torch.where(keep[:, None], w2, w)
                else:
                    d2 = d - w[pick, t]
                    keep = no & (d2 > 0)
                    d = torch.where(keep, d2, d)
                    w[pick, t] = torch.where(keep, 0.0, w[pick, t])
        if T == 0.0:
            last = best
        else:
            run_sum = torch.cumsum(w, -1)
            last = (run_sum > s["u_sample"].double()[:, None] * run_sum[:, -1:]).int().argmax(-1)
        on = taken >= 0
        tokens[:, level] = torch.where(alive, torch.where(on, s["token"][row[pick, taken.clamp_min(0)]], last), tokens[:, level])
        n_out += alive.int()
        alive = alive & on
        node = torch.where(on, taken, node)
    return tokens, path, n_out


def _depth(par):
    d = []
    for p in par:
        d.append(1 + (d[p] if p >= 0 else 0))
    return max(d)


# ---------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "kv":
        out = []
        for name in ("k", "v"):
            x = s[name].double()
            if case["cache"] == "bf16":
                out.append(x.to(torch.bfloat16).double())
                continue
            amax = x.abs().amax(-1, keepdim=True)
            a = torch.maximum((amax / QMAX[case["cache"]]).float(), torch.tensor(TINY, device=DEV)).double()
            y = (x / a).float().double()
            if case["cache"] == "i8":
                c = torch.round(y)
            else:                                                                # three fraction bits, exponents from -6 up
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
                c = torch.round(y / step) * step
            out.append(c * a)
        return tuple(out)
    if case["op"] == "attn":
        H, Hkv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
        out, at = torch.empty(sum(s["nodes"]), H, hd, dtype=torch.double, device=DEV), 0
        for b, (ctx, n) in enumerate(zip(s["ctx"], s["nodes"])):
            see = torch.zeros(n, ctx + n, dtype=torch.bool, device=DEV)
            see[:, :ctx] = True
            for i in range(n):
                j = i
                while j >= 0:
                    see[i, ctx + j] = True
                    j = s["parents"][b][j]
            where = torch.arange(ctx, device=DEV)
            pg = s["bt"][b][where // page].long()
            for h in range(Hkv):
                kv = []
                for name in ("k", "v"):
                    old = s[name + "_pages"].view(torch.uint8 if case["cache"] != "bf16" else torch.bfloat16)[pg, h, where % page]
                    old = old.view(CODE[case["cache"]]).double()
                    if case["cache"] != "bf16":
                        old = old * s[name + "_scale"][pg, h, where % page].double()[:, None]
                    kv.append(torch.cat([old, s[name][at:at + n, h].double()]))
                for hq in range(h * (H // Hkv), (h + 1) * (H // Hkv)):
                    score = (s["q"][at:at + n, hq].double() @ kv[0].T) / math.sqrt(hd)
                    out[at:at + n, hq] = torch.softmax(score.masked_fill(~see, -math.inf), -1) @ kv[1]
            at += n
        return out
    B, D, T = case["batch"], max(s["nodes"]), case["T"]
    tokens, path, n_out = np.zeros((B, D), np.int64), np.full((B, D), -1, np.int32), np.zeros(B, np.int32)
    tok, ua, us = s["token"].tolist(), s["u_accept"].tolist(), s["u_sample"].tolist()
    first = 0
    for b, par in enumerate(s["parents"]):
        node, level = 0, 0
        while True:
            z = s["logits"][first + node].double()
            kids = [i for i, p in enumerate(par) if p == node]
            nxt = None
            if T == 0.0:
                last = int((z == z.max()).nonzero()[0])
                nxt = next((c for c in kids if tok[first + c] == last), None)
            else:
                p = torch.softmax(z / T, 0)
                q = s["draft"][first + node].double() if s["draft"] is not None else None
                res = p.clone()                                                  # normalised residual
                for c in kids:
                    t = tok[first + c]
                    drawn_with = float(q[t]) if q is not None else 1.0
                    if ua[first + c] * drawn_with < float(res[t]):
                        nxt = c
                        break
                    r = (res - q).clamp_min(0.0) if q is not None else res.index_fill(0, torch.tensor([t], device=DEV), 0.0)
                    if float(r.sum()) > 0:
                        res = r / r.sum()
                c_sum = torch.cumsum(res, 0)
                last = int((c_sum > us[b] * float(c_sum[-1])).nonzero()[0])
            path[b, level] = first + node
            tokens[b, level] = tok[first + nxt] if nxt is not None else last
            n_out[b] += 1
            level += 1
            if nxt is None:
                break
            node = nxt
        first += len(par)
    return tokens, path, n_out
