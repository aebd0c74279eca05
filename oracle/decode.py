"""Decode operators restated in 64 bits, one row at a time where that is the plainest: quantised rows of a paged cache, attention of
drafted trees over it, verification of drafted tokens.  No code of pcp_b200 is used."""
from __future__ import annotations

import math

import torch

Q = {"e4m3": 448.0, "i8": 127.0}
TORCH = {"e4m3": torch.float8_e4m3fn, "i8": torch.int8, "bf16": torch.bfloat16}


def quantise(x: torch.Tensor, kind: str):
    """Codes and f32 scales of rows [..., width] on the CPU (f32 divisions, rounded to nearest even)."""
    x = x.detach().cpu().float()
    amax = x.abs().amax(-1)
    amax = torch.where(x.isnan().any(-1), torch.tensor(math.nan), amax)
    a = torch.maximum(amax / torch.full_like(amax, Q[kind]), torch.tensor(2.0 ** -126))
    a = torch.where(amax.isfinite(), a, torch.tensor(math.nan))
    y = torch.where(amax.isfinite()[..., None], x / a[..., None], torch.zeros_like(x))
    return (y.clamp(-448, 448).to(torch.float8_e4m3fn) if kind == "e4m3" else y.round().clamp(-127, 127).to(torch.int8)), a


def values(codes: torch.Tensor, scale) -> torch.Tensor:
    return codes.double() if scale is None else codes.float().double() * scale.double()[..., None]


def cached_rows(pages, scales, table_row, page_tokens, n):
    """Rows [n, heads, width] in 64 bits and which of them exist (their page is one of the cache)."""
    val = values(pages.cpu(), None if scales is None else scales.cpu())
    rows, there = [], []
    for t in range(n):
        lp = t // page_tokens
        p = int(table_row[lp]) if lp < len(table_row) else -1
        ok = 0 <= p < val.shape[0]
        there.append(ok)
        rows.append(val[p if ok else 0, :, t % page_tokens])
    return torch.stack(rows) if rows else torch.zeros(0, *val[0, :, 0].shape, dtype=torch.float64), torch.tensor(there, dtype=torch.bool)


def ancestors(parents):
    """[n, n] truth: j is i or above it; a parent that does not come before its child counts as none."""
    m = torch.zeros(len(parents), len(parents), dtype=torch.bool)
    for i, p in enumerate(parents):
        m[i, i] = True
        if 0 <= p < i:
            m[i] |= m[p]
    return m


def tree_attention(q, k_new, v_new, k_old, v_old, there, parents, scale, null_self=False):
    """One sequence.  q [n, H, d]; k_new, v_new [n, Hkv, d]; k_old, v_old [ctx, Hkv, d] with truth there [ctx].
    -> out [n, H, d], lse [n, H], spread [n, H, d] = sum of weight * |value| and slack [n, H] = largest sum |q k| * scale: what error bounds
    are made of.  Masked values never enter, whatever they hold."""
    n, H, d = q.shape
    Hkv = k_new.shape[1]
    see = torch.cat([there[None, :].expand(n, -1), ancestors(parents)], 1)
    out, lse = torch.zeros(n, H, d, dtype=torch.float64), torch.full((n, H), -math.inf, dtype=torch.float64)
    spread, slack = torch.zeros(n, H, d, dtype=torch.float64), torch.zeros(n, H, dtype=torch.float64)
    K, V = torch.cat([k_old, k_new.double()]), torch.cat([v_old, v_new.double()])
    ctx = k_old.shape[0]
    for i in range(n):
        at = see[i].nonzero()[:, 0]
        if len(at) == 0:
            continue
        for h in range(H):
            kk, vv = K[at, h // (H // Hkv)].clone(), V[at, h // (H // Hkv)].clone()
            if null_self:
                own = at == ctx + i
                kk[own], vv[own] = 0.0, 0.0
            s = (kk * q[i, h].double()).sum(-1) * scale
            w = torch.softmax(s, 0)
            out[i, h], lse[i, h] = (w[:, None] * vv).sum(0), torch.logsumexp(s, 0)
            spread[i, h] = (w[:, None] * vv.abs()).sum(0)
            slack[i, h] = ((kk * q[i, h].double()).abs().sum(-1) * abs(scale)).max()
    return out, lse, spread, slack


def verify(logits, token, parents, u_accept, u_sample, temperature, draft=None, max_out=None):
    """One sequence's walk -> (tokens, nodes)."""
    tokens, nodes, node = [], [], 0
    n, V = len(parents), logits.shape[-1]
    max_out = max_out or n
    par = [p if 0 <= p < i else -1 for i, p in enumerate(parents)]
    while n and len(tokens) < max_out:
        z = logits[node].double().cpu()
        nodes.append(node)
        top = z[~z.isnan()].max() if (~z.isnan()).any() else torch.tensor(-math.inf)
        if not bool(top.isfinite()):
            tokens.append(-1)
            break
        kids = [c for c in range(n) if par[c] == node and 0 <= token[c] < V] if len(tokens) + 1 < max_out else []
        taken = None
        if temperature < 1e-6:
            last = int((z == top).nonzero()[0])
            taken = next((c for c in kids if token[c] == last), None)
        else:
            w = torch.exp((z - top) / temperature)
            w = torch.where(z.isnan(), 0.0, w)
            left = w / w.sum()                                   # normalised distribution that is left
            q = draft[node].double().cpu() if draft is not None else None
            for c in kids:
                t = token[c]
                if u_accept[c] * (float(q[t]) if q is not None else 1.0) < float(left[t]):
                    taken = c
                    break
                nxt = (left - q).clamp_min(0.0) if q is not None else left.index_fill(0, torch.tensor([t]), 0.0)
                if float(nxt.sum()) > 0:
                    left = nxt / nxt.sum()
            run = torch.cumsum(left, 0)
            hit = (run > u_sample * float(run[-1])).nonzero()
            last = int(hit[0]) if len(hit) else int((left > 0).nonzero()[-1])
        tokens.append(token[taken] if taken is not None else last)
        if taken is None:
            break
        node = taken
    return tokens, nodes
