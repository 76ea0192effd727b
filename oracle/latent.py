"""CPU restatement of latent attention as include/fused_attn.h defines it, in float64.  TEST INFRASTRUCTURE ONLY.

What pins it (tests/test_latent.py, on the CPU): the absorbed form over latents is the expanded form over the keys and values that the
same latents expand to, with queries and outputs through the same maps; the expanded form against torch's softmax of whole
matrices.
"""
import math

import torch


def visible(starts, lens, L, most, causal):
    """How many keys token i of sequence b sees, [B, L]; lens and starts are lists."""
    seen = torch.zeros(len(starts), L, dtype=torch.int64)
    for b, (start, n) in enumerate(zip(starts, lens)):
        n = max(0, min(n, L))
        for i in range(n):
            seen[b, i] = max(0, min(start + (i + 1 if causal else n), most))
    return seen


def rows_attention(q, keys, values, seen, scale):
    """q [n, D], keys [K, D], values [K, V] (NaN rows of keys: no key there), seen [n]: out, lse, and for tolerances the attention over
    |values| and the largest scale * sum |q k| of a row that it sees."""
    K = keys.shape[0]
    there = ~torch.isnan(keys).all(dim=1) if K else torch.zeros(0, dtype=torch.bool)
    mask = (torch.arange(K)[None] < seen[:, None]) & there[None]
    k = torch.where(there[:, None], keys, 0.0)
    s = torch.where(mask, (q @ k.T) * scale, -math.inf)
    top = s.amax(dim=1, keepdim=True) if K else torch.full((q.shape[0], 1), -math.inf, dtype=torch.float64)
    p = torch.where(mask, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = p.sum(dim=1, keepdim=True)
    v = torch.where(there[:, None], values, 0.0)
    norm = torch.where(total == 0, 1.0, total)
    out, spread = p @ v / norm, p @ v.abs() / norm
    lse = torch.where(total == 0, -math.inf, top + total.log())[:, 0]
    size = torch.where(mask, q.abs() @ k.abs().T * scale, 0.0).amax(dim=1) if K else torch.zeros(q.shape[0], dtype=torch.float64)
    return out, lse, spread, size


def gathered(cache, table, b):
    """The cached tokens of sequence b in order, float64 [W * P, channels]; NaN where there is no page."""
    N, P, D = cache.shape
    out = torch.full((table.shape[1], P, D), math.nan, dtype=torch.float64)
    for w, page in enumerate(table[b].tolist()):
        if 0 <= page < N:
            out[w] = cache[page].double()
    return out.flatten(0, 1)


def absorbed(q, r, cache, table, starts, lens, scale, causal=True):
    """q [B, L, R, C], r [B, L, R, DR], cache [N, P, C + DR] -> out [B, L, R, C], lse [B, R, L], spread, size, all float64."""
    B, L, R, C = q.shape
    seen = visible(starts, lens, L, table.shape[1] * cache.shape[1], causal)
    x = torch.cat([q, r], -1).double()
    out, spread = torch.zeros(B, L, R, C, dtype=torch.float64), torch.zeros(B, L, R, C, dtype=torch.float64)
    lse, size = torch.full((B, R, L), -math.inf, dtype=torch.float64), torch.zeros(B, L, R, dtype=torch.float64)
    for b in range(B):
        keys = gathered(cache, table, b)[:int(seen[b].max())]
        o, s, a, z = rows_attention(x[b].flatten(0, 1), keys, keys[:, :C], seen[b].repeat_interleave(R), scale)
        out[b], spread[b], lse[b], size[b] = o.view(L, R, C), a.view(L, R, C), s.view(L, R).T, z.view(L, R)
    return out, lse, spread, size


def expanded(q, k, kr, v, starts, lens, scale, causal=True):
    """q [B, L, R, DN + DR], k [B, K, R, DN], kr [B, K, DR], v [B, K, R, DV] -> as `absorbed`."""
    B, L, R, _ = q.shape
    K, DV = k.shape[1], v.shape[3]
    seen = visible(starts, lens, L, K, causal)
    out, spread = torch.zeros(B, L, R, DV, dtype=torch.float64), torch.zeros(B, L, R, DV, dtype=torch.float64)
    lse, size = torch.full((B, R, L), -math.inf, dtype=torch.float64), torch.zeros(B, L, R, dtype=torch.float64)
    for b in range(B):
        n = int(seen[b].max())
        for h in range(R):
            keys = torch.cat([k[b, :n, h], kr[b, :n]], -1).double()
            o, s, a, z = rows_attention(q[b, :, h].double(), keys, v[b, :n, h].double(), seen[b], scale)
            out[b, :, h], spread[b, :, h], lse[b, h], size[b, :, h] = o, a, s, z
    return out, lse, spread, size
