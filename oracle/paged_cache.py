"""CPU restatement of the paged 8-bit key/value cache.  TEST INFRASTRUCTURE ONLY.

The reference has no cache (its keys and values are the call's own, reference src/fused_attn_extention.cu:15-22); what is
restated here are the definitions in include/fused_attn.h, token by token and head by head in float64, with the rotation in
float32 as the definition has it.

What pins each function (tests/test_paged_cache.py, on the CPU):
  e4m3         against torch's float8_e4m3fn over every code and the midpoints between codes
  exponent_of  against its definition at every border 448 * 2^e and its neighbours
  append       what was appended comes back within half a step of e4m3; parts give what the whole gives
  attention    against `oracle.attention` on the values that the cache stands for
  select       the score of a page is no smaller than what any of its keys scores with the rounded query, as appended, nor by more than
               the rounding to e4m3 smaller than what the stored ones do, and closed forms
"""
import math

import numpy as np
import torch

LEAST_EXPONENT = -80


def e4m3(x):
    """float64 x rounded to e4m3 (OCP FP8, to nearest even): the values, not the codes.  |x| <= 448 or NaN."""
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        step = np.exp2(np.maximum(np.floor(np.log2(np.abs(x))), -6) - 3)
    step = np.where(np.isfinite(step) & (step > 0), step, 2.0 ** -9)
    return np.rint(x / step) * step


def exponent_of(amax):
    """The smallest e with amax <= 448 * 2^e, not below LEAST_EXPONENT."""
    e = LEAST_EXPONENT
    if amax > 0:
        e = max(e, int(math.floor(math.log2(amax / 448.0))) - 1)
        while amax > 448.0 * 2.0 ** e:
            e += 1
    return e


def rotate(x, cos, sin):
    """x [..., H] float32 rotated by the tables' rows cos, sin [H / 2], each product and each sum rounded to float32."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * cos - b * sin, b * cos + a * sin], axis=-1)


class Cache:
    """The cache's tensors as numpy arrays; codes as the float64 values they have."""

    def __init__(self, k, v, k_exponents, v_exponents, page_table, key_bounds=None):
        self.codes = {"k": k.float().double().cpu().numpy().copy(), "v": v.float().double().cpu().numpy().copy()}
        self.exponents = {"k": k_exponents.cpu().numpy().astype(np.int64), "v": v_exponents.cpu().numpy().astype(np.int64)}
        self.bounds = None if key_bounds is None else key_bounds.cpu().numpy().astype(np.int64)
        self.table = page_table.cpu().numpy().astype(np.int64)
        self.pages, self.heads, self.P, self.H = self.codes["k"].shape

    def page(self, b, w):
        """The page of tokens w P .. w P + P - 1, or None."""
        if not 0 <= w < self.table.shape[1]:
            return None
        page = self.table[b, w]
        return int(page) if 0 <= page < self.pages else None

    def values(self, name, page, head):
        return self.codes[name][page, head] * 2.0 ** self.exponents[name][page, head]

    def codes_tensor(self, name):
        return torch.from_numpy(self.codes[name]).float().to(torch.float8_e4m3fn)


def append(cache, k, v, starts, lens, cos=None, sin=None):
    """k, v [B, L, heads, H] (16-bit tensors) appended in place; starts and lens are lists."""
    rows = None if cos is None else cos.shape[0]
    for b in range(k.shape[0]):
        first, end = starts[b], starts[b] + max(0, min(lens[b], k.shape[1]))
        tokens = [t for t in range(max(first, 0), end) if rows is None or t < rows]
        for w in sorted({t // cache.P for t in tokens}):
            page = cache.page(b, w)
            if page is None:
                continue
            here = [t for t in tokens if t // cache.P == w]
            before = here[0] - w * cache.P                         # earlier tokens on the page
            for name, x in (("k", k), ("v", v)):
                for head in range(cache.heads):
                    y = np.stack([x[b, t - first, head].float().numpy() for t in here])
                    if name == "k" and cos is not None:
                        with np.errstate(over="ignore", invalid="ignore"):
                            y = np.stack([rotate(y[n], cos[t].numpy(), sin[t].numpy()) for n, t in enumerate(here)])
                    y = y.astype(np.float64)
                    counted = np.where(np.isfinite(y), y, 0.0)
                    old = int(cache.exponents[name][page, head])
                    e = exponent_of(np.abs(counted).max())
                    if before:
                        e = max(e, old)
                        codes = cache.codes[name][page, head]
                        codes[:before] = e4m3(codes[:before] * 2.0 ** (old - e))
                    cache.exponents[name][page, head] = e
                    cache.codes[name][page, head, before:before + len(here)] = e4m3(np.where(np.isfinite(y), y, np.nan) * 2.0 ** -e)
                    if name == "k" and cache.bounds is not None:
                        steps = counted * 2.0 ** (-e - 2)
                        up, down = np.ceil(steps.max(axis=0)), np.floor(steps.min(axis=0))
                        if before:
                            up = np.maximum(up, np.ceil(cache.bounds[page, head, 0] * 2.0 ** (old - e)))
                            down = np.minimum(down, np.floor(cache.bounds[page, head, 1] * 2.0 ** (old - e)))
                        cache.bounds[page, head] = np.stack([up, down]).astype(np.int64)


def rotated_queries(q, starts, lens, cos=None, sin=None):
    """q [B, L, R, H] rotated, rounded once to its type; zeros for tokens that do not exist or have no row in the tables."""
    out = torch.zeros_like(q)
    for b in range(q.shape[0]):
        for i in range(max(0, min(lens[b], q.shape[1]))):
            if cos is None:
                out[b, i] = q[b, i]
            elif 0 <= starts[b] + i < cos.shape[0]:
                with np.errstate(over="ignore", invalid="ignore"):
                    y = rotate(q[b, i].float().numpy(), cos[starts[b] + i].numpy(), sin[starts[b] + i].numpy())
                out[b, i] = torch.from_numpy(y).to(q.dtype)
    return out


def _visible(cache, starts, lens, b, i, L, causal):
    n = max(0, min(lens[b], L))
    if i >= n:
        return 0
    return max(0, min(starts[b] + (i + 1 if causal else n), cache.table.shape[1] * cache.P))


def attention(cache, q, starts, lens, selected=None, causal=True, scale=None):
    """out [B, L, R, H], lse [B, R, L] and, for tolerances, the attention over |values| and the largest sum of |q k| of a row, all float64.
    selected: [B, L, heads, count] places in the page table, or None."""
    B, L, R, H = q.shape
    scale = 1.0 / math.sqrt(H) if scale is None else scale
    group = R // cache.heads
    out, spread = np.zeros((B, L, R, H)), np.zeros((B, L, R, H))
    lse, size = np.full((B, R, L), -np.inf), np.zeros((B, L, R))
    x = q.double().numpy()
    for b in range(B):
        for head in range(cache.heads):
            keys, values, at = [], [], []
            for w in range(cache.table.shape[1]):
                page = cache.page(b, w)
                if page is not None:
                    keys.append(cache.values("k", page, head))
                    values.append(cache.values("v", page, head))
                    at.append(np.arange(w * cache.P, (w + 1) * cache.P))
            if not keys:
                continue
            keys, values, at = np.concatenate(keys), np.concatenate(values), np.concatenate(at)
            rows = slice(head * group, (head + 1) * group)
            seen = at < np.array([_visible(cache, starts, lens, b, i, L, causal) for i in range(L)])[:, None]      # [L, keys]
            if selected is not None:
                seen &= np.stack([np.isin(at // cache.P, selected[b, i, head].numpy()) for i in range(L)])
            seen = np.repeat(seen, group, axis=0)                  # a row per token and query head
            with np.errstate(invalid="ignore", divide="ignore"):
                y = x[b, :, rows].reshape(L * group, H)
                s = np.where(seen, y @ keys.T * scale, -np.inf)
                top = s.max(axis=1, keepdims=True)
                p = np.where(seen, np.exp(s - np.where(top == -np.inf, 0.0, top)), 0.0)
                total = p.sum(axis=1, keepdims=True)
                # a NaN that a row does not see is none of its business: zero in its place, and counted apart
                bad = np.isnan(values)
                o = p @ np.where(bad, 0.0, values) / np.where(total == 0, 1.0, total)
                o[(seen.astype(np.float64) @ bad) > 0] = np.nan
                a = p @ np.where(bad, 0.0, np.abs(values)) / np.where(total == 0, 1.0, total)
                z = np.where(seen, np.abs(y) @ np.abs(keys).T, 0.0).max(axis=1) * scale
                out[b, :, rows], spread[b, :, rows] = o.reshape(L, group, H), a.reshape(L, group, H)
                lse[b, rows] = np.where(total == 0, -np.inf, top + np.log(total))[:, 0].reshape(L, group).T
                size[b, :, rows] = z.reshape(L, group)
    return torch.from_numpy(out), torch.from_numpy(lse), torch.from_numpy(spread), torch.from_numpy(size)


def select(cache, q, starts, lens, count):
    """int32 [B, L, heads, count]."""
    B, L, R, H = q.shape
    group = R // cache.heads
    out = torch.full((B, L, cache.heads, count), -1, dtype=torch.int32)
    for b in range(B):
        for i in range(L):
            n = -(-_visible(cache, starts, lens, b, i, L, True) // cache.P)
            for head in range(cache.heads):
                x = q[b, i, head * group:(head + 1) * group].double().numpy()
                x = np.where(np.isfinite(x), x, 0.0)
                e = 0
                if np.abs(x).max() > 0:
                    e = int(math.floor(math.log2(np.abs(x).max() / 127.0))) - 1
                    while np.abs(x).max() > 127.0 * 2.0 ** e:
                        e += 1
                x = np.rint(x * 2.0 ** -e).astype(np.int64)
                scores = []
                for w in range(n):
                    page = cache.page(b, w)
                    if page is None:
                        continue
                    up, down = cache.bounds[page, head]
                    dot = int((np.maximum(x, 0) @ up + np.minimum(x, 0) @ down).max())
                    scores.append((math.inf if w == n - 1 else dot * 2.0 ** int(cache.exponents["k"][page, head]), w))
                best = sorted(w for _, w in sorted(scores, key=lambda s: (-s[0], s[1]))[:count])
                out[b, i, head, :len(best)] = torch.tensor(best, dtype=torch.int32)
    return out
