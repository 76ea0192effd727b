"""Latent attention: the oracle and the refusals on the CPU; on the GPU appending bit by bit, and the absorbed and the expanded form
against the oracle in 64 bits and against each other.

Tolerance of the attention, from its roundings.  With u half a step of the element type (fp16 2^-11, bf16 2^-8), D the channels of a
key, n the keys of a row, A = sum p |v| / sum p, and d = (D + 8) 2^-24 max_j scale sum |q k_j| + |s| 2^-22 what a float32 score may be off by
(products of 16-bit numbers are exact, D of them are summed; the scale and the exponential's argument):
  each weight is rounded once to the element type and off by e^d, the exponential itself by 2^-22, its row's sum's reciprocal by 2^-22:
                                                                                    A (u + 2 d + 2^-20)
  sums of n terms, joined over lanes, waves and parts, in float32:                  A 2 (n + 64) 2^-24
  fp16 weights below what fp16 holds, half of 2^-24 against a reference of 2^8:     n 2^-33 max |v|
  the result is rounded once:                                                       u |out| + 2^-25 (fp16)
"""
import ctypes
import math

import pytest
import torch

from fused_attention_amd import capi
from oracle import latent as lo
from oracle import rotary as ro

F16, BF16, I32 = torch.float16, torch.bfloat16, torch.int32


def _module():
    import fused_attn

    return fused_attn


class Problem:
    """A latent cache and a call, on the CPU."""

    def __init__(self, B=2, L=1, R=4, C=128, DR=32, P=16, W=4, dtype=BF16, seed=0, extra=3):
        self.B, self.L, self.R, self.C, self.DR, self.P, self.W, self.dtype = B, L, R, C, DR, P, W, dtype
        self.gen = torch.Generator().manual_seed(seed)
        N = B * W + extra
        self.cache = self.normal(N, P, C + DR)
        self.table = torch.randperm(N, generator=self.gen)[:B * W].to(I32).view(B, W)
        self.starts, self.lens = [0] * B, [L] * B
        self.q, self.r = self.normal(B, L, R, C), self.normal(B, L, R, DR)
        self.scale = 1.0 / math.sqrt(128 + DR)

    def normal(self, *shape, std=1.0):
        return (std * torch.randn(*shape, generator=self.gen)).to(self.dtype)

    def on(self, dev):
        t = {"latent_cache": self.cache, "page_table": self.table, "starts": torch.tensor(self.starts, dtype=I32),
             "new_lens": torch.tensor(self.lens, dtype=I32)}
        return {name: x.to(dev) for name, x in t.items()}

    def want(self, causal=True):
        return lo.absorbed(self.q, self.r, self.cache, self.table, self.starts, self.lens, self.scale, causal)


def _check(got, lse, want, D, n, dtype, most):
    """got [B, L, R, V]; want: what the oracle returns; most: the largest |value|."""
    out, want_lse, spread, size = want
    u = 2.0 ** -11 if dtype == F16 else 2.0 ** -8
    s = torch.where(torch.isfinite(want_lse), want_lse, 0.0).abs().transpose(1, 2) + math.log(max(n, 2))
    d = (D + 8) * 2.0 ** -24 * size + s * 2.0 ** -22
    tol = spread * (u + 2 * d[..., None] + 2.0 ** -20 + 2 * (n + 64) * 2.0 ** -24) + u * out.abs() + 2.0 ** -133
    if dtype == F16:
        tol = tol + n * 2.0 ** -33 * most + 2.0 ** -25
    got = got.cpu().double()
    assert not torch.isnan(got).any()
    excess = (got - out).abs() - tol
    assert excess.max().item() <= 0, "max excess %.3e" % excess.max().item()
    nothing = (want_lse == -math.inf).transpose(1, 2)[..., None].expand_as(got)
    assert torch.equal(got[nothing], torch.zeros_like(got[nothing]))
    if lse is not None:
        lse = lse.cpu().double()
        at = torch.isfinite(want_lse)
        assert torch.equal(at, torch.isfinite(lse)) and torch.equal(lse[~at], want_lse[~at])
        off = (lse - want_lse)[at].abs() - (d.transpose(1, 2)[at] + 2.0 ** -20 + want_lse[at].abs() * 2.0 ** -22 + (n + 64) * 2.0 ** -24)
        assert off.numel() == 0 or off.max().item() <= 0


def _compare(gpu, p, causal=True, m=None, q=None, r=None, table=None):
    t = p.on(gpu)
    if table is not None:
        t["page_table"] = table
    got, lse = (m or _module()).latent_attention(p.q.to(gpu) if q is None else q, p.r.to(gpu) if r is None else r, scale=p.scale, causal=causal,
                                                 return_lse=True, **t)
    assert got.dtype == p.dtype and tuple(got.shape) == (p.B, p.L, p.R, p.C) and got.is_contiguous() and lse.dtype == torch.float32
    _check(got, lse, p.want(causal), p.C + p.DR, p.W * p.P, p.dtype, p.cache[torch.isfinite(p.cache)].abs().max().item())
    return got, lse


# ---- the oracle, on the CPU ----

def test_the_two_forms_of_the_oracle_are_one():
    # keys W_h c, values U_h c: queries absorb W_h, outputs go through U_h
    g = torch.Generator().manual_seed(1)
    B, L, R, C, DR, D, P, W = 2, 5, 3, 32, 8, 16, 4, 6
    cache = torch.randn(B * W, P, C + DR, generator=g, dtype=torch.float64)
    table = torch.randperm(B * W, generator=g).view(B, W)
    wk, wv = torch.randn(R, C, D, generator=g, dtype=torch.float64), torch.randn(R, C, D, generator=g, dtype=torch.float64)
    q, r = torch.randn(B, L, R, D, generator=g, dtype=torch.float64), torch.randn(B, L, R, DR, generator=g, dtype=torch.float64)
    starts, lens = [7, 18], [5, 3]
    out, lse, _, _ = lo.absorbed(torch.einsum("blrd,rcd->blrc", q, wk), r, cache, table, starts, lens, 0.3)
    kept = torch.stack([lo.gathered(cache, table, b) for b in range(B)])
    k, v = (torch.einsum("bkc,rcd->bkrd", kept[..., :C], w) for w in (wk, wv))
    want, want_lse, _, _ = lo.expanded(torch.cat([q, r], -1), k, kept[..., C:], v, starts, lens, 0.3)
    assert (torch.einsum("blrc,rcd->blrd", out, wv) - want).abs().max() < 1e-12 and torch.equal(lse == -math.inf, want_lse == -math.inf)
    assert (lse - want_lse)[torch.isfinite(lse)].abs().max() < 1e-12 and (out[1, 3:] == 0).all()
    # against whole matrices
    s = torch.einsum("lrd,krd->rlk", torch.cat([q, r], -1)[0], torch.cat([k[0], kept[0, :, None, C:].expand(-1, R, -1)], -1)) * 0.3
    s = s.masked_fill(torch.arange(W * P)[None, None] > 7 + torch.arange(L)[None, :, None], -math.inf)
    assert (torch.einsum("rlk,krd->lrd", s.softmax(-1), v[0]) - want[0]).abs().max() < 1e-12


# ---- refusals, on the CPU ----

def test_the_library_refuses_what_its_header_says():
    lib, ok = capi.load_library(), 0x1000                          # never dereferenced: every case is refused before a launch
    good = dict(latents=ok, page_table=ok, pages=10, page_size=64, latent_dim=128, rope_dim=32, sequences=3, table_width=4, table_stride=4)

    def cache(**kw):
        return ctypes.byref(capi.LatentCache(**{**good, **kw}))

    def append(c=None, x=ok, xs=(256, 128), k=ok, ks=(64, 32), q=ok, qs=(256, 32, 128), out=ok, os=(256, 32, 128), starts=ok, lens=None, L=2, R=4, cos=None,
               sin=None, rows=0, flags=0):
        return lib.fa_latent_append(cache() if c is None else c, x, *xs, k, *ks, q, *qs, out, *os, starts, lens, L, R, cos, sin, rows, flags, None)

    def attend(c=None, q=ok, qs=(1024, 128, 512), r=ok, rs=(256, 32, 128), out=ok, os=(1024, 128, 512), lse=None, starts=ok, lens=None, L=2, R=4,
               scale=0.125, flags=0, ws=None, n=0):
        return lib.fa_latent_attention(cache() if c is None else c, q, *qs, r, *rs, out, *os, lse, starts, lens, L, R, scale, flags, ws, n, None)

    for call in (append, attend):
        assert [call(c=cache(latent_dim=n)) for n in (0, 64, 192, 1024)] == [-2] * 4 and [call(c=cache(rope_dim=n)) for n in (0, 16, 128)] == [-2] * 3
        assert [call(c=cache(page_size=n)) for n in (0, 8, 48, 256)] == [-9] * 4
        for name in ("pages", "sequences", "table_width"):
            assert call(c=cache(**{name: 0})) == -3, name
        assert call(L=0) == -3 and call(R=0) == -3
        assert call(c=cache(table_stride=3)) == -4
        assert call(c=cache(latents=None)) == -1 and call(c=cache(page_table=None)) == -1 and call(starts=None) == -1 and call(out=None) == -1
        assert call(c=cache(latents=ok + 8)) == -5 and call(c=cache(page_table=ok + 2)) == -5 and call(starts=ok + 1) == -5 and call(lens=ok + 2) == -5
        assert call(c=cache(pages=2 ** 31)) == -6 and call(c=cache(table_width=2 ** 27, table_stride=2 ** 27)) == -6 and call(L=2 ** 31) == -6
        assert call(flags=16) == -7 and call(flags=8) == -7
        assert call(q=ok + 2) == -5 and call(out=ok + 8) == -5 and call(qs=(1024, 60, 512)) == -4 and call(qs=(-8, 128, 512)) == -4
        assert call(os=(0, 128, 512)) == -4 and call(os=(1024, 8, 512)) == -4
    assert append(flags=1) == -7 and attend(flags=4) == -7
    assert append(x=None) == -1 and append(k=None) == -1 and append(xs=(256, 120)) == -4 and append(ks=(64, 24)) == -4 and append(q=None) == -1
    assert append(cos=ok) == -1 and append(cos=ok, sin=ok) == -3 and append(cos=ok + 4, sin=ok, rows=9) == -5
    assert attend(q=None) == -1 and attend(r=None) == -1 and attend(rs=(256, 30, 128)) == -4 and attend(lse=ok + 2) == -5
    assert [attend(scale=s) for s in (0.0, -1.0, math.inf, math.nan, 2.9e38)] == [-8] * 5
    long = dict(table_width=4096, table_stride=4096)
    need = lib.fa_latent_attention_workspace(cache(**long), 2, 4)
    assert need > 0 and attend(c=cache(**long)) == -10 and attend(c=cache(**long), ws=ok, n=need - 1) == -10 and attend(c=cache(**long), ws=ok + 4, n=need) == -5
    assert lib.fa_latent_attention_workspace(cache(latent_dim=3), 1, 4) == -2 and lib.fa_latent_attention_plan(cache(), 1, 4, None) == -1
    i64 = ctypes.c_int64

    def expanded(scale=0.125, flags=0, ws=None, n=0, **kw):
        x = capi.Expanded(**{**dict(q=ok, k=ok, rope_k=ok, v=ok, out=ok, sequences=3, tokens=2, heads=4, keys=9, key_dim=64, rope_dim=32, value_dim=64,
                                    q_strides=(i64 * 3)(768, 96, 384), k_strides=(i64 * 3)(2304, 64, 256), rope_k_strides=(i64 * 2)(288, 32),
                                    v_strides=(i64 * 3)(2304, 64, 256), out_strides=(i64 * 3)(512, 64, 256)), **kw})
        return lib.fa_expanded_attention(ctypes.byref(x), scale, flags, ws, n, None)

    assert lib.fa_expanded_attention(None, 0.1, 0, None, 0, None) == -1
    for name in ("q", "k", "rope_k", "v", "out"):
        assert expanded(**{name: None}) == -1 and expanded(**{name: ok + 8}) == -5, name
    for kw in (dict(key_dim=32, value_dim=32), dict(value_dim=128), dict(rope_dim=16)):
        assert expanded(**kw) == -2, kw
    for name in ("sequences", "tokens", "heads", "keys"):
        assert expanded(**{name: 0}) == -3 and expanded(**{name: 2 ** 31}) == -6, name
    for name, bad in (("q_strides", (768, 90, 384)), ("k_strides", (2304, 64, -8)), ("v_strides", (2304, 4, 256)), ("out_strides", (512, 0, 256))):
        assert expanded(**{name: (i64 * 3)(*bad)}) == -4, name
    assert expanded(rope_k_strides=(i64 * 2)(288, 30)) == -4 and expanded(k_strides=(i64 * 3)(0, 64, 2 ** 24 + 8)) == -6
    assert expanded(flags=4) == -7 and expanded(scale=0.0) == -8 and expanded(lse=ok + 2) == -5 and expanded(starts=ok + 1) == -5 and expanded(new_lens=ok + 1) == -5
    assert expanded(keys=65536) == -10 and expanded(keys=65536, ws=ok + 4, n=1 << 40) == -5


@pytest.mark.parametrize("how", ["module", "capi"])
def test_the_entry_points_refuse_wrong_tensors(how):
    m = _module() if how == "module" else capi
    errors = RuntimeError if how == "module" else (ValueError, TypeError)
    p = Problem(B=2, L=3, R=4, C=128, DR=32)
    t = p.on("cpu")
    x, k, qr = p.normal(2, 3, 128), p.normal(2, 3, 32), p.normal(2, 3, 4, 32)
    calls = {"append": lambda **kw: m.latent_append(**{**t, "latents": x, "rope_keys": k, "queries": qr, **kw}),
             "attend": lambda **kw: m.latent_attention(**{**t, "queries": p.q, "rope_queries": p.r, "scale": 0.1, **kw})}

    def refused(match, which=("append", "attend"), **kw):
        for name in which:
            with pytest.raises(errors, match=match):
                calls[name](**kw)

    refused("GPU")
    refused("latent_cache must", latent_cache=p.cache.float())
    refused("latent_cache must", latent_cache=p.cache[0])
    refused("contiguous", latent_cache=p.cache.transpose(0, 1))
    refused("latent channels must", latent_cache=p.cache[..., :96].contiguous())
    refused("must hold 16, 32, 64 or 128", latent_cache=p.cache[:, :8].contiguous())
    refused("page_table must be", page_table=t["page_table"].long())
    refused("page_table must be", page_table=t["page_table"].t())
    refused("starts must", starts=t["starts"][:1])
    refused("new_lens must", new_lens=t["new_lens"].float())
    a, b = ("append",), ("attend",)
    refused("rotary channels must", a, rope_keys=k[..., :16])
    refused("latents must", a, latents=x[..., :64])
    refused("latents must", a, latents=x.half())
    refused("rope_keys must", a, rope_keys=k[:, :2])
    refused("queries must", a, queries=qr[:, :2])
    refused("queries must", a, queries=qr.half())
    refused("last dimension", a, latents=x.repeat_interleave(2, 2)[..., ::2])
    table = torch.zeros(9, 16)
    if how == "module":
        refused("go together", a, rope_cos=table)
        refused("must be", a, rope_cos=table, rope_sin=table.double())
        refused("must be", a, rope_cos=table[:, :8].contiguous(), rope_sin=table[:, :8].contiguous())
    else:
        refused("pair", a, rope=table)
        refused("must be", a, rope=(table[:, :8].contiguous(),) * 2)
    refused("rotary channels must", b, rope_queries=p.r[..., :16])
    refused("queries must", b, queries=p.q[..., :64])
    refused("rope_queries must", b, rope_queries=p.r[:, :, :2])
    refused("queries must", b, queries=p.q.half())
    refused("batch", ("attend",), queries=p.q[:1]) if how == "module" else refused("queries must", b, queries=p.q[:1])
    q, kv, kr = torch.zeros(2, 3, 4, 96, dtype=F16), torch.zeros(2, 5, 4, 64, dtype=F16), torch.zeros(2, 5, 32, dtype=F16)

    def bad(match, **kw):
        with pytest.raises(errors, match=match):
            m.expanded_attention(**{**dict(queries=q, keys=kv, rope_keys=kr, values=kv), **kw})

    bad("GPU")
    bad("queries must be float16 or bfloat16", queries=q.float())
    bad("keys must", keys=kv[:, :, :2])
    bad("values must", values=kv[:, :4])
    bad("64 or 128 channels", keys=kv[..., :32], values=kv[..., :32])
    bad("rotary channels", queries=q[..., :80])
    bad("rope_keys must", rope_keys=kr[:, :4])
    bad("dtype", keys=kv.bfloat16())
    bad("at least as many", queries=q.repeat(1, 2, 1, 1))
    bad("starts must", starts=torch.zeros(1, dtype=I32))
    bad("new_lens must", new_lens=torch.zeros(2))


def test_launches_are_within_what_the_kernels_take():
    for B, L, R, C, DR, P, W in [(1, 1, 1, 128, 32, 16, 1), (64, 1, 16, 512, 64, 64, 128), (1, 1, 128, 512, 64, 128, 1024), (3, 4096, 128, 256, 64, 64, 64),
                                 (1024, 1, 16, 512, 64, 64, 100), (1025, 1, 16, 512, 64, 64, 100)]:
        plan = capi.latent_attention_plan(B, L, R, C, DR, P, W)
        assert plan["rows"] in (16, 32, 64) and plan["workgroups"] >= 1
        if plan["shared"]:
            assert plan["workgroups"] <= 512 and B * -(-L * R // plan["rows"]) <= 1024
        else:
            assert plan["workgroups"] == B * -(-L * R // plan["rows"])
    assert capi.latent_attention_plan(64, 1, 16, 512, 64, 64, 128) == {"rows": 16, "shared": 1, "workgroups": 256}
    for B, L, R, K, D, DR in [(1, 1, 1, 1, 64, 32), (1, 4096, 32, 16384, 128, 64), (1, 2, 1, 16384, 64, 32), (64, 1000, 128, 1000, 128, 64)]:
        plan = capi.expanded_attention_plan(B, L, R, K, D, DR)
        assert plan["rows"] in (128, 256) and 1 <= plan["splits"] <= 128 and plan["workgroups"] == B * R * -(-L // plan["rows"]) * plan["splits"]


# ---- on the GPU: appending ----

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("C,DR,P", [(128, 32, 16), (256, 64, 32), (512, 64, 128), (512, 32, 64)])
@pytest.mark.parametrize("interleaved,rope", [(False, True), (True, True), (False, False)])
def test_append_is_the_oracles(gpu, dtype, C, DR, P, interleaved, rope):
    B, L, R, W = 5, 21, 3, 5
    p = Problem(B, L, R, C, DR, P, W, dtype, seed=C + P)
    p.starts, p.lens = [0, 13, P * W - 9, -4, 17], [21, 9, 21, 21, -3]
    p.table[1, 0], p.table[0, 1] = -1, p.cache.shape[0]            # no pages there
    p.cache[0, 0, 0] = math.nan                                    # whatever stands elsewhere stays
    both = p.normal(B, L, C + DR)                                  # slices of one projection
    both[4, 0] = math.inf
    heads = p.normal(B, L, R, 16 + DR)
    rows = P * W - 5                                               # the tables end before the cache does
    cos, sin = (torch.from_numpy(x).float() for x in ro.tables(rows, DR))
    starts, lens = torch.tensor(p.starts), torch.tensor(p.lens)
    at = starts[:, None] + torch.arange(L)
    exists = torch.arange(L)[None] < lens[:, None]
    if rope:
        keys = ro.rotate(both[:, :, None, C:], cos, sin, at, interleaved=interleaved, exists=exists)[:, :, 0]
        want_q = ro.rotate(heads[..., 16:], cos, sin, at, interleaved=interleaved, exists=exists)
    else:
        keys, want_q = both[..., C:], torch.where(exists[:, :, None, None], heads[..., 16:], 0.0)
    want = p.cache.clone()
    for b in range(B):
        for i in range(L):
            pos = p.starts[b] + i
            if exists[b, i] and 0 <= pos < P * W and (not rope or pos < rows) and 0 <= p.table[b, pos // P] < len(want):
                want[p.table[b, pos // P], pos % P] = torch.cat([both[b, i, :C], keys[b, i]])
    for m in (_module(), capi):
        t = p.on(gpu)
        d, h = both.to(gpu), heads.to(gpu)
        tables = (cos.to(gpu), sin.to(gpu)) if rope else None
        kw = {"rope": tables} if m is capi else dict(zip(("rope_cos", "rope_sin"), tables or (None, None)))
        got = m.latent_append(d[..., :C], d[..., C:], queries=h[..., 16:], interleaved=interleaved, **kw, **t)
        assert torch.equal(got.cpu(), want_q) and got.is_contiguous()
        assert torch.equal(t["latent_cache"].cpu().view(torch.int16), want.view(torch.int16))
        assert m.latent_append(d[..., :C], d[..., C:], interleaved=interleaved, **kw, **t) is None
        assert torch.equal(t["latent_cache"].cpu().view(torch.int16), want.view(torch.int16))


# ---- on the GPU: the absorbed form ----

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("C,DR", [(128, 32), (128, 64), (256, 32), (256, 64), (512, 32), (512, 64)])
@pytest.mark.parametrize("R,L,P,W", [(1, 1, 16, 1), (4, 1, 64, 3), (16, 1, 32, 40), (5, 3, 16, 33), (31, 1, 128, 9), (40, 2, 64, 12), (128, 1, 16, 45), (3, 50, 32, 6),
                                     (16, 33, 64, 3)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_is_the_oracles(gpu, dtype, C, DR, R, L, P, W, causal):
    p = Problem(3, L, R, C, DR, P, W, dtype, seed=R + L + W)
    most = P * W
    p.lens = [L, max(1, L - 1), L // 2 + 1]
    p.starts = [most - L, (most - L) // 2, min(most - L, 17)]
    _compare(gpu, p, causal)
    _compare(gpu, p, causal, m=capi)


@pytest.mark.gpu
@pytest.mark.parametrize("R,L,W", [(4, 1, 3), (16, 1, 60), (40, 3, 60), (16, 20, 5), (64, 1, 60)])
@pytest.mark.parametrize("C,DR", [(128, 32), (256, 64), (512, 64)])
def test_rows_that_see_nothing_and_odd_lengths(gpu, R, L, W, C, DR):
    # no token yet, no token in the call, lengths beyond both ends, positions beyond the table and before it, tables without pages
    p = Problem(10, L, R, C, DR, 16, W, F16, seed=L)
    most = 16 * W
    p.starts = [-L, 0, 5, most, most - 1, most + 100, -1, 30, 0, 40]
    p.lens = [L, 0, -7, L, L + 9, L, L, L, 1, L]
    p.table[7] = -1
    p.table[9, 0], p.table[9, 2] = 2 ** 31 - 1, -2 ** 31
    got, lse = _compare(gpu, p)
    assert (got[7] == 0).all() and (lse[7] == -math.inf).all()
    _compare(gpu, p, causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,R,C,DR,P,W", [(1, 1, 16, 128, 32, 16, 8192), (1, 1, 3, 512, 64, 128, 1000), (300, 1, 4, 128, 64, 16, 11), (1030, 1, 2, 128, 32, 16, 13),
                                            (2, 300, 16, 256, 64, 32, 30), (40, 3, 40, 128, 32, 64, 9)])
def test_many_keys_and_many_rows(gpu, B, L, R, C, DR, P, W):
    p = Problem(B, L, R, C, DR, P, W, BF16, seed=B)
    most = P * W
    p.lens = [max(1, (L * (7 + b % 3)) // 9) for b in range(B)]
    p.starts = [(most - L) * (b * 7 % 11 + 1) // 11 for b in range(B)]
    p.starts[0] = most - L
    _compare(gpu, p)


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,R,C,DR,P,W,lens", [(200, 1, 20, 256, 32, 64, 16, "even"), (300, 1, 4, 512, 64, 16, 64, "ragged"), (260, 1, 16, 512, 32, 16, 40, "few"),
                                                 (130, 2, 24, 256, 64, 32, 20, "ragged"), (7, 3, 50, 128, 32, 32, 50, "ragged"), (70, 1, 3, 512, 64, 16, 40, "none"),
                                                 (2, 700, 3, 128, 64, 64, 30, "ragged"), (1, 9, 16, 512, 64, 16, 300, "even"), (90, 1, 40, 256, 32, 16, 60, "few")])
def test_shares_of_many_sequences(gpu, B, L, R, C, DR, P, W, lens):
    # both ways to share out keys, and a launch where there is nothing to share out
    p = Problem(B, L, R, C, DR, P, W, F16, seed=B + R)
    most = P * W - L
    p.starts = [{"even": most, "ragged": (most * (b * 37 % 101)) // 100, "few": most if b % 29 == 3 else -L, "none": -L}[lens] for b in range(B)]
    p.lens = [L if b % 3 else max(1, L // 2) for b in range(B)]
    assert capi.latent_attention_plan(B, L, R, C, DR, P, W)["shared"] == 1
    first = _compare(gpu, p)
    again = _compare(gpu, p)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("C,DR,R,L,W", [(128, 32, 4, 1, 3), (512, 64, 16, 1, 60), (512, 64, 40, 2, 30), (256, 64, 16, 9, 4), (128, 64, 8, 40, 5)])
def test_what_is_not_finite_stays_where_it_is_seen(gpu, dtype, C, DR, R, L, W):
    P = 16
    p = Problem(3, L, R, C, DR, P, W, dtype, seed=C)
    p.starts = [P * W - L - 5, 2 * P + 3 if P * W >= 2 * P + 3 + L else 0, 0]
    p.lens = [L, L, L]
    clean = _compare(gpu, p)
    bad = p.cache.clone()
    seen = set()
    for b in range(3):                                             # everything that nobody sees, of pages and beside them
        end = p.starts[b] + L
        for pos in range(P * W):
            if pos < end:
                seen.add((int(p.table[b, pos // P]), pos % P))
    for page in range(bad.shape[0]):
        for slot in range(P):
            if (page, slot) not in seen:
                bad[page, slot] = (math.nan, math.inf, -math.inf)[(page + slot) % 3]
    t = p.on(gpu)
    t["latent_cache"] = bad.to(gpu)
    got = _module().latent_attention(p.q.to(gpu), p.r.to(gpu), scale=p.scale, return_lse=True, **t)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
    # a token of the call that only later ones see, and one behind a page boundary: those rows alone
    for b, i, channel, value in ((0, L - 1, 3, math.nan), (1, L // 2, C - 1, math.inf), (0, L // 2, C + 1, math.nan), (2, 0, 0, -math.inf)):
        pos = p.starts[b] + i
        cache = bad.clone()
        cache[p.table[b, pos // P], pos % P, channel] = value
        t["latent_cache"] = cache.to(gpu)
        out, lse = _module().latent_attention(p.q.to(gpu), p.r.to(gpu), scale=p.scale, return_lse=True, **t)
        sees = torch.zeros(3, L, dtype=torch.bool)
        sees[b, i:] = True
        assert torch.equal(out.cpu()[~sees], clean[0].cpu()[~sees])
        if channel < C:
            assert not torch.isfinite(out.cpu()[sees][..., channel]).any()
        elif math.isnan(value):
            assert torch.isnan(out.cpu()[sees]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("R,C,DR", [(16, 128, 32), (40, 512, 64)])
def test_scores_that_rise_and_fall(gpu, dtype, R, C, DR):
    # references that have to follow from tile to tile, rows apart from each other, and keys far below the largest one
    p = Problem(2, 2, R, C, DR, 16, 60, dtype, seed=3)
    p.starts = [60 * 16 - 2, 500]
    for b in range(2):
        for w in range(60):
            p.cache[p.table[b, w]] = (p.cache[p.table[b, w]].float() * (0.05 + 3.0 * ((w * 7) % 13) / 13)).to(dtype)
    _compare(gpu, p)
    p.q *= 4
    _compare(gpu, p)
    p.cache[p.table[0, 30], 5] = p.cache[p.table[0, 30], 5] * 8    # one key far above the others
    _compare(gpu, p)


def _end_to_end(p):
    """Whether the workgroups lay the key tiles of all sequences end to end (causal calls): equal parts of a sequence's keys need more workgroups than
    there are, or make one of them have too much.  A restatement of what each workgroup works out from the lengths."""
    plan = capi.latent_attention_plan(p.B, p.L, p.R, p.C, p.DR, p.P, p.W)
    tiles, steps = -(-p.L * p.R // plan["rows"]), -(-p.W * p.P // 64)
    groups = min(p.B * tiles * -(-steps // 2), 512 if p.C == 128 else 256)
    of = [-(-max(0, min(start + n, p.W * p.P)) // 64) if n > 0 else 0 for start, n in zip(p.starts, p.lens)]
    share = max(2, -(-sum(of) * tiles // groups))
    fits = [part for part in (share + (share * t + 7) // 8 for t in range(16)) if sum(-(-n // part) for n in of) * tiles <= groups]
    return not fits or fits[0] > share + 5


def _unseen(p):
    """[pages, P]: the places of the cache that no row of a call sees."""
    unseen = torch.ones(p.cache.shape[:2], dtype=torch.bool)
    for b in range(p.B):
        pos = torch.arange(max(0, min(p.starts[b] + p.lens[b], p.W * p.P)) if p.lens[b] > 0 else 0)
        unseen[p.table[b, pos // p.P].long(), pos % p.P] = False
    return unseen


WIDE = [(140, 4, 16, 512, 64, 16, 24, "end to end"), (140, 4, 16, 256, 32, 16, 24, "end to end"), (16, 33, 16, 512, 64, 16, 40, "parts"), (2, 100, 16, 512, 32, 32, 64, "parts"), (60, 20, 16, 512, 64, 16, 20, "end to end"),
        (60, 20, 16, 512, 32, 16, 20, "end to end"), (16, 128, 16, 512, 64, 16, 12, "alone"), (16, 128, 16, 512, 32, 16, 12, "alone"),
        (10, 40, 16, 256, 32, 16, 40, "parts"), (60, 20, 16, 256, 64, 16, 24, "end to end"), (8, 128, 16, 256, 64, 16, 16, "alone"),
        (20, 40, 16, 128, 32, 16, 40, "parts"), (110, 20, 16, 128, 32, 16, 36, "end to end"), (16, 128, 16, 128, 64, 16, 16, "alone")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B,L,R,C,DR,P,W,way", WIDE)
def test_workgroups_of_64_rows(gpu, dtype, B, L, R, C, DR, P, W, way):
    # (and of 32 where two of them are a sequence's) each way to share keys out and none, ragged lengths, scores that rise and fall from page to page
    p = Problem(B, L, R, C, DR, P, W, dtype, seed=B + C)
    most = P * W - L
    p.starts = [most if b % 4 == 0 else (most * (b * 37 % 101)) // 100 for b in range(B)]
    p.lens = [L if b % 3 else max(1, L // 2 + 1) for b in range(B)]
    if B > 8:
        p.starts[5], p.lens[6] = -L, 0                             # a sequence that sees nothing, and one without tokens
    p.cache = (p.cache.float() * (0.05 + 2.0 * (torch.arange(p.cache.shape[0]) * 7 % 13) / 13)[:, None, None]).to(dtype)
    plan = capi.latent_attention_plan(B, L, R, C, DR, P, W)
    assert plan["rows"] == (32 if L == 4 else 64) and plan["shared"] == (way != "alone")
    if way != "alone":
        assert _end_to_end(p) == (way == "end to end")
    clean = _compare(gpu, p)
    _compare(gpu, p, causal=False)
    again = _compare(gpu, p)
    assert torch.equal(again[0], clean[0]) and torch.equal(again[1], clean[1])
    # what nobody sees may be anything, and what some rows see reaches no others
    unseen = _unseen(p)
    bad = p.cache.clone()
    bad[unseen] = torch.tensor([math.nan, math.inf, -math.inf], dtype=dtype)[torch.arange(int(unseen.sum())) % 3][:, None]
    t = p.on(gpu)
    for b, i, channel, value in ((0, L // 3, None, None), (0, L // 3, 5, math.nan), (1, L // 2, C - 1, math.inf), (0, L // 2, C + 1, math.nan)):
        cache = bad.clone()
        pos = p.starts[b] + i
        if channel is not None:
            cache[p.table[b, pos // P], pos % P, channel] = value
        t["latent_cache"] = cache.to(gpu)
        out, lse = _module().latent_attention(p.q.to(gpu), p.r.to(gpu), scale=p.scale, return_lse=True, **t)
        sees = torch.zeros(B, L, dtype=torch.bool)
        if channel is not None:
            sees[b, i:p.lens[b]] = True
            assert sees.any()
        assert torch.equal(out.cpu()[~sees], clean[0].cpu()[~sees])
        assert torch.equal(lse.cpu().transpose(1, 2)[~sees], clean[1].cpu().transpose(1, 2)[~sees])
        if channel is not None and channel < C:
            assert not torch.isfinite(out.cpu()[sees][..., channel]).any()
        elif channel is not None:
            assert torch.isnan(out.cpu()[sees]).all()


@pytest.mark.gpu
def test_views_and_tables_with_rows_apart(gpu):
    p = Problem(3, 2, 6, 256, 32, 32, 7, F16, seed=11)
    p.starts = [200, 31, 3]
    want = _compare(gpu, p)
    q = p.q.to(gpu).transpose(1, 2).contiguous().transpose(1, 2)   # [B, R, L, C] tensors
    wide = torch.randn(3, 2, 6, 96 + 32, generator=p.gen).to(F16).to(gpu)
    wide[..., 96:] = p.r.to(gpu)
    table = torch.full((3, 11), -5, dtype=I32, device=gpu)
    table[:, :7] = p.table.to(gpu)
    got = _compare(gpu, p, q=q, r=wide[..., 96:], table=table[:, :7])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # heads and tokens that are one and the same
    p.q, p.r = p.q[:, :1, :1].expand(3, 2, 6, 256), p.r[:, :1, :1].expand(3, 2, 6, 32)
    _compare(gpu, p, q=p.q[:, :1, :1].contiguous().to(gpu).expand(3, 2, 6, 256), r=p.r[:, :1, :1].contiguous().to(gpu).expand(3, 2, 6, 32))


@pytest.mark.gpu
def test_pages_beyond_32_bits_of_bytes(gpu):
    m = _module()
    N, P, C, DR = 32000, 128, 512, 64                              # 4.7 GB
    cache = torch.zeros(N, P, C + DR, dtype=BF16, device=gpu)
    p = Problem(1, 1, 16, C, DR, P, 4, BF16, seed=12)
    p.starts = [4 * P - 1]
    want = p.on(gpu)
    out = m.latent_attention(p.q.to(gpu), p.r.to(gpu), scale=p.scale, **want)
    pages = [31999, 30000, 3, 29999]
    for w, page in enumerate(pages):
        cache[page] = p.cache[p.table[0, w]].to(gpu)
    t = {**want, "latent_cache": cache, "page_table": torch.tensor([pages], dtype=I32, device=gpu)}
    assert torch.equal(m.latent_attention(p.q.to(gpu), p.r.to(gpu), scale=p.scale, **t), out)
    x = p.normal(1, 1, C + DR).to(gpu)
    m.latent_append(x[..., :C], x[..., C:], cache, t["page_table"], t["starts"])
    assert torch.equal(cache[29999, P - 1], x[0, 0])


# ---- on the GPU: the expanded form ----

def _expanded(gpu, B, L, K, R, D, DR, dtype, seed, starts=None, lens=None, causal=True, m=None, kv=None, q=None, kr=None, packed=True):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g).to(dtype)
    q = normal(B, L, R, D + DR) if q is None else q
    kv = normal(B, K, R, 2 * D) if kv is None else kv              # one product's output
    kr = normal(B, K, DR) if kr is None else kr
    k, v = kv[..., :D], kv[..., D:]
    dq, dkv, dkr = (x.to(gpu) for x in (q, kv, kr))
    kw = {}
    if starts is not None:
        kw["starts"] = torch.tensor(starts, dtype=I32, device=gpu)
    if lens is not None:
        kw["new_lens"] = torch.tensor(lens, dtype=I32, device=gpu)
    got, lse = (m or _module()).expanded_attention(dq, dkv[..., :D], dkr, dkv[..., D:], causal=causal, return_lse=True, **kw)
    assert tuple(got.shape) == (B, L, R, D) and got.dtype == dtype
    return got, lse, (q, k, kr, v, [K - L] * B if starts is None else starts, [L] * B if lens is None else lens, 1 / math.sqrt(D + DR), causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,DR", [(64, 32), (64, 64), (128, 32), (128, 64)])
@pytest.mark.parametrize("B,L,K,R", [(2, 1, 1, 1), (1, 1, 200, 3), (2, 17, 17, 2), (1, 130, 130, 2), (2, 100, 333, 2), (1, 300, 1000, 1), (1, 5, 3000, 2), (3, 65, 64 + 65, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_expanded_attention_is_the_oracles(gpu, dtype, D, DR, B, L, K, R, causal):
    for m in (_module(), capi):
        got, lse, args = _expanded(gpu, B, L, K, R, D, DR, dtype, seed=L + K, causal=causal, m=m)
        _check(got, lse, lo.expanded(*args), D + DR, K, dtype, args[3].abs().max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("D,DR", [(64, 32), (128, 64)])
@pytest.mark.parametrize("L,K", [(40, 40), (40, 700), (300, 290)])
def test_expanded_padded_batches_and_odd_lengths(gpu, D, DR, L, K):
    starts = [0, K - L, K + 5, -L, -3, K - 1, 7, 0]
    lens = [L, L // 2, L, L, L, L + 9, 0, -1]
    for causal in (True, False):
        got, lse, args = _expanded(gpu, 8, L, K, 2, D, DR, F16, seed=K, starts=starts, lens=lens, causal=causal)
        _check(got, lse, lo.expanded(*args), D + DR, K, F16, args[3].abs().max().item())
    assert (got[3] == 0).all() and (lse[6] == -math.inf).all() and (got[1, L // 2:] == 0).all()


@pytest.mark.gpu
def test_expanded_attention_of_long_prompts(gpu):
    # 256 rows a workgroup, whole chip; a sample of heads against the oracle
    B, L, K, R, D, DR = 1, 2100, 4200, 40, 128, 64
    got, lse, (q, k, kr, v, starts, lens, scale, causal) = _expanded(gpu, B, L, K, R, D, DR, BF16, seed=4)
    assert capi.expanded_attention_plan(B, L, R, K, D, DR)["rows"] == 256
    for h in (0, 39):
        want = lo.expanded(q[:, :, h:h + 1], k[:, :, h:h + 1], kr, v[:, :, h:h + 1], starts, lens, scale, causal)
        _check(got[:, :, h:h + 1], lse[:, h:h + 1], want, D + DR, K, BF16, v.abs().max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("DR", [32, 64])
def test_expanded_attention_of_many_narrow_heads(gpu, dtype, DR):
    # more than two workgroups of 128 rows for every compute unit; a sample of heads against the oracle
    B, L, K, R, D = 3, 700, 731, 36, 64
    starts, lens = [31, 0, -5], [700, 411, 700]
    plan = capi.expanded_attention_plan(B, L, R, K, D, DR)
    assert plan["rows"] == 128 and plan["workgroups"] > 512
    for causal in (True, False):
        got, lse, (q, k, kr, v, _, _, scale, _) = _expanded(gpu, B, L, K, R, D, DR, dtype, seed=DR, starts=starts, lens=lens, causal=causal)
        for h in (0, 17, 35):
            want = lo.expanded(q[:, :, h:h + 1], k[:, :, h:h + 1], kr, v[:, :, h:h + 1], starts, lens, scale, causal)
            _check(got[:, :, h:h + 1], lse[:, h:h + 1], want, D + DR, K, dtype, v.abs().max().item())
    # what only some rows see, and nobody
    kv = torch.cat([k, v], -1)
    bad, bad_r = kv.clone(), kr.clone()
    bad[1, 411:], bad_r[1, 411:] = math.nan, math.inf
    bad[0, 500, 4, D + 7] = math.inf
    clean = _expanded(gpu, B, L, K, R, D, DR, dtype, seed=DR, starts=starts, lens=lens, kv=kv, kr=kr, q=q)[0].cpu()
    got = _expanded(gpu, B, L, K, R, D, DR, dtype, seed=DR, starts=starts, lens=lens, kv=bad, kr=bad_r, q=q)[0].cpu()
    hit = torch.zeros(B, L, R, D, dtype=torch.bool)
    hit[0, 500 - 31:, 4, 7] = True
    assert torch.equal(got[~hit], clean[~hit]) and not torch.isfinite(got[hit]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("L,K,D,DR", [(30, 100, 64, 32), (300, 300, 128, 64), (3, 2000, 128, 32)])
def test_expanded_what_is_not_finite_stays_where_it_is_seen(gpu, dtype, L, K, D, DR):
    g = torch.Generator().manual_seed(7)
    kv, kr = torch.randn(2, K, 2, 2 * D, generator=g).to(dtype), torch.randn(2, K, DR, generator=g).to(dtype)
    starts, lens = [K - L - 1, 2], [L, L]
    clean, clean_lse, args = _expanded(gpu, 2, L, K, 2, D, DR, dtype, seed=1, starts=starts, lens=lens, kv=kv, kr=kr)
    _check(clean, clean_lse, lo.expanded(*args), D + DR, K, dtype, kv.abs().max().item())
    bad, bad_r = kv.clone(), kr.clone()
    for b in range(2):                                             # behind what anybody sees
        bad[b, starts[b] + L:] = math.nan
        bad[b, starts[b] + L + 1::2] = math.inf
        bad_r[b, starts[b] + L:] = -math.inf
    got, lse, _ = _expanded(gpu, 2, L, K, 2, D, DR, dtype, seed=1, starts=starts, lens=lens, kv=bad, kr=bad_r)
    assert torch.equal(got, clean) and torch.equal(lse, clean_lse)
    for b, i, h, channel, value in ((0, L - 1, 1, D - 1, math.nan), (1, L // 2, 0, 3, math.inf), (0, 0, 0, 0, math.nan)):
        at = (starts[b] + i) % K                                   # (a token before the first key: the last key, which nobody sees)
        one = bad.clone()
        one[b, at, h, D + channel] = value                         # a value: in its channel and head, where it is seen
        got, lse, _ = _expanded(gpu, 2, L, K, 2, D, DR, dtype, seed=1, starts=starts, lens=lens, kv=one, kr=bad_r)
        hit = torch.zeros(2, L, 2, D, dtype=torch.bool)
        hit[b, at - starts[b]:, h, channel] = True
        assert torch.equal(got.cpu()[~hit], clean.cpu()[~hit]) and not torch.isfinite(got.cpu()[hit]).any() and torch.equal(lse, clean_lse)
        one = bad.clone()
        one[b, at, h, channel] = math.nan                          # a key: the rows that see it
        got, lse, _ = _expanded(gpu, 2, L, K, 2, D, DR, dtype, seed=1, starts=starts, lens=lens, kv=one, kr=bad_r)
        hit = torch.zeros(2, L, 2, D, dtype=torch.bool)
        hit[b, at - starts[b]:, h] = True
        assert torch.equal(got.cpu()[~hit], clean.cpu()[~hit]) and torch.isnan(got.cpu()[hit]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,DR", [(64, 32), (64, 64), (128, 32), (128, 64)])
def test_expanded_workgroups_of_256_rows(gpu, dtype, D, DR):
    # two blocks of rows a wave: ragged lengths, row tiles without a token, causal or not; a sample of heads against the oracle
    B, L, K, R = (5, 500, 520, 36) if D == 64 else (3, 520, 820, 40)
    assert capi.expanded_attention_plan(B, L, R, K, D, DR)["rows"] == 256
    starts, lens = [K - L, 0, 11, K - 1, -4][:B], [L, L - 30, 200, L, L][:B]
    heads = (0, 21, R - 1)
    for causal in (False, True):
        got, lse, (q, k, kr, v, _, _, scale, _) = _expanded(gpu, B, L, K, R, D, DR, dtype, seed=D + DR, starts=starts, lens=lens, causal=causal)
        for h in heads:
            want = lo.expanded(q[:, :, h:h + 1], k[:, :, h:h + 1], kr, v[:, :, h:h + 1], starts, lens, scale, causal)
            _check(got[:, :, h:h + 1], lse[:, h:h + 1], want, D + DR, K, dtype, v.abs().max().item())
    got, lse = got.cpu(), lse.cpu()
    # behind what anybody sees, and a value and a key that some rows see
    bad, bad_r = torch.cat([k, v], -1), kr.clone()
    for b in range(B):
        bad[b, starts[b] + lens[b]:], bad_r[b, starts[b] + lens[b]:] = math.nan, -math.inf
        bad[b, starts[b] + lens[b] + 1::2] = math.inf
    for b, i, h, channel in ((None,) * 4, (0, 300, 21, D + 3), (1, L - 31, 0, 2 * D - 1), (2, 7, R - 1, 5)):
        one, hit, all_of = bad.clone(), torch.zeros(B, L, R, D, dtype=torch.bool), torch.zeros(B, R, L, dtype=torch.bool)
        if b is not None:
            one[b, starts[b] + i, h, channel] = math.nan
            hit[b, i:lens[b], h, channel - D if channel >= D else slice(None)] = True
            all_of[b, h, i:lens[b]] = channel < D
        out, sums, _ = _expanded(gpu, B, L, K, R, D, DR, dtype, seed=0, starts=starts, lens=lens, kv=one, kr=bad_r, q=q)
        out, sums = out.cpu(), sums.cpu()
        assert torch.equal(out[~hit], got[~hit]) and torch.isnan(out[hit]).all()
        assert torch.equal(sums[~all_of], lse[~all_of]) and torch.isnan(sums[all_of]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("L,R,K,D,DR,splits", [(300, 2, 8192, 64, 32, 32), (1, 1, 16384, 64, 64, 128), (1, 1, 16384, 128, 64, 128), (1, 4, 16384, 128, 32, 64),
                                                 (1000, 8, 16384, 128, 64, 8), (1000, 8, 16384, 128, 32, 8)])
def test_expanded_keys_in_many_parts(gpu, dtype, L, R, K, D, DR, splits):
    # joined by sixteen waves a row, or parts of 256 rows; parts that no row sees among them; the first and the last head against the oracle
    plan = capi.expanded_attention_plan(1, L, R, K, D, DR)
    assert plan["splits"] == splits and plan["rows"] == (256 if splits == 8 else 128)
    for starts in ([K - L], [K // 3], [-1]):
        got, lse, (q, k, kr, v, _, lens, scale, causal) = _expanded(gpu, 1, L, K, R, D, DR, dtype, seed=splits, starts=starts)
        for h in {0, R - 1}:
            want = lo.expanded(q[:, :, h:h + 1], k[:, :, h:h + 1], kr, v[:, :, h:h + 1], starts, lens, scale, causal)
            _check(got[:, :, h:h + 1], lse[:, h:h + 1], want, D + DR, K, dtype, v.abs().max().item())
        again = _expanded(gpu, 1, L, K, R, D, DR, dtype, seed=splits, starts=starts)
        assert torch.equal(again[0], got) and torch.equal(again[1], lse)


@pytest.mark.gpu
def test_expanded_views(gpu):
    # separate tensors, [B, heads, L, D] tensors, keys that heads share
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(2, n, 3, d, generator=g).to(F16).to(gpu) for n, d in ((50, 96), (70, 64), (70, 64)))
    kr = torch.randn(2, 70, 32, generator=g).to(F16).to(gpu)
    m = _module()
    want = m.expanded_attention(q, k, kr, v)
    turned = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    wide = torch.randn(2, 70, 64, generator=g).to(F16).to(gpu)
    wide[..., 32:] = kr
    assert torch.equal(m.expanded_attention(turned[0], turned[1], wide[..., 32:], turned[2]), want)
    shared = m.expanded_attention(q, k[:, :, :1].expand(-1, -1, 3, -1), kr, v)
    assert torch.equal(shared, m.expanded_attention(q, k[:, :, :1].repeat(1, 1, 3, 1), kr, v))


# ---- on the GPU: together ----

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_an_answer_by_both_forms(gpu, dtype):
    # a prompt in the expanded form, then token by token in the absorbed one, over pages that are taken and forked as they are needed: every
    # token's output is that of the expanded form over the whole text.  The maps of latents to keys and values select channels, so that both forms
    # stand for the same numbers exactly, and each is within its own tolerance of the oracle.
    m = _module()
    B, R, C, DR, D, P, W, L0, steps = 2, 4, 128, 32, 64, 16, 8, 37, 21
    g = torch.Generator().manual_seed(21)
    normal = lambda *shape: torch.randn(*shape, generator=g).to(dtype)
    n = L0 + steps
    text_c, text_k, text_q = normal(B, n, C), normal(B, n, DR), normal(B, n, R, D + DR)
    pick_k = [torch.randperm(C, generator=g)[:D] for _ in range(R)]
    pick_v = [torch.randperm(C, generator=g)[:D] for _ in range(R)]
    cos, sin = m.rotary_tables(W * P, DR, gpu, scaling="linear", factor=2.0)
    S = B + 1                                                      # one more row, for a fork
    cache = torch.full((S * W, P, C + DR), math.nan, dtype=dtype, device=gpu)
    table, starts = torch.full((S, W), -1, dtype=I32, device=gpu), torch.zeros(S, dtype=I32, device=gpu)
    uses = torch.zeros(S * W, dtype=I32, device=gpu)
    scale = 1 / math.sqrt(D + DR)

    def padded(x, L):
        return torch.cat([x, torch.zeros(S - B, *x.shape[1:], dtype=dtype)]).to(gpu)[:, :L].contiguous()

    def step(first, L, lens):
        c, k, q = (padded(x[:, first:first + L], L) for x in (text_c, text_k, text_q))
        lens = torch.tensor(lens, dtype=I32, device=gpu)
        assert m.take_pages(table, starts, uses, P, L, lens).sum() == 0
        r = m.latent_append(c, k, cache, table, starts, new_lens=lens, queries=q[..., D:], rope_cos=cos, rope_sin=sin)
        absorbed = torch.zeros(S, L, R, C, dtype=dtype, device=gpu)
        for h in range(R):
            absorbed[:, :, h].index_copy_(2, pick_k[h].to(gpu), q[:, :, h, :D].contiguous())
        out = m.latent_attention(absorbed, r, cache, table, starts, scale, new_lens=lens)
        out = torch.stack([out[:, :, h][..., pick_v[h].to(gpu)] for h in range(R)], dim=2)
        starts.add_(lens)
        return out[:B].cpu(), r[:B]

    outs, queries = [], []
    lens = [L0] * B + [0]
    out, r = step(0, L0, lens)
    outs.append(out), queries.append(r.cpu())
    for i in range(steps):
        if i == 5:                                                 # sequence 1 goes on as a fork, whose parent ends
            assert m.fork_pages([cache], table, starts, uses, P, torch.tensor([1], dtype=I32, device=gpu), torch.tensor([2], dtype=I32, device=gpu)).tolist() == [1]
            m.free_pages(table, starts, uses, torch.tensor([1], dtype=I32, device=gpu))
            m.compact_pages([cache], table, uses)
            assert m.fork_pages([cache], table, starts, uses, P, torch.tensor([2], dtype=I32, device=gpu), torch.tensor([1], dtype=I32, device=gpu)).tolist() == [1]
            m.free_pages(table, starts, uses, torch.tensor([2], dtype=I32, device=gpu))
        out, r = step(L0 + i, 1, [1] * B + [0])
        outs.append(out), queries.append(r.cpu())
    got, rotated = torch.cat(outs, 1), torch.cat(queries, 1)
    keys_r = m.rotate(text_k.to(gpu), cos, sin, DR)                # the rotary keys of the whole text, as appended
    k = torch.stack([text_c[..., pick_k[h]] for h in range(R)], 2)
    v = torch.stack([text_c[..., pick_v[h]] for h in range(R)], 2)
    q = torch.cat([text_q[..., :D], rotated], -1)
    whole = m.expanded_attention(q.to(gpu), k.to(gpu), keys_r, v.to(gpu)).cpu()
    want = lo.expanded(q, k, keys_r.cpu(), v, [0] * B, [n] * B, scale)
    _check(whole, None, want, D + DR, n, dtype, v.abs().max().item())
    _check(got, None, want, C + DR, n, dtype, text_c.abs().max().item())


@pytest.mark.gpu
def test_steps_captured_in_graphs(gpu):
    # append and attend in one graph, and the expanded form beside it, and a second graph of the same: replayed in turn with eager work between
    m = _module()
    p = Problem(3, 1, 40, 512, 64, 16, 60, BF16, seed=16)
    p.starts = [700, 123, 0]
    cos, sin = m.rotary_tables(960, 64, gpu)
    scale = p.scale

    def step(t, x, qr, q, kv):
        r = m.latent_append(x[..., :512], x[..., 512:], queries=qr, rope_cos=cos, rope_sin=sin, interleaved=True, **t)
        e = torch.cat([q[..., :128], r], -1)
        return (r, *m.latent_attention(q, r, scale=scale, return_lse=True, **t), m.expanded_attention(e, kv[..., :128], x[..., 512:].expand(3, 70, 64), kv[..., 128:]))

    runs = []
    for _ in range(2):
        t = p.on(gpu)
        x = [p.normal(3, 1, 576).to(gpu), p.normal(3, 1, 40, 64).to(gpu), p.q.to(gpu), p.normal(3, 70, 40, 256).to(gpu)]
        warm = {name: value.clone() for name, value in t.items()}
        side = torch.cuda.Stream(device=gpu)
        side.wait_stream(torch.cuda.current_stream(gpu))
        with torch.cuda.stream(side):
            step(warm, *x)
        torch.cuda.current_stream(gpu).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(t, *x)
        runs.append((graph, t, x, out, p.on(gpu)))
    for _ in range(4):
        for graph, t, x, out, eager in runs:
            for y in x:
                y.copy_(torch.randn(y.shape, generator=p.gen).to(y.dtype))
            graph.replay()
            want = step(eager, *x)
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            assert torch.equal(t["latent_cache"], eager["latent_cache"])
            t["starts"] += 1
            eager["starts"] += 1


@pytest.mark.gpu
def test_steps_on_two_streams(gpu):
    m = _module()
    problems = [Problem(2, 3, R, 512, 64, 16, 200, F16, seed=s) for s, R in ((17, 16), (18, 40))]
    alone, tensors, streams = [], [], []
    for p in problems:
        p.starts = [3000, 2500]
        tensors.append((p.on(gpu), p.q.to(gpu), p.r.to(gpu)))
        t, q, r = tensors[-1]
        alone.append(m.latent_attention(q, r, scale=p.scale, return_lse=True, **t))
        streams.append(torch.cuda.Stream(device=gpu))
    torch.cuda.synchronize()
    for _ in range(3):
        got = [None, None]
        for n in range(2):
            with torch.cuda.stream(streams[n]):
                t, q, r = tensors[n]
                got[n] = m.latent_attention(q, r, scale=problems[n].scale, return_lse=True, **t)
        torch.cuda.synchronize()
        for n in range(2):
            assert all(torch.equal(a, b) for a, b in zip(alone[n], got[n]))
