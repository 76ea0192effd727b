"""The paged 8-bit key/value cache: its oracle and its refusals on the CPU, and on the GPU the three operators against the
oracle in 64 bits and against each other.

Codes, exponents, bounds, rotated queries and selections are compared for equality: their definitions leave nothing open.

Tolerance of the attention, from its roundings.  With u half a step of the element type (fp16 2^-11, bf16 2^-8), n the
keys of a row, A = sum p |v| / sum p, and d = (H + 8) 2^-24 max_j scale sum |q k_j| + |s| 2^-22 what a float32 score may be off
by (products of 16-bit numbers and codes are exact, H of them are summed; the factors and the exponential's argument):
  each weight is rounded once to the element type and off by e^d, the exponential itself by 2^-22:   A (u + 2 d + 2^-21)
  sums of n terms, joined over waves and splits, in float32:                                       A 2 (n + 64) 2^-24
  values below the reach of fp16 next to the largest power of two of the row's pages E:             2^(E - 25), fp16 only
  weights below it, 2^-24 of the reference's 2^7, n of them:                                        n 2^-32 448 2^E, fp16 only
  the result is rounded once:                                                                       u |out| + 2^-25 (fp16)
"""
import ctypes
import math
import random

import numpy as np
import pytest
import torch

from fused_attention_amd import capi
from oracle import attention as full_attention
from oracle import paged_cache as pc
from oracle import rope_tables

E4M3 = torch.float8_e4m3fn


class Problem:
    """Tensors of a cache and a call, on the CPU."""

    def __init__(self, B=2, L=1, R=4, Rkv=2, H=64, P=16, W=4, dtype=torch.float16, seed=0, extra=3, bounds=True, layout="blf"):
        self.B, self.L, self.R, self.Rkv, self.H, self.P, self.W = B, L, R, Rkv, H, P, W
        self.dtype, self.layout = dtype, layout
        self.gen = torch.Generator().manual_seed(seed)
        N = B * W + extra
        self.k_cache = self.codes(N)
        self.v_cache = self.codes(N)
        self.k_exponents = torch.randint(-9, -6, (N, Rkv), generator=self.gen).to(torch.int8)
        self.v_exponents = torch.randint(-9, -6, (N, Rkv), generator=self.gen).to(torch.int8)
        self.key_bounds = None
        if bounds:
            y = self.k_cache.float()
            self.key_bounds = torch.stack([(y.amax(2) / 4).ceil(), (y.amin(2) / 4).floor()], 2).to(torch.int8)
        self.page_table = torch.randperm(N, generator=self.gen)[:B * W].to(torch.int32).view(B, W)
        self.starts = [0] * B
        self.lens = [L] * B
        self.q, self.k, self.v = (self.normal(B, L, heads, H) for heads in (R, Rkv, Rkv))

    def codes(self, N):
        return (100 * torch.randn(N, self.Rkv, self.P, self.H, generator=self.gen)).clamp(-448, 448).to(E4M3)

    def normal(self, *shape, std=1.0):
        return (std * torch.randn(*shape, generator=self.gen)).to(self.dtype)

    def cache(self):
        return pc.Cache(self.k_cache, self.v_cache, self.k_exponents, self.v_exponents, self.page_table, self.key_bounds)

    def laid_out(self, x):
        """[B, L, heads, H] as a caller has it."""
        return x.flatten(2) if self.layout == "blf" else x.transpose(1, 2).contiguous()

    def by_token(self, x, heads):
        x = x.cpu()
        return x.view(self.B, self.L, heads, self.H) if self.layout == "blf" else x.transpose(1, 2)

    def on(self, dev):
        """The cache's tensors on the GPU, as keyword arguments by name."""
        t = {name: getattr(self, name).to(dev) for name in ("k_cache", "v_cache", "k_exponents", "v_exponents", "page_table")}
        t["starts"] = torch.tensor(self.starts, dtype=torch.int32, device=dev)
        t["new_lens"] = torch.tensor(self.lens, dtype=torch.int32, device=dev)
        if self.key_bounds is not None:
            t["key_bounds"] = self.key_bounds.to(dev)
        return t


def _only(t, *names):
    return {name: t[name] for name in names if name in t}


CACHE = ("k_cache", "v_cache", "k_exponents", "v_exponents", "page_table", "starts", "new_lens")


def _equal_codes(got, want):
    """The same values, NaN where there is NaN."""
    got, want = got.cpu().float().double().numpy(), np.asarray(want, dtype=np.float64)
    np.testing.assert_array_equal(got, want)


def _check_appended(t, cache):
    for name in ("k", "v"):
        np.testing.assert_array_equal(t[name + "_exponents"].cpu().numpy(), cache.exponents[name])
        _equal_codes(t[name + "_cache"], cache.codes[name])
    if cache.bounds is not None:
        np.testing.assert_array_equal(t["key_bounds"].cpu().numpy(), cache.bounds)


def _check_attention(p, got, lse, want, most_exponent=None):
    """got [B, L, R, H]; want: what the oracle's attention returns."""
    out, want_lse, spread, size = want
    u = 2.0 ** -11 if p.dtype == torch.float16 else 2.0 ** -8
    n = p.W * p.P
    seen = (want_lse != -math.inf).transpose(1, 2)[..., None]
    s = torch.where(torch.isfinite(want_lse), want_lse, 0.0).abs().transpose(1, 2) + math.log(max(n, 2))
    d = (p.H + 8) * 2.0 ** -24 * size + s * 2.0 ** -22
    tol = spread * (u + 2 * d[..., None] + 2.0 ** -21 + 2 * (n + 64) * 2.0 ** -24) + u * out.abs() + 2.0 ** -133
    if p.dtype == torch.float16:
        E = int(p.v_exponents.max()) if most_exponent is None else most_exponent
        tol = tol + 2.0 ** (E - 25) + n * 2.0 ** -32 * 448 * 2.0 ** E + 2.0 ** -25
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    excess = torch.where(torch.isnan(out), 0.0, (got - out).abs() - tol)
    assert excess.max().item() <= 0, "max excess %.3e" % excess.max().item()
    assert torch.equal(got[~seen.expand_as(got)], torch.zeros_like(got[~seen.expand_as(got)]))   # rows that see nothing
    if lse is not None:
        assert lse.dtype == torch.float32
        lse = lse.cpu().double()
        at = torch.isfinite(want_lse)
        assert torch.equal(at, torch.isfinite(lse)) and torch.equal(lse[~at & ~torch.isnan(want_lse)], want_lse[~at & ~torch.isnan(want_lse)])
        off = (lse - want_lse)[at].abs() - (d.transpose(1, 2)[at] + 2.0 ** -20 + want_lse[at].abs() * 2.0 ** -22 + (n + 64) * 2.0 ** -24)
        assert off.numel() == 0 or off.max().item() <= 0


# ---- the oracle, on the CPU ----

def test_e4m3_of_the_oracle_is_torchs():
    codes = torch.arange(256, dtype=torch.uint8).view(E4M3).float().double()
    codes = codes[torch.isfinite(codes)].unique()
    x = torch.cat([codes, (codes[1:] + codes[:-1]) / 2, codes * 1.01, torch.tensor([1e-9, -1e-9, 2.0 ** -10, 3 * 2.0 ** -10])])
    x = x[x.abs() <= 448]
    np.testing.assert_array_equal(pc.e4m3(x.numpy()), x.float().to(E4M3).float().double().numpy())


def test_exponents_of_the_oracle_are_the_smallest():
    for e in list(range(-79, 120)):
        for amax, want in ((448.0 * 2.0 ** e, e), (448.0 * 2.0 ** e * (1 + 2.0 ** -20), e + 1), (448.0 * 2.0 ** e * (1 - 2.0 ** -20), e)):
            assert pc.exponent_of(amax) == want
    assert pc.exponent_of(0.0) == pc.LEAST_EXPONENT == pc.exponent_of(1e-30)


def test_appended_values_come_back_and_parts_give_the_whole():
    p = Problem(B=1, L=37, P=16, W=3, seed=3)
    whole, parts = p.cache(), p.cache()
    pc.append(whole, p.k, p.v, [5], [37])
    for first, n in ((0, 1), (1, 7), (8, 20), (28, 9)):
        pc.append(parts, p.k[:, first:first + n], p.v[:, first:first + n], [5 + first], [n])
    np.testing.assert_array_equal(whole.bounds, parts.bounds)
    for name, x in (("k", p.k), ("v", p.v)):
        np.testing.assert_array_equal(whole.exponents[name], parts.exponents[name])
        for i in range(37):
            page = whole.page(0, (5 + i) // 16)
            got = whole.codes[name][page, :, (5 + i) % 16] * 2.0 ** whole.exponents[name][page][:, None]
            y = x[0, i].double().numpy()
            step = 2.0 ** (whole.exponents[name][page][:, None] - 9.0)
            assert (np.abs(got - y) <= np.maximum(np.abs(y) * 2.0 ** -4, step / 2)).all()


def test_attention_of_the_oracle_is_the_full_one():
    p = Problem(B=2, L=5, R=4, Rkv=2, H=32, P=16, W=2, seed=4)
    p.starts = [20, 27]
    cache = p.cache()
    out, lse, _, _ = pc.attention(cache, p.q, p.starts, p.lens)
    for b in range(2):
        n = p.starts[b] + 5
        keys, values = (np.concatenate([cache.codes[name][cache.page(b, w)] * 2.0 ** cache.exponents[name][cache.page(b, w)][:, None, None]
                                        for w in range(2)], axis=1) for name in ("k", "v"))        # [Rkv, 32, H]
        keys, values = (torch.from_numpy(x).repeat_interleave(2, dim=0).transpose(0, 1).reshape(1, 32, 4 * 32)[:, :n] for x in (keys, values))
        q = torch.zeros(1, n, 4 * 32)
        q[0, p.starts[b]:] = p.q[b].flatten(1)
        want = full_attention(q, keys, values, 32, mask=torch.full((n, n), -math.inf).triu(1)[None])
        assert (want[0, p.starts[b]:].double() - out[b].flatten(1)).abs().max() < 1e-5


def test_selection_of_the_oracle_bounds_the_scores():
    p = Problem(B=1, L=1, R=4, Rkv=2, H=32, P=16, W=6, seed=5)
    p.starts = [6 * 16 - 1]
    cache = p.cache()
    picked = pc.select(cache, p.q, p.starts, p.lens, 3)[0, 0]
    for head in range(2):
        x = p.q[0, 0, 2 * head:2 * head + 2].double().numpy()
        step = 2.0 ** math.ceil(math.log2(np.abs(x).max() / 127))
        best = []
        for w in range(6):
            page = cache.page(0, w)
            exact = (cache.values("k", page, head) @ x.T).max()
            up, down = cache.bounds[page, head] * 4.0 * 2.0 ** cache.exponents["k"][page, head]
            bound = (np.maximum(x, 0) @ up + np.minimum(x, 0) @ down).max()
            assert exact <= bound
            best.append(bound)
        others = sorted(set(range(5)) - set(picked[head].tolist()))
        slack = step / 2 * 448 * 2.0 ** -6 * 32                    # the rounding of q, times the largest key, in each channel
        assert 5 in picked[head] and all(best[w] <= best[o] + 2 * slack for w in others for o in picked[head].tolist())
    assert pc.select(cache, p.q, [0], p.lens, 3)[0, 0].tolist() == [[0, -1, -1]] * 2
    assert pc.select(cache, p.q, p.starts, [0], 3)[0, 0].tolist() == [[-1] * 3] * 2
    # equal scores: the lowest places
    cache.bounds[:], cache.exponents["k"][:] = 1, 0
    assert pc.select(cache, p.q, p.starts, p.lens, 3)[0, 0].tolist() == [[0, 1, 5]] * 2


@pytest.mark.parametrize("H,P,n", [(32, 16, 96), (64, 64, 150), (16, 128, 128)])
def test_scores_bound_the_keys_as_appended(H, P, n):
    # The bounds that appending makes are of the keys before their rounding to e4m3: what was appended lies within, in every channel, and
    # scores no more with the rounded query than its page.  The codes may lie outside: 433 becomes 448 behind a bound of 436.  By their
    # rounding alone: half a step, 2^-4 of a normal number or 2^-10, and where exponents grew afterwards up to 2^-10 once more.
    p = Problem(B=1, L=n, R=4, Rkv=2, H=H, P=P, W=-(-n // P), seed=31)
    p.k *= torch.linspace(-2, 3, n).exp2()[:, None, None].half()   # exponents grow within pages
    p.k[0, 3, 0, 2] = 433.0
    cache = p.cache()
    first = 0
    for part in (1, 2, 40, n):                                     # in parts
        part = min(part, n - first)
        pc.append(cache, p.k[:, first:first + part], p.v[:, first:first + part], [first], [part])
        first += part
    assert first == n
    outside = 0
    for w in range(p.W):
        page, here = cache.page(0, w), p.k[0, w * P:(w + 1) * P].double().numpy()
        for head in range(2):
            e = cache.exponents["k"][page, head]
            keys = here[:, head] * 2.0 ** -e
            codes = cache.codes["k"][page, head, :len(keys)]
            up, down = cache.bounds[page, head] * 4.0
            assert (keys <= up).all() and (keys >= down).all() and (keys.max(0) > up - 4).all() and (keys.min(0) < down + 4).all()
            slack = np.abs(keys).max(0) * 2.0 ** -4 + 2.0 ** -9
            assert (codes <= up + slack).all() and (codes >= down - slack).all()
            outside += (codes > up).sum() + (codes < down).sum()
            x = p.q[0, 0, 2 * head:2 * head + 2].double().numpy()
            q8 = np.rint(x * 2.0 ** -math.ceil(math.log2(np.abs(x).max() / 127)))
            score = (np.maximum(q8, 0) @ up + np.minimum(q8, 0) @ down).max()
            assert (keys @ q8.T).max() <= score and (codes @ q8.T).max() <= score + (np.abs(q8) @ slack).max()
    at = cache.page(0, 0)
    assert cache.exponents["k"][at, 0] == 0 and cache.codes["k"][at, 0, 3, 2] == 448 and cache.bounds[at, 0, 0, 2] * 4 == 436
    assert outside > 1


# ---- refusals, on the CPU ----

def test_the_library_refuses_what_its_header_says():
    lib = capi.load_library()
    ok = 0x1000                                                    # never dereferenced: every case is refused before a launch
    good = dict(keys=ok, values=ok, key_exponents=ok, value_exponents=ok, key_bounds=ok, page_table=ok, pages=10, heads=2, page_size=64,
                head_dim=64, sequences=3, table_width=4, table_stride=4)

    def cache(**kw):
        return ctypes.byref(capi.Cache(**{**good, **kw}))

    def append(c=None, k=ok, v=ok, kv=(512, 64, 128), q=ok, qs=(512, 64, 256), out=ok, os=(512, 64, 256), starts=ok, lens=None, L=2, R=4,
               cos=None, sin=None, rows=0, flags=0):
        return lib.fa_cache_append(cache() if c is None else c, k, v, *kv, q, *qs, out, *os, starts, lens, L, R, cos, sin, rows, flags, None)

    def attend(c=None, q=ok, qs=(512, 64, 256), out=ok, os=(512, 64, 256), lse=None, sel=None, count=0, starts=ok, lens=None, L=2, R=4,
               scale=0.125, flags=0, ws=None, n=0):
        return lib.fa_cached_attention(cache() if c is None else c, q, *qs, out, *os, lse, sel, count, starts, lens, L, R, scale, flags, ws, n,
                                       None)

    def select(c=None, q=ok, qs=(512, 64, 256), sel=ok, count=2, starts=ok, lens=None, L=2, R=4, flags=0):
        return lib.fa_select_pages(cache() if c is None else c, q, *qs, sel, count, starts, lens, L, R, flags, None)

    for call in (append, attend, select):
        assert call(c=cache(head_dim=48)) == -2 and call(c=cache(head_dim=256)) == -2
        assert [call(c=cache(page_size=n)) for n in (0, 8, 48, 256, -64)] == [-9] * 5
        for name in ("pages", "heads", "sequences", "table_width"):
            assert call(c=cache(**{name: 0})) == -3, name
        assert call(L=0) == -3
        assert call(c=cache(table_stride=3)) == -4
        assert call(c=cache(key_exponents=None)) == -1 and call(c=cache(page_table=None)) == -1 and call(starts=None) == -1
        assert call(c=cache(page_table=ok + 2)) == -5 and call(starts=ok + 1) == -5 and call(lens=ok + 2) == -5
        assert call(c=cache(key_bounds=ok + 8)) == -5
        assert call(c=cache(pages=2 ** 31)) == -6 and call(c=cache(pages=2 ** 28, page_size=128)) == -6
        assert call(c=cache(table_width=2 ** 27, table_stride=2 ** 27)) == -6 and call(L=2 ** 31) == -6 and call(c=cache(sequences=2 ** 29)) == -6
        assert call(flags=8) == -7
        assert call(q=None) == -1
        assert call(qs=(512, 64, 56)) == -4 and call(qs=(512, 60, 256)) == -4 and call(qs=(-512, 64, 256)) == -4
        assert call(q=ok + 2) == -5
        assert call(qs=(2 ** 62, 64, 256)) == -6
        assert call(R=3) == -3 and call(R=0) == -3
    assert lib.fa_cache_append(None, ok, ok, 512, 64, 128, None, 0, 0, 0, None, 0, 0, 0, ok, None, 2, 4, None, None, 0, 0, None) == -1
    for call in (append, attend):
        for name in ("keys", "values", "value_exponents"):
            assert call(c=cache(**{name: None})) == -1, name
        assert call(c=cache(keys=ok + 8)) == -5 and call(c=cache(values=ok + 4)) == -5
        assert call(out=None) == -1 and call(os=(512, 64, 8)) == -4 and call(out=ok + 8) == -5
        assert call(os=(0, 64, 256)) == -4 and call(os=(512, 0, 256)) == -4        # rows in one place
    assert append(k=None) == -1 and append(v=ok + 8) == -5 and append(kv=(512, 64, 60)) == -4
    assert append(q=None, out=ok) == -1
    assert append(cos=ok) == -1 and append(cos=ok, sin=ok, rows=0) == -3 and append(cos=ok + 4, sin=ok, rows=9) == -5
    assert append(flags=1) == -7 and select(flags=1) == -7
    assert [attend(scale=s) for s in (0.0, -1.0, math.inf, math.nan)] == [-8] * 4
    assert attend(sel=ok, count=0) == -3 and attend(sel=ok, count=4097) == -6 and attend(sel=ok + 2, count=2) == -5 and attend(lse=ok + 2) == -5
    assert select(sel=None) == -1 and select(c=cache(key_bounds=None)) == -1 and select(count=0) == -3 and select(count=4097) == -6
    assert select(c=cache(table_width=32769, table_stride=32769, page_size=16)) == -6
    # a long cache and few rows: the keys are split, and the sums need room
    long = dict(table_width=4096, table_stride=4096, sequences=1)
    need = lib.fa_cached_attention_workspace(cache(**long), 1, 4, 0)
    assert need > 0 and need % 4 == 0
    assert attend(c=cache(**long), L=1) == -10 and attend(c=cache(**long), L=1, ws=ok, n=need - 1) == -10
    assert attend(c=cache(**long), L=1, ws=ok + 4, n=need) == -5
    assert lib.fa_cached_attention_workspace(cache(head_dim=3), 1, 4, 0) == -2 and lib.fa_cached_attention_workspace(cache(), 1, 4, 5000) == -6
    plan = (ctypes.c_int * 5)()
    assert lib.fa_cached_attention_plan(cache(), 1, 4, 0, None) == -1 and lib.fa_select_pages_plan(cache(), 1, 4, None) == -1
    assert lib.fa_cached_attention_plan(cache(page_size=3), 1, 4, 0, plan) == -9 and lib.fa_cached_attention_plan(cache(), 1, 4, -1, plan) == -3
    assert lib.fa_cached_attention_plan(cache(), 1, 4, 5000, plan) == -6 and lib.fa_select_pages_plan(cache(heads=3), 1, 4, plan) == -3
    assert lib.fa_select_pages_plan(cache(table_width=32769, table_stride=32769, page_size=16), 1, 4, plan) == -6
    assert "page_size" in capi.strerror(-9) and "workspace" in capi.strerror(-10)


def test_scales_beyond_float32_in_units_of_log2_are_refused():
    # the kernels' exponentials are of base 2: scale * log2(e) would be infinite, and a score of zero times it NaN
    lib = capi.load_library()
    ok = 0x1000                                                    # never dereferenced: without a workspace, nothing is launched
    c = capi.Cache(keys=ok, values=ok, key_exponents=ok, value_exponents=ok, page_table=ok, pages=10, heads=2, page_size=64, head_dim=64,
                   sequences=1, table_width=4096, table_stride=4096)

    def attend(scale):
        return lib.fa_cached_attention(ctypes.byref(c), ok, 256, 64, 256, ok, 256, 64, 256, None, None, 0, ok, None, 1, 4, scale, 0, None, 0, None)

    largest = torch.finfo(torch.float32).max
    assert [attend(s) for s in (largest, 2.9e38, largest / math.log2(math.e) * 1.001)] == [-8] * 3
    assert [attend(s) for s in (largest / math.log2(math.e) * 0.999, 1.0, 1e-38)] == [-10] * 3


def test_outputs_whose_rows_overlap_are_refused():
    # by zero strides, by strides that are too small, between any two dimensions; rows that lie apart are not: with nothing else wrong
    # those calls fail later, at the workspace that they lack
    lib = capi.load_library()
    ok = 0x1000                                                    # never dereferenced
    # one long table and few rows: the keys are in parts, which need a workspace
    c = capi.Cache(keys=ok, values=ok, key_exponents=ok, value_exponents=ok, key_bounds=ok, page_table=ok, pages=10, heads=2, page_size=64,
                   head_dim=64, sequences=3, table_width=4096, table_stride=4096)

    def attend(os, L=2, R=4, sequences=3):
        c.sequences = sequences
        return lib.fa_cached_attention(ctypes.byref(c), ok, 512, 64, 256, ok, *os, None, None, 0, ok, None, L, R, 0.125, 0, None, 0, None)

    def append(os, L=2, R=4):
        c.sequences = 3
        # a flag of the rotation that is out of order behind the strides
        return lib.fa_cache_append(ctypes.byref(c), ok, ok, 512, 64, 128, ok, 512, 64, 256, ok, *os, ok, None, L, R, ok, None, 9, 0, None)

    apart = [(512, 64, 256), (512, 128, 64), (64, 384, 192), (4096, 1024, 64), (128, 64 * 12, 64), (64, 64 * 6, 64 * 3), (520, 64, 256),
             (520, 64, 264)]
    overlapping = [(512, 8, 256), (8, 64, 256), (504, 64, 256), (512, 56, 256), (512, 64, 248), (512, 64, 64), (64, 64, 256), (256, 64, 256),
                   (512, 120, 64), (448, 128, 64), (0, 64, 256), (512, 0, 256), (64, 384, 184), (512, 64, 264), (2 ** 60, 2 ** 60, 2 ** 59)]
    for os in apart:
        assert attend(os) == -10 and append(os) == -1, os
    for os in overlapping:
        assert attend(os) == -4 and append(os) == -4, os
    # a dimension of one element places nothing
    assert attend((0, 64, 256), sequences=1) == -10 and attend((8, 64, 256), sequences=1) == -10
    assert attend((256, 64, 64), L=1) == -10 and attend((192, 64, 64), L=1) == -4
    c.heads = 1
    assert attend((128, 0, 64), R=1) == -10 and attend((64, 8, 64), R=1) == -4


def _entries():
    import fused_attn

    return fused_attn


def test_names_and_defaults_of_the_entry_points():
    import re

    m = _entries()

    def names(f):
        return re.findall(r"(\w+): ", f.__doc__.split("->")[0])

    assert names(m.cache_append) == ["keys", "values", "k_cache", "v_cache", "k_exponents", "v_exponents", "page_table", "starts", "new_lens",
                                     "queries", "rope_cos", "rope_sin", "key_bounds", "layout"]
    assert names(m.cached_attention) == ["queries", "k_cache", "v_cache", "k_exponents", "v_exponents", "page_table", "starts", "new_lens",
                                         "pages", "causal", "return_lse", "layout", "scale"]
    assert names(m.select_pages) == ["queries", "key_bounds", "k_exponents", "page_table", "starts", "page_size", "count", "new_lens", "layout"]
    assert "causal: bool = True" in m.cached_attention.__doc__ and "layout: str = 'blf'" in m.select_pages.__doc__


@pytest.mark.parametrize("how", ["module", "capi"])
def test_the_entry_points_refuse_wrong_tensors(how):
    m = _entries() if how == "module" else capi
    errors = RuntimeError if how == "module" else (ValueError, TypeError)
    p = Problem(B=2, L=3, R=4, Rkv=2, H=64, P=16, W=4)
    t = p.on("cpu")
    q, k, v = (p.laid_out(x) for x in (p.q, p.k, p.v))
    pages = torch.zeros(2, 3, 2, 2, dtype=torch.int32)
    calls = {
        "append": lambda **kw: m.cache_append(**{**_only(t, *CACHE, "key_bounds"), "keys": k, "values": v, "queries": q, **kw}),
        "attend": lambda **kw: m.cached_attention(**{**_only(t, *CACHE), "queries": q, "pages": pages, **kw}),
        "select": lambda **kw: m.select_pages(**{**_only(t, "k_exponents", "page_table", "starts", "new_lens", "key_bounds"), "queries": q,
                                                 "page_size": 16, "count": 2, **kw}),
    }

    def refused(match, which=("append", "attend", "select"), **kw):
        for name in which:
            with pytest.raises(errors, match=match):
                calls[name](**kw)

    refused("GPU")                                                 # everything else in order
    refused("k_exponents must be", k_exponents=t["k_exponents"].float())
    refused("k_exponents must be", k_exponents=t["k_exponents"][0])
    refused("page_table must be", page_table=t["page_table"].long())
    refused("page_table must be", page_table=t["page_table"].t())
    refused("starts must", starts=t["starts"].long())
    refused("starts must", starts=t["starts"][:1])
    refused("new_lens must", new_lens=t["new_lens"][:1])
    refused("new_lens must", new_lens=t["new_lens"].float())
    refused("queries must be float16 or bfloat16", queries=q.float())
    refused("takes 4-D", layout="bhld")
    refused("layout must be", layout="lbf")
    refused("features of queries", queries=q[..., :40])
    refused("heads of queries", queries=q[..., :192])
    refused("batch of page_table", queries=q[:1])
    refused("empty dimension", queries=q[:, :0])
    refused("last dimension", queries=q.repeat_interleave(2, dim=2)[..., ::2])
    both = ("append", "attend")
    refused("k_cache must be", both, k_cache=t["k_cache"].float())
    refused("k_cache must", both, k_cache=t["k_cache"][:-1])
    refused("v_cache must", both, v_cache=t["v_cache"][:, :, :, :32])
    refused("v_cache must be", both, v_cache=t["v_cache"].transpose(1, 2).contiguous().transpose(1, 2))
    refused("v_exponents must", both, v_exponents=t["v_exponents"][:-1])
    refused("k_cache must be", both, k_cache=t["k_cache"][0])
    refused("must hold 16, 32, 64 or 128", both, k_cache=t["k_cache"][:, :, :8].contiguous(), v_cache=t["v_cache"][:, :, :8].contiguous())
    refused("must hold 16, 32, 64 or 128", ("select",), page_size=48)
    refused("head_dim must be", both, k_cache=t["k_cache"][..., :48].contiguous(), v_cache=t["v_cache"][..., :48].contiguous())
    refused("key_bounds must", ("append", "select"), key_bounds=t["key_bounds"][:-1])
    refused("key_bounds must", ("append", "select"), key_bounds=t["key_bounds"].float())
    refused("keys must have the key heads", ("append",), keys=q, values=q)
    refused("values must", ("append",), values=v.bfloat16())
    refused("values must", ("append",), values=v[:, :2])
    refused("values must", ("append",), values=torch.cat([v, v], dim=2)[:, :, :128])
    refused("queries must have the", ("append",), queries=q.bfloat16())
    refused("queries must have the seq_len", ("append",), queries=q[:, :2])
    table = torch.zeros(64, 32)
    for bad in (table.double(), torch.zeros(64, 16), torch.zeros(64, 64)[:, ::2]):
        refused("rope", ("append",), **({"rope_cos": table, "rope_sin": bad} if how == "module" else {"rope": (table, bad)}))
    if how == "module":
        refused("go together", ("append",), rope_cos=table)
        refused("one shape", ("append",), rope_cos=table, rope_sin=table[:9])
    else:
        refused("pair", ("append",), rope=table)
        refused("rope sin", ("append",), rope=(table, table[:9]))
        refused("rope cos", ("append",), rope=(table[:0], table[:0]))
        refused("rope cos must be", ("append",), rope=([1.0], table))
        refused("out", both, out=q[:, :2])
        for name, which in (("queries", ("append", "attend", "select")), ("k_cache", both), ("v_cache", both), ("out", both), ("pages", ("attend",)),
                            ("keys", ("append",)), ("values", ("append",)), ("key_bounds", ("append", "select")), ("starts", both)):
            refused(name + " must be a torch.Tensor", which, **{name: [0]})
    refused("pages must be", ("attend",), pages=pages.long())
    refused("pages must be", ("attend",), pages=pages[:, :2])
    refused("pages must be", ("attend",), pages=pages[..., :0])
    refused("count must be", ("select",), count=0)
    refused("count must be", ("select",), count=4097)


# ---- on the GPU ----

def _append(m, p, t, q=True, rope=None, **kw):
    args = {**_only(t, *CACHE, "key_bounds"), "keys": p.laid_out(p.k).to(t["starts"].device), "values": p.laid_out(p.v).to(t["starts"].device),
            "queries": p.laid_out(p.q).to(t["starts"].device) if q else None, "layout": p.layout, **kw}
    if rope is not None:
        cos, sin = (x.to(t["starts"].device) for x in rope)
        args.update({"rope": (cos, sin)} if m is capi else {"rope_cos": cos, "rope_sin": sin})
    return m.cache_append(**args)


def _attend(m, p, t, q=None, **kw):
    q = p.laid_out(p.q).to(t["starts"].device) if q is None else q
    return m.cached_attention(queries=q, layout=p.layout, **{**_only(t, *CACHE), **kw})


def _select(m, p, t, count, q=None, **kw):
    q = p.laid_out(p.q).to(t["starts"].device) if q is None else q
    return m.select_pages(queries=q, page_size=p.P, count=count, layout=p.layout,
                          **{**_only(t, "k_exponents", "page_table", "starts", "new_lens", "key_bounds"), **kw})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,P", [(16, 16), (16, 128), (32, 64), (64, 32), (64, 128), (128, 16), (128, 64), (128, 128)])
@pytest.mark.parametrize("L,layout,rope,bounds", [(1, "blf", True, True), (3, "bhld", False, True), (50, "blf", True, False),
                                                  (150, "bhld", True, True)])
def test_append_is_the_oracles(gpu, dtype, H, P, L, layout, rope, bounds):
    W = max(3, -(-170 // P))
    p = Problem(B=4, L=L, R=6, Rkv=3, H=H, P=P, W=W, dtype=dtype, seed=H + P + L, bounds=bounds, layout=layout)
    # from the first place of a page, from inside one, over a page's end, and nothing new
    p.starts = [P, 5, min(W * P - L, 2 * P - 1), 7]
    p.lens = [L, L - L // 3, L, 0]
    tables = rope_tables(W * P, H) if rope else None
    p.k[1, 0] *= 40                                                # the page's exponent grows over its earlier tokens'
    p.k[2] *= 2.0 ** -9                                            # ... or not
    cache = p.cache()
    pc.append(cache, p.k, p.v, p.starts, p.lens, *(tables or (None, None)))
    want_q = pc.rotated_queries(p.q, p.starts, p.lens, *(tables or (None, None)))
    for m in (_entries(), capi):
        t = p.on(gpu)
        got = _append(m, p, t, rope=tables)
        assert got.dtype == dtype and got.is_contiguous()
        _check_appended(t, cache)
        assert torch.equal(p.by_token(got, p.R), want_q)
        t2 = p.on(gpu)
        assert _append(m, p, t2, q=False, rope=tables) is None
        _check_appended(t2, cache)


@pytest.mark.gpu
@pytest.mark.parametrize("H,P,dtype", [(64, 64, torch.float16), (128, 32, torch.bfloat16)])
def test_tokens_appended_in_parts(gpu, H, P, dtype):
    # one by one, by drafts, by chunks: the same exponents and bounds, and codes that differ only where one was subnormal
    # before its page's exponent grew; each part as the oracle appends it
    m = _entries()
    p = Problem(B=1, L=150, R=2, Rkv=2, H=H, P=P, W=6, dtype=dtype, seed=1)
    p.k[0] *= torch.linspace(-3, 6, 150).exp2()[:, None, None].to(dtype)
    p.v[0, 70] *= 1000
    tables = rope_tables(6 * P, H)
    whole, cache = p.on(gpu), p.cache()
    p.starts = [9]
    whole["starts"] = torch.tensor([9], dtype=torch.int32, device=gpu)
    _append(m, p, whole, rope=tables)
    parts = p.on(gpu)
    first = 0
    for n in [1] * 12 + [4, 5, 60, 1, 40, 28]:
        part = Problem(B=1, L=n, R=2, Rkv=2, H=H, P=P, W=6, dtype=dtype)
        part.q, part.k, part.v = (x[:, first:first + n] for x in (p.q, p.k, p.v))
        parts["starts"] = torch.tensor([9 + first], dtype=torch.int32, device=gpu)
        parts["new_lens"] = torch.tensor([n], dtype=torch.int32, device=gpu)
        _append(m, part, parts, rope=tables)
        pc.append(cache, part.k, part.v, [9 + first], [n], *tables)
        first += n
    assert first == 150
    _check_appended(parts, cache)
    for name in ("k_exponents", "v_exponents", "key_bounds"):
        assert torch.equal(parts[name], whole[name])
    for name in ("k_cache", "v_cache"):
        a, b = parts[name].float(), whole[name].float()
        assert ((a == b) | ((a - b).abs() <= 2.0 ** -9)).all() and (a != b).float().mean() < 0.2


@pytest.mark.gpu
def test_appended_values_that_are_not_finite_and_extremes(gpu):
    m = _entries()
    p = Problem(B=2, L=20, R=2, Rkv=2, H=64, P=16, W=3, dtype=torch.bfloat16, seed=2)
    big = torch.finfo(torch.bfloat16).max
    p.k[0, 3, 0, 5], p.k[0, 4, 1, 60], p.v[0, 5, 0, 0] = math.inf, math.nan, -math.inf
    p.k[1, :, 0], p.v[1, :, 0] = 0, 0                             # pages of zeros
    p.k[1, 2, 1, 3], p.v[1, 2, 1, 3] = big, -big
    p.v[1, 17:, 1] *= 1e-30
    p.k[0, 18:] = math.nan                                         # a page's tokens of which none is finite
    p.k[0, 16:18] = math.nan
    p.k[0, 10, 0], p.q[0, 0, 0, :2] = big, torch.tensor([math.inf, math.nan])   # overflows where it is rotated
    p.starts = [0, 9]
    for tables in (None, rope_tables(48, 64)):
        cache = p.cache()
        pc.append(cache, p.k, p.v, p.starts, p.lens, *(tables or (None, None)))
        t = p.on(gpu)
        got = _append(m, p, t, rope=tables)
        _check_appended(t, cache)
        want = pc.rotated_queries(p.q, p.starts, p.lens, *(tables or (None, None)))
        np.testing.assert_array_equal(p.by_token(got, 2).float().numpy(), want.float().numpy())
    # exactly on the borders of the exponents, and one step beyond
    p = Problem(B=1, L=16, R=2, Rkv=2, H=16, P=16, W=1, dtype=torch.bfloat16, seed=3)
    for amax in (448.0, 450.0, 446.0, 224.0, 2.0 ** -72, 2.0 ** -73):
        p.k[:], p.v[:] = 0.25 * amax * torch.rand(1, 16, 2, 16), amax
        p.k[0, 7, 0, 3] = -amax
        cache, t = p.cache(), p.on(gpu)
        pc.append(cache, p.k, p.v, [0], [16])
        _append(m, p, t)
        _check_appended(t, cache)


@pytest.mark.gpu
def test_append_writes_nothing_else(gpu):
    # pages of others, places behind the last token, tables that name no page or the same one outside the call's reach, positions
    # behind the table, the rotation's tables and before zero
    m = _entries()
    p = Problem(B=6, L=40, R=2, Rkv=2, H=64, P=16, W=4, seed=4, extra=4)
    N = p.k_cache.shape[0]
    p.page_table[1, 1] = -1
    p.page_table[2, 2] = N
    p.page_table[3, 3] = 2 ** 31 - 1
    p.starts = [50, 10, 20, 30, -5, 2 ** 31 - 30]                 # the first passes the table's end
    p.lens = [40, 40, 33, 99, 40, 40]
    for rows in (64, 45):
        tables = rope_tables(rows, 64)
        cache, t = p.cache(), p.on(gpu)
        lens = [min(n, 40) for n in p.lens]
        pc.append(cache, p.k, p.v, p.starts, lens, *tables)
        _append(m, p, t, rope=tables)
        _check_appended(t, cache)
    p.starts, p.lens = [-2 ** 31, 2 ** 31 - 1, 64, 63, 0, 0], [40, 40, 40, 1, -7, -2 ** 31]
    cache, t = p.cache(), p.on(gpu)
    pc.append(cache, p.k, p.v, p.starts, [max(0, n) for n in p.lens])
    _append(m, p, t)
    _check_appended(t, cache)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,P,R,Rkv,L,W,layout", [
    (64, 16, 1, 1, 1, 1, "blf"),           # one head, one page
    (64, 64, 4, 4, 1, 9, "bhld"),          # keys split over workgroups
    (128, 64, 10, 2, 1, 5, "blf"),         # five query heads to a key head
    (128, 16, 17, 1, 1, 20, "blf"),        # more query heads than a tile's rows
    (128, 128, 8, 2, 5, 2, "blf"),         # drafted tokens: 20 rows
    (32, 32, 3, 3, 40, 3, "bhld"),
    (16, 16, 4, 2, 33, 7, "blf"),
    (64, 32, 6, 2, 70, 5, "blf"),          # tiles that end inside a token's group
    (128, 64, 4, 1, 150, 3, "bhld"),
    (64, 64, 2, 2, 300, 6, "blf"),
])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_is_the_oracles(gpu, dtype, H, P, R, Rkv, L, W, layout, causal):
    _compare_attention(gpu, 3, dtype, H, P, R, Rkv, L, W, layout, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,H,P,R,Rkv,L,W,layout", [
    (32, 16, 16, 24, 8, 40, 4, "blf"),
    (1, 16, 32, 12, 4, 500, 100, "blf"),   # keys in parts
    (48, 32, 16, 16, 2, 40, 4, "bhld"),
    (8, 32, 64, 6, 2, 130, 100, "blf"),    # keys in parts, head_dim 32
    (16, 64, 64, 16, 8, 100, 2, "blf"),
    (32, 64, 16, 8, 8, 100, 8, "bhld"),
    (1, 128, 16, 8, 1, 40, 4, "blf"),      # two tiles of rows
    (1, 128, 32, 3, 1, 45, 2, "blf"),      # three query heads to a key head, rows that end inside a wave's
    (4, 128, 64, 64, 8, 70, 2, "bhld"),
    (1, 128, 64, 64, 8, 130, 100, "blf"),  # keys in parts, head_dim 128
    # 256 rows to a workgroup, in parts the last two
    (32, 16, 32, 128, 8, 9, 2, "blf"), (32, 32, 64, 128, 8, 9, 1, "bhld"), (32, 64, 16, 128, 8, 9, 1, "blf"), (8, 128, 32, 256, 8, 17, 2, "bhld"),
    (2, 16, 64, 12, 4, 131, 85, "blf"), (1, 128, 64, 32, 1, 259, 114, "blf"),
])
def test_attention_of_many_rows_is_the_oracles(gpu, dtype, B, H, P, R, Rkv, L, W, layout):
    assert capi.cached_attention_plan(B, L, R, Rkv, H, P, W)["kernel"] == "many"
    for causal in (True, False):
        _compare_attention(gpu, B, dtype, H, P, R, Rkv, L, W, layout, causal)


def test_launches_are_within_what_the_kernels_take():
    # as the kernels count on: row tiles times parts times heads, lanes for the join, parts with keys to take
    rng = random.Random(5)
    kinds = set()
    for _ in range(4000):
        H, P = rng.choice([16, 32, 64, 128]), rng.choice([16, 32, 64, 128])
        B, Rkv, group = int(2 ** rng.uniform(0, 8)), rng.choice([1, 2, 3, 8, 16]), rng.choice([1, 2, 3, 4, 5, 8, 17, 64])
        L, W = int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 12))
        count = rng.choice([0, 0, 0, rng.randint(1, 4096)])
        plan = capi.cached_attention_plan(B, L, Rkv * group, Rkv, H, P, W, count)
        rows = plan["rows"]
        joined = plan["kernel"] == "joined"
        tiles = -(-L // min(L, 16 // group)) if joined else L * -(-group // rows) if count else -(-L * group // rows)
        keys = (count or W) * P
        assert plan["workgroups"] == B * Rkv * tiles * plan["splits"]
        assert 1 <= plan["splits"] <= 64 and (plan["splits"] - 1) * 64 < keys
        if plan["kernel"] == "many":
            assert plan["waves"] == 8 and rows in (128, 256) and not count
        elif joined:
            assert count and L > 1 and group <= 8 and W <= 8192 and plan["waves"] in (2, 4) and (rows, plan["splits"]) == (16, 1)
        else:
            assert plan["waves"] == 4 or (count and plan["waves"] in (1, 8))
            assert rows in (16, 32) and (rows == 16 or (L * group > 16 and not count))
        kinds.add((plan["kernel"], plan["waves"], rows, plan["splits"] > 1))
        if W <= 2048:
            plan = capi.select_pages_plan(B, L, Rkv * group, Rkv, H, P, W)
            assert plan["workgroups"] == B * Rkv * -(-L // plan["tokens"])
            assert plan["tokens"] == 1 or (plan["tokens"] * group == 16 and plan["tokens"] * W <= 8192 and plan["waves"] == 4)
            kinds.add(("select", plan["tokens"] > 1, plan["waves"]))
    assert len(kinds) == 6 + 4 + 2 + 3, kinds                     # few rows, many rows, joined lists, selections


def _compare_attention(gpu, B, dtype, H, P, R, Rkv, L, W, layout, causal):
    p = Problem(B=B, L=L, R=R, Rkv=Rkv, H=H, P=P, W=W, dtype=dtype, seed=H + P + L, layout=layout)
    p.starts = ([W * P - L, max(0, (W * P - L) // 2 - 3), 0] + [(7 * b) % (W * P - L + 1) for b in range(B)])[:B]
    p.lens = ([L, L - L // 4, L] + [L - b % L for b in range(B)])[:B]
    want = pc.attention(p.cache(), p.q, p.starts, p.lens, causal=causal)
    for m in (_entries(), capi):
        t = p.on(gpu)
        got, lse = _attend(m, p, t, causal=causal, return_lse=True)
        assert got.dtype == dtype and got.is_contiguous()
        _check_attention(p, p.by_token(got, R), lse, want)
        again = _attend(m, p, t, causal=causal)
        assert torch.equal(again, got)


@pytest.mark.gpu
@pytest.mark.parametrize("W,P,B,starts", [(700, 16, 1, [11190]), (100, 128, 2, [3, 12700]), (513, 64, 1, [100])])
def test_attention_over_long_tables(gpu, W, P, B, starts):
    # keys in many parts, most of them empty in the short sequences
    p = Problem(B=B, L=2, R=4, Rkv=2, H=64, P=P, W=W, seed=W)
    p.starts = starts
    want = pc.attention(p.cache(), p.q, p.starts, p.lens)
    got, lse = _attend(_entries(), p, p.on(gpu), return_lse=True)
    _check_attention(p, p.by_token(got, 4), lse, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,R,L,kernel", [(64, 4, 16, "few"), (128, 32, 64, "many"), (64, 128, 60, "many")])
def test_attention_over_rows_that_see_nothing(gpu, dtype, H, R, L, kernel):
    p = Problem(B=6, L=L, R=R, Rkv=2, H=H, P=16, W=4, dtype=dtype, seed=7)
    assert capi.cached_attention_plan(6, L, R, 2, H, 16, 4)["kernel"] == kernel
    N = p.k_cache.shape[0]
    p.page_table[1] = -1                                           # no page at all
    p.page_table[2] = torch.tensor([N, 3, -9, 2 ** 31 - 1])
    p.page_table[5, 0] = -1                                        # the first tokens' page is missing
    p.starts = [44, 44, 30, 100, -7, 0]                            # behind the table; before zero
    p.lens = [0] + [L] * 5
    for causal in (True, False):
        want = pc.attention(p.cache(), p.q, p.starts, p.lens, causal=causal)
        got, lse = _attend(_entries(), p, p.on(gpu), causal=causal, return_lse=True)
        _check_attention(p, p.by_token(got, R), lse, want)
    p.starts, p.lens = [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 5, 40, 0, 63], [L, L, -3, 500, -2 ** 31, 1]
    p.q[3, L - 1], p.q[5, 1:] = math.nan, math.inf                 # rows that do not exist hold anything
    p.lens[3] = L - 1
    want = pc.attention(p.cache(), p.q, p.starts, p.lens)
    got, lse = _attend(_entries(), p, p.on(gpu), return_lse=True)
    _check_attention(p, p.by_token(got, R), lse, want)


@pytest.mark.gpu
@pytest.mark.parametrize("H,L,R,kernel", [(64, 1, 4, "few"), (64, 20, 4, "few"), (64, 150, 2, "few"), (128, 150, 64, "many"), (64, 90, 192, "many")])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_that_are_not_numbers_stay_where_they_are_seen(gpu, dtype, H, L, R, kernel):
    # behind the last token, on pages that nobody names, and in tokens that some rows of a tile see and others do not
    p = Problem(B=2, L=L, R=R, Rkv=2, H=H, P=16, W=12, dtype=dtype, seed=8 + L)
    assert capi.cached_attention_plan(2, L, R, 2, H, 16, 12)["kernel"] == kernel
    p.starts = [12 * 16 - L - 30, 5]
    nan = torch.tensor(0x7f, dtype=torch.uint8)
    clean_k, clean_v = p.k_cache.clone(), p.v_cache.clone()
    for cache in (p.k_cache.view(torch.uint8), p.v_cache.view(torch.uint8)):
        for b in range(2):
            for pos in range(p.starts[b] + L, 12 * 16):
                cache[p.page_table[b, pos // 16], :, pos % 16] = nan
    want = pc.attention(p.cache(), p.q, p.starts, p.lens)
    assert torch.isfinite(want[0]).all()
    got, lse = _attend(_entries(), p, p.on(gpu), return_lse=True)
    _check_attention(p, p.by_token(got, R), lse, want)
    if L > 1:
        for pos, channel in ((p.starts[0] + L // 2, 7), (p.starts[0] + L - 1, 33)):
            p.v_cache.view(torch.uint8)[p.page_table[0, pos // 16], 1, pos % 16, channel] = nan + 128 * (channel == 7)
        p.k_cache.view(torch.uint8)[p.page_table[1, (5 + L - 2) // 16], 0, (5 + L - 2) % 16, 9] = nan
        want = pc.attention(p.cache(), p.q, p.starts, p.lens)
        assert torch.isnan(want[0]).any() and torch.isfinite(want[0]).any()
        got, lse = _attend(_entries(), p, p.on(gpu), return_lse=True)
        _check_attention(p, p.by_token(got, R), None, want)
    # queries: their own rows only
    p.k_cache, p.v_cache = clean_k, clean_v
    p.q[0, L - 1, 1, 3], p.q[1, 0, 0, 0] = math.nan, math.inf
    want = pc.attention(p.cache(), p.q, p.starts, p.lens)
    got = p.by_token(_attend(_entries(), p, p.on(gpu)), R)
    rows = torch.isnan(want[0]).any(-1)
    assert rows.sum() == 2 and torch.isnan(got[rows]).all()
    assert torch.isfinite(got[~rows]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,R,L,kernel", [(64, 4, 9, "few"), (128, 128, 90, "many")])
def test_attention_over_pages_of_different_sizes(gpu, dtype, H, R, L, kernel):
    # exponents that grow and shrink along a sequence, scores far apart, scales of the caller's
    p = Problem(B=2, L=L, R=R, Rkv=2, H=H, P=16, W=10, dtype=dtype, seed=9)
    assert capi.cached_attention_plan(2, L, R, 2, H, 16, 10)["kernel"] == kernel
    p.starts = [160 - L, 70]
    p.k_exponents += torch.randint(-2, 3, p.k_exponents.shape, generator=p.gen).to(torch.int8)
    p.v_exponents += torch.randint(-6, 7, p.v_exponents.shape, generator=p.gen).to(torch.int8)
    for scale in (None, 0.9, 1e-4):
        want = pc.attention(p.cache(), p.q, p.starts, p.lens, scale=scale)
        got, lse = _attend(_entries(), p, p.on(gpu), return_lse=True, scale=scale)
        _check_attention(p, p.by_token(got, R), lse, want)
    if dtype == torch.bfloat16:                                    # values far outside of fp16
        p.v_exponents += 60
        want = pc.attention(p.cache(), p.q, p.starts, p.lens)
        got = _attend(_entries(), p, p.on(gpu))
        _check_attention(p, p.by_token(got, R), None, want)


@pytest.mark.gpu
@pytest.mark.parametrize("H,R,L,kernel", [(64, 4, 1, "few"), (64, 4, 9, "few"), (64, 256, 90, "many"), (128, 128, 90, "many")])
@pytest.mark.parametrize("dtype,large,small", [(torch.float16, 0, -14), (torch.float16, 5, -20), (torch.bfloat16, 30, -80), (torch.bfloat16, 60, -80)])
def test_small_values_beside_large_ones_without_weight(gpu, dtype, large, small, H, R, L, kernel):
    # A page of large values that every row sees and gives no weight to: what the header says of the others' bits.  The tolerance is that of
    # the attention without the large page, and of a value next to its power of two: half a step of the smallest fp16 numbers,
    # 2^-25, or with bfloat16 the largest code, below 2^9, times the least scale of its conversion, 2^-126.
    p = Problem(B=2, L=L, R=R, Rkv=2, H=H, P=16, W=10, dtype=dtype, seed=25)
    assert capi.cached_attention_plan(2, L, R, 2, H, 16, 10)["kernel"] == kernel
    p.starts = [160 - L, 70]
    p.q[:] = p.q[:1, :1, :1].clone()                               # every row the same, and a key far below all others: e^-100 at least
    p.v_exponents[:] = small
    at = p.page_table[:, 2].long()
    p.v_exponents[at], p.k_exponents[at] = large, -3
    p.k_cache[at] = (-448 * torch.sign(p.q[0, 0, 0].float())).expand(2, 2, 16, H).to(E4M3)
    assert p.q[0, 0, 0].float().abs().sum() * 448 * 2.0 ** -3 / math.sqrt(H) > 100 + 4 * 448 * 2.0 ** -7
    with_it = pc.attention(p.cache(), p.q, p.starts, p.lens)[0]
    table, p.page_table[:, 2] = p.page_table.clone(), -1
    want, _, spread, size = pc.attention(p.cache(), p.q, p.starts, p.lens)
    p.page_table = table
    assert ((with_it - want).abs() <= 2.0 ** -30 * spread).all()
    u, least = (2.0 ** -11, 2.0 ** -25) if dtype == torch.float16 else (2.0 ** -8, 2.0 ** -117)
    d = (H + 8) * 2.0 ** -24 * size + 20 * 2.0 ** -22              # no score beyond 20 in float32's exponential
    tol = spread * (u + 2 * d[..., None] + 2.0 ** -21 + 2 * (160 + 64) * 2.0 ** -24) + u * want.abs() + 2.0 ** large * least
    tol = tol + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    got = p.by_token(_attend(_entries(), p, p.on(gpu)), R).double()
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.gpu
@pytest.mark.parametrize("H,R,L,kernel", [(64, 4, 9, "few"), (64, 256, 90, "many"), (128, 128, 90, "many")])
def test_scores_too_small_for_a_factor(gpu, H, R, L, kernel):
    # the caller's scale times a page's power of two below any float32: what a row does not see stays out of it all the same
    p = Problem(B=2, L=L, R=R, Rkv=2, H=H, P=16, W=10, seed=23)
    assert capi.cached_attention_plan(2, L, R, 2, H, 16, 10)["kernel"] == kernel
    p.starts = [150 - L, 70]
    pages = torch.randint(0, 10, (2, L, 2, 4), generator=p.gen).to(torch.int32)
    for exponent, scale in ((None, 1e-30), (-80, 1e-30), (-128, 1e-6), (None, 1e-38)):
        if exponent is not None:
            p.k_exponents[::2] = exponent
        for selected in (None, pages):
            want = pc.attention(p.cache(), p.q, p.starts, p.lens, scale=scale, selected=selected)
            got, lse = _attend(_entries(), p, p.on(gpu), return_lse=True, scale=scale, **({} if selected is None else {"pages": selected.to(gpu)}))
            _check_attention(p, p.by_token(got, R), lse, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,P,R,Rkv,L,W,count,layout", [
    (64, 16, 2, 2, 1, 1, 1, "blf"), (64, 16, 4, 2, 3, 12, 4, "bhld"), (128, 64, 20, 4, 1, 30, 8, "blf"), (128, 32, 32, 1, 2, 9, 5, "blf"),
    (16, 128, 4, 2, 5, 6, 3, "blf"), (32, 64, 6, 3, 30, 5, 2, "bhld"), (64, 16, 8, 2, 2, 300, 64, "blf"), (128, 16, 40, 1, 1, 600, 33, "blf"),
    # sixteen rows of several tokens to a workgroup of the selection, and more attention tiles than a chip holds
    (64, 16, 8, 8, 300, 25, 5, "blf"), (16, 16, 16, 8, 150, 12, 4, "bhld"), (128, 32, 32, 8, 70, 40, 9, "blf"), (32, 64, 64, 8, 35, 5, 3, "blf"),
    (64, 16, 24, 8, 120, 20, 20, "blf"),
])
def test_selection_and_attention_over_it_are_the_oracles(gpu, dtype, H, P, R, Rkv, L, W, count, layout):
    p = Problem(B=2, L=L, R=R, Rkv=Rkv, H=H, P=P, W=W, dtype=dtype, seed=H + W, layout=layout)
    p.starts = [W * P - L, max(0, W * P // 2 - 3)]
    p.lens = [L, L - L // 3]
    if W > 2:
        p.page_table[0, 1] = -1                                    # never selected
    cache = p.cache()
    want_pages = pc.select(cache, p.q, p.starts, p.lens, count)
    want = pc.attention(cache, p.q, p.starts, p.lens, selected=want_pages)
    for m in (_entries(), capi):
        t = p.on(gpu)
        plan = capi.select_pages_plan(2, L, R, Rkv, H, P, W)
        assert (plan["tokens"] > 1) == (L > 30 and R // Rkv in (1, 2, 4, 8))
        pages = _select(m, p, t, count)
        assert torch.equal(pages.cpu(), want_pages)
        got, lse = _attend(m, p, t, pages=pages, return_lse=True)
        _check_attention(p, p.by_token(got, R), lse, want)


@pytest.mark.gpu
@pytest.mark.parametrize("L,R,Rkv", [(2, 4, 2), (90, 16, 8), (45, 4, 4)])
def test_selections_with_ties_and_odd_queries(gpu, L, R, Rkv):
    m = _entries()
    p = Problem(B=3, L=L, R=R, Rkv=Rkv, H=64, P=16, W=40, seed=11)
    p.starts = [640 - L, 333, 0]
    p.key_bounds[:, :, 0], p.key_bounds[:, :, 1] = 1, -1          # every page the same score
    p.k_exponents[:] = -7
    for count in (1, 2, 7, 39, 40, 64):
        assert torch.equal(_select(m, p, p.on(gpu), count).cpu(), pc.select(p.cache(), p.q, p.starts, p.lens, count))
    p.k_exponents[torch.randperm(p.k_exponents.shape[0], generator=p.gen)[:60]] = -6
    p.q[0, 0, 0, 0], p.q[0, 1, 3, 5], p.q[1, 0] = math.inf, math.nan, 0
    p.q[1, 1, 2:] = -p.q[1, 1, 2:].abs() * 1000
    for count in (1, 5, 17):
        assert torch.equal(_select(m, p, p.on(gpu), count).cpu(), pc.select(p.cache(), p.q, p.starts, p.lens, count))
    # negative scores throughout, and exponents at their ends
    p.key_bounds[:, :, 0], p.key_bounds[:, :, 1] = -3, -90
    p.q = p.q.nan_to_num(posinf=9.0).abs()
    p.k_exponents[:] = torch.randint(-80, 121, p.k_exponents.shape, generator=p.gen).to(torch.int8)
    p.starts, p.lens = [638, 400, -1], [L, L - 1, L]
    assert torch.equal(_select(m, p, p.on(gpu), 9).cpu(), pc.select(p.cache(), p.q, p.starts, p.lens, 9))


@pytest.mark.gpu
def test_lists_of_pages_as_they_come(gpu):
    # in any order, named twice, outside the table, behind the token, empty
    p = Problem(B=2, L=3, R=4, Rkv=2, H=64, P=16, W=6, seed=12)
    p.starts = [90, 40]
    lists = [[0, 0, 3, 3, 3, 0], [5, 2, 1, -1, 2, 5], [6, 7, -1, 2 ** 31 - 1, -2 ** 31, 99], [4, 3, 2, 1, 0, 5], [1, 1, 1, 1, 1, 1], [-1] * 6]
    pages = torch.tensor(lists * 2, dtype=torch.int32).view(2, 3, 2, 6)
    for count in (6, 3, 1):
        want = pc.attention(p.cache(), p.q, p.starts, p.lens, selected=pages[..., :count])
        got, lse = _attend(_entries(), p, p.on(gpu), pages=pages[..., :count].contiguous().to(gpu), return_lse=True)
        _check_attention(p, p.by_token(got, 4), lse, want)
    # every page listed, repeated over the longest list there may be: what it is without a list
    many = torch.arange(4096, dtype=torch.int32).remainder(6).expand(2, 3, 2, 4096).contiguous()
    want = pc.attention(p.cache(), p.q, p.starts, p.lens)
    got, lse = _attend(_entries(), p, p.on(gpu), pages=many.to(gpu), return_lse=True)
    _check_attention(p, p.by_token(got, 4), lse, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,R,Rkv,L,H,P,W,count,waves,causal,layout", [
    (4, 8, 8, 128, 64, 16, 9, 3, 4, True, "blf"), (8, 80, 16, 7, 128, 16, 9, 6, 4, True, "blf"), (8, 16, 16, 100, 16, 16, 7, 2, 2, True, "bhld"),
    (3, 32, 4, 90, 32, 32, 5, 4, 4, False, "blf"), (4, 24, 8, 150, 128, 16, 12, 5, 2, True, "blf"), (16, 32, 16, 40, 128, 64, 3, 1, 2, False, "bhld"),
    (6, 24, 12, 90, 64, 128, 2, 2, 2, True, "blf"), (4, 32, 16, 35, 16, 32, 130, 70, 4, True, "blf"),
])
@pytest.mark.parametrize("nan", [False, True])
def test_joined_lists(gpu, dtype, B, R, Rkv, L, H, P, W, count, waves, causal, layout, nan):
    # lists of several tokens in one tile: repeats, gaps, numbers outside the table, tokens that do not exist, and values that are not
    # numbers on pages that some of the tokens list
    p = Problem(B=B, L=L, R=R, Rkv=Rkv, H=H, P=P, W=W, dtype=dtype, seed=H + L + count, layout=layout)
    plan = capi.cached_attention_plan(B, L, R, Rkv, H, P, W, count)
    assert (plan["kernel"], plan["waves"]) == ("joined", waves)
    p.starts = [max(0, W * P - L - 5 * b * b) if b % 3 < 2 else b for b in range(B)]
    p.lens = [L - (b * L) // (2 * B) for b in range(B)]
    lists = torch.randint(-1, W + 1, (B, L, Rkv, count), generator=p.gen).to(torch.int32)
    lists[0, ::2] = lists[0, 0].clone()                  # some alike,
    lists[-1, 1] = -1                                    # one empty
    if nan:
        code = torch.tensor(0x7f, dtype=torch.uint8)
        p.v_cache.view(torch.uint8)[p.page_table[0, W // 2], 1, 3, H - 1] = code
        p.k_cache.view(torch.uint8)[p.page_table[0, 0], 0, P - 1, 2] = code + 128
        p.v_cache.view(torch.uint8)[p.page_table[B - 1, W - 1], :, P - 1] = code
        p.q[1, 0, 0, 0] = math.nan
    want = pc.attention(p.cache(), p.q, p.starts, p.lens, selected=lists, causal=causal)
    assert not nan or (torch.isnan(want[0]).any() and torch.isfinite(want[0]).any())
    got, lse = _attend(_entries(), p, p.on(gpu), pages=lists.to(gpu), return_lse=True, causal=causal)
    _check_attention(p, p.by_token(got, R), lse, want)


@pytest.mark.gpu
def test_lists_with_gaps(gpu):
    # a page named on both sides of numbers that name nothing still counts once
    p = Problem(B=2, L=3, R=4, Rkv=2, H=64, P=16, W=6, seed=22)
    p.starts = [90, 40]
    lists = [[5, -1, 5, -1, 5, -1], [0, 1, -1, 0, 1, 2], [-1, 2, -5, 2, 3, 4], [1, 6, -1, 1, 6, -1], [-1, -1, 3, 4, -1, 3], [0, -2 ** 31, 0, 2, 2 ** 31 - 1, 2]]
    pages = torch.tensor(lists * 2, dtype=torch.int32).view(2, 3, 2, 6)
    for repeats in (1, 60):                              # entries of one thread, and of several
        some = torch.cat([pages] * repeats, dim=3)
        want = pc.attention(p.cache(), p.q, p.starts, p.lens, selected=some)
        got, lse = _attend(_entries(), p, p.on(gpu), pages=some.to(gpu), return_lse=True)
        _check_attention(p, p.by_token(got, 4), lse, want)


@pytest.mark.gpu
def test_the_widest_table_and_the_longest_lists(gpu):
    # 32768 pages in a table, 4096 of them selected; the longest lists on each form of the attention kernel
    m = _entries()
    p = Problem(B=1, L=2, R=2, Rkv=1, H=16, P=16, W=32768, seed=20, extra=0)
    p.starts = [32768 * 16 - 2]
    pages = _select(m, p, p.on(gpu), 4096)
    cache = p.cache()
    want = pc.select(cache, p.q, p.starts, p.lens, 4096)
    assert torch.equal(pages.cpu(), want)
    got, lse = _attend(m, p, p.on(gpu), pages=pages, return_lse=True)
    _check_attention(p, p.by_token(got, 2), lse, pc.attention(cache, p.q, p.starts, p.lens, selected=want))
    for B, L, R, kernel, waves in ((2, 1, 2, "few", 4), (100, 1, 2, "few", 8), (3, 200, 18, "few", 1), (4, 100, 16, "joined", 4), (4, 200, 16, "joined", 2)):
        p = Problem(B=B, L=L, R=R, Rkv=2, H=128, P=16, W=16, seed=21)
        plan = capi.cached_attention_plan(B, L, R, 2, 128, 16, 16, 4096)
        assert (plan["kernel"], plan["waves"]) == (kernel, waves)
        p.starts = [(31 * b) % (256 - L + 1) for b in range(B)]
        lists = torch.full((B, L, 2, 4096), -1, dtype=torch.int32)
        lists[..., 5], lists[..., 100], lists[..., 101], lists[..., 4095] = 3, 9, 3, 0
        want = pc.attention(p.cache(), p.q, p.starts, p.lens, selected=lists)
        got, lse = _attend(m, p, p.on(gpu), pages=lists.to(gpu), return_lse=True)
        _check_attention(p, p.by_token(got, R), lse, want)


@pytest.mark.gpu
@pytest.mark.parametrize("L,W,waves", [(512, 8192, 4), (1536, 8191, 2)])
def test_joined_lists_of_the_longest_tables(gpu, L, W, waves):
    # queries of zero give every key one weight, so that the log-sum-exp counts the keys that a row's list names: a page more or less
    # among some 3200 moves it by 2^-12, rounding by 2^-18 at most: the sum of n weights of 2^7 is exact below 2^24, its logarithm of
    # base 2, below 24, is off by 2^-20 and its product with ln 2 by 2^-20
    p = Problem(B=1, L=L, R=8, Rkv=8, H=16, P=16, W=W, dtype=torch.bfloat16, seed=24, extra=0, bounds=False)
    plan = capi.cached_attention_plan(1, L, 8, 8, 16, 16, W, 4096)
    assert (plan["kernel"], plan["waves"]) == ("joined", waves)
    p.q = torch.zeros_like(p.q)
    p.starts = [16 * W - L]
    lists = torch.randint(-1, W + 1, (1, L, 8, 4096), generator=p.gen).to(torch.int32).to(gpu)
    got, lse = _attend(_entries(), p, p.on(gpu), pages=lists, return_lse=True)
    named = torch.zeros(L, 8, W + 2, dtype=torch.bool, device=gpu)
    named.scatter_(2, lists[0].long() + 1, True)
    limit = p.starts[0] + 1 + torch.arange(L, device=gpu)
    seen = (limit[:, None] - 16 * torch.arange(W, device=gpu)).clamp(0, 16)
    n = torch.stack([(named[:, head, 1:-1] * seen).sum(-1) for head in range(8)], 0).double()
    assert (lse[0].double() - n.log()).abs().max().item() < 2.0 ** -14
    assert torch.isfinite(got).all()


@pytest.mark.gpu
def test_pages_beyond_32_bits_of_bytes(gpu):
    # a cache of 5 GB for keys and for values each, its last pages in use
    m = _entries()
    p = Problem(B=1, L=40, R=4, Rkv=2, H=128, P=128, W=3, seed=13, extra=1)
    N = 5 * 2 ** 30 // (2 * 128 * 128)
    small, t = p.on(gpu), p.on(gpu)
    high = torch.tensor([[N - 1, N - 3, N - 2]], dtype=torch.int32, device=gpu)
    for name, value in list(t.items()):
        if name in ("k_cache", "v_cache", "k_exponents", "v_exponents", "key_bounds"):
            big = torch.empty((N,) + tuple(value.shape[1:]), dtype=value.dtype, device=gpu)
            big.view(torch.uint8)[high[0].long()] = value.view(torch.uint8)[t["page_table"][0].long()]
            t[name] = big
    t["page_table"] = high
    for s in (small, t):
        s["starts"] = torch.tensor([300], dtype=torch.int32, device=gpu)
    tables = rope_tables(384, 128)
    q1, q2 = (_append(m, p, s, rope=tables) for s in (small, t))
    assert torch.equal(q1, q2)
    for name in ("k_cache", "v_cache", "k_exponents", "v_exponents", "key_bounds"):
        assert torch.equal(t[name].view(torch.uint8)[high[0].long()], small[name].view(torch.uint8)[small["page_table"][0].long()])
    s1, s2 = (_select(m, p, s, 2, q=q1) for s in (small, t))
    assert torch.equal(s1, s2)
    assert torch.equal(_attend(m, p, small, q=q1), _attend(m, p, t, q=q1))
    assert torch.equal(_attend(m, p, small, q=q1, pages=s1), _attend(m, p, t, q=q1, pages=s1))


@pytest.mark.gpu
def test_views_and_tables_with_rows_apart(gpu):
    # slices of a packed projection, single tokens with strides that mean nothing, a slice of a wider page table, `out` views
    m = _entries()
    p = Problem(B=2, L=6, R=2, Rkv=2, H=64, P=16, W=5, seed=14)
    p.starts = [60, 33]
    t = p.on(gpu)
    packed = torch.stack([p.laid_out(x) for x in (p.q, p.k, p.v)], dim=2).to(gpu)
    q, k, v = (packed[:, :, n] for n in range(3))
    table = torch.full((2, 9), -1, dtype=torch.int32, device=gpu)
    table[:, 2:7] = t["page_table"]
    t["page_table"] = table[:, 2:7]
    cache = p.cache()
    pc.append(cache, p.k, p.v, p.starts, p.lens)
    got_q = m.cache_append(keys=k, values=v, queries=q, **_only(t, *CACHE, "key_bounds"))
    assert torch.equal(got_q, q)
    _check_appended(t, cache)
    want = pc.attention(cache, p.q, p.starts, p.lens)
    _check_attention(p, p.by_token(_attend(m, p, t, q=q), 2), None, want)
    wide = torch.full((2, 6, 4, 64), 7.0, dtype=torch.float16, device=gpu)
    out = wide.view(2, 6, 256)[:, :, 64:192]
    assert _attend(capi, p, t, q=q, out=out) is out
    assert torch.equal(out, _attend(m, p, t, q=q)) and (wide[:, :, 0] == 7).all() and (wide[:, :, 3] == 7).all()
    one = q[:, 2:3].transpose(0, 1).contiguous().transpose(0, 1)
    one = one.as_strided((2, 1, 128), (one.stride(0), 1, 1))
    t["starts"], t["new_lens"] = t["starts"] + 2, torch.ones_like(t["new_lens"])
    assert torch.equal(_attend(m, p, t, q=one), _attend(m, p, t, q=q[:, 2:3].contiguous()))


@pytest.mark.gpu
def test_an_answer_token_by_token(gpu):
    # projection, append with rotation, attention; selection once the context is longer than what is selected.  Against the
    # oracle's cache step by step, and the dense attention kernel on what the cache stands for.
    import fused_attn

    B, R, H, P, W = 2, 4, 64, 16, 6
    F = R * H
    p = Problem(B=B, L=1, R=R, Rkv=R, H=H, P=P, W=W, dtype=torch.float16, seed=15)
    t, cache = p.on(gpu), p.cache()
    tables = rope_tables(W * P, H)
    cos, sin = (x.to(gpu) for x in tables)
    weight = (torch.randn(F, 3 * F, generator=p.gen) / math.sqrt(F)).half().to(gpu)
    lens = [37, 21]
    starts = [0, 0]
    for step in range(12):
        L = 37 if step == 0 else 3 if step == 5 else 1
        new = lens if step == 0 else [L, L]
        t["starts"] = torch.tensor(starts, dtype=torch.int32, device=gpu)
        t["new_lens"] = torch.tensor(new, dtype=torch.int32, device=gpu)
        hidden = torch.randn(B, L, F, generator=p.gen).half().to(gpu)
        qkv = fused_attn.qkv_projection(hidden, weight, None, R, H)
        q, k, v = (qkv[:, :, n] for n in range(3))
        p.L = L
        q = fused_attn.cache_append(k, v, queries=q, rope_cos=cos, rope_sin=sin, **_only(t, *CACHE, "key_bounds"))
        pc.append(cache, *(x.cpu().reshape(B, L, R, H) for x in (k, v)), starts, new, *tables)
        _check_appended(t, cache)
        assert torch.equal(p.by_token(q, R), pc.rotated_queries(qkv[:, :, 0].cpu().reshape(B, L, R, H), starts, new, *tables))
        got, lse = _attend(_entries(), p, t, q=q, return_lse=True)
        most = int(cache.exponents["v"].max())
        _check_attention(p, p.by_token(got, R), lse, pc.attention(cache, p.by_token(q, R), starts, new), most)
        pages = _select(_entries(), p, t, 3, q=q)
        assert torch.equal(pages.cpu(), pc.select(cache, p.by_token(q, R), starts, new, 3))
        got = _attend(_entries(), p, t, q=q, pages=pages)
        _check_attention(p, p.by_token(got, R), None, pc.attention(cache, p.by_token(q, R), starts, new, selected=pages.cpu()), most)
        if step == 0:                                              # the first prompt is the whole context: the dense kernel's case
            dense = []
            for name in ("k", "v"):
                x = np.stack([np.concatenate([cache.codes[name][cache.page(0, w)] * 2.0 ** cache.exponents[name][cache.page(0, w)][:, None, None]
                                              for w in range(W)], axis=1)])
                dense.append(torch.from_numpy(x)[:, :, :37].transpose(1, 2).reshape(1, 37, F).half().to(gpu))
            want = fused_attn.attention_forward_ex(q[:1], *dense, H, causal=True)
            whole = _attend(_entries(), p, t, q=q)
            # both round their weights and results: two of each
            assert (whole[0].float() - want[0].float()).abs().max() <= 4 * 2.0 ** -11 * dense[1].abs().max()
        starts = [a + b for a, b in zip(starts, new)]


@pytest.mark.gpu
def test_steps_captured_in_graphs(gpu):
    # append, select and attend in one graph, and a second graph of the same calls: replayed in turn with eager work between,
    # each against eager calls on copies.  starts live on the device, so that a replay is the next token's step.
    m = _entries()
    p = Problem(B=2, L=1, R=4, Rkv=2, H=64, P=16, W=40, seed=16)
    p.starts = [500, 123]
    tables = rope_tables(640, 64)

    def step(t, q, k, v, cos, sin):
        q = m.cache_append(k, v, queries=q, rope_cos=cos, rope_sin=sin, **_only(t, *CACHE, "key_bounds"))
        pages = m.select_pages(q, page_size=16, count=5, **_only(t, "k_exponents", "page_table", "starts", "new_lens", "key_bounds"))
        return (q, pages, m.cached_attention(q, **_only(t, *CACHE)), m.cached_attention(q, pages=pages, **_only(t, *CACHE)))

    cos, sin = (x.to(gpu) for x in tables)
    runs = []
    for _ in range(2):
        t = p.on(gpu)
        x = [p.laid_out(y).to(gpu) for y in (p.q, p.k, p.v)]
        warm = {name: value.clone() for name, value in t.items()}
        side = torch.cuda.Stream(device=gpu)
        side.wait_stream(torch.cuda.current_stream(gpu))
        with torch.cuda.stream(side):
            step(warm, *x, cos, sin)
        torch.cuda.current_stream(gpu).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(t, *x, cos, sin)
        runs.append((graph, t, x, out, p.on(gpu)))
    for n in range(5):
        for graph, t, x, out, eager in runs:
            for y in x:
                y.copy_(torch.randn(y.shape, generator=p.gen).to(y.dtype))
            graph.replay()
            want = step(eager, *x, cos, sin)
            for a, b in zip(out, want):
                assert torch.equal(a, b)
            for name in ("k_cache", "v_cache", "k_exponents", "v_exponents", "key_bounds"):
                assert torch.equal(t[name].view(torch.uint8), eager[name].view(torch.uint8))
            t["starts"] += 1
            eager["starts"] += 1


@pytest.mark.gpu
def test_steps_on_two_streams(gpu):
    # two answers, each on a stream of its own, at the same time: what each is by itself
    m = _entries()
    problems = [Problem(B=2, L=3, R=4, Rkv=2, H=64, P=16, W=200, seed=s) for s in (17, 18)]
    for p in problems:
        p.starts = [3000, 2500]
    alone, tensors, streams = [], [], []
    for p in problems:
        t = p.on(gpu)
        q = _append(m, p, t)
        alone.append((q, _attend(m, p, t, q=q), _select(m, p, t, 9, q=q)))
        tensors.append((p.on(gpu), [p.laid_out(x).to(gpu) for x in (p.q, p.k, p.v)]))
        streams.append(torch.cuda.Stream(device=gpu))
    torch.cuda.synchronize()
    got = [None, None]
    for rep in range(3):
        for n in range(2):
            with torch.cuda.stream(streams[n]):
                p, (t, (q, k, v)) = problems[n], tensors[n]
                q = m.cache_append(k, v, queries=q, **_only(t, *CACHE, "key_bounds"))
                got[n] = (q, _attend(m, p, t, q=q), _select(m, p, t, 9, q=q))
        torch.cuda.synchronize()
        for n in range(2):
            assert all(torch.equal(a, b) for a, b in zip(alone[n], got[n]))
