"""Rotary positions: the oracle and the refusals on the CPU; on the GPU the tables against 64 bits and the rotation against the oracle bit
by bit, since its definition leaves nothing open.

Tolerance of the tables: the angle of position p in 64 bits is off by 4 roundings of 2^-53 of p f (frequency, its share of a turn, the
product, the way back), the series by 7e-12, and the result is rounded once to float32: amplitude (p f 2^-51 + 1e-11) + |value| 2^-24 +
2^-149.
"""
import ctypes
import math
import random

import numpy as np
import pytest
import torch

from fused_attention_amd import capi
from oracle import rotary as ro

F16, BF16 = torch.float16, torch.bfloat16
SCALINGS = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
            dict(scaling="turns", factor=8.0, original_rows=512.0, low=1.0, high=4.0),
            dict(scaling="index", factor=16.0, original_rows=256.0, low=1.0, high=32.0, amplitude=1.2772588722239782),
            dict(base=500000.0, scaling="turns", factor=32.0, original_rows=8192.0, low=1.0, high=4.0)]


def _module():
    import fused_attn

    return fused_attn


# ---- the oracle, on the CPU ----

def test_frequencies_of_the_oracle():
    plain = ro.frequencies(64)
    np.testing.assert_allclose(plain, [10000.0 ** (-j / 32) for j in range(32)], rtol=1e-14)
    for scaling in ("linear", "base", "turns", "index"):
        np.testing.assert_allclose(ro.frequencies(64, scaling=scaling, factor=1.0, original_rows=512.0, high=32.0), plain, rtol=1e-14)
    np.testing.assert_allclose(ro.frequencies(64, scaling="linear", factor=4.0), plain / 4, rtol=1e-14)
    turns = 512 * plain / (2 * np.pi)
    for scaling, high in (("turns", 4.0), ("index", 32.0)):
        f = ro.frequencies(64, scaling=scaling, factor=4.0, original_rows=512.0, low=1.0, high=high)
        assert np.all(f[turns > 2 * high] == plain[turns > 2 * high]) and np.allclose(f[turns < 0.5], plain[turns < 0.5] / 4, rtol=1e-14)
        assert np.all(f <= plain * (1 + 1e-15)) and np.all(f >= plain / 4 * (1 - 1e-15))
    # the last column's wave is `factor` times as long, the first one stays
    f = ro.frequencies(64, scaling="base", factor=4.0)
    assert f[0] == 1.0 and math.isclose(f[-1], plain[-1] / 4, rel_tol=1e-12)


def test_tables_and_rotation_of_the_oracle():
    cos, sin = ro.tables(40, 32, scaling="turns", factor=3.0, original_rows=10.0)
    assert np.all(cos[0] == 1) and np.all(sin[0] == 0)
    np.testing.assert_allclose(cos[5] * cos[7] - sin[5] * sin[7], cos[12], atol=1e-14)
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 5, 3, 48, generator=g).to(BF16)
    c, s = (torch.from_numpy(t).float() for t in (cos, sin))
    at = torch.tensor([[0, 3, 39, 40, -1], [7, 7, 1, 2, 38]])
    for il in (False, True):
        y = ro.rotate(x, c, s, at, first=8, interleaved=il)
        part = x[..., 8:40].double()
        z = torch.complex(part[..., 0::2], part[..., 1::2]) if il else torch.complex(part[..., :16], part[..., 16:])
        z = z * torch.polar(torch.ones(2, 5, 16, dtype=torch.float64), torch.atan2(s, c).double()[at.clamp(0, 39)])[:, :, None]
        want = torch.stack([z.real, z.imag], -1).flatten(-2) if il else torch.cat([z.real, z.imag], -1)
        ok = (at >= 0) & (at < 40)
        assert ((y[..., 8:40].double() - want)[ok].abs() <= want[ok].abs() * 2.0 ** -8 + 1e-5).all()
        assert torch.equal(y[ok][..., :8], x[ok][..., :8]) and torch.equal(y[ok][..., 40:], x[ok][..., 40:]) and (y[~ok] == 0).all()
        back = ro.rotate(y, c, s, at, first=8, interleaved=il, inverse=True)
        assert ((back - x).float()[ok].abs() <= 2.0 ** -6 * x.float()[ok].abs().amax(-1, keepdim=True)).all()
    q, k = (torch.randn(1, 1, 1, 32, generator=g).to(F16).expand(1, 2, 1, 32) for _ in range(2))
    a = (ro.rotate(q, c, s, torch.tensor([[3, 13]])).double() * ro.rotate(k, c, s, torch.tensor([[8, 18]])).double()).sum(-1)
    assert abs(a[0, 0] - a[0, 1]) < 0.05


# ---- refusals, on the CPU ----

def test_the_library_refuses_what_its_header_says():
    lib, ok = capi.load_library(), 0x1000                          # never dereferenced: every case is refused before a launch

    def tables(cos=ok, sin=ok, rows=4, dims=32, how=(0, 10000.0, 1.0, 1.0, 1.0, 4.0, 1.0)):
        return lib.fa_rotary_tables(cos, sin, rows, dims, None if how is None else ctypes.byref(capi.Rotary(*how)), None)

    assert tables(cos=None) == -1 and tables(sin=None) == -1 and tables(how=None) == -1
    assert tables(rows=0) == -3 and tables(dims=0) == -3 and tables(dims=40) == -3 and tables(dims=272) == -6 and tables(rows=2 ** 31) == -6
    assert tables(cos=ok + 4) == -5 and tables(sin=ok + 8) == -5
    assert tables(how=(5, 10000.0, 1, 1, 1, 4, 1)) == -7 and tables(how=(-1, 10000.0, 1, 1, 1, 4, 1)) == -7
    for how in ((0, 1.0, 1, 1, 1, 4, 1), (0, math.inf, 1, 1, 1, 4, 1), (0, 1e4, 1, 1, 1, 4, 0.0), (0, 1e4, 1, 1, 1, 4, math.nan), (1, 1e4, 0.0, 1, 1, 4, 1),
                (2, 1e4, -1.0, 1, 1, 4, 1), (3, 1e4, 2, 0.0, 1, 4, 1), (3, 1e4, 2, 9, 4, 4, 1), (4, 1e4, 2, 9, -1, 4, 1), (4, 1e4, 2, 9, 1, math.inf, 1),
                (2, 1e300, 1e300, 1, 1, 4, 1)):
        assert tables(how=how) == -8, how

    def rotate(q=ok, qs=(512, 64, 256), out=ok, os=(512, 64, 256), k=None, ks=(0, 0, 0), k_out=None, kos=(0, 0, 0), B=2, L=2, R=4, Rkv=0, H=64, first=0,
               dims=64, cos=ok, sin=ok, rows=9, positions=None, starts=None, lens=None, flags=0):
        return lib.fa_rotate(q, *qs, out, *os, k, *ks, k_out, *kos, B, L, R, Rkv, H, first, dims, cos, sin, rows, positions, starts, lens, flags, None)

    assert rotate(flags=1) == -7 and rotate(flags=16) == -7
    assert [rotate(H=h) for h in (0, 8, 40, 1040)] == [-2] * 4
    assert rotate(q=None) == -1 and rotate(out=None) == -1 and rotate(cos=None) == -1 and rotate(sin=None) == -1 and rotate(k=ok, Rkv=1) == -1
    assert rotate(B=0) == -3 and rotate(L=0) == -3 and rotate(R=0) == -3 and rotate(rows=0) == -3
    assert rotate(dims=0) == -3 and rotate(dims=24) == -3 and rotate(dims=80) == -3 and rotate(first=4, dims=32) == -3 and rotate(first=40, dims=32) == -3
    assert rotate(first=-8, dims=32) == -3 and rotate(positions=ok, starts=ok) == -3
    assert rotate(q=ok + 2) == -5 and rotate(out=ok + 8) == -5 and rotate(cos=ok + 4) == -5 and rotate(starts=ok + 2) == -5 and rotate(lens=ok + 1) == -5
    assert rotate(qs=(512, 64, 56)) == -4 and rotate(qs=(512, 60, 256)) == -4 and rotate(os=(512, 0, 256)) == -4 and rotate(os=(504, 64, 256)) == -4
    assert rotate(B=2 ** 20, L=2 ** 20) == -6 and rotate(L=2 ** 31) == -6
    assert rotate(k=ok, ks=(256, 64, 128), k_out=ok, kos=(256, 64, 64), Rkv=2) == -4 and rotate(k=ok, ks=(256, 64, 128), k_out=ok, kos=(256, 64, 128), Rkv=0) == -3


@pytest.mark.parametrize("how", ["module", "capi"])
def test_in_place_refuses_what_autograd_would_go_on_with(how):
    # its gradient would pass as if nothing had been rotated
    errors = RuntimeError if how == "module" else ValueError
    cos = torch.zeros(9, 16)

    def call(q, k):
        if how == "module":
            return _module().rotate(q, cos, cos, 64, keys=k, in_place=True)
        return capi.rotate(q, (cos, cos), 64, keys=k, out=(q, k))

    def both():
        return torch.zeros(2, 3, 256, dtype=F16), torch.zeros(2, 3, 128, dtype=F16)

    for which in (0, 1):
        x = both()
        x[which].requires_grad_()
        for y in (x, tuple(t * 1 for t in x)):                     # a leaf, and what follows from one
            with pytest.raises(errors, match="gradient"):
                call(*y)
            with torch.no_grad(), pytest.raises(errors, match="GPU"):
                call(*y)
    with pytest.raises(errors, match="GPU"):
        call(*both())


def test_outputs_that_share_places_with_what_is_read_or_written_beside_them():
    # against all places of small views, written out; without a GPU a call that is not refused ends at its launch
    lib, ok, H = capi.load_library(), 0x100000, 16
    g = random.Random(1)

    def places(at, s, B, heads, L):
        return {at // 2 + b * s[0] + h * s[1] + l * s[2] + c for b in range(B) for h in range(heads) for l in range(L) for c in range(H)}

    seen = set()
    for n in range(400):
        B, L, R, Rkv = (g.choice([1, 2, 3]) for _ in range(4))
        wide = g.choice([3, 4, 6]) * H                             # a token's values in the one tensor that all are views of
        s = (wide * 5, H, wide)
        at = [ok + 2 * (8 * g.randrange(0, 4 * H // 8) + wide * g.randrange(0, 3) + s[0] * g.randrange(0, 3)) for _ in range(4)]
        if g.random() < 0.5:
            at[1] = at[0]                                          # in place
        if g.random() < 0.5:
            at[3] = at[2]
        if max(R, Rkv) * H > wide:
            continue
        of = [places(a, s, B, heads, L) for a, heads in zip(at, (R, R, Rkv, Rkv))]
        bad = (at[0] != at[1] and of[0] & of[1]) or (at[2] != at[3] and of[2] & of[3]) or of[1] & of[3] or of[1] & of[2] or of[3] & of[0]
        seen.add(bool(bad))
        if bad or not torch.cuda.is_available():                   # (addresses of nothing: what is not refused goes to no GPU)
            got = lib.fa_rotate(at[0], *s, at[1], *s, at[2], *s, at[3], *s, B, L, R, Rkv, H, 0, H, ok, ok, 9, None, None, None, 0, None)
            assert got == -4 if bad else got > 0, (n, at, s, B, L, R, Rkv)
    assert seen == {True, False}
    one = lambda q_out, k, k_out, ks=(512, 64, 256): lib.fa_rotate(ok, 512, 64, 256, q_out, 512, 64, 256, k, *ks, k_out, *ks, 2, 2, 4, 1, 64, 0, 64, ok, ok, 9, None, None,
                                                                   None, 0, None)
    assert one(ok, ok, ok) == -4 and one(ok + 0x10000, ok, ok + 0x10000) == -4           # the same tensor twice, one output for both
    assert one(ok, ok + 128, ok + 128, (64, 64, 64)) == -4                               # other strides, on one of the queries' heads
    assert one(ok + 16, ok + 0x10000, ok + 0x10000) == -4                                # written 8 values behind what is read


@pytest.mark.parametrize("how", ["module", "capi"])
def test_the_entry_points_refuse_wrong_tensors(how):
    m = _module() if how == "module" else capi
    errors = RuntimeError if how == "module" else (ValueError, TypeError)
    q, k = torch.zeros(2, 3, 256, dtype=F16), torch.zeros(2, 3, 128, dtype=F16)
    cos = torch.zeros(9, 16)

    def call(queries=q, keys=k, cos=cos, sin=cos, head_dim=64, **kw):
        return m.rotate(queries, *((cos, sin) if how == "module" else ((cos, sin),)), head_dim, keys=keys, **kw)

    def refused(match, **kw):
        with pytest.raises(errors, match=match):
            call(**kw)

    refused("GPU")
    refused("head_dim must be", head_dim=40)
    refused("layout must be", layout="x")
    refused("dimensions", layout="bhld")
    refused("queries must be float16 or bfloat16", queries=q.float())
    refused("features of queries", queries=q[..., :40])
    refused("dtype", keys=k.bfloat16())
    refused("empty dimension", queries=q[:, :0], keys=None)
    refused("keys must have the batch", keys=k[:, :2])
    refused("last dimension", queries=q.repeat_interleave(2, 2)[..., ::2], keys=None)
    refused("one shape", sin=cos[:8])
    refused("must be", cos=cos.double(), sin=cos.double())
    refused("multiple of 8", cos=cos[:, :4].contiguous(), sin=cos[:, :4].contiguous())
    refused("first", first=4)
    refused("first", first=40)
    refused("exclude", starts=torch.zeros(2, dtype=torch.int32), positions=torch.zeros(2, 3, dtype=torch.int32))
    refused("starts must", starts=torch.zeros(3, dtype=torch.int32))
    refused("starts must", starts=torch.zeros(2))
    refused("new_lens must", new_lens=torch.zeros(2, dtype=torch.int64))
    refused("positions must", positions=torch.zeros(2, 2, dtype=torch.int32))
    for kw in (dict(rows=0), dict(rotary_dim=24), dict(rotary_dim=272), dict(scaling="x"), dict(factor=0.0, scaling="linear"), dict(device="cpu")):
        with pytest.raises(errors):
            m.rotary_tables(**{**dict(rows=4, rotary_dim=32, device="cuda"), **kw})


# ---- on the GPU ----

@pytest.mark.gpu
@pytest.mark.parametrize("rows,dims", [(1, 16), (7, 32), (1000, 48), (4099, 128), (131072, 64), (300, 256)])
@pytest.mark.parametrize("n", range(len(SCALINGS)))
def test_tables_are_the_oracles(gpu, rows, dims, n):
    how = SCALINGS[n]
    f = ro.frequencies(dims, **{key: value for key, value in how.items() if key != "amplitude"})
    want = ro.tables(rows, dims, **how)
    amplitude = how.get("amplitude", 1.0)
    for m in (_module(), capi):
        for got, w in zip(m.rotary_tables(rows, dims, gpu, **how), want):
            assert got.dtype == torch.float32 and tuple(got.shape) == (rows, dims // 2) and got.device == gpu
            tol = amplitude * (np.arange(rows)[:, None] * f[None] * 2.0 ** -51 + 1e-11) + np.abs(w) * 2.0 ** -24 + 2.0 ** -149
            assert (np.abs(got.cpu().numpy().astype(np.float64) - w) <= tol).all()


def _case(dtype, B, L, R, Rkv, H, layout, seed=0):
    g = torch.Generator().manual_seed(seed)
    both = torch.randn(B, L, (R + Rkv) * H, generator=g).to(dtype)
    q, k = both[..., :R * H], both[..., R * H:]                    # slices of one projection
    if layout == "bhld":
        return tuple(x.reshape(B, L, -1, H).transpose(1, 2) for x in (q, k))
    return q, k


def _by_token(x, H, layout):
    return x.reshape(x.shape[0], x.shape[1], -1, H) if layout == "blf" else x.transpose(1, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,dims,first", [(16, 16, 0), (64, 64, 0), (64, 32, 32), (128, 64, 0), (128, 32, 48), (192, 64, 128), (48, 32, 8), (1024, 256, 512)])
@pytest.mark.parametrize("interleaved,inverse", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("layout", ["blf", "bhld"])
def test_rotation_is_the_oracles(gpu, dtype, H, dims, first, interleaved, inverse, layout):
    B, L, R, Rkv = 3, 5, 6, 1
    q, k = _case(dtype, B, L, R, Rkv, H, layout)
    cos, sin = (torch.from_numpy(x).float() for x in ro.tables(40, dims))
    starts, lens = torch.tensor([0, 37, -2], dtype=torch.int32), torch.tensor([5, 9, 3], dtype=torch.int32)
    at = starts[:, None] + torch.arange(L)
    exists = torch.arange(L)[None] < lens[:, None]
    kw = dict(first=first, interleaved=interleaved, inverse=inverse)
    want = [ro.rotate(_by_token(x, H, layout), cos, sin, at, exists=exists, **kw) for x in (q, k)]
    dq, dk, dc, ds, dst, dl = (x.to(gpu) for x in (q, k, cos, sin, starts, lens))
    m = _module()
    a = m.rotate(dq, dc, ds, H, keys=dk, starts=dst, new_lens=dl, layout=layout, **kw)
    b = capi.rotate(dq, (dc, ds), H, keys=dk, starts=dst, new_lens=dl, layout=layout, **kw)
    positions = at.to(gpu).int().contiguous()
    c = m.rotate(dq, dc, ds, H, keys=dk, positions=positions, new_lens=dl, layout=layout, **kw)
    own_q, own_k = dq.clone(), dk.clone()
    d = m.rotate(own_q, dc, ds, H, keys=own_k, starts=dst, new_lens=dl, layout=layout, in_place=True, **kw)
    assert d[0].data_ptr() == own_q.data_ptr() and d[1].data_ptr() == own_k.data_ptr()
    for got in (a, b, c, d):
        for x, w in zip(got, want):
            assert torch.equal(_by_token(x.cpu(), H, layout), w)
    alone = m.rotate(dq, dc, ds, H, layout=layout, **kw)           # queries alone, positions from 0
    assert torch.equal(_by_token(alone.cpu(), H, layout), ro.rotate(_by_token(q, H, layout), cos, sin, torch.arange(L).expand(B, L), **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,R,Rkv,H", [(2, 700, 40, 8, 128), (1, 1, 1, 1, 64), (64, 1, 40, 8, 128), (1, 20000, 8, 8, 64)])
def test_rotation_of_many_rows(gpu, B, L, R, Rkv, H):
    # the kernel that takes four heads a thread, and the largest and smallest calls
    q, k = _case(BF16, B, L, R, Rkv, H, "blf", seed=3)
    cos, sin = (torch.from_numpy(x).float() for x in ro.tables(L + 100, H))
    starts = torch.arange(B, dtype=torch.int32)
    at = starts[:, None] + torch.arange(L)
    got = _module().rotate(q.to(gpu), cos.to(gpu), sin.to(gpu), H, keys=k.to(gpu), starts=starts.to(gpu))
    for x, y in zip(got, (q, k)):
        assert torch.equal(_by_token(x.cpu(), H, "blf"), ro.rotate(_by_token(y, H, "blf"), cos, sin, at))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,layout,interleaved,inverse,first,dims", [(F16, "blf", False, True, 40, 64), (BF16, "bhld", True, False, 0, 128), (F16, "bhld", True, True, 96, 32),
                                                                         (BF16, "blf", False, False, 24, 96)])
def test_rotation_of_four_heads_a_thread(gpu, dtype, layout, interleaved, inverse, first, dims):
    # enough heads of 16 channels that a thread takes four of them; head counts that are no multiple of it, copied channels, absent tokens, in place
    B, L, R, Rkv, H = 2, 4100, 37, 6, 128
    assert B * L * (R + Rkv) * (H // 16) >= 4 * 2048 * 256
    q, k = _case(dtype, B, L, R, Rkv, H, layout, seed=dims)
    cos, sin = (torch.from_numpy(x).float() for x in ro.tables(4096, dims))
    starts, lens = torch.tensor([-3, 70], dtype=torch.int32), torch.tensor([4100, 3001], dtype=torch.int32)
    exists = torch.arange(L)[None] < lens[:, None]
    kw = dict(first=first, interleaved=interleaved, inverse=inverse)
    want = [ro.rotate(_by_token(x, H, layout), cos, sin, starts[:, None] + torch.arange(L), exists=exists, **kw) for x in (q, k)]
    dq, dk, dc, ds, dst, dl = (x.to(gpu) for x in (q, k, cos, sin, starts, lens))
    m = _module()
    calls = [m.rotate(dq, dc, ds, H, keys=dk, starts=dst, new_lens=dl, layout=layout, **kw),
             capi.rotate(dq, (dc, ds), H, keys=dk, starts=dst, new_lens=dl, layout=layout, **kw),
             m.rotate(dq, dc, ds, H, keys=dk, starts=dst, new_lens=dl, layout=layout, in_place=True, **kw)]
    for got in calls:
        for x, w in zip(got, want):
            assert torch.equal(_by_token(x.cpu(), H, layout), w)


@pytest.mark.gpu
def test_rotation_is_the_caches(gpu):
    # the same tables give the same queries as appending to the 8-bit cache does
    m = _module()
    B, L, R, Rkv, H, P = 2, 7, 4, 2, 64, 16
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(B, L, h * H, generator=g).to(BF16).to(gpu) for h in (R, Rkv, Rkv))
    cos, sin = m.rotary_tables(64, H, gpu, scaling="turns", factor=4.0, original_rows=16.0)
    starts = torch.tensor([3, 20], dtype=torch.int32, device=gpu)
    cache = [torch.zeros(8, Rkv, P, H, dtype=torch.float8_e4m3fn, device=gpu) for _ in range(2)]
    cache += [torch.zeros(8, Rkv, dtype=torch.int8, device=gpu) for _ in range(2)]
    table = torch.arange(4, dtype=torch.int32, device=gpu).view(B, 2)
    want = m.cache_append(k, v, *cache, table, starts, queries=q, rope_cos=cos, rope_sin=sin)
    assert torch.equal(m.rotate(q, cos, sin, H, keys=k, starts=starts)[0], want)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_the_gradient_is_the_rotation_back(gpu, interleaved):
    # d/dx sum(w * rotate(x)) = rotate back of w: against differences of the oracle in 64 bits, half a step (2^-11) and the tables' 2^-24
    m = _module()
    B, L, H, D, first = 1, 3, 64, 32, 16
    g = torch.Generator().manual_seed(6)
    x, w = (torch.randn(B, L, 2, H, generator=g).to(F16) for _ in range(2))
    cos, sin = m.rotary_tables(50, D, gpu)
    starts = torch.tensor([41], dtype=torch.int32, device=gpu)
    got = m.rotate(w.flatten(2).to(gpu), cos, sin, H, starts=starts, first=first, interleaved=interleaved, inverse=True).cpu().view(B, L, 2, H)
    c, s = (t.cpu().double()[41:44][None, :, None] for t in (cos, sin))

    def f(y):
        part = y[..., first:first + D]
        a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :D // 2], part[..., D // 2:])
        a, b = a * c - b * s, b * c + a * s
        turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
        return (torch.cat([y[..., :first], turned, y[..., first + D:]], -1) * w.double()).sum()

    y = x.double()
    for at in [(0, 0, 0, 3), (0, 1, 1, 16), (0, 2, 0, 31), (0, 1, 1, 32), (0, 2, 1, 47), (0, 0, 0, 63)]:
        e = torch.zeros_like(y)
        e[at] = 0.5
        want = f(y + e) - f(y - e)                                 # linear: exact but for rounding in 64 bits
        assert abs(got[at].double() - want) <= want.abs() * 2.0 ** -11 + 4 * 2.0 ** -24 * 8 + 2.0 ** -25
    leaf = y.clone().requires_grad_()
    f(leaf).backward()
    assert ((got.double() - leaf.grad).abs() <= leaf.grad.abs() * 2.0 ** -11 + 4 * 2.0 ** -24 * 8 + 2.0 ** -25).all()


@pytest.mark.gpu
def test_rotation_in_place_of_views_of_one_tensor(gpu):
    m = _module()
    B, L, H = 2, 5, 64
    both = torch.randn(B, L, 8 * H, generator=torch.Generator().manual_seed(9)).to(BF16).to(gpu)
    cos, sin = m.rotary_tables(16, H, gpu)
    want_q, want_k = m.rotate(both[..., :4 * H], cos, sin, H, keys=both[..., 4 * H:6 * H])
    kept = both.clone()
    for call in (lambda q, k: m.rotate(q, cos, sin, H, keys=k, in_place=True), lambda q, k: capi.rotate(q, (cos, sin), H, keys=k, out=(q, k))):
        for q, k in ((both, both), (both[..., :4 * H], both[..., 3 * H:5 * H]), (both[:, 1:], both[:, :-1])):
            with pytest.raises(RuntimeError, match="stride"):
                call(q, k)
        assert torch.equal(both, kept)
        call(both[..., :4 * H], both[..., 4 * H:6 * H])
        assert torch.equal(both[..., :4 * H], want_q) and torch.equal(both[..., 4 * H:6 * H], want_k) and torch.equal(both[..., 6 * H:], kept[..., 6 * H:])
        both.copy_(kept)
    with pytest.raises(RuntimeError, match="stride"):              # each other's place
        capi.rotate(both[..., :2 * H], (cos, sin), H, keys=both[..., 2 * H:4 * H], out=(both[..., 2 * H:4 * H], both[..., :2 * H]))
    assert torch.equal(both, kept)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["module", "capi"])
def test_autograd_sees_a_rotation_in_place(gpu, how):
    cos, sin = capi.rotary_tables(8, 64, gpu)

    def rotate(q, k, in_place):
        if how == "module":
            return _module().rotate(q, cos, sin, 64, keys=k, in_place=in_place)
        return capi.rotate(q, (cos, sin), 64, keys=k, out=(q, k) if in_place else None)

    w = torch.ones(1, 4, 192, dtype=F16, device=gpu, requires_grad=True)
    both = torch.randn(1, 4, 192, generator=torch.Generator().manual_seed(2)).to(F16).to(gpu)
    y = (w * both).float().sum()                                   # keeps `both` for the backward pass
    versions = both._version
    rotate(both[..., :128], both[..., 128:], False)
    assert both._version == versions
    rotate(both[..., :128], both[..., 128:], True)
    assert both._version > versions
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        kept = both.clone()
        rotate(kept[..., :128], kept[..., 128:], True)             # has no version
    assert torch.equal(kept[..., :128], rotate(both[..., :128], both[..., 128:], False)[0])


@pytest.mark.gpu
def test_a_function_with_the_rotation_back_as_its_gradient(gpu):
    # as a caller has it, in place of its input too: the gradient of both is that of the rotation written out
    m = _module()
    cos, sin = m.rotary_tables(8, 64, gpu)

    class Rotate(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, in_place):
            if in_place:
                ctx.mark_dirty(x)
            return m.rotate(x, cos, sin, 64, in_place=in_place)

        @staticmethod
        def backward(ctx, g):
            return m.rotate(g.contiguous(), cos, sin, 64, inverse=True), None

    g = torch.Generator().manual_seed(3)
    x, w = (torch.randn(2, 5, 128, generator=g).to(BF16).to(gpu) for _ in range(2))
    want = m.rotate(w, cos, sin, 64, inverse=True)
    for in_place in (False, True):
        leaf = x.clone().requires_grad_()
        out = Rotate.apply(leaf * 1, in_place)
        assert torch.equal(out, m.rotate(x, cos, sin, 64))
        out.backward(w)
        assert torch.equal(leaf.grad, want)


@pytest.mark.gpu
def test_rotation_captured_and_on_another_stream(gpu):
    m = _module()
    q, k = (x.to(gpu) for x in _case(F16, 2, 3, 4, 2, 64, "blf", seed=8))
    starts = torch.tensor([3, 9], dtype=torch.int32, device=gpu)
    side = torch.cuda.Stream(device=gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        cos, sin = m.rotary_tables(64, 64, gpu)
        want = m.rotate(q, cos, sin, 64, keys=k, starts=starts)
    torch.cuda.current_stream(gpu).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tables = m.rotary_tables(64, 64, gpu)
        out = m.rotate(q, *tables, 64, keys=k, starts=starts)
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = m.rotate(q, cos, sin, 64, keys=k, starts=starts)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        starts += 5
        q.mul_(0.5)
