"""Keeping the pages of a cache: closed forms of the oracle and the refusals on the CPU; on the GPU every operation against the oracle.
Whole numbers and copies: everything is compared for equality.
"""
import ctypes
import random

import pytest
import torch

from fused_attention_amd import capi
from oracle.pages import Keeper

I32 = torch.int32


def _module():
    import fused_attn

    return fused_attn


def _ints(x, dev="cpu"):
    return torch.tensor(x, dtype=I32, device=dev)


# ---- the oracle, on the CPU ----

def test_operations_of_the_oracle():
    k = Keeper([[4, 2, -1], [-1, -1, -1], [5, -1, -1]], [20, 0, 16], [0, 0, 1, 0, 1, 1], 16)
    assert k.check()
    assert k.fork([0], [1]) == [1]
    assert k.table[1] == [4, 0, -1] and k.starts == [20, 20, 16] and k.uses == [1, 0, 1, 0, 2, 1] and k.holds[0] == 2 and k.check()
    assert k.take([30, 0, 1], 30) == [1, 0, 0]                     # places 2 and 3, of which the table has one
    assert k.table == [[4, 2, 1], [4, 0, -1], [5, 3, -1]] and k.check()
    k.free([0])
    assert k.uses == [1, 0, 0, 1, 1, 1] and k.table[0] == [-1, -1, -1] and k.starts[0] == 0 and k.check()
    assert k.compact() == [0, -1, -1, 3, 1, 2]
    assert k.table == [[-1, -1, -1], [1, 0, -1], [2, 3, -1]] and k.uses == [1, 1, 1, 1, 0, 0] and k.holds[:4] == [2, 4, 5, 3] and k.check()
    assert k.fork([1, 1, 0, 9, 2, 1], [0, 0, 0, 0, 2, 1]) == [1, 0, 0, 0, 0, 0]
    k.copy([0, 99], [5, 0])
    assert k.holds[5] == 2 and k.holds[0] == 2


def test_a_fork_of_a_sequence_without_tokens_in_the_oracle():
    # the child goes on from nothing, and what its row named before is given back
    k = Keeper([[-1, -1], [3, 1], [0, -1]], [0, 0, -5], [1, 1, 0, 1], 16)
    assert k.fork([0, 2], [1, 0]) == [1, 1]
    assert k.table == [[-1, -1], [-1, -1], [0, -1]] and k.uses == [1, 0, 0, 0] and k.starts == [0, 0, -5] and k.check()


# ---- refusals, on the CPU ----

def test_the_library_refuses_what_its_header_says():
    lib, ok = capi.load_library(), 0x1000                          # never dereferenced: every case is refused before a launch

    def pages(**kw):
        c = capi.Pages(**{**dict(page_table=ok, starts=ok, uses=ok, pages=10, page_size=16, sequences=3, table_width=4, table_stride=4, tensors=1),
                          **{key: value for key, value in kw.items() if key not in ("data", "page_bytes")}})
        c.data[0], c.page_bytes[0] = kw.get("data", ok), kw.get("page_bytes", 32)
        return ctypes.byref(c)

    def copy(c=None, a=ok, b=ok, n=2):
        return lib.fa_copy_pages(pages() if c is None else c, a, b, n, None)

    def free(c=None, a=ok, n=2):
        return lib.fa_free_pages(pages() if c is None else c, a, n, None)

    def take(c=None, lens=None, L=2, missing=ok, ws=ok, size=40):
        return lib.fa_take_pages(pages() if c is None else c, lens, L, missing, ws, size, None)

    def fork(c=None, a=ok, b=ok, n=2, forked=ok, ws=ok, size=24):
        return lib.fa_fork_pages(pages() if c is None else c, a, b, n, forked, ws, size, None)

    def compact(c=None, moved=ok, ws=ok, size=56):
        return lib.fa_compact_pages(pages() if c is None else c, moved, ws, size, None)

    for call in (free, take, fork, compact):
        for name in ("pages", "sequences", "table_width"):
            assert call(c=pages(**{name: 0})) == -3, name
        assert call(c=pages(table_stride=3)) == -4 and call(c=pages(table_stride=-1, sequences=1)) == -4
        assert call(c=pages(page_table=None)) == -1 and call(c=pages(uses=None)) == -1
        assert call(c=pages(page_table=ok + 2)) == -5 and call(c=pages(uses=ok + 1)) == -5
        assert call(c=pages(pages=2 ** 31)) == -6 and call(c=pages(sequences=2 ** 31)) == -6 and call(c=pages(table_width=2 ** 25, table_stride=2 ** 25)) == -6
    for call in (free, take, fork):
        assert [call(c=pages(page_size=n)) for n in (0, 8, 24, 256)] == [-9] * 4
        assert call(c=pages(starts=None)) == -1 and call(c=pages(starts=ok + 2)) == -5
    for call in (copy, fork, compact):
        assert call(c=pages(tensors=0)) == -3 and call(c=pages(tensors=9)) == -6 and call(c=pages(data=None)) == -1 and call(c=pages(page_bytes=0)) == -3
        assert call(c=pages(page_bytes=2 ** 41)) == -6
    assert lib.fa_copy_pages(None, ok, ok, 1, None) == -1 and lib.fa_free_pages(None, ok, 1, None) == -1
    assert copy(a=None) == -1 and copy(b=None) == -1 and copy(a=ok + 1) == -5 and copy(n=-1) == -3 and copy(n=0) == 0
    assert free(a=None) == -1 and free(a=ok + 2) == -5 and free(n=-1) == -3 and free(n=65537) == -6 and free(n=0) == 0
    assert take(L=0) == -3 and take(L=2 ** 31) == -6 and take(missing=None) == -1 and take(missing=ok + 2) == -5 and take(lens=ok + 2) == -5
    assert take(ws=None) == -10 and take(size=39) == -10 and take(ws=ok + 4) == -5
    assert fork(a=None) == -1 and fork(b=None) == -1 and fork(forked=None) == -1 and fork(n=-1) == -3 and fork(n=4097) == -6 and fork(n=0) == 0
    assert fork(ws=None) == -10 and fork(size=23) == -10 and fork(ws=ok + 8) == -5
    assert compact(moved=None) == -1 and compact(moved=ok + 1) == -5 and compact(ws=None) == -10 and compact(size=55) == -10 and compact(ws=ok + 8) == -5
    assert lib.fa_take_pages_workspace(pages()) == 40 and lib.fa_compact_pages_workspace(pages()) == 56 and lib.fa_fork_pages_workspace(2) == 24
    assert lib.fa_take_pages_workspace(pages(pages=0)) == -3 and lib.fa_fork_pages_workspace(-1) == -3 and lib.fa_fork_pages_workspace(5000) == -6


@pytest.mark.parametrize("S,W", [(140000, 16384), (1 << 20, 2048), (1 << 16, 32767)])
def test_tables_whose_places_32_bits_cannot_count(S, W):
    # refused from the sizes alone; 2^31 - 2^16 - 1 places are the most
    ok = 0x1000
    c = capi.Pages(page_table=ok, starts=ok, uses=ok, pages=10, page_size=16, sequences=S, table_width=W, table_stride=W)
    assert S * W >= 2 ** 31 - 2 ** 16
    assert capi.load_library().fa_take_pages(ctypes.byref(c), None, 1, ok, ok, 40, None) == -6


@pytest.mark.parametrize("how", ["module", "capi"])
def test_the_entry_points_refuse_wrong_tensors(how):
    m = _module() if how == "module" else capi
    errors = RuntimeError if how == "module" else (ValueError, TypeError)
    t = dict(page_table=torch.full((3, 4), -1, dtype=I32), starts=torch.zeros(3, dtype=I32), uses=torch.zeros(10, dtype=I32))
    data, two = [torch.zeros(10, 4)], _ints([0, 1])
    calls = {
        "copy": lambda tensors=data, sources=two, targets=two, **kw: m.copy_pages(tensors, sources, targets),
        "free": lambda sequences=two, **kw: m.free_pages(**{**t, **{key: kw[key] for key in t if key in kw}}, sequences=sequences),
        "take": lambda page_size=16, seq_len=2, new_lens=None, **kw: m.take_pages(**{**t, **{key: kw[key] for key in t if key in kw}}, page_size=page_size,
                                                                                   seq_len=seq_len, new_lens=new_lens),
        "fork": lambda tensors=data, page_size=16, parents=two, children=two, **kw: m.fork_pages(
            tensors, **{**t, **{key: kw[key] for key in t if key in kw}}, page_size=page_size, parents=parents, children=children),
        "compact": lambda tensors=data, **kw: m.compact_pages(tensors, kw.get("page_table", t["page_table"]), kw.get("uses", t["uses"])),
    }

    def refused(match, which, **kw):
        for name in which:
            with pytest.raises(errors, match=match):
                calls[name](**kw)

    refused("GPU", calls)
    keeping = ("free", "take", "fork", "compact")
    refused("uses must be", keeping, uses=t["uses"].long())
    refused("uses must", keeping, uses=t["uses"][:0])
    refused("page_table must be", keeping, page_table=t["page_table"].long())
    refused("page_table must be", keeping, page_table=t["page_table"].t())
    refused("starts must", keeping[:3], starts=t["starts"][:2])
    refused("page_size must be", ("take", "fork"), page_size=24)
    refused("seq_len must be", ("take",), seq_len=0)
    refused("new_lens must", ("take",), new_lens=two)
    tensors = ("copy", "fork", "compact")
    refused("tensors must be one to eight", tensors, tensors=[])
    refused("tensors must be one to eight", tensors, tensors=data * 9)
    refused("tensors must be contiguous", tensors, tensors=[torch.zeros(4, 10).t()])
    refused("same pages", tensors, tensors=data + [torch.zeros(9, 4)])
    refused("targets must be as many", ("copy",), targets=_ints([0]))
    refused("children must be as many", ("fork",), children=_ints([0]))
    refused("at most 4096", ("fork",), parents=torch.zeros(4097, dtype=I32), children=torch.zeros(4097, dtype=I32))
    refused("sequences must", ("free",), sequences=two.long())
    refused("sources must", ("copy",), sources=two.long())


# ---- on the GPU ----

class Both:
    """A page table, its counts and a cache's tensors on the GPU, and the oracle beside them."""

    def __init__(self, dev, S, W, N, P, seed, shapes=((16, torch.float16),), stride=0):
        self.rng, self.dev, self.P, self.S, self.W, self.N = random.Random(seed), dev, P, S, W, N
        self.k = Keeper([[-1] * W for _ in range(S)], [0] * S, [0] * N, P)
        g = torch.Generator().manual_seed(seed)
        self.first = [torch.randint(-100, 100, (N,) + (n if isinstance(n, tuple) else (n,)), generator=g).to(dtype) for n, dtype in shapes]
        self.tensors = [x.to(dev) for x in self.first]
        self.table = torch.full((S, W + stride), -1, dtype=I32, device=dev)[:, :W]
        self.starts = torch.zeros(S, dtype=I32, device=dev)
        self.uses = torch.zeros(N, dtype=I32, device=dev)

    def check(self):
        assert self.k.check()
        assert self.table.tolist() == self.k.table
        assert self.starts.tolist() == self.k.starts and self.uses.tolist() == self.k.uses
        holds = torch.tensor(self.k.holds)
        for x, first in zip(self.tensors, self.first):
            assert torch.equal(x.cpu().view(torch.uint8), first[holds].view(torch.uint8))

    def step(self, m, op):
        r, k = self.rng, self.k
        rows = lambda n: [r.randrange(-1, self.S + 1) for _ in range(n)]
        args = (self.table, self.starts, self.uses)
        if op == "take":
            lens = [r.choice([0, 0, 1, r.randrange(-2, 3 * self.P)]) for _ in range(self.S)]
            got = m.take_pages(*args, self.P, 2 * self.P + 3, _ints(lens, self.dev))
            assert got.tolist() == k.take(lens, 2 * self.P + 3)
            grown = [min(max(n, 0), 2 * self.P + 3) for n in lens]
            self.starts += _ints(grown, self.dev)
            k.starts = [a + b for a, b in zip(k.starts, grown)]
        elif op == "free":
            which = rows(r.randrange(1, 5))
            m.free_pages(*args, _ints(which, self.dev))
            k.free(which)
        elif op == "fork":
            n = r.randrange(1, 6)
            a, b = rows(n), rows(n)
            assert m.fork_pages(self.tensors, *args, self.P, _ints(a, self.dev), _ints(b, self.dev)).tolist() == k.fork(a, b)
        elif op == "compact":
            assert m.compact_pages(self.tensors, self.table, self.uses).tolist() == k.compact()
        else:                                                      # from used pages into free ones and back: no target twice, none a source
            pages = list(range(-2, self.N + 2))
            r.shuffle(pages)
            n = r.randrange(1, len(pages) // 2)
            a, b = [r.choice(pages[n:]) for _ in range(n)], pages[:n]
            m.copy_pages(self.tensors, _ints(a, self.dev), _ints(b, self.dev))
            k.copy(a, b)
        self.check()


SHAPES = {
    "latent": (((16, 160), torch.float16),),
    "8bit": (((3, 16, 16), torch.int8), ((3, 16, 16), torch.int8), (3, torch.int8), (3, torch.int8), ((3, 2, 16), torch.int8)),   # pages of 3 bytes
    "odd": ((1, torch.int8), (2, torch.int16), (3, torch.float32), ((2, 5000), torch.int16), (20001, torch.int8)),
}


@pytest.mark.gpu
@pytest.mark.parametrize("S,W,N,P,stride", [(6, 5, 24, 16, 0), (1, 1, 1, 128, 0), (2, 3, 7, 32, 3), (40, 9, 150, 64, 1)])
@pytest.mark.parametrize("kind", list(SHAPES))
@pytest.mark.parametrize("how", ["module", "capi"])
def test_a_server_at_work(gpu, S, W, N, P, stride, kind, how):
    # every operation in a random order, with lists that name what does not exist, twice or itself, and pages that run out
    both = Both(gpu, S, W, N, P, seed=S + N, shapes=SHAPES[kind], stride=stride)
    m = _module() if how == "module" else capi
    for _ in range(40):
        both.step(m, both.rng.choice(["take", "take", "take", "free", "fork", "fork", "compact", "copy"] if N > 4 else ["take", "free", "fork", "compact"]))


@pytest.mark.gpu
def test_more_pages_and_sequences_than_threads(gpu):
    # the plans go through 4096 pages, and 1024 sequences or forks, at a time
    both = Both(gpu, 2500, 3, 9001, 16, seed=9, shapes=(((8,), torch.float16),))
    m = _module()
    for op in ("take", "take", "free", "fork", "take", "compact", "fork", "take"):
        both.step(m, op)
    k, S = both.k, both.S
    parents, children = [n % 7 for n in range(2400)], [S - 1 - n for n in range(2400)]
    m.free_pages(both.table, both.starts, both.uses, _ints(children[:2000] * 2, gpu))
    k.free(children[:2000])
    got = m.fork_pages(both.tensors, both.table, both.starts, both.uses, 16, _ints(parents, gpu), _ints(children, gpu))
    assert got.tolist() == k.fork(parents, children)
    both.check()
    both.step(m, "compact")


@pytest.mark.gpu
@pytest.mark.parametrize("N,enough", [(9001, True), (5000, False)])
@pytest.mark.parametrize("how", ["module", "capi"])
def test_more_pages_taken_at_once_than_stay_in_a_workgroup(gpu, N, enough, how):
    # above 2048 wanted pages the free ones are listed in the workspace: with enough of them, and running out in the middle of a row
    both = Both(gpu, 2500, 3, N, 16, seed=N, shapes=(((8,), torch.float16),))
    m = _module() if how == "module" else capi
    held = list(range(0, N, 7))[:300]                              # some pages are somebody's already
    for n, page in enumerate(held):
        both.k.table[8 * n][0], both.k.uses[page] = page, 1
    both.table.copy_(_ints(both.k.table))
    both.uses.copy_(_ints(both.k.uses))
    lens = [17 + n * 7 % 24 for n in range(2500)]
    wanted = sum(-(-n // 16) - (s % 8 == 0 and s // 8 < len(held)) for s, n in enumerate(lens))
    assert wanted > 2048 and (wanted <= N - len(held)) == enough
    got = m.take_pages(both.table, both.starts, both.uses, 16, 40, _ints(lens, gpu))
    assert got.tolist() == both.k.take(lens, 40) and (int(got.sum()) == 0) == enough
    both.check()
    more = m.take_pages(both.table, both.starts, both.uses, 16, 48)      # places that stayed empty, and one more of many rows
    assert more.tolist() == both.k.take([48] * 2500, 48)
    both.check()


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["module", "capi"])
def test_a_fork_of_a_sequence_without_tokens(gpu, how):
    # its child's row is cleared as any child's is, and pages that were taken for it, or that it shares, lose the use
    m = _module() if how == "module" else capi
    both = Both(gpu, 6, 4, 30, 16, seed=5)
    k, args = both.k, (both.table, both.starts, both.uses)
    lens = [0, 40, 17, 33, 0, 20]
    assert m.take_pages(*args, 16, 40, _ints(lens, gpu)).tolist() == k.take(lens, 40)
    both.starts[5] = k.starts[5] = 20                              # of those with pages only the last one gets tokens
    both.starts[4] = k.starts[4] = -7
    both.table[3, 3], k.table[3][3] = both.table[5, 0], k.table[5][0]
    both.uses[k.table[5][0]] += 1
    k.uses[k.table[5][0]] += 1
    both.check()
    parents, children = [0, 4, 5, 1], [1, 3, 2, 0]
    assert m.fork_pages(both.tensors, *args, 16, _ints(parents, gpu), _ints(children, gpu)).tolist() == k.fork(parents, children) == [1, 1, 1, 1]
    assert both.table[1].tolist() == [-1] * 4 and both.table[3].tolist() == [-1] * 4 and int((both.uses > 0).sum()) == 3 and int(both.uses.sum()) == 4
    both.check()


@pytest.mark.gpu
def test_lists_of_nothing_and_pages_beyond_32_bits(gpu):
    m = _module()
    both = Both(gpu, 3, 3, 6, 16, seed=2)
    none = torch.zeros(0, dtype=I32, device=gpu)
    for m in (_module(), capi):
        m.copy_pages(both.tensors, none, none)
        m.free_pages(both.table, both.starts, both.uses, none)
        assert m.fork_pages(both.tensors, both.table, both.starts, both.uses, 16, none, none).numel() == 0
        both.check()
    big = torch.zeros(2100, 1 << 20, dtype=torch.int16, device=gpu)       # pages of 2 MiB: the last ones lie behind 4 GiB
    big[7] = torch.arange(1 << 20, device=gpu) % 30011
    m.copy_pages([big], _ints([7, 2099], gpu), _ints([2098, 0], gpu))
    assert torch.equal(big[2098], big[7]) and int(big[2097].abs().max()) == 0 and int(big[2099].abs().max()) == 0
    uses = torch.zeros(2100, dtype=I32, device=gpu)
    uses[2098] = 3
    table = _ints([[2098, 5]], gpu)
    moved = m.compact_pages([big], table, uses)
    assert torch.equal(big[0], big[7]) and table.tolist() == [[0, -1]] and int(moved[2098]) == 0 and int((moved >= 0).sum()) == 1 and int(uses[0]) == 3


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["module", "capi"])
def test_pages_of_more_tensors_than_a_call_takes(gpu, how):
    # the layers of a model: the first eight tensors go with the table, the others follow by copies
    m = _module() if how == "module" else capi
    P, S, W = 16, 14, 5
    both = Both(gpu, S, W, 60, P, seed=6, shapes=(((16, 24), torch.float16), (7, torch.int8)) * 10)
    k, args, rng = both.k, (both.table, both.starts, both.uses), random.Random(3)
    everything = torch.arange(both.N, dtype=I32, device=gpu)
    groups = [both.tensors[n:n + 8] for n in range(8, len(both.tensors), 8)]
    assert [len(g) for g in groups] == [8, 4]
    copied = 0
    for turn in range(12):
        gone = [rng.randrange(S) for _ in range(4)]
        m.free_pages(*args, _ints(gone, gpu))
        k.free(gone)
        moved = m.compact_pages(both.tensors[:8], both.table, both.uses)
        assert moved.tolist() == k.compact()
        for rest in groups:
            m.copy_pages(rest, everything, moved)
        both.check()
        lens = [rng.choice([0, 16, 23, 48]) if n % 2 else 0 for n in range(S)]
        m.take_pages(*args, P, 48, _ints(lens, gpu))
        k.take(lens, 48)
        both.starts += _ints(lens, gpu)
        k.starts = [a + b for a, b in zip(k.starts, lens)]
        parents, children = [_ints([rng.randrange(S) for _ in range(9)], gpu) for _ in range(2)]
        ok = m.fork_pages(both.tensors[:8], *args, P, parents, children)
        assert ok.tolist() == k.fork(parents.tolist(), children.tolist())
        tokens = both.starts[parents]
        place = (tokens // P).clamp(max=both.table.shape[1] - 1)
        last, copy = both.table[parents, place], both.table[children, place]
        copy = torch.where((ok == 1) & (tokens % P != 0), copy, -1)
        copied += int(((copy >= 0) & (last >= 0)).sum())
        for rest in groups:
            m.copy_pages(rest, last, copy)
        both.check()
    assert copied > 5


@pytest.mark.gpu
def test_a_turn_captured_in_a_graph(gpu):
    # a turn of a server, replayed: the lists' and the table's contents decide, as the host's steps do
    m = _module()
    both = Both(gpu, 8, 6, 40, 16, seed=4, shapes=SHAPES["8bit"])
    k = both.k
    lens, gone = _ints([0] * 8, gpu), _ints([7, 7], gpu)
    parents, children = _ints([0, 0], gpu), _ints([7, 7], gpu)

    def turn():
        m.free_pages(both.table, both.starts, both.uses, gone)
        moved = m.compact_pages(both.tensors, both.table, both.uses)
        missing = m.take_pages(both.table, both.starts, both.uses, 16, 40, lens)
        both.starts.add_(lens)
        return moved, missing, m.fork_pages(both.tensors, both.table, both.starts, both.uses, 16, parents, children)

    def host():
        k.free(gone.tolist())
        moved = k.compact()
        missing = k.take(lens.tolist(), 40)
        k.starts = [a + b for a, b in zip(k.starts, lens.tolist())]
        return moved, missing, k.fork(parents.tolist(), children.tolist())

    side = torch.cuda.Stream(device=gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        turn()
    torch.cuda.current_stream(gpu).wait_stream(side)
    host()
    both.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = turn()
    rng = random.Random(1)
    for _ in range(8):
        lens.copy_(_ints([rng.choice([0, 1, 17, 40]) for _ in range(8)]))
        gone.copy_(_ints([rng.randrange(8), rng.randrange(8)]))
        parents.copy_(_ints([rng.randrange(8), rng.randrange(8)]))
        children.copy_(gone)
        want = host()
        graph.replay()
        torch.cuda.synchronize()
        assert [x.tolist() for x in out] == [list(x) for x in want]
        both.check()
