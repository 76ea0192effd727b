"""What a program that answers with a model asks for besides plain attention and the 8-bit cache: rotary positions of every kind,
the dealing out, sharing and moving of a cache's pages, and attention whose keys and values come from one latent vector a token.

`listed()` names twelve calls, `draw(rng)` gives more from the same ranges; `prepare` makes the tensors that a program holds
before the call, `run` is one call (or the calls of one step) and `work` the bytes and operations it cannot do without.
`run` makes the module's calls where `own` is true; otherwise it computes the same from elementary operations in 32 bits (angles
of positions in 64). `exact` has the same results from the definitions in 64 bits, or whole numbers on the host.

Keys of a case:
  op       "rotate" (queries and keys rotated by their positions), "tables_rotate" (the tables made first), "pages" (a turn of a
           server's page keeping, see _pages_turn), "append" (rotate and append to the latent cache), "attend" (the absorbed form
           over the latent cache), "step" (append, then attend) or "expanded" (attention with keys and values of each head)
  B L      sequences, and new tokens of each: 1 for an answer's next token, a few for drafted ones, many for a prompt
  R        query heads
  dtype    "fp16" or "bf16"
  ragged   sequences are shorter than the longest, down to half of it, and bring fewer new tokens
  rotate:   Rkv H  key heads, head_dim; D first  channels first .. first + D of a head are rotated; interleaved: channels 2j and
            2j + 1 are a pair, otherwise j and j + D/2; scaling, factor: how frequencies are scaled for long contexts; ctx:
            positions in the tables; inverse: rotated back (the gradient); layout as elsewhere ("blf", "bhld")
  pages:    kind "latent" (one tensor, [pages, P, C + Dr]) or "8bit" (five, Rkv heads of H); n prompts and c forks of them in each
            of two halves, ctx tokens of the longest, P tokens of a page
  latent:   C Dr   channels of the latent and of the rotary key; Dn  channels of a query that stand before its rotary ones;
            P ctx  tokens of a page; tokens of the longest sequence, the new ones among them; lse: returned as well
  expanded: Dn Dr Dv  channels of a head's own keys, of the shared rotary key and of the values; ctx: keys
"""
import math

import torch

own = False

# Pairs of a token and a key times flop: what a drawn case has at most (the largest listed one has 1.2e12), and bytes of a cache.
MOST_FLOPS = 1.0e12
MOST_CACHED = 1 << 30

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_DEVICE = "cuda"


def _rotate_case(name, op, B, L, R, Rkv, H, D, ctx, dtype="fp16", first=0, interleaved=False, scaling="none", factor=1.0, inverse=False,
                 ragged=False, layout="blf"):
    case = {"op": op, "B": B, "L": L, "R": R, "Rkv": Rkv, "H": H, "D": D, "ctx": ctx, "dtype": dtype, "first": first,
            "interleaved": interleaved, "scaling": scaling, "factor": factor, "inverse": inverse, "ragged": ragged, "layout": layout}
    return {**case, "name": name} if name else case


def _pages_case(name, kind, n, c, ctx, P, Rkv=0, H=0, C=0, Dr=0, dtype="fp16"):
    case = {"op": "pages", "kind": kind, "n": n, "c": c, "ctx": ctx, "P": P, "Rkv": Rkv, "H": H, "C": C, "Dr": Dr, "dtype": dtype}
    return {**case, "name": name} if name else case


def _latent_case(name, op, B, L, R, C, Dr, P, ctx, dtype="bf16", Dn=128, ragged=False, interleaved=False, lse=False):
    case = {"op": op, "B": B, "L": L, "R": R, "C": C, "Dr": Dr, "Dn": Dn, "P": P, "ctx": ctx, "dtype": dtype, "ragged": ragged,
            "interleaved": interleaved, "lse": lse}
    return {**case, "name": name} if name else case


def _expanded_case(name, B, L, R, Dn, Dr, ctx, dtype="bf16", ragged=False, lse=False):
    case = {"op": "expanded", "B": B, "L": L, "R": R, "Dn": Dn, "Dr": Dr, "Dv": Dn, "ctx": ctx, "dtype": dtype, "ragged": ragged, "lse": lse}
    return {**case, "name": name} if name else case


def listed():
    return [
        # one answer's next token in a small model, tables at hand: latency
        _rotate_case("rotate_token", "rotate", 1, 1, 4, 4, 64, 64, 256),
        # four prompts of forty 128-wide heads on eight key heads, half of each head rotated in neighbouring pairs, frequencies stretched
        _rotate_case("rotate_prompts", "tables_rotate", 4, 2048, 40, 8, 128, 64, 8192, dtype="bf16", interleaved=True, scaling="turns",
                     factor=8.0, ragged=True),
        # a chunk of a very long document, tables for all of its positions
        _rotate_case("tables_long", "tables_rotate", 1, 2048, 32, 8, 128, 128, 131072, scaling="index", factor=32.0),
        # a turn of page keeping of a small server over its latent cache: latency
        _pages_case("pages_small", "latent", 4, 4, 500, 16, C=128, Dr=32),
        # the same for 32 answers over the 8-bit cache
        _pages_case("pages_cache", "8bit", 16, 8, 8192, 64, Rkv=8, H=128, dtype="fp16"),
        # four long prompts appended to the latent cache, sixteen query heads
        _latent_case("append_prompts", "append", 4, 4096, 16, 512, 64, 64, 4096, interleaved=True),
        # one answer's next token over a short context: latency
        _latent_case("latent_token", "step", 1, 1, 4, 128, 32, 64, 256, dtype="fp16", Dn=64),
        # four drafted tokens of sixteen answers, forty heads, the log-sum-exp kept
        _latent_case("latent_drafted", "step", 16, 4, 40, 512, 64, 32, 2000, ragged=True, interleaved=True, lse=True),
        # the next tokens of 64 answers
        _latent_case("latent_batch", "attend", 64, 1, 16, 512, 64, 64, 8192, ragged=True),
        # the next token over one very long document, many heads
        _latent_case("latent_long", "attend", 1, 1, 128, 512, 64, 128, 131072, dtype="fp16"),
        # short prompts of a padded batch, an odd length, twelve narrow heads, the log-sum-exp kept
        _expanded_case("expanded_prompts", 8, 1001, 12, 64, 32, 1001, dtype="fp16", ragged=True, lse=True),
        # a chunk of a long prompt behind what was expanded before
        _expanded_case("expanded_chunk", 1, 4096, 32, 128, 64, 16384),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "tables_rotate", "pages", "pages", "append", "attend", "attend", "attend", "step", "expanded", "expanded"])
    dtype, ragged = rng.choice(["fp16", "bf16"]), rng.random() < 0.6
    if op in ("rotate", "tables_rotate"):
        H = rng.choice([16, 32, 64, 64, 128, 128])
        D = max(16, rng.choice([H, H, H // 2, H // 4]))
        Rkv = rng.choice([1, 2, 4, 8, 12])
        R = Rkv * rng.choice([1, 1, 2, 4, 5])
        B = _log_int(rng, 1, 64)
        ctx = _log_int(rng, 64, 131072)
        L = 1 if rng.random() < 0.3 else _log_int(rng, 2, 4096)
        L = max(1, min(L, ctx, (1 << 26) // (B * R * H)))
        scaling = rng.choice(["none", "linear", "base", "turns", "index"]) if op == "tables_rotate" else "none"
        return _rotate_case(None, op, B, L, R, Rkv, H, D, ctx, dtype=dtype, first=rng.choice([0, H - D]), interleaved=rng.random() < 0.5,
                            scaling=scaling, factor=1.0 if scaling == "none" else round(rng.uniform(1.5, 40.0), 2),
                            inverse=rng.random() < 0.3, ragged=ragged, layout=rng.choice(["blf", "blf", "bhld"]))
    P = rng.choice([16, 32, 64, 64, 128])
    C, Dr = rng.choice([128, 256, 512, 512]), rng.choice([32, 64, 64])
    if op == "pages":
        n, c, ctx = _log_int(rng, 1, 32), _log_int(rng, 1, 16), _log_int(rng, 16, 16384)
        kind = rng.choice(["latent", "8bit"])
        Rkv, H = (rng.choice([1, 2, 4, 8]), rng.choice([16, 32, 64, 128])) if kind == "8bit" else (0, 0)
        per_token = 2 * Rkv * H if kind == "8bit" else 2 * (C + Dr)
        ctx = max(16, min(ctx, MOST_CACHED // (4 * (n + c) * per_token)))
        return _pages_case(None, kind, n, c, ctx, P, Rkv=Rkv, H=H, C=C if kind == "latent" else 0, Dr=Dr if kind == "latent" else 0, dtype=dtype)
    R = rng.choice([1, 4, 8, 12, 16, 16, 24, 32, 40, 64, 128])
    L = 1 if rng.random() < 0.5 else rng.randint(2, 8) if rng.random() < 0.4 else _log_int(rng, 8, 4096)
    B = _log_int(rng, 1, 64)
    if op == "expanded":
        Dn = rng.choice([64, 128])
        L = _log_int(rng, 2, 4096)
        ctx = max(L, _log_int(rng, 16, 16384))
        B = max(1, min(B, int(MOST_CACHED // (ctx * R * 4 * Dn)), int(MOST_FLOPS // (2.0 * L * ctx * R * (2 * Dn + Dr)))))
        L = max(1, min(L, int(MOST_FLOPS // (2.0 * B * ctx * R * (2 * Dn + Dr)))))
        return _expanded_case(None, B, L, R, Dn, Dr, ctx, dtype=dtype, ragged=ragged, lse=rng.random() < 0.4)
    ctx = max(16, min(_log_int(rng, 64, 131072), MOST_CACHED // (B * 2 * (C + Dr))))
    L = max(1, min(L, ctx, int(0.4 * MOST_FLOPS // (2.0 * B * ctx * R * (2 * C + Dr))), (1 << 26) // (B * R * C)))
    return _latent_case(None, op, B, L, R, C, Dr, P, ctx, dtype=dtype, Dn=rng.choice([64, 128]), ragged=ragged,
                        interleaved=rng.random() < 0.5, lse=op != "append" and rng.random() < 0.4)


# ---- what the program holds ----

def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=_DEVICE, dtype=torch.float32)


def _lengths(case, gen, longest):
    """Tokens of each sequence, and its new ones among them."""
    B, L = case["B"], case["L"]
    totals = torch.full((B,), longest, device=_DEVICE, dtype=torch.int64)
    new_lens = torch.full((B,), L, device=_DEVICE, dtype=torch.int64)
    if case["ragged"]:
        totals -= torch.randint(0, longest // 2 + 1, (B,), generator=gen, device=_DEVICE)
        new_lens -= torch.randint(0, (L + 1) // 2, (B,), generator=gen, device=_DEVICE)
        totals[0], new_lens[0] = longest, L
        new_lens = torch.minimum(new_lens, totals)
    return totals, new_lens


def _plain_tables(rows, D):
    inv = 10000.0 ** (-torch.arange(0, D, 2, device=_DEVICE, dtype=torch.float64) / D)
    angle = torch.arange(rows, device=_DEVICE, dtype=torch.float64)[:, None] * inv[None, :]
    return angle.cos().to(torch.float32), angle.sin().to(torch.float32)


def _prepare_rotate(case, gen):
    B, L, R, Rkv, H = (case[key] for key in ("B", "L", "R", "Rkv", "H"))
    dtype = _DTYPES[case["dtype"]]
    if case["layout"] == "blf":
        both = _normal(gen, B, L, (R + 2 * Rkv) * H).to(dtype)     # one projection's output
        state = {"q": both[:, :, :R * H], "k": both[:, :, R * H:(R + Rkv) * H]}
    else:
        state = {"q": _normal(gen, B, R, L, H).to(dtype), "k": _normal(gen, B, Rkv, L, H).to(dtype)}
    totals, new_lens = _lengths(case, gen, case["ctx"])
    state["starts"] = (totals - new_lens).to(torch.int32)
    state["new_lens"] = new_lens.to(torch.int32) if case["ragged"] else None
    if case["op"] == "rotate":
        state["cos"], state["sin"] = _plain_tables(case["ctx"], case["D"])
    return state


def _prepare_pages(case, gen):
    n, c, ctx, P = (case[key] for key in ("n", "c", "ctx", "P"))
    dev, dtype = torch.device(_DEVICE), _DTYPES[case["dtype"]]
    half, W = n + c, -(-(ctx + 1) // P)
    S = 2 * half + 2                                               # two halves of prompts and their forks, and two rows of a fixed text
    N = 2 * n * W + 2 * c + 2 * W + 2 * half + 8
    if case["kind"] == "latent":
        tensors = [_normal(gen, N, P, case["C"] + case["Dr"]).to(dtype)]
    else:
        Rkv, H = case["Rkv"], case["H"]
        tensors = [_normal(gen, N, Rkv, P, H).to(torch.float8_e4m3fn) for _ in range(2)]
        tensors += [torch.randint(-20, 20, (N, Rkv), generator=gen, device=dev).to(torch.int8) for _ in range(2)]
        tensors += [torch.randint(-100, 100, (N, Rkv, 2, H), generator=gen, device=dev).to(torch.int8)]
    lens = torch.zeros(2, S, dtype=torch.int64, device=dev)        # what each half's new prompts bring
    which = torch.arange(S, device=dev)
    for h in range(2):
        prompts = (which >= h * half) & (which < h * half + n)
        lens[h] = torch.where(prompts, ctx - torch.randint(0, ctx // 2 + 1, (S,), generator=gen, device=dev), 0)
    starts = lens.sum(dim=0)
    fixed = min(W, max(1, ctx // (4 * P)))                         # pages of the fixed text
    starts[S - 2:] = fixed * P
    order = torch.randperm(N, generator=gen, device=dev)
    page = torch.arange(W, device=dev)
    held = page[None, :] * P < starts[:, None]
    rank = held.flatten().cumsum(0).view(S, W) - 1
    table = torch.where(held, order[rank.clamp(min=0)], -1).to(torch.int32)
    uses = torch.zeros(N, dtype=torch.int32, device=dev)
    uses[table[held].long()] = 1
    halves = []
    for h in range(2):
        parents = h * half + torch.randint(0, n, (c,), generator=gen, device=dev)
        children = h * half + n + torch.arange(c, device=dev)
        halves.append({"all": (h * half + torch.arange(half, device=dev)).to(torch.int32), "lens": lens[h].to(torch.int32),
                       "parents": parents.to(torch.int32), "children": children.to(torch.int32)})
    return {"tensors": tensors, "table": table, "starts": starts.to(torch.int32), "uses": uses, "halves": halves}


def _prepare_latent(case, gen):
    B, L, R, C, Dr, Dn, P, ctx = (case[key] for key in ("B", "L", "R", "C", "Dr", "Dn", "P", "ctx"))
    dtype, W = _DTYPES[case["dtype"]], -(-ctx // P)
    N = B * W + max(1, B * W // 16)                                # some pages are free
    size = (0.4 * _normal(gen, C + Dr)).exp_()                     # channels of different size, as models have them
    cache = torch.empty(N, P, C + Dr, dtype=dtype, device=_DEVICE)
    for at in range(0, N, 4096):
        cache[at:at + 4096] = (_normal(gen, min(4096, N - at), P, C + Dr) * size).to(dtype)
    state = {"cache": cache}
    state["table"] = torch.randperm(N, generator=gen, device=_DEVICE)[:B * W].to(torch.int32).view(B, W)
    totals, new_lens = _lengths(case, gen, ctx)
    state["starts"] = (totals - new_lens).to(torch.int32)
    state["new_lens"] = new_lens.to(torch.int32) if case["ragged"] else None
    both = (_normal(gen, B, L, C + Dr) * size).to(dtype)           # one projection's output
    state["c"], state["k"] = both[:, :, :C], both[:, :, C:]
    state["qr"] = _normal(gen, B, L, R, Dn + Dr).to(dtype)[..., Dn:]
    if case["op"] != "append":
        state["q"] = _normal(gen, B, L, R, C).to(dtype)
    state["cos"], state["sin"] = _plain_tables(ctx, Dr)
    state["scale"] = 1.0 / math.sqrt(Dn + Dr)
    return state


def _prepare_expanded(case, gen):
    B, L, R, Dn, Dr, Dv, K = (case[key] for key in ("B", "L", "R", "Dn", "Dr", "Dv", "ctx"))
    dtype = _DTYPES[case["dtype"]]
    kv = torch.empty(B, K, R, Dn + Dv, dtype=dtype, device=_DEVICE)    # one product's output
    for b in range(B):
        kv[b] = _normal(gen, K, R, Dn + Dv).to(dtype)
    state = {"q": _normal(gen, B, L, R, Dn + Dr).to(dtype), "k": kv[..., :Dn], "v": kv[..., Dn:], "kr": _normal(gen, B, K, Dr).to(dtype)}
    totals, new_lens = _lengths(case, gen, K)
    state["starts"] = (totals - new_lens).to(torch.int32) if case["ragged"] else None
    state["new_lens"] = new_lens.to(torch.int32) if case["ragged"] else None
    return state


_FAMILY = {"rotate": "rotate", "tables_rotate": "rotate", "pages": "pages", "append": "latent", "attend": "latent", "step": "latent",
           "expanded": "expanded"}


def prepare(case, seed):
    gen = torch.Generator(device=torch.device(_DEVICE)).manual_seed(seed)
    make = {"rotate": _prepare_rotate, "pages": _prepare_pages, "latent": _prepare_latent, "expanded": _prepare_expanded}
    return {"case": case, **make[_FAMILY[case["op"]]](case, gen)}


# ---- the plain form ----

def _lens(s, B, L):
    return s["new_lens"].long() if s["new_lens"] is not None else torch.full((B,), L, device=_DEVICE, dtype=torch.int64)


def _frequencies(case):
    """What the tables' columns turn by for each position, in 64 bits."""
    D, factor, n = case["D"], case["factor"], case["ctx"] / case["factor"]      # n: positions of the model before it was stretched
    j = torch.arange(D // 2, device=_DEVICE, dtype=torch.float64)
    base = 10000.0
    if case["scaling"] == "base":
        base = base * factor ** (D / (D - 2))
    f = base ** (-2.0 * j / D)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "turns":
        keep = ((n * f / (2.0 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
    if case["scaling"] == "index":
        a = max(math.floor(D * math.log(n / (2.0 * math.pi * 32.0)) / (2.0 * math.log(base))), 0)
        b = min(math.ceil(D * math.log(n / (2.0 * math.pi * 1.0)) / (2.0 * math.log(base))), D - 1)
        keep = 1.0 - ((j - a) / max(b - a, 0.001)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
    return f


def _amplitude(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "index" else 1.0


def _tables(s):
    case = s["case"]
    angle = torch.arange(case["ctx"], device=_DEVICE, dtype=torch.float64)[:, None] * _frequencies(case)[None, :]
    return (angle.cos() * _amplitude(case)).to(torch.float32), (angle.sin() * _amplitude(case)).to(torch.float32)


def _turned(x, cos, sin, at, interleaved, inverse=False):
    """x [B, L, ..., D] in 32 bits by the tables' rows at [B, L]; products and their sums each rounded."""
    at = at.clamp(0, cos.shape[0] - 1)
    cos, sin = cos[at], sin[at]
    while cos.dim() < x.dim():
        cos, sin = cos.unsqueeze(2), sin.unsqueeze(2)
    if inverse:
        sin = -sin
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, dim=-1)
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)


def _rotate(s, cos, sin):
    case = s["case"]
    B, L, H, D, first = (case[key] for key in ("B", "L", "H", "D", "first"))
    i = torch.arange(L, device=_DEVICE)
    at = s["starts"].long()[:, None] + i
    exists = (i < _lens(s, B, L)[:, None])[:, :, None, None]
    out = []
    for x in (s["q"], s["k"]):
        y = (x.view(B, L, -1, H) if case["layout"] == "blf" else x.transpose(1, 2)).to(torch.float32)
        turned = _turned(y[..., first:first + D], cos, sin, at, case["interleaved"], case["inverse"])
        y = torch.cat([y[..., :first], turned, y[..., first + D:]], dim=-1)
        y = torch.where(exists, y, 0.0).to(x.dtype)
        out.append(y.flatten(2) if case["layout"] == "blf" else y.transpose(1, 2).contiguous())
    return out


def _as_bytes(t):
    return t.flatten(1).view(torch.uint8)


def _plain_copy(tensors, sources, targets):
    N = tensors[0].shape[0]
    sources, targets = sources.long(), targets.long()
    ok = (sources >= 0) & (sources < N) & (targets >= 0) & (targets < N)
    for t in tensors:
        _as_bytes(t)[targets[ok]] = _as_bytes(t)[sources[ok]]


def _plain_free(table, starts, uses, sequences):
    rows = sequences.long()
    named = table[rows].flatten().long()
    named = named[(named >= 0) & (named < uses.shape[0])]
    uses.sub_(torch.zeros_like(uses).index_add_(0, named, torch.ones_like(named, dtype=torch.int32)))
    table[rows] = -1
    starts[rows] = 0


def _plain_take(table, starts, uses, P, L, new_lens):
    S, W = table.shape
    first = starts.long().clamp(min=0)
    end = (starts.long() + new_lens.long().clamp(0, L)).clamp(min=0)
    w = torch.arange(W, device=table.device)
    wanted = (w >= -(-first // P)[:, None]) & (w < -(-end // P)[:, None]) & (new_lens > 0)[:, None]
    beyond = torch.where(new_lens > 0, (-(-end // P) - torch.maximum(-(-first // P), torch.full_like(first, W))).clamp(min=0), 0)
    wanted &= (table < 0) | (table >= uses.shape[0])
    free = torch.nonzero(uses <= 0).flatten()
    rank = wanted.flatten().cumsum(0).view(S, W) - 1
    given = wanted & (rank < free.shape[0])
    pages = free[rank[given]]
    table[wanted] = -1
    table[given] = pages.to(torch.int32)
    uses[pages] = 1
    return ((wanted & ~given).sum(dim=1) + beyond).to(torch.int32)


def _plain_fork(tensors, table, starts, uses, P, parents, children):
    """Parents and children that exist, children that are empty and named once: what this file's lists hold."""
    W = table.shape[1]
    parents, children = parents.long(), children.long()
    length = starts[parents].long()
    full, partial = length // P, length % P != 0
    free = torch.nonzero(uses <= 0).flatten()
    rank = partial.long().cumsum(0) - 1
    ok = ~partial | (rank < free.shape[0])
    w = torch.arange(W, device=table.device)
    rows = torch.where(w < full[:, None], table[parents], -1)
    copied = partial & ok
    to = free[rank[copied]]
    of = table[parents[copied], full[copied]]
    rows[copied, full[copied]] = to.to(torch.int32)
    shared = torch.where((w < full[:, None]) & ok[:, None], rows, -1).flatten().long()
    shared = shared[shared >= 0]
    uses.add_(torch.zeros_like(uses).index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32)))
    uses[to] = 1
    table[children[ok]] = rows[ok]
    starts[children[ok]] = starts[parents[ok]]
    _plain_copy(tensors, of, to)
    return ok.to(torch.int32)


def _plain_compact(tensors, table, uses):
    N = uses.shape[0]
    used = uses > 0
    U = used.sum()
    page = torch.arange(N, device=uses.device)
    holes, movers = torch.nonzero(~used & (page < U)).flatten(), torch.nonzero(used & (page >= U)).flatten()
    moved = torch.where(used, page, -1)
    moved[movers] = holes
    _plain_copy(tensors, movers, holes)
    uses[holes] = uses[movers]
    uses[movers] = 0
    named = (table >= 0) & (table < N)
    table.copy_(torch.where(named, moved[table.clamp(0, N - 1).long()].to(torch.int32), -1))
    return moved.to(torch.int32)


def _latent_append(s):
    case = s["case"]
    B, L, P = case["B"], case["L"], case["P"]
    dtype, starts, lens = s["cache"].dtype, s["starts"].long(), _lens(s, B, L)
    i = torch.arange(L, device=_DEVICE)
    at, exists = starts[:, None] + i, i < lens[:, None]
    keys = _turned(s["k"].to(torch.float32), s["cos"], s["sin"], at, case["interleaved"]).to(dtype)
    new = torch.cat([s["c"], keys], dim=-1)[exists]
    pages = torch.gather(s["table"].long(), 1, (at // P).clamp(max=s["table"].shape[1] - 1))
    s["cache"][pages[exists], (at % P)[exists]] = new
    q = _turned(s["qr"].to(torch.float32), s["cos"], s["sin"], at, case["interleaved"])
    return torch.where(exists[:, :, None, None], q, 0.0).to(dtype)


def _visible(starts, lens, L, causal_to):
    """How many keys the rows see, [B, L]: those up to their own; none in rows behind the new tokens."""
    i = torch.arange(L, device=starts.device)
    return torch.where(i < lens[:, None], (starts[:, None] + i + 1).clamp(max=causal_to), 0)


def _softmax(scores, seen):
    """scores [..., rows, keys] in place, seen [..., rows]: weights, their sums' reciprocals and the log-sum-exp."""
    at = torch.arange(scores.shape[-1], device=scores.device)
    scores.masked_fill_(at >= seen[..., None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    scores.sub_(top).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    return scores, torch.where(total > 0, 1.0 / total, 0.0), (top + total.log())[..., 0]


def _latent_attend(s, qr):
    case = s["case"]
    B, L, R, C, Dr, P, ctx = (case[key] for key in ("B", "L", "R", "C", "Dr", "P", "ctx"))
    W = s["table"].shape[1]
    seen = _visible(s["starts"].long(), _lens(s, B, L), L, ctx)
    out = torch.empty(B, L, R, C, dtype=s["cache"].dtype, device=_DEVICE)
    lse = torch.empty(B, R, L, dtype=torch.float32, device=_DEVICE)
    step = max(1, (1 << 30) // (L * R * W * P + W * P * (C + Dr)))
    for b in range(0, B, step):
        pick = slice(b, min(B, b + step))
        keys = s["cache"][s["table"][pick].long()].flatten(1, 2).to(torch.float32)
        q = torch.cat([s["q"][pick], qr[pick]], dim=-1).to(torch.float32).flatten(1, 2)
        scores = (q * s["scale"]) @ keys.transpose(1, 2)
        weights, inverse, sums = _softmax(scores, seen[pick, :, None].expand(-1, -1, R).flatten(1))
        out[pick] = ((weights @ keys[..., :C]) * inverse).view(-1, L, R, C).to(out.dtype)
        lse[pick] = sums.view(-1, L, R).transpose(1, 2)
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def _expanded(s):
    case = s["case"]
    B, L, R, Dn, Dr, Dv, K = (case[key] for key in ("B", "L", "R", "Dn", "Dr", "Dv", "ctx"))
    starts = s["starts"].long() if s["starts"] is not None else torch.full((B,), K - L, device=_DEVICE)
    seen = _visible(starts, _lens(s, B, L), L, K)
    out = torch.empty(B, L, R, Dv, dtype=s["q"].dtype, device=_DEVICE)
    lse = torch.empty(B, R, L, dtype=torch.float32, device=_DEVICE)
    step = max(1, (1 << 30) // (L * K))
    for b in range(B):
        for h in range(0, R, step):
            pick = slice(h, min(R, h + step))
            heads = pick.stop - h
            q = s["q"][b, :, pick].transpose(0, 1).to(torch.float32) * (1.0 / math.sqrt(Dn + Dr))
            k = torch.cat([s["k"][b, :, pick], s["kr"][b, :, None].expand(-1, heads, -1)], dim=-1).to(torch.float32)
            scores = q @ k.permute(1, 2, 0)
            weights, inverse, sums = _softmax(scores, seen[b].expand(heads, -1))
            o = (weights @ s["v"][b, :, pick].transpose(0, 1).to(torch.float32)) * inverse
            out[b, :, pick], lse[b, pick] = o.transpose(0, 1).to(out.dtype), sums
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


# ---- the calls ----

def _own_tables(s):
    import fused_attn

    case = s["case"]
    options = {"none": {}, "linear": {}, "base": {}, "turns": {"low": 1.0, "high": 4.0}, "index": {"low": 1.0, "high": 32.0}}
    return fused_attn.rotary_tables(case["ctx"], case["D"], s["q"].device, base=10000.0, scaling=case["scaling"], factor=case["factor"],
                                    original_rows=case["ctx"] / case["factor"], amplitude=_amplitude(case), **options[case["scaling"]])


def _own_rotate(s, cos, sin):
    import fused_attn

    case = s["case"]
    return fused_attn.rotate(s["q"], cos, sin, case["H"], keys=s["k"], starts=s["starts"], new_lens=s["new_lens"], first=case["first"],
                             interleaved=case["interleaved"], inverse=case["inverse"], layout=case["layout"])


def _own_append(s):
    import fused_attn

    return fused_attn.latent_append(s["c"], s["k"], s["cache"], s["table"], s["starts"], new_lens=s["new_lens"], queries=s["qr"],
                                    rope_cos=s["cos"], rope_sin=s["sin"], interleaved=s["case"]["interleaved"])


def _own_attend(s, qr):
    import fused_attn

    r = fused_attn.latent_attention(s["q"], qr, s["cache"], s["table"], s["starts"], s["scale"], new_lens=s["new_lens"],
                                    return_lse=s["case"]["lse"])
    return {"out": r[0], "lse": r[1]} if s["case"]["lse"] else {"out": r}


def _own_expanded(s):
    import fused_attn

    r = fused_attn.expanded_attention(s["q"], s["k"], s["kr"], s["v"], starts=s["starts"], new_lens=s["new_lens"],
                                      return_lse=s["case"]["lse"])
    return {"out": r[0], "lse": r[1]} if s["case"]["lse"] else {"out": r}


def _pages_turn(s):
    """The fixed text's pages are written afresh from their master copy; then, for each half of the sequences, as when its answers have
    ended: their pages are freed, what is left is moved together, new prompts take pages, and each fork continues one of them."""
    if own:
        from fused_attn import compact_pages as compact, copy_pages as copy, fork_pages as fork, free_pages as free, take_pages as take
    else:
        copy, free, compact, take, fork = _plain_copy, _plain_free, _plain_compact, _plain_take, _plain_fork
    tensors, table, starts, uses = s["tensors"], s["table"], s["starts"], s["uses"]
    P, most = s["case"]["P"], s["case"]["ctx"]
    got = {}
    copy(tensors, table[-2], table[-1])
    for h, half in enumerate(s["halves"]):
        free(table, starts, uses, half["all"])
        moved = compact(tensors, table, uses)
        missing = take(table, starts, uses, P, most, half["lens"])
        starts.add_(half["lens"])
        forked = fork(tensors, table, starts, uses, P, half["parents"], half["children"])
        got.update({"moved%d" % h: moved, "missing%d" % h: missing, "forked%d" % h: forked})
    got.update({"table": table, "starts": starts, "uses": uses})
    got.update({"tensor%d" % n: t for n, t in enumerate(tensors)})
    return got


def run(state):
    op = state["case"]["op"]
    if op in ("rotate", "tables_rotate"):
        got = {}
        if op == "tables_rotate":
            cos, sin = (_own_tables if own else _tables)(state)
            got = {"cos": cos, "sin": sin}
        else:
            cos, sin = state["cos"], state["sin"]
        got["q"], got["k"] = (_own_rotate if own else _rotate)(state, cos, sin)
        return got
    if op == "pages":
        return _pages_turn(state)
    if op == "expanded":
        return (_own_expanded if own else _expanded)(state)
    got, qr = {}, state["qr"]
    if op in ("append", "step"):
        qr = (_own_append if own else _latent_append)(state)
        got = {"q": qr, "cache": state["cache"]}
    if op in ("attend", "step"):
        got.update((_own_attend if own else _latent_attend)(state, qr))
    return got


def work(case):
    op = case["op"]
    nbytes = flops = 0.0
    if op in ("rotate", "tables_rotate"):
        B, L, R, Rkv, H, D = (float(case[key]) for key in ("B", "L", "R", "Rkv", "H", "D"))
        T = B * L * ((1.0 + 0.75 * (B - 1)) / B if case["ragged"] and L > 1 else 1.0)
        nbytes = (T + B * L) * (R + Rkv) * H * 2                   # (rows of tokens that do not exist are written, not read)
        flops = 3.0 * T * (R + Rkv) * D
        if op == "tables_rotate":
            nbytes += 4.0 * case["ctx"] * D
            flops += 20.0 * case["ctx"] * D                        # a sine or a cosine of a 64-bit angle
        else:
            nbytes += 4.0 * min(T, case["ctx"]) * D
    elif op == "pages":
        n, c, ctx, P = (float(case[key]) for key in ("n", "c", "ctx", "P"))
        page = P * 2.0 * (case["C"] + case["Dr"]) if case["kind"] == "latent" else 2.0 * case["Rkv"] * (P * case["H"] + 1 + case["H"])
        pages = 0.75 * ctx / P                                     # of a sequence, on average
        # each turn moves one half's pages (half of them lie behind the others) and each fork copies one
        copied = max(1.0, ctx / (4 * P)) + 2 * (0.5 * n * pages + c)
        nbytes = 2.0 * page * copied + 4.0 * 2 * 4 * (2 * n * pages + (n + c) * ctx / P)
        flops = 0.0
    elif op == "expanded":
        B, L, R, Dn, Dr, Dv, K = (float(case[key]) for key in ("B", "L", "R", "Dn", "Dr", "Dv", "ctx"))
        share = (1.0 + 0.75 * (B - 1)) / B if case["ragged"] else 1.0
        T, keys = B * L * share, max(1.0, K * share - L * share / 2.0)
        nbytes = 2.0 * T * R * (Dn + Dr) + 2.0 * B * L * R * Dv + 2.0 * B * K * share * (R * (Dn + Dv) + Dr) + 4.0 * B * R * L * case["lse"]
        flops = 2.0 * T * keys * R * (Dn + Dr + Dv)
    else:
        B, L, R, C, Dr, P, ctx = (float(case[key]) for key in ("B", "L", "R", "C", "Dr", "P", "ctx"))
        share = (1.0 + 0.75 * (B - 1)) / B if case["ragged"] else 1.0
        T = B * L * (share if L > 1 else 1.0)
        if op in ("append", "step"):
            nbytes += 2.0 * T * ((C + Dr) * 2 + R * Dr * 2) + 4.0 * min(T, ctx) * Dr
            flops += 3.0 * T * (R + 1) * Dr
        if op in ("attend", "step"):
            keys = max(1.0, ctx * share - (T / B) / 2.0 + 0.5)
            nbytes += 2.0 * B * ctx * share * (C + Dr) + 2.0 * T * R * (C + (Dr if op == "attend" else 0.0)) + 2.0 * B * L * R * C
            nbytes += 4.0 * B * R * L * case["lse"]
            flops += 2.0 * T * keys * R * (2 * C + Dr)
    return {"bytes": nbytes, "flops": flops}


# ---- from the definitions ----

def _exact_tables(case):
    D, s, n = case["D"], case["factor"], case["ctx"] / case["factor"]
    f = []
    for j in range(D // 2):
        if case["scaling"] == "base":
            f.append(math.exp(-2.0 * j / D * (math.log(10000.0) + D / (D - 2.0) * math.log(s))))
            continue
        x = math.exp(-2.0 * j / D * math.log(10000.0))
        turns = n * x / math.tau
        if case["scaling"] == "linear":
            x /= s
        elif case["scaling"] == "turns":
            x = x if turns >= 4.0 else x / s if turns <= 1.0 else x * ((turns - 1.0) + (4.0 - turns) / s) / 3.0
        elif case["scaling"] == "index":
            low = max(math.floor(D * math.log(n / (math.tau * 32.0)) / math.log(1e8)), 0)
            high = min(math.ceil(D * math.log(n / math.tau) / math.log(1e8)), D - 1)
            away = min(max((j - low) / max(high - low, 0.001), 0.0), 1.0)
            x = x * (1.0 - away) + x / s * away
        f.append(x)
    f = torch.tensor(f, dtype=torch.float64, device=_DEVICE)
    angle = torch.outer(torch.arange(case["ctx"], device=_DEVICE).double(), f)
    z = torch.polar(torch.full_like(angle, _amplitude(case)), angle)
    return z.real, z.imag


def _exact_turn(x, turn, interleaved):
    """x [n, heads, D] by the complex numbers turn [n, D/2]."""
    half = x.shape[-1] // 2
    pairs = x.double().unflatten(-1, (half, 2)) if interleaved else x.double().unflatten(-1, (2, half)).transpose(-1, -2)
    z = torch.view_as_complex(pairs.contiguous()) * turn[:, None]
    y = torch.view_as_real(z)
    return (y if interleaved else y.transpose(-1, -2)).flatten(-2)


def _exact_rotate(case, s):
    B, L, H, D, first = (case[key] for key in ("B", "L", "H", "D", "first"))
    got = {}
    if case["op"] == "tables_rotate":
        cos, sin = _exact_tables(case)
        got = {"cos": cos, "sin": sin}
        cos, sin = cos.float().double(), sin.float().double()      # as the rotation gets them
    else:
        cos, sin = s["cos"].double(), s["sin"].double()
    starts = s["starts"].tolist()
    lens = s["new_lens"].tolist() if case["ragged"] else [L] * B
    for name in ("q", "k"):
        x = s[name].unflatten(2, (-1, H)) if case["layout"] == "blf" else s[name].transpose(1, 2)
        y = torch.zeros(x.shape, dtype=torch.float64, device=_DEVICE)
        for b in range(B):
            rows = slice(starts[b], starts[b] + lens[b])
            turn = torch.complex(cos[rows], -sin[rows] if case["inverse"] else sin[rows])
            y[b, :lens[b]] = x[b, :lens[b]].double()
            y[b, :lens[b], :, first:first + D] = _exact_turn(x[b, :lens[b], :, first:first + D], turn, case["interleaved"])
        got[name] = y.flatten(2) if case["layout"] == "blf" else y.transpose(1, 2).contiguous()
    return got


def _exact_pages(case, s):
    """A page's contents by the page that held them at first; all else in lists on the host."""
    P, most = case["P"], case["ctx"]
    table, starts, uses = s["table"].tolist(), s["starts"].tolist(), s["uses"].tolist()
    S, W, N = len(table), len(table[0]), len(uses)
    holds = list(range(N))
    got = {}
    for a, b in zip(table[-2], table[-1]):
        if 0 <= a < N and 0 <= b < N:
            holds[b] = a

    def free_pages():
        return iter([page for page in range(N) if uses[page] <= 0])

    for h, half in enumerate(s["halves"]):
        for row in half["all"].tolist():
            for page in table[row]:
                if 0 <= page < N:
                    uses[page] -= 1
            table[row], starts[row] = [-1] * W, 0
        used = [page for page in range(N) if uses[page] > 0]
        U = len(used)
        moved = [page if uses[page] > 0 else -1 for page in range(N)]
        for hole, page in zip([p for p in range(U) if uses[p] <= 0], [p for p in used if p >= U]):
            moved[page], holds[hole], uses[hole], uses[page] = hole, holds[page], uses[page], 0
        table = [[moved[page] if 0 <= page < N else -1 for page in row] for row in table]
        free, missing = free_pages(), [0] * S
        for row, n in enumerate(half["lens"].tolist()):
            if n > 0:
                for w in range(-(-starts[row] // P), -(-(starts[row] + min(n, most)) // P)):
                    page = next(free, None) if w < W else None
                    if page is None:
                        missing[row] += 1
                    else:
                        table[row][w], uses[page] = page, 1
            starts[row] += n
        free, forked = free_pages(), []
        for parent, child in zip(half["parents"].tolist(), half["children"].tolist()):
            n = starts[parent]
            row = [page if (w + 1) * P <= n else -1 for w, page in enumerate(table[parent])]
            page = next(free, None) if n % P else -1
            forked.append(int(page is not None))
            if page is None:
                continue
            for shared in row:
                if shared >= 0:
                    uses[shared] += 1
            if n % P:
                row[n // P], uses[page], holds[page] = page, 1, holds[table[parent][n // P]]
            table[child], starts[child] = row, n
        got.update({"moved%d" % h: moved, "missing%d" % h: missing, "forked%d" % h: forked})
    got.update({"table": table, "starts": starts, "uses": uses})
    got = {key: torch.tensor(x, dtype=torch.int32, device=_DEVICE) for key, x in got.items()}
    holds = torch.tensor(holds, device=_DEVICE)
    for n, t in enumerate(s["tensors"]):
        got["tensor%d" % n] = _as_bytes(t)[holds].view(t.dtype).view(t.shape)
    return got


def _exact_latent(case, s):
    B, L, R, C, Dr, P, ctx = (case[key] for key in ("B", "L", "R", "C", "Dr", "P", "ctx"))
    starts, lens = s["starts"].tolist(), s["new_lens"].tolist() if case["ragged"] else [L] * B
    got, qr = {}, s["qr"].double()
    if case["op"] != "attend":
        q, cache = torch.zeros(B, L, R, Dr, dtype=torch.float64, device=_DEVICE), s["cache"].double()
        for b in range(B):
            n, first = lens[b], starts[b]
            turn = torch.complex(s["cos"][first:first + n].double(), s["sin"][first:first + n].double())
            q[b, :n] = _exact_turn(s["qr"][b, :n], turn, case["interleaved"])
            new = torch.cat([s["c"][b, :n].double(), _exact_turn(s["k"][b, :n, None], turn, case["interleaved"])[:, 0]], dim=-1)
            at = torch.arange(first, first + n, device=_DEVICE)
            pages = s["table"][b].long()[at // P]
            cache[pages, at % P] = new
            s["cache"][pages, at % P] = new.to(s["cache"].dtype)
        got = {"q": q, "cache": cache}
        qr = q.to(s["cache"].dtype).double()                       # as the attention gets it
    if case["op"] == "append":
        return got
    out = torch.zeros(B, L, R, C, dtype=torch.float64, device=_DEVICE)
    lse = torch.full((B, R, L), -math.inf, dtype=torch.float64, device=_DEVICE)
    for b in range(B):
        n, keys = lens[b], starts[b] + lens[b]
        if n == 0 or keys == 0:
            continue
        cached = s["cache"][s["table"][b, :-(-keys // P)].long()].flatten(0, 1)[:keys].double()
        hidden = torch.arange(keys, device=_DEVICE) > starts[b] + torch.arange(n, device=_DEVICE)[:, None]
        for h in range(R):
            scores = (s["q"][b, :n, h].double() @ cached[:, :C].T + qr[b, :n, h] @ cached[:, C:].T) * s["scale"]
            scores.masked_fill_(hidden, -math.inf)
            lse[b, h, :n] = scores.logsumexp(dim=1)
            out[b, :n, h] = (scores - lse[b, h, :n, None]).exp() @ cached[:, :C]
    return {**got, "out": out, **({"lse": lse} if case["lse"] else {})}


def _exact_expanded(case, s):
    B, L, R, Dn, Dr, Dv, K = (case[key] for key in ("B", "L", "R", "Dn", "Dr", "Dv", "ctx"))
    starts = s["starts"].tolist() if case["ragged"] else [K - L] * B
    lens = s["new_lens"].tolist() if case["ragged"] else [L] * B
    out = torch.zeros(B, L, R, Dv, dtype=torch.float64, device=_DEVICE)
    lse = torch.full((B, R, L), -math.inf, dtype=torch.float64, device=_DEVICE)
    for b in range(B):
        n, keys = lens[b], starts[b] + lens[b]
        hidden = torch.arange(keys, device=_DEVICE) > starts[b] + torch.arange(n, device=_DEVICE)[:, None]
        for h in range(R):
            q = s["q"][b, :n, h].double()
            scores = q[:, :Dn] @ s["k"][b, :keys, h].double().T + q[:, Dn:] @ s["kr"][b, :keys].double().T
            scores = (scores / math.sqrt(Dn + Dr)).masked_fill_(hidden, -math.inf)
            lse[b, h, :n] = scores.logsumexp(dim=1)
            out[b, :n, h] = (scores - lse[b, h, :n, None]).exp() @ s["v"][b, :keys, h].double()
    return {"out": out, **({"lse": lse} if case["lse"] else {})}


def exact(case, seed):
    if case["op"] in ("attend", "step", "expanded") and case["B"] * case["R"] > 2048:
        return None                                                # loops that would take long
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "pages": _exact_pages, "latent": _exact_latent, "expanded": _exact_expanded}[_FAMILY[case["op"]]](case, s)
