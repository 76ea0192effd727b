"""What a program that answers with a model asks of the key/value cache: appending tokens to it, attention over it, and
attention over those of its pages that a cheap score selects.

`listed()` names twelve calls, `draw(rng)` gives more from the same ranges; `prepare` makes the tensors that a program holds
before the call, `run` is one call (or the calls of one step) and `work` the bytes and operations it cannot do without.
`run` makes the module's calls where `own` is true; otherwise it computes the same from elementary operations in 32 bits.
`exact` has the same results from the definitions in 64 bits.

The cache: pages of P tokens for each key head, keys and values in 8 bits (e4m3), a power of two for each page and head
([pages, Rkv] exponents), and for every page the largest and the smallest key of each channel in steps of 2^(exponent + 2).
Token i of the call has the position starts[b] + i; sequence b brings new_lens[b] tokens of the L that its rows have room for.

Keys of a case:
  op       "append" (rotate and append), "attend", "select", "step" (append, then attend), "sparse" (select, then
           attend to the selected pages) or "sparse_step" (append, select, attend)
  B L      sequences, and new tokens of each: 1 for an answer's next token, a few for drafted ones, many for a prompt
  R Rkv H  query heads, key/value heads, head_dim
  P ctx    tokens of a page; tokens of the longest sequence, the new ones among them
  ragged   the other sequences are shorter, down to half of it, and bring fewer new tokens
  dtype    "fp16" or "bf16"
  layout   "blf" ([B, L, heads * H], slices of one projection's output) or "bhld" ([B, heads, L, H])
  rope     keys (and queries) are rotated by their positions on the way into the cache
  bounds   the pages' largest and smallest keys are kept as well
  lse      the log-sum-exp of every row is returned as well
  count    pages that are selected for each token and key head
"""
import math

import torch

own = False

# Keys of one head that a listed case holds at most (times its heads and head_dim), and its scores.
MOST_CACHED = 32 * 8192 * 8 * 128
MOST_SCORES = 32 * 2048 * 16384

LEAST_EXPONENT = -80
LARGEST_CODE = 448.0

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_DEVICE = "cuda"


def _case(name, op, B, L, R, Rkv, H, P, ctx, dtype="fp16", ragged=False, layout="blf", rope=False, bounds=False, lse=False,
          count=0):
    case = {"op": op, "B": B, "L": L, "R": R, "Rkv": Rkv, "H": H, "P": P, "ctx": ctx, "ragged": ragged, "dtype": dtype,
            "layout": layout, "rope": rope, "bounds": bounds, "lse": lse, "count": count}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one answer's next token in a small model: latency
        _case("append_token", "append", 1, 1, 4, 4, 64, 64, 256, rope=True),
        # the next tokens of 64 answers, forty 128-wide heads on eight key heads, selection in use
        _case("append_tokens", "append", 64, 1, 40, 8, 128, 64, 4096, dtype="bf16", ragged=True, rope=True, bounds=True),
        # four long prompts, twelve 64-wide heads without sharing
        _case("append_prompts", "append", 4, 4096, 12, 12, 64, 64, 4096, rope=True),
        # one answer's next token over a short context: latency
        _case("attend_token", "attend", 1, 1, 4, 4, 64, 64, 256),
        # four drafted tokens of sixteen answers, twelve 64-wide heads without sharing, small pages, the log-sum-exp kept
        _case("attend_drafted", "attend", 16, 4, 12, 12, 64, 16, 1000, ragged=True, lse=True),
        # the next tokens of 32 answers, five query heads to a key head
        _case("attend_batch", "attend", 32, 1, 40, 8, 128, 64, 8192, dtype="bf16", ragged=True),
        # the next token over one very long document
        _case("attend_long", "attend", 1, 1, 32, 8, 128, 128, 131072),
        # a chunk of a long prompt behind what is cached already
        _case("attend_chunk", "attend", 1, 2048, 32, 8, 128, 64, 16384, dtype="bf16"),
        # whole short prompts of a batch, nothing cached before: append, then attend, [B, R, L, H] tensors
        _case("step_prompts", "step", 8, 1000, 12, 12, 64, 32, 1000, ragged=True, layout="bhld", rope=True),
        # the selection alone, for sixteen answers over long contexts
        _case("select_tokens", "select", 16, 1, 32, 8, 128, 64, 32768, dtype="bf16", ragged=True, bounds=True, count=32),
        # a whole step of the same: append, select, attend to a sixteenth of the pages
        _case("sparse_tokens", "sparse_step", 16, 1, 32, 8, 128, 64, 32768, ragged=True, rope=True, bounds=True, count=32),
        # a chunk of a prompt, every token with a selection of its own
        _case("sparse_chunk", "sparse", 1, 500, 32, 8, 128, 32, 8000, dtype="bf16", bounds=True, count=48),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "step", "select", "sparse", "sparse_step"])
    H = rng.choice([16, 32, 64, 64, 128, 128, 128])
    Rkv = rng.choice([1, 2, 4, 8, 8, 12, 16])
    group = rng.choice([1, 1, 2, 3, 4, 4, 5, 8, 16])
    P = rng.choice([16, 32, 64, 64, 128])
    B = _log_int(rng, 1, 64)
    ctx = _log_int(rng, 64, 65536)
    if rng.random() < 0.3:
        ctx = -(-ctx // 64) * 64
    ctx = max(16, min(ctx, MOST_CACHED // (B * Rkv * H)))
    sparse = op in ("select", "sparse", "sparse_step")
    if sparse:
        ctx = max(ctx, 8 * P)                                      # a selection that leaves something out
    L = 1
    if rng.random() < 0.5:
        L = rng.randint(2, 8) if rng.random() < 0.4 else _log_int(rng, 8, 256 if sparse else 4096)
    L = max(1, min(L, ctx, MOST_SCORES // (2 * B * Rkv * group * ctx), (1 << 25) // (B * Rkv * group * H)))
    count = min(_log_int(rng, 2, 128), ctx // (2 * P)) if sparse else 0
    return _case(None, op, B, L, Rkv * group, Rkv, H, P, ctx, dtype=rng.choice(["fp16", "bf16"]), ragged=rng.random() < 0.6,
                 layout=rng.choice(["blf", "blf", "bhld"]), rope=op in ("append", "step", "sparse_step") and rng.random() < 0.8,
                 bounds=sparse or (op == "append" and rng.random() < 0.5), lse=op == "attend" and rng.random() < 0.3, count=count)


def _pow2(e):
    """2^e in 32 bits, e a tensor of whole numbers in [-126, 127]."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent_of(amax):
    """The smallest e with amax <= 448 * 2^e, not below LEAST_EXPONENT."""
    m, e = torch.frexp(amax)                                       # amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    return torch.where(m <= 0.875, e - 9, e - 8).clamp_min(LEAST_EXPONENT).where(amax > 0, LEAST_EXPONENT)


def _codes(x):
    return x.to(torch.float8_e4m3fn)


def prepare(case, seed):
    dev = torch.device(_DEVICE)
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    B, L, R, Rkv, H, P, ctx = (case[key] for key in ("B", "L", "R", "Rkv", "H", "P", "ctx"))
    W = -(-ctx // P)
    N = B * W + max(1, B * W // 16)                                # some pages are free

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device=dev, dtype=dtype)

    # channels of keys and heads of values of different size, as models have them
    k_size = (0.5 * normal(Rkv, 1, H)).exp_()
    v_size = (0.7 * normal(Rkv, 1, 1)).exp_()
    state = {"case": case}
    for name, size in (("k", k_size), ("v", v_size)):
        y = normal(N, Rkv, P, H).mul_(size)
        exponents = _exponent_of(y.abs().amax(dim=(2, 3)))
        y.mul_(_pow2(-exponents)[:, :, None, None])
        state[name + "_cache"] = _codes(y)
        state[name + "_exponents"] = exponents.to(torch.int8)
        if name == "k" and case["bounds"]:
            y = state["k_cache"].to(torch.float32)
            state["key_bounds"] = torch.stack([(y.amax(dim=2) / 4).ceil(), (y.amin(dim=2) / 4).floor()], dim=2).to(torch.int8)
        del y
    state["page_table"] = torch.randperm(N, generator=gen, device=dev)[:B * W].to(torch.int32).view(B, W)
    totals = torch.full((B,), ctx, device=dev, dtype=torch.int64)
    new_lens = torch.full((B,), L, device=dev, dtype=torch.int64)
    if case["ragged"]:
        totals -= torch.randint(0, ctx // 2 + 1, (B,), generator=gen, device=dev)
        new_lens -= torch.randint(0, (L + 1) // 2, (B,), generator=gen, device=dev)
        totals[0], new_lens[0] = ctx, L
        new_lens = torch.minimum(new_lens, totals)
    state["starts"] = (totals - new_lens).to(torch.int32)
    state["new_lens"] = new_lens.to(torch.int32) if case["ragged"] else None
    # one projection's output, or its three parts as [B, heads, L, H] tensors
    k_std = k_size.view(Rkv, H)
    if case["layout"] == "blf":
        both = normal(B, L, R + 2 * Rkv, H)
        both[:, :, R:R + Rkv] *= k_std
        both[:, :, R + Rkv:] *= v_size.view(Rkv, 1)
        both = both.to(dtype).view(B, L, (R + 2 * Rkv) * H)
        parts = both[:, :, :R * H], both[:, :, R * H:(R + Rkv) * H], both[:, :, (R + Rkv) * H:]
    else:
        parts = (normal(B, R, L, H).to(dtype), (normal(B, Rkv, L, H) * k_std[:, None]).to(dtype),
                 (normal(B, Rkv, L, H) * v_size).to(dtype))
    state["q"], state["k"], state["v"] = parts
    state["cos"] = state["sin"] = None
    if case["rope"]:
        inv = 10000.0 ** (-torch.arange(0, H, 2, device=dev, dtype=torch.float64) / H)
        angle = torch.arange(W * P, device=dev, dtype=torch.float64)[:, None] * inv[None, :]
        state["cos"], state["sin"] = angle.cos().to(torch.float32), angle.sin().to(torch.float32)
    return state


# ---- the plain form ----

def _by_token(x, heads, H, layout):
    """[B, L, heads, H] in 32 bits."""
    x = x.view(x.shape[0], x.shape[1], heads, H) if layout == "blf" else x.transpose(1, 2)
    return x.to(torch.float32)


def _by_layout(x, layout):
    """[B, L, heads, H] as the caller has it."""
    return x.flatten(2) if layout == "blf" else x.transpose(1, 2).contiguous()


def _lens(s):
    case = s["case"]
    return s["new_lens"].long() if s["new_lens"] is not None else torch.full((case["B"],), case["L"], device=s["starts"].device)


def _rotated(x, s):
    """x [B, L, heads, H] rotated by the tokens' positions, products and their sums each rounded to 32 bits."""
    if s["cos"] is None:
        return x
    L, half = x.shape[1], x.shape[3] // 2
    at = (s["starts"].long()[:, None] + torch.arange(L, device=x.device)).clamp(0, s["cos"].shape[0] - 1)
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _append(s):
    case = s["case"]
    L, R, Rkv, H, P = (case[key] for key in ("L", "R", "Rkv", "H", "P"))
    starts, lens = s["starts"].long(), _lens(s)
    dev, W = starts.device, s["page_table"].shape[1]
    # the pages that the new tokens reach, slot by slot: [B, pages, P]
    NP = (L + P - 2) // P + 1
    page = starts[:, None] // P + torch.arange(NP, device=dev)
    at = page[:, :, None] * P + torch.arange(P, device=dev)
    token = at - starts[:, None, None]
    new = (token >= 0) & (token < lens[:, None, None])
    live = token < 0
    old_page = live.any(dim=2)
    reached = new.any(dim=2) & (page < W)
    ids = torch.gather(s["page_table"].long(), 1, page.clamp(max=W - 1))
    which = torch.arange(case["B"], device=dev)[:, None, None]
    token = token.clamp(0, L - 1)
    q = _by_token(s["q"], R, H, case["layout"])
    k = _by_token(s["k"], Rkv, H, case["layout"])
    v = _by_token(s["v"], Rkv, H, case["layout"])
    for name, x in (("k", _rotated(k, s)), ("v", v)):
        cache, exponents = s[name + "_cache"], s[name + "_exponents"]
        y = x[which, token].permute(0, 1, 3, 2, 4)                 # [B, pages, Rkv, P, H]
        is_new, is_live = new[:, :, None, :, None], live[:, :, None, :, None]
        counted = torch.where(is_new & y.isfinite(), y, 0.0)
        e_old = exponents[ids].long()
        e = _exponent_of(counted.abs().amax(dim=(3, 4))).long()
        e = torch.where(old_page[:, :, None], torch.maximum(e, e_old), e)
        shift = _pow2(e_old.clamp_min(-126) - e)[..., None, None]
        was = cache[ids.reshape(-1)].view(ids.shape + cache.shape[1:])
        moved = _codes(was.to(torch.float32) * shift)
        fresh = _codes(torch.where(is_new, y, 0.0) * _pow2(-e)[..., None, None])
        as_bytes = torch.where(is_new, fresh.view(torch.uint8), torch.where(is_live, moved.view(torch.uint8), was.view(torch.uint8)))
        cache.view(torch.uint8)[ids[reached]] = as_bytes[reached]
        exponents[ids[reached]] = e[reached].to(torch.int8)
        if name == "k" and "key_bounds" in s:
            step = counted * _pow2(-e - 2)[..., None, None]
            up = torch.where(is_new, step.ceil(), -128.0).amax(dim=3)
            low = torch.where(is_new, step.floor(), 127.0).amin(dim=3)
            was = s["key_bounds"][ids].to(torch.float32) * shift[..., 0, :, None]
            merge = old_page[:, :, None, None]
            up = torch.where(merge, torch.maximum(up, was[..., 0, :].ceil()), up)
            low = torch.where(merge, torch.minimum(low, was[..., 1, :].floor()), low)
            s["key_bounds"][ids[reached]] = torch.stack([up, low], dim=3)[reached].to(torch.int8)
    q = torch.where((torch.arange(L, device=dev) < lens[:, None])[:, :, None, None], _rotated(q, s), 0.0)
    return _by_layout(q.to(s["q"].dtype), case["layout"])


def _visible(s):
    """How many keys the rows see, [B, L]: those up to their own; none in rows behind the new tokens."""
    i = torch.arange(s["case"]["L"], device=s["starts"].device)
    return torch.where(i < _lens(s)[:, None], s["starts"].long()[:, None] + i + 1, 0)


def _select(s, q):
    case = s["case"]
    B, L, R, Rkv, H, P, count = (case[key] for key in ("B", "L", "R", "Rkv", "H", "P", "count"))
    W = s["page_table"].shape[1]
    x = _by_token(q, R, H, case["layout"]).view(B, L, Rkv, R // Rkv, H)
    amax = x.abs().amax(dim=(3, 4))
    m, e = torch.frexp(amax)
    e = torch.where(m <= 127 / 128, e - 7, e - 6).where(amax > 0, 0)
    x = (x * _pow2(-e)[..., None, None]).round()                   # whole numbers of at most 127
    x = x.permute(0, 2, 1, 3, 4).reshape(B * Rkv, -1, H)
    ids = s["page_table"].long()
    bounds = s["key_bounds"][ids].to(torch.float32).permute(0, 2, 3, 4, 1).reshape(B * Rkv, 2, H, W)
    dots = x.clamp_min(0) @ bounds[:, 0] + x.clamp_max(0) @ bounds[:, 1]
    dots = dots.view(B, Rkv, L, R // Rkv, W).amax(dim=3).transpose(1, 2)
    scores = dots * _pow2(s["k_exponents"][ids].long().clamp(-100, 120) - 20).transpose(1, 2)[:, None]
    seen = _visible(s)[:, :, None, None]
    page = torch.arange(W, device=x.device)
    scores = torch.where(page * P < seen, scores, -math.inf)
    scores = torch.where((page == (seen - 1) // P) & (seen > 0), math.inf, scores)
    order = torch.sort(scores, dim=3, descending=True, stable=True)[1][..., :count]
    pages = torch.where(torch.gather(scores, 3, order) > -math.inf, order, W).sort(dim=3)[0]
    return torch.where(pages < W, pages, -1).to(torch.int32)


def _dequantised(s, name):
    """Keys or values of every sequence, [B, Rkv, W * P, H]."""
    ids = s["page_table"].long()
    x = s[name + "_cache"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).to(torch.float32)
    x = x * _pow2(s[name + "_exponents"][ids].long().clamp_min(-126))[..., None, None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _attend(s, q, pages=None):
    case = s["case"]
    B, L, R, Rkv, H, P = (case[key] for key in ("B", "L", "R", "Rkv", "H", "P"))
    G, W = R // Rkv, s["page_table"].shape[1]
    x = _by_token(q, R, H, case["layout"]).view(B, L, Rkv, G, H).permute(0, 2, 1, 3, 4).reshape(B * Rkv, L * G, H)
    keys = _dequantised(s, "k").flatten(0, 1)
    scores = ((x * (1.0 / math.sqrt(H))) @ keys.transpose(1, 2)).view(B, Rkv, L, G, W * P)
    del keys
    at = torch.arange(W * P, device=x.device)
    seen = (at < _visible(s)[:, :, None])[:, None]                 # [B, 1, L, keys]
    if pages is not None:
        chosen = torch.zeros(B, L, Rkv, W + 1, dtype=torch.bool, device=x.device)
        chosen.scatter_(3, torch.where(pages >= 0, pages, W).long(), True)
        seen = seen & chosen.transpose(1, 2)[..., at // P]
    scores.masked_fill_(~seen[:, :, :, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    scores.sub_(top).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    out = (scores.view(B * Rkv, L * G, W * P) @ _dequantised(s, "v").flatten(0, 1)).view(B, Rkv, L, G, H)
    out = torch.where(total > 0, out / total, 0.0)
    out = _by_layout(out.permute(0, 2, 1, 3, 4).flatten(2, 3), case["layout"]).to(q.dtype)
    if not case["lse"]:
        return {"out": out}
    return {"out": out, "lse": (top + total.log())[..., 0].permute(0, 1, 3, 2).flatten(1, 2).contiguous()}


# ---- the calls ----

def _own_append(s):
    import fused_attn

    return fused_attn.cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_exponents"], s["v_exponents"], s["page_table"],
                                   s["starts"], new_lens=s["new_lens"], queries=s["q"], rope_cos=s["cos"], rope_sin=s["sin"],
                                   key_bounds=s.get("key_bounds"), layout=s["case"]["layout"])


def _own_select(s, q):
    import fused_attn

    return fused_attn.select_pages(q, s["key_bounds"], s["k_exponents"], s["page_table"], s["starts"], s["case"]["P"],
                                   s["case"]["count"], new_lens=s["new_lens"], layout=s["case"]["layout"])


def _own_attend(s, q, pages=None):
    import fused_attn

    r = fused_attn.cached_attention(q, s["k_cache"], s["v_cache"], s["k_exponents"], s["v_exponents"], s["page_table"], s["starts"],
                                    new_lens=s["new_lens"], pages=pages, return_lse=s["case"]["lse"], layout=s["case"]["layout"])
    return {"out": r[0], "lse": r[1]} if s["case"]["lse"] else {"out": r}


def _cache_of(s):
    return {key: s[key] for key in ("k_cache", "v_cache", "k_exponents", "v_exponents", "key_bounds") if key in s}


def run(state):
    op = state["case"]["op"]
    append, select, attend = (_own_append, _own_select, _own_attend) if own else (_append, _select, _attend)
    got, q = {}, state["q"]
    if op in ("append", "step", "sparse_step"):
        q = append(state)
        got = {"q": q, **_cache_of(state)}
    pages = None
    if op in ("select", "sparse", "sparse_step"):
        pages = got["pages"] = select(state, q)
    if op in ("attend", "step", "sparse", "sparse_step"):
        got.update(attend(state, q, pages))
    return got


def work(case):
    B, L, R, Rkv, H, P = (float(case[key]) for key in ("B", "L", "R", "Rkv", "H", "P"))
    op, ctx = case["op"], float(case["ctx"])
    # of the other sequences three quarters, on average; a chunk's tokens see half of it
    share = (1.0 + 0.75 * (B - 1)) / B if case["ragged"] else 1.0
    T = B * L * (share if L > 1 else 1.0)
    cached = B * ctx * share
    nbytes = flops = 0.0
    if op in ("append", "step", "sparse_step"):
        nbytes += T * H * (2 * R + 2 * 2 * Rkv + 2 * R + 2 * Rkv)  # read q, k, v; write q and the codes
        nbytes += 4.0 * min(T, ctx) * H if case["rope"] else 0.0
        nbytes += 2.0 * (T / P + B) * Rkv * (1 + (H if case["bounds"] else 0))
        flops += 3.0 * T * (R + Rkv) * H if case["rope"] else 0.0
    if op in ("select", "sparse", "sparse_step"):
        nbytes += cached / P * Rkv * 2 * H + 2.0 * T * R * H * (op == "select") + 4.0 * T * Rkv * case["count"]
        flops += 2.0 * T * R * 2 * H * cached / B / P
    if op in ("attend", "step", "sparse", "sparse_step"):
        keys = max(1.0, ctx * share - L / 2.0)                     # that a token sees
        if case["count"]:
            keys = min(keys, case["count"] * P)
        nbytes += min(cached, T * keys) * 2 * Rkv * H + 2.0 * T * R * H * (2 if op in ("attend", "sparse") else 1)
        nbytes += 4.0 * T * R if case["lse"] else 0.0
        flops += 4.0 * T * keys * R * H
    return {"bytes": nbytes, "flops": flops}


# ---- from the definitions, in 64 bits ----

def _two(e):
    """2^e in 64 bits, to the last bit (a power computed on the GPU may not be)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_append(s):
    """The queries, and of each cache tensor the values before they are rounded to 8 bits; the state's own tensors get the
    rounded ones."""
    case = s["case"]
    B, L, R, Rkv, H, P = (case[key] for key in ("B", "L", "R", "Rkv", "H", "P"))
    dev, half = s["starts"].device, H // 2
    starts, table = s["starts"].tolist(), s["page_table"].tolist()
    lens = s["new_lens"].tolist() if s["new_lens"] is not None else [L] * B

    def rotated(x, first):                                         # [n, heads, H]
        if s["cos"] is None:
            return x
        rows = slice(first, first + x.shape[0])
        turn = torch.complex(s["cos"][rows].double(), s["sin"][rows].double())[:, None]
        z = torch.complex(x[..., :half], x[..., half:]) * turn
        return torch.cat([z.real, z.imag], dim=-1)

    def tokens(x, b, n, heads):
        x = x[b, :n].view(n, heads, H) if case["layout"] == "blf" else x[b, :, :n].transpose(0, 1)
        return x.double()

    values = {name: s[name + "_cache"].to(torch.float64) for name in ("k", "v")}
    q = torch.zeros(B, L, R, H, dtype=torch.float64, device=dev)
    for b in range(B):
        first, n = starts[b], lens[b]
        q[b, :n] = rotated(tokens(s["q"], b, n, R), first)
        for name in ("k", "v"):
            y = tokens(s[name], b, n, Rkv)
            y = rotated(y, first) if name == "k" else y
            exponents = s[name + "_exponents"]
            for w in range(first // P, (first + n - 1) // P + 1):
                low, high = max(first, w * P), min(first + n, (w + 1) * P)
                page, part = table[b][w], y[low - first:high - first].transpose(0, 1)
                amax = part.abs().amax(dim=(1, 2)).clamp_min(1e-300)
                e = (amax / LARGEST_CODE).log2().ceil().clamp_min(LEAST_EXPONENT)
                e = torch.where(amax > LARGEST_CODE * _two(e), e + 1, torch.where(amax <= LARGEST_CODE * _two(e - 1), e - 1, e))
                e = e.clamp_min(LEAST_EXPONENT)
                before = exponents[page].double()
                e = torch.maximum(e, before) if low > w * P else e
                if low > w * P:
                    moved = values[name][page, :, :low - w * P] * _two(before - e)[:, None, None]
                    values[name][page, :, :low - w * P] = moved
                    s[name + "_cache"][page, :, :low - w * P] = _codes(moved.float())
                part = part * _two(-e)[:, None, None]
                values[name][page, :, low - w * P:high - w * P] = part
                s[name + "_cache"][page, :, low - w * P:high - w * P] = _codes(part.float())
                exponents[page] = e.to(torch.int8)
                if name == "k" and "key_bounds" in s:
                    up, down = (part.amax(dim=1) / 4).ceil(), (part.amin(dim=1) / 4).floor()
                    if low > w * P:
                        was = s["key_bounds"][page].double() * _two(before - e)[:, None, None]
                        up, down = torch.maximum(up, was[:, 0].ceil()), torch.minimum(down, was[:, 1].floor())
                    s["key_bounds"][page] = torch.stack([up, down], dim=1).to(torch.int8)
    return q, {**_cache_of(s), "k_cache": values["k"], "v_cache": values["v"]}


def _exact_select(s, q):
    """q [B, L, R, H] as the selection gets it, in 64 bits."""
    case = s["case"]
    B, L, R, Rkv, P, count = (case[key] for key in ("B", "L", "R", "Rkv", "P", "count"))
    seen = _visible(s).tolist()
    pages = torch.full((B, L, Rkv, count), -1, dtype=torch.int32, device=q.device)
    for b in range(B):
        W = -(-max(seen[b]) // P)
        ids = s["page_table"][b, :W].long()
        least = torch.tensor([max(n, 1) for n in seen[b]], device=q.device)
        page = torch.arange(W, device=q.device)
        for h in range(Rkv):
            x = q[b, :, h * (R // Rkv):(h + 1) * (R // Rkv)]
            amax = x.abs().amax(dim=(1, 2), keepdim=True).clamp_min(1e-300)
            e = (amax / 127).log2().ceil()
            e = torch.where(amax > 127 * _two(e), e + 1, torch.where(amax <= 127 * _two(e - 1), e - 1, e))
            x = (x * _two(-e)).round()
            up, down = (s["key_bounds"][ids, h, n].double() for n in (0, 1))
            dots = (x[:, :, None] * torch.where(x[:, :, None] > 0, up, down)).sum(dim=-1) if L * W < 4096 else \
                torch.relu(x) @ up.T - torch.relu(-x) @ down.T
            scores = dots.amax(dim=1) * _two(s["k_exponents"][ids, h])
            scores = torch.where(page * P < least[:, None], scores, -math.inf)
            scores[page == ((least - 1) // P)[:, None]] = math.inf
            order = torch.argsort(-scores, dim=1, stable=True)[:, :count]
            kept = torch.gather(scores, 1, order) > -math.inf
            order = torch.where(kept, order, W).sort(dim=1)[0]
            pages[b, :, h, :order.shape[1]] = torch.where(order < W, order, -1).to(torch.int32)
        pages[b, [i for i, n in enumerate(seen[b]) if n == 0]] = -1
    return pages


def _exact_attend(s, q, pages=None):
    """q [B, L, R, H] in 64 bits."""
    case = s["case"]
    B, L, R, Rkv, H, P = (case[key] for key in ("B", "L", "R", "Rkv", "H", "P"))
    G = R // Rkv
    seen = _visible(s)
    out = torch.zeros(B, L, R, H, dtype=torch.float64, device=q.device)
    lse = torch.full((B, R, L), -math.inf, dtype=torch.float64, device=q.device)
    most, lens = seen.amax(dim=1).tolist(), _lens(s).tolist()
    for b in range(B):
        n, keys = lens[b], most[b]
        ids = s["page_table"][b, :-(-keys // P)].long()
        hidden = torch.arange(keys, device=q.device) >= seen[b, :n, None]
        for h in range(Rkv):
            k, v = ((s[name + "_cache"][:, h].view(torch.uint8)[ids].view(torch.float8_e4m3fn).to(torch.float64) *
                     _two(s[name + "_exponents"][ids, h])[:, None, None]).flatten(0, 1)[:keys] for name in ("k", "v"))
            away = hidden
            if pages is not None:
                named = (pages[b, :n, h, :, None] == torch.arange(len(ids), device=q.device)).any(dim=1)
                away = hidden | ~named.repeat_interleave(P, dim=1)[:, :keys]
            heads = slice(h * G, (h + 1) * G)
            scores = (q[b, :n, heads].reshape(-1, H) @ k.T).div_(math.sqrt(H)).view(n, G, keys)
            scores.masked_fill_(away[:, None], -math.inf)
            sums = torch.logsumexp(scores, dim=2)
            scores = scores.sub_(sums[..., None]).exp_()
            out[b, :n, heads] = (scores.view(-1, keys) @ v).view(n, G, H)
            lse[b, heads, :n] = sums.T
    return {"out": _by_layout(out, case["layout"]), **({"lse": lse} if case["lse"] else {})}


def exact(case, seed):
    if case["B"] * case["Rkv"] > 1024 or case["B"] * -(-case["L"] // case["P"]) > 2048:
        return None                                                # loops that would take long
    s = prepare(case, seed)
    op = case["op"]
    q = (s["q"].view(case["B"], case["L"], case["R"], case["H"]) if case["layout"] == "blf" else s["q"].transpose(1, 2)).double()
    got = {}
    if op in ("append", "step", "sparse_step"):
        q, caches = _exact_append(s)
        got = {"q": _by_layout(q, case["layout"]), **caches}
        q = q.to(s["q"].dtype).double()                            # as the other operators get it
    pages = None
    if op in ("select", "sparse", "sparse_step"):
        pages = got["pages"] = _exact_select(s, q)
    if op in ("attend", "step", "sparse", "sparse_step"):
        got.update(_exact_attend(s, q, pages))
    return got
