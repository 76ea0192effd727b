"""ctypes view of libfused_attn_gfx950.so (the C ABI declared in include/fused_attn.h).

`forward` and `forward_timed` check what the library cannot see from raw addresses (tensor
devices, shapes, the mask's extent) and raise before any address reaches it; value ranges,
alignment and strides are checked by the library and reported through its status codes.
"""
import ctypes
import math
import os

_PKG_DIR = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG_DIR, "libfused_attn_gfx950.so")

# every symbol include/fused_attn.h declares
EXPORTS = ("fa_fwd", "fa_fwd_ex", "fa_fwd_strided", "fa_fwd_plan", "fa_fwd_variant", "fa_fwd_query", "fa_fwd_reference_bias", "fa_strerror",
           "fa_fwd_timed", "fa_fwd_timed_ex", "fa_qkv_proj", "fa_qkv_proj_plan", "fa_qkv_proj_variant",
           "fa_cache_append", "fa_cached_attention", "fa_cached_attention_workspace", "fa_cached_attention_plan", "fa_select_pages", "fa_select_pages_plan",
           "fa_rotary_tables", "fa_rotate", "fa_copy_pages", "fa_free_pages", "fa_take_pages", "fa_take_pages_workspace", "fa_fork_pages",
           "fa_fork_pages_workspace", "fa_compact_pages", "fa_compact_pages_workspace", "fa_latent_append", "fa_latent_attention",
           "fa_latent_attention_workspace", "fa_latent_attention_plan", "fa_expanded_attention", "fa_expanded_attention_workspace",
           "fa_expanded_attention_plan")
FLAG_CAUSAL = 1
FLAG_BF16 = 2
FLAG_INTERLEAVED = 4
FLAG_INVERSE = 8
ROTARY_SCALINGS = ("none", "linear", "base", "turns", "index")

_lib = None


class Cache(ctypes.Structure):
    """fa_cache: addresses and sizes of a paged key/value cache and its page table."""

    _fields_ = ([(name, ctypes.c_void_p) for name in ("keys", "values", "key_exponents", "value_exponents", "key_bounds", "page_table")] +
                [(name, ctypes.c_int64) for name in ("pages", "heads", "page_size", "head_dim", "sequences", "table_width", "table_stride")])


class Rotary(ctypes.Structure):
    """fa_rotary: how the frequencies of a rotary encoding are scaled."""

    _fields_ = [("scaling", ctypes.c_int)] + [(name, ctypes.c_double) for name in ("base", "factor", "original_rows", "low", "high", "amplitude")]


class Pages(ctypes.Structure):
    """fa_pages: a page table, the pages' uses and the tensors that pages hold."""

    _fields_ = ([(name, ctypes.c_void_p) for name in ("page_table", "starts", "uses")] +
                [(name, ctypes.c_int64) for name in ("pages", "page_size", "sequences", "table_width", "table_stride", "tensors")] +
                [("data", ctypes.c_void_p * 8), ("page_bytes", ctypes.c_int64 * 8)])


class LatentCache(ctypes.Structure):
    """fa_latent_cache: addresses and sizes of a paged cache of latents and its page table."""

    _fields_ = ([(name, ctypes.c_void_p) for name in ("latents", "page_table")] +
                [(name, ctypes.c_int64) for name in ("pages", "page_size", "latent_dim", "rope_dim", "sequences", "table_width", "table_stride")])


class Expanded(ctypes.Structure):
    """fa_expanded: addresses, sizes and strides of attention in the expanded form."""

    _fields_ = ([(name, ctypes.c_void_p) for name in ("q", "k", "rope_k", "v", "out", "lse", "starts", "new_lens")] +
                [(name, ctypes.c_int64) for name in ("sequences", "tokens", "heads", "keys", "key_dim", "rope_dim", "value_dim")] +
                [(name, ctypes.c_int64 * n) for name, n in (("q_strides", 3), ("k_strides", 3), ("rope_k_strides", 2), ("v_strides", 3),
                                                            ("out_strides", 3))])


class FusedAttnError(RuntimeError):
    """A non-zero status from the kernel library."""

    def __init__(self, status, text):
        super().__init__("%s (status %d)" % (text, status))
        self.status = status


def load_library():
    """Loads the kernel library once.  Raises OSError if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise OSError(
            "%s is missing: build it with `python -m fused_attention_amd.build` "
            "(there is no fallback implementation)" % LIB_PATH)
    lib = ctypes.CDLL(LIB_PATH)
    i64, vp, f32 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
    fwd_args = [vp, vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, f32, vp]
    lib.fa_fwd.argtypes = fwd_args
    lib.fa_fwd.restype = ctypes.c_int
    lib.fa_fwd_ex.argtypes = [vp, vp, vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, f32,
                              ctypes.c_int, vp]
    lib.fa_fwd_ex.restype = ctypes.c_int
    lib.fa_fwd_strided.argtypes = [vp, vp, vp, vp, vp, vp, i64, i64, i64, i64, i64, i64, i64, i64, i64, i64,
                                   f32, ctypes.c_int, vp]
    lib.fa_fwd_strided.restype = ctypes.c_int
    lib.fa_fwd_timed.argtypes = fwd_args + [ctypes.c_int, ctypes.POINTER(ctypes.c_float)]
    lib.fa_fwd_timed.restype = ctypes.c_int
    lib.fa_fwd_timed_ex.argtypes = lib.fa_fwd_strided.argtypes + [ctypes.c_int, ctypes.POINTER(ctypes.c_float)]
    lib.fa_fwd_timed_ex.restype = ctypes.c_int
    lib.fa_qkv_proj.argtypes = [vp, vp, vp, vp, i64, i64, i64, i64, i64, vp, vp, ctypes.c_int, vp]
    lib.fa_qkv_proj.restype = ctypes.c_int
    lib.fa_qkv_proj_plan.argtypes = [i64, i64, i64, i64, i64, ctypes.POINTER(ctypes.c_int)]
    lib.fa_qkv_proj_plan.restype = ctypes.c_int
    lib.fa_qkv_proj_variant.argtypes = [i64, i64, i64, i64, i64, ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    lib.fa_qkv_proj_variant.restype = ctypes.c_int
    lib.fa_fwd_plan.argtypes = [i64, i64, i64, i64, ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    lib.fa_fwd_plan.restype = ctypes.c_int
    lib.fa_fwd_variant.argtypes = lib.fa_fwd_plan.argtypes
    lib.fa_fwd_variant.restype = ctypes.c_int
    lib.fa_fwd_query.argtypes = [i64]
    lib.fa_fwd_query.restype = ctypes.c_int
    lib.fa_fwd_reference_bias.argtypes = [i64]
    lib.fa_fwd_reference_bias.restype = f32
    cache = ctypes.POINTER(Cache)
    lib.fa_cache_append.argtypes = [cache, vp, vp, i64, i64, i64, vp, i64, i64, i64, vp, i64, i64, i64, vp, vp, i64, i64, vp, vp, i64,
                                    ctypes.c_int, vp]
    lib.fa_cache_append.restype = ctypes.c_int
    lib.fa_cached_attention.argtypes = [cache, vp, i64, i64, i64, vp, i64, i64, i64, vp, vp, i64, vp, vp, i64, i64, f32, ctypes.c_int,
                                        vp, i64, vp]
    lib.fa_cached_attention.restype = ctypes.c_int
    lib.fa_cached_attention_workspace.argtypes = [cache, i64, i64, i64]
    lib.fa_cached_attention_workspace.restype = i64
    lib.fa_cached_attention_plan.argtypes = [cache, i64, i64, i64, ctypes.POINTER(ctypes.c_int)]
    lib.fa_cached_attention_plan.restype = ctypes.c_int
    lib.fa_select_pages.argtypes = [cache, vp, i64, i64, i64, vp, i64, vp, vp, i64, i64, ctypes.c_int, vp]
    lib.fa_select_pages.restype = ctypes.c_int
    lib.fa_select_pages_plan.argtypes = [cache, i64, i64, ctypes.POINTER(ctypes.c_int)]
    lib.fa_select_pages_plan.restype = ctypes.c_int
    pages, latent, expanded = ctypes.POINTER(Pages), ctypes.POINTER(LatentCache), ctypes.POINTER(Expanded)
    four = [vp, i64, i64, i64]                                     # a tensor and its strides
    for name, args, restype in (
            ("fa_rotary_tables", [vp, vp, i64, i64, ctypes.POINTER(Rotary), vp], ctypes.c_int),
            ("fa_rotate", four * 4 + [i64] * 7 + [vp, vp, i64, vp, vp, vp, ctypes.c_int, vp], ctypes.c_int),
            ("fa_copy_pages", [pages, vp, vp, i64, vp], ctypes.c_int),
            ("fa_free_pages", [pages, vp, i64, vp], ctypes.c_int),
            ("fa_take_pages", [pages, vp, i64, vp, vp, i64, vp], ctypes.c_int),
            ("fa_take_pages_workspace", [pages], i64),
            ("fa_fork_pages", [pages, vp, vp, i64, vp, vp, i64, vp], ctypes.c_int),
            ("fa_fork_pages_workspace", [i64], i64),
            ("fa_compact_pages", [pages, vp, vp, i64, vp], ctypes.c_int),
            ("fa_compact_pages_workspace", [pages], i64),
            ("fa_latent_append", [latent, vp, i64, i64, vp, i64, i64] + four * 2 + [vp, vp, i64, i64, vp, vp, i64, ctypes.c_int, vp], ctypes.c_int),
            ("fa_latent_attention", [latent] + four * 3 + [vp, vp, vp, i64, i64, f32, ctypes.c_int, vp, i64, vp], ctypes.c_int),
            ("fa_latent_attention_workspace", [latent, i64, i64], i64),
            ("fa_latent_attention_plan", [latent, i64, i64, ctypes.POINTER(ctypes.c_int)], ctypes.c_int),
            ("fa_expanded_attention", [expanded, f32, ctypes.c_int, vp, i64, vp], ctypes.c_int),
            ("fa_expanded_attention_workspace", [expanded], i64),
            ("fa_expanded_attention_plan", [expanded, ctypes.POINTER(ctypes.c_int)], ctypes.c_int)):
        getattr(lib, name).argtypes, getattr(lib, name).restype = args, restype
    lib.fa_strerror.argtypes = [ctypes.c_int]
    lib.fa_strerror.restype = ctypes.c_char_p
    _lib = lib
    return lib


def strerror(status):
    return load_library().fa_strerror(int(status)).decode()


def _check(status):
    if status != 0:
        raise FusedAttnError(status, strerror(status))


def launch_plan(B, R, L, H, causal=False, has_mask=False):
    """What fa_fwd_plan reports for a problem, as a dict.  Needs no GPU."""
    out = (ctypes.c_int * 7)()
    _check(load_library().fa_fwd_plan(B, R, L, H, FLAG_CAUSAL if causal else 0, 1 if has_mask else 0, out))
    keys = ("waves", "rows_per_wave", "workgroups", "working", "per_head", "heads_per_xcd", "matrix_tile")
    return dict(zip(keys, out))


def launch_variant(B, R, L, H, causal=False, has_mask=False):
    """What fa_fwd_variant reports for a problem, as a dict.  Needs no GPU."""
    out = (ctypes.c_int * 7)()
    _check(load_library().fa_fwd_variant(B, R, L, H, FLAG_CAUSAL if causal else 0, 1 if has_mask else 0, out))
    keys = ("kernel", "waves", "rows", "key_groups", "workgroups", "working", "per_head")
    res = dict(zip(keys, out))
    res["kernel"] = ("tile", "split", "group")[res["kernel"]]
    return res


def projection_plan(B, L, F_in, R, H):
    """What fa_qkv_proj_plan reports for a problem, as a dict.  Needs no GPU."""
    out = (ctypes.c_int * 4)()
    _check(load_library().fa_qkv_proj_plan(B, L, F_in, R, H, out))
    keys = ("workgroups", "working", "tiles", "tiles_n")
    return dict(zip(keys, out))


def projection_variant(B, L, F_in, R, H, rope=False):
    """What fa_qkv_proj_variant reports for a problem, as a dict.  Needs no GPU."""
    out = (ctypes.c_int * 6)()
    _check(load_library().fa_qkv_proj_variant(B, L, F_in, R, H, int(rope), out))
    return dict(zip(("tile_m", "tile_n", "workgroups", "working", "tiles", "tiles_n"), out))


def fwd_raw(q_ptr, k_ptr, v_ptr, mask_ptr, out_ptr, B, R, L, H, stride_b, stride_h, stride_l,
            scale, stream=0):
    """fa_fwd on raw device addresses (ints).  Returns the status code without raising."""
    return load_library().fa_fwd(q_ptr, k_ptr, v_ptr, mask_ptr or None, out_ptr, B, R, L, H,
                                 stride_b, stride_h, stride_l, scale, stream or None)


def _layout(q, head_dim, layout):
    if layout == "blf":      # [B, L, R*H]: the reference layout
        B, L, F = q.shape
        R = F // head_dim
        return B, R, L, L * F, head_dim, F
    if layout == "bhld":     # [B, R, L, H]
        B, R, L, H = q.shape
        return B, R, L, R * L * H, L * H, H
    raise ValueError("layout must be 'blf' or 'bhld'")


def _strides(t, head_dim, layout, name):
    """(stride_b, stride_h, stride_l) in elements of a tensor or view whose last dimension is dense."""
    if t.stride(-1) != 1:
        raise ValueError("%s: the last dimension must be contiguous" % name)
    if layout == "blf":
        return t.stride(0), head_dim, t.stride(1)
    return t.stride(0), t.stride(1), t.stride(2)


def _current_stream(q):
    import torch

    return torch.cuda.current_stream(q.device).cuda_stream


def _checked_problem(q, k, v, head_dim, out, mask, layout):
    """Everything the library cannot see from raw addresses, checked before any address reaches it
    (the same checks as the torch binding, reference src/fused_attn_extention.cu:24-64): dtypes,
    GPU residency on one device, dimensionality, equal shapes and strides, num_features a
    multiple of head_dim, a contiguous [B, L, L] mask.  Returns (B, R, L, q/k/v strides).
    Raises TypeError / ValueError; needs neither the library nor a GPU to do so."""
    import torch

    named = (("q", q), ("k", k), ("v", v), ("out", out), ("mask", mask))
    for name, t in named:
        if t is not None and not isinstance(t, torch.Tensor):
            raise TypeError("%s must be a torch.Tensor, got %s" % (name, type(t).__name__))
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("q, k, v must be float16 or bfloat16, got %s" % q.dtype)
    for name, t in named[1:]:
        if t is not None and t.dtype != q.dtype:
            raise TypeError("%s must have the dtype of q (%s), got %s" % (name, q.dtype, t.dtype))
    if int(head_dim) != head_dim or head_dim not in (16, 32, 64, 128):
        raise ValueError("head_dim must be 16, 32, 64 or 128, got %r" % (head_dim,))
    if layout not in ("blf", "bhld"):
        raise ValueError("layout must be 'blf' or 'bhld'")
    want_dim = 3 if layout == "blf" else 4
    if q.dim() != want_dim:
        raise ValueError("layout %r takes %d-D tensors, q has %d dimensions" % (layout, want_dim, q.dim()))
    if layout == "blf":
        if q.shape[2] % head_dim != 0:
            raise ValueError("num_features (%d) must be a multiple of head_dim (%d)" % (q.shape[2], head_dim))
    elif q.shape[3] != head_dim:
        raise ValueError("the last dimension (%d) must equal head_dim (%d)" % (q.shape[3], head_dim))
    if min(q.shape) < 1:
        raise ValueError("q must not have an empty dimension, got %s" % (tuple(q.shape),))
    if k.shape != q.shape or v.shape != q.shape:
        raise ValueError("q, k, v must have one shape")
    if out is not None and out.shape != q.shape:
        raise ValueError("out must have the shape of q")
    B, R, L = _layout(q, head_dim, layout)[:3]
    strides = _strides(q, head_dim, layout, "q")
    if _strides(k, head_dim, layout, "k") != strides or _strides(v, head_dim, layout, "v") != strides:
        raise ValueError("q, k, v must have the same strides")
    if mask is not None:
        if tuple(mask.shape) != (B, L, L):
            raise ValueError("mask must have shape [batch, seq_len, seq_len] = [%d, %d, %d], got %s"
                             % (B, L, L, tuple(mask.shape)))
        if not mask.is_contiguous():
            raise ValueError("mask must be contiguous")
    # last, so that the checks above can be exercised on host tensors
    for name, t in named:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("%s must be a GPU tensor, got device %s" % (name, t.device))
        if t.device != q.device:
            raise ValueError("%s is on %s but q is on %s" % (name, t.device, q.device))
    return B, R, L, strides


def forward(q, k, v, head_dim, out=None, mask=None, layout="blf", scale=None, causal=False,
            return_lse=False):
    """Runs fa_fwd_strided on torch GPU tensors (fp16 or bf16) on torch's current stream.

    layout 'blf' takes [B, L, R*head_dim] tensors, 'bhld' takes [B, R, L, head_dim] tensors.
    q, k and v may be views (slices of one packed projection output, say) as long as their last
    dimension is dense and the three have the same strides; `out` may be a view of its own.  The
    mask is contiguous [B, L, L].  causal=True restricts query i to keys j <= i.  q, k, v (and out,
    mask when given) must share one dtype and one GPU; bfloat16 tensors set FA_FLAG_BF16.  Returns
    `out` (allocated like q when not given), or (out, lse) with lse a float32 [B, R, L] tensor
    when return_lse is set.
    """
    import torch

    B, R, L, (sb, sh, sl) = _checked_problem(q, k, v, head_dim, out, mask, layout)
    flags = (FLAG_CAUSAL if causal else 0) | (FLAG_BF16 if q.dtype == torch.bfloat16 else 0)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ob, oh, ol = _strides(out, head_dim, layout, "out")
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    lse = torch.empty((B, R, L), dtype=torch.float32, device=q.device) if return_lse else None
    with torch.cuda.device(q.device):
        status = load_library().fa_fwd_strided(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), mask.data_ptr() if mask is not None else None,
            out.data_ptr(), lse.data_ptr() if lse is not None else None, B, R, L, head_dim, sb, sh, sl,
            ob, oh, ol, scale, flags, _current_stream(q) or None)
    _check(status)
    return (out, lse) if return_lse else out


def forward_timed(q, k, v, head_dim, out, iters, mask=None, layout="blf", scale=None, causal=False):
    """Average milliseconds per launch over `iters` back-to-back launches of the launch `forward`
    would make (HIP events on the launch stream, measured inside the library by fa_fwd_timed_ex).
    Same tensors as `forward` (fp16 or bf16, views allowed); `out` is required."""
    import torch

    B, R, L, (sb, sh, sl) = _checked_problem(q, k, v, head_dim, out, mask, layout)
    if out is None:
        raise ValueError("forward_timed needs an `out` tensor")
    flags = (FLAG_CAUSAL if causal else 0) | (FLAG_BF16 if q.dtype == torch.bfloat16 else 0)
    ob, oh, ol = _strides(out, head_dim, layout, "out")
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    ms = ctypes.c_float(0.0)
    with torch.cuda.device(q.device):
        status = load_library().fa_fwd_timed_ex(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), mask.data_ptr() if mask is not None else None,
            out.data_ptr(), None, B, R, L, head_dim, sb, sh, sl, ob, oh, ol, scale, flags,
            _current_stream(q) or None, int(iters), ctypes.byref(ms))
    _check(status)
    return float(ms.value)


def qkv_project(x, w, num_heads, head_dim, bias=None, rope=None, out=None):
    """fa_qkv_proj on torch GPU tensors, on torch's current stream: x [B, L, F_in] times w
    [F_in, 3 * num_heads * head_dim] (+ bias) -> packed [B, L, 3, num_heads * head_dim] (fp16 or
    bf16, like x).  rope = (cos, sin), float32 [L, head_dim / 2] tables of a rotate-half rotary
    encoding applied to the q and k slices.  The three slices out[:, :, s] are views that
    `forward` takes as q, k and v without a copy."""
    import torch

    for name, t in (("x", x), ("w", w), ("bias", bias), ("out", out)):
        if t is not None and not isinstance(t, torch.Tensor):
            raise TypeError("%s must be a torch.Tensor, got %s" % (name, type(t).__name__))
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("x must be float16 or bfloat16, got %s" % x.dtype)
    if x.dim() != 3 or w.dim() != 2:
        raise ValueError("x must be [B, L, F_in] and w [F_in, 3 F]")
    if int(head_dim) != head_dim or head_dim not in (16, 32, 64, 128):
        raise ValueError("head_dim must be 16, 32, 64 or 128, got %r" % (head_dim,))
    if int(num_heads) != num_heads or num_heads < 1:
        raise ValueError("num_heads must be a positive integer, got %r" % (num_heads,))
    B, L, f_in = x.shape
    F = num_heads * head_dim
    if F % 64 != 0:
        raise ValueError("num_heads * head_dim (%d) must be a multiple of 64: the three slices of the packed "
                         "output start on 64-feature boundaries" % F)
    if f_in % 64 != 0:
        raise ValueError("F_in (%d) must be a multiple of 64: the contraction is walked in steps of 64" % f_in)
    if tuple(w.shape) != (f_in, 3 * F):
        raise ValueError("w must have shape [F_in, 3 * num_heads * head_dim] = [%d, %d], got %s"
                         % (f_in, 3 * F, tuple(w.shape)))
    if bias is not None and tuple(bias.shape) != (3 * F,):
        raise ValueError("bias must have shape [%d], got %s" % (3 * F, tuple(bias.shape)))
    if out is None:
        out = torch.empty((B, L, 3, F), dtype=x.dtype, device=x.device)
    elif tuple(out.shape) != (B, L, 3, F):
        raise ValueError("out must have shape [%d, %d, 3, %d], got %s" % (B, L, F, tuple(out.shape)))
    tables = (None, None)
    if rope is not None:
        if isinstance(rope, torch.Tensor) or not isinstance(rope, (tuple, list)) or len(rope) != 2:
            raise ValueError("rope must be a pair (cos, sin) of float32 [L, head_dim / 2] tensors")
        tables = tuple(rope)
        for name, t in zip(("rope cos", "rope sin"), tables):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or tuple(t.shape) != (L, head_dim // 2):
                raise ValueError("%s must be a float32 tensor of shape [%d, %d]" % (name, L, head_dim // 2))
    for name, t in (("x", x), ("w", w), ("bias", bias), ("out", out), ("rope cos", tables[0]), ("rope sin", tables[1])):
        if t is None:
            continue
        if name in ("w", "bias", "out") and t.dtype != x.dtype:
            raise TypeError("%s must have the dtype of x (%s), got %s" % (name, x.dtype, t.dtype))
        if not t.is_contiguous():
            raise ValueError("%s must be contiguous" % name)
        if not t.is_cuda or t.device != x.device:
            raise ValueError("%s must be on the GPU of x, got device %s" % (name, t.device))
    flags = FLAG_BF16 if x.dtype == torch.bfloat16 else 0
    with torch.cuda.device(x.device):
        status = load_library().fa_qkv_proj(
            x.data_ptr(), w.data_ptr(), bias.data_ptr() if bias is not None else None, out.data_ptr(),
            B, L, f_in, num_heads, head_dim, tables[0].data_ptr() if rope is not None else None,
            tables[1].data_ptr() if rope is not None else None, flags, _current_stream(x) or None)
    _check(status)
    return out


def _kind(name, t, dtype, shape=None, contiguous=True):
    import torch

    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch.Tensor, got %s" % (name, type(t).__name__))
    if t.dtype != dtype:
        raise TypeError("%s must be %s, got %s" % (name, dtype, t.dtype))
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError("%s must have shape %s, got %s" % (name, list(shape), tuple(t.shape)))
    if contiguous and not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    return t


def _cache(k_exponents, page_table, starts, new_lens, page_size, head_dim, k_cache=None, v_cache=None, v_exponents=None,
           key_bounds=None):
    """The fa_cache of checked tensors, and the tensors."""
    import torch

    _kind("k_exponents", k_exponents, torch.int8)
    if k_exponents.dim() != 2 or k_exponents.numel() == 0:
        raise ValueError("k_exponents must be [pages, key heads], got %s" % (tuple(k_exponents.shape),))
    pages, heads = k_exponents.shape
    if head_dim not in (16, 32, 64, 128):
        raise ValueError("head_dim must be 16, 32, 64 or 128, got %r" % (head_dim,))
    if page_size not in (16, 32, 64, 128):
        raise ValueError("the pages must hold 16, 32, 64 or 128 tokens, got %r" % (page_size,))
    _kind("page_table", page_table, torch.int32, contiguous=False)
    if page_table.dim() != 2 or page_table.numel() == 0 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("page_table must be [batch, width] with dense rows, got %s" % (tuple(page_table.shape),))
    B, W = page_table.shape
    tensors = [k_exponents, page_table, _kind("starts", starts, torch.int32, (B,))]
    if new_lens is not None:
        tensors.append(_kind("new_lens", new_lens, torch.int32, (B,)))
    c = Cache(key_exponents=k_exponents.data_ptr(), page_table=page_table.data_ptr(), pages=pages, heads=heads, page_size=page_size,
              head_dim=head_dim, sequences=B, table_width=W, table_stride=page_table.stride(0) if B > 1 else W)
    if k_cache is not None:
        shape = (pages, heads, page_size, head_dim)
        c.keys = _kind("k_cache", k_cache, torch.float8_e4m3fn, shape).data_ptr()
        c.values = _kind("v_cache", v_cache, torch.float8_e4m3fn, shape).data_ptr()
        c.value_exponents = _kind("v_exponents", v_exponents, torch.int8, (pages, heads)).data_ptr()
        tensors += [k_cache, v_cache, v_exponents]
    if key_bounds is not None:
        c.key_bounds = _kind("key_bounds", key_bounds, torch.int8, (pages, heads, 2, head_dim)).data_ptr()
        tensors.append(key_bounds)
    return c, tensors


def _tokens(name, t, layout, c):
    """(L, heads, (stride_b, stride_h, stride_l)) of new tokens; the strides of dimensions of one element, which mean nothing,
    as the library takes them."""
    import torch

    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch.Tensor, got %s" % (name, type(t).__name__))
    if t.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("%s must be float16 or bfloat16, got %s" % (name, t.dtype))
    if layout not in ("blf", "bhld"):
        raise ValueError("layout must be 'blf' or 'bhld'")
    if t.dim() != (3 if layout == "blf" else 4):
        raise ValueError("layout %r takes %d-D tensors, %s has %d dimensions" % (layout, 3 if layout == "blf" else 4, name, t.dim()))
    if min(t.shape) < 1:
        raise ValueError("%s must not have an empty dimension, got %s" % (name, tuple(t.shape)))
    if t.shape[0] != c.sequences:
        raise ValueError("%s must have the batch of page_table (%d), got %s" % (name, c.sequences, tuple(t.shape)))
    if layout == "blf" and t.shape[2] % c.head_dim != 0:
        raise ValueError("the features of %s (%d) must be a multiple of head_dim (%d)" % (name, t.shape[2], c.head_dim))
    if layout == "bhld" and t.shape[3] != c.head_dim:
        raise ValueError("the last dimension of %s (%d) must equal head_dim (%d)" % (name, t.shape[3], c.head_dim))
    L, heads = (t.shape[1], t.shape[2] // c.head_dim) if layout == "blf" else (t.shape[2], t.shape[1])
    sb, sh, sl = _strides(t, c.head_dim, layout, name)
    return L, heads, (sb if c.sequences > 1 else 0, sh if heads > 1 else 0, sl if L > 1 else c.head_dim)


def _on_one_gpu(tensors):
    """Last, so that the checks before it can be exercised on host tensors."""
    for t in tensors:
        if not t.is_cuda or t.device != tensors[0].device:
            raise ValueError("all tensors must be on one GPU, got devices %s and %s" % (tensors[0].device, t.device))


def _query_tokens(queries, out, layout, c):
    import torch

    L, R, strides = _tokens("queries", queries, layout, c)
    if R % c.heads != 0:
        raise ValueError("the heads of queries (%d) must be a multiple of the key heads (%d)" % (R, c.heads))
    if out is not None and not isinstance(out, torch.Tensor):
        raise TypeError("out must be a torch.Tensor, got %s" % type(out).__name__)
    if out is not None and (out.shape != queries.shape or out.dtype != queries.dtype):
        raise ValueError("out must have the shape and dtype of queries")
    return L, R, strides


def cache_append(keys, values, k_cache, v_cache, k_exponents, v_exponents, page_table, starts, new_lens=None, queries=None,
                 rope=None, key_bounds=None, layout="blf", out=None):
    """fa_cache_append on torch GPU tensors, on torch's current stream: appends keys (rotated by rope = (cos, sin), float32
    [positions, head_dim / 2] tables) and values to the cache in place.  Returns the rotated queries (`out`, allocated when not
    given), or None without queries.  The cache's tensors are described in include/fused_attn.h."""
    import torch

    if _kind("k_cache", k_cache, torch.float8_e4m3fn).dim() != 4:
        raise ValueError("k_cache must be [pages, key heads, page_size, head_dim], got %s" % (tuple(k_cache.shape),))
    c, tensors = _cache(k_exponents, page_table, starts, new_lens, k_cache.shape[2], k_cache.shape[3], k_cache, v_cache, v_exponents,
                        key_bounds)
    L, heads, kv = _tokens("keys", keys, layout, c)
    if heads != c.heads:
        raise ValueError("keys must have the key heads of the cache (%d), got %d" % (c.heads, heads))
    if _tokens("values", values, layout, c) != (L, heads, kv) or values.dtype != keys.dtype or values.shape != keys.shape:
        raise ValueError("values must have the dtype, shape and strides of keys")
    R, q, o = c.heads, (0, 0, 0), (0, 0, 0)
    if queries is None and out is not None:
        raise ValueError("out goes with queries")
    if queries is not None:
        Lq, R, q = _query_tokens(queries, out, layout, c)
        if Lq != L or queries.dtype != keys.dtype:
            raise ValueError("queries must have the seq_len and dtype of keys")
        out = torch.empty(queries.shape, dtype=queries.dtype, device=queries.device) if out is None else out
        o = _tokens("out", out, layout, c)[2]
    tables = (None, None)
    if rope is not None:
        if isinstance(rope, torch.Tensor) or not isinstance(rope, (tuple, list)) or len(rope) != 2:
            raise ValueError("rope must be a pair (cos, sin) of float32 [positions, head_dim / 2] tensors")
        tables = tuple(rope)
        for name, t in zip(("rope cos", "rope sin"), tables):
            _kind(name, t, torch.float32)
            if tuple(t.shape) != (len(tables[0]), c.head_dim // 2) or len(t) == 0:
                raise ValueError("%s must be [positions, head_dim / 2 = %d], one shape for both, got %s" % (name, c.head_dim // 2, tuple(t.shape)))
    _on_one_gpu(tensors + [keys, values] + [t for t in (queries, out) + tables if t is not None])
    with torch.cuda.device(keys.device):
        _check(load_library().fa_cache_append(
            ctypes.byref(c), keys.data_ptr(), values.data_ptr(), *kv, queries.data_ptr() if queries is not None else None, *q,
            out.data_ptr() if queries is not None else None, *o, starts.data_ptr(),
            new_lens.data_ptr() if new_lens is not None else None, L, R, tables[0].data_ptr() if rope is not None else None,
            tables[1].data_ptr() if rope is not None else None, tables[0].shape[0] if rope is not None else 0,
            FLAG_BF16 if keys.dtype == torch.bfloat16 else 0, _current_stream(keys) or None))
    return out


def _bytes(status):
    if status < 0:
        _check(int(status))
    return status


def cached_attention(queries, k_cache, v_cache, k_exponents, v_exponents, page_table, starts, new_lens=None, pages=None, causal=True,
                     return_lse=False, layout="blf", scale=None, out=None):
    """fa_cached_attention on torch GPU tensors, on torch's current stream: attention of new tokens over the cache, or over the
    pages that `pages`, int32 [batch, seq_len, key heads, count], lists.  Returns `out` (allocated when not given), or
    (out, lse)."""
    import torch

    if _kind("k_cache", k_cache, torch.float8_e4m3fn).dim() != 4:
        raise ValueError("k_cache must be [pages, key heads, page_size, head_dim], got %s" % (tuple(k_cache.shape),))
    c, tensors = _cache(k_exponents, page_table, starts, new_lens, k_cache.shape[2], k_cache.shape[3], k_cache, v_cache, v_exponents)
    L, R, q = _query_tokens(queries, out, layout, c)
    count = 0
    if pages is not None:
        _kind("pages", pages, torch.int32)
        if pages.dim() != 4 or tuple(pages.shape[:3]) != (c.sequences, L, c.heads) or pages.shape[3] < 1:
            raise ValueError("pages must be [batch, seq_len, key heads, count], got %s" % (tuple(pages.shape),))
        count = pages.shape[3]
    out = torch.empty(queries.shape, dtype=queries.dtype, device=queries.device) if out is None else out
    o = _tokens("out", out, layout, c)[2]
    _on_one_gpu(tensors + [queries, out] + ([pages] if pages is not None else []))
    lib = load_library()
    lse = torch.empty((c.sequences, R, L), dtype=torch.float32, device=queries.device) if return_lse else None
    nbytes = _bytes(lib.fa_cached_attention_workspace(ctypes.byref(c), L, R, count))
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=queries.device) if nbytes else None
    flags = (FLAG_CAUSAL if causal else 0) | (FLAG_BF16 if queries.dtype == torch.bfloat16 else 0)
    with torch.cuda.device(queries.device):
        _check(lib.fa_cached_attention(
            ctypes.byref(c), queries.data_ptr(), *q, out.data_ptr(), *o, lse.data_ptr() if return_lse else None,
            pages.data_ptr() if pages is not None else None, count, starts.data_ptr(),
            new_lens.data_ptr() if new_lens is not None else None, L, R, 1.0 / math.sqrt(c.head_dim) if scale is None else scale, flags,
            workspace.data_ptr() if nbytes else None, nbytes, _current_stream(queries) or None))
    return (out, lse) if return_lse else out


def select_pages(queries, key_bounds, k_exponents, page_table, starts, page_size, count, new_lens=None, layout="blf"):
    """fa_select_pages on torch GPU tensors, on torch's current stream.  Returns int32 [batch, seq_len, key heads, count]."""
    import torch

    if _kind("key_bounds", key_bounds, torch.int8).dim() != 4:
        raise ValueError("key_bounds must be [pages, key heads, 2, head_dim], got %s" % (tuple(key_bounds.shape),))
    c, tensors = _cache(k_exponents, page_table, starts, new_lens, page_size, key_bounds.shape[3], key_bounds=key_bounds)
    L, R, q = _query_tokens(queries, None, layout, c)
    if int(count) != count or not 1 <= count <= 4096:
        raise ValueError("count must be between 1 and 4096, got %r" % (count,))
    _on_one_gpu(tensors + [queries])
    selected = torch.empty((c.sequences, L, c.heads, count), dtype=torch.int32, device=queries.device)
    with torch.cuda.device(queries.device):
        _check(load_library().fa_select_pages(
            ctypes.byref(c), queries.data_ptr(), *q, selected.data_ptr(), count, starts.data_ptr(),
            new_lens.data_ptr() if new_lens is not None else None, L, R, FLAG_BF16 if queries.dtype == torch.bfloat16 else 0,
            _current_stream(queries) or None))
    return selected


def _sizes(B, Rkv, H, P, W, pages=1):
    return ctypes.byref(Cache(pages=pages, heads=Rkv, page_size=P, head_dim=H, sequences=B, table_width=W, table_stride=W))


def cached_attention_plan(B, L, R, Rkv, H, P, W, count=0):
    """What fa_cached_attention_plan reports for a problem, as a dict.  Needs no GPU."""
    out = (ctypes.c_int * 5)()
    _check(load_library().fa_cached_attention_plan(_sizes(B, Rkv, H, P, W), L, R, count, out))
    res = dict(zip(("kernel", "waves", "rows", "splits", "workgroups"), out))
    res["kernel"] = ("few", "many", "joined")[res["kernel"]]
    return res


def select_pages_plan(B, L, R, Rkv, H, P, W):
    """What fa_select_pages_plan reports for a problem, as a dict.  Needs no GPU."""
    out = (ctypes.c_int * 3)()
    _check(load_library().fa_select_pages_plan(_sizes(B, Rkv, H, P, W), L, R, out))
    return dict(zip(("tokens", "waves", "workgroups"), out))


# ---- rotary positions, the pages of a cache, latent attention ----

def _half(name, t, like=None, dims=None):
    import torch

    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch.Tensor, got %s" % (name, type(t).__name__))
    if t.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("%s must be float16 or bfloat16, got %s" % (name, t.dtype))
    if like is not None and t.dtype != like.dtype:
        raise TypeError("%s must have the dtype %s, got %s" % (name, like.dtype, t.dtype))
    if dims is not None and t.dim() != dims:
        raise ValueError("%s must have %d dimensions, got %s" % (name, dims, tuple(t.shape)))
    if t.numel() == 0:
        raise ValueError("%s must not have an empty dimension, got %s" % (name, tuple(t.shape)))
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError("the last dimension of %s must be contiguous" % name)
    return t


def _ints(name, t, n=None):
    import torch

    if t is None:
        return None
    _kind(name, t, torch.int32)
    if t.dim() != 1 or (n is not None and t.shape[0] != n):
        raise ValueError("%s must have shape %s, got %s" % (name, "[n]" if n is None else [n], tuple(t.shape)))
    return t


def _rope(rope, dims=None):
    """(cos, sin) and what they are, or Nones."""
    import torch

    if rope is None:
        return None, None, 0, 0
    if isinstance(rope, torch.Tensor) or not isinstance(rope, (tuple, list)) or len(rope) != 2:
        raise ValueError("rope must be a pair (cos, sin) of float32 [positions, dimensions / 2] tensors")
    cos, sin = rope
    for name, t in (("rope cos", cos), ("rope sin", sin)):
        _kind(name, t, torch.float32)
        if t.dim() != 2 or t.numel() == 0 or t.shape != cos.shape or (dims is not None and t.shape[1] != dims // 2):
            raise ValueError("%s must be [positions, %s], one shape for both, got %s" % (name, "dimensions / 2" if dims is None else dims // 2, tuple(t.shape)))
    return cos, sin, cos.shape[0], 2 * cos.shape[1]


def _address(t):
    return t.data_ptr() if t is not None else None


def _bf16(t):
    import torch

    return FLAG_BF16 if t.dtype == torch.bfloat16 else 0


def rotary_tables(rows, rotary_dim, device="cuda", base=10000.0, scaling="none", factor=1.0, original_rows=None, low=1.0, high=4.0, amplitude=1.0):
    """fa_rotary_tables on torch's current stream: (cos, sin), float32 [rows, rotary_dim / 2]."""
    import torch

    if scaling not in ROTARY_SCALINGS:
        raise ValueError("scaling must be one of %s, got %r" % (", ".join(ROTARY_SCALINGS), scaling))
    if int(rows) != rows or rows < 1:
        raise ValueError("rows must be at least 1, got %r" % (rows,))
    if int(rotary_dim) != rotary_dim or rotary_dim % 16 != 0 or not 16 <= rotary_dim <= 256:
        raise ValueError("rotary_dim must be a multiple of 16 up to 256, got %r" % (rotary_dim,))
    if not (factor > 0 and math.isfinite(factor)):
        raise ValueError("factor must be positive, got %r" % (factor,))
    how = Rotary(ROTARY_SCALINGS.index(scaling), base, factor, rows / factor if original_rows is None else original_rows, low, high, amplitude)
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("device must be a GPU, got %s" % device)
    cos, sin = (torch.empty((rows, rotary_dim // 2), dtype=torch.float32, device=device) for _ in range(2))
    with torch.cuda.device(cos.device):
        _check(load_library().fa_rotary_tables(cos.data_ptr(), sin.data_ptr(), rows, rotary_dim, ctypes.byref(how), _current_stream(cos) or None))
    return cos, sin


def _head_rows(name, t, layout, head_dim, like):
    """(batch, L, heads, strides) in either layout, strides of dimensions of one element as the library takes them."""
    _half(name, t, like, 3 if layout == "blf" else 4)
    if layout == "blf" and t.shape[2] % head_dim != 0:
        raise ValueError("the features of %s (%d) must be a multiple of head_dim (%d)" % (name, t.shape[2], head_dim))
    if layout == "bhld" and t.shape[3] != head_dim:
        raise ValueError("the last dimension of %s (%d) must equal head_dim (%d)" % (name, t.shape[3], head_dim))
    B, L, heads = (t.shape[0], t.shape[1], t.shape[2] // head_dim) if layout == "blf" else (t.shape[0], t.shape[2], t.shape[1])
    sb, sh, sl = (t.stride(0), head_dim, t.stride(1)) if layout == "blf" else t.stride()[:3]
    return B, L, heads, (sb if B > 1 else 0, sh if heads > 1 else 0, sl if L > 1 else head_dim)


def rotate(queries, rope, head_dim, keys=None, starts=None, new_lens=None, positions=None, first=0, interleaved=False, inverse=False, layout="blf",
           out=None):
    """fa_rotate on torch GPU tensors, on torch's current stream: queries, and keys beside them, rotated by rope = (cos, sin), float32
    [positions, dimensions / 2].  `out`: what is written, queries or (queries, keys); the inputs themselves rotate in place.  Returns it."""
    import torch

    if int(head_dim) != head_dim or head_dim % 16 != 0 or not 16 <= head_dim <= 1024:
        raise ValueError("head_dim must be a multiple of 16 up to 1024, got %r" % (head_dim,))
    if layout not in ("blf", "bhld"):
        raise ValueError("layout must be 'blf' or 'bhld'")
    if rope is None:
        raise ValueError("rope must be a pair (cos, sin)")
    cos, sin, rows, dims = _rope(rope)
    if dims % 16 != 0 or int(first) != first or first < 0 or first % 8 != 0 or first + dims > head_dim:
        raise ValueError("first must be a multiple of 8 and the tables' %d channels, a multiple of 16, must lie within head_dim (%d), got first %r"
                         % (dims, head_dim, first))
    inputs = [queries] if keys is None else [queries, keys]
    shapes = [_head_rows(name, t, layout, head_dim, queries) for name, t in zip(("queries", "keys"), inputs)]
    B, L, R, _ = shapes[0]
    if keys is not None and shapes[1][:2] != (B, L):
        raise ValueError("keys must have the batch and seq_len of queries, got %s" % (tuple(keys.shape),))
    if starts is not None and positions is not None:
        raise ValueError("starts and positions exclude each other")
    _ints("starts", starts, B), _ints("new_lens", new_lens, B)
    if positions is not None:
        _kind("positions", positions, torch.int32, (B, L))
    outs = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in inputs] if out is None else list(out) if isinstance(out, (tuple, list)) else [out]
    if len(outs) != len(inputs):
        raise ValueError("out must be as many tensors as are rotated")
    for t, x in zip(outs, inputs):
        if not isinstance(t, torch.Tensor) or t.shape != x.shape or t.dtype != x.dtype:
            raise ValueError("out must have the shape and dtype of what is rotated")
    outs_at = [_head_rows("out", t, layout, head_dim, queries)[3] for t in outs]
    if out is not None and torch.is_grad_enabled() and any(t.requires_grad for t in outs):
        raise ValueError("out requires a gradient, which the call does not record: rotate within a torch.autograd.Function, or under torch.no_grad()")
    _on_one_gpu(inputs + outs + [t for t in (cos, sin, starts, new_lens, positions) if t is not None])
    flags = _bf16(queries) | (FLAG_INTERLEAVED if interleaved else 0) | (FLAG_INVERSE if inverse else 0)
    k = (keys.data_ptr(), *shapes[1][3], outs[1].data_ptr(), *outs_at[1]) if keys is not None else (None, 0, 0, 0) * 2
    with torch.cuda.device(queries.device):
        _check(load_library().fa_rotate(
            queries.data_ptr(), *shapes[0][3], outs[0].data_ptr(), *outs_at[0], *k, B, L, R, shapes[-1][2] if keys is not None else 0, head_dim,
            first, dims, cos.data_ptr(), sin.data_ptr(), rows, _address(positions), _address(starts), _address(new_lens), flags,
            _current_stream(queries) or None))
    if out is not None:                                            # autograd sees that what it may have kept of them is gone
        torch.autograd.graph.increment_version([t for t in outs if not t.is_inference()])
    return outs[0] if keys is None else tuple(outs)


def _pages(page_table, uses, starts=None, page_size=16, tensors=None):
    """The fa_pages of checked tensors, and the tensors."""
    import torch

    c, held = Pages(page_size=page_size), []
    if uses is not None:
        _ints("uses", uses)
        if uses.numel() == 0:
            raise ValueError("uses must be [pages], got %s" % (tuple(uses.shape),))
        _kind("page_table", page_table, torch.int32, contiguous=False)
        if page_table.dim() != 2 or page_table.numel() == 0 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
            raise ValueError("page_table must be [sequences, width] with dense rows, got %s" % (tuple(page_table.shape),))
        if page_size not in (16, 32, 64, 128):
            raise ValueError("page_size must be 16, 32, 64 or 128, got %r" % (page_size,))
        S, W = page_table.shape
        c.page_table, c.uses, c.pages, c.sequences, c.table_width = page_table.data_ptr(), uses.data_ptr(), uses.shape[0], S, W
        c.table_stride = page_table.stride(0) if S > 1 else W
        held = [uses, page_table]
    if starts is not None:
        c.starts = _ints("starts", starts, page_table.shape[0]).data_ptr()
        held.append(starts)
    if tensors is not None:
        if isinstance(tensors, torch.Tensor) or not 1 <= len(tensors) <= 8:
            raise ValueError("tensors must be one to eight of a cache")
        for n, t in enumerate(tensors):
            if not isinstance(t, torch.Tensor):
                raise TypeError("tensors must be torch.Tensors, got %s" % type(t).__name__)
            if t.dim() < 1 or t.numel() == 0 or not t.is_contiguous():
                raise ValueError("tensors must be contiguous [pages, ...], got %s" % (tuple(t.shape),))
            c.pages = c.pages or t.shape[0]
            if t.shape[0] != c.pages:
                raise ValueError("tensors must have the same pages (%d), got %s" % (c.pages, tuple(t.shape)))
            c.data[n], c.page_bytes[n] = t.data_ptr(), t.numel() // t.shape[0] * t.element_size()
        c.tensors = len(tensors)
        held += list(tensors)
    return c, held


def _keep(call, like, c, *args, workspace=None):
    """One of the page keeping's calls, with a workspace of its size where it takes one."""
    import torch

    lib = load_library()
    if workspace is not None:
        nbytes = _bytes(workspace(lib))
        room = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=like.device)
        args += (room.data_ptr(), nbytes)
    with torch.cuda.device(like.device):
        _check(getattr(lib, call)(ctypes.byref(c), *args, _current_stream(like) or None))


def copy_pages(tensors, sources, targets):
    """fa_copy_pages on torch GPU tensors, on torch's current stream: page sources[n] into page targets[n] of every tensor."""
    c, held = _pages(None, None, tensors=tensors)
    _ints("sources", sources), _ints("targets", targets)
    if len(sources) != len(targets):
        raise ValueError("targets must be as many as sources (%d), got %d" % (len(sources), len(targets)))
    _on_one_gpu(held + [sources, targets])
    if len(sources):
        _keep("fa_copy_pages", sources, c, sources.data_ptr(), targets.data_ptr(), len(sources))


def free_pages(page_table, starts, uses, sequences):
    """fa_free_pages on torch GPU tensors, on torch's current stream."""
    c, held = _pages(page_table, uses, starts)
    _ints("sequences", sequences)
    _on_one_gpu(held + [sequences])
    if len(sequences):
        _keep("fa_free_pages", uses, c, sequences.data_ptr(), len(sequences))


def take_pages(page_table, starts, uses, page_size, seq_len, new_lens=None):
    """fa_take_pages on torch GPU tensors, on torch's current stream.  Returns int32 [sequences]: the pages that each lacks."""
    import torch

    c, held = _pages(page_table, uses, starts, page_size)
    if int(seq_len) != seq_len or seq_len < 1:
        raise ValueError("seq_len must be at least 1, got %r" % (seq_len,))
    _ints("new_lens", new_lens, page_table.shape[0])
    _on_one_gpu(held + ([new_lens] if new_lens is not None else []))
    missing = torch.empty(page_table.shape[0], dtype=torch.int32, device=uses.device)
    _keep("fa_take_pages", uses, c, _address(new_lens), seq_len, missing.data_ptr(), workspace=lambda lib: lib.fa_take_pages_workspace(ctypes.byref(c)))
    return missing


def fork_pages(tensors, page_table, starts, uses, page_size, parents, children):
    """fa_fork_pages on torch GPU tensors, on torch's current stream.  Returns int32 [forks]: 1 for each that happened."""
    import torch

    c, held = _pages(page_table, uses, starts, page_size, tensors)
    _ints("parents", parents), _ints("children", children)
    if len(parents) != len(children):
        raise ValueError("children must be as many as parents (%d), got %d" % (len(parents), len(children)))
    if len(parents) > 4096:
        raise ValueError("at most 4096 forks at once, got %d" % len(parents))
    _on_one_gpu(held + [parents, children])
    forked = torch.empty(len(parents), dtype=torch.int32, device=uses.device)
    if len(parents):
        _keep("fa_fork_pages", uses, c, parents.data_ptr(), children.data_ptr(), len(parents), forked.data_ptr(),
              workspace=lambda lib: lib.fa_fork_pages_workspace(len(parents)))
    return forked


def compact_pages(tensors, page_table, uses):
    """fa_compact_pages on torch GPU tensors, on torch's current stream.  Returns int32 [pages]: where each is now, -1 for free ones."""
    import torch

    c, held = _pages(page_table, uses, tensors=tensors)
    _on_one_gpu(held)
    moved = torch.empty(uses.shape[0], dtype=torch.int32, device=uses.device)
    _keep("fa_compact_pages", uses, c, moved.data_ptr(), workspace=lambda lib: lib.fa_compact_pages_workspace(ctypes.byref(c)))
    return moved


def _latent_cache(latent_cache, page_table, starts, new_lens, rope_dim):
    import torch

    _half("latent_cache", latent_cache, dims=3)
    if not latent_cache.is_contiguous():
        raise ValueError("latent_cache must be contiguous")
    pages, page_size, channels = latent_cache.shape
    if rope_dim not in (32, 64):
        raise ValueError("the rotary channels must be 32 or 64, got %r" % (rope_dim,))
    if channels - rope_dim not in (128, 256, 512):
        raise ValueError("the latent channels must be 128, 256 or 512, got %d beside %d rotary ones" % (channels - rope_dim, rope_dim))
    if page_size not in (16, 32, 64, 128):
        raise ValueError("the pages must hold 16, 32, 64 or 128 tokens, got %r" % (page_size,))
    _kind("page_table", page_table, torch.int32, contiguous=False)
    if page_table.dim() != 2 or page_table.numel() == 0 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("page_table must be [batch, width] with dense rows, got %s" % (tuple(page_table.shape),))
    B, W = page_table.shape
    _kind("starts", starts, torch.int32, (B,)), _ints("new_lens", new_lens, B)
    c = LatentCache(latents=latent_cache.data_ptr(), page_table=page_table.data_ptr(), pages=pages, page_size=page_size, latent_dim=channels - rope_dim,
                    rope_dim=rope_dim, sequences=B, table_width=W, table_stride=page_table.stride(0) if B > 1 else W)
    return c, [latent_cache, page_table, starts] + ([new_lens] if new_lens is not None else [])


def _by_heads(name, t, like, batch, shape=None):
    """The strides (b, h, l) of [batch, seq_len, heads, channels]."""
    _half(name, t, like, 4)
    if t.shape[0] != batch or (shape is not None and tuple(t.shape) != tuple(shape)):
        raise ValueError("%s must be [%d, seq_len, heads, channels]%s, got %s" % (name, batch, "" if shape is None else " = %s" % (list(shape),), tuple(t.shape)))
    return (t.stride(0) if batch > 1 else 0, t.stride(2) if t.shape[2] > 1 else 0, t.stride(1) if t.shape[1] > 1 else t.shape[3])


def _by_rows(name, t, like, shape):
    """The strides (b, l) of [batch, seq_len, channels]."""
    _half(name, t, like, 3)
    if tuple(t.shape) != tuple(shape):
        raise ValueError("%s must be %s, got %s" % (name, list(shape), tuple(t.shape)))
    return (t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else t.shape[2])


def latent_append(latents, rope_keys, latent_cache, page_table, starts, new_lens=None, queries=None, rope=None, interleaved=False):
    """fa_latent_append on torch GPU tensors, on torch's current stream.  Returns the rotated queries, or None without queries."""
    import torch

    _half("rope_keys", rope_keys, dims=3), _half("latents", latents, dims=3)
    c, held = _latent_cache(latent_cache, page_table, starts, new_lens, rope_keys.shape[2])
    L = latents.shape[1]
    x = _by_rows("latents", latents, latent_cache, (c.sequences, L, c.latent_dim))
    k = _by_rows("rope_keys", rope_keys, latent_cache, (c.sequences, L, c.rope_dim))
    q, o, out, R = (0, 0, 0), (0, 0, 0), None, 1
    if queries is not None:
        _half("queries", queries, dims=4)
        R = queries.shape[2]
        q = _by_heads("queries", queries, latent_cache, c.sequences, (c.sequences, L, R, c.rope_dim))
    cos, sin, rows, _ = _rope(rope, c.rope_dim)
    _on_one_gpu(held + [latents, rope_keys] + [t for t in (queries, cos, sin) if t is not None])
    if queries is not None:
        out = torch.empty(queries.shape, dtype=queries.dtype, device=queries.device)
        o = _by_heads("out", out, latent_cache, c.sequences)
    with torch.cuda.device(latent_cache.device):
        _check(load_library().fa_latent_append(
            ctypes.byref(c), latents.data_ptr(), *x, rope_keys.data_ptr(), *k, _address(queries), *q, _address(out), *o, starts.data_ptr(),
            _address(new_lens), L, R, _address(cos), _address(sin), rows, _bf16(latent_cache) | (FLAG_INTERLEAVED if interleaved else 0),
            _current_stream(latent_cache) or None))
    return out


def latent_attention(queries, rope_queries, latent_cache, page_table, starts, scale, new_lens=None, causal=True, return_lse=False):
    """fa_latent_attention on torch GPU tensors, on torch's current stream.  Returns out, or (out, lse)."""
    import torch

    _half("rope_queries", rope_queries, dims=4), _half("queries", queries, dims=4)
    c, held = _latent_cache(latent_cache, page_table, starts, new_lens, rope_queries.shape[3])
    B, L, R, _ = queries.shape
    q = _by_heads("queries", queries, latent_cache, c.sequences, (c.sequences, L, R, c.latent_dim))
    r = _by_heads("rope_queries", rope_queries, latent_cache, c.sequences, (c.sequences, L, R, c.rope_dim))
    _on_one_gpu(held + [queries, rope_queries])
    lib = load_library()
    out = torch.empty(queries.shape, dtype=queries.dtype, device=queries.device)
    o = _by_heads("out", out, latent_cache, c.sequences)
    lse = torch.empty((B, R, L), dtype=torch.float32, device=queries.device) if return_lse else None
    nbytes = _bytes(lib.fa_latent_attention_workspace(ctypes.byref(c), L, R))
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=queries.device) if nbytes else None
    with torch.cuda.device(queries.device):
        _check(lib.fa_latent_attention(
            ctypes.byref(c), queries.data_ptr(), *q, rope_queries.data_ptr(), *r, out.data_ptr(), *o, _address(lse), starts.data_ptr(),
            _address(new_lens), L, R, scale, (FLAG_CAUSAL if causal else 0) | _bf16(queries), _address(workspace), nbytes,
            _current_stream(queries) or None))
    return (out, lse) if return_lse else out


def expanded_attention(queries, keys, rope_keys, values, starts=None, new_lens=None, causal=True, return_lse=False, scale=None):
    """fa_expanded_attention on torch GPU tensors, on torch's current stream.  Returns out, or (out, lse)."""
    import torch

    for name, t in (("queries", queries), ("keys", keys), ("values", values)):
        _half(name, t, dims=4)
    B, L, R, _ = queries.shape
    K, D = keys.shape[1], keys.shape[3]
    DR = queries.shape[3] - D
    if D not in (64, 128):
        raise ValueError("keys must have 64 or 128 channels, got %d" % D)
    if DR not in (32, 64):
        raise ValueError("queries must have 32 or 64 rotary channels behind the %d of keys, got %d" % (D, queries.shape[3]))
    q = _by_heads("queries", queries, queries, B)
    k, v = (_by_heads(name, t, queries, B, (B, K, R, D)) for name, t in (("keys", keys), ("values", values)))
    kr = _by_rows("rope_keys", rope_keys, queries, (B, K, DR))
    if starts is None and K < L:
        raise ValueError("without starts the keys (%d) must be at least as many as the queries (%d)" % (K, L))
    _ints("starts", starts, B), _ints("new_lens", new_lens, B)
    _on_one_gpu([queries, keys, rope_keys, values] + [t for t in (starts, new_lens) if t is not None])
    lib = load_library()
    out = torch.empty((B, L, R, D), dtype=queries.dtype, device=queries.device)
    o = _by_heads("out", out, queries, B)
    lse = torch.empty((B, R, L), dtype=torch.float32, device=queries.device) if return_lse else None
    i64 = ctypes.c_int64
    x = Expanded(q=queries.data_ptr(), k=keys.data_ptr(), rope_k=rope_keys.data_ptr(), v=values.data_ptr(), out=out.data_ptr(), lse=_address(lse),
                 starts=_address(starts), new_lens=_address(new_lens), sequences=B, tokens=L, heads=R, keys=K, key_dim=D, rope_dim=DR, value_dim=D,
                 q_strides=(i64 * 3)(*q), k_strides=(i64 * 3)(*k), rope_k_strides=(i64 * 2)(*kr), v_strides=(i64 * 3)(*v), out_strides=(i64 * 3)(*o))
    nbytes = _bytes(lib.fa_expanded_attention_workspace(ctypes.byref(x)))
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=queries.device) if nbytes else None
    with torch.cuda.device(queries.device):
        _check(lib.fa_expanded_attention(ctypes.byref(x), 1.0 / math.sqrt(D + DR) if scale is None else scale,
                                         (FLAG_CAUSAL if causal else 0) | _bf16(queries), _address(workspace), nbytes, _current_stream(queries) or None))
    return (out, lse) if return_lse else out


def latent_attention_plan(B, L, R, C, DR, P, W, pages=1):
    """What fa_latent_attention_plan reports for a problem, as a dict.  Needs no GPU."""
    out = (ctypes.c_int * 3)()
    _check(load_library().fa_latent_attention_plan(ctypes.byref(LatentCache(pages=pages, page_size=P, latent_dim=C, rope_dim=DR, sequences=B, table_width=W,
                                                                            table_stride=W)), L, R, out))
    return dict(zip(("rows", "shared", "workgroups"), out))


def expanded_attention_plan(B, L, R, K, D, DR):
    """What fa_expanded_attention_plan reports for a problem, as a dict.  Needs no GPU."""
    out = (ctypes.c_int * 3)()
    _check(load_library().fa_expanded_attention_plan(ctypes.byref(Expanded(sequences=B, tokens=L, heads=R, keys=K, key_dim=D, rope_dim=DR, value_dim=D)), out))
    return dict(zip(("rows", "splits", "workgroups"), out))
