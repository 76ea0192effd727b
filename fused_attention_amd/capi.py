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
           "fa_cache_append", "fa_cached_attention", "fa_cached_attention_workspace", "fa_cached_attention_plan", "fa_select_pages", "fa_select_pages_plan")
FLAG_CAUSAL = 1
FLAG_BF16 = 2

_lib = None


class Cache(ctypes.Structure):
    """fa_cache: addresses and sizes of a paged key/value cache and its page table."""

    _fields_ = ([(name, ctypes.c_void_p) for name in ("keys", "values", "key_exponents", "value_exponents", "key_bounds", "page_table")] +
                [(name, ctypes.c_int64) for name in ("pages", "heads", "page_size", "head_dim", "sequences", "table_width", "table_stride")])


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
