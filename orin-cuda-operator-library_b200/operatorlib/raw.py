"""Tensor-level calls straight onto the C-ABI (no torch binding involved).

Each ``*_into`` function takes contiguous CUDA tensors with preallocated
outputs, passes their device pointers and the current CUDA stream (or
``stream``) to the matching ``opl_*`` entry point and raises ``OplError`` on a
non-zero return -- the same contract a C, cgo or JNI caller gets.  The paged
cache functions (``rope_into``, ``kv_append_into``, ``paged_attention_into``)
take strided tensors whose last dimension is contiguous, and raise ``ValueError``
for operands whose shapes, types or devices do not go together: the C entries
see pointers only and would read or write past them.
"""
from __future__ import annotations


def _ptr(t) -> int:
    return t.data_ptr()


def _stream(t, stream) -> int:
    import torch

    s = stream if stream is not None else torch.cuda.current_stream(t.device)
    return s.cuda_stream


def _lib():
    from . import capi

    return capi()


def _check(op, code):
    from . import check

    check(op, code)


def reduce_sum_into(x, out, stream=None) -> None:
    _check("reduce_sum", _lib().opl_reduce_sum_f32(
        _ptr(x), _ptr(out), x.numel(), _stream(x, stream)))


def reduce_sum_partial_f64_into(x, out, stream=None) -> None:
    _check("reduce_sum_partial_f64", _lib().opl_reduce_sum_partial_f64(
        _ptr(x), _ptr(out), x.numel(), _stream(x, stream)))


def _dtype_fn(base: str, dtype):
    import torch

    suffix = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}[dtype]
    return getattr(_lib(), f"opl_{base}_{suffix}")


def softmax_into(x, out, stream=None) -> None:
    """FP32, FP16 or BF16 (out has x's dtype; arithmetic in FP32)."""
    cols = x.shape[-1]
    _check("softmax", _dtype_fn("softmax", x.dtype)(
        _ptr(x), _ptr(out), x.numel() // cols, cols, _stream(x, stream)))


def transpose_into(x, out, stream=None) -> None:
    rows, cols = x.shape
    _check("transpose", _lib().opl_transpose_f32(
        _ptr(x), _ptr(out), rows, cols, _stream(x, stream)))


def rmsnorm_into(x, w, out, eps: float, stream=None) -> None:
    """FP32, FP16 or BF16 (w and out have x's dtype; arithmetic in FP32)."""
    hidden = x.shape[-1]
    _check("rmsnorm", _dtype_fn("rmsnorm", x.dtype)(
        _ptr(x), _ptr(w), _ptr(out), x.numel() // hidden, hidden, float(eps),
        _stream(x, stream)))


def gemm_into(a, b, c, stream=None) -> None:
    import torch

    m, k = a.shape
    n = b.shape[1]
    fn = _lib().opl_gemm_f16 if a.dtype == torch.float16 else _lib().opl_gemm_f32
    _check("gemm", fn(_ptr(a), _ptr(b), _ptr(c), m, n, k, _stream(a, stream)))


def attention_into(q, k, v, out, causal: bool, stream=None) -> None:
    import torch

    b, h, s, d = q.shape
    fn = (_lib().opl_attention_f16 if q.dtype == torch.float16
          else _lib().opl_attention_f32)
    _check("attention", fn(_ptr(q), _ptr(k), _ptr(v), _ptr(out), b, h, s, d,
                           int(bool(causal)), _stream(q, stream)))


def _require_rows(name, t, dtype, device, shape=None, written=False) -> None:
    """A strided operand: the last dimension contiguous, at least the first
    dimension's rows."""
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must have the other tensors' dtype and device")
    own = t.shape
    if shape is not None and own != shape and (len(own) != len(shape) or own[1:] != shape[1:]
                                               or own[0] < shape[0]):
        raise ValueError(f"{name} must have the shape {list(shape)}, or more rows")
    strides = t.stride()
    if strides[-1] != 1 and own[-1] != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    if written and 0 in strides and any(s == 0 and n > 1 for s, n in zip(strides, own)):
        raise ValueError(f"{name} is written and must not be expanded")


def _require_flat(name, t, dtype, device, count, exact=False) -> None:
    """Contiguous numbers, at least (or exactly) `count`."""
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {str(dtype).split('.')[-1]} on the other tensors' device")
    size = t.numel()
    if size < count or (exact and size != count) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous with {'' if exact else 'at least '}{count} "
                         "elements")


def _require_dims(name, t, dims) -> None:
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions")


def _rope_spec(tokens, device, positions, inv_freq, sections, adjacent, inverse):
    import torch

    from . import RopeSpec

    pairs = inv_freq.numel()
    sections = list(sections) if sections else [pairs]
    if len(sections) > 4:
        raise ValueError("a rotary embedding has at most 4 position axes")
    _require_flat("inv_freq", inv_freq, torch.float32, device, pairs)
    if pairs > 0:  # the kernel finds an axis at axis * tokens
        _require_flat("positions", positions, torch.int64, device, len(sections) * tokens,
                      exact=len(sections) > 1)
    spec = RopeSpec(positions=_ptr(positions), inv_freq=_ptr(inv_freq), rot_dim=2 * pairs,
                    axes=len(sections), adjacent=int(bool(adjacent)),
                    inverse=int(bool(inverse)))
    spec.sections[:len(sections)] = sections
    return spec


def _kv_cache(q, dtype, device, k_cache, v_cache, written):
    from . import KvCache

    _require_dims("k_cache", k_cache, 4)
    shape = k_cache.shape
    _require_rows("k_cache", k_cache, dtype, device, written=written)
    _require_rows("v_cache", v_cache, dtype, device, shape, written)
    if shape[3] != q.shape[2]:
        raise ValueError("the caches must be [pages, page_size, kv_heads, head_dim] with q's "
                         "head_dim")
    return KvCache(_ptr(k_cache), _ptr(v_cache), *shape, *k_cache.stride()[:3], *v_cache.stride()[:3])


def rope_into(x, out, positions, inv_freq, sections=None, adjacent=False, inverse=False,
              stream=None) -> None:
    """Rotary embedding of x [tokens, heads, head_dim] (FP32, FP16 or BF16)
    into out, which may be x.  positions: int64 [tokens] or [axes, tokens],
    contiguous; inv_freq: FP32 [rotated pairs]; sections: pairs of each axis."""
    import ctypes

    import torch

    _require_dims("x", x, 3)
    dtype, device, shape = x.dtype, x.device, x.shape
    tokens, heads, head_dim = shape
    _require_rows("x", x, dtype, device)
    _require_rows("out", out, dtype, device, shape, True)
    spec = _rope_spec(tokens, device, positions, inv_freq, sections, adjacent, inverse)
    with torch.cuda.device(device):
        _check("rope", _dtype_fn("rope", dtype)(
            _ptr(x), _ptr(out), tokens, heads, head_dim, *x.stride()[:2], *out.stride()[:2],
            ctypes.byref(spec), _stream(x, stream)))


def kv_append_into(q, k, v, q_out, k_cache, v_cache, slots, positions, inv_freq, sections=None,
                   adjacent=False, stream=None) -> None:
    """Rotates q into q_out (which may be q) and k into the cache, and copies v
    there.  The caches are [pages, page_size, kv_heads, head_dim]; slots: int64
    [tokens], contiguous, page * page_size + token of the page, negative for a
    token that is not kept; the rest as in rope_into."""
    import ctypes

    import torch

    _require_dims("q", q, 3)
    dtype, device, shape = q.dtype, q.device, q.shape
    tokens, heads, head_dim = shape
    _require_rows("q", q, dtype, device)
    _require_rows("q_out", q_out, dtype, device, shape, True)
    cache = _kv_cache(q, dtype, device, k_cache, v_cache, True)
    new = (tokens, cache.kv_heads, head_dim)
    _require_rows("k", k, dtype, device, new)
    _require_rows("v", v, dtype, device, new)
    _require_flat("slots", slots, torch.int64, device, tokens)
    spec = _rope_spec(tokens, device, positions, inv_freq, sections, adjacent, False)
    with torch.cuda.device(device):
        _check("kv_append", _dtype_fn("kv_append", dtype)(
            _ptr(q), *q.stride()[:2], _ptr(k), *k.stride()[:2], _ptr(v), *v.stride()[:2],
            _ptr(q_out), *q_out.stride()[:2], ctypes.byref(cache), _ptr(slots), tokens,
            heads, ctypes.byref(spec), _stream(q, stream)))


def paged_attention_workspace(heads: int, kv_heads: int, head_dim: int, device) -> "torch.Tensor":
    """Scratch for paged_attention_into; calls that may overlap need one each."""
    import ctypes

    import torch

    size = ctypes.c_size_t()
    with torch.cuda.device(device):
        _check("paged_attention", _lib().opl_paged_attention_workspace(
            heads, kv_heads, head_dim, ctypes.byref(size)))
        return torch.empty(size.value, dtype=torch.uint8, device=device)


def paged_attention_into(q, k_cache, v_cache, block_table, seq_lens, out, workspace, scale=None,
                         stream=None) -> None:
    """Attention of q [batch, heads, head_dim], one new token per sequence,
    over the cache (see kv_append_into) into the contiguous out.  block_table:
    int32 [batch, pages of the longest sequence]; seq_lens: int32 [batch];
    workspace from paged_attention_workspace; scale: 1 / sqrt(head_dim)."""
    import ctypes

    import torch

    _require_dims("q", q, 3)
    dtype, device = q.dtype, q.device
    batch, heads, head_dim = q.shape
    _require_rows("q", q, dtype, device)
    _require_flat("out", out, dtype, device, q.numel())
    cache = _kv_cache(q, dtype, device, k_cache, v_cache, False)
    _require_dims("block_table", block_table, 2)
    rows, columns = block_table.shape
    table_row, step = block_table.stride()
    if (block_table.dtype != torch.int32 or block_table.device != device or rows < batch
            or (step != 1 and columns != 1)):
        raise ValueError("block_table must be int32 [batch, pages] on the other tensors' device, "
                         "contiguous in its last dimension")
    _require_flat("seq_lens", seq_lens, torch.int32, device, batch)
    if workspace.device != device or not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous on the other tensors' device")
    scale = head_dim ** -0.5 if scale is None else float(scale)
    with torch.cuda.device(device):
        _check("paged_attention", _dtype_fn("paged_attention", dtype)(
            _ptr(q), *q.stride()[:2], ctypes.byref(cache), _ptr(block_table),
            table_row, columns, _ptr(seq_lens), _ptr(out), batch, heads,
            scale, _ptr(workspace), workspace.numel() * workspace.element_size(),
            _stream(q, stream)))
