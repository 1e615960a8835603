"""Plain (non-differential) cross-attention of query tokens to an encoder's states, as sm_100a kernels through the
C ABI (`hb_context_attn`): the attention of `sa3jax.dit._cross_attention` for a model without the differential
branch (dit.py:131-147, 203-215), with what serving it needs beside the differential kernel in `cross_attention`:
contexts of any length, padded batches (`lens`, `mask`), fewer kv heads than query heads, head_dim 64 or 128, bf16
or fp16, single query tokens against long contexts, and states that the whole batch shares.

* `context_attention(q, kv, num_heads, head_dim)` -> `(B, Lq, H * D)`;
* `shared_context_attention(q, shared_kv, kv, num_heads, head_dim)`: one softmax over the shared states, which are
  read once for the whole batch, and each batch element's own.

Inference only: tensors that require gradients are refused. `ValueError` on unsupported shapes.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from hummingbird_b200 import _lib
from hummingbird_b200._tensors import check_cuda, launch

_DTYPES = {torch.bfloat16: _lib.HB_BF16, torch.float16: _lib.HB_FP16}
_ARGS = struct.Struct("=9Q9q8i2f")  # HbContextArgs: pointers, strides, sizes, eps and scale
_PLANS: dict = {}                   # checked calls by the sizes, strides and types of their tensors
_MAX_PLANS = 4096


def _layout(t: torch.Tensor):
    return t.shape, t.stride(), t.dtype


def _readable(t: torch.Tensor, width: int) -> bool:
    """Whether a tensor map describes the rows of `t`: unit stride in the last dim, the others multiples of 16 bytes,
    no row over another, batch elements behind one another, interleaved or all the same."""
    *outer, row, col = t.stride()
    if col != 1 or row < width or row % 8:
        return False
    return not outer or outer[0] == 0 or (outer[0] >= width and outer[0] % 8 == 0
                                          and (outer[0] % row == 0 or row % outer[0] == 0))


def _plan(q, shared_kv, kv, num_heads, head_dim, kv_heads, lens, mask, shared_mask, q_weight, out):
    """Check a call by its sizes and types: (tensors that need a copy, workspace bytes, sizes for HbContextArgs)."""
    if head_dim not in (64, 128) or num_heads < 1 or kv_heads < 1 or num_heads % kv_heads:
        raise ValueError(f"context attention takes head_dim 64 or 128 and num_heads a multiple of kv_heads, got "
                         f"head_dim={head_dim}, {num_heads} heads, {kv_heads} kv heads")
    width, kv_width, dtype = num_heads * head_dim, 2 * kv_heads * head_dim, q.dtype
    if q.dim() != 3 or dtype not in _DTYPES or q.shape[-1] != width:
        raise ValueError(f"q must be bf16 or fp16 (B, Lq, {width}), got {tuple(q.shape)} {dtype}")
    batch, q_len, _ = q.shape
    if kv.dim() != 3 or kv.shape[0] != batch or kv.shape[-1] != kv_width or kv.dtype != dtype:
        raise ValueError(f"kv must be {dtype} ({batch}, Lkv, {kv_width}), got {tuple(kv.shape)} {kv.dtype}")
    kv_len, shared_len = kv.shape[1], 0
    if shared_kv is not None:
        if shared_kv.dim() != 2 or shared_kv.shape[-1] != kv_width or shared_kv.dtype != dtype:
            raise ValueError(f"shared_kv must be {dtype} (Ls, {kv_width}), got {tuple(shared_kv.shape)} "
                             f"{shared_kv.dtype}")
        shared_len = shared_kv.shape[0]
    if lens is not None and (lens.dtype != torch.int32 or lens.shape != (batch,)):
        raise ValueError(f"lens must be int32 ({batch},), got {tuple(lens.shape)} {lens.dtype}")
    for name, t, shape in (("mask", mask, (batch, kv_len)), ("shared_mask", shared_mask, (shared_len,))):
        if t is not None and (t.dtype not in (torch.bool, torch.uint8) or t.shape != shape):
            raise ValueError(f"{name} must be bool {shape}, got {tuple(t.shape)} {t.dtype}")
    if q_weight is not None and q_weight.shape != (head_dim,):
        raise ValueError(f"q_weight must be ({head_dim},), got {tuple(q_weight.shape)}")
    if out is not None and (out.shape != q.shape or out.dtype != dtype or out.stride(-1) != 1):
        raise ValueError(f"out must be {dtype} {tuple(q.shape)} with unit stride in its last dim")
    check_cuda(*(t for t in (q, kv, shared_kv, lens, mask, shared_mask, q_weight, out) if t is not None))
    copies = (not _readable(q, width), not _readable(kv, kv_width),
              shared_kv is not None and not _readable(shared_kv, kv_width),
              lens is not None and lens.stride(0) != 1,
              mask is not None and kv_len > 1 and mask.stride(1) != 1,
              shared_mask is not None and shared_len > 1 and shared_mask.stride(0) != 1,
              q_weight is not None and (q_weight.dtype != torch.float32 or q_weight.stride(0) != 1))
    need = 0
    if batch and q_len:
        n = ctypes.c_size_t(0)
        _lib.call("hb_context_workspace_bytes", batch, q_len, kv_len, shared_len, num_heads, kv_heads, head_dim,
                  int((mask is not None and kv_len > 0) or (shared_mask is not None and shared_len > 0)),
                  ctypes.byref(n))
        need = n.value
    strides = (q.stride(0), q.stride(1), kv.stride(0), kv.stride(1), 0 if shared_kv is None else shared_kv.stride(0),
               0 if mask is None else mask.stride(0))
    sizes = (batch, q_len, kv_len, shared_len, num_heads, kv_heads, head_dim, _DTYPES[dtype])
    return (any(copies) and copies, need, strides, sizes, q.is_contiguous() and batch * q_len > 0,
            _lib.lib().hb_context_attn)


def _own_copy(t: torch.Tensor, copy: bool, dtype=None):
    return t.to(dtype or t.dtype, copy=True, memory_format=torch.contiguous_format) if copy else t


def _attend(q, shared_kv, kv, num_heads, head_dim, kv_heads, lens, mask, shared_mask, q_weight, eps, scale, out):
    if kv_heads is None:
        kv_heads = num_heads
    key = (num_heads, head_dim, kv_heads, q.shape, q.stride(), q.dtype, kv.shape, kv.stride(), kv.dtype,
           None if shared_kv is None else _layout(shared_kv), None if lens is None else _layout(lens),
           None if mask is None else _layout(mask), None if shared_mask is None else _layout(shared_mask),
           None if q_weight is None else _layout(q_weight), None if out is None else _layout(out))
    plan = _PLANS.get(key)
    if plan is None:
        plan = _plan(q, shared_kv, kv, num_heads, head_dim, kv_heads, lens, mask, shared_mask, q_weight, out)
        if len(_PLANS) >= _MAX_PLANS:
            _PLANS.clear()
        _PLANS[key] = plan
    copies, need, strides, sizes, like_q, call = plan
    device = q.get_device()
    if device < 0 or kv.get_device() != device or (shared_kv is not None and shared_kv.get_device() != device) \
            or (lens is not None and lens.get_device() != device) or (mask is not None and mask.get_device() != device) \
            or (shared_mask is not None and shared_mask.get_device() != device) \
            or (q_weight is not None and q_weight.get_device() != device) \
            or (out is not None and out.get_device() != device):
        check_cuda(*(t for t in (q, kv, shared_kv, lens, mask, shared_mask, q_weight, out) if t is not None))
        raise ValueError("the tensors of a context attention must be on one device")
    if (q.requires_grad or kv.requires_grad or (shared_kv is not None and shared_kv.requires_grad)
            or (q_weight is not None and q_weight.requires_grad) or (out is not None and out.requires_grad)) \
            and torch.is_grad_enabled():
        raise RuntimeError("context attention has no backward pass: call it under torch.no_grad()")
    q_at, kv_at = q.data_ptr(), kv.data_ptr()
    shared_at = 0 if shared_kv is None else shared_kv.data_ptr()
    weight_at = 0 if q_weight is None else q_weight.data_ptr()
    if copies or (q_at | kv_at | shared_at | weight_at) & 15:
        if out is None:
            out = q.new_empty(q.shape)
        c = copies or (False,) * 7
        return _attend(_own_copy(q, c[0] or q_at & 15), shared_kv if shared_kv is None else
                       _own_copy(shared_kv, c[2] or shared_at & 15), _own_copy(kv, c[1] or kv_at & 15), num_heads,
                       head_dim, kv_heads, lens if lens is None else _own_copy(lens, c[3]),
                       mask if mask is None else _own_copy(mask, c[4]),
                       shared_mask if shared_mask is None else _own_copy(shared_mask, c[5]),
                       q_weight if q_weight is None else _own_copy(q_weight, c[6] or weight_at & 15, torch.float32),
                       eps, scale, out)
    if out is None:
        out = torch.empty_like(q) if like_q else q.new_empty(q.shape)
    if not sizes[0] or not sizes[1]:
        return out
    # Partial results in a block of the caching allocator: it belongs to this call's stream, or to the graph that is
    # being captured, so calls on other streams and other graphs have theirs.
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    out_strides = out.stride()
    args = _ARGS.pack(q_at, kv_at, shared_at, 0 if lens is None else lens.data_ptr(),
                      mask.data_ptr() if mask is not None and sizes[2] else 0,  # (one without a state is none)
                      shared_mask.data_ptr() if shared_mask is not None and sizes[3] else 0,
                      weight_at, out.data_ptr(), 0 if ws is None else ws.data_ptr(), *strides, out_strides[0],
                      out_strides[1], need, *sizes, eps, head_dim ** -0.5 if scale is None else scale)
    launch(device, "hb_context_attn", call, args)
    return out


def context_attention(q: torch.Tensor, kv: torch.Tensor, num_heads: int, head_dim: int = 64, *,
                      kv_heads: int | None = None, lens: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                      q_weight: torch.Tensor | None = None, eps: float = 1e-6, scale: float | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """`(B, Lq, H * D)` queries and `(B, Lkv, [k | v])` states, `kv_heads * D` columns each -> `(B, Lq, H * D)`.

    `lens` int32 `(B,)` and `mask` bool `(B, Lkv)` (True: read) say which states of a padded batch count; what lies
    at the others is not read, and a batch element without any gets zeros. Query head h reads kv head
    `h // (num_heads // kv_heads)`. `q_weight` `(D,)` RMS-norms every query head first (`eps`), as the DiT does.
    `scale` defaults to `D ** -0.5`. `out`, where given, has 16-byte aligned rows and overlaps no input."""
    return _attend(q, None, kv, num_heads, head_dim, kv_heads, lens, mask, None, q_weight, eps, scale, out)


def shared_context_attention(q: torch.Tensor, shared_kv: torch.Tensor, kv: torch.Tensor, num_heads: int,
                             head_dim: int = 64, *, kv_heads: int | None = None, lens: torch.Tensor | None = None,
                             mask: torch.Tensor | None = None, shared_mask: torch.Tensor | None = None,
                             q_weight: torch.Tensor | None = None, eps: float = 1e-6, scale: float | None = None,
                             out: torch.Tensor | None = None) -> torch.Tensor:
    """`context_attention` over `(Ls, [k | v])` states that every batch element reads (bool `shared_mask` `(Ls,)`)
    and its own `kv` (`lens`, `mask`; `kv` may have length 0): one softmax over both."""
    return _attend(q, shared_kv, kv, num_heads, head_dim, kv_heads, lens, mask, shared_mask, q_weight, eps, scale, out)
