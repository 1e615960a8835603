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
import functools

import torch

from hummingbird_b200 import _lib
from hummingbird_b200._tensors import check_cuda

_DTYPES = {torch.bfloat16: _lib.HB_BF16, torch.float16: _lib.HB_FP16}


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(*sizes: int) -> int:
    n = ctypes.c_size_t(0)
    _lib.call("hb_context_workspace_bytes", *sizes, ctypes.byref(n))
    return n.value


def _rows(t: torch.Tensor, name: str, width: int, dtype: torch.dtype, device: torch.device,
          batch: int | None) -> torch.Tensor:
    """`t` checked, and copied only where the kernels cannot read its layout (unit stride in the last dim, other
    strides multiples of 16 bytes, no row over another)."""
    if t.dim() != (2 if batch is None else 3) or t.shape[-1] != width or (batch is not None and t.shape[0] != batch):
        raise ValueError(f"{name} must be {'(Ls' if batch is None else '(B, Lkv'}, {width}), got {tuple(t.shape)}")
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {dtype} on {device}, got {t.dtype} on {t.device}")
    return _readable(t, width)


def _readable(t: torch.Tensor, width: int) -> torch.Tensor:
    """`t`, or a copy of it where a tensor map cannot describe its rows."""
    strides = t.stride()
    if strides[-1] == 1 and t.data_ptr() % 16 == 0 and strides[-2] >= width and strides[-2] % 8 == 0:
        if t.dim() == 2:
            return t
        row, batch = strides[1], strides[0]
        if batch == 0 or (batch >= width and batch % 8 == 0 and (batch % row == 0 or row % batch == 0)):
            return t
    return t.contiguous() if not t.is_contiguous() else t.clone()


def _byte_mask(t: torch.Tensor | None, name: str, shape: tuple, device: torch.device) -> torch.Tensor | None:
    if t is None:
        return None
    if t.dtype not in (torch.bool, torch.uint8) or tuple(t.shape) != shape or t.device != device:
        raise ValueError(f"{name} must be a bool {shape} tensor on {device}, got {tuple(t.shape)} {t.dtype}")
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _attend(q, shared_kv, kv, num_heads, head_dim, kv_heads, lens, mask, shared_mask, q_weight, eps, scale, out):
    kv_heads = num_heads if kv_heads is None else kv_heads
    if head_dim not in (64, 128) or num_heads < 1 or kv_heads < 1 or num_heads % kv_heads:
        raise ValueError(f"context attention takes head_dim 64 or 128 and num_heads a multiple of kv_heads, got "
                         f"head_dim={head_dim}, {num_heads} heads, {kv_heads} kv heads")
    width, dtype, device = num_heads * head_dim, q.dtype, q.device
    if q.dim() != 3 or dtype not in _DTYPES or q.shape[-1] != width:
        raise ValueError(f"q must be bf16 or fp16 (B, Lq, {width}), got {tuple(q.shape)} {dtype}")
    batch, q_len, _ = q.shape
    kv = _rows(kv, "kv", 2 * kv_heads * head_dim, dtype, device, batch)
    kv_len = kv.shape[1]
    shared_len = 0
    if shared_kv is not None:
        shared_kv = _rows(shared_kv, "shared_kv", 2 * kv_heads * head_dim, dtype, device, None)
        shared_len = shared_kv.shape[0]
    if lens is not None and (lens.dtype != torch.int32 or tuple(lens.shape) != (batch,) or lens.device != device):
        raise ValueError(f"lens must be int32 ({batch},) on {device}, got {tuple(lens.shape)} {lens.dtype}")
    mask = _byte_mask(mask, "mask", (batch, kv_len), device)
    shared_mask = _byte_mask(shared_mask, "shared_mask", (shared_len,), device)
    if out is not None and (out.shape != q.shape or out.dtype != dtype or out.device != device
                            or out.stride(-1) != 1):
        raise ValueError(f"out must be {dtype} {tuple(q.shape)} on {device} with unit stride in its last dim")
    check_cuda(q)
    if torch.is_grad_enabled() and (q.requires_grad or kv.requires_grad
                                    or (shared_kv is not None and shared_kv.requires_grad)):
        raise RuntimeError("context attention has no backward pass: call it under torch.no_grad()")
    q = _readable(q, width)
    if lens is not None and lens.stride(0) != 1:
        lens = lens.contiguous()
    if q_weight is not None:
        if tuple(q_weight.shape) != (head_dim,) or q_weight.device != device:
            raise ValueError(f"q_weight must be ({head_dim},) on {device}, got {tuple(q_weight.shape)}")
        q_weight = q_weight.to(torch.float32).contiguous()
        if q_weight.data_ptr() % 16:
            q_weight = q_weight.clone()
    if out is None:
        out = torch.empty(batch, q_len, width, dtype=dtype, device=device)
    if not batch or not q_len:
        return out
    need = _workspace_bytes(batch, q_len, kv_len, shared_len, num_heads, kv_heads, head_dim,
                            int(mask is not None or shared_mask is not None))
    # partial results in a block of the caching allocator: it belongs to this call's stream, or to the graph that
    # is being captured, so calls on other streams and other graphs have theirs
    with torch.cuda.device(device):
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        _lib.call("hb_context_attn", q.data_ptr(), q.stride(0), q.stride(1), kv.data_ptr(), kv.stride(0), kv.stride(1),
                  None if shared_kv is None else shared_kv.data_ptr(), 0 if shared_kv is None else shared_kv.stride(0),
                  None if lens is None else lens.data_ptr(), None if mask is None else mask.data_ptr(),
                  0 if mask is None else mask.stride(0), None if shared_mask is None else shared_mask.data_ptr(),
                  None if q_weight is None else q_weight.data_ptr(), eps,
                  head_dim ** -0.5 if scale is None else scale, out.data_ptr(), out.stride(0), out.stride(1), batch,
                  q_len, kv_len, shared_len, num_heads, kv_heads, head_dim, _DTYPES[dtype],
                  None if ws is None else ws.data_ptr(), need, torch.cuda.current_stream(device).cuda_stream)
    return out


def context_attention(q: torch.Tensor, kv: torch.Tensor, num_heads: int, head_dim: int = 64, *,
                      kv_heads: int | None = None, lens: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                      q_weight: torch.Tensor | None = None, eps: float = 1e-6, scale: float | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """`(B, Lq, H * D)` queries and `(B, Lkv, [k | v])` states, `kv_heads * D` columns each -> `(B, Lq, H * D)`.

    `lens` int32 `(B,)` and `mask` bool `(B, Lkv)` (True: read) say which states of a padded batch count; what lies
    at the others is not read, and a batch element without any gets zeros. Query head h reads kv head
    `h // (num_heads // kv_heads)`. `q_weight` `(D,)` RMS-norms every query head first (`eps`), as the DiT does.
    `scale` defaults to `D ** -0.5`."""
    return _attend(q, None, kv, num_heads, head_dim, kv_heads, lens, mask, None, q_weight, eps, scale, out)


def shared_context_attention(q: torch.Tensor, shared_kv: torch.Tensor, kv: torch.Tensor, num_heads: int,
                             head_dim: int = 64, *, kv_heads: int | None = None, lens: torch.Tensor | None = None,
                             mask: torch.Tensor | None = None, shared_mask: torch.Tensor | None = None,
                             q_weight: torch.Tensor | None = None, eps: float = 1e-6, scale: float | None = None,
                             out: torch.Tensor | None = None) -> torch.Tensor:
    """`context_attention` over `(Ls, [k | v])` states that every batch element reads (bool `shared_mask` `(Ls,)`)
    and its own `kv` (`lens`, `mask`; `kv` may have length 0): one softmax over both."""
    return _attend(q, shared_kv, kv, num_heads, head_dim, kv_heads, lens, mask, shared_mask, q_weight, eps, scale, out)
