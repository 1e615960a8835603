"""Linear layers with 4-bit weights and group scales for a few rows, on sm_100a (`hb_w4_linear`).

The DiT's timestep, global and adaLN embedders (dit.py:39-42) run once per step on one row per clip, so they cost
the bytes of their weights; at 4 bits those are a quarter of bf16's. `W4Linear` is the drop-in for their `_linear`
(dit.py:33-36) when `DiTConfig.cond_quant == "w4"`; the MLP's thousands of rows take `w8a8`. Weights are quantised
and laid out once (`quantize_w4`).
"""
from __future__ import annotations

import struct

import torch

from hummingbird_b200 import _lib
from hummingbird_b200._tensors import check_cuda, launch, stream_handle

_ARGS = struct.Struct("=5Q2q6i")  # HbW4Args
GROUPS = (32, 64, 128)
_ACTS = {None: 0, "none": 0, "silu": 1}
_DTYPES = {torch.bfloat16: _lib.HB_BF16, torch.float16: _lib.HB_FP16}


def _blocks(out_features: int, in_features: int, group: int) -> tuple[int, int]:
    if group not in GROUPS or in_features < 1 or in_features % group or out_features < 1:
        raise ValueError(f"W4 takes groups of 32, 64 or 128 inputs that divide the row, got group={group}, "
                         f"weight ({out_features}, {in_features})")
    return -(-out_features // 16), -(-in_features // 128)


def quantize_w4(weight: torch.Tensor, group: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 `(N, K)` -> `packed` uint8 `(ceil(N / 16), ceil(K / 128), 1024)` and `scales` bf16 `(ceil(N / 16),
    ceil(K / 128), 128 // group, 16)` in the layout `hb_w4_linear` reads: per row and group of inputs s =
    bf16(absmax / 7) (1 where that is 0), q = clamp(rint(w / s), -7, 7)."""
    if weight.dim() != 2 or weight.dtype != torch.bfloat16:
        raise ValueError("quantize_w4 expects a 2-D bf16 tensor")
    n, k = weight.shape
    tiles, blocks = _blocks(n, k, group)
    check_cuda(weight)
    if weight.stride(1) != 1 or weight.stride(0) % 8 or weight.stride(0) < k or weight.data_ptr() % 16:
        weight = weight.clone(memory_format=torch.contiguous_format)
    packed = torch.empty(tiles, blocks, 1024, dtype=torch.uint8, device=weight.device)
    scales = torch.empty(tiles, blocks, 128 // group, 16, dtype=torch.bfloat16, device=weight.device)
    with torch.cuda.device(weight.device):
        _lib.call("hb_quant_w4", weight.data_ptr(), weight.stride(0), n, k, group, packed.data_ptr(),
                  scales.data_ptr(), stream_handle(weight.device))
    return packed, scales


def dequantize_w4(packed: torch.Tensor, scales: torch.Tensor, out_features: int, in_features: int,
                  group: int) -> torch.Tensor:
    """The fp32 `(N, K)` matrix that `packed` and `scales` stand for (torch ops; any device)."""
    tiles, blocks = _blocks(out_features, in_features, group)
    _check_weights(packed, scales, tiles, blocks, group)
    by = packed.view(tiles, blocks, 2, 8, 4, 4, 4)
    nib = torch.stack([by & 15, by >> 4], -1).flatten(-2).float() - 8  # (tile, block, half, row, t, word, nibble)
    nib = nib.view(*nib.shape[:-1], 2, 4).transpose(-1, -2).flatten(-2)  # nibbles 0 2 4 6 | 1 3 5 7 -> 0 .. 7
    q = nib.permute(0, 2, 3, 1, 5, 4, 6).reshape(tiles * 16, blocks * 128)
    s = scales.float().permute(0, 3, 1, 2).reshape(tiles * 16, -1)
    w = (q.unflatten(1, (-1, group)) * s[..., None]).flatten(1)
    return w[:out_features, :in_features].contiguous()


def _check_weights(packed, scales, tiles, blocks, group):
    if packed.shape != (tiles, blocks, 1024) or packed.dtype != torch.uint8 or not packed.is_contiguous():
        raise ValueError(f"packed must be contiguous uint8 ({tiles}, {blocks}, 1024), got {tuple(packed.shape)} "
                         f"{packed.dtype}")
    if scales.shape != (tiles, blocks, 128 // group, 16) or scales.dtype != torch.bfloat16 \
            or not scales.is_contiguous():
        raise ValueError(f"scales must be contiguous bf16 ({tiles}, {blocks}, {128 // group}, 16), got "
                         f"{tuple(scales.shape)} {scales.dtype}")


_PLANS: dict = {}  # checked calls by the sizes, strides and types of their tensors
_MAX_PLANS = 4096


def _plan(x, packed, scales, out_features, group, bias, act, out):
    """Check a call by its sizes and types: (copy x, copy bias, act code, type code)."""
    if x.dim() != 2 or x.dtype not in _DTYPES:
        raise ValueError(f"x must be bf16 or fp16 (M, K), got {tuple(x.shape)} {x.dtype}")
    if act not in _ACTS:
        raise ValueError(f"act must be 'silu' or None, not {act!r}")
    m, k = x.shape
    _check_weights(packed, scales, *_blocks(out_features, k, group), group)
    if bias is not None and (bias.shape != (out_features,) or bias.dtype != x.dtype):
        raise ValueError(f"bias must be {x.dtype} ({out_features},), got {tuple(bias.shape)} {bias.dtype}")
    if out is not None and (out.shape != (m, out_features) or out.dtype != x.dtype or out.stride(1) != 1):
        raise ValueError(f"out must be {x.dtype} ({m}, {out_features}) with unit stride in its last dim")
    check_cuda(*(t for t in (x, packed, scales, bias, out) if t is not None))
    return (x.stride(1) != 1 or x.stride(0) % 8 != 0 or x.stride(0) < k, bias is not None and bias.stride(0) != 1,
            _ACTS[act], _DTYPES[x.dtype])


def w4_linear(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, out_features: int, group: int,
              bias: torch.Tensor | None = None, *, act: str | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """`act(x @ W^T + bias)` of bf16 or fp16 `x` `(M, K)` with the weights of `quantize_w4`: fp32 sums, one rounding
    to x's type. `bias` `(N,)` of x's type; `act` "silu" or None ("none"). `out`, where given, overlaps no input."""
    key = (x.shape, x.stride(), x.dtype, packed.shape, packed.stride(), packed.dtype, scales.shape, scales.stride(),
           scales.dtype, out_features, group, act, None if bias is None else (bias.shape, bias.stride(), bias.dtype),
           None if out is None else (out.shape, out.stride(), out.dtype))
    plan = _PLANS.get(key)
    if plan is None:
        plan = _plan(x, packed, scales, out_features, group, bias, act, out)
        if len(_PLANS) >= _MAX_PLANS:
            _PLANS.clear()
        _PLANS[key] = plan
    copy_x, copy_bias, act_code, dtype_code = plan
    device = x.get_device()
    if device < 0 or packed.get_device() != device or scales.get_device() != device \
            or (bias is not None and bias.get_device() != device) or (out is not None and out.get_device() != device):
        check_cuda(*(t for t in (x, packed, scales, bias, out) if t is not None))
        raise ValueError("x, packed, scales, bias and out must be on one device")
    if (x.requires_grad or scales.requires_grad or (bias is not None and bias.requires_grad)
            or (out is not None and out.requires_grad)) and torch.is_grad_enabled():
        raise RuntimeError("W4 linear layers have no backward pass: call them under torch.no_grad()")
    x_at = x.data_ptr()
    if copy_x or x_at & 15:
        x = x.clone(memory_format=torch.contiguous_format)
        x_at = x.data_ptr()
    if copy_bias:
        bias = bias.contiguous()
    m, k = x.shape
    if out is None:
        out = torch.empty(m, out_features, dtype=x.dtype, device=x.device)
    if m:
        launch(device, "hb_w4_linear", _lib.lib().hb_w4_linear,
               _ARGS.pack(x_at, packed.data_ptr(), scales.data_ptr(), 0 if bias is None else bias.data_ptr(),
                          out.data_ptr(), x.stride(0), out.stride(0), m, out_features, k, group, act_code, dtype_code))
    return out


class W4Linear:
    """`nn.Linear` with weight `[out, in]` (the checkpoint layout, dit.py:34) and 4-bit weights: rounded to bf16 and
    quantised once, applied to the few rows of a conditioning vector. `act="silu"` takes the activation that follows
    along. fp16 inputs are taken and answered in fp16, all others in bf16."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, *, group: int = 128,
                 act: str | None = None):
        self.packed, self.scales = quantize_w4(weight.to(torch.bfloat16), group)
        self.bias = None if bias is None else bias.to(torch.bfloat16).contiguous()
        self._bias_fp16 = None if bias is None else bias.to(torch.float16).contiguous()
        self.out_features, self.in_features = weight.shape
        self.group, self.act = group, act

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise ValueError(f"x must have {self.in_features} columns, got {tuple(x.shape)}")
        fp16 = x.dtype == torch.float16
        x2 = x.reshape(-1, self.in_features).to(torch.float16 if fp16 else torch.bfloat16)
        y = w4_linear(x2, self.packed, self.scales, self.out_features, self.group,
                      self._bias_fp16 if fp16 else self.bias, act=self.act)
        return y.reshape(*x.shape[:-1], self.out_features)
