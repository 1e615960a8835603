"""GPU: W4 linear layers wide enough, over rows enough, that a CTA takes two tiles of outputs: against float64 products
within the bound of `oracle.w4`."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
UNIT = {BF16: 2.0 ** -8, FP16: 2.0 ** -11}


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k,group,act,with_bias", [
    (9, 4745, 9120, 32, None, True),       # 297 tiles of outputs, the last one partial; 71 1/4 blocks of inputs
    (16, 4752, 5184, 64, "silu", False),   # 297 whole tiles; 40 1/2 blocks
    (16, 8201, 8192, 128, None, True),
    (17, 4737, 4864, 128, None, True),     # one output in the last tile, which is a CTA's first
    (32, 4768, 2592, 32, "silu", True),    # 298 tiles: pairs
    (32, 4900, 4160, 64, None, False),     # 307 tiles
    (33, 8201, 2560, 128, "silu", True),   # rows past one CTA's
    (70, 4745, 1248, 32, None, True),
])
def test_two_tiles_of_outputs_to_a_cta(cuda_lib, m, n, k, group, act, with_bias, dtype):
    from hummingbird_b200 import w4
    assert m > 8 and m * k * 2 > 160 * 1024 and n > 2 * 148 * 16
    g = torch.Generator(device="cuda").manual_seed(n + m)
    weight = (torch.randn(n, k, generator=g, device="cuda") / k ** 0.5).to(BF16)
    packed, scales = w4.quantize_w4(weight, group)
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    bias = torch.randn(n, generator=g, device="cuda").to(dtype) if with_bias else None
    buf = torch.full((m + 2, n + 9), 5.0, dtype=dtype, device="cuda")
    got = w4.w4_linear(x, packed, scales, n, group, bias, act=act, out=buf[1:-1, 3:3 + n]).double()
    w = w4.dequantize_w4(packed, scales, n, k, group).double()
    ref, mag = x.double() @ w.T, x.double().abs() @ w.abs().T
    if bias is not None:
        ref, mag = ref + bias.double(), mag + bias.double().abs()
    tol = (k + 1) * 2.0 ** -23 * mag
    if act == "silu":
        ref = ref * torch.special.expit(ref)
        tol = 1.1 * tol + 2.0 ** -20 * ref.abs()
    tol = tol + UNIT[dtype] * (ref.abs() + tol) + 1e-38
    over = ((got - ref).abs() - tol).max().item()
    assert over <= 0, f"off by {(got - ref).abs().max().item():.3e}, {over:.3e} over the bound"
    rest = buf.clone()
    rest[1:-1, 3:3 + n] = 5.0
    assert (rest == 5.0).all()
    assert torch.equal(w4.w4_linear(x[:8], packed, scales, n, group, bias, act=act), got[:8].to(dtype))  # one tile a CTA


def test_linear_class_keeps_fp16(cuda_lib):
    """fp16 inputs go through the fp16 kernel with the bias in fp16 (values that bf16 would round), and come back so."""
    from hummingbird_b200.w4 import W4Linear, dequantize_w4, w4_linear
    g = torch.Generator(device="cuda").manual_seed(1)
    weight, bias = torch.randn(96, 256, generator=g, device="cuda"), torch.randn(96, generator=g, device="cuda")
    x = torch.randn(2, 3, 256, generator=g, device="cuda").to(FP16)
    for b in (bias, None):
        lin = W4Linear(weight, b, group=64)
        y = lin(x)
        w = dequantize_w4(lin.packed, lin.scales, 96, 256, 64).double()
        ref = x.double() @ w.T + (0 if b is None else b.double())
        mag = x.double().abs() @ w.abs().T + 4
        assert y.dtype == FP16 and y.shape == (2, 3, 96)
        assert ((y.double() - ref).abs() <= UNIT[FP16] * (ref.abs() + 4) * 1.01 + 257 * 2.0 ** -23 * mag).all()
        bf = lin(x.to(BF16))
        assert bf.dtype == BF16 and lin(x.float()).dtype == BF16
        assert torch.equal(bf, w4_linear(x.to(BF16).view(6, 256), lin.packed, lin.scales, 96, 64, lin.bias).view(2, 3, 96))
