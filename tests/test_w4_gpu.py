"""GPU: W4 linear layers and their quantiser (`hummingbird_b200.w4`, through the C ABI) against exact arithmetic."""
import numpy as np
import pytest
import torch

from oracle import w4 as ow4

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
UNIT = {BF16: 2.0 ** -8, FP16: 2.0 ** -11}


def _weights(n, k, group, seed=0):
    from hummingbird_b200 import w4
    w = (torch.randn(n, k, generator=torch.Generator().manual_seed(seed)) / k ** 0.5).to(BF16)
    packed, scales = w4.quantize_w4(w.cuda(), group)
    return w, packed, scales


@pytest.mark.parametrize("n,k,group", [(16, 128, 128), (1, 32, 32), (37, 352, 32), (33, 192, 64), (48, 640, 128),
                                       (17, 1056, 32)])
def test_quantiser_is_exact(cuda_lib, n, k, group):
    from hummingbird_b200 import w4
    w = (torch.randn(n, k, generator=torch.Generator().manual_seed(n)) * 3).to(BF16)
    w[0] = 0                                          # a zero group: scale 1
    w[-1, :group] = torch.tensor([2.0 ** -133, 0.0] * (group // 2)).to(BF16)  # absmax / 7 rounds to 0
    if n > 2:
        w[1, :8] = torch.tensor([7.0, 3.5, 2.5, 1.5, 0.5, -0.5, -1.5, -7.0])   # ties, with s = 1
        w[1, 8:group] = 0
    q, s = ow4.quantize(w.float().numpy(), group)
    want, want_s = ow4.pack(q, s, group)
    packed, scales = w4.quantize_w4(w.cuda(), group)
    assert np.array_equal(packed.cpu().numpy(), want)
    assert np.array_equal(scales.double().cpu().numpy(), want_s)
    back = w4.dequantize_w4(packed, scales, n, k, group).double().cpu().numpy()
    assert np.array_equal(back, (q.reshape(n, -1, group) * s[..., None]).reshape(n, k))


def test_quantiser_takes_strided_rows(cuda_lib):
    from hummingbird_b200 import w4
    w = torch.randn(40, 300, device="cuda").to(BF16)
    ref = w4.quantize_w4(w[:, :256].contiguous(), 64)
    for view in (w[:, :256], torch.nn.functional.pad(w, (8, 4))[:, 8:264], w.T.contiguous().T[:, :256]):
        got = w4.quantize_w4(view, 64)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,n,k,group,act,with_bias", [
    (1, 16, 128, 128, None, False),
    (1, 1, 32, 32, "silu", True),
    (2, 1024, 256, 128, "silu", False),
    (2, 6144, 1024, 128, "none", True),
    (3, 33, 192, 64, None, True),
    (7, 257, 2048, 64, "silu", True),
    (8, 64, 4096, 128, None, False),
    (9, 130, 1056, 32, None, True),
    (16, 48, 640, 128, "silu", False),
    (17, 47, 96, 32, None, True),
    (31, 200, 1408, 128, None, False),
    (32, 128, 512, 64, None, True),
    (33, 40, 160, 32, "silu", True),
    (100, 50, 384, 128, None, True),
])
def test_linear_matches_exact(cuda_lib, m, n, k, group, act, with_bias, dtype):
    from hummingbird_b200 import w4
    _, packed, scales = _weights(n, k, group, seed=m)
    g = torch.Generator().manual_seed(m + n)
    x = torch.randn(m, k, generator=g).to(dtype)
    bias = torch.randn(n, generator=g).to(dtype) if with_bias else None
    y = w4.w4_linear(x.cuda(), packed, scales, n, group, None if bias is None else bias.cuda(), act=act)
    w = w4.dequantize_w4(packed, scales, n, k, group).double().cpu().numpy()
    ref, tol = ow4.linear(x.double().numpy(), w, None if bias is None else bias.double().numpy(), act == "silu",
                          UNIT[dtype])
    got = y.double().cpu().numpy()
    assert y.dtype == dtype and np.isfinite(got).all()
    assert (np.abs(got - ref) <= tol).all(), f"off by {np.abs(got - ref).max():.3e}"


def test_every_weight_value_and_input_position(cuda_lib):
    """A one-hot input reads one column of the matrix, exactly: all 16 nibble values, at every position."""
    from hummingbird_b200 import w4
    n, k, group = 48, 288, 32
    q = torch.randint(-8, 8, (n, k), generator=torch.Generator().manual_seed(3)).double().numpy()
    s = 2.0 ** np.random.default_rng(3).integers(-6, 6, (n, k // group)).astype(np.float64)
    pk, sc = ow4.pack(q, s, group)
    packed, scales = torch.from_numpy(pk).cuda(), torch.from_numpy(sc).to(BF16).cuda()
    want = torch.from_numpy((q.reshape(n, -1, group) * s[..., None]).reshape(n, k))
    for dtype in (BF16, FP16):
        eye = torch.eye(k, dtype=dtype, device="cuda")
        got = torch.cat([w4.w4_linear(eye[a:a + 5], packed, scales, n, group) for a in range(0, k, 5)])
        assert torch.equal(got.double().cpu(), want.T)
        assert torch.equal(w4.w4_linear(eye, packed, scales, n, group).double().cpu(), want.T)


def test_strided_rows_and_output(cuda_lib):
    from hummingbird_b200 import w4
    m, n, k = 5, 70, 256
    _, packed, scales = _weights(n, k, 128)
    x = torch.randn(m, k, device="cuda").to(BF16)
    ref = w4.w4_linear(x, packed, scales, n, 128)
    wide = torch.full((m, k + 40), float("nan"), dtype=BF16, device="cuda")
    wide[:, 16:16 + k] = x
    buf = torch.full((m + 2, n + 9), 5.0, dtype=BF16, device="cuda")
    out = w4.w4_linear(wide[:, 16:16 + k], packed, scales, n, 128, out=buf[1:-1, 3:3 + n])
    assert torch.equal(out, ref)
    rest = buf.clone()
    rest[1:-1, 3:3 + n] = 5.0
    assert (rest == 5.0).all()
    wide[:, 17:17 + k] = x                           # rows that are not 16-byte aligned
    assert torch.equal(w4.w4_linear(wide[:, 17:17 + k], packed, scales, n, 128), ref)
    assert torch.equal(w4.w4_linear(x.T.contiguous().T, packed, scales, n, 128), ref)
    assert w4.w4_linear(x[:0], packed, scales, n, 128).shape == (0, n)


def test_same_bits_whatever_the_batch_and_in_a_graph(cuda_lib):
    from hummingbird_b200 import w4
    n, k = 500, 4096
    _, packed, scales = _weights(n, k, 64)
    x = torch.randn(8, k, device="cuda").to(BF16)
    ref = w4.w4_linear(x, packed, scales, n, 64)
    assert torch.equal(torch.cat([w4.w4_linear(x[i:i + 1], packed, scales, n, 64) for i in range(8)]), ref)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = w4.w4_linear(x, packed, scales, n, 64)
    x.mul_(-1)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, -ref)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = w4.w4_linear(x, packed, scales, n, 64)
    torch.cuda.synchronize()
    assert torch.equal(other, -ref)


def test_linear_class_and_extreme_activations(cuda_lib):
    from hummingbird_b200.w4 import W4Linear, dequantize_w4
    w = torch.randn(96, 128, device="cuda").to(BF16)
    lin = W4Linear(w, torch.randn(96, device="cuda"), act="silu")
    x = torch.randn(2, 3, 128, device="cuda").to(BF16) * 40  # SiLU far out on both sides
    y = lin(x)
    assert y.shape == (2, 3, 96) and y.dtype == BF16
    wd = dequantize_w4(lin.packed, lin.scales, 96, 128, 128).double().cpu().numpy()
    ref, tol = ow4.linear(x.reshape(6, 128).double().cpu().numpy(), wd, lin.bias.double().cpu().numpy(), True,
                          UNIT[BF16])
    assert (np.abs(y.reshape(6, 96).double().cpu().numpy() - ref) <= tol).all()
    with pytest.raises(ValueError):
        lin(x[..., :64])
    xg = x.float().requires_grad_(True)
    with pytest.raises(RuntimeError):
        lin(xg)
