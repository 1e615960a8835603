"""CPU: the W4 entry points check their arguments on the host before anything is launched (stand-in addresses,
never dereferenced); the layout's torch reader against the documented one; the exact quantiser's rules."""
import numpy as np
import pytest
import torch

from hummingbird_b200 import _lib, w4
from oracle import w4 as ow4

P = 0x7F0000001000


@pytest.fixture(scope="module")
def lib():
    from hummingbird_b200 import build
    build.build()
    return _lib.lib()


def _linear(**kw):
    a = dict(x=P, packed=P, scales=P, bias=0, y=P, ldx=1024, ldy=6144, m=2, n=6144, k=1024, group=128, silu=0,
             dtype=_lib.HB_BF16)
    assert set(kw) <= set(a)
    a.update(kw)
    return w4._ARGS.pack(*(0 if v is None else v for v in a.values())), None


@pytest.mark.parametrize("override,status", [
    (dict(x=None), _lib.HB_ERR_NULL), (dict(packed=None), _lib.HB_ERR_NULL), (dict(scales=None), _lib.HB_ERR_NULL),
    (dict(y=None), _lib.HB_ERR_NULL), (dict(m=0), _lib.HB_ERR_SHAPE), (dict(n=0), _lib.HB_ERR_SHAPE),
    (dict(k=0), _lib.HB_ERR_SHAPE), (dict(k=1000), _lib.HB_ERR_SHAPE), (dict(group=16), _lib.HB_ERR_SHAPE),
    (dict(group=0), _lib.HB_ERR_SHAPE), (dict(ldx=1016), _lib.HB_ERR_SHAPE), (dict(ldy=6143), _lib.HB_ERR_SHAPE),
    (dict(silu=2), _lib.HB_ERR_SHAPE), (dict(dtype=7), _lib.HB_ERR_SHAPE), (dict(m=1 << 30), _lib.HB_ERR_SHAPE),
    (dict(x=P + 8), _lib.HB_ERR_ALIGN), (dict(packed=P + 4), _lib.HB_ERR_ALIGN), (dict(scales=P + 2), _lib.HB_ERR_ALIGN),
    (dict(ldx=1028), _lib.HB_ERR_ALIGN), (dict(y=P + 1), _lib.HB_ERR_ALIGN), (dict(bias=P + 1), _lib.HB_ERR_ALIGN),
])
def test_linear_rejects(lib, override, status):
    assert lib.hb_w4_linear(*_linear(**override)) == status


def test_struct_has_the_header_s_size_and_null_is_refused(lib):
    assert w4._ARGS.size == 5 * 8 + 2 * 8 + 6 * 4
    assert lib.hb_w4_linear(None, None) == _lib.HB_ERR_NULL


@pytest.mark.parametrize("args,status", [
    ((None, 256, 16, 256, 128, P, P, None), _lib.HB_ERR_NULL), ((P, 256, 16, 256, 128, None, P, None), _lib.HB_ERR_NULL),
    ((P, 256, 16, 256, 128, P, None, None), _lib.HB_ERR_NULL), ((P, 256, 0, 256, 128, P, P, None), _lib.HB_ERR_SHAPE),
    ((P, 256, 16, 200, 64, P, P, None), _lib.HB_ERR_SHAPE), ((P, 248, 16, 256, 128, P, P, None), _lib.HB_ERR_SHAPE),
    ((P, 256, 16, 256, 256, P, P, None), _lib.HB_ERR_SHAPE), ((P + 8, 256, 16, 256, 128, P, P, None), _lib.HB_ERR_ALIGN),
    ((P, 260, 16, 256, 128, P, P, None), _lib.HB_ERR_ALIGN),
])
def test_quantiser_rejects(lib, args, status):
    assert lib.hb_quant_w4(*args) == status


@pytest.mark.parametrize("n,k,group", [(16, 128, 128), (5, 96, 32), (37, 320, 64)])
def test_dequantize_reads_the_documented_layout(n, k, group):
    rng = np.random.default_rng(n)
    q = rng.integers(-8, 8, (n, k)).astype(np.float64)
    s = 2.0 ** rng.integers(-5, 5, (n, k // group)).astype(np.float64)
    packed, scales = ow4.pack(q, s, group)
    got = w4.dequantize_w4(torch.from_numpy(packed), torch.from_numpy(scales).bfloat16(), n, k, group)
    assert np.array_equal(got.numpy(), (q.reshape(n, -1, group) * s[..., None]).reshape(n, k))


def test_exact_quantiser_rules():
    w = np.zeros((2, 64), np.float32)
    w[0, :6] = [7, 3.5, 2.5, -2.5, 0.5, -7]
    q, s = ow4.quantize(w, 32)
    assert s[0, 0] == 1 and list(q[0, :6]) == [7, 4, 2, -2, 0, -7]
    assert (s[1] == 1).all() and (q[1] == 0).all() and s[0, 1] == 1
    r = np.random.default_rng(0).normal(size=(8, 256)).astype(np.float32)
    q, s = ow4.quantize(r, 64)
    err = np.abs(q.reshape(8, 4, 64) * s[..., None] - r.reshape(8, 4, 64))
    # half a step, and a clamped value's distance: the scale's rounding, at most 2^-8 of 7 steps
    assert (err <= s[..., None] * (0.5 + 7 * 2.0 ** -8)).all()


def _w(n, k, group):
    return (torch.zeros(-(-n // 16), -(-k // 128), 1024, dtype=torch.uint8),
            torch.zeros(-(-n // 16), -(-k // 128), 128 // group, 16, dtype=torch.bfloat16))


@pytest.mark.parametrize("call", [
    lambda: w4.quantize_w4(torch.zeros(4, 64)),                                            # fp32
    lambda: w4.quantize_w4(torch.zeros(4, 96, dtype=torch.bfloat16), 64),
    lambda: w4.quantize_w4(torch.zeros(4, 64, dtype=torch.bfloat16), 16),
    lambda: w4.w4_linear(torch.zeros(2, 128), *_w(16, 128, 128), 16, 128),
    lambda: w4.w4_linear(torch.zeros(2, 256, dtype=torch.bfloat16), *_w(16, 128, 128), 16, 128),
    lambda: w4.w4_linear(torch.zeros(2, 128, dtype=torch.bfloat16), *_w(16, 128, 128), 32, 128),
    lambda: w4.w4_linear(torch.zeros(2, 128, dtype=torch.bfloat16), *_w(16, 128, 64), 16, 128),
    lambda: w4.w4_linear(torch.zeros(2, 128, dtype=torch.bfloat16), *_w(16, 128, 128), 16, 128, act="gelu"),
    lambda: w4.w4_linear(torch.zeros(2, 128, dtype=torch.bfloat16), *_w(16, 128, 128), 16, 128, torch.zeros(16)),
    lambda: w4.w4_linear(torch.zeros(2, 128, dtype=torch.bfloat16), *_w(16, 128, 128), 16, 128,
                         out=torch.zeros(2, 17, dtype=torch.bfloat16)),
])
def test_python_refusals(call):
    with pytest.raises(ValueError):
        call()


def test_no_cpu_path():
    with pytest.raises(RuntimeError):
        w4.w4_linear(torch.zeros(2, 128, dtype=torch.bfloat16), *_w(16, 128, 128), 16, 128)
