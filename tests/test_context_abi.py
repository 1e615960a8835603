"""CPU: the context attention checks its arguments on the host before anything is launched (stand-in addresses,
never dereferenced), and the Python entry points refuse what the kernels do not take."""
import ctypes

import pytest
import torch

from hummingbird_b200 import _lib
from hummingbird_b200.context_attention import _ARGS

P = 0x7F0000001000


@pytest.fixture(scope="module")
def lib():
    from hummingbird_b200 import build
    build.build()
    return _lib.lib()


def _need(lib, *sizes, masked=0):
    n = ctypes.c_size_t(0)
    assert lib.hb_context_workspace_bytes(*sizes, masked, ctypes.byref(n)) == _lib.HB_OK
    return n.value


def _args(**kw):
    a = dict(q=P, kv=P, skv=0, lens=0, mask=0, smask=0, q_w=0, out=P, ws=P, q_bs=300 * 1024, q_rs=1024,
             kv_bs=257 * 2048, kv_rs=2048, skv_rs=0, mask_bs=0, o_bs=300 * 1024, o_rs=1024, ws_bytes=1 << 40, batch=2,
             q_len=300, kv_len=257, shared_len=0, heads=16, kv_heads=16, head_dim=64, dtype=_lib.HB_BF16, eps=1e-6,
             scale=0.125)
    assert set(kw) <= set(a)
    a.update(kw)
    return _ARGS.pack(*(0 if v is None else v for v in a.values())), None


@pytest.mark.parametrize("override,status", [
    (dict(q=None), _lib.HB_ERR_NULL),
    (dict(out=None), _lib.HB_ERR_NULL),
    (dict(kv=None), _lib.HB_ERR_NULL),
    (dict(shared_len=8, skv_rs=2048), _lib.HB_ERR_NULL),
    (dict(batch=0), _lib.HB_ERR_SHAPE),
    (dict(q_len=0), _lib.HB_ERR_SHAPE),
    (dict(kv_len=-1), _lib.HB_ERR_SHAPE),
    (dict(shared_len=-1), _lib.HB_ERR_SHAPE),
    (dict(kv_heads=5), _lib.HB_ERR_SHAPE),
    (dict(kv_heads=0), _lib.HB_ERR_SHAPE),
    (dict(head_dim=96), _lib.HB_ERR_SHAPE),
    (dict(dtype=2), _lib.HB_ERR_SHAPE),
    (dict(scale=0.0), _lib.HB_ERR_SHAPE),
    (dict(scale=-1.0), _lib.HB_ERR_SHAPE),
    (dict(scale=float("nan")), _lib.HB_ERR_SHAPE),
    (dict(scale=float("inf")), _lib.HB_ERR_SHAPE),
    (dict(q_w=P, eps=-1.0), _lib.HB_ERR_SHAPE),
    (dict(q_rs=1016), _lib.HB_ERR_SHAPE),
    (dict(kv_rs=2040), _lib.HB_ERR_SHAPE),
    (dict(o_rs=1016), _lib.HB_ERR_SHAPE),
    (dict(o_bs=1024), _lib.HB_ERR_SHAPE),                      # output rows of two batch elements on one another
    (dict(q_bs=-1024), _lib.HB_ERR_SHAPE),
    (dict(batch=1 << 20, q_len=1 << 20), _lib.HB_ERR_SHAPE),
    (dict(kv_len=(1 << 24) + 1), _lib.HB_ERR_SHAPE),
    (dict(kv_bs=1024), _lib.HB_ERR_SHAPE),                     # batch elements closer than a row
    (dict(kv_bs=257 * 2048 + 8), _lib.HB_ERR_ALIGN),           # neither stride a multiple of the other
    (dict(kv_bs=2056, kv_rs=4096), _lib.HB_ERR_ALIGN),
    (dict(kv_rs=1 << 40), _lib.HB_ERR_SHAPE),
    (dict(q=P + 8), _lib.HB_ERR_ALIGN),
    (dict(ws=P + 16), _lib.HB_ERR_ALIGN),
    (dict(kv=P + 2), _lib.HB_ERR_ALIGN),
    (dict(out=P + 4), _lib.HB_ERR_ALIGN),
    (dict(q_rs=1028), _lib.HB_ERR_ALIGN),
    (dict(kv_rs=2052), _lib.HB_ERR_ALIGN),
    (dict(lens=P + 2), _lib.HB_ERR_ALIGN),
    (dict(q_w=P + 4), _lib.HB_ERR_ALIGN),
])
def test_rejects(lib, override, status):
    assert lib.hb_context_attn(*_args(**override)) == status


def test_struct_has_the_header_s_size_and_null_is_refused(lib):
    assert _ARGS.size == 9 * 8 + 9 * 8 + 8 * 4 + 2 * 4
    assert lib.hb_context_attn(None, None) == _lib.HB_ERR_NULL


def test_workspace_is_asked_for_and_checked(lib):
    sizes = (1, 1, 100000, 0, 16, 4, 64)
    need = _need(lib, *sizes)
    assert need > 0
    one = dict(batch=1, q_len=1, kv_len=100000, kv_heads=4, kv_rs=512, kv_bs=0)
    assert lib.hb_context_attn(*_args(**one, ws=None, ws_bytes=0)) == _lib.HB_ERR_WORKSPACE
    assert lib.hb_context_attn(*_args(**one, ws_bytes=need - 1)) == _lib.HB_ERR_WORKSPACE
    assert _need(lib, 1, 1, 16, 0, 16, 16, 64) == 0             # one part: written directly
    n = ctypes.c_size_t(0)
    assert lib.hb_context_workspace_bytes(1, 1, 16, 0, 16, 5, 64, 0, ctypes.byref(n)) == _lib.HB_ERR_SHAPE
    assert lib.hb_context_workspace_bytes(1, 1, 16, 0, 16, 16, 64, 0, None) == _lib.HB_ERR_NULL


def test_more_work_units_than_32_bits_count_are_refused(lib):
    """A broadcast batch (stride 0) makes long masked contexts of very many elements possible: 2^22 x 1,024 units."""
    big = dict(batch=1 << 22, q_len=40, kv_len=1 << 24, heads=1, kv_heads=1, q_bs=40 * 64, q_rs=64, kv_bs=0, kv_rs=128,
               o_bs=40 * 64, o_rs=64, mask=P)
    assert lib.hb_context_attn(*_args(**big)) == _lib.HB_ERR_SHAPE
    n = ctypes.c_size_t(0)
    assert lib.hb_context_workspace_bytes(1 << 22, 40, 1 << 24, 0, 1, 1, 64, 1, ctypes.byref(n)) == _lib.HB_ERR_SHAPE


def test_workspace_stays_small_against_the_inputs(lib):
    """Only calls with few rows are cut along the keys, so partial results stay below a few passes over q."""
    for b, lq, lkv, ls, h, hkv, d in [(2, 2648, 8184, 0, 16, 16, 64), (8, 646, 128, 2584, 16, 16, 64),
                                      (32, 1, 257, 16384, 16, 4, 64), (8, 1, 32768, 0, 16, 4, 64)]:
        assert _need(lib, b, lq, lkv, ls, h, hkv, d) <= 64 << 20


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call", [
    lambda f, s: f(_t(2, 3, 128), _t(2, 4, 256), 2, 80),                                  # head_dim
    lambda f, s: f(_t(2, 3, 192), _t(2, 4, 256), 3, 64, kv_heads=2),                      # heads per kv head
    lambda f, s: f(_t(2, 3, 128), _t(2, 4, 128), 2, 64),                                  # kv width
    lambda f, s: f(_t(2, 3, 100), _t(2, 4, 256), 2, 64),                                  # q width
    lambda f, s: f(_t(2, 3, 128), _t(1, 4, 256), 2, 64),                                  # batch
    lambda f, s: f(_t(2, 3, 128, dtype=torch.float32), _t(2, 4, 256, dtype=torch.float32), 2, 64),
    lambda f, s: f(_t(2, 3, 128), _t(2, 4, 256, dtype=torch.float16), 2, 64),             # mixed types
    lambda f, s: f(_t(2, 3, 128), _t(2, 4, 256), 2, 64, lens=torch.zeros(2, dtype=torch.int64)),
    lambda f, s: f(_t(2, 3, 128), _t(2, 4, 256), 2, 64, lens=torch.zeros(3, dtype=torch.int32)),
    lambda f, s: f(_t(2, 3, 128), _t(2, 4, 256), 2, 64, mask=torch.ones(2, 5, dtype=torch.bool)),
    lambda f, s: f(_t(2, 3, 128), _t(2, 4, 256), 2, 64, mask=torch.ones(2, 4)),
    lambda f, s: f(_t(2, 3, 128), _t(2, 4, 256), 2, 64, out=_t(2, 3, 64)),
    lambda f, s: s(_t(2, 3, 128), _t(4, 128), _t(2, 4, 256), 2, 64),
    lambda f, s: s(_t(2, 3, 128), _t(1, 4, 256), _t(2, 4, 256), 2, 64),
    lambda f, s: s(_t(2, 3, 128), _t(5, 256), _t(2, 4, 256), 2, 64, shared_mask=torch.ones(4, dtype=torch.bool)),
])
def test_python_refusals(call):
    from hummingbird_b200.context_attention import context_attention, shared_context_attention
    with pytest.raises(ValueError):
        call(context_attention, shared_context_attention)


def test_no_cpu_path():
    from hummingbird_b200.context_attention import context_attention
    with pytest.raises(RuntimeError):
        context_attention(_t(2, 3, 128), _t(2, 4, 256), 2, 64)
