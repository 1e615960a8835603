"""GPU: context attention (`hummingbird_b200.context_attention`, through the C ABI) against a plain float64
implementation, element by element within the bound that the roundings of its documented arithmetic give
(`oracle.context`)."""
import numpy as np
import pytest
import torch

from oracle.context import context_attention as plain

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
UNIT = {BF16: 2.0 ** -8, FP16: 2.0 ** -11}


def _np(t):
    return None if t is None else t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _make(seed, b, lq, lkv, h, hkv, d, dtype, ls=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    q = (scale * torch.randn(b, lq, h * d, generator=g)).to(dtype).cuda()
    kv = torch.randn(b, lkv, 2 * hkv * d, generator=g).to(dtype).cuda()
    sh = torch.randn(ls, 2 * hkv * d, generator=g).to(dtype).cuda() if ls else None
    return q, kv, sh


def _call(q, kv, h, d, shared_kv=None, **kw):
    from hummingbird_b200.context_attention import context_attention, shared_context_attention
    if shared_kv is None:
        return context_attention(q, kv, h, d, **kw)
    return shared_context_attention(q, shared_kv, kv, h, d, **kw)


def _check(out, q, kv, h, d, **kw):
    ref, tol = plain(_np(q), np.nan_to_num(_np(kv), posinf=0, neginf=0), h, d, unit=UNIT[q.dtype],
                     **{k: _np(v) if torch.is_tensor(v) else v for k, v in kw.items()})
    got = _np(out)
    assert np.isfinite(got).all(), "non-finite output"
    over = np.abs(got - ref) - tol
    assert over.max() <= 0, f"off by {np.abs(got - ref).max():.3e}, {over.max():.3e} over the bound"


SHAPES = [
    # b, lq, lkv, heads, kv heads, head_dim
    (1, 1, 1, 1, 1, 64),
    (1, 1, 257, 16, 16, 64),
    (2, 3, 31, 4, 2, 64),
    (3, 5, 130, 6, 2, 128),
    (1, 16, 64, 2, 1, 128),
    (2, 17, 33, 3, 3, 64),
    (1, 127, 129, 2, 2, 64),
    (2, 128, 128, 2, 1, 128),
    (1, 129, 300, 4, 4, 64),
    (2, 300, 257, 4, 2, 64),
    (1, 1, 5000, 8, 2, 64),
    (2, 2, 3001, 4, 1, 128),
    (1, 700, 1421, 3, 1, 128),
    (2, 33, 16, 8, 1, 64),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,lq,lkv,h,hkv,d", SHAPES)
def test_matches_plain(cuda_lib, b, lq, lkv, h, hkv, d, dtype):
    q, kv, _ = _make(lq + lkv, b, lq, lkv, h, hkv, d, dtype)
    _check(_call(q, kv, h, d, kv_heads=hkv), q, kv, h, d, kv_heads=hkv)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,lq,lkv,h,hkv,d", [(4, 1, 300, 4, 2, 64), (4, 9, 129, 2, 2, 128), (4, 200, 385, 4, 4, 64),
                                              (4, 140, 1000, 4, 1, 128), (4, 1, 4000, 2, 1, 64)])
def test_lens_mask_and_garbage(cuda_lib, b, lq, lkv, h, hkv, d, dtype):
    """Lengths (one of them 0, one past the end, one negative), holes in the mask, and NaN or infinities wherever
    a state is not valid."""
    q, kv, _ = _make(7, b, lq, lkv, h, hkv, d, dtype)
    g = torch.Generator().manual_seed(8)
    lens = torch.tensor([lkv + 5, 0, -3, max(1, lkv // 3)], dtype=torch.int32)[:b].cuda()
    mask = (torch.rand(b, lkv, generator=g) < 0.6).cuda()
    mask[3, : lkv // 4] = False  # whole tiles without a valid state
    mask[3, lkv // 4] = True
    j = torch.arange(lkv, device="cuda")[None]
    for use_lens, use_mask in ((True, False), (False, True), (True, True)):
        valid = torch.ones(b, lkv, dtype=torch.bool, device="cuda")
        if use_lens:
            valid &= j < lens[:, None]
        if use_mask:
            valid &= mask
        for bad in (float("nan"), float("inf"), -float("inf")):
            dirty = kv.masked_fill(~valid[..., None], bad)
            kw = dict(kv_heads=hkv, lens=lens if use_lens else None, mask=mask if use_mask else None)
            out = _call(q, dirty, h, d, **kw)
            _check(out, q, dirty, h, d, **kw)
            if use_lens:
                assert (out[1:3] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,lq,lkv,ls,h,hkv,d", [(2, 1, 5, 300, 4, 2, 64), (5, 3, 40, 1000, 8, 2, 64),
                                                 (3, 17, 33, 201, 4, 4, 128), (3, 200, 64, 257, 2, 2, 64),
                                                 (2, 130, 129, 16, 4, 1, 128), (32, 1, 257, 2048, 8, 2, 64),
                                                 (1, 1, 7, 900, 4, 1, 128), (40, 1, 3, 100, 2, 2, 128)])
def test_shared_states(cuda_lib, b, lq, lkv, ls, h, hkv, d, dtype):
    q, kv, sh = _make(9, b, lq, lkv, h, hkv, d, dtype, ls=ls)
    g = torch.Generator().manual_seed(10)
    lens = torch.randint(0, lkv + 1, (b,), generator=g, dtype=torch.int32).cuda()
    mask = (torch.rand(b, lkv, generator=g) < 0.7).cuda()
    smask = (torch.rand(ls, generator=g) < 0.7).cuda()
    dirty = sh.masked_fill(~smask[:, None], float("nan"))
    for kw in (dict(), dict(lens=lens), dict(lens=lens, mask=mask)):
        _check(_call(q, kv, h, d, shared_kv=sh, kv_heads=hkv, **kw), q, kv, h, d, shared_kv=sh, kv_heads=hkv, **kw)
    out = _call(q, kv, h, d, shared_kv=dirty, shared_mask=smask, kv_heads=hkv, mask=mask)
    _check(out, q, kv, h, d, shared_kv=sh, shared_mask=smask, kv_heads=hkv, mask=mask)
    # no own states at all; no valid state anywhere
    none = kv[:, :0]
    _check(_call(q, none, h, d, shared_kv=sh, kv_heads=hkv), q, none, h, d, shared_kv=sh, kv_heads=hkv)
    empty = _call(q, kv, h, d, shared_kv=sh, kv_heads=hkv, shared_mask=torch.zeros_like(smask),
                  lens=torch.zeros_like(lens))
    assert (empty == 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,lq,lkv,ls,h,hkv,d", [
    (2, 1, 7, 70000, 8, 2, 64),      # pooled rows and own rows in the few-rows kernel
    (33, 1, 257, 4200, 8, 2, 64),    # pooled rows in the tcgen05 kernel, own rows beside it
    (6, 60, 33, 16000, 4, 2, 64),    # both in the tcgen05 kernel
    (24, 3, 65, 3100, 6, 2, 128),
])
def test_long_shared_states_are_pooled(cuda_lib, b, lq, lkv, ls, h, hkv, d, dtype):
    """Long enough shared states that all batch elements' rows take them in one pass, apart from their own."""
    assert (b - 1) * ls * hkv * d * 4 > 32 << 20 and lq * h // hkv < 128
    q, kv, sh = _make(30, b, lq, lkv, h, hkv, d, dtype, ls=ls)
    g = torch.Generator().manual_seed(31)
    lens = torch.randint(0, lkv + 1, (b,), generator=g, dtype=torch.int32).cuda()
    lens[0] = 0
    valid = torch.arange(lkv, device="cuda")[None] < lens[:, None]
    kw = dict(kv_heads=hkv, lens=lens)
    out = _call(q, kv.masked_fill(~valid[..., None], float("nan")), h, d, shared_kv=sh, **kw)
    _check(out, q, kv, h, d, shared_kv=sh, **kw)
    smask = (torch.rand(ls, generator=g) < 0.5).cuda()
    smask[100:1000] = False
    kw["shared_mask"] = smask
    dirty = sh.masked_fill(~smask[:, None], float("inf"))
    _check(_call(q, kv, h, d, shared_kv=dirty, **kw), q, kv, h, d, shared_kv=sh, **kw)
    none = kv[:, :0]
    _check(_call(q, none, h, d, shared_kv=sh, kv_heads=hkv), q, none, h, d, shared_kv=sh, kv_heads=hkv)


@pytest.mark.parametrize("lq,lkv,ls,h,hkv,d", [(10200, 1000, 0, 8, 4, 64), (4700, 900, 300, 16, 16, 64),
                                               (9590, 1100, 0, 4, 4, 128)])
def test_items_of_a_last_round_are_cut(cuda_lib, lq, lkv, ls, h, hkv, d):
    """More tiles of rows than run at once: the last round's key lists are cut and merged; rows sampled from every
    tile, the last, partly empty one whole."""
    q, kv, sh = _make(32, 1, lq, lkv, h, hkv, d, BF16, ls=ls)
    out = _call(q, kv, h, d, kv_heads=hkv, shared_kv=sh)
    rows = torch.cat([torch.arange(0, lq, 61), torch.arange(lq - 130, lq)]).unique().cuda()
    _check(out[:, rows], q[:, rows], kv, h, d, kv_heads=hkv, shared_kv=sh)
    assert torch.isfinite(out).all()


def test_long_masked_context_of_many_rows(cuda_lib):
    """Mask bits of more keys than a CTA holds: the key list is cut however many rows there are."""
    lq, lkv = 76000, 17000
    q, kv, _ = _make(33, 1, lq, lkv, 1, 1, 64, FP16)
    mask = (torch.rand(1, lkv, generator=torch.Generator().manual_seed(34)) < 0.5).cuda()
    mask[0, 3000:9000] = False
    out = _call(q, kv.masked_fill(~mask[..., None], float("nan")), 1, 64, mask=mask)
    rows = torch.arange(0, lq, 997).cuda()
    _check(out[:, rows], q[:, rows], kv, 1, 64, mask=mask)
    assert torch.isfinite(out).all()


def test_no_states_gives_zeros(cuda_lib):
    q, kv, _ = _make(11, 2, 5, 4, 2, 2, 64, BF16)
    assert (_call(q, kv[:, :0], 2, 64) == 0).all()
    for d in (64, 128):  # many rows: there is no key to make a tensor map of
        wide, states, sh = _make(11, 2, 300, 4, 2, 2, d, BF16, ls=3)
        assert (_call(wide, states[:, :0], 2, d) == 0).all()
        assert (_call(wide, states[:, :0], 2, d, shared_kv=sh[:0]) == 0).all()
    assert _call(q[:, :0], kv, 2, 64).shape == (2, 0, 128)
    assert _call(q[:0], kv[:0], 2, 64).shape == (0, 5, 128)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,lq,lkv,h,hkv,d", [(2, 2, 70, 4, 2, 64), (1, 260, 257, 2, 2, 64), (2, 150, 90, 4, 2, 128)])
def test_query_norm_and_scale(cuda_lib, b, lq, lkv, h, hkv, d, dtype):
    q, kv, _ = _make(12, b, lq, lkv, h, hkv, d, dtype, scale=3.0)
    w = (1 + 0.1 * torch.randn(d, generator=torch.Generator().manual_seed(13))).cuda()
    kw = dict(kv_heads=hkv, q_weight=w, eps=1e-5, scale=0.11)
    _check(_call(q, kv, h, d, **kw), q, kv, h, d, **kw)


@pytest.mark.parametrize("b,lq,lkv,d", [(2, 3, 200, 64), (2, 140, 200, 128)])
def test_strided_inputs_and_output(cuda_lib, b, lq, lkv, d):
    """Column slices of wider projections, a window of a longer cache, token-major tensors, an expanded batch; the
    output goes between rows that stay as they were."""
    h, hkv = 4, 2
    q, kv, _ = _make(14, b, lq, lkv, h, hkv, d, BF16)
    ref = _call(q, kv, h, d, kv_heads=hkv)
    wide_q = torch.full((b, lq + 2, h * d + 64), float("nan"), dtype=BF16, device="cuda")
    wide_q[:, 1:-1, 32:32 + h * d] = q
    cache = torch.full((b, lkv + 50, 2 * hkv * d + 8), float("nan"), dtype=BF16, device="cuda")
    cache[:, 20:20 + lkv, :2 * hkv * d] = kv
    buf = torch.full((b, lq + 3, h * d + 16), 7.0, dtype=BF16, device="cuda")
    out = buf[:, 1:1 + lq, 8:8 + h * d]
    got = _call(wide_q[:, 1:-1, 32:32 + h * d], cache[:, 20:20 + lkv, :2 * hkv * d], h, d, kv_heads=hkv, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, ref)
    rest = buf.clone()
    rest[:, 1:1 + lq, 8:8 + h * d] = 7.0
    assert (rest == 7.0).all()
    tok = q.transpose(0, 1).contiguous().transpose(0, 1)          # (Lq, B, W) in memory
    tok_out = torch.empty(lq, b, h * d, dtype=BF16, device="cuda").transpose(0, 1)
    assert torch.equal(_call(tok, kv.transpose(0, 1).contiguous().transpose(0, 1), h, d, kv_heads=hkv, out=tok_out), ref)
    one = kv[:1].expand(b, -1, -1)                                  # batch stride 0
    assert torch.equal(_call(q, one, h, d, kv_heads=hkv), _call(q, one.contiguous(), h, d, kv_heads=hkv))
    odd = torch.empty(b, lq, h * d + 1, dtype=BF16, device="cuda")[..., 1:]  # unaligned rows are copied
    odd.copy_(q)
    assert torch.equal(_call(odd, kv, h, d, kv_heads=hkv), ref)


def test_offsets_past_32_bits(cuda_lib):
    """Rows 2 MiB apart: the last ones lie more than 2^32 bytes and 2^31 elements behind the first."""
    lkv, stride = 2200, 1 << 20
    q, kv, _ = _make(15, 1, 2, lkv, 2, 1, 64, BF16)
    far = torch.empty(lkv * stride, dtype=BF16, device="cuda").as_strided((1, lkv, 128), (lkv * stride, stride, 1))
    far.copy_(kv)
    ref = _call(q, kv, 2, 64, kv_heads=1)
    assert torch.equal(_call(q, far, 2, 64, kv_heads=1), ref)
    q2, _, _ = _make(16, 1, 200, 1, 2, 1, 64, BF16)
    assert torch.equal(_call(q2, far, 2, 64, kv_heads=1), _call(q2, kv, 2, 64, kv_heads=1))
    assert torch.equal(_call(q, kv[:, :5], 2, 64, kv_heads=1, shared_kv=far[0]),
                       _call(q, kv[:, :5], 2, 64, kv_heads=1, shared_kv=kv[0]))


def test_large_scores(cuda_lib):
    """Scores in the hundreds, in rising order along the keys, so the running maximum moves at every step."""
    for lq in (2, 200):
        q = torch.full((1, lq, 64), 1.0, dtype=BF16, device="cuda")
        kv = torch.randn(1, 900, 128, generator=torch.Generator().manual_seed(17)).to(BF16).cuda()
        kv[0, :, :64] = (torch.arange(900, device="cuda")[:, None] / 8).to(BF16)
        for sign in (1, -1):
            x = kv.clone()
            x[..., :64] *= sign
            _check(_call(q, x, 1, 64), q, x, 1, 64)


def test_same_call_same_bits_and_streams(cuda_lib):
    q, kv, sh = _make(18, 4, 2, 3000, 8, 2, 64, BF16, ls=22000)  # pooled: two kernels and a merge
    ref = _call(q, kv, 8, 64, shared_kv=sh, kv_heads=2)
    for _ in range(3):
        assert torch.equal(_call(q, kv, 8, 64, shared_kv=sh, kv_heads=2), ref)
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(_call(q, kv, 8, 64, shared_kv=sh, kv_heads=2))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)


def test_two_graphs_replayed_together(cuda_lib):
    """Two captured calls with split key lists, replayed on two streams at once, each on inputs refilled in place."""
    sets = [_make(20, 2, 1, 6000, 8, 2, 64, BF16, ls=70000), _make(21, 9, 4, 2000, 8, 2, 64, BF16, ls=9000)]
    graphs, outs = [], []
    for q, kv, sh in sets:
        _call(q, kv, 8, 64, shared_kv=sh, kv_heads=2)
    torch.cuda.synchronize()
    for q, kv, sh in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_call(q, kv, 8, 64, shared_kv=sh, kv_heads=2))
        graphs.append(g)
    for q, kv, sh in sets:
        q.mul_(-1)
    refs = [_call(q, kv, 8, 64, shared_kv=sh, kv_heads=2) for q, kv, sh in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, r) for o, r in zip(outs, refs))


def test_refuses_gradients(cuda_lib):
    q, kv, _ = _make(22, 1, 2, 8, 2, 2, 64, BF16)
    q.requires_grad_(True)
    with pytest.raises(RuntimeError):
        _call(q, kv, 2, 64)
    with torch.no_grad():
        _check(_call(q, kv, 2, 64), q.detach(), kv, 2, 64)
    with pytest.raises(RuntimeError):
        _call(q.detach(), kv, 2, 64, q_weight=torch.ones(64, device="cuda", requires_grad=True))
