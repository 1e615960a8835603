"""GPU: context attention at its edges: mask buffers handed from unit to unit, launches that overlap, values that are
not finite, weights far below the largest one, key lists that are cut for a last round of CTAs."""
import numpy as np
import pytest
import torch

from oracle.context import context_attention as plain

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
UNIT = {BF16: 2.0 ** -8, FP16: 2.0 ** -11}


def _np(t):
    return None if t is None else t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _make(seed, b, lq, lkv, h, hkv, d, dtype, ls=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b, lq, h * d, generator=g).to(dtype).cuda()
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


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,lq,h,d", [(3, 2000, 16, 64), (3, 2000, 8, 128)])
def test_units_without_keys_between_masked_ones(cuda_lib, b, lq, h, d, dtype):
    """Several units to a CTA (768 on 592, 384 on 296), so its two mask buffers are filled again and again: one batch
    element whose last tiles hold no valid key (every role skips them and gives the buffer back), one without any key,
    one with a single key in the last tile."""
    lkv = 401
    q, kv, _ = _make(40, b, lq, lkv, h, h, d, dtype)
    mask = (torch.rand(b, lkv, generator=torch.Generator().manual_seed(41)) < 0.5).cuda()
    mask[0, 0], mask[0, 70:] = True, False
    mask[1] = False
    mask[2, 64:], mask[2, 400] = False, True
    dirty = kv.masked_fill(~mask[..., None], float("nan"))
    ref = _call(q, dirty, h, d, mask=mask)
    assert (ref[1] == 0).all() and torch.isfinite(ref).all()
    rows = torch.arange(0, lq, 53).cuda()
    _check(ref[:, rows], q[:, rows], dirty, h, d, mask=mask)
    for _ in range(5):
        assert torch.equal(_call(q, dirty, h, d, mask=mask), ref)


def test_early_launches_of_both_head_dims_on_two_streams(cuda_lib):
    """Each launch may start under the end of the one before it, and its CTAs then hold tensor memory while they wait:
    calls that take 128 and 256 columns a CTA in turn, on two streams at once, more CTAs than run at once."""
    sets = [(*_make(42 + i, b, lq, 300, h, h, d, BF16)[:2], h, d)
            for i, (b, lq, h, d) in enumerate([(2, 700, 16, 64), (1, 900, 6, 128), (1, 130, 2, 64), (2, 1500, 16, 128)])]
    refs = [_call(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for turn in range(12):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                for i in range(len(sets)):
                    j = (i * (k + 1) + turn) % len(sets)
                    outs.append((j, _call(*sets[j])))
    torch.cuda.synchronize()
    assert all(torch.equal(out, refs[j]) for j, out in outs)
    from hummingbird_b200 import _lib
    assert _lib.device_status() == 0


FP16_FLOOR = 2.0 ** -36  # of the row's largest weight: the error of an fp16 weight below the type's normal range


@pytest.mark.parametrize("gap", [14.3, 17.0, 21.3, 25.2, 29.0])
@pytest.mark.parametrize("b,lq,d", [(300, 1, 64), (600, 40, 64), (300, 40, 128), (1, 1, 64), (1, 200, 128)])
def test_fp16_weights_far_below_the_largest(cuda_lib, b, lq, d, gap):
    """One key with weight 1 and value 0 in front of 20,000 whose weights are 2^-gap and whose values are 1: fp16's
    normal range ends at 2^-14, and what is lost below it adds up. Key lists walked whole by either kernel (many batch
    elements) and cut."""
    n = 20000
    kv = torch.zeros(1, n + 1, 2 * d, dtype=FP16)
    kv[0, 0, :d] = gap * np.log(2) / d ** 0.5
    kv[0, 1:, :d] = 0.01 * torch.randn(n, d, generator=torch.Generator().manual_seed(50))
    kv[0, 1:, d:] = 1.0
    kv = kv.cuda().expand(b, -1, -1)
    q = torch.ones(b, lq, d, dtype=FP16, device="cuda")
    q[:, 1::2] = 0.75
    out = _call(q, kv, 1, d)
    pick = torch.tensor(sorted({0, b // 2, b - 1}))
    rows = torch.arange(min(2, lq))
    ref, tol = plain(_np(q[pick][:, rows]), _np(kv[pick]), 1, d, unit=UNIT[FP16], floor=FP16_FLOOR)
    got = _np(out[pick][:, rows])
    over = np.abs(got - ref) - tol
    assert over.max() <= 0, f"{got.flat[0]:.4e} instead of {ref.flat[0]:.4e}, bound {tol.flat[0]:.1e}"
    assert torch.equal(out[0, :lq], out[b - 1, :lq])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,lq,lkv,ls,h,hkv,d", [
    (2, 2, 300, 0, 4, 2, 64),          # few rows, whole
    (2, 2, 9000, 0, 4, 2, 128),        # few rows, cut
    (2, 200, 300, 0, 2, 2, 64),        # many rows
    (1, 200, 3000, 0, 2, 2, 128),      # many rows, cut
    (2, 1, 7, 70000, 8, 2, 64),        # pooled, few rows
    (33, 1, 257, 4200, 8, 2, 64),      # pooled in the tcgen05 kernel
    (1, 10200, 1000, 0, 8, 4, 64),     # the last round's items cut
])
def test_a_query_that_is_nan_shows(cuda_lib, b, lq, lkv, ls, h, hkv, d, dtype):
    """A NaN query gives NaN in its own row and head, whether the key list is cut or not, and changes nothing else."""
    q, kv, sh = _make(52, b, lq, lkv, h, hkv, d, dtype, ls=ls)
    ref = _call(q, kv, h, d, kv_heads=hkv, shared_kv=sh)
    at = [(0, 0, 0), (b - 1, lq - 1, h - 1)]
    for bq, i, hq in at:
        q[bq, i, hq * d + 5] = float("nan")
    out = _call(q, kv, h, d, kv_heads=hkv, shared_kv=sh)
    for bq, i, hq in at:
        assert out[bq, i, hq * d:(hq + 1) * d].isnan().all(), f"NaN query {bq, i, hq} is lost"
        out[bq, i, hq * d:(hq + 1) * d] = ref[bq, i, hq * d:(hq + 1) * d]
    assert torch.equal(out, ref)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lq,d", [(2, 64), (2, 128), (200, 64), (200, 128)])
def test_a_valid_key_that_is_not_finite_shows(cuda_lib, lq, d, dtype):
    """NaN in a valid key, or a score of +inf, makes the softmax NaN, wherever in a tile the key lies; the other batch
    elements keep their bits."""
    b, h, lkv = 3, 2, 150
    q, kv, _ = _make(51, b, lq, lkv, h, h, d, dtype)
    q[..., ::d] = 1.0
    ref = _call(q, kv, h, d)
    for bad in (float("nan"), float("inf")):
        for key in (*range(64, 72), 3, 6, 15, 127, lkv - 1):
            x = kv.clone()
            x[1, key, 0] = bad                       # head 0 of batch element 1
            out = _call(q, x, h, d)
            assert out[1, :, :d].isnan().all(), f"{bad} at key {key} is lost"
            assert torch.equal(out[1, :, d:], ref[1, :, d:]) and torch.equal(out[::2], ref[::2])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,lq,lkv,d", [(2, 2, 100, 64), (2, 2, 5000, 128), (2, 200, 100, 64), (2, 200, 100, 128),
                                        (1, 200, 3000, 64)])
def test_scores_of_minus_infinity(cuda_lib, b, lq, lkv, d, dtype):
    """Keys of score -inf have weight 0; where every valid key has it there is no weight at all, and the row is zero."""
    q, kv, _ = _make(53, b, lq, lkv, 1, 1, d, dtype)
    q[..., 0] = 1.0
    kv[..., 0] = -float("inf")
    assert (_call(q, kv, 1, d) == 0).all()
    kv[:, lkv // 2, 0] = 0.5
    assert torch.equal(_call(q, kv, 1, d), kv[:, lkv // 2, d:][:, None].expand(b, lq, d))


CUT_LAST_ROUND = [
    # b, lq, lkv, heads, kv heads, head_dim: more row tiles than run at once, and a last round that leaves CTAs idle
    (3, 3400, 1000, 8, 4, 64),    # 648 on 592: all of the last round is the last batch element's
    (2, 2648, 2000, 16, 16, 64),  # 672
    (5, 1630, 900, 5, 5, 128),    # 325 on 296
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,lq,lkv,h,hkv,d", CUT_LAST_ROUND)
def test_last_round_with_lengths_masks_and_norm(cuda_lib, b, lq, lkv, h, hkv, d, dtype):
    """The items of a last, partly filled round are cut along the keys: over lengths (cut units without keys, or with
    fewer tiles than parts), masks, the query norm, shared states and several batch elements."""
    ctas, items = (592 if d == 64 else 296), b * hkv * -(-lq * (h // hkv) // 128)
    assert items > ctas and items % ctas
    q, kv, sh = _make(60, b, lq, lkv, h, hkv, d, dtype, ls=100)
    g = torch.Generator().manual_seed(61)
    w = (1 + 0.1 * torch.randn(d, generator=g)).cuda()
    rows = torch.cat([torch.arange(0, lq, 211), torch.arange(lq - 130, lq, 9)]).unique().cuda()
    j = torch.arange(lkv, device="cuda")[None]
    mask = (torch.rand(b, lkv, generator=g) < 0.5).cuda()
    mask[-1, 150:] = False                       # the last element's later tiles hold no valid key
    for last in (lkv, 100, 1, 0):
        lens = torch.full((b,), lkv, dtype=torch.int32, device="cuda")
        lens[-1], lens[0] = last, lkv - 37
        for use_mask, shared in ((False, None), (True, None), (True, sh)):
            valid = (j < lens[:, None]) & (mask if use_mask else True)
            dirty = kv.masked_fill(~valid[..., None], float("nan"))
            kw = dict(kv_heads=hkv, lens=lens, mask=mask if use_mask else None, q_weight=w, shared_kv=shared)
            out = _call(q, dirty, h, d, **kw)
            assert torch.isfinite(out).all()
            _check(out[:, rows], q[:, rows], dirty, h, d, **kw)
            assert torch.equal(_call(q, dirty, h, d, **kw), out)


def test_inputs_rewritten_in_place_before_every_call(cuda_lib):
    """Kernels that start under the end of the one before read only what it leaves behind: queries, norm weights, lengths
    and masks that the kernel right before each call rewrites, through both kernels, side by side, and W4 layers."""
    from hummingbird_b200 import w4
    shapes = [(4, 2, 300, 0, 4, 2, 64), (2, 200, 300, 0, 2, 2, 64), (33, 1, 257, 4200, 8, 2, 64), (2, 200, 300, 0, 2, 2, 128)]
    for b, lq, lkv, ls, h, hkv, d in shapes:
        qa, kv, sh = _make(70, b, lq, lkv, h, hkv, d, BF16, ls=ls)
        qb, _, _ = _make(71, b, lq, 1, h, hkv, d, BF16)
        g = torch.Generator().manual_seed(72)
        sets = [(x, (1 + 0.3 * torch.randn(d, generator=g)).cuda(),
                 torch.randint(1, lkv + 1, (b,), generator=g, dtype=torch.int32).cuda(),
                 (torch.rand(b, lkv, generator=g) < 0.5).cuda()) for x in (qa, qb)]
        live = [t.clone() for t in sets[0]]
        one = lambda q, w, n, m: _call(q, kv, h, d, kv_heads=hkv, shared_kv=sh, q_weight=w, lens=n, mask=m)  # noqa: E731
        refs = []
        for s in sets:
            refs.append(one(*s))
            torch.cuda.synchronize()
        outs = []
        for turn in range(60):
            for which, t in enumerate(live):     # one of them by the last kernel before the call, each in its turn
                if which != turn % 4:
                    t.copy_(sets[turn % 2][which])
            live[turn % 4].copy_(sets[turn % 2][turn % 4])
            outs.append(one(*live))
        assert all(torch.equal(o, refs[i % 2]) for i, o in enumerate(outs))
    packed, scales = w4.quantize_w4(torch.randn(2000, 1024, device="cuda").to(BF16), 128)
    for m in (1, 9, 32):
        x = torch.randn(m, 1024, device="cuda").to(BF16)
        ref = w4.w4_linear(x, packed, scales, 2000, 128)
        outs = []
        for _ in range(60):
            x.neg_()
            outs.append(w4.w4_linear(x, packed, scales, 2000, 128))
        assert all(torch.equal(o, ref if i % 2 else -ref) for i, o in enumerate(outs))


@pytest.mark.parametrize("b,lq,ls,h,hkv,d", [(6, 1820, 25804, 8, 4, 128), (2, 3, 40, 2, 2, 64)])
def test_masks_of_no_state(cuda_lib, b, lq, ls, h, hkv, d):
    """A batch whose elements have no own states may still pass its (empty) mask: the call is that of none, workspace
    included, however many shared states there are."""
    q, kv, sh = _make(80, b, lq, 0, h, hkv, d, BF16, ls=ls)
    mask = torch.ones(b, 0, dtype=torch.bool, device="cuda")
    kw = dict(kv_heads=hkv, shared_kv=sh)
    out = _call(q, kv, h, d, mask=mask, **kw)
    assert torch.equal(out, _call(q, kv, h, d, **kw))
    rows = torch.arange(0, lq, max(1, lq // 3)).cuda()
    _check(out[:1, rows], q[:1, rows], kv[:1], h, d, **kw)
    empty = _call(q[:, :3], kv, h, d, kv_heads=hkv, mask=mask, shared_kv=sh[:0],
                  shared_mask=torch.ones(0, dtype=torch.bool, device="cuda"))
    assert (empty == 0).all()


@pytest.mark.parametrize("h,d", [(16, 64), (8, 128)])
def test_right_behind_library_products(cuda_lib, h, d):
    """As the DiT calls it: each call right behind the matrix product that makes its queries, which may let it in early."""
    b, lq, w = 2, 1500, h * d
    g = torch.Generator(device="cuda").manual_seed(90)
    bf = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF16)  # noqa: E731
    x, kv, proj = bf(b, lq, w), bf(b, 257, 2 * w), bf(4, w, w) / w ** 0.5
    refs = []
    for p in proj:
        q = x @ p
        torch.cuda.synchronize()
        refs.append(_call(q, kv, h, d))
        torch.cuda.synchronize()
    outs = [_call(x @ proj[i % 4], kv, h, d) for i in range(40)]
    assert all(torch.equal(o, refs[i % 4]) for i, o in enumerate(outs))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lq,lkv,d", [(2, 250, 64), (2, 2040, 64), (2, 2040, 128), (200, 250, 64), (200, 2040, 64),
                                      (200, 2040, 128)])
def test_scores_in_the_ten_thousands(cuda_lib, lq, lkv, d, dtype):
    """Scores around 60,000 in rising order, exact in fp32, within two of one another: the parts of a list have different
    maxima, and a rounding of one against the weights that it stands for would show (half a unit of 87,000 is 2^-8). Bound:
    roundings of the weights and of the output, 1e-4 for exponentials and fp32 sums."""
    big = (d - 1) * 16 * 60 * 64 // d
    q = torch.full((1, lq, d), 16.0 * 64 / d, dtype=dtype, device="cuda")
    q[..., 0] = 2.0 ** -7
    kv = torch.full((1, lkv, 2 * d), 60.0)
    kv[..., 0] = torch.arange(lkv) // (lkv // 250)
    kv[..., d:] = torch.randn(1, lkv, d, generator=torch.Generator().manual_seed(91))
    kv = kv.to(dtype).cuda()
    out = _call(q, kv, 1, d, scale=1.0).double()
    s = (q.double() @ kv[..., :d].double().transpose(1, 2))
    assert s.min() > big - 1 and s.max() < big + 3
    p, v = torch.softmax(s, -1), kv[..., d:].double()
    ref, a = p @ v, p @ v.abs()
    u = UNIT[dtype]
    assert ((out - ref).abs() <= u * (a + ref.abs()) * (1 + u) + 1e-4 * a).all(), (out - ref).abs().max().item()
