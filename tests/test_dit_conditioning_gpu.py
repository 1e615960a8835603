"""GPU: the DiT with the conditioning operators together, as a clip uses them: plain cross-attention over a padded
prompt and shared states (`cross_differential=False`), and 4-bit embedders (`cond_quant="w4"`)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPE = dict(batch=2, latents=150, depth=2, steps=2, context=130)


def _inputs(seed, batch=2, latents=150, context=130, steps=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    bf = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    mask = torch.rand(batch, context, generator=g, device="cuda") < 0.5
    mask[:, -1] = True  # the duration token behind the prompt's padding
    return (bf(batch, context, 768), bf(batch, 768), bf(batch, 64, latents), bf(steps, batch, 64, latents), mask,
            bf(300, 768))


def _step(model, inputs, masked=True, shared=True):
    cross, glob, x, eps, mask, shared_cond = inputs
    static = model.prepare_static(cross, glob, **({"cross_mask": mask} if masked else {}),
                                  **({"shared_cond": shared_cond} if shared else {}))
    t = torch.full((2,), 0.9, device="cuda", dtype=torch.bfloat16)
    return model.step(x, t, torch.full_like(t, 0.5), eps[0], static).float()


@pytest.mark.parametrize("kv_heads", [None, 4])
@pytest.mark.parametrize("masked,shared", [(False, False), (True, False), (False, True), (True, True)])
def test_plain_cross_attention_matches_torch_glue(cuda_lib, kv_heads, masked, shared):
    """The same tolerance as the differential DiT's fused glue against torch ops."""
    from hummingbird_b200.config import DiTConfig
    from hummingbird_b200.dit import ClipShape, DiT
    cfg = DiTConfig(cross_differential=False, cross_kv_heads=kv_heads)
    inputs = _inputs(1)
    outs = [_step(DiT(cfg, ClipShape(**SHAPE), "cuda", glue=glue), inputs, masked, shared) for glue in ("cuda", "torch")]
    rel = ((outs[0] - outs[1]).norm() / outs[1].norm()).item()
    assert torch.isfinite(outs[0]).all() and rel < 2e-2, f"relative difference {rel:.3e}"


def test_padding_and_its_contents_do_not_matter(cuda_lib):
    """Context tokens that the mask leaves out change nothing, whatever they hold; those it keeps do."""
    from hummingbird_b200.config import DiTConfig
    from hummingbird_b200.dit import ClipShape, DiT
    model = DiT(DiTConfig(cross_differential=False), ClipShape(**SHAPE), "cuda")
    cross, glob, x, eps, mask, shared = _inputs(2)
    ref = _step(model, (cross, glob, x, eps, mask, shared))
    other = torch.where(mask[..., None], cross, torch.full_like(cross, float("nan")))
    assert torch.equal(_step(model, (other, glob, x, eps, mask, shared)), ref)
    moved = torch.where(mask[..., None], cross * 2, cross)
    assert not torch.equal(_step(model, (moved, glob, x, eps, mask, shared)), ref)


def test_w4_embedders_match_their_dequantised_weights(cuda_lib):
    """The 4-bit embedders against the same model holding the matrices that they stand for, in fp64: bf16 roundings
    of the activations between the two layers and of the result (2^-8 each, the first through the second layer)."""
    from hummingbird_b200.config import DiTConfig
    from hummingbird_b200.dit import ClipShape, DiT
    from hummingbird_b200.w4 import dequantize_w4
    model = DiT(DiTConfig(cond_quant="w4"), ClipShape(**SHAPE), "cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    for name, layers in model.cond_layers.items():
        x = torch.randn(2, layers[0].in_features, generator=g, device="cuda").to(torch.bfloat16)
        w = [dequantize_w4(m.packed, m.scales, m.out_features, m.in_features, m.group).double() for m in layers]
        mid = torch.nn.functional.silu(x.double() @ w[0].T)
        ref = mid @ w[1].T
        tol = 2.0 ** -8 * (mid.abs() @ w[1].abs().T + ref.abs()) * (1 + 2.0 ** -7) + 1e-4
        got = model._embed(name, x).double()
        assert got.shape == ref.shape and ((got - ref).abs() <= tol).all(), name


def test_whole_clip_in_one_graph_equals_eager(cuda_lib):
    """All of them in the denoise loop: W4 embedders, plain masked cross-attention over shared states, W8A8 MLP,
    captured once and replayed on refilled latents, against the same steps run eagerly."""
    from hummingbird_b200 import _lib
    from hummingbird_b200.config import DiTConfig
    from hummingbird_b200.dit import ClipShape, DiT
    cfg = DiTConfig(cross_differential=False, cross_kv_heads=8, cond_quant="w4", ff_quant="w8a8")
    model = DiT(cfg, ClipShape(**SHAPE), "cuda")
    cross, glob, x, eps, mask, shared = _inputs(4)
    static = model.prepare_static(cross, glob, cross_mask=mask, shared_cond=shared)
    x0 = x.clone()
    run, graph = model.denoise_graph(x0, eps, static, steps=2)
    sched = [float(v) for v in model.schedule(2, device=x.device)]
    for scale in (1.0, 0.5):
        x0.copy_(x * scale)
        got = run().clone()
        y = x * scale
        for s in range(2):
            full = lambda v: torch.full((2,), v, device="cuda", dtype=torch.bfloat16)  # noqa: E731
            y = model.step(y, full(sched[s]), full(sched[s + 1]), eps[s], static)
        torch.cuda.synchronize()
        assert torch.isfinite(got).all() and torch.equal(got, y)
    del run, graph
    assert _lib.device_status() == 0


def test_refuses_what_the_configuration_does_not_have(cuda_lib):
    from hummingbird_b200.config import DiTConfig
    from hummingbird_b200.dit import ClipShape, DiT
    with pytest.raises(ValueError):
        DiT(DiTConfig(cross_differential=False, cross_kv_heads=5), ClipShape(**SHAPE), "cuda")
    with pytest.raises(ValueError):
        DiT(DiTConfig(cross_kv_heads=4), ClipShape(**SHAPE), "cuda")
    model = DiT(DiTConfig(), ClipShape(**SHAPE), "cuda")
    cross, glob, x, eps, mask, shared = _inputs(5)
    with pytest.raises(ValueError):
        model.prepare_static(cross, glob, cross_mask=mask)
    with pytest.raises(ValueError):
        model.prepare_static(cross, glob, shared_cond=shared)
