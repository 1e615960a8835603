"""CPU (gloo): the DiT's plain cross-attention with a padding mask and shared states over ranks, and the refusals of its
configuration."""
import pytest
import torch
import torch.distributed as dist

from tests.test_parallel import _dit_inputs, _run, _stand_in_attention


def _dit(group, split_batch=True, **cfg):
    from hummingbird_b200.config import DiTConfig
    from hummingbird_b200.dit import ClipShape, DiT
    config = DiTConfig(embed_dim=512, num_heads=8, num_memory_tokens=8, cross_differential=False, **cfg)
    shape = ClipShape(batch=2, latents=88, io_channels=16, context=8, context_dim=32, depth=2, steps=2)
    return DiT(config, shape, "cpu", group=group, attend=_stand_in_attention, glue="torch",
               split_batch=split_batch), shape


def _worker(rank, world, split_batch, shared):
    full, shape = _dit(None, cross_kv_heads=4)
    cross, glob, x = _dit_inputs(shape)
    mask = torch.tensor([[True] * 3 + [False] * 4 + [True], [False] * 6 + [True] * 2])  # a different one per batch row
    states = torch.randn(11, shape.context_dim, generator=torch.Generator().manual_seed(8)) if shared else None
    t = torch.tensor([0.7, 0.4]).bfloat16()
    static = lambda m: m.prepare_static(cross, glob, cross_mask=mask, shared_cond=states)  # noqa: E731
    expect = full.forward(x, t, static(full)).float()
    model, _ = _dit(dist.group.WORLD, split_batch, cross_kv_heads=4)
    got = model.gather_latents(model.forward(model.local_view(x), t, static(model))).float()
    rel = ((got - expect).norm() / expect.norm()).item()
    assert got.shape == expect.shape and rel < 1e-2, f"rank {rank}: relative difference {rel:.2e}"
    if split_batch and world == 2:  # one batch row per rank, its own row of the mask: the same bits
        assert torch.equal(got, expect)
    other = full.forward(x, t, full.prepare_static(cross, glob, cross_mask=mask.flip(0), shared_cond=states)).float()
    assert not torch.equal(other, expect)  # the mask's rows are not interchangeable


@pytest.mark.parametrize("world,split_batch,shared", [(2, True, False), (2, False, True), (4, True, True)])
def test_masked_cross_attention_over_ranks(world, split_batch, shared):
    """Each rank takes its batch rows of the mask; shared states go to all of them."""
    _run(_worker, world, split_batch, shared)


@pytest.mark.parametrize("cfg", [dict(cross_kv_heads=0), dict(cross_kv_heads=-4), dict(cross_kv_heads=3)])
def test_kv_heads_that_do_not_divide_the_heads_are_refused(cfg):
    with pytest.raises(ValueError):
        _dit(None, **cfg)
