"""Hooks on the modules that the fused channels-last group norm stands for run as without it.  On the CPU, where the fused
kernel itself refuses its tensors: what runs here runs through the modules."""
import pytest
import torch

from style_transfer_amd import unet as U

KINDS = {
    "forward": lambda m, f: m.register_forward_hook(lambda *a: f()),
    "forward pre": lambda m, f: m.register_forward_pre_hook(lambda *a: f()),
    "backward": lambda m, f: m.register_full_backward_hook(lambda *a: f()),
    "backward pre": lambda m, f: m.register_full_backward_pre_hook(lambda *a: f()),
}


def block():
    torch.manual_seed(1)
    b = U.ResBlock(32, 16, 64).to(memory_format=torch.channels_last)
    b.fused_norm = True
    return b


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("which", ["layers", "norm", "act"])
def test_resblock_hooks_run(which, kind):
    b, seen = block(), []
    hooks = []
    for name in ("in_layers", "out_layers"):
        layers = getattr(b, name)
        m = {"layers": layers, "norm": layers[0], "act": layers[1]}[which]
        hooks.append(KINDS[kind](m, lambda name=name: seen.append(name)))
    x, emb = torch.randn(2, 32, 6, 5, requires_grad=True), torch.randn(2, 16)
    y = b(x, emb)
    y.sum().backward()
    assert sorted(set(seen)) == ["in_layers", "out_layers"]
    b.fused_norm = False
    assert torch.equal(b(x, emb), y)
    b.fused_norm = True
    for h in hooks:                                     # gone: the fused kernel again
        h.remove()
    with pytest.raises(RuntimeError, match="GPU memory"):
        b(x, emb)


def test_global_hooks_see_every_module():
    b, seen = block(), []
    h = torch.nn.modules.module.register_module_forward_hook(lambda m, *a: seen.append(m))
    try:
        b(torch.randn(1, 32, 4, 4), torch.randn(1, 16))
    finally:
        h.remove()
    assert all(m in seen for m in (b.in_layers, *b.in_layers, b.out_layers, *b.out_layers))


def test_transformer_norm_hook_runs():
    t, seen = U.SpatialTransformer(32, 4, 8), []
    t.fused_norm = True
    t.norm.register_forward_hook(lambda *a: seen.append(1))
    t.proj_in.register_forward_pre_hook(lambda *a: seen.append(2))
    try:
        t(torch.randn(1, 32, 4, 4))
    except (RuntimeError, TypeError):                   # the attention behind it needs a GPU
        pass
    assert seen == [1, 2]


def test_output_layers_hook_runs():
    """The network's last layers, with stock blocks and no transformers before them."""
    model = U.UNetModel(model_channels=32, num_heads=4, channel_mult=(1,), num_res_blocks=1, attention_resolutions=(), context_dim=16)
    model.use_channels_last()
    seen = []
    for m in model.modules():
        if isinstance(m, U.ResBlock):
            m.fused_norm = False
        elif isinstance(m, U.SpatialTransformer):
            m.forward = lambda x, *a, **kw: x
    model.out.register_forward_hook(lambda *a: seen.append(1))
    with torch.no_grad():
        y = model(torch.randn(1, 4, 8, 8), torch.tensor([3]), torch.randn(1, 5, 16))
    assert seen == [1] and y.is_contiguous()
