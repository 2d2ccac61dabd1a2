"""The step in which convolutions are tuned trains like every other one."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("winner", ["hip128", "miopen"])
@pytest.mark.parametrize("kind", ["conv", "deconv"])
def test_weights_have_gradients_in_the_tuning_step(kind, winner, monkeypatch):
    from deepof_amd.ops import conv, deconv

    if kind == "conv":
        cache, module = conv._dispatch_cache, conv.FusedConvAct(64, 64, 3, 1, None)
    else:
        cache, module = deconv._deconv_cache, deconv.FusedDeconvAct(64, 64, None)
    cache.clear()
    # both candidates are timed as ever; which one wins is set here
    tune = type(module)._autotune

    def tuned(self, x, key):
        tune(self, x, key)
        choice = winner if kind == "conv" or winner == "miopen" else "hip"
        cache[key] = choice
        return choice

    monkeypatch.setattr(type(module), "_autotune", tuned)
    module.to(DEV).to(memory_format=torch.channels_last)
    x = torch.randn(2, 64, 16, 16, device=DEV).contiguous(
        memory_format=torch.channels_last)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = module(x.bfloat16())
    y.float().square().sum().backward()
    for p in module.parameters():
        assert p.grad is not None and float(p.grad.abs().sum()) > 0
    cache.clear()
