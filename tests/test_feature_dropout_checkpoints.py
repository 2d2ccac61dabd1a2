"""Feature dropout has no parameters: checkpoints are the same with and
without it."""

import pytest
import torch

from deepof_amd import ops
from deepof_amd.models import build_model

SMALL = {"st_single": {"input_hw": (64, 64), "fc_dim": 32, "num_classes": 5},
         "st_baseline": {"input_hw": (64, 64), "fc_dim": 32, "num_classes": 5}}


@pytest.mark.parametrize("name", ["flownets", "flownetc", "vgg16",
                                  "inception_v3", "st_single", "st_baseline"])
@pytest.mark.parametrize("norm", [None, "group"])
def test_checkpoints_fit_with_and_without(name, norm):
    kw = SMALL.get(name, {})
    torch.manual_seed(0)
    plain, _, _ = build_model(name, norm=norm, **kw)
    dropped, _, _ = build_model(name, norm=norm, feature_dropout=0.3, **kw)
    assert any(getattr(m, "dropout", 0.0) == 0.3 or (
        isinstance(m, ops.CounterDropout) and m.p == 0.3)
        for m in dropped.modules())
    assert list(plain.state_dict()) == list(dropped.state_dict())
    dropped.load_state_dict(plain.state_dict())
    plain.eval(), dropped.eval()
    x = torch.randn(1, 6, 64, 64)
    with torch.no_grad():
        want, got = plain(x), dropped(x)
    if isinstance(want, tuple):
        want, got = want[0] + [want[1]], got[0] + [got[1]]
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)
    # and back, from the state while training
    dropped.train()
    plain.load_state_dict(dropped.state_dict())


@pytest.mark.parametrize("name", ["flownets", "vgg16"])
def test_earlier_checkpoints_with_dropout_are_read(name):
    """Where each layer was the first of two modules."""
    model, _, _ = build_model(name, feature_dropout=0.3)
    layers = [n for n, m in model.named_modules()
              if getattr(m, "drop", None) is not None]
    assert layers
    old = {}
    for key, value in model.state_dict().items():
        for n in layers:
            if key.startswith(n + "."):
                key = f"{n}.0.{key[len(n) + 1:]}"
                break
        old[key] = torch.full_like(value, 0.5)
    for feature_dropout in (0.0, 0.3):
        model, _, _ = build_model(name, feature_dropout=feature_dropout)
        model.load_state_dict(old)
        assert all(bool((p == 0.5).all()) for p in model.parameters())
    # a normed model's are not taken for those
    normed, _, _ = build_model(name, norm="group")
    with pytest.raises(RuntimeError):
        model.load_state_dict(normed.state_dict())


def test_layers_drop_behind_their_activation():
    from deepof_amd.models.common import conv, deconv

    torch.manual_seed(0)
    x = torch.randn(2, 8, 6, 6)
    for build in (conv, deconv):
        plain, dropped = build(8, 16), build(8, 16, dropout=0.5)
        dropped.load_state_dict(plain.state_dict())
        y, want = dropped(x), plain(x)
        kept = y != 0
        assert 0.3 < float(kept.float().mean()) < 0.7
        torch.testing.assert_close(y[kept], 2 * want[kept])
        y.sum().backward()
        assert all(p.grad.abs().sum() > 0 for p in dropped.parameters())
