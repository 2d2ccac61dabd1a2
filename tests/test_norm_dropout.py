"""Group norm and counter-based dropout on the CPU: the plain forms that the
kernels are held to, and what the public entry points refuse."""

import math

import pytest
import torch
import torch.nn.functional as F

from deepof_amd import ops
from deepof_amd.ops import reference as ref


def _words(*v):
    return [torch.tensor([w]) for w in v]


@pytest.mark.parametrize("counter,key,want", [
    # the known answers published with the generator
    ((0, 0, 0, 0), (0, 0),
     (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2,
     (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344),
     (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_philox_known_answers(counter, key, want):
    got = ref.philox4x32(_words(*counter), _words(*key))
    assert tuple(int(w) for w in got) == want


def test_dropout_numbers_layout():
    """u(i)'s halves come from the two counters, eight elements a block."""
    rng = torch.tensor([0x1234567_89ABCDEF, 77 + (5 << 32)])
    u = ref.dropout_numbers(21, rng)
    for i in (0, 1, 7, 8, 20):
        j, s = i // 8, i % 8
        halves = []
        for tag in (0, 1 << 31):
            w = ref.philox4x32(_words(j, tag, 77, 5),
                               _words(0x89ABCDEF, 0x1234567))
            halves.append(int(w[s // 2]) >> (16 * (s % 2)) & 0xFFFF)
        assert int(u[i]) == halves[0] << 16 | halves[1]
    assert int(u.min()) >= 0 and int(u.max()) < 2**32


@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
def test_keep_rate_and_independence(p):
    n = 1 << 18
    x = torch.ones(n)
    y = ops.dropout(x, p, (3, 4))
    keep = (y != 0).double()
    # 6 standard deviations of n draws
    assert abs(float(keep.mean()) - (1 - p)) < 6 * math.sqrt(p * (1 - p) / n)
    torch.testing.assert_close(y[y != 0], torch.full_like(y[y != 0], 1 / (1 - p)))
    other = (ops.dropout(x, p, (3, 5)) != 0).double()
    for a, b in ((keep, other), (keep[1:], keep[:-1]), (keep[8:], keep[:-8])):
        cov = float(((a - (1 - p)) * (b - (1 - p))).mean())
        assert abs(cov) < 6 * p * (1 - p) / math.sqrt(a.numel())


def test_dropout_edges():
    x = torch.tensor([1.0, float("inf"), float("nan"), -2.0])
    assert torch.equal(ops.dropout(x, 1.0, (1, 2)), torch.zeros(4))
    torch.testing.assert_close(ops.dropout(x, 0.0), x, equal_nan=True)
    assert ops.dropout(torch.empty(0, 3), 0.5, (1, 2)).shape == (0, 3)
    g = torch.ones(4, requires_grad=True)
    ops.dropout(g, 1.0, (1, 2)).sum().backward()
    assert torch.equal(g.grad, torch.zeros(4))


def test_dropout_follows_memory_order():
    x = torch.randn(2, 6, 3, 5)
    last = x.contiguous(memory_format=torch.channels_last)
    flat = x.permute(0, 2, 3, 1).reshape(-1)
    want = ops.dropout(flat, 0.4, (9, 1)).reshape(2, 3, 5, 6)
    assert torch.equal(ops.dropout(last, 0.4, (9, 1)).permute(0, 2, 3, 1), want)
    # neither contiguous nor channels last: made contiguous
    t = x.transpose(2, 3)
    assert torch.equal(ops.dropout(t, 0.4, (9, 1)),
                       ops.dropout(t.contiguous(), 0.4, (9, 1)))


def test_rng_forms_agree_and_follow_the_seed():
    x = torch.randn(1000)
    a = ops.dropout(x, 0.3, (11, 12))
    assert torch.equal(a, ops.dropout(x, 0.3, torch.tensor([11, 12])))
    torch.manual_seed(5)
    b = ops.dropout(x, 0.3)
    torch.manual_seed(5)
    rng = ops.draw_rng("cpu")
    assert torch.equal(b, ops.dropout(x, 0.3, rng))
    assert not torch.equal(b, ops.dropout(x, 0.3))


def test_dropout_under_recomputation_is_the_same():
    from torch.utils.checkpoint import checkpoint

    x = torch.randn(64, 64, dtype=torch.float64, requires_grad=True)

    def block(t):
        return ops.dropout(t, 0.5, act="elu") * t

    torch.manual_seed(1)
    want = torch.autograd.grad(block(x).sum(), x)[0]
    torch.manual_seed(1)
    got = torch.autograd.grad(
        checkpoint(block, x, use_reentrant=False).sum(), x)[0]
    assert torch.equal(got, want)


@pytest.mark.parametrize("act", [None, "elu", "leaky_relu", "relu", "silu"])
def test_group_norm_plain_form(act):
    torch.manual_seed(0)
    x = torch.randn(3, 12, 5, 7, dtype=torch.float64)
    w, b = torch.randn(12).double(), torch.randn(12).double()
    want = F.group_norm(x, 4, w, b, eps=1e-3)
    want = ref.activation(want, act)
    got = ops.group_norm(x, 4, w, b, eps=1e-3, act=act)
    torch.testing.assert_close(got, want, rtol=1e-10, atol=1e-12)
    assert got.is_contiguous(memory_format=torch.channels_last)


@pytest.mark.parametrize("act", [None, "elu", "silu"])
def test_gradients_against_differences(act):
    torch.manual_seed(0)
    x = torch.randn(2, 6, 3, 4, dtype=torch.float64, requires_grad=True)
    w = torch.randn(6, dtype=torch.float64, requires_grad=True)
    b = torch.randn(6, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(
        lambda *t: ops.group_norm(t[0], 2, t[1], t[2], act=act, dropout=0.3,
                                  rng=(1, 2)), (x, w, b))
    assert torch.autograd.gradcheck(
        lambda t: ops.dropout(t, 0.3, (1, 2), act=act), (x,))


def test_group_norm_drops_as_dropout_does():
    x = torch.randn(2, 8, 4, 6).contiguous(memory_format=torch.channels_last)
    y = ops.group_norm(x, 4, act="elu", dropout=0.4, rng=(7, 8))
    want = ops.dropout(ops.group_norm(x, 4, act="elu"), 0.4, (7, 8))
    torch.testing.assert_close(y, want)
    assert torch.equal(y == 0, want == 0)


def test_empty_inputs_have_gradients():
    for shape in ((0, 4, 3, 3), (2, 4, 0, 3)):
        x = torch.randn(shape, requires_grad=True)
        w = torch.ones(4, requires_grad=True)
        b = torch.ones(4, requires_grad=True)
        y = ops.group_norm(x, 2, w, b, act="relu")
        assert y.shape == shape
        y.sum().backward()
        assert torch.equal(w.grad, torch.zeros(4))
        assert torch.equal(b.grad, torch.zeros(4))


X = torch.zeros(2, 8, 3, 3)


@pytest.mark.parametrize("error,call", [
    (ValueError, lambda d: ops.group_norm(X.to(d)[0], 2)),
    (ValueError, lambda d: ops.group_norm(X.to(d), 3)),
    (ValueError, lambda d: ops.group_norm(X.to(d), 0)),
    (ValueError, lambda d: ops.group_norm(X.to(d), -2)),
    (ValueError, lambda d: ops.group_norm(X.to(d)[:, :0], 1)),
    (ValueError, lambda d: ops.group_norm(
        torch.zeros(1, 8192, 1, 1, device=d), 8192)),
    (TypeError, lambda d: ops.group_norm(X.to(d), 2.0)),
    (TypeError, lambda d: ops.group_norm(X.to(d), True)),
    (TypeError, lambda d: ops.group_norm(X.to(d).int(), 2)),
    (TypeError, lambda d: ops.group_norm([1.0], 2)),
    (ValueError, lambda d: ops.group_norm(X.to(d), 2, torch.ones(7, device=d))),
    (ValueError, lambda d: ops.group_norm(
        X.to(d), 2, None, torch.ones(8, 1, device=d))),
    (TypeError, lambda d: ops.group_norm(
        X.to(d), 2, torch.ones(8, dtype=torch.int64, device=d))),
    (ValueError, lambda d: ops.group_norm(X.to(d), 2, eps=0.0)),
    (ValueError, lambda d: ops.group_norm(X.to(d), 2, eps=float("nan"))),
    (ValueError, lambda d: ops.group_norm(X.to(d), 2, act="gelu")),
    (ValueError, lambda d: ops.group_norm(X.to(d), 2, dropout=1.5)),
    (ValueError, lambda d: ops.dropout(X.to(d), -0.1)),
    (ValueError, lambda d: ops.dropout(X.to(d), float("nan"))),
    (TypeError, lambda d: ops.dropout(X.to(d), "0.5")),
    (TypeError, lambda d: ops.dropout(X.to(d).long(), 0.5)),
    (ValueError, lambda d: ops.dropout(X.to(d), 0.5, act="tanh")),
    (ValueError, lambda d: ops.dropout(X.to(d), 0.5, (-1, 0))),
    (ValueError, lambda d: ops.dropout(X.to(d), 0.5, (0, 2**63))),
    (TypeError, lambda d: ops.dropout(X.to(d), 0.5, (0, 1, 2))),
    (TypeError, lambda d: ops.dropout(X.to(d), 0.5, 7)),
    (ValueError, lambda d: ops.dropout(
        X.to(d), 0.5, torch.zeros(2, device=d))),
    (ValueError, lambda d: ops.dropout(
        X.to(d), 0.5, torch.zeros(3, dtype=torch.int64, device=d))),
])
def test_refusals(error, call):
    with pytest.raises(error):
        call("cpu")


# ---------------------------------------------------------------------------
# modules, models and configs
# ---------------------------------------------------------------------------
def test_modules_train_and_eval():
    torch.manual_seed(0)
    x = torch.randn(2, 48, 5, 6)
    m = ops.GroupNormAct(48, "elu", dropout=0.5)
    assert m.groups == 16
    m.eval()
    want = F.elu(F.group_norm(x, 16, m.weight, m.bias))
    torch.testing.assert_close(m(x), want)
    m.train()
    assert 0.4 < float((m(x) == 0).float().mean()) < 0.6
    d = ops.CounterDropout(0.5, "relu")
    assert 0.7 < float((d(x) == 0).float().mean()) < 0.8
    assert not torch.equal(d(x), d(x))
    d.eval()
    assert torch.equal(d(x), F.relu(x))
    for bad in (lambda: ops.GroupNormAct(10, groups=3),
                lambda: ops.GroupNormAct(8, "gelu"),
                lambda: ops.GroupNormAct(8, dropout=2.0),
                lambda: ops.CounterDropout(-1.0),
                lambda: ops.CounterDropout(0.5, "tanh")):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("name", ["flownets", "flownetc", "vgg16",
                                  "inception_v3"])
def test_models_with_group_norm(name):
    from deepof_amd.models import build_model

    torch.manual_seed(0)
    model, scales, _ = build_model(name, norm="group", feature_dropout=0.1)
    norms = [m for m in model.modules() if isinstance(m, ops.GroupNormAct)]
    assert norms and all(m.dropout == 0.1 for m in norms)
    assert not any(isinstance(m, torch.nn.BatchNorm2d)
                   for m in model.modules())
    x = torch.randn(1, 6, 64, 64)
    flows = model(x)
    assert len(flows) == len(scales) and flows[0].shape == (1, 2, 32, 32)
    sum(f.square().sum() for f in flows).backward()
    for p in model.parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all()
    model.eval()
    with torch.no_grad():
        a, b = model(x), model(x)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_models_are_as_before_without():
    from deepof_amd.models import build_model
    from deepof_amd.models.ucf101 import STSingle

    for name in ("flownets", "inception_v3"):
        model, _, _ = build_model(name)
        assert not any(isinstance(m, (ops.GroupNormAct, ops.CounterDropout))
                       for m in model.modules())
    kw = {"input_hw": (64, 64), "fc_dim": 32, "num_classes": 5}
    plain, counter = STSingle(**kw), STSingle(**kw, dropout_rng="counter")
    assert sum(isinstance(m, torch.nn.Dropout) for m in plain.modules()) == 2
    assert sum(isinstance(m, ops.CounterDropout)
               for m in counter.modules()) == 2
    # one's checkpoint is the other's
    counter.load_state_dict(plain.state_dict())
    x = torch.randn(2, 6, 64, 64)
    plain.eval(), counter.eval()
    torch.testing.assert_close(counter(x)[1], plain(x)[1])
    counter.train()
    counter(x)[1].sum().backward()
    with pytest.raises(ValueError):
        STSingle(**kw, dropout_rng="other")
    with pytest.raises(ValueError):
        build_model("flownets", norm="layer")


def test_inception_feature_dropout_without_group_norm():
    from deepof_amd.models import build_model

    model, _, _ = build_model("inception_v3", feature_dropout=0.2)
    drops = [m for m in model.modules() if isinstance(m, ops.CounterDropout)]
    assert drops and any(isinstance(m, torch.nn.BatchNorm2d)
                         for m in model.modules())
    model.eval()
    with torch.no_grad():
        assert torch.isfinite(model(torch.randn(1, 6, 64, 64))[0]).all()


def test_config_keys():
    from deepof_amd.config import Config

    cfg = Config().apply_overrides(["norm=group", "feature_dropout=0.1",
                                    "dropout_rng=counter"])
    assert (cfg.norm, cfg.feature_dropout, cfg.dropout_rng) == (
        "group", 0.1, "counter")
    assert Config().norm is None and Config().dropout_rng == "torch"
    for bad in ("norm=batch", "feature_dropout=1.5", "dropout_rng=x"):
        with pytest.raises(ValueError):
            Config().apply_overrides([bad])


def test_train_then_eval_from_the_command_line(tmp_path, capsys):
    """A checkpoint of a normed model is evaluated by the same config."""
    from deepof_amd.cli import main

    common = ["dataset=synthetic", "image_size=[64, 64]", "batch_size=2",
              "num_workers=0", "device=cpu", "norm=group",
              "feature_dropout=0.1", f"log_dir={tmp_path}", "run_name=r"]
    main(["train", "--max-steps", "1"] + common)
    ckpt = tmp_path / "r" / "ckpt_last.pt"
    assert ckpt.exists()
    main(["eval", "--checkpoint", str(ckpt)] + common)
    assert "AEE" in capsys.readouterr().out
