"""Group norm and counter-based dropout on the GPU against the plain forms in
64 bits."""

import math
import threading

import pytest
import torch

from deepof_amd import ops
from deepof_amd.ops import reference as ref
from test_norm_dropout import test_refusals as cpu_refusals

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
LAST = torch.channels_last

# Tolerances.  A stored value is off by at most half a step, eps / 2 of it.
# Before it is rounded it comes out of fp32 arithmetic: at the sizes here the
# longest chain from an input to an output is below 200 additions in a thread,
# 20 joins and 30 other operations, each off by at most 2^-24 of the largest
# value that takes part.  256 steps of 2^-24 bound that, times the largest
# magnitude in the chain, which each test names.
CHAIN = 256 * 2.0**-24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def features(shape, dtype, seed, spread=1.0, shift=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    x = x * spread + shift * torch.randn(shape[1], generator=g).view(1, -1, 1, 1)
    return x.to(dtype).contiguous(memory_format=LAST)


def params(c, seed):
    g = torch.Generator().manual_seed(seed + 1000)
    return (1 + 0.3 * torch.randn(c, generator=g),
            0.3 * torch.randn(c, generator=g))


def assert_near(got, want, dtype, magnitude):
    """got, of `dtype`, against want in 64 bits."""
    got = got.detach().cpu().double()
    bound = half_step(dtype) * want.abs() + CHAIN * (magnitude + want.abs())
    if dtype == FP16:
        bound = bound + 2.0**-25  # half the step of its smallest values
    off = (got - want).abs() - bound
    assert got.shape == want.shape and not torch.isnan(got).any()
    assert float(off.max()) <= 0, (
        f"over the bound by {float(off.max()):.3g} at "
        f"{int(off.argmax())}: {float(got.flatten()[off.argmax()])} for "
        f"{float(want.flatten()[off.argmax()])}")


SHAPES = [  # b, c, h, w, groups
    (1, 1, 1, 1, 1),          # a single value
    (2, 8, 1, 1, 2),          # one pixel
    (1, 6, 3, 5, 3),          # single channels are moved
    (2, 32, 7, 9, 32),        # a group per channel
    (3, 80, 5, 7, 16),        # groups of 5 straddle a thread's 8 channels
    (2, 20, 9, 11, 4),        # 4 channels are moved
    (2, 64, 33, 17, 32),      # groups of 2
    (2, 96, 10, 13, 6),       # groups of 16, 12 columns
    (1, 1024, 6, 8, 32),      # few pixels, many channels
    (1, 4104, 2, 3, 1),       # a group wider than a block, its last columns few
    (2, 515, 3, 4, 5),        # odd channels, groups that cross a block's width
    (2, 16, 130, 67, 4),      # many pixels: split over blocks
    (70, 24, 3, 3, 3),        # many samples
    (2, 256, 1, 40, 8),
    (3, 2048, 4, 5, 16),
    (1, 48, 211, 97, 2),
    (2, 32, 64, 64, 4),       # a tile of more than 64 KB of LDS
    (1, 4096, 50, 70, 4096),  # as many groups as there may be, split
]
IDS = ["x".join(map(str, s)) for s in SHAPES]


def oracle(x, groups, w, b, act, p=0.0, rng=None, gy=None, eps=1e-5):
    """The plain form in 64 bits on the CPU, and its gradients."""
    x = x.detach().cpu().double().requires_grad_(True)
    w, b = (t if t is None else t.detach().cpu().double().requires_grad_(True)
            for t in (w, b))
    y = ref.group_norm(x, groups, w, b, eps, act, p, rng)
    if gy is None:
        return y.detach()
    leaves = [t for t in (x, w, b) if t is not None]
    return (y.detach(),) + torch.autograd.grad(y, leaves, gy.cpu().double())


def magnitudes(x, groups, w, b, gy, scale, eps=1e-5):
    """Bounds of what takes part in y, dx, dw and db (64 bits)."""
    x = x.detach().cpu().double()
    n, c, h, wd = x.shape
    v = x.reshape(n, groups, -1)
    rstd = 1 / torch.sqrt(v.var(2, unbiased=False) + eps)
    hat = ((v.abs().amax(2) + v.mean(2).abs()) * rstd).max()
    wm = 1.0 if w is None else float(w.abs().max())
    bm = 0.0 if b is None else float(b.abs().max())
    y = scale * (wm * float(hat) + bm)
    if gy is None:
        return y
    g = scale * 1.2 * gy.cpu().double().abs()  # silu's slope is below 1.1
    dx = float(rstd.max()) * wm * float(g.max()) * (2 + float(hat)) ** 2
    db = float(g.sum((0, 2, 3)).max())
    return y, dx, db * (1 + float(hat)), db


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_group_norm_forward(shape, dtype):
    *dims, groups = shape
    x = features(dims, dtype, sum(shape))
    w, b = params(dims[1], 0)
    want = oracle(x, groups, w, b, "elu")
    got = ops.group_norm(x.to(DEV), groups, w.to(DEV), b.to(DEV), act="elu")
    assert got.dtype == dtype and got.is_contiguous(memory_format=LAST)
    assert_near(got, want, dtype, magnitudes(x, groups, w, b, None, 1.0))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_group_norm_backward(shape, dtype):
    *dims, groups = shape
    x = features(dims, dtype, sum(shape))
    w, b = params(dims[1], 0)
    gy = features(dims, dtype, 7 + sum(shape))
    y, dx, dw, db = oracle(x, groups, w, b, "silu", gy=gy)
    xs, ws, bs = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    got = ops.group_norm(xs, groups, ws, bs, act="silu")
    gx, gw, gb = torch.autograd.grad(got, (xs, ws, bs), gy.to(DEV))
    my, mx, mw, mb = magnitudes(x, groups, w, b, gy, 1.0)
    assert gx.dtype == dtype and gw.dtype == FP32 and gb.dtype == FP32
    assert_near(got, y, dtype, my)
    assert_near(gx, dx, dtype, mx)
    assert_near(gw, dw, FP32, mw)
    assert_near(gb, db, FP32, mb)


@pytest.mark.parametrize("act", [None, "elu", "leaky_relu", "relu", "silu"])
@pytest.mark.parametrize("shape", [(2, 24, 9, 7, 3), (1, 35, 4, 6, 7),
                                   (2, 64, 40, 33, 4)],
                         ids=["v8", "v1", "split"])
def test_group_norm_activations_and_dropout(act, shape):
    *dims, groups = shape
    rng = torch.tensor([123456789012345, 42])
    x = features(dims, FP32, 3)
    w, b = params(dims[1], 3)
    gy = features(dims, FP32, 4)
    y, dx, dw, db = oracle(x, groups, w, b, act, 0.3, rng, gy)
    z = oracle(x, groups, w, b, None)
    jump = act in ("relu", "leaky_relu")
    if jump:
        # where rounding may take z across the jump of the slope, the incoming
        # gradient is 0 on both sides
        gy = torch.where(z.abs() < CHAIN * 8, 0.0, gy.double()).float()
        gy = gy.contiguous(memory_format=LAST)
        y, dx, dw, db = oracle(x, groups, w, b, act, 0.3, rng, gy)
    xs, ws, bs = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    got = ops.group_norm(xs, groups, ws, bs, act=act, dropout=0.3,
                         rng=rng.to(DEV))
    gx, gw, gb = torch.autograd.grad(got, (xs, ws, bs), gy.to(DEV))
    my, mx, mw, mb = magnitudes(x, groups, w, b, gy, 1 / 0.7)
    assert_near(got, y, FP32, my)
    assert_near(gx, dx, FP32, mx)
    assert_near(gw, dw, FP32, mw)
    assert_near(gb, db, FP32, mb)
    if act is None:  # z is nowhere 0: zeros are what was dropped
        keep = ref.dropout_keep(x, 0.3, rng)
        assert torch.equal(got.detach().cpu() == 0, ~keep)


@pytest.mark.parametrize("have", ["weight", "bias", "neither"])
def test_group_norm_without_parameters(have):
    x = features((2, 16, 12, 10), FP32, 1)
    gy = features((2, 16, 12, 10), FP32, 2)
    w, b = params(16, 1)
    w, b = w if have == "weight" else None, b if have == "bias" else None
    want = oracle(x, 4, w, b, "elu", gy=gy)
    xs, ws, bs = (t if t is None else t.to(DEV).requires_grad_(True)
                  for t in (x, w, b))
    got = ops.group_norm(xs, 4, ws, bs, act="elu")
    leaves = [t for t in (xs, ws, bs) if t is not None]
    grads = torch.autograd.grad(got, leaves, gy.to(DEV))
    my, mx, mw, mb = magnitudes(x, 4, w, b, gy, 1.0)
    assert_near(got, want[0], FP32, my)
    for g, t in zip(grads, want[1:]):
        assert_near(g, t, FP32, max(mx, mw, mb))


def test_group_norm_parameters_at_any_address():
    x = features((2, 16, 12, 10), BF16, 1)
    w, b = params(16, 1)
    want = oracle(x, 4, w, b, None)
    both = torch.cat([torch.zeros(1), w, torch.zeros(2), b]).to(DEV)
    got = ops.group_norm(x.to(DEV), 4, both[1:17], both[19:35])
    assert_near(got, want, BF16, magnitudes(x, 4, w, b, None, 1.0))


@pytest.mark.parametrize("which", [0, 1, 2])
def test_group_norm_one_gradient_alone(which):
    x = features((3, 32, 20, 30), FP32, 5)
    gy = features((3, 32, 20, 30), FP32, 6)
    w, b = params(32, 5)
    want = oracle(x, 8, w, b, "elu", gy=gy)[1 + which]
    leaves = [t.to(DEV) for t in (x, w, b)]
    leaves[which].requires_grad_(True)
    y = ops.group_norm(leaves[0], 8, leaves[1], leaves[2], act="elu")
    g = torch.autograd.grad(y, leaves[which], gy.to(DEV))[0]
    assert_near(g, want, FP32, magnitudes(x, 8, w, b, gy, 1.0)[1 + which])


@pytest.mark.parametrize("which", [0, 1, 2])
def test_group_norm_one_gradient_alone_of_a_large_sample(which):
    x = features((1, 16, 130, 67), FP32, 5)
    gy = features((1, 16, 130, 67), FP32, 6)
    w, b = params(16, 5)
    want = oracle(x, 4, w, b, "elu", gy=gy)[1 + which]
    leaves = [t.to(DEV) for t in (x, w, b)]
    leaves[which].requires_grad_(True)
    y = ops.group_norm(leaves[0], 4, leaves[1], leaves[2], act="elu")
    g = torch.autograd.grad(y, leaves[which], gy.to(DEV))[0]
    assert_near(g, want, FP32, magnitudes(x, 4, w, b, gy, 1.0)[1 + which])


@pytest.mark.parametrize("hw", [(9, 8), (120, 130)], ids=["tile", "split"])
def test_group_norm_squares_beyond_fp32(hw):
    """Finite values whose squares are not: no result that looks like one."""
    x = features((1, 16) + hw, FP32, 60) * 1e25
    y = ops.group_norm(x.to(DEV), 4)
    assert not (torch.isfinite(y) & (y != 0)).any()


def test_many_samples_of_one_pixel():
    x = features((20000, 8, 1, 1), FP32, 61)
    gy = features((20000, 8, 1, 1), FP32, 62)
    w, b = params(8, 63)
    want = oracle(x, 2, w, b, "elu", gy=gy)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = ops.group_norm(leaves[0], 2, *leaves[1:], act="elu")
    got = (y,) + torch.autograd.grad(y, leaves, gy.to(DEV))
    for a, t, m in zip(got, want, magnitudes(x, 2, w, b, gy, 1.0)):
        assert_near(a, t, FP32, m)


def test_too_many_samples_are_refused():
    x = torch.empty(1, 8, 1, 1, device=DEV).expand(9_000_000, -1, -1, -1)
    with pytest.raises(RuntimeError, match="too large"):
        ops.group_norm(x, 2)


def test_group_norm_16_bit_parameters():
    x = features((2, 16, 5, 6), BF16, 1)
    gy = features((2, 16, 5, 6), BF16, 2)
    w, b = (t.bfloat16() for t in params(16, 1))
    _, dx, dw, db = oracle(x, 4, w, b, None, gy=gy)
    xs, ws, bs = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    y = ops.group_norm(xs, 4, ws, bs)
    gx, gw, gb = torch.autograd.grad(y, (xs, ws, bs), gy.to(DEV))
    assert gw.dtype == BF16 and gb.dtype == BF16
    _, mx, mw, mb = magnitudes(x, 4, w, b, gy, 1.0)
    assert_near(gx, dx, BF16, mx)
    assert_near(gw, dw, BF16, mw)
    assert_near(gb, db, BF16, mb)


@pytest.mark.parametrize("kind", ["nchw", "batch", "channels", "crop",
                                  "offset", "expanded"])
def test_group_norm_strides(kind):
    base = features((4, 48, 12, 15), BF16, 9).to(DEV)
    if kind == "nchw":
        x = base.contiguous()
    elif kind == "batch":
        x = base[::2]
    elif kind == "channels":
        x = base[:, 8:32]
    elif kind == "crop":
        x = base[..., 1:11, 2:14]
    elif kind == "expanded":
        x = base[:1].expand(4, -1, -1, -1)
    else:  # dense, at an address that is no multiple of a vector
        flat = torch.empty(base.numel() + 3, dtype=BF16, device=DEV)
        flat[3:] = base.permute(0, 2, 3, 1).reshape(-1)
        x = flat[3:].view(4, 12, 15, 48).permute(0, 3, 1, 2)
    c = x.shape[1]
    w, b = params(c, 2)
    gy = features(tuple(x.shape), BF16, 10)
    want = oracle(x, 8, w, b, "elu", gy=gy)
    xs = x.detach().requires_grad_(True)
    y = ops.group_norm(xs, 8, w.to(DEV), b.to(DEV), act="elu")
    g = torch.autograd.grad(y, xs, gy.to(DEV).contiguous())[0]
    my, mx, _, _ = magnitudes(x, 8, w, b, gy, 1.0)
    assert_near(y, want[0], BF16, my)
    assert_near(g, want[1], BF16, mx)


@pytest.mark.parametrize("shape", [(1, 16, 8, 8, 2), (2, 32, 150, 160, 4)],
                         ids=["small", "large"])
def test_group_norm_mean_far_from_zero(shape):
    """A mean of 1000 deviations: sums of squares about 0 would lose them."""
    *dims, groups = shape
    x = features(dims, FP32, 11, shift=0.0) + 1000
    want = oracle(x, groups, None, None, None)
    got = ops.group_norm(x.to(DEV), groups).cpu().double()
    # mean is rounded to fp32 once more: 1000 * 2^-24; the rest as everywhere
    assert float((got - want).abs().max()) < 1000 * 2**-23 + CHAIN * 20


@pytest.mark.parametrize("at", [0, 1, -1])
def test_group_norm_outlier(at):
    """One value far from all others, the first among them: a sum about the
    first value alone would leave nothing of the others' spread."""
    x = features((1, 8, 120, 130), FP32, 12, shift=0.0)
    x.permute(0, 2, 3, 1).reshape(-1, 8)[at] = 3e4
    want = oracle(x, 2, None, None, None)
    got = ops.group_norm(x.to(DEV), 2).cpu().double()
    assert_near(got, want, FP32, magnitudes(x, 2, None, None, None, 1.0))


def test_group_norm_constant_groups():
    x = torch.full((2, 16, 30, 20), 3.7).contiguous(memory_format=LAST)
    w, b = params(16, 4)
    xs = x.to(DEV).requires_grad_(True)
    y = ops.group_norm(xs, 4, w.to(DEV), b.to(DEV), act="relu")
    want = b.clamp(min=0).view(1, -1, 1, 1).expand_as(x)
    # the mean may be off by a step of 3.7, which rstd = 1 / sqrt(eps) widens
    assert float((y.cpu() - want).abs().max()) < 3.7 * 2**-23 / math.sqrt(1e-5) * 2
    g = torch.autograd.grad(y.sum(), xs)[0]
    assert torch.isfinite(g).all()


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_group_norm_keeps_what_is_not_finite_in_its_group(bad):
    x = features((2, 16, 40, 30), BF16, 13)
    clean = ops.group_norm(x.to(DEV), 4, act="elu").cpu()
    x[1, 5, 3, 3] = bad
    got = ops.group_norm(x.to(DEV), 4, act="elu").cpu()
    assert torch.equal(got[0], clean[0])
    others = [c for c in range(16) if c // 4 != 1]
    assert torch.equal(got[1, others], clean[1, others])
    assert torch.isnan(got[1, 4:8]).all()


def test_group_norm_is_the_same_every_time():
    x = features((3, 64, 60, 50), BF16, 14).to(DEV).requires_grad_(True)
    w, b = (t.to(DEV).requires_grad_(True) for t in params(64, 6))
    gy = features((3, 64, 60, 50), BF16, 15).to(DEV)

    def once():
        y = ops.group_norm(x, 32, w, b, act="elu", dropout=0.1, rng=(1, 2))
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), gy)

    first = once()
    for _ in range(3):
        for a, t in zip(once(), first):
            assert torch.equal(a, t)


@pytest.mark.parametrize("shape", [(8, 64, 6, 8), (4, 64, 120, 90)],
                         ids=["tile", "split"])
def test_group_norm_backward_again_and_again(shape):
    """One graph's backward several times, as a whole and in part, and from
    saved tensors that were moved to the host and back."""
    x = features(shape, BF16, 70).to(DEV).requires_grad_(True)
    w, b = (t.to(DEV).requires_grad_(True) for t in params(64, 71))
    gy = features(shape, BF16, 72).to(DEV)
    y = ops.group_norm(x, 8, w, b, act="silu", dropout=0.2, rng=(1, 2))
    want = torch.autograd.grad(y, (x, w, b), gy, retain_graph=True)
    for _ in range(3):
        got = torch.autograd.grad(y, (x, w, b), gy, retain_graph=True)
        for a, t in zip(got, want):
            assert torch.equal(a, t)
        assert torch.equal(
            torch.autograd.grad(y, w, gy, retain_graph=True)[0], want[1])
        assert torch.equal(
            torch.autograd.grad(y, x, gy, retain_graph=True)[0], want[0])
    with torch.autograd.graph.save_on_cpu():
        y = ops.group_norm(x, 8, w, b, act="silu", dropout=0.2, rng=(1, 2))
    for _ in range(2):
        got = torch.autograd.grad(y, (x, w, b), gy, retain_graph=True)
        for a, t in zip(got, want):
            assert torch.equal(a, t)


@pytest.mark.parametrize("shape", [(2, 32, 7, 9, 8), (2, 64, 90, 120, 16)])
def test_group_norm_one_tensor_as_weight_and_bias(shape):
    b, c, h, w, groups = shape
    x = features((b, c, h, w), BF16, 80).to(DEV).requires_grad_()
    gy = features((b, c, h, w), BF16, 81).to(DEV)
    both = params(c, 80)[0].to(DEV).requires_grad_()
    one, two = (both.detach().clone().requires_grad_() for _ in range(2))
    y = ops.group_norm(x, groups, both, both, act="silu")
    dx, d = torch.autograd.grad(y, (x, both), gy)
    y2 = ops.group_norm(x, groups, one, two, act="silu")
    dx2, d1, d2 = torch.autograd.grad(y2, (x, one, two), gy)
    assert torch.equal(y, y2) and torch.equal(dx, dx2)
    assert torch.equal(d, d1 + d2)


def test_group_norm_against_differences():
    x = features((2, 16, 9, 8), FP32, 16)
    w, b = params(16, 7)
    gy = features((2, 16, 9, 8), FP32, 17)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]

    def f(*t):
        return ops.group_norm(t[0], 4, t[1], t[2], act="silu", dropout=0.2,
                              rng=(5, 6))

    grads = torch.autograd.grad(f(*leaves), leaves, gy.to(DEV))
    h = 2.0**-7
    for i, g in enumerate(grads):
        v = torch.randn(g.shape, generator=torch.Generator().manual_seed(i))
        v = (v / v.norm()).to(DEV)
        up, down = list(leaves), list(leaves)
        up[i], down[i] = leaves[i] + h * v, leaves[i] - h * v
        with torch.no_grad():
            diff = ((f(*up) - f(*down)).double() * gy.to(DEV).double()).sum()
        got = (g.double() * v.double()).sum()
        # h^2 / 6 of a third derivative below 100 along a unit vector, and
        # values off by 2^-22 each over 2 h, 2304 of them at random signs
        norm = float(gy.norm())
        assert abs(float(diff) / (2 * h) - float(got)) < norm * (
            100 * h * h / 6 + 2.0**-22 * 2 / (2 * h))


def test_group_norm_empty():
    for shape in ((0, 8, 3, 3), (2, 8, 0, 3)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        w, b = (t.to(DEV).requires_grad_(True) for t in params(8, 1))
        y = ops.group_norm(x, 2, w, b, act="elu", dropout=0.5, rng=(1, 2))
        assert y.shape == shape
        gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
        assert gx.shape == shape
        assert not gw.any() and not gb.any()


def test_group_norm_refuses_a_second_derivative():
    x = features((1, 4, 3, 3), FP32, 1).to(DEV).requires_grad_(True)
    g = torch.autograd.grad(ops.group_norm(x, 2).square().sum(), x,
                            create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 8192, 8193, 100003])
def test_dropout_mask_and_values(n, dtype):
    rng = torch.tensor([2**62 + 12345, 2**40 + 3])
    g = torch.Generator().manual_seed(n)
    x = (torch.randn(n, generator=g).abs() + 0.5).to(dtype)  # nowhere 0
    for p in (0.1, 0.5, 2.0**-20 * 3, 1 - 2.0**-18 * 3):
        got = ops.dropout(x.to(DEV), p, rng.to(DEV)).cpu()
        keep = ref.dropout_keep(x, p, rng)
        assert torch.equal(got != 0, keep)
        want = torch.where(keep, x.double() / (1 - p), 0.0)
        if dtype != FP16 or p < 0.9:  # 1 / (1 - p) takes fp16 beyond its range
            assert_near(got, want, dtype, 0.0)


def test_dropout_of_any_64_bits():
    x = torch.ones(5000, device=DEV)
    for rng in ([-1, -1], [-2**63, 2**63 - 1], [0, 0], [5, -7]):
        rng = torch.tensor(rng)
        keep = ref.dropout_keep(x.cpu(), 0.3, rng)
        assert torch.equal((ops.dropout(x, 0.3, rng.to(DEV)) != 0).cpu(), keep)


def test_dropout_undecided_upper_halves():
    """p so placed that the upper 16 bits leave many elements undecided, and
    the lower ones decide: every one of 2^20 elements as the definition says."""
    n = 1 << 20
    rng = torch.tensor([77, 78])
    u = ref.dropout_numbers(n, rng)
    x = torch.ones(n, device=DEV)
    for quantile in (0.25, 0.5, 0.75):
        border = int(u.double().quantile(quantile))
        border = (border & ~0xFFFF) | 0x8000
        got = ops.dropout(x, border / 2**32, rng.to(DEV)).cpu()
        assert torch.equal(got != 0, u >= border)
        assert int(((u >> 16) == (border >> 16)).sum()) > 0


@pytest.mark.parametrize("act", [None, "elu", "leaky_relu", "relu", "silu"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_dropout_activation_and_gradient(act, dtype):
    rng = torch.tensor([9, 8])
    g = torch.Generator().manual_seed(1)
    x = torch.randn(37, 41, generator=g).to(dtype)
    x.view(-1)[:3] = torch.tensor([0.0, -30.0, 30.0])
    gy = torch.randn(37, 41, generator=g).to(dtype)
    xd = x.double().requires_grad_(True)
    want = ref.dropout(xd, 0.3, rng, act)
    dwant = torch.autograd.grad(want, xd, gy.double())[0]
    xs = x.to(DEV).requires_grad_(True)
    y = ops.dropout(xs, 0.3, rng.to(DEV), act=act)
    dx = torch.autograd.grad(y, xs, gy.to(DEV))[0]
    # pointwise: no sums, all magnitudes are the values' own, except that
    # silu' = t (1 + z (1 - t)) may cancel to less than its terms
    tiny = 1.0 if act in ("elu", "silu") else 0.0
    assert_near(y, want.detach(), dtype, tiny)
    assert_near(dx, dwant, dtype, tiny * float(gy.abs().max()) * 2)


@pytest.mark.parametrize("kind", ["last", "transposed", "offset", "scalar",
                                  "five", "expanded"])
def test_dropout_strides(kind):
    rng = (5, 7)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(4, 10, 6, 9, generator=g)
    if kind == "last":
        x = x.contiguous(memory_format=LAST)
    elif kind == "transposed":
        x = x.transpose(1, 3)
    elif kind == "offset":
        x = x.flatten()[1:]
    elif kind == "scalar":
        x = x[0, 0, 0, 0]
    elif kind == "five":
        x = x.unsqueeze(2)
    else:
        x = x[:1].expand(3, -1, -1, -1)
    want = ops.dropout(x, 0.4, rng, act="elu")
    xs = x.to(DEV)
    if kind == "transposed":
        xs = x.transpose(1, 3).to(DEV).transpose(1, 3)
    elif kind == "offset":
        buf = torch.empty(x.numel() + 1, device=DEV)
        buf[1:] = x.to(DEV)
        xs = buf[1:]
    xs = xs.detach().requires_grad_(True)
    got = ops.dropout(xs, 0.4, rng, act="elu")
    assert got.shape == x.shape
    assert torch.equal(got.cpu() != 0, want != 0)
    assert_near(got, want.double(), FP32, 1.0)
    grad = torch.autograd.grad(got.sum(), xs)[0]
    assert torch.equal((grad != 0).cpu(), want != 0)


@pytest.mark.parametrize("shape", [(3, 5, 1, 1), (3, 1, 4, 5)])
def test_dropout_layouts_of_single_extents(shape):
    """Shapes that are contiguous and channels last at once."""
    for fmt in (LAST, torch.contiguous_format):
        x = torch.randn(shape).contiguous(memory_format=fmt)
        xs = x.to(DEV).requires_grad_(True)
        y = ops.dropout(xs, 0.5, (1, 1), act="elu")
        want = ops.dropout(x, 0.5, (1, 1), act="elu")
        assert torch.equal(y.cpu() != 0, want != 0)
        for gfmt in (LAST, torch.contiguous_format):
            gy = torch.ones(shape, device=DEV).contiguous(memory_format=gfmt)
            g = torch.autograd.grad(y, xs, gy, retain_graph=True)[0]
            assert torch.equal((g != 0).cpu(), want != 0)


def test_dropped_places_leave_no_trace():
    keep = ref.dropout_keep(torch.empty(64), 0.5, torch.tensor([1, 2]))
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = torch.ones(64)
        x[~keep] = bad
        xs = x.to(DEV).requires_grad_(True)
        for act in (None, "elu", "silu"):
            y = ops.dropout(xs, 0.5, (1, 2), act=act)
            assert torch.isfinite(y).all() and not y[~keep.to(DEV)].any()
            gy = torch.where(keep, 1.0, bad).to(DEV)
            g = torch.autograd.grad(y, xs, gy)[0]
            assert torch.isfinite(g).all() and not g[~keep.to(DEV)].any()


def test_dropout_all_none_and_empty():
    x = torch.randn(100, device=DEV, requires_grad=True)
    y = ops.dropout(x, 1.0)
    assert not y.any() and not torch.autograd.grad(y.sum(), x)[0].any()
    assert torch.equal(ops.dropout(x, 0.0), x)
    e = torch.empty(0, 4, device=DEV, requires_grad=True)
    assert torch.autograd.grad(ops.dropout(e, 0.5).sum(), e)[0].shape == (0, 4)


# ---------------------------------------------------------------------------
# streams, graphs, sizes, refusals
# ---------------------------------------------------------------------------
def _block(x, w, b, rng=None):
    y = ops.group_norm(x, 8, w, b, act="elu", dropout=0.2, rng=rng)
    return ops.dropout(y, 0.3, rng, act="silu")


def test_on_another_stream():
    x = features((2, 64, 40, 30), BF16, 18).to(DEV).requires_grad_(True)
    w, b = (t.to(DEV).requires_grad_(True) for t in params(64, 8))
    want = torch.autograd.grad(_block(x, w, b, (3, 4)).sum(), (x, w, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = _block(x, w, b, (3, 4))
        got = torch.autograd.grad(y.sum(), (x, w, b))
    torch.cuda.current_stream().wait_stream(side)
    for a, t in zip(got, want):
        assert torch.equal(a, t)


@pytest.mark.parametrize("shape", [(2, 64, 6, 8), (2, 64, 60, 50),
                                   (1, 64, 64, 64), (2, 64, 120, 90)],
                         ids=["small", "large", "lds", "split"])
def test_graph_replays(shape):
    """Forward and backward captured; replays between eager work give what the
    eager calls give for the rng that the graph reads."""
    x = features(shape, BF16, 19).to(DEV)
    w, b = (t.to(DEV) for t in params(64, 9))
    rng = torch.tensor([1, 0], device=DEV)

    def step(x, rng):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = _block(*leaves, rng)
        return (y.detach(),) + torch.autograd.grad(y, leaves, torch.ones_like(y))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, rng)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, rng)
    for i in range(4):
        x.copy_(features(shape, BF16, 20 + i))
        rng.fill_(100 + i)
        want = [t.clone() for t in step(x, rng.clone())]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, t in zip(out, want):
            assert torch.equal(a, t)


def test_two_threads_at_once():
    """Calls of two host threads on streams of their own give what they give
    one after the other."""
    cases = [(4, 64, 24, 32, 16), (2, 64, 160, 200, 32)]
    data = []
    for k, (b, c, h, w, groups) in enumerate(cases):
        data.append((groups, features((b, c, h, w), BF16, 90 + k).to(DEV),
                     *(t.to(DEV) for t in params(c, 90 + k)),
                     features((b, c, h, w), BF16, 95 + k).to(DEV)))

    def calls(k):
        groups, x, weight, bias, gy = data[k]
        leaves = [t.detach().requires_grad_() for t in (x, weight, bias)]
        y = ops.group_norm(leaves[0], groups, *leaves[1:], act="elu",
                           dropout=0.3, rng=(7, k))
        z = ops.dropout(y, 0.2, rng=(8, k), act="relu")
        return [y.detach(), z.detach(), *torch.autograd.grad(z, leaves, gy)]

    want = [calls(k) for k in range(2)]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream(DEV)):
                for i in range(20):
                    got = calls(k)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(g, e)
                               for g, e in zip(got, want[k])):
                        wrong.append((k, i))
        except Exception as e:  # a thread's error would be lost
            wrong.append((k, repr(e)))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("shape", [(4, 64, 24, 32, 16), (2, 64, 160, 200, 32)])
def test_two_graphs_of_one_backward(shape):
    """Backwards of one call, recorded twice and replayed side by side with
    eager ones, share no counter."""
    b, c, h, w, groups = shape
    side = [torch.cuda.Stream(DEV) for _ in range(3)]
    x = features((b, c, h, w), BF16, 70).to(DEV).requires_grad_()
    weight, bias = (t.to(DEV).requires_grad_() for t in params(c, 70))
    leaves = (x, weight, bias)
    gys = [features((b, c, h, w), BF16, 71 + i).to(DEV) for i in range(3)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    with torch.cuda.stream(side[0]):
        y = ops.group_norm(x, groups, weight, bias, act="elu")
        want = [torch.autograd.grad(y, leaves, gy, retain_graph=True)
                for gy in gys]
    torch.cuda.synchronize()
    for gy in gys[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side[0]):
            outs.append(torch.autograd.grad(y, leaves, gy, retain_graph=True))
        graphs.append(g)
    for _ in range(20):
        for out in outs:
            for t in out:
                t.fill_(7.0)
        torch.cuda.synchronize()
        for g, s in zip(graphs, side[1:]):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(side[0]):
            eager = torch.autograd.grad(y, leaves, gys[2], retain_graph=True)
        torch.cuda.synchronize()
        for got, exact in zip([*outs, eager], want):
            assert all(torch.equal(a, e) for a, e in zip(got, exact))


def test_graph_draws_anew_at_every_replay():
    x = torch.ones(4096, device=DEV)
    ops.dropout(x, 0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.dropout(x, 0.5)
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        seen.append(y.clone())
        rate = float((y != 0).float().mean())
        assert abs(rate - 0.5) < 6 * 0.5 / 64
    assert not torch.equal(seen[0], seen[1])
    assert not torch.equal(seen[1], seen[2])


def test_graph_draws_differ_between_captures_of_one_program():
    """Two graphs in flight share no workspace."""
    xs = [features((2, 64, 60, 50), BF16, 30 + i).to(DEV) for i in range(2)]
    ops.group_norm(xs[0], 8)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.group_norm(x, 8, act="elu"))
        graphs.append(g)
    want = [ops.group_norm(x, 8, act="elu") for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, t in zip(outs, want):
            assert torch.equal(o, t)


def test_recomputation_draws_the_same_mask():
    from torch.utils.checkpoint import checkpoint

    x = features((2, 64, 20, 20), BF16, 31).to(DEV).requires_grad_(True)
    w, b = (t.to(DEV).requires_grad_(True) for t in params(64, 10))
    torch.manual_seed(3)
    want = torch.autograd.grad(_block(x, w, b).float().square().sum(), (x, w, b))
    torch.manual_seed(3)
    y = checkpoint(_block, x, w, b, use_reentrant=False)
    got = torch.autograd.grad(y.float().square().sum(), (x, w, b))
    for a, t in zip(got, want):
        assert torch.equal(a, t)


def test_more_than_32_bits_of_elements():
    """Elements behind 2^31 and 2^32 bytes: the last sample on its own."""
    b, c, h, w = 3, 64, 3400, 3400  # 2.2e9 elements
    rng = torch.tensor([5, 6], device=DEV)
    x = torch.empty(b, h, w, c, dtype=BF16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    for i in range(b):
        x[i].normal_(generator=g)
    x = x.permute(0, 3, 1, 2)
    assert x.numel() > 2**31
    y = ops.group_norm(x, 8, act="elu")
    last = ops.group_norm(x[-1:].clone(memory_format=LAST), 8, act="elu")
    # the sample alone is split otherwise: one rounding to bf16 apart at most
    d = (y[-1:].float() - last.float()).abs()
    assert float((d - 2.0**-7 * last.float().abs()).max()) <= 2.0**-20
    del d, last
    z = ops.dropout(y, 0.5, rng)
    n, tail = x.numel(), 4096
    at = n // 8 * 8 - tail
    j = torch.arange(at // 8, n // 8)
    words = ref.philox4x32(
        (j & 0xFFFFFFFF, j >> 32, torch.tensor(6), torch.tensor(0)),
        (torch.tensor(5), torch.tensor(0)))
    half = torch.stack([t >> s & 0xFFFF for t in words for s in (0, 16)], 1)
    keep = half.reshape(-1) >= 0x8000
    flat = z.permute(0, 2, 3, 1).reshape(-1)[at:at + tail].cpu()
    source = y.permute(0, 2, 3, 1).reshape(-1)[at:at + tail].cpu()
    assert torch.equal(flat, torch.where(keep, source.float() * 2, 0.0).bfloat16())


@pytest.mark.parametrize("error,call", cpu_refusals.pytestmark[0].args[1])
def test_refusals(error, call):
    with pytest.raises(error):
        call(DEV)


def test_refuses_tensors_of_other_devices():
    x = features((1, 8, 3, 3), FP32, 1)
    with pytest.raises(ValueError):
        ops.group_norm(x.to(DEV), 2, torch.ones(8))
    with pytest.raises(ValueError):
        ops.group_norm(x, 2, torch.ones(8, device=DEV))
    with pytest.raises(ValueError):
        ops.dropout(x.to(DEV), 0.5, torch.tensor([1, 2]))
    with pytest.raises(TypeError):
        ops.dropout(x.to(DEV).double(), 0.5)


# ---------------------------------------------------------------------------
# together, as models use them
# ---------------------------------------------------------------------------
def test_block_as_models_build_it():
    """conv -> norm + act + dropout -> conv -> act + dropout: the GPU's kernels
    against the plain forms in 64 bits, the same masks on both sides."""
    import torch.nn.functional as F

    g = torch.Generator().manual_seed(50)
    x = features((2, 8, 14, 18), FP32, 51)
    w1, w2 = (torch.randn(16, c, 3, 3, generator=g) * 0.1 for c in (8, 16))
    gamma, beta = params(16, 52)
    gy = features((2, 16, 14, 18), FP32, 53)

    def block(x, w1, w2, gamma, beta, norm, drop):
        y = F.conv2d(x, w1, padding=1)
        y = norm(y, 4, gamma, beta, act="elu", dropout=0.2, rng=(1, 2))
        y = F.conv2d(y, w2, padding=1).contiguous(memory_format=LAST)
        return drop(y, 0.3, (3, 4), act="silu")

    leaves = [t.double().requires_grad_(True)
              for t in (x, w1, w2, gamma, beta)]
    want = block(*leaves, ops.group_norm, ops.dropout)  # CPU, 64 bits
    dwant = torch.autograd.grad(want, leaves, gy.double())
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w1, w2, gamma, beta)]
    got = block(*leaves, ops.group_norm, ops.dropout)
    dgot = torch.autograd.grad(got, leaves, gy.to(DEV))
    # chains of two convolutions (72 and 144 terms) and a norm: 2^12 steps of
    # fp32 relative to the largest value bound them
    for a, t in zip((got,) + dgot, (want.detach(),) + dwant):
        bound = 2.0**12 * 2.0**-24 * float(t.abs().max())
        assert float((a.detach().cpu().double() - t).abs().max()) < bound


@pytest.mark.parametrize("name", ["flownets", "inception_v3"])
def test_model_step_with_group_norm(name):
    from deepof_amd.models import build_model

    torch.manual_seed(0)
    model, _, _ = build_model(name, norm="group", feature_dropout=0.1)
    model.to(DEV).to(memory_format=LAST)
    x = torch.randn(2, 6, 128, 128, device=DEV).contiguous(memory_format=LAST)
    with torch.autocast("cuda", dtype=BF16):
        flows = model(x)
    sum(f.float().square().mean() for f in flows).backward()
    for n, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), n
    norms = [m for m in model.modules() if isinstance(m, ops.GroupNormAct)]
    assert all(float(m.weight.grad.abs().sum()) > 0 for m in norms)
