"""Group norm's sums where they are long: many values per thread, outliers in
front of them, many samples.  Against sums in 64 bits.

Tolerances are those of the other group norm tests: half a step of what is
stored, and 256 steps of 2^-24 of the largest magnitude in the chain.  Sums
keep to that at any length because none is one chain: a thread's values are
added up in runs of at most 64, which are joined, below 64 + 8192 / 64 additions
at the sizes here, 40 more over a block and over blocks, and 64 where shares of
the samples meet; a share's own sum carries along what its roundings lose.
"""

import pytest
import torch

from deepof_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
LAST = torch.channels_last
CHAIN = 256 * 2.0**-24


def assert_close(got, want, magnitude):
    assert not torch.isnan(got).any()
    half = torch.finfo(got.dtype).eps / 2
    off = (got.double() - want).abs() - (
        half * want.abs() + CHAIN * (magnitude + want.abs()))
    assert float(off.max()) <= 0, f"over the bound by {float(off.max()):.3g}"


def normalise(x, groups, eps=1e-5):
    """Group norm in 64 bits where x is, and the largest |xhat|."""
    b, c, h, w = x.shape
    v = x.double().permute(0, 2, 3, 1).reshape(b, h * w, groups, c // groups)
    mean = v.mean((1, 3), keepdim=True)
    v = v - mean
    rstd = 1 / torch.sqrt(v.square().mean((1, 3), keepdim=True) + eps)
    v = v * rstd
    largest = float(v.abs().max() + (mean.abs() * rstd).max())
    return v.reshape(b, h, w, c).permute(0, 3, 1, 2), largest


LONG = [  # b, c, h, w, groups
    (1, 1, 120, 150, 1),       # a tile, 36 values a thread
    (1, 33, 1500, 2000, 3),    # single channels are moved, 782 values
    (1, 36, 1500, 2000, 4),    # 4 at a time, 209
    (1, 64, 1800, 2900, 2),    # 8 at a time, 319
    (600, 16, 512, 160, 2),    # a block per sample, 320
]


@pytest.mark.parametrize("kind", ["pixel", "rows", "pixel of zeros"])
@pytest.mark.parametrize("shape", LONG, ids=["x".join(map(str, s)) for s in LONG])
def test_statistics_behind_outliers(shape, kind):
    """The first values that threads meet lie far from all others: sums about
    them are of nearly equal numbers, and round the same way again and again."""
    b, c, h, w, groups = shape
    g = torch.Generator(device=DEV).manual_seed(c)
    x = torch.empty(b, h, w, c, device=DEV)
    for i in range(b):
        x[i].normal_(generator=g)
    x = x.permute(0, 3, 1, 2)
    if kind == "pixel":
        x[:, :, 0, 0] = 3e4
    elif kind == "rows":  # bright rows above darkness
        rows = max(1, 20000 // w)
        x[:, :, rows:] = 0.0
        x[:, :, :rows] += 30
    else:
        x.zero_()
        x[:, :, 0, 0] = 17.3
    step = max(1, 200_000_000 // (c * h * w))  # samples compared at once
    y = ops.group_norm(x, groups)
    for i in range(0, b, step):
        want, largest = normalise(x[i:i + step], groups)
        assert_close(y[i:i + step], want, largest)


def test_gradient_sums_of_many_values():
    """8192 values a thread.  What a mean hands back is the same everywhere."""
    b, c, h, w = 1, 511, 1448, 1448
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.empty(b, h, w, c, device=DEV)
    x.normal_(generator=g)
    x = x.permute(0, 3, 1, 2)
    bias = torch.zeros(c, device=DEV, requires_grad=True)
    gy = torch.full_like(x, 0.1)
    y = ops.group_norm(x, 7, None, bias)
    db = torch.autograd.grad(y, bias, gy)[0]
    want = torch.full((c,), float(gy[0, 0, 0, 0].double()) * h * w,
                      device=DEV, dtype=torch.float64)
    assert_close(db, want, float(want[0]))


@pytest.mark.parametrize("shape", [(100_000, 512, 1, 1, 32),
                                   (4096, 8, 3, 3, 2), (2048, 515, 2, 2, 5)])
def test_parameter_gradients_over_many_samples(shape):
    b, c, h, w, groups = shape
    g = torch.Generator(device=DEV).manual_seed(6)
    x = torch.randn(b, h, w, c, device=DEV, generator=g).permute(0, 3, 1, 2)
    weight = torch.ones(c, device=DEV, requires_grad=True)
    bias = torch.zeros(c, device=DEV, requires_grad=True)
    gy = torch.full_like(x, 0.1)
    y = ops.group_norm(x, groups, weight, bias)
    dw, db = torch.autograd.grad(y, (weight, bias), gy)
    step = float(gy[0, 0, 0, 0].double())
    n = b * h * w
    want = torch.full((c,), step * n, device=DEV, dtype=torch.float64)
    assert_close(db, want, step * n)
    xhat, largest = normalise(x, groups)
    assert_close(dw, step * xhat.sum((0, 2, 3)), step * n * (1 + largest))


@pytest.mark.parametrize("shape", [
    (1, 33, 1500, 2000, 3), (1, 36, 1500, 2000, 4), (1, 64, 1800, 2900, 2),
    (1, 4096, 132, 131, 4096),  # as much of LDS as there may be
], ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_long_threads(shape):
    b, c, h, w, groups = shape
    g = torch.Generator(device=DEV).manual_seed(7)
    x, gy = (torch.randn(b, h, w, c, device=DEV, generator=g)
             .permute(0, 3, 1, 2) for _ in range(2))
    weight = 1 + 0.3 * torch.randn(c, device=DEV, generator=g)
    leaves = [t.requires_grad_() for t in
              (x, weight, torch.zeros(c, device=DEV))]
    y = ops.group_norm(x, groups, *leaves[1:])
    dx, dw, db = torch.autograd.grad(y, leaves, gy)
    del y
    x, weight = x.detach(), weight.detach()
    xhat, largest = normalise(x, groups)
    gz = gy.double()
    total = float(gz.abs().sum((0, 2, 3)).max())
    assert_close(db, gz.sum((0, 2, 3)), total)
    assert_close(dw, (gz * xhat).sum((0, 2, 3)), total * (1 + largest))
    gz *= weight.double().view(1, -1, 1, 1)
    top = float(gz.abs().max())

    def over_groups(t):  # the mean of each value's group
        v = t.reshape(b, groups, -1).mean(2)
        return v.repeat_interleave(c // groups, 1).view(b, c, 1, 1)

    var = over_groups((x.double() - over_groups(x.double())).square())
    rstd = 1 / torch.sqrt(var + 1e-5)
    want = rstd * (gz - over_groups(gz) - xhat * over_groups(gz * xhat))
    assert_close(dx, want, float(rstd.max()) * top * (2 + largest) ** 2)


def test_statistics_behind_2_31_elements():
    """The last sample, whose every element lies behind 2^31: 1056 values a
    thread, against sums in 64 bits."""
    b, c, h, w, groups = 3, 64, 3400, 3400, 8
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.empty(b, h, w, c, dtype=torch.bfloat16, device=DEV)
    for i in range(b):
        x[i].normal_(generator=g)
    x = x.permute(0, 3, 1, 2)
    assert x.numel() > 2**31
    y = ops.group_norm(x, groups)
    for group in (0, groups - 1):
        at = slice(group * c // groups, (group + 1) * c // groups)
        want, largest = normalise(x[-1:, at], 1)
        assert_close(y[-1:, at], want, largest)


@pytest.mark.parametrize("shape", [
    (2048, 515, 2, 2, 5),     # parameters' gradients by a launch of their own
    (2, 64, 700, 800, 8),     # totals in LDS
], ids=lambda s: "x".join(map(str, s)))
def test_replays_of_long_sums(shape):
    b, c, h, w, groups = shape
    g = torch.Generator(device=DEV).manual_seed(8)
    x, gy = (torch.randn(b, h, w, c, device=DEV, generator=g).bfloat16()
             .permute(0, 3, 1, 2) for _ in range(2))
    weight, bias = (torch.randn(c, device=DEV, generator=g) for _ in range(2))

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, weight, bias)]
        y = ops.group_norm(leaves[0], groups, *leaves[1:], act="silu")
        return [y.detach(), *torch.autograd.grad(y, leaves, gy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        x.normal_(generator=g)
        gy.normal_(generator=g)
        want = step()
        for t in out:
            t.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(out, want):
            assert torch.equal(a, e)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("at", [0, 5 * 800 + 3, -1], ids=["first", "amid", "last"])
def test_what_is_not_finite_stays_in_its_group(bad, at):
    """Wherever among a thread's runs it comes."""
    x = torch.randn(600, 800, 16, device=DEV)
    x = x.permute(2, 0, 1).unsqueeze(0)
    clean = ops.group_norm(x, 4)
    x.permute(0, 2, 3, 1).view(-1, 16)[at, 5] = bad
    y = ops.group_norm(x, 4)
    assert torch.isnan(y[:, 4:8]).all()
    assert torch.equal(y[:, :4], clean[:, :4])
    assert torch.equal(y[:, 8:], clean[:, 8:])
