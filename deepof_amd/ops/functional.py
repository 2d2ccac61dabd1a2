"""Device-dispatching functional ops.

On GPU (torch "cuda" == ROCm/HIP here) every op runs the hand-written
CDNA4 HIP kernel from deepof_amd.ops.hip — and FAILS LOUDLY if the
extension is not built (no silent eager fallback on a GPU box).  On CPU
the pure-torch reference implementations run instead, so the same model
code is testable without a GPU.
"""

from __future__ import annotations

import torch

from . import reference as ref

_HIP = None
_HIP_ERR: str | None = None


def _load_hip():
    global _HIP, _HIP_ERR
    if _HIP is not None or _HIP_ERR is not None:
        return _HIP
    try:
        from .hip import _deepof_hip  # built in-tree by setup.py / __graft_entry__

        _HIP = _deepof_hip
    except ImportError as e:  # pragma: no cover - exercised on GPU boxes only
        _HIP_ERR = str(e)
    return _HIP


def hip_available() -> bool:
    return _load_hip() is not None


def require_hip():
    m = _load_hip()
    if m is None:
        raise RuntimeError(
            "deepof_amd HIP extension is not built but a GPU tensor reached a "
            "deepof_amd op. Build it in-tree first: `python setup.py "
            f"build_ext --inplace` (import error: {_HIP_ERR})"
        )
    return m


def _on_gpu(*tensors) -> bool:
    return any(t.is_cuda for t in tensors if isinstance(t, torch.Tensor))


# ---------------------------------------------------------------------------
# warp
# ---------------------------------------------------------------------------
class _WarpBilinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, img2, flow):
        hip = require_hip()
        recon = hip.warp_forward(img2.contiguous(), flow.contiguous())
        ctx.save_for_backward(img2, flow)
        return recon

    @staticmethod
    def backward(ctx, grad_out):
        img2, flow = ctx.saved_tensors
        hip = require_hip()
        gimg2, gflow = hip.warp_backward(
            grad_out.contiguous(), img2.contiguous(), flow.contiguous()
        )
        return gimg2, gflow


def warp_bilinear(img2: torch.Tensor, flow: torch.Tensor) -> torch.Tensor:
    """Backward-warp img2 ([B,C,H,W]) by pixel-scaled flow ([B,2,H,W])."""
    if _on_gpu(img2, flow):
        return _WarpBilinear.apply(img2, flow.float())
    return ref.warp_bilinear(img2, flow)


# ---------------------------------------------------------------------------
# resize / lrn (loss-branch image preprocessing; inputs are constants)
# ---------------------------------------------------------------------------
def resize_bilinear(x: torch.Tensor, out_h: int, out_w: int) -> torch.Tensor:
    if x.is_cuda:
        if x.requires_grad and torch.is_grad_enabled():
            # differentiable path (same legacy-TF sampling, torch ops);
            # the HIP kernel serves the no-grad image-pyramid hot path
            return ref.resize_bilinear(x, out_h, out_w)
        return require_hip().resize_bilinear(x.contiguous(), out_h, out_w)
    return ref.resize_bilinear(x, out_h, out_w)


def lrn(x, depth_radius: int = 4, bias: float = 1.0, alpha: float = 1.0,
        beta: float = 0.7) -> torch.Tensor:
    if x.is_cuda:
        if x.requires_grad and torch.is_grad_enabled():
            # differentiable torch-op path (a future loss backprops
            # through the image branch); the HIP kernel serves the
            # no-grad image-pyramid hot path
            return ref.lrn(x, depth_radius, bias, alpha, beta)
        return require_hip().lrn_forward(x.contiguous(), depth_radius, bias, alpha, beta)
    return ref.lrn(x, depth_radius, bias, alpha, beta)


# ---------------------------------------------------------------------------
# correlation (FlowNetC)
# ---------------------------------------------------------------------------
class _Correlation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, f1, f2, md):
        hip = require_hip()
        out = hip.correlation_forward(f1.contiguous(), f2.contiguous(), md)
        ctx.save_for_backward(f1, f2)
        ctx.md = md
        return out

    @staticmethod
    def backward(ctx, grad_out):
        f1, f2 = ctx.saved_tensors
        hip = require_hip()
        gf1, gf2 = hip.correlation_backward(
            grad_out.contiguous(), f1.contiguous(), f2.contiguous(), ctx.md
        )
        return gf1, gf2, None


def correlation(f1: torch.Tensor, f2: torch.Tensor, max_displacement: int = 10):
    """FlowNetC cost volume, (2*md+1)^2 channels, zero-padded, /C."""
    if _on_gpu(f1, f2):
        return _Correlation.apply(f1, f2, max_displacement)
    return ref.correlation(f1, f2, max_displacement)


# ---------------------------------------------------------------------------
# fused per-scale unsupervised loss
# ---------------------------------------------------------------------------
class _FusedUnsupLoss(torch.autograd.Function):
    """HIP fused warp + Charbonnier photometric + smoothness for one scale.

    Forward returns raw SUMS (photo_sum, u_sum, v_sum) and the recon
    image; normalization and the lambda-weighted total happen in Python.
    Backward produces d(flow_raw) only — images are data, not params.
    """

    @staticmethod
    def forward(ctx, flow_raw, img1, img2, flow_scale, eps, alpha_c, alpha_s,
                want_recon):
        hip = require_hip()
        photo_sum, u_sum, v_sum, recon = hip.unsup_loss_forward(
            flow_raw.contiguous(), img1.contiguous(), img2.contiguous(),
            flow_scale, eps, alpha_c, alpha_s, want_recon,
        )
        ctx.save_for_backward(flow_raw, img1, img2)
        ctx.params = (flow_scale, eps, alpha_c, alpha_s)
        return photo_sum, u_sum, v_sum, recon

    @staticmethod
    def backward(ctx, g_photo, g_u, g_v, g_recon):
        flow_raw, img1, img2 = ctx.saved_tensors
        flow_scale, eps, alpha_c, alpha_s = ctx.params
        hip = require_hip()
        # upstream grads stay on device (no .item() sync; hipGraph-safe)
        dev = flow_raw.device
        def _g(t):
            return (t.float().reshape(1) if isinstance(t, torch.Tensor)
                    else torch.zeros(1, device=dev))
        gs = torch.cat([_g(g_photo), _g(g_u), _g(g_v)])
        gflow = hip.unsup_loss_backward(
            flow_raw.contiguous(), img1.contiguous(), img2.contiguous(),
            flow_scale, eps, alpha_c, alpha_s, gs,
        )
        return gflow, None, None, None, None, None, None, None


def unsup_loss_scale(
    flow_raw: torch.Tensor,
    img1: torch.Tensor,
    img2: torch.Tensor,
    flow_scale: float,
    epsilon: float = 1e-4,
    alpha_c: float = 0.25,
    alpha_s: float = 0.37,
    lambda_smooth: float = 1.0,
    return_recon: bool = False,
):
    """One pyramid scale of the unsupervised warp loss (see
    deepof_amd.ops.reference.unsup_loss_scale for the semantics spec)."""
    if not _on_gpu(flow_raw, img1, img2):
        return ref.unsup_loss_scale(
            flow_raw, img1, img2, flow_scale, epsilon, alpha_c, alpha_s,
            lambda_smooth, return_recon,
        )
    b, c, h, w = img1.shape
    import math

    # mirror the kernel's border-mask fallback for degenerate scales
    bw = math.ceil(h * 0.1)
    if (h - 2 * bw) > 0 and (w - 2 * bw) > 0:
        num_valid = float(b * c * (h - 2 * bw) * (w - 2 * bw))
        num_valid_flows = num_valid / c * 2
    else:
        num_valid = float(b * c * h * w)
        num_valid_flows = float(2 * b * h * w)
    photo_sum, u_sum, v_sum, recon = _FusedUnsupLoss.apply(
        flow_raw.float(), img1, img2, flow_scale, epsilon, alpha_c, alpha_s,
        return_recon,
    )
    photo = photo_sum / num_valid
    u_loss = u_sum / num_valid_flows
    v_loss = v_sum / num_valid_flows
    total = photo + lambda_smooth * (u_loss + v_loss)
    out = {"total": total, "photo": photo, "u_loss": u_loss, "v_loss": v_loss}
    if return_recon:
        out["recon"] = recon
    return out


# ---------------------------------------------------------------------------
# EPE reduction (eval)
# ---------------------------------------------------------------------------
def endpoint_error_sum(flow: torch.Tensor, flow_gt: torch.Tensor) -> torch.Tensor:
    """Sum over all pixels of sqrt(du^2+dv^2); divide by B*H*W for AEE."""
    if _on_gpu(flow, flow_gt):
        return require_hip().epe_sum(flow.contiguous().float(),
                                     flow_gt.contiguous().float())
    d = (flow.float() - flow_gt.float())
    return torch.sqrt(d[:, 0] ** 2 + d[:, 1] ** 2).sum()


# ---------------------------------------------------------------------------
# dropout from a counter-based generator; group norm + activation + dropout
# ---------------------------------------------------------------------------
_ACT_CODES = {None: 0, "none": 0, "elu": 1, "leaky_relu": 2, "relu": 3,
              "silu": 4}
_MAX_GROUPS = 4096  # the kernels hold a sample's group statistics in LDS


def draw_rng(device, generator: torch.Generator | None = None) -> torch.Tensor:
    """A fresh (seed, offset) for `dropout` and `group_norm`: two int64 drawn
    from torch's generator of `device`, and left there.

    Follows torch.manual_seed, a saved and restored generator state
    (activation recomputation) and graph capture: every replay draws anew.
    """
    return torch.randint(0, 2**63 - 1, (2,), device=device,
                         generator=generator)


def _act_code(act) -> int:
    try:
        return _ACT_CODES[act]
    except (KeyError, TypeError):
        raise ValueError(f"unknown activation {act!r}") from None


def _check_float(x, name):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name}: a tensor expected, got {type(x).__name__}")
    allowed = (torch.float64, torch.float32, torch.float16, torch.bfloat16)
    if x.dtype not in allowed:
        raise TypeError(f"{name}: a floating tensor expected, got {x.dtype}")


def _check_dropout(p, rng, x):
    """-> (p, rng tensor or None, seed, offset)"""
    if isinstance(p, bool) or not isinstance(p, (int, float)):
        raise TypeError(f"dropout probability: a number expected, got {p!r}")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must lie in [0, 1], got {p}")
    if p == 0.0:
        return p, None, 0, 0
    if rng is None:
        return p, draw_rng(x.device), 0, 0
    if isinstance(rng, torch.Tensor):
        if rng.dtype != torch.int64 or rng.shape != (2,):
            raise ValueError("rng: an int64 tensor [seed, offset] expected, "
                             f"got {rng.dtype} {tuple(rng.shape)}")
        if rng.device != x.device:
            raise ValueError(f"rng is on {rng.device}, the input on {x.device}")
        return p, rng.contiguous(), 0, 0
    if (isinstance(rng, (tuple, list)) and len(rng) == 2
            and all(isinstance(v, int) and not isinstance(v, bool)
                    for v in rng)):
        if not all(0 <= v < 2**63 for v in rng):
            raise ValueError(f"rng: seed and offset lie in [0, 2^63), got {rng}")
        return p, None, rng[0], rng[1]
    raise TypeError("rng: an int64 tensor of 2 or a pair of ints expected, got "
                    f"{rng!r}")


def _rng_tensor(rng, seed, offset):
    return torch.tensor([seed, offset]) if rng is None else rng


def _dense_format(x):
    if (x.dim() == 4 and not x.is_contiguous()
            and x.is_contiguous(memory_format=torch.channels_last)):
        return torch.channels_last
    return torch.contiguous_format


def dropout(x: torch.Tensor, p: float = 0.5, rng=None,
            act: str | None = None) -> torch.Tensor:
    """act(x) / (1 - p) where kept, 0 where dropped (with probability p).

    x: float32, float16 or bfloat16, any shape.  rng: what the mask is a
    function of, an int64 tensor [seed, offset] on x's device or a pair of
    ints in [0, 2^63); None draws one (`draw_rng`).  The mask is computed from
    (seed, offset, element) by Philox4x32-10 in both directions and never
    stored; elements are counted in memory order, channels fastest in
    channels-last tensors, and tensors of other strides are made contiguous.
    p is held to 2^-32.  A captured graph replays the mask of a pair of ints;
    it reads a tensor anew, and draws anew where rng is None.

    On the GPU forward-mode derivatives and tracing (torch.jit.trace, make_fx)
    raise NotImplementedError.
    """
    code = _act_code(act)
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"dropout: a tensor expected, got {type(x).__name__}")
    p, rng, seed, offset = _check_dropout(p, rng, x)
    if x.is_cuda:  # x is checked by the native call
        return require_hip().dropout(x, code, p, rng, seed, offset)
    _check_float(x, "dropout")
    x = x.contiguous(memory_format=_dense_format(x))
    return ref.dropout(x, p, _rng_tensor(rng, seed, offset), act)


def group_norm(x: torch.Tensor, num_groups: int,
               weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5,
               act: str | None = None, dropout: float = 0.0,
               rng=None) -> torch.Tensor:
    """Group norm, affine, activation and dropout of [B, C, H, W] in one go.

    x: float32, float16 or bfloat16; the result is channels last, and an x
    that is not is copied.  Statistics and all arithmetic are fp32.  act: None,
    "elu", "leaky_relu" (0.1), "relu" or "silu".  dropout: its probability;
    rng as for `dropout`, whose mask for the same rng is the same.

    On the GPU forward-mode derivatives and tracing (torch.jit.trace, make_fx)
    raise NotImplementedError.
    """
    code = _act_code(act)
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"group_norm: a tensor expected, got "
                        f"{type(x).__name__}")
    if type(num_groups) is not int:
        raise TypeError(f"group_norm: num_groups must be an int, got "
                        f"{num_groups!r}")
    p, rng, seed, offset = _check_dropout(dropout, rng, x)
    if x.is_cuda:  # tensors, groups and eps are checked by the native call
        return require_hip().group_norm(x, num_groups, weight, bias, eps, code,
                                        p, rng, seed, offset)
    _check_float(x, "group_norm")
    if x.dim() != 4:
        raise ValueError(f"group_norm: [B, C, H, W] expected, got "
                         f"{tuple(x.shape)}")
    c = x.shape[1]
    if not 1 <= num_groups <= _MAX_GROUPS or c == 0 or c % num_groups:
        raise ValueError(f"group_norm: {c} channels in {num_groups} groups "
                         f"(at most {_MAX_GROUPS})")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _check_float(t, f"group_norm {name}")
        if t.shape != (c,) or t.device != x.device:
            raise ValueError(f"group_norm: {name} must be [{c}] on {x.device}, "
                             f"got {tuple(t.shape)} on {t.device}")
    if not 0.0 < eps < float("inf"):
        raise ValueError(f"group_norm: eps must be positive, got {eps}")
    x = x.contiguous(memory_format=torch.channels_last)
    y = ref.group_norm(x, num_groups, weight, bias, eps, act, p,
                       _rng_tensor(rng, seed, offset) if p else None)
    return y.contiguous(memory_format=torch.channels_last)
