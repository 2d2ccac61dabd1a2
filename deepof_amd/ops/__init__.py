from .functional import (
    warp_bilinear,
    resize_bilinear,
    lrn,
    correlation,
    unsup_loss_scale,
    endpoint_error_sum,
    draw_rng,
    dropout,
    group_norm,
    hip_available,
    require_hip,
)
from .norm import CounterDropout, GroupNormAct

__all__ = [
    "CounterDropout",
    "GroupNormAct",
    "warp_bilinear",
    "resize_bilinear",
    "lrn",
    "correlation",
    "unsup_loss_scale",
    "endpoint_error_sum",
    "draw_rng",
    "dropout",
    "group_norm",
    "hip_available",
    "require_hip",
]
