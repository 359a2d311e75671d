"""Mamba-2 operators of ``metal_kernelops.cv`` on MI355X (HIP kernels).

The names follow the reference's ``cv/__init__.py:15-40`` for the SSM scan path and
its neighbours in a Mamba block: the chunked SSD scan and the single-token decode
update (each with its pure-torch twin), the four-path 2D scan (VMamba's ss2d) built
on the Mamba-1 scan kernels, the causal depthwise conv1d ahead of the scan and the
gated RMSNorm after it.  Beside them, for layers around those scans, stand operators that the
reference does not have: the gated linear recurrence and its one-token update, the RMS norm of
the residual stream, and the projections in 8-bit integers.  The reference's other ``cv`` operators (NSA selection,
RoIAlign and the rest) are not part of this package.  Importing it registers the
``mko::`` custom ops and launches nothing.
"""

from .causal_conv1d import causal_conv1d_fn, causal_conv1d_ref, causal_conv1d_update
from .gated_norm import rmsnorm_gated, rmsnorm_gated_reference
from .gated_recurrence import (
    gated_recurrence,
    gated_recurrence_reference,
    gated_recurrence_update,
    gated_recurrence_update_reference,
)
from .int8_linear import int8_linear, int8_linear_reference, quantize_int8, quantize_int8_reference
from .mamba2_chunk import last_path, mamba2_chunk_scan, mamba2_chunk_scan_reference
from .mamba2_state import CHECKED_TORCH, mamba2_state_update, mamba2_state_update_reference
from .path_scan import MAX_STATES, MERGE_MODES, path_orders, ss2d_scan, ss2d_scan_reference
from .residual_norm import (
    rmsnorm_residual,
    rmsnorm_residual_int8,
    rmsnorm_residual_int8_reference,
    rmsnorm_residual_reference,
)

__all__ = [
    "CHECKED_TORCH",
    "MAX_STATES",
    "MERGE_MODES",
    "causal_conv1d_fn",
    "causal_conv1d_ref",
    "causal_conv1d_update",
    "gated_recurrence",
    "gated_recurrence_reference",
    "gated_recurrence_update",
    "gated_recurrence_update_reference",
    "int8_linear",
    "int8_linear_reference",
    "last_path",
    "mamba2_chunk_scan",
    "mamba2_chunk_scan_reference",
    "mamba2_state_update",
    "mamba2_state_update_reference",
    "path_orders",
    "quantize_int8",
    "quantize_int8_reference",
    "rmsnorm_gated",
    "rmsnorm_gated_reference",
    "rmsnorm_residual",
    "rmsnorm_residual_int8",
    "rmsnorm_residual_int8_reference",
    "rmsnorm_residual_reference",
    "ss2d_scan",
    "ss2d_scan_reference",
]
