"""cpmi355 -- host-side plumbing over libcpmi355.so (ctypes), MI355X / gfx950 only."""
from .capi import (CP_BF16, CP_CD_DELTA, CP_CD_RECIPROCAL, CP_E4M3, CP_E5M2, CP_F16, CP_F32, CP_F64,  # noqa: F401
                   CP_QUANT_POW2, Blocks, Context, CpError, DevBuf, OrthoJobs, OrthoStepJobs, default_context, device_count,
                   load, ortho_workspace)
from .pruner import LayerProblem, prune_layer, prune_layers_batched  # noqa: F401
