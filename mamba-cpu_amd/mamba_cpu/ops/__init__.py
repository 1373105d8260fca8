from mamba_cpu.ops.causal_conv1d import causal_conv1d_fn, causal_conv1d_update
from mamba_cpu.ops.embedding import embedding_fn
from mamba_cpu.ops.gated_linear import gated_linear_scan_fn, gated_linear_update
from mamba_cpu.ops.layer_norm import layer_norm_fn
from mamba_cpu.ops.mamba_inner import mamba_inner_fn
from mamba_cpu.ops.sampling import sample_fn
from mamba_cpu.ops.selective_scan_interface import selective_scan_fn
from mamba_cpu.ops.selective_state_update import selective_state_update
from mamba_cpu.ops.ssd_combined import mamba_chunk_scan_combined

__all__ = [
    "causal_conv1d_fn",
    "causal_conv1d_update",
    "embedding_fn",
    "gated_linear_scan_fn",
    "gated_linear_update",
    "layer_norm_fn",
    "mamba_chunk_scan_combined",
    "mamba_inner_fn",
    "sample_fn",
    "selective_scan_fn",
    "selective_state_update",
]
