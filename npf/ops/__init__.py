"""MI355X ops layer: fused CDNA4 HIP kernels with torch reference fallbacks."""

from ._backend import extension, has_extension, require_extension
from .functional import (attention_qkv, clip_grad_norm_, conv_block_1d,
                         conv_block_2d, differential_attention,
                         gaussian_kl_sum, gaussian_nll_logmeanexp,
                         gaussian_nll_sum, grad_norm, grid_density, layer_norm,
                         mlp_chain, setconv_gaussian)

__all__ = [
    "attention_qkv",
    "clip_grad_norm_",
    "differential_attention",
    "grad_norm",
    "layer_norm",
    "conv_block_1d",
    "conv_block_2d",
    "grid_density",
    "gaussian_kl_sum",
    "mlp_chain",
    "setconv_gaussian",
    "gaussian_nll_sum",
    "gaussian_nll_logmeanexp",
    "extension",
    "has_extension",
    "require_extension",
]
