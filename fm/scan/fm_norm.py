"""Norm with the residual's addition (`from fm.scan.fm_norm import fm_norm`), served by fm_amd."""
from fm_amd.scan.fm_norm import FM_Norm, fm_norm, fm_norm_quantized  # noqa: F401
