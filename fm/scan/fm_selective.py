"""Operators of a selective state space layer (`from fm.scan.fm_selective import fm_conv`), served by fm_amd."""
from fm_amd.scan.fm_selective import FM_Conv, fm_conv, fm_conv_step  # noqa: F401
