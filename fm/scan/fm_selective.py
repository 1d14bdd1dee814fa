"""Operators of a selective state space layer (`from fm.scan.fm_selective import fm_selective_scan`), served by fm_amd."""
from fm_amd.scan.fm_selective import (FM_Conv, FM_Selective, fm_conv, fm_conv_step, fm_selective_scan,  # noqa: F401
                                      fm_selective_step)
