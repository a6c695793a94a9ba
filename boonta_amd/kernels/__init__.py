"""Stand-alone kernels behind boonta's network blocks (boonta/networks/kernels)."""
from .attention import linear_attention, linear_attention_step, qk_norm_rotary, rotary_frequencies
from .scan import get_scan_implementation, hip, scan, ssm, ssm_scan

__all__ = ["get_scan_implementation", "hip", "linear_attention", "linear_attention_step", "qk_norm_rotary",
           "rotary_frequencies", "scan", "ssm", "ssm_scan"]
