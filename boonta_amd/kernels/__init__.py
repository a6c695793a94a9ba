"""Stand-alone kernels behind boonta's network blocks (boonta/networks/kernels)."""
from .attention import linear_attention, linear_attention_step, qk_norm_rotary, rotary_frequencies
from .gated import gated_scan, gated_scan_step
from .residual import residual_norm
from .scan import get_scan_implementation, hip, scan, ssm, ssm_scan
from .tokens import TokenLogProbs, token_log_probs

__all__ = ["TokenLogProbs", "gated_scan", "gated_scan_step", "get_scan_implementation", "hip", "linear_attention",
           "linear_attention_step", "qk_norm_rotary", "residual_norm", "rotary_frequencies", "scan", "ssm", "ssm_scan",
           "token_log_probs"]
