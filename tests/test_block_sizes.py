"""Sizes past 32 bits are refused: an entry point takes them as C ints, which would keep the low half of them."""
import pytest
import torch

from boonta_amd.kernels import gated_scan, gated_scan_step, linear_attention, qk_norm_rotary, residual_norm, token_log_probs

LONG = (1 << 32) + 5


def wide(*shape, dtype=torch.float32):
    return torch.zeros((), dtype=dtype).expand(shape)


@pytest.mark.parametrize("shape", [(1, LONG, 1), (LONG, 1, 1), (1 << 31, 1, 1)])
def test_sizes_past_32_bits_are_refused(shape):
    x = wide(*shape)
    tokens = wide(*shape[:2], dtype=torch.int64)
    heads = wide(*shape[:2], 1, 8)
    for call in (lambda: residual_norm(x, x), lambda: gated_scan(x, x, x, torch.ones(1)), lambda: token_log_probs(x, tokens),
                 lambda: token_log_probs(x[:, 0] if shape[1] == 1 else x[0], tokens[:, 0] if shape[1] == 1 else tokens[0]),
                 lambda: linear_attention(heads, heads, heads, torch.zeros(1)), lambda: qk_norm_rotary(heads, heads)):
        with pytest.raises(ValueError, match="up to 2\\^31 - 1"):
            call()
    if shape[0] > 1:
        y = x[:, 0]
        with pytest.raises(ValueError, match="up to 2\\^31 - 1"):
            gated_scan_step(y, y, y, torch.ones(1), y)
    with pytest.raises(ValueError, match="up to 2\\^31 - 1"):
        qk_norm_rotary(wide(1, 1, 1, 8), wide(1, 1, LONG, 8))
    with pytest.raises(ValueError, match="up to 2\\^31 - 1"):
        gated_scan(wide(1, 1, LONG), wide(1, 1, LONG), wide(1, 1, LONG), wide(LONG))
