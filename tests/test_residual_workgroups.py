"""How the norms around a block spread many rows over the chip, from the sizes of the backward's workspace: two sums
of each column for each workgroup."""
import pytest

from boonta_amd import _lib

CUS = 256


def workgroups(dtype, rows, width):
    nbytes = _lib.load().ppo_residual_norm_bwd_workspace(dtype, 1, rows, width)
    assert nbytes % (8 * width) == 0
    return nbytes // (8 * width)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("width", [1, 8, 40, 300, 512, 513, 640, 768, 769, 1000, 1100, 1536, 2048, 2300, 2560, 3000, 3500, 4096, 4097,
                                   5000, 6144, 7000, 8192])
def test_every_cu_gets_as_many_workgroups(dtype, width):
    groups, waves = workgroups(dtype, 1 << 20, width), max(4 if width <= 512 else 0, -(-width // 512))
    assert groups % CUS == 0 and 8 <= groups // CUS * waves <= 16
    assert workgroups(dtype, 1, width) == 1
    if width > 512:   # (a row each)
        assert workgroups(dtype, 100, width) == 100 and workgroups(dtype, 0, width) == 0
