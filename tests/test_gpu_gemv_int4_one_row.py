"""Products of one row of x with 4-bit weights around the K up to which one kernel takes
it, and across it: the same answer either way."""
import pytest

from test_gpu_gemv_int4 import compare

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n,k,group", [(40, 4096, 128), (40, 4128, 32), (1, 6144, 64), (33, 8160, 32), (300, 8192, 128),
                                       (300, 8192, 8192), (65, 8224, 32), (17, 8320, 160), (4100, 5120, 128)])
def test_one_row(n, k, group, zeros, dt):
    compare(1, n, k, group, zeros, dt)
