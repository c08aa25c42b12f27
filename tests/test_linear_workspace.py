"""The workspace that a product asks for is enough for every plan of its sizes,
whether its rows can be copied into LDS or, off 16-byte words, go through registers
(no GPU)."""
import ctypes

import pytest

from tecoops import _lib
from test_layer_abi import plan  # noqa: F401

MOST = 512 << 20


def asked(m, n, k, gated):
    size = ctypes.c_size_t()
    _lib.call("tecoopsGetLinearWorkspaceSize", m, n, k, gated, ctypes.byref(size))
    return size.value


@pytest.mark.parametrize("copy", [0, 1])
@pytest.mark.parametrize("gated", [0, 1])
def test_asked_is_enough(plan, gated, copy):  # noqa: F811
    split = 0
    for m in (1, 2, 8, 17, 33, 64, 65, 128, 200, 333, 1000):
        for n in (32, 70, 256, 1024, 4096, 14336):
            for k in (64, 512, 588, 4096, 14336, 14337):
                if copy and k % 8:
                    continue
                ws = asked(m, n, k, gated)
                best, got = plan(m, n, k, gated, copy, MOST), plan(m, n, k, gated, copy, ws)
                assert got == best, (m, n, k)
                split += got[4] > 1
    assert split > 50


def test_views_of_few_rows_are_split(plan):  # noqa: F811
    """Rows that would stream W if they could be copied still get their splits."""
    for m, n, k in ((1, 4096, 4096), (8, 4096, 14336), (24, 4096, 4096)):
        assert plan(m, n, k)[7] and plan(m, n, k, copy=0, ws=asked(m, n, k, 0))[4] > 1
