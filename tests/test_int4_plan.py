"""How attention over the 4-bit cache is cut (fa_int4.h), for every type's route and for
bounds far past what the tensors hold, on the CPU: the header built as host C++."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "teco-ops_amd", "csrc")
MOST = (1 << 31) - 1


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text("""#include "fa_int4.h"
extern "C" void plan(int b, int h, int hkv, int d, int rows, int keys, unsigned long long room, int exact, long long *o) {
    const auto p = tecoops::fa4::make_plan(b, h, hkv, d, rows, keys, room, 256, exact != 0);
    o[0] = p.split; o[1] = p.split ? p.ct * 16 : p.waves * 32; o[2] = p.tiles; o[3] = p.cols;
    o[4] = p.split_len; o[5] = p.splits; o[6] = (long long)p.bytes;
}
extern "C" int row_bound(int most, int total, int batch) { return tecoops::fa4::row_bound(most, total, batch); }
""")
    # (a signed overflow ends the program)
    subprocess.run(["g++", "-std=c++17", "-O1", "-ftrapv", "-fPIC", "-shared", "-I", CSRC, str(d / "plan.cpp"), "-o",
                    str(d / "plan.so")], check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))
    lib.plan.argtypes = [ctypes.c_int] * 6 + [ctypes.c_ulonglong, ctypes.c_int, ctypes.c_void_p]
    return lib


def test_rows_are_bounded_by_what_is_there(lib):
    """At least the mean, at most all rows, whatever the caller's bound."""
    for total, batch in ((1, 1), (64, 64), (91, 3), (5000, 7), (MOST, 1), (0, 4)):
        mean = max(1, -(-total // batch))
        for most in (-5, 0, 1, mean, mean + 3, 8192, 131072, MOST):
            got = lib.row_bound(most, total, batch)
            assert got == min(max(most, mean), max(total, 1))
            assert mean <= got <= max(total, 1)


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("room", [0, 1 << 20, 1 << 63])
def test_grids_hold_and_splits_are_whole(lib, exact, room):
    """For every bound a grid that can be launched, splits of whole blocks of pages
    (which are followed by 16 keys) that cover the keys, states within the workspace."""
    o = (ctypes.c_longlong * 7)()
    for b in (1, 2, 5, 64, 4096, 65536, 1 << 22):
        for h, hkv in ((1, 1), (8, 1), (32, 8), (64, 1), (40, 8), (128, 2)):
            if b * hkv > 1 << 22:
                continue
            for rows in (1, 2, 5, 17, 33, 100, 203, 1000, 68536, 1 << 24, MOST):
                for keys in (1, 31, 128, 777, 2049, 8192, 16300, 100000, MOST - 4096):
                    for d in (32, 128, 192):
                        lib.plan(b, h, hkv, d, rows, keys, room, exact, o)
                        split, tile, tiles, cols, length, splits, need = o
                        want = min(h // hkv * rows, MOST)
                        assert split == (exact or want <= 64)
                        assert cols <= want and (tiles - 1) * tile < cols <= tiles * tile
                        assert b * hkv * tiles * splits <= 1 << 22
                        assert splits <= 65535 and (split or tiles * splits <= 65535)
                        # fewer columns than the bound only where the grid is full
                        assert cols == want or b * hkv * (tiles + 1) > 1 << 22 or tiles == 65535
                        assert length > 0 and (splits == 1 or length % (128 if split else 96) == 0)
                        assert splits >= 1 and (splits - 1) * length < keys
                        assert splits * length >= keys or splits == 1
                        assert need == (0 if splits == 1 else b * hkv * splits * cols * (d + 2) * 4) and need <= room
