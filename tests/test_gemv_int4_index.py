"""Index arithmetic of products with 4-bit weights over a long K (gemv_int4.h), on the
CPU: the header built as host C++."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "teco-ops_amd", "csrc")
MOST_K = (1 << 31) - 32  # whole groups of 32


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("index")
    (d / "index.cpp").write_text("""#include "gemv_int4.h"
extern "C" {
int stages(int k) { return tecoops::gemv_int4_stages(k); }
int past(int from, int count, int end) { return tecoops::gemv_int4_past(from, count, end); }
int group(int slot, int slots, int most) {
    return tecoops::gemv_int4_quotient(slot, slots, tecoops::gemv_int4_inverse(slots, most));
}
int product(int slots, int most) { return tecoops::gemv_int4_inverse(slots, most) != 0; }
int parts(int b, int n, int k) { return tecoops::gemv_int4_plan(b, n, k, ~size_t{0}, 256).parts; }
}
""")
    # (a signed overflow ends the program)
    subprocess.run(["g++", "-std=c++17", "-O1", "-ftrapv", "-fPIC", "-shared", "-I", CSRC, str(d / "index.cpp"), "-o",
                    str(d / "index.so")], check=True)
    return ctypes.CDLL(str(d / "index.so"))


KS = [32, 64, 480, 512, 544, 1024, 14336, 1 << 20, 201332160, (1 << 30) + 32, MOST_K - 512, MOST_K - 32, MOST_K]


@pytest.mark.parametrize("k", KS)
def test_stages_and_words_past_k(lib, k):
    n = lib.stages(k)
    assert (n - 1) * 512 < k <= n * 512
    assert 1 <= lib.parts(1, 1, k) <= max(1, n // 2)
    for st in {0, n // 2, n - 1}:
        for at in range(0, 512, 8):
            assert lib.past(st * 512 + at, 8, k) == max(0, st * 512 + at + 8 - k)
        for at in range(0, 256, 16):
            assert lib.past(st * 256 + at, 16, k // 2) == max(0, st * 256 + at + 16 - k // 2)


@pytest.mark.parametrize("slots", [1, 2, 3, 5, 7, 12, 100, 1000, 65535, 6291456, (1 << 26) - 1])
@pytest.mark.parametrize("most", [16, 4096, 6291630, 1 << 26])
def test_groups_of_uses(lib, slots, most):
    """The quotient for all uses up to the last of a K, beside multiples and at random
    (with a float's 24 bits the first wrong one of three a group is 6291458)."""
    g = random.Random(slots + most)
    at = {0, 1, most - 1, 6291458} | {g.randrange(most) for _ in range(200)}
    for _ in range(200):
        m = g.randrange(most // slots + 1) * slots
        at |= {m - 1, m, m + 1}
    for a in at:
        if 0 <= a <= most:
            assert lib.group(a, slots, most) == a // slots, (a, slots, most)


def test_ordinary_sizes_take_a_product(lib):
    for slots in (2, 3, 5, 32, 112):
        assert lib.product(slots, 65536 // 32)
