"""The build's check of the wait states behind matrix products
(teco-ops_amd/build.py check_matrix_waits), on hand-written assembly."""
import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "teco-ops_amd"))
import build  # noqa: E402

PRODUCT = "\tv_mfma_f32_16x16x32_f16 v[24:27], v[20:23], v[10:13], 0\n"
READ = "\tv_cndmask_b32_e64 v30, v26, v24, s[8:9]\n"


def run(body):
    return build.check_matrix_waits("_Zkernel:\n" + body + "\ts_endpgm\n.Lfunc_end0:\n", "test.hip")


def test_a_full_wait_passes():
    assert run(PRODUCT + "\ts_nop 7\n" + READ) == 1
    assert run(PRODUCT + "\tv_add_f32_e32 v1, v2, v3\n" * 8 + READ) == 1


@pytest.mark.parametrize("between", ["", "\ts_nop 6\n", "\tv_add_f32_e32 v1, v2, v3\n" * 7])
def test_a_short_wait_is_refused(between):
    with pytest.raises(RuntimeError, match="wait states behind"):
        run(PRODUCT + between + READ)


def test_the_shorter_path_counts():
    body = PRODUCT + "\ts_cbranch_scc1 .LBB0_2\n\ts_nop 7\n.LBB0_2:\n" + READ
    with pytest.raises(RuntimeError, match="only 1 wait"):
        run(body)
    assert run(PRODUCT + "\ts_nop 6\n\ts_cbranch_scc1 .LBB0_2\n.LBB0_2:\n" + READ) == 1


def test_a_chain_of_products_needs_no_wait_for_its_sums():
    chain = "\tv_mfma_f32_16x16x32_f16 v[24:27], v[20:23], v[10:13], v[24:27]\n"
    assert run(PRODUCT + chain + "\ts_nop 7\n" + READ) == 2
    with pytest.raises(RuntimeError):
        run(PRODUCT + "\tv_mfma_f32_16x16x32_f16 v[0:3], v[24:27], v[10:13], 0\n")
