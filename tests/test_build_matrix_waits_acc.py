"""The build's check of the wait states behind matrix products whose results lie in
accumulation registers, operands by their place, and that every source is checked
(teco-ops_amd/build.py), on hand-written assembly."""
import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "teco-ops_amd"))
import build  # noqa: E402

PRODUCT = "\tv_mfma_f32_16x16x32_f16 a[24:27], v[20:23], v[10:13], a[24:27]\n"
READS = ["\tv_accvgpr_read_b32 v1, a25\n", "\tglobal_store_dwordx4 v[2:3], a[24:27], off\n",
         "\tds_write_b32 v2, a27\n", "\tv_accvgpr_write_b32 a26, v2\n",
         "\tv_mfma_f32_16x16x32_f16 v[0:3], a[24:27], v[10:13], 0\n",
         "\tv_mfma_f32_16x16x32_f16 v[0:3], v[10:13], a[24:27], 0\n"]


def run(body):
    return build.check_matrix_waits("_Zkernel:\n" + body + "\ts_endpgm\n.Lfunc_end0:\n", "test.hip")


@pytest.mark.parametrize("read", READS)
def test_short_waits_are_refused(read):
    for between in ("", "\ts_nop 6\n", "\tv_add_f32_e32 v1, v2, v3\n" * 7):
        with pytest.raises(RuntimeError, match="wait states behind"):
            run(PRODUCT + between + read)
    run(PRODUCT + "\ts_nop 7\n" + read)


def test_sums_of_a_part_wait_two_states_less():
    part = "\tv_mfma_f32_16x16x32_f16 a[26:29], v[10:13], v[14:17], a[26:29]\n"
    with pytest.raises(RuntimeError, match="only 5 wait"):
        run(PRODUCT + "\ts_nop 4\n" + part)
    assert run(PRODUCT + "\ts_nop 5\n" + part) == 2


def test_register_files_are_apart():
    assert run(PRODUCT + "\tv_add_f32_e32 v24, v25, v26\n") == 1
    assert run(PRODUCT + "\tv_mfma_f32_16x16x32_f16 v[0:3], v[24:27], v[10:13], 0\n\ts_nop 7\n") == 2
    # its own operands may be loaded anew, and the whole result added to at once
    assert run(PRODUCT + "\tv_mov_b32_e32 v20, v1\n" + PRODUCT) == 2


def test_what_another_product_writes_is_that_ones():
    over = "\tv_mfma_f32_16x16x32_f16 a[22:25], v[10:13], v[14:17], a[40:43]\n"
    add = "\tv_mfma_f32_16x16x32_f16 a[40:43], v[10:13], v[14:17], a[22:25]\n"
    assert run(PRODUCT + over + add + "\ts_nop 7\n") == 3
    with pytest.raises(RuntimeError, match="only 2 wait"):
        run(PRODUCT + over + "\tv_accvgpr_read_b32 v1, a2\n" + "\tv_accvgpr_read_b32 v1, a27\n")
    with pytest.raises(RuntimeError, match="only 0 wait"):
        run(PRODUCT + over + "\tv_accvgpr_read_b32 v1, a24\n")


@pytest.mark.parametrize("result", ["v[24:27]", "a[24:27]"])
def test_operands_go_by_their_place(result):
    """The first operand counts also where the result is of the other file."""
    product = f"\tv_mfma_f32_16x16x32_f16 {result}, v[20:23], v[10:13], 0\n"
    second = f"\tv_mfma_f32_16x16x32_f16 a[0:3], {result}, v[10:13], a[0:3]\n"
    with pytest.raises(RuntimeError):
        run(product + second)


def test_every_device_source_is_checked(monkeypatch, tmp_path):
    """Products are looked for in all sources, and copies in a source that is not listed
    for them are an error."""
    seen = []
    monkeypatch.setattr(build, "_check_assembly", lambda src: seen.append(src))
    monkeypatch.setattr(build, "_compile", lambda src: (src, ""))
    monkeypatch.setattr(build, "BUILD", str(tmp_path))

    class Linked(Exception):
        pass

    def link(*a, **kw):
        raise Linked
    monkeypatch.setattr(build.subprocess, "run", link)
    with pytest.raises(Linked):
        build.build()
    assert sorted(seen) == sorted(s for s in build.SOURCES if s.endswith(".hip"))
    assert "gemv_int4.hip" in seen
