"""Attention over the 4-bit cache where keys that a row does not see (they come after it)
are far larger than those that it sees: they change nothing for it, by either route."""
import pytest
import torch

from int4_reference import DTYPES, attention, check, rand
from test_gpu_attention_int4 import bound, cache, run
from test_gpu_attention_int4_routes import widened

pytestmark = pytest.mark.gpu

# rows, query heads (2 kv heads), keys of two sequences: a prompt within a block of keys,
# columns held once to four times, two tiles, widened tiles of four and of twelve waves,
# keys in several splits, head sizes of each kind of value word
SHAPES = [([2, 1], 2, [2, 3], 128), ([8, 5], 2, [8, 5], 128), ([4, 4], 4, [4, 33], 64), ([9, 3], 8, [200, 3], 128),
          ([20, 16], 4, [20, 300], 96), ([70, 70], 4, [70, 200], 128), ([70, 70], 2, [200, 75], 192),
          ([40, 40], 8, [1500, 40], 128), ([150, 130], 8, [150, 140], 32), ([6, 6], 16, [40, 6], 160)]


def larger(held, lens, which, power, constant=False):
    """The last key (or value) of every sequence 2^power times what it was, or all its
    elements 2^power."""
    out = [t.clone() for t in held]
    for b, S in enumerate(lens):
        at = held[4][b, (S - 1) // 16].long(), slice(None), (S - 1) % 16
        pair = held[which][at].double()
        pair = torch.stack([0 * pair[..., 0], torch.full_like(pair[..., 0], 2.0 ** power)], -1) if constant \
            else pair * 2.0 ** power
        out[which][at] = pair.to(held[which].dtype)
    return out


def compare(held, changed, lens, rows, H, dt):
    """Over `changed`: the rows that do not see the last key against the formula over
    `held` (a weight of 0 times an infinite value would be none), the others returned."""
    dtype = DTYPES[dt]
    q = rand(sum(rows), H, 2 * held[0].shape[3], dtype=dtype, seed=2)
    got, cu = run(q, changed, lens, rows)
    last = torch.zeros(sum(rows), dtype=torch.bool)
    last[torch.tensor(cu[1:]) - 1] = True
    of = []
    for h in (held, changed):
        ref, mass, reach = attention(q, *h[:4], cu, lens, h[4])
        of.append((ref, bound(ref, mass, reach, dtype, widened(dtype, H // 2, rows))))
    check(got.cpu()[~last], of[0][0][~last], of[0][1][~last], f"{lens} {rows}")
    return got.cpu()[last], of[1][0][last], of[1][1][last]


@pytest.mark.parametrize("rows,H,lens,D", SHAPES)
@pytest.mark.parametrize("which,constant", [(2, False), (3, False), (3, True)])
@pytest.mark.parametrize("dt,power", [("bf16", 8), ("bf16", 20), ("bf16", 26), ("bf16", 30), ("bf16", 45), ("bf16", 80),
                                      ("bf16", 120), ("f16", 12), ("f16", 15)])
def test_hidden_keys_and_values(dt, power, which, constant, rows, H, lens, D):
    held = cache(lens, 2, D, 16, DTYPES[dt], seed=1)
    got, ref, limit = compare(held, larger(held, lens, which, power, constant), lens, rows, H, dt)
    if which == 3:  # (the rows that see a large value: it is most of their output, or all)
        fine = torch.isfinite(ref)
        check(got[fine], ref[fine], limit[fine], "last rows")
        assert not torch.isfinite(got[~fine]).any()


@pytest.mark.parametrize("rows,H,lens,D", SHAPES)
@pytest.mark.parametrize("power", [-16, -20, -26, -40])
def test_small_rows_before_ordinary_ones(power, rows, H, lens, D):
    """The values of all but the last rows' keys are small: so are the outputs."""
    held = cache(lens, 2, D, 16, torch.bfloat16, seed=1)
    held[3].mul_(2.0 ** power)
    got, ref, limit = compare(held, larger(held, lens, 3, -power), lens, rows, H, "bf16")
    check(got, ref, limit, "last rows")


@pytest.mark.parametrize("rows,H", [([70], 2), ([70], 8)])
def test_fp16_small_rows_before_ordinary_ones(rows, H):
    held = cache([70], 2, 128, 16, torch.float16, seed=1)
    held[3].mul_(2.0 ** -9)
    got, ref, limit = compare(held, larger(held, [70], 3, 20), [70], rows, H, "f16")
    check(got, ref, limit, "last rows")


def test_rows_far_apart_in_splits():
    """Keys cut into splits, a large value in the last: states of either kind join."""
    rows, lens = [30, 30], [1500, 700]
    for dt, power in (("bf16", 40), ("bf16", 110)):
        held = cache(lens, 2, 128, 16, DTYPES[dt], seed=1)
        for H in (4, 16):
            got, ref, limit = compare(held, larger(held, lens, 3, power), lens, rows, H, dt)
            check(got, ref, limit, "last rows")


def test_nan_and_far_rows():
    """A NaN value row among rows far apart, in the widened tiles' plain form too."""
    rows, lens = [70], [90]
    held = larger(cache(lens, 2, 128, 16, torch.bfloat16, seed=1), lens, 3, 60)
    for key, which in ((80, 3), (82, 2)):
        held[which][held[4][0, key // 16], 0, key % 16] = float("nan")
    q = rand(70, 8, 128, dtype=torch.bfloat16)
    got, _ = run(q, held, lens, rows)
    nan = torch.zeros(70, 8, dtype=torch.bool)
    nan[60:, :4] = True  # (row r sees keys up to 20 + r)
    assert torch.equal(torch.isnan(got.cpu()).all(-1), nan) and torch.equal(torch.isnan(got.cpu()).any(-1), nan)


@pytest.mark.parametrize("dt,what", [(t, x) for t in ("f16", "bf16") for x in (float("inf"), float("nan"), 2.0 ** 13)] +
                         [("bf16", 2.0 ** 30), ("bf16", 2.0 ** 100)])
@pytest.mark.parametrize("rows,H,lens,D", SHAPES)
def test_query_rows_of_other_sizes(rows, H, lens, D, what, dt):
    """One query row (of one head) infinite, none or large: the others are what they are."""
    dtype = DTYPES[dt]
    held = cache(lens, 2, D, 16, dtype, seed=1)
    q = rand(sum(rows), H, D, dtype=dtype, seed=2)
    ref, mass, reach = attention(q, *held[:4], [0, rows[0], sum(rows)], lens, held[4])
    r, h = rows[0] // 2, H - 1
    if what - what == 0:
        q[r, h] *= what / 4
    else:
        q[r, h, 3] = what
    got, _ = run(q, held, lens, rows)
    others = torch.ones(sum(rows), H, dtype=torch.bool)
    others[r, h] = False
    check(got.cpu()[others], ref[others], bound(ref, mass, reach, dtype, widened(dtype, H // 2, rows))[others], "others")
    if what - what != 0:
        assert torch.isnan(got[r, h]).all()


@pytest.mark.parametrize("power", [0, 60])
@pytest.mark.parametrize("rows,H", [(3, 4), (9, 8), (70, 8), (100, 8)])
def test_infinite_value_rows_are_none(power, rows, H):
    """A value row whose pair is infinite makes the rows that see it NaN, and no others, in
    every form (2^60 apart: key by key)."""
    held = larger(cache([130], 2, 128, 16, torch.bfloat16, seed=1), [130], 3, power)
    for i, (key, pair) in enumerate(((127, (float("inf"), 0.0)), (128, (0.0, -float("inf"))))):
        held[3][held[4][0, key // 16], i, key % 16] = torch.tensor(pair, dtype=torch.bfloat16)
    q = rand(rows, H, 128, dtype=torch.bfloat16)
    got, _ = run(q, held, [130], [rows])
    nan = torch.zeros(rows, H, dtype=torch.bool)
    nan[rows - 3:, :H // 2] = True  # (row r sees keys up to 130 - rows + r)
    nan[rows - 2:, H // 2:] = True
    assert torch.equal(torch.isnan(got.cpu()).all(-1), nan) and torch.isfinite(got.cpu()[~nan]).all()
