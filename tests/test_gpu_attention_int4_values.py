"""Attention over the 4-bit cache whose value rows are constant (scale 0), large, or of
both kinds in one sequence."""
import math

import pytest
import torch

from int4_reference import DTYPES, attention, check, pack, quantised, rand
from test_gpu_attention_int4 import bound, cache, run
from test_gpu_attention_int4_routes import widened

pytestmark = pytest.mark.gpu


def constant(held, lens, bs, keys, low, seed=0):
    """The values of these keys of every sequence are `low` in all channels."""
    _, vc, _, vs, table = held
    for b, S in enumerate(lens):
        for j in keys:
            if j < S:
                page = table[b, j // bs]
                vs[page, :, j % bs, 0], vs[page, :, j % bs, 1] = 0.0, low


def compare(held, lens, rows, H, dt, causal=True, q_scale=1.0):
    dtype = DTYPES[dt]
    q = rand(sum(rows), H, held[0].shape[3] * 2, dtype=dtype, scale=q_scale, seed=3)
    got, cu = run(q, held, lens, rows, causal)
    ref, mass, reach = attention(q, *held[:4], cu, lens, held[4], None, causal)
    tiles = widened(dtype, H // held[0].shape[1], rows)
    over = ref.to(dtype).isinf()  # (past the type's range)
    assert not over.all()
    check(torch.where(over, torch.zeros_like(ref), got.cpu().double()), torch.where(over, torch.zeros_like(ref), ref),
          bound(ref, mass, reach, dtype, tiles), f"{lens} {rows}")


# rows and query heads (2 kv heads): columns held four, two times and once, two tiles
# of them, and more than a tile's; keys in one split and in several
ROWS = [([1], 4, [200]), ([1], 4, [5000]), ([1, 1], 16, [333, 40]), ([1], 32, [700]), ([9], 8, [200]),
        ([70], 8, [200]), ([70], 2, [1500])]


@pytest.mark.parametrize("rows,H,lens", ROWS)
@pytest.mark.parametrize("dt,low", [("bf16", 1.0), ("bf16", -1e9), ("bf16", 2.0 ** 28), ("bf16", 1e30),
                                    ("bf16", -1e38), ("bf16", 3e38), ("bf16", 1e-30), ("bf16", 0.0), ("f16", 60000.0),
                                    ("f16", -1.0), ("f16", 6e-8)])
def test_all_rows_constant(dt, low, rows, H, lens):
    """The answer is that constant (in fp32 weights sum to 1 but for 2^-18)."""
    held = cache(lens, 2, 128, 16, DTYPES[dt])
    constant(held, lens, 16, range(max(lens)), low)
    compare(held, lens, rows, H, dt)


@pytest.mark.parametrize("rows,H,lens", ROWS)
@pytest.mark.parametrize("keys", [range(0, 40), range(0, 128), range(150, 200), [7], [199]])
@pytest.mark.parametrize("dt,low", [("bf16", 1.0), ("bf16", 1e9), ("bf16", 1e30), ("bf16", -1e38), ("f16", 60000.0)])
def test_constant_rows_beside_ordinary_ones(dt, low, keys, rows, H, lens):
    held = cache(lens, 2, 128, 16, DTYPES[dt])
    constant(held, lens, 16, keys, low)
    compare(held, lens, rows, H, dt, causal=False)


@pytest.mark.parametrize("rows,H,lens", ROWS)
@pytest.mark.parametrize("scale", [2.0 ** 40, 1e20, 2.0 ** 101, 1e33, 2e37])
def test_large_values(scale, rows, H, lens):
    """Values up to the type's largest, and constant rows before them."""
    held = list(cache(lens, 2, 128, 16, torch.bfloat16, seed=1))
    n, pair = quantised((torch.randn(held[1].shape[0], 2, 16, 128, generator=torch.Generator().manual_seed(9))
                         .clamp(-8, 8) * scale).bfloat16())
    held[1], held[3] = pack(n), pair
    compare(held, lens, rows, H, "bf16")
    constant(held, lens, 16, range(0, 128), -3.0 * min(scale, 1e38))
    compare(held, lens, rows, H, "bf16")


# scales and lows of the blocks of 128 keys, (factor, constant or None): a wave sees each
# in turn, since 128 sequences of 2 kv heads leave keys unsplit
BLOCKS = {
    "constant rows, then large ones": [(1, 2.0 ** -80), (2.0 ** 45, None), (1, None)],
    "ordinary, then large, then ordinary": [(1, None), (2.0 ** 60, None), (1, None), (1, 5.0)],
    "constants far apart": [(1, 2.0 ** -100), (1, 1.0), (1, 2.0 ** 50), (1, -2.0 ** 100)],
    "large, then larger": [(2.0 ** 39, None), (2.0 ** 41, None), (2.0 ** 100, None), (2.0 ** 123, None)],
    "zeros, then small ones": [(1, 0.0), (2.0 ** -100, None), (2.0 ** -90, None)],
    "from the smallest to the largest": [(2.0 ** -120, None), (2.0 ** -40, None), (2.0 ** 40, None), (2.0 ** 118, None)],
}


@pytest.mark.parametrize("what", list(BLOCKS))
@pytest.mark.parametrize("rows,H", [(1, 2), (1, 4), (1, 16), (1, 32), (5, 8)])
def test_blocks_of_one_wave(what, rows, H):
    blocks, S, B = BLOCKS[what], 520, 128
    lens = [S] * 3 + [128 * len(blocks) - 40] + [1] * (B - 4)
    held = list(cache(lens, 2, 64, 16, torch.bfloat16, seed=1))
    for b in range(4):
        for i, (factor, low) in enumerate(blocks):
            j = torch.arange(128 * i, min(128 * i + 128, lens[b]))
            at = held[4][b, j // 16].long(), slice(None), j % 16
            pair = held[3][at].double() / 8 * factor  # (|values| below 1 * factor, unless far out)
            if low is not None:
                pair = torch.stack([torch.zeros_like(pair[..., 0]), torch.full_like(pair[..., 0], low)], -1)
            held[3][at] = pair.to(torch.bfloat16)
    compare(held, lens, [rows] * 4 + [1] * (B - 4), H, "bf16", causal=False)


@pytest.mark.parametrize("rows,H,lens", ROWS)
@pytest.mark.parametrize("dt,low", [("bf16", 1e9), ("bf16", 1e36), ("f16", 50000.0)])
def test_nan_rows_among_large_ones(dt, low, rows, H, lens):
    """A value row of NaN among large constants reaches the rows that see it alone."""
    held = cache(lens, 2, 128, 16, DTYPES[dt])
    constant(held, lens, 16, range(max(lens)), low)
    b, j = 0, lens[0] - 1
    held[3][held[4][b, j // 16], 1, j % 16] = math.nan
    q = rand(sum(rows), H, 128, dtype=DTYPES[dt], seed=3)
    got, cu = run(q, held, lens, rows, True)
    nan = torch.zeros(sum(rows), H, dtype=torch.bool)
    nan[rows[0] - 1, H // 2:] = True
    assert torch.equal(torch.isnan(got.cpu()).all(-1), nan) and torch.equal(torch.isnan(got.cpu()).any(-1), nan)


@pytest.mark.parametrize("rows", [1, 9])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_many_keys_of_one_value(rows, dt):
    """20000 keys: sums of weights and of weight * value stay within fp32."""
    S, D = 20000, 64
    g = torch.Generator().manual_seed(2)
    n, ks = quantised(torch.randn(S // 16, 1, 16, D, generator=g).to(DTYPES[dt]))
    low = 60000.0 if dt == "f16" else 1e30
    vs = torch.zeros(S // 16, 1, 16, 2, dtype=DTYPES[dt])
    vs[..., 1] = low
    held = (pack(n), torch.zeros_like(pack(n)), ks, vs, torch.arange(S // 16, dtype=torch.int32)[None])
    compare(held, [S], [rows], 4, dt, q_scale=0.05)
