"""Attention over the 4-bit cache against the formula in 64 bits."""
import math

import pytest
import torch

import tecoops
from int4_reference import DTYPES, HALF_STEP, SMALLEST, attention, check, pack, quantised, rand

pytestmark = pytest.mark.gpu


def cache(lens, Hkv, D, bs, dtype, seed=0, scale=1.0, shift=0.0):
    """A cache of random rows, its pages shuffled; what lies behind a sequence's last
    key is NaN. Codes, pairs of keys and values, table."""
    g = torch.Generator().manual_seed(seed)
    need = [(s + bs - 1) // bs for s in lens]
    NB = sum(need) + 2
    perm = torch.randperm(NB, generator=g).int()
    table = torch.full((len(lens), max(max(need), 1) + 1), -7, dtype=torch.int32)
    at, held = 0, []
    for i in range(2):
        n, pair = quantised(((torch.randn(NB, Hkv, bs, D, generator=g) + shift) * scale).to(dtype))
        held.append((pack(n), pair))
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
        if lens[b] % bs:
            for _, pair in held:
                pair[table[b, n - 1], :, lens[b] % bs:] = math.nan
    return held[0][0], held[1][0], held[0][1], held[1][1], table


def bound(ref, mass, reach, dtype, tiles):
    """The weights (times a scale) are rounded to fp16, 2^-11 of each, in either
    route; in the split route W = fp16(p s) multiplies n - 7.5, that is, an error of W
    moves the sum by it times the value's distance from the middle of its row.  The tile route also rounds keys and values to fp16: a score moves by
    2^-11 reach, its weight by twice that against the others, the values by 2^-11.
    In fp32: scores (128 products, 2^-18 reach, and their exponential), sums 2^-18.
    Then one rounding of the result."""
    unit = 2.0 ** -11
    soft = unit + 2.0 ** -17 + 2.0 ** -16 * reach
    if tiles:
        soft = soft + unit * (1.0 + 2.2 * reach)
    return HALF_STEP[dtype] * ref.abs() + soft * mass * 1.01 + SMALLEST[dtype]


def run(q, held, lens, rows, causal=True, scale=None, most_q=None, most_k=None, extra=0):
    kc, vc, ks, vs, table = [t.cuda() for t in held]
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    out = torch.full((q.shape[0] + extra, *q.shape[1:]), 5.0, dtype=q.dtype, device="cuda")
    qd = torch.cat([q, torch.ones(extra, *q.shape[1:], dtype=q.dtype)]).cuda()
    tecoops.flash_attn_varlen_int4(qd, kc, vc, ks, vs, max(rows) if most_q is None else most_q,
                                   torch.tensor(cu, dtype=torch.int32).cuda(),
                                   max(lens) if most_k is None else most_k,
                                   torch.tensor(lens, dtype=torch.int32).cuda(), scale, causal, table, out)
    torch.cuda.synchronize()
    assert (out[q.shape[0]:] == 0).all()
    return out[:q.shape[0]], cu


def compare(dt, H, Hkv, D, bs, lens, rows, causal=True, scale=None, q_scale=1.0, seed=0, k_scale=1.0,
            shift=0.0, **kw):
    dtype = DTYPES[dt]
    held = cache(lens, Hkv, D, bs, dtype, seed, k_scale, shift)
    q = rand(sum(rows), H, D, dtype=dtype, scale=q_scale, seed=seed + 1)
    got, cu = run(q, held, lens, rows, causal, scale, **kw)
    ref, mass, reach = attention(q, *held[:4], cu, lens, held[4], scale, causal)
    tiles = H // Hkv * max(max(rows), kw.get("most_q") or 0, -(-(sum(rows) + kw.get("extra", 0)) // len(rows))) > 64
    check(got, ref, bound(ref, mass, reach, dtype, tiles), f"{lens} {rows}")
    # over all rows the roundings add up as independent ones do
    off = float((got.cpu().double() - ref).norm() / ref.norm().clamp(min=1e-30))
    assert off < 1.5 * HALF_STEP[dtype] + (6 if tiles else 2) * 2.0 ** -11, off
    return got


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D,bs,lens", [
    (32, 8, 128, 16, [1]), (32, 8, 128, 16, [777]), (4, 4, 128, 32, [5, 0, 130, 33]),
    (8, 1, 64, 24, [300, 17]), (16, 2, 96, 16, [100, 511, 64]), (6, 2, 192, 64, [1000]),
    (10, 2, 160, 4, [77, 260]), (16, 8, 32, 7, [63, 200]), (40, 8, 128, 1, [90]),
    (64, 8, 128, 16, [129, 2049]), (20, 1, 128, 48, [400, 31]), (64, 1, 128, 16, [333])])
def test_single_tokens(H, Hkv, D, bs, lens, dt):
    compare(dt, H, Hkv, D, bs, lens, [1] * len(lens))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D,bs,lens,rows", [
    (32, 8, 128, 16, [200, 5, 40], [4, 5, 1]),      # a few rows each
    (32, 8, 128, 16, [500], [9]),                   # two tiles of columns
    (16, 4, 64, 16, [64, 90], [16, 0]),
    (16, 2, 128, 24, [70, 3], [3, 8]),              # more rows than keys
    (8, 2, 128, 16, [333, 40], [100, 40]),          # query tiles
    (8, 2, 96, 32, [150], [150]), (6, 2, 64, 24, [97], [65]), (3, 3, 192, 16, [140], [70]),
    (4, 1, 160, 16, [90], [33]), (8, 8, 32, 5, [130], [100]), (5, 1, 128, 1, [60], [60]),
    (4, 2, 128, 16, [1300], [1200]), (2, 1, 192, 16, [1100], [1090])])
@pytest.mark.parametrize("causal", [True, False])
def test_several_rows(H, Hkv, D, bs, lens, rows, causal, dt):
    compare(dt, H, Hkv, D, bs, lens, rows, causal)


@pytest.mark.parametrize("rows", [[1, 1, 1], [3, 0, 7], [70, 1, 20]])
@pytest.mark.parametrize("most_q,most_k", [(None, 100000), (1, None), (None, 1), (0, 0), (500, 64)])
def test_bounds_shape_the_launch_alone(rows, most_q, most_k):
    compare("f16", 8, 2, 128, 16, [300, 0, 1100], rows, most_q=most_q, most_k=most_k)


@pytest.mark.parametrize("rows", [[1, 0, 1], [80, 0, 3]])
def test_padding_rows_are_zero(rows):
    compare("bf16", 8, 2, 128, 16, [100, 30, 0], rows, extra=5)


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("dt,q_scale,k_scale,shift", [
    ("f16", 1.0, 1.0, 40.0),       # rows far from zero
    ("f16", 20.0, 4.0, 0.0),       # sharp: scores of hundreds
    ("f16", 1.0, 2.0 ** -12, 0.0),  # values in fp16's small exponents
    ("f16", 2.0 ** -3, 8000.0, 0.0),
    ("bf16", 1e-20, 1e20, 0.0), ("bf16", 1e10, 1e-12, 0.0), ("bf16", 1.0, 1e-30, 0.0),
    ("bf16", 1.0, 1.0, -100.0)])
def test_ranges(dt, q_scale, k_scale, shift, rows):
    compare(dt, 4, 2, 128, 16, [200], [rows], q_scale=q_scale, k_scale=k_scale, shift=shift)


def test_scores_far_below_zero():
    """Every score negative and large: the softmax is of their differences."""
    held = cache([50], 1, 64, 16, torch.float16, shift=3.0)
    for rows in (1, 70):
        q = -rand(rows, 1, 64, scale=0.3).abs() * 60
        got, cu = run(q, held, [50], [rows], causal=False)
        ref, mass, reach = attention(q, *held[:4], cu, [50], held[4], None, False)
        assert float((ref.abs().amax())) > 0.1
        check(got, ref, bound(ref, mass, reach, torch.float16, rows > 1), "far")


@pytest.mark.parametrize("rows", [1, 70])
def test_nan_rows_reach_their_columns_only(rows):
    """A visible NaN row makes the rows that see it NaN; a hidden one nothing."""
    lens, D = [200, 90], 128
    held = list(cache(lens, 2, D, 16, torch.bfloat16))
    held[2][held[4][0, 12], 0, 3] = math.nan  # key 195 of kv head 0
    q = rand(2 * rows, 4, D, dtype=torch.bfloat16)
    got, cu = run(q, held, lens, [rows, rows])
    seen = torch.zeros(2 * rows, 4, dtype=torch.bool)
    for r in range(rows):
        seen[r, :2] = 200 - rows + r >= 195
    assert torch.equal(torch.isnan(got.cpu()).all(-1), seen)
    assert torch.equal(torch.isnan(got.cpu()).any(-1), seen)


@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("rows,G", [(1, 4), (3, 1), (3, 4), (9, 2), (14, 1), (14, 4), (70, 4)])
def test_nan_rows_of_keys_and_values(rows, G, which):
    """The same for keys and values, where rows share a tile of columns (held in one or
    several copies), and for more of them."""
    lens, D = [200, 90], 128
    held = list(cache(lens, 2, D, 16, torch.float16))
    held[which][held[4][0, 12], 0, 6] = math.nan  # row 198 of kv head 0
    q = rand(2 * rows, 2 * G, D, dtype=torch.float16)
    got, cu = run(q, held, lens, [rows, rows])
    seen = torch.zeros(2 * rows, 2 * G, dtype=torch.bool)
    for r in range(rows):
        seen[r, :G] = 200 - rows + r >= 198
    assert torch.equal(torch.isnan(got.cpu()).all(-1), seen)
    assert torch.equal(torch.isnan(got.cpu()).any(-1), seen)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192])
@pytest.mark.parametrize("G,rows", [(1, 1), (2, 1), (4, 1), (3, 1), (8, 1), (5, 1), (12, 1), (16, 1),
                                    (1, 3), (2, 4), (1, 17), (4, 9)])
@pytest.mark.parametrize("bs", [16, 48, 20])
def test_columns_of_every_number(G, rows, bs, D, dt):
    """Columns that are held once, twice and four times, one and two tiles of them, in
    pages of whole halves of a block and others, at keys that end inside blocks."""
    compare(dt, 2 * G, 2, D, bs, [37, 129 + 16 * G, 260], [rows] * 3)


def test_long_context_of_small_weights():
    """Many keys of equal weight: none may be lost to fp16's range."""
    S, D = 40000, 64
    n, pair = quantised(rand(S // 16, 1, 16, D, dtype=torch.float16, seed=4) * 0.0 + 1.0)
    kc, ks = pack(n), pair
    vn, vs = quantised(torch.ones(S // 16, 1, 16, D, dtype=torch.float16)
                       + rand(S // 16, 1, 16, D, dtype=torch.float16, scale=0.01, seed=5))
    table = torch.arange(S // 16, dtype=torch.int32)[None]
    ks[0, 0, 0, 1] = 3.0  # one key far ahead of all others
    held = (kc, pack(vn), ks, vs, table)
    q = torch.full((1, 1, D), 0.9, dtype=torch.float16)
    got, cu = run(q, held, [S], [1])
    ref, mass, reach = attention(q, *held[:4], cu, [S], table)
    check(got, ref, bound(ref, mass, reach, torch.float16, False), "long")


def test_far_pages():
    """Offsets past 2^31 bytes into the cache."""
    H, Hkv, D, bs = 4, 1, 128, 16
    NB = (1 << 31) // (bs * D // 2) + 64
    held = cache([100], Hkv, D, bs, torch.float16)
    kc = torch.zeros(NB, Hkv, bs, D // 2, dtype=torch.uint8, device="cuda")
    vc = torch.zeros_like(kc)
    ks = torch.zeros(NB, Hkv, bs, 2, dtype=torch.float16, device="cuda")
    vs = torch.zeros_like(ks)
    need = 7
    far = torch.arange(NB - need, NB, dtype=torch.int32)
    src = held[4][0, :need].long()
    for dst, t in ((kc, held[0]), (vc, held[1]), (ks, held[2]), (vs, held[3])):
        dst[NB - need:] = t[src].cuda()
    for rows in (1, 40):
        q = rand(rows, H, D)
        out = torch.empty(rows, H, D, dtype=torch.float16, device="cuda")
        tecoops.flash_attn_varlen_int4(q.cuda(), kc, vc, ks, vs, rows,
                                       torch.tensor([0, rows], dtype=torch.int32).cuda(), 100,
                                       torch.tensor([100], dtype=torch.int32).cuda(), None, True,
                                       far[None].cuda(), out)
        want, _ = run(q, held, [100], [rows])
        assert torch.equal(out, want)


def test_captured_replayed_and_two_streams():
    lens, H, Hkv, D = [700, 90, 1500], 8, 2, 128
    held = [t.cuda() for t in cache(lens, Hkv, D, 16, torch.float16)]
    kc, vc, ks, vs, table = held
    q = rand(3, H, D).cuda()
    cu = torch.arange(4, dtype=torch.int32).cuda()
    used = torch.tensor(lens, dtype=torch.int32).cuda()
    out, other = torch.empty_like(q), torch.empty_like(q)

    def step(o):
        tecoops.flash_attn_varlen_int4(q, kc, vc, ks, vs, 1, cu, 1500, used, None, True, table, o)

    step(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out)
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        step(other)
    side = torch.cuda.Stream()
    for i in range(3):
        q.copy_(rand(3, H, D, seed=i).cuda())
        used.copy_(torch.tensor([x - 5 * i for x in lens], dtype=torch.int32))
        torch.cuda.synchronize()
        want = torch.empty_like(q)
        step(want)
        torch.cuda.synchronize()
        out.zero_(), other.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            second.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(other, want)
