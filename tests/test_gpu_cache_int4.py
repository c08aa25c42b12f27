"""Keys and values stored in 4 bits: codes and pairs equal to the definition's."""
import math

import pytest
import torch

import tecoops
from int4_reference import DTYPES, pack, quantised, rand

pytestmark = pytest.mark.gpu


def run(key, value, slots, NB, bs, rows=None):
    T, H, D = key.shape
    kc = torch.full((NB, H, bs, D // 2), 0xA5, dtype=torch.uint8, device="cuda")
    ks = torch.full((NB, H, bs, 2), 3.0, dtype=key.dtype, device="cuda")
    vc, vs = kc.clone(), ks.clone()
    k, v = (key.cuda(), value.cuda()) if rows is None else rows
    tecoops.reshape_and_cache_int4(k, v, slots.cuda(), kc, vc, ks, vs)
    return [t.cpu() for t in (kc, vc, ks, vs)]


def expected(x, slots, NB, bs):
    T, H, D = x.shape
    held = torch.full((NB, H, bs, D // 2), 0xA5, dtype=torch.uint8)
    pairs = torch.full((NB, H, bs, 2), 3.0, dtype=x.dtype)
    n, pair = quantised(x)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < NB * bs:
            held[s // bs, :, s % bs], pairs[s // bs, :, s % bs] = pack(n[t]), pair[t]
    return held, pairs


def same(got, want):
    assert torch.equal(got[0], want[0]), "codes"
    a, b = got[1].view(torch.int16), want[1].view(torch.int16)
    nan = torch.isnan(want[1])
    assert torch.equal(torch.isnan(got[1]), nan) and torch.equal(a[~nan], b[~nan]), "pairs"


def slots_of(T, NB, bs, seed=0):
    return torch.randperm(NB * bs, generator=torch.Generator().manual_seed(seed))[:T]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("T,H,D,bs", [(1, 1, 8, 16), (3, 8, 128, 16), (65, 2, 64, 24), (33, 5, 96, 1),
                                      (17, 3, 192, 7), (9, 2, 256, 32), (5, 1, 512, 16),
                                      (700, 8, 128, 64), (4, 3, 24, 16)])
def test_store(T, H, D, bs, dt):
    NB = (T + bs - 1) // bs + 2
    key, value = rand(T, H, D, dtype=DTYPES[dt], seed=T), rand(T, H, D, dtype=DTYPES[dt], scale=9, seed=D)
    slots = slots_of(T, NB, bs)
    if T > 2:
        slots[1], slots[2] = -1, NB * bs
    got = run(key, value, slots, NB, bs)
    same((got[0], got[2]), expected(key, slots, NB, bs))
    same((got[1], got[3]), expected(value, slots, NB, bs))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("off", [0, 8, 1])
def test_rows_of_a_wider_product(dt, off):
    T, H, D, bs, NB = 21, 3, 64, 16, 4
    flat = rand(T * (2 * H * D + 40) + 64, dtype=DTYPES[dt])
    dev = flat.cuda()
    views = []
    for t in (flat, dev):
        w = t[off:off + T * (2 * H * D + 40)].view(T, -1)
        views.append([w[:, i:i + H * D].view(T, H, D) for i in (0, H * D)])
    slots = slots_of(T, NB, bs)
    got = run(*views[0], slots, NB, bs, rows=views[1])
    same((got[0], got[2]), expected(views[0][0], slots, NB, bs))
    same((got[1], got[3]), expected(views[0][1], slots, NB, bs))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_rows_of_special_values(dt):
    """Equal elements, ties between codes, tiny and wide ranges, infinities, NaN."""
    dtype, D, bs, NB = DTYPES[dt], 64, 16, 2
    x = rand(16, 1, D, dtype=dtype)
    x[0] = 0
    x[1] = 3.5
    x[2] = (torch.arange(D) % 31).to(dtype) * 0.5   # scale 1: halves are ties
    x[3] = (torch.arange(D) % 61).to(dtype) * 0.25
    x[4] = torch.finfo(dtype).tiny * (torch.arange(D) % 5).to(dtype)
    x[5] = torch.finfo(dtype).smallest_normal / 128 * (torch.arange(D) % 2).to(dtype)
    x[6, 0, ::2], x[6, 0, 1::2] = torch.finfo(dtype).max, torch.finfo(dtype).min
    x[7, 0, 9] = math.inf
    x[8, 0, 9] = -math.inf
    x[9, 0, 40] = math.nan
    x[10] = math.inf
    x[11] = -x[2]
    x[12, 0, 0] = 60000.0
    x[13, 0, D - 1] = math.nan
    x[14] = -0.0
    slots = slots_of(16, NB, bs)
    got = run(x, x.flip(0), slots, NB, bs)
    same((got[0], got[2]), expected(x, slots, NB, bs))
    same((got[1], got[3]), expected(x.flip(0), slots, NB, bs))


def test_captured_and_replayed():
    T, H, D, bs, NB = 8, 2, 128, 16, 2
    key, slots = rand(T, H, D).cuda(), slots_of(T, NB, bs).cuda()
    kc = torch.zeros(NB, H, bs, D // 2, dtype=torch.uint8, device="cuda")
    ks = torch.zeros(NB, H, bs, 2, dtype=torch.float16, device="cuda")
    vc, vs = kc.clone(), ks.clone()
    tecoops.reshape_and_cache_int4(key, key, slots, kc, vc, ks, vs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tecoops.reshape_and_cache_int4(key, key, slots, kc, vc, ks, vs)
    for i in range(3):
        key.copy_(rand(T, H, D, seed=i + 1).cuda())
        kc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        same((kc.cpu(), ks.cpu()), [torch.where(torch.zeros(1, dtype=torch.bool), a, a) for a in
                                    _zeroed(expected(key.cpu(), slots.cpu(), NB, bs), slots.cpu(), bs)])


def _zeroed(want, slots, bs):
    """Rows that no token was stored in hold the zeros that were there."""
    used = torch.zeros(want[0].shape[0] * bs, dtype=torch.bool)
    used[slots] = True
    used = used.view(-1, 1, bs, 1)
    return [torch.where(used, t, torch.zeros_like(t)) for t in want]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("low", [0.0, -7.0])
def test_values_at_the_middle_of_two_codes(dt, low):
    """Middles of codes and their neighbours, at scales from the smallest on: the
    codes are those of the quotients, ties to even."""
    T, D, bs, NB = 96, 128, 16, 8
    dtype = DTYPES[dt]
    tiny, huge = (-24, 11) if dt == "f16" else (-133, 123)
    unit = torch.logspace(0, 1, T, base=2, dtype=torch.float64).mul(
        torch.pow(2.0, torch.linspace(tiny, huge, T, dtype=torch.float64).floor())).to(dtype).double()
    middle = torch.cat([torch.arange(0, 15) + 0.5, torch.arange(0, 16)]).double()
    x = (unit[:, None] * (middle + low)[None]).to(dtype)  # [T, 31]
    bits = x.view(torch.int16)
    row = torch.cat([x, (bits + 1).view(dtype), (bits - (bits & 0x7fff).clamp(max=1)).view(dtype), x], 1)
    row = torch.where(torch.isfinite(row), row, torch.zeros_like(row))
    key = torch.cat([row, row[:, :4]], 1).view(T, 1, D)
    value = key.flip(0).contiguous()
    slots = slots_of(T, NB, bs)
    got = run(key, value, slots, NB, bs)
    same((got[0], got[2]), expected(key, slots, NB, bs))
    same((got[1], got[3]), expected(value, slots, NB, bs))
