"""Norms of queries and keys with the rotation, against the formulas in 64 bits."""
import math

import pytest
import torch

import tecoops
from int4_reference import DTYPES, HALF_STEP, SMALLEST, check, norm_rotary, rand

pytestmark = pytest.mark.gpu
EPS = 1e-6


def angles(positions, rot, base):
    a = positions.double()[:, None] * base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return a.cos(), a.sin()


def bound(ref, size, dtype):
    # one rounding to the type; in fp32 a sum of squares (2^-18 for up to 1024
    # elements), a reciprocal root, four products and an angle: 2^-17 of the terms
    return HALF_STEP[dtype] * ref.abs() + 2.0 ** -17 * size + SMALLEST[dtype]


# tokens, heads, kv heads, head, rot, neox
CASES = [(1, 1, 1, 64, 64, True), (5, 32, 8, 128, 128, True), (3, 4, 2, 128, 64, True),
         (7, 3, 1, 80, 80, True), (4, 16, 4, 96, 32, False), (2, 8, 1, 256, 256, True),
         (2, 5, 5, 192, 192, True), (3, 2, 2, 512, 128, False), (2, 3, 1, 40, 24, True),
         (2, 2, 1, 20, 12, False), (1, 1, 1, 1024, 512, True), (3, 2, 1, 33, 2, True),
         (700, 9, 3, 128, 128, False), (2, 6, 2, 8, 8, False), (3, 2, 1, 600, 512, True)]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("T,H,Hkv,D,rot,neox", CASES)
def test_in_place(T, H, Hkv, D, rot, neox, dt):
    dtype = DTYPES[dt]
    qkv = rand(T, (H + 2 * Hkv) * D, dtype=dtype, scale=3.0, seed=T + D)
    qw, kw = rand(D, dtype=dtype, seed=1) + 1, rand(D, dtype=dtype, seed=2) + 1
    pos = torch.randint(0, 300000, (T,), generator=torch.Generator().manual_seed(3))
    dev = qkv.cuda()
    q, k, v = dev.split([H * D, Hkv * D, Hkv * D], 1)
    tecoops.qk_norm_rotary(pos.cuda(), q, k, qw.cuda(), kw.cuda(), D, eps=EPS, base=1e6, rot_dim=rot,
                           is_neox=neox)
    cos, sin = angles(pos, rot, float(torch.tensor(1e6)))
    for got, n0, n, w in ((q, 0, H, qw), (k, H, Hkv, kw)):
        x = qkv[:, n0 * D:(n0 + n) * D].view(T, n, D)
        ref, size = norm_rotary(x, w, EPS, cos, sin, rot, neox)
        check(got.reshape(T, n, D), ref, bound(ref, size, dtype), f"{n} heads")
    assert torch.equal(v.cpu(), qkv[:, (H + Hkv) * D:])


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("bs", [16, 24, 1])
@pytest.mark.parametrize("write_key", [False, True])
def test_fused_store_is_both_calls(odd, neox, bs, write_key):
    """Bit-identical to the call in place and reshape_and_cache, for rows aligned or
    not, with tokens of no slot or outside the table left out or as they are."""
    T, H, Hkv, D, rot, NB = 13, 8, 2, 128, 128, 40
    dtype, off = torch.bfloat16, 1 if odd else 0
    flat = rand(T * (H + 2 * Hkv) * D + 1, dtype=dtype, scale=2.0).cuda()
    qw, kw = (rand(D, dtype=dtype, seed=5) + 1).cuda(), (rand(D, dtype=dtype, seed=6) + 1).cuda()
    cos, sin = angles(torch.arange(100), rot, 1e4)
    table = torch.cat([cos, sin], 1).float().cuda()
    pos = torch.arange(T) * 7 % 100
    pos[4], pos[9] = 100, -1
    slots = torch.randperm(NB * bs, generator=torch.Generator().manual_seed(1))[:T]
    slots[2], slots[9], slots[11] = -1, NB * bs + 3, -5

    def rows():
        x = flat.clone()[off:off + T * (H + 2 * Hkv) * D].view(T, -1)
        return x.split([H * D, Hkv * D, Hkv * D], 1)

    q1, k1, v1 = rows()
    tecoops.qk_norm_rotary(pos.cuda(), q1, k1, qw, kw, D, cos_sin_cache=table, is_neox=neox)
    kc1 = torch.full((NB, Hkv, bs, D), 7.0, dtype=dtype, device="cuda")
    vc1 = kc1.clone()
    tecoops.reshape_and_cache(k1.reshape(T, Hkv, D).contiguous(), v1.reshape(T, Hkv, D).contiguous(),
                              slots.cuda(), kc1, vc1)
    q2, k2, v2 = rows()
    before = k2.clone()
    kc2, vc2 = torch.full_like(kc1, 7.0), torch.full_like(kc1, 7.0)
    tecoops.qk_norm_rotary_reshape_and_cache(pos.cuda(), q2, k2, v2, qw, kw, slots.cuda(), kc2, vc2, D,
                                             cos_sin_cache=table, is_neox=neox, write_key=write_key)
    assert torch.equal(q1, q2) and torch.equal(kc1, kc2) and torch.equal(vc1, vc2)
    assert torch.equal(k2, k1 if write_key else before) and torch.equal(v1, v2)
    raw = rows()
    for t in (4, 9):  # outside the table
        assert torch.equal(q2[t], raw[0][t])


def test_axes_and_no_key():
    """Positions of several axes turn as rotary_embedding_axes turns the normalised
    rows; a query alone."""
    T, H, D, sections = 50, 4, 128, [16, 24, 24]
    x = rand(T, H * D, dtype=torch.float16, scale=2.0, seed=9)
    w = rand(D, dtype=torch.float16, seed=1) + 1
    pos = torch.randint(0, 5000, (3, T), generator=torch.Generator().manual_seed(3))
    q = x.cuda()
    tecoops.qk_norm_rotary(pos.cuda(), q, None, w.cuda(), None, D, sections=sections, eps=1e-5)
    axis = torch.tensor([0] * 16 + [1] * 24 + [2] * 24)
    a = pos[axis].t().double() * 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    ref, size = norm_rotary(x.view(T, H, D), w, 1e-5, a.cos(), a.sin(), D, True)
    check(q.view(T, H, D), ref, bound(ref, size, torch.float16), "axes")


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_zero_small_and_infinite_rows(dt):
    dtype, D = DTYPES[dt], 128
    x = rand(4, 2 * D, dtype=dtype)
    x[0] = 0
    x[1] *= 2.0 ** -12  # eps decides
    x[2, 5] = math.nan
    x[3] *= 2.0 ** 12
    w = rand(D, dtype=dtype, seed=1) + 1
    pos = torch.arange(4)
    q = x.cuda()
    tecoops.qk_norm_rotary(pos.cuda(), q, None, w.cuda(), None, D)
    cos, sin = angles(pos, D, 1e4)
    ref, size = norm_rotary(x.view(4, 2, D), w, EPS, cos, sin, D, True)
    check(q.view(4, 2, D), ref, bound(ref, size, dtype), "rows")


def test_captured_and_replayed():
    T, H, D = 4, 8, 128
    w = (rand(D, dtype=torch.float16, seed=1) + 1).cuda()
    src, q = rand(T, H * D).cuda(), torch.empty(T, H * D, dtype=torch.float16, device="cuda")
    pos = torch.arange(T).cuda()

    def step():
        q.copy_(src)
        tecoops.qk_norm_rotary(pos, q, None, w, None, D)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        src.copy_(rand(T, H * D, seed=i).cuda())
        step()
        want = q.clone()
        q.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, want)
