"""Products with 4-bit weights against the formula in 64 bits."""
import math

import pytest
import torch

import tecoops
from int4_reference import DTYPES, HALF_STEP, SMALLEST, check, pack, rand, weights

pytestmark = pytest.mark.gpu


def make(n, k, group, zeros, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g)
    scales = ((torch.rand(n, k // group, generator=g) + 0.5) * 0.1).to(dtype)
    z = (torch.rand(n, k // group, generator=g) * 4 + 5.5).to(dtype) if zeros else None
    return codes, scales, z


def bound(x, codes, scales, zeros, group, ref, dtype):
    """One rounding, and sums in fp32: products of codes under an exponent (up to 1024
    + 15) and what takes it off again, 2^-24 of each partial sum; a lane or matrix
    instruction adds at most 32 at a time and a sum runs over at most 2^10 such."""
    size = (x.double().abs().view(*x.shape[:-1], -1, group).sum(-1) @ scales.double().abs().t()) * 1040
    return HALF_STEP[dtype] * ref.abs() + 2.0 ** -24 * 4 * size + SMALLEST[dtype]


def compare(b, n, k, group, zeros, dt, x=None, offset=0):
    dtype = DTYPES[dt]
    codes, scales, z = make(n, k, group, zeros, dtype, n + k)
    x = rand(b, k, dtype=dtype, seed=b) if x is None else x
    w = pack(codes).cuda()
    store = torch.empty(b * k + offset, dtype=dtype, device="cuda")
    xd = store[offset:].view(b, k)
    xd.copy_(x)
    out = torch.full((b, n), 7.0, dtype=dtype, device="cuda")
    tecoops.gemv_int4(w, scales.cuda(), xd, out, zeros=None if z is None else z.cuda())
    ref = x.double() @ weights(codes, scales, z, group).t()
    check(out, ref, bound(x, codes, scales, z, group, ref, dtype), f"{b} {n} {k} {group}")
    rel = float((out.cpu().double() - ref).norm() / ref.norm().clamp(min=1e-30))
    assert rel < HALF_STEP[dtype] + 2.0 ** -14, rel


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n,k,group", [(64, 128, 128), (1, 32, 32), (17, 96, 32), (33, 192, 64),
                                       (129, 1024, 256), (300, 4096, 128), (50, 160, 160),
                                       (16, 2048, 32), (95, 4480, 64), (1000, 512, 128)])
@pytest.mark.parametrize("b", [1, 2, 3, 5, 16])
def test_sizes(b, n, k, group, zeros, dt):
    compare(b, n, k, group, zeros, dt)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("b", [7, 8, 9, 17, 32, 33, 48, 64, 65, 130])
def test_batches(b, dt):
    compare(b, 130, 1088, 64, True, dt)


@pytest.mark.parametrize("b", [1, 2, 4, 20, 64])
def test_long_rows(b):
    """More of K than is staged at once."""
    compare(b, 40, 40960, 128, True, "bf16")
    compare(b, 24, 33344, 32, False, "f16")


@pytest.mark.parametrize("b", [1, 3, 16])
def test_x_off_16_byte_addresses(b):
    compare(b, 70, 256, 64, True, "f16", offset=1)
    compare(b, 70, 256, 64, True, "bf16", offset=4)


@pytest.mark.parametrize("b", [1, 4, 16])
def test_values(b):
    """Zero and large x, a column of one element; NaN stays in its row."""
    k, n, dtype = 512, 48, torch.float16
    x = rand(b, k, dtype=dtype)
    x[0] = 0
    x[-1] *= 1000.0
    compare(b, n, k, 128, True, "f16", x=x)
    one = torch.zeros(b, k, dtype=torch.bfloat16)
    one[:, 131] = 1e20
    compare(b, n, k, 128, False, "bf16", x=one)
    codes, scales, z = make(n, k, 128, True, dtype)
    x[0, 77] = math.nan
    out = torch.empty(b, n, dtype=dtype, device="cuda")
    tecoops.gemv_int4(pack(codes).cuda(), scales.cuda(), x.cuda(), out, zeros=z.cuda())
    assert torch.isnan(out[0]).all() and not torch.isnan(out[1:]).any()


def test_a_vector_and_no_rows():
    codes, scales, z = make(32, 64, 32, False, torch.float16)
    x, out = rand(64).cuda(), torch.empty(32, dtype=torch.float16, device="cuda")
    tecoops.gemv_int4(pack(codes).cuda(), scales.cuda(), x, out)
    two = torch.empty(1, 32, dtype=torch.float16, device="cuda")
    tecoops.gemv_int4(pack(codes).cuda(), scales.cuda(), x[None], two)
    assert torch.equal(out, two[0])
    tecoops.gemv_int4(pack(codes).cuda(), scales.cuda(), x[None][:0], two[:0])


@pytest.mark.parametrize("b", [1, 16])
def test_captured_and_replayed(b):
    codes, scales, z = make(64, 256, 64, True, torch.float16)
    w, s, zd = pack(codes).cuda(), scales.cuda(), z.cuda()
    x, out = rand(b, 256).cuda(), torch.empty(b, 64, dtype=torch.float16, device="cuda")
    tecoops.gemv_int4(w, s, x, out, zeros=zd)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tecoops.gemv_int4(w, s, x, out, zeros=zd)
    for i in range(3):
        x.copy_(rand(b, 256, seed=i + 5).cuda())
        want = torch.empty_like(out)
        tecoops.gemv_int4(w, s, x, want, zeros=zd)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
