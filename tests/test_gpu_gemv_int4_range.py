"""Products with 4-bit weights of x that is infinite or close to the largest number:
what an offset of the codes overflows is still what the formula gives.

Bound: that of the products at large (test_gpu_gemv_int4.bound).  The codes' sums carry
an offset of up to 1024 that the sums of x take off again, each rounded by 2^-24 of its
partial sums; so an x of 2.4e36 whose weight is 0 and whose multiples are still finite
leaves 2^-24 * 143 * 2.4e36 * scale in the output, whatever its weight: the error is
relative to sum |x| scale, not to sum |x| |W|.  Where the sums are not finite the
products are summed one by one, which is closer (2^-24 (K / 64 + 8) of sum |x| |W|,
with |W| at most 15 scales: 2^-24 * 15 * 264 < 2^-24 * 4 * 1040 for K up to 16384)."""
import math

import pytest
import torch

import tecoops
from int4_reference import DTYPES, check, pack, rand, weights
from test_gpu_gemv_int4 import bound

pytestmark = pytest.mark.gpu

# rows of x, n, k, group: one row over a short K, one over a long K, parts of K, tiles of
# every number of rows of x, a K that ends inside a stage
SIZES = [(1, 40, 512, 128), (1, 300, 4096, 64), (1, 48, 14336, 128), (2, 70, 256, 64), (9, 33, 1088, 32),
         (33, 64, 14336, 128), (64, 20, 4160, 160), (70, 130, 512, 64)]


def compare(x, n, group, zeros, seed):
    b, k = x.shape
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (n, k), generator=g)
    scales = ((torch.rand(n, k // group, generator=g) + 0.5) * 0.05).to(x.dtype)
    z = (torch.rand(n, k // group, generator=g) * 4 + 5.5).to(x.dtype) if zeros else None
    out = torch.full((b, n), 7.0, dtype=x.dtype, device="cuda")
    tecoops.gemv_int4(pack(codes).cuda(), scales.cuda(), x.cuda(), out, zeros=None if z is None else z.cuda())
    w = weights(codes, scales, z, group)
    ref = x.double() @ w.t()
    got = out.cpu().double()
    ends = torch.isinf(ref)
    assert torch.equal(got[ends], ref[ends])
    check(got, ref, bound(x, codes, scales, z, group, ref, x.dtype), f"{b} {n} {k} {group}")


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("b,n,k,group", SIZES)
def test_infinities(b, n, k, group, zeros, dt):
    """One infinite element of a row: infinite outputs, NaN where its weight is 0."""
    x = rand(b, k, dtype=DTYPES[dt], seed=b + k)
    x[0, k // 3] = math.inf
    x[b - 1, k - 1] = -math.inf
    compare(x, n, group, zeros, n)


@pytest.mark.parametrize("b,n,k,group", SIZES)
@pytest.mark.parametrize("big", [2.4e36, 3e37, -1e38])
def test_large_finite_rows(b, n, k, group, big):
    """A finite x whose multiple by a code under an exponent is not."""
    x = rand(b, k, dtype=torch.bfloat16, seed=b + k)
    x[0, k // 5] = big
    x[b - 1, 7] = big
    compare(x, n, group, True, n)


def test_rows_beside_one_that_is_none():
    """NaN and infinite rows of x leave the others what they are."""
    b, n, k, group = 20, 80, 1024, 64
    x = rand(b, k, dtype=torch.bfloat16, seed=1)
    x[3, 5], x[17, 900], x[9] = math.nan, math.inf, math.nan
    compare(x, n, group, False, 2)


@pytest.mark.parametrize("b", [1, 2])
def test_groups_of_a_very_long_row(b):
    """The last groups of a K of 2 * 10^8: x is 0 but there."""
    n, group, k, used = 2, 96, 201332160, 5472
    dtype, far = torch.float16, k - 5472
    g = torch.Generator().manual_seed(3)
    w = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.ones(n, k // group, dtype=dtype, device="cuda")
    x = torch.zeros(b, k, dtype=dtype, device="cuda")
    codes = torch.randint(0, 16, (n, used), generator=g)
    tail = ((torch.rand(n, used // group, generator=g) + 0.5) * 0.1).to(dtype)
    xt = rand(b, used, dtype=dtype, seed=4)
    w[:, far // 2:], scales[:, far // group:], x[:, far:] = pack(codes).cuda(), tail.cuda(), xt.cuda()
    out = torch.empty(b, n, dtype=dtype, device="cuda")
    tecoops.gemv_int4(w, scales, x, out)
    ref = xt.double() @ weights(codes, tail, None, group).t()
    check(out, ref, bound(xt, codes, tail, None, group, ref, dtype), "the end of a long row")
