"""Attention over the 4-bit cache by each of its routes: codes as they are (fp16, and
bf16 of few rows) and widened tiles (bf16 of many rows)."""
import pytest
import torch

import tecoops
from int4_reference import DTYPES, HALF_STEP, attention, check, rand
from test_gpu_attention_int4 import bound, cache, run

pytestmark = pytest.mark.gpu
MOST = (1 << 31) - 1


def widened(dtype, G, rows, most_q=None, extra=0):
    """Whether the call takes the widened tiles: bf16, more than 64 columns by the bound."""
    total = sum(rows) + extra
    most = max(rows) if most_q is None else most_q
    return dtype == torch.bfloat16 and G * min(max(most, -(-total // len(rows))), total) > 64


def compare(dt, H, Hkv, D, bs, lens, rows, causal=True, most_q=None, most_k=None, seed=0):
    dtype = DTYPES[dt]
    held = cache(lens, Hkv, D, bs, dtype, seed)
    q = rand(sum(rows), H, D, dtype=dtype, seed=seed + 1)
    got, cu = run(q, held, lens, rows, causal, most_q=most_q, most_k=most_k)
    ref, mass, reach = attention(q, *held[:4], cu, lens, held[4], None, causal)
    tiles = widened(dtype, H // Hkv, rows, most_q)
    check(got, ref, bound(ref, mass, reach, dtype, tiles), f"{lens} {rows} {most_q} {most_k}")
    return got, ref


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [[1, 1, 1], [3, 0, 7], [70, 1, 20], [300, 10, 10]])
@pytest.mark.parametrize("most_q,most_k", [(None, None), (1, None), (0, 0), (500, 64), (None, MOST), (8192, None),
                                           (131072, 100000), (MOST, None), (MOST, MOST), (-1, 1)])
def test_bounds_shape_the_launch_alone(rows, most_q, most_k, dt):
    compare(dt, 8, 2, 128, 16, [300, 0, 1100], rows, most_q=most_q, most_k=most_k)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_more_tiles_than_a_grid_has(dt):
    """65536 sequences of one row and one of 3000, with no bound on them: each workgroup
    goes on to further tiles of the long one."""
    dtype, D, bs, B, L, at = DTYPES[dt], 32, 16, 65536, 3000, 40000
    held = cache([40], 1, D, bs, dtype)
    kc, vc, ks, vs, pages = [t.cuda() for t in held]
    lens = torch.full((B,), 20, dtype=torch.int32)
    lens[at] = 40
    cu = torch.arange(B + 1, dtype=torch.int32)
    cu[at + 1:] += L - 1
    q = rand(B + L - 1, 1, D, dtype=dtype)
    out = torch.full_like(q, 5.0).cuda()
    tecoops.flash_attn_varlen_int4(q.cuda(), kc, vc, ks, vs, MOST, cu.cuda(), 40, lens.cuda(), None, True,
                                   pages.expand(B, -1).contiguous(), out)
    pick = [0, 1, at, at + 1, B - 1]
    some = torch.cat([q[cu[b]:cu[b + 1]] for b in pick])
    got = torch.cat([out[cu[b]:cu[b + 1]] for b in pick])
    offs = [0, 1, 2, 2 + L, 3 + L, 4 + L]
    ref, mass, reach = attention(some, *held[:4], offs, [int(lens[b]) for b in pick], held[4].expand(5, -1))
    check(got, ref, bound(ref, mass, reach, dtype, dtype == torch.bfloat16), "picked")
    assert torch.isfinite(out).all()


def test_more_columns_than_a_grid_has():
    """One sequence of more rows than 65535 tiles of columns hold."""
    D, L = 32, 65535 * 384 + 5000
    held = cache([16], 1, D, 16, torch.bfloat16)
    kc, vc, ks, vs, pages = [t.cuda() for t in held]
    q = torch.randn(L, 1, D, generator=torch.Generator("cuda").manual_seed(1), device="cuda", dtype=torch.bfloat16)
    out = torch.full_like(q, 5.0)
    tecoops.flash_attn_varlen_int4(q, kc, vc, ks, vs, L, torch.tensor([0, L], dtype=torch.int32).cuda(), 16,
                                   torch.tensor([16], dtype=torch.int32).cuda(), None, False, pages, out)
    some = torch.cat([torch.arange(0, 500), torch.arange(L // 2, L // 2 + 500), torch.arange(L - 5500, L)])
    ref, mass, reach = attention(q[some.cuda()].cpu(), *held[:4], [0, len(some)], [16], held[4], None, False)
    check(out[some.cuda()], ref, bound(ref, mass, reach, torch.bfloat16, True), "picked")
    assert torch.isfinite(out).all() and float(out.float().abs().max()) < 5.0
