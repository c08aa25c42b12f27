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


@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("rows,G,keys", [(3, 4, 200), (70, 1, 200), (70, 4, 200), (20, 4, 1500), (150, 4, 200)])
def test_nan_rows_reach_the_rows_that_see_them(rows, G, keys, dt, which):
    """NaN rows of keys and of values, one seen by the last rows alone, in either route,
    in tiles of four waves and of twelve, in one split and in several."""
    lens, hidden = [keys, 90], keys - 2
    held = list(cache(lens, 2, 128, 16, DTYPES[dt]))
    held[which][held[4][0, hidden // 16], 0, hidden % 16] = float("nan")
    q = rand(2 * rows, 2 * G, 128, dtype=DTYPES[dt])
    got, cu = run(q, held, lens, [rows, rows])
    seen = torch.zeros(2 * rows, 2 * G, dtype=torch.bool)
    for r in range(rows):
        seen[r, :G] = keys - rows + r >= hidden
    assert torch.equal(torch.isnan(got.cpu()).all(-1), seen)
    assert torch.equal(torch.isnan(got.cpu()).any(-1), seen)
    # and the others are what they are without it
    held[which][held[4][0, hidden // 16], 0, hidden % 16] = 0.0
    ref, mass, reach = attention(q, *held[:4], cu, lens, held[4])
    fine = ~seen
    check(got.cpu()[fine], ref[fine], bound(ref, mass, reach, DTYPES[dt], widened(DTYPES[dt], G, [rows] * 2))[fine],
          "others")


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 40, 100])
def test_far_pages(rows, dt):
    """Offsets past 2^31 bytes into the cache and 2^32 into its rows, in either route."""
    H, D, bs, need = 4, 128, 16, 7
    NB = (1 << 32) // (bs * D // 2) + 64
    held = cache([100], 1, D, bs, DTYPES[dt])
    far = torch.arange(NB - need, NB, dtype=torch.int32)
    dev = []
    for t in held[:4]:
        whole = torch.zeros(NB, *t.shape[1:], dtype=t.dtype, device="cuda")
        whole[NB - need:] = t[held[4][0, :need].long()].cuda()
        dev.append(whole)
    q = rand(rows, H, D, dtype=DTYPES[dt])
    out = torch.empty_like(q, device="cuda")
    tecoops.flash_attn_varlen_int4(q.cuda(), *dev, rows, torch.tensor([0, rows], dtype=torch.int32).cuda(), 100,
                                   torch.tensor([100], dtype=torch.int32).cuda(), None, True, far[None].cuda(), out)
    want, _ = run(q, held, [100], [rows])
    assert torch.equal(out, want)


def off_of(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


def rounded_weights(q, held, S, one_term):
    """What a form with fewer bits gives in fp16: the weights times the scales in one fp16
    term, or (else) keys, values and weights in fp16."""
    from int4_reference import rows_of
    kc, vc, ks, vs, table = held
    out = torch.zeros(q.shape, dtype=torch.float64)
    rows, G = q.shape[0], q.shape[1] // kc.shape[1]
    seen = torch.arange(S)[None] <= S - rows + torch.arange(rows)[:, None]
    for h in range(q.shape[1]):
        K, V = rows_of(kc, ks, table[0], S, h // G), rows_of(vc, vs, table[0], S, h // G)
        if not one_term:
            K, V = K.half().double(), V.half().double()
        s = (q[:, h].double() @ K.t() * q.shape[2] ** -0.5).masked_fill(~seen, -float("inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        if one_term:
            j = torch.arange(S)
            pair = vs[table[0].long()[j // 16], h // G, j % 16].double()
            scale, middle = pair[:, 0], pair[:, 1] + 7.5 * pair[:, 0]
            w = (p * scale * 1024).half().double() / 1024
            out[:, h] = w @ ((V - middle[:, None]) / scale[:, None]) + p @ middle[:, None]
        else:
            out[:, h] = (p.half().double() @ V)
        out[:, h] /= p.sum(-1, keepdim=True)
    return out.half()


@pytest.mark.parametrize("H,S,rows", [(8, 40, 1), (32, 60, 1), (8, 50, 6), (8, 60, 40), (16, 64, 64)])
def test_fp16_is_as_close_as_its_output(H, S, rows):
    """fp16 over exact codes, with weights in two terms: off by the rounding of the output
    (its rms error from the reference alone) and little else.  Else is 2^-22 of each
    weight and some 2^-17 of fp32, relative to sums of magnitudes that are up to 8 times
    an output of 64 keys of random signs: 2^-14 at most beside a rounding of some 2^-12.3
    (sqrt(1 + 2^-3.4) = 1.05), were those to add up: 1.08 is allowed.  Weights in one term
    are off by 1.15 times that rounding or more, widened keys and values by 1.6."""
    held = cache([S], 2, 128, 16, torch.float16, seed=S)
    q = rand(rows, H, 128, dtype=torch.float16, seed=rows)
    got, cu = run(q, held, [S], [rows])
    ref, _, _ = attention(q, *held[:4], cu, [S], held[4])
    own = off_of(ref.half(), ref)
    assert off_of(rounded_weights(q, held, S, True), ref) > 1.13 * own
    assert off_of(rounded_weights(q, held, S, False), ref) > 1.5 * own
    assert off_of(got.cpu(), ref) < 1.08 * own


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hkv,D,bs,lens,rows", [
    (8, 2, 128, 16, [333, 40], [100, 40]), (8, 2, 96, 32, [150], [150]), (6, 2, 64, 24, [97], [65]),
    (3, 3, 192, 16, [140], [70]), (4, 1, 160, 16, [90], [33]), (8, 8, 32, 5, [130], [100]),
    (4, 2, 128, 16, [1300], [600]), (2, 1, 192, 16, [1100], [300])])
def test_fp16_of_many_rows(H, Hkv, D, bs, lens, rows, causal):
    """Held to the bound of exact codes, whatever the number of rows."""
    compare("f16", H, Hkv, D, bs, lens, rows, causal)
