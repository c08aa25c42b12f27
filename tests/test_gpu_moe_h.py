"""How the expert layer (tecoops.moe_layer) holds h, the operand of its second
product.  h keeps 16 bits of its mantissa in bf16 and 22 in fp16, so that the
result is off by its own rounding, which an h of the operands' type would double:
against 64 bits the bound has 2^-16 (fp16 2^-22) of each h, of independent signs
(within 4 times the root sum of squares of what they move: 7 standard deviations of
a uniform error) where one rounding to the type has 2^-8 (2^-11)."""
import math

import pytest
import torch

import tecoops

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
OF_H = {"f16": 2.0 ** -22, "bf16": 2.0 ** -16}


def weights64(logits, ids):
    top = logits.double().gather(1, ids.long())
    return torch.softmax(top, -1)


def layer64(x, w_in, w_out, ids, weights):
    """(out, root sum of squares of the terms w W h) in 64 bits."""
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    spread, inter = torch.zeros_like(out), w_out.shape[2]
    for e in sorted(set(ids.flatten().tolist())):
        t, j = (ids == e).nonzero(as_tuple=True)
        w = weights[t, j][:, None]
        y = x[t].double() @ w_in[e].double().t().contiguous()
        h = y[:, :inter] * torch.sigmoid(y[:, :inter]) * y[:, inter:]
        w2 = w_out[e].double().t().contiguous()
        out.index_add_(0, t, w * (h @ w2))
        spread.index_add_(0, t, w * w * ((h * h) @ (w2 * w2)))
    return out, spread.sqrt()


# every size of item and of rows per workgroup, the sum in the second product and in
# parts, widths outside 16-byte words, h far from 1 both ways
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -6, 2.0 ** 4])
@pytest.mark.parametrize("T,H,I,E,k", [(1, 512, 384, 8, 2), (3, 4096, 256, 4, 2), (4, 256, 1000, 16, 4),
                                       (7, 256, 200, 16, 4), (8, 4104, 136, 9, 4), (6, 64, 4096, 64, 8),
                                       (14, 192, 264, 32, 3), (60, 2048, 136, 8, 2), (130, 96, 72, 4, 2),
                                       (300, 520, 64, 4, 1), (520, 136, 40, 4, 2), (5, 45, 35, 4, 2)])
def test_result_is_off_by_its_own_rounding(T, H, I, E, k, scale, dtype):
    dt = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(T + H)

    def real(*shape, size=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * size).to(dt)

    x = real(T, H, size=scale)
    w_in, w_out = real(E, 2 * I, H, size=H ** -0.5), real(E, H, I, size=I ** -0.5)
    logits = torch.randn(T, E, generator=g, device="cuda")
    out, ids = torch.empty_like(x), torch.empty(T, k, dtype=torch.int32, device="cuda")
    tecoops.moe_layer(x, w_in, w_out, logits, k, out, topk_ids=ids)
    ref, spread = layer64(x, w_in, w_out, ids, weights64(logits, ids))
    half = torch.finfo(dt).eps / 2
    # The fp32 sums of both products, H + I terms in runs of 8 with roundings of
    # either sign; the activation, whose exponential is off by 2^-24 |v|; the softmax
    sums = ((H + I) / 8 + 60) * 2.0 ** -24
    bound = half * ref.abs() * 1.01 + (4.1 * OF_H[dtype] + 6 * sums) * spread
    bound += 20 * 2.0 ** -24 * ref.abs() + torch.finfo(dt).smallest_normal * half * 2
    # fp16's lo ends at 2^-27 (half of it, as above, I terms of weights of 1 / sqrt(I))
    bound += 0 if dtype == "bf16" else 4.1 * 2.0 ** -28 * w_out.float().abs().max().item() * math.sqrt(k * I)
    err = (out.double() - ref).abs()
    assert (err <= bound).all(), (err / bound).max().item()


@pytest.mark.parametrize("T", [1, 4, 7, 12, 40, 200])
@pytest.mark.parametrize("I", [64, 40, 33])
def test_h_past_the_range_of_fp16(T, I):
    """gate and up 2047 (up 4094 in one row of I: an h of 8380418): finite, and exact
    where the down weights keep the result within fp16."""
    H, E, dt = 32, 2, torch.float16
    x = torch.zeros(T, H, dtype=dt, device="cuda")
    x[:, 0], x[:, 1] = 2047, 4094
    w_in = torch.zeros(E, 2 * I, H, dtype=dt, device="cuda")
    w_in[:, :, 0] = 1
    w_in[:, 2 * I - 1, 0], w_in[:, 2 * I - 1, 1] = 0, 1
    w_out = torch.zeros(E, H, I, dtype=dt, device="cuda")
    w_out[:, 0, :2], w_out[:, 1, I - 1], w_out[:, 2, 3] = 2.0 ** -10, -2.0 ** -8, 2.0 ** -14
    out = torch.empty_like(x)
    tecoops.moe_layer(x, w_in, w_out, torch.zeros(T, E, device="cuda"), 2, out, activation="relu")
    ref = torch.zeros(H, dtype=torch.float64)
    ref[0], ref[1], ref[2] = 2047 ** 2 * 2.0 ** -9, -2047 ** 2 * 2.0 ** -7, 2047 ** 2 * 2.0 ** -14
    assert torch.equal(out, ref.to(dt).cuda().expand(T, H))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T", [2, 8, 30])
def test_infinite_h_stays_in_its_token(T, dtype):
    """A token whose h is infinite or NaN gets infinities or NaN, the others their values."""
    H, I, E, dt = 64, 40, 4, DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randint(-2, 3, (T, H), generator=g, device="cuda").to(dt)
    w_in = torch.randint(-1, 2, (E, 2 * I, H), generator=g, device="cuda").to(dt)
    w_out = torch.randint(-1, 2, (E, H, I), generator=g, device="cuda").to(dt)
    logits = torch.randn(T, E, generator=g, device="cuda")
    first, out = torch.empty_like(x), torch.empty_like(x)
    tecoops.moe_layer(x, w_in, w_out, logits, 2, first, activation="relu")
    x[T - 1] = float("inf")
    tecoops.moe_layer(x, w_in, w_out, logits, 2, out, activation="relu")
    assert torch.isfinite(first).all() and torch.equal(out[:T - 1], first[:T - 1])
    assert not torch.isfinite(out[T - 1]).all()
    tecoops.moe_layer(x, w_in, w_out, logits.index_fill(0, torch.tensor([T - 1], device="cuda"), -math.inf), 2,
                      out, activation="relu")
    assert torch.equal(out[:T - 1], first[:T - 1]) and (out[T - 1] == 0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("I", [64, 35])
@pytest.mark.parametrize("T", [1, 4, 8, 30, 200])
def test_infinite_down_weight(T, I, dtype):
    """An infinite weight gives an infinity of h's sign, not NaN, whatever terms h
    falls into, and only in its row of the result."""
    H, E, dt = 72, 2, DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.rand(T, H, generator=g, device="cuda").to(dt) + 0.5
    w_in, w_out = (torch.rand(*s, generator=g, device="cuda").to(dt) for s in ((E, 2 * I, H), (E, H, I)))
    w_out[:, 3, I - 1], w_out[:, 5, 0] = math.inf, -math.inf
    out = torch.empty_like(x)
    tecoops.moe_layer(x, w_in / 8, w_out / 8, torch.zeros(T, E, device="cuda"), 2, out)
    assert (out[:, 3] == math.inf).all() and (out[:, 5] == -math.inf).all()
    rest = [i for i in range(H) if i not in (3, 5)]
    assert torch.isfinite(out[:, rest]).all()
