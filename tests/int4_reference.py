"""Plain 64-bit forms of the operators of a decode path held in 4 bits, written
from their formulas, and the inputs that their tests share."""
import math

import torch

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
# half a step of a rounding to the type, relative to the value
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def rand(*shape, dtype=torch.float16, scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def pack(codes):
    """Codes [..., K] of 0..15 as bytes [..., K / 2], the even ones in the low half."""
    c = codes.to(torch.int32)
    return (c[..., 0::2] + 16 * c[..., 1::2]).to(torch.uint8)


def unpack(held):
    h = held.to(torch.int32)
    return torch.stack([h % 16, h // 16], -1).flatten(-2)


def quantised(x):
    """Codes and (scale, low) of the rows of x, from the definition."""
    f = x.double()
    low, top = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    scale = ((top - low).float() / 15).to(x.dtype)
    n = torch.where(scale > 0, (f - low) / scale.double(), torch.zeros_like(f))
    pair = torch.cat([scale, low.to(x.dtype)], -1)
    bad = ~torch.isfinite(f).all(-1, keepdim=True) | ~torch.isfinite((top - low).float())
    n = torch.where(bad, torch.zeros_like(n), n).round().clamp(0, 15)
    return n.to(torch.int32), torch.where(bad, torch.full_like(pair, math.nan), pair)


def dequantised(held, pairs):
    p = pairs.double()
    return unpack(held).double() * p[..., :1] + p[..., 1:]


def rows_of(held, pairs, table, length, kv_head):
    """[length, head_size] rows of a sequence of the cache."""
    bs = held.shape[2]
    j = torch.arange(length)
    page = table.long()[j // bs]
    return dequantised(held[page, kv_head, j % bs], pairs[page, kv_head, j % bs])


def attention(q, kc, vc, ks, vs, cu, lens, table, scale=None, causal=True):
    """Output [rows, heads, D] and, for each element, what a relative error of the
    weights moves it by, sum_j p_j max(|V_j|, |V_j - middle of row j|), and the
    largest sum |q| |K| over the keys that its row sees (for error bounds)."""
    T, H, D = q.shape
    Hkv = kc.shape[1]
    scale = scale or 1.0 / math.sqrt(D)
    out = torch.zeros(T, H, D, dtype=torch.float64)
    mass, reach = torch.zeros_like(out), torch.zeros(T, H, 1, dtype=torch.float64)
    for b, S in enumerate(lens):
        q0, L = cu[b], cu[b + 1] - cu[b]
        if L <= 0:
            continue
        first = max(S - L, 0) if causal else 0
        for kvh in range(Hkv):
            K = rows_of(kc, ks, table[b], S, kvh)
            V = rows_of(vc, vs, table[b], S, kvh)
            M = rows_of(torch.zeros_like(vc), vs, table[b], S, kvh) + 7.5 * rows_of(
                torch.zeros_like(vc), torch.stack([vs[..., 0] * 0, vs[..., 0]], -1), table[b], S, kvh)
            for h in range(kvh * (H // Hkv), (kvh + 1) * (H // Hkv)):
                qr = q[q0:q0 + L, h].double()
                s = qr @ K.t() * scale
                seen = torch.ones(L, S, dtype=torch.bool)
                if causal:
                    seen = torch.arange(S)[None] <= first + torch.arange(L)[:, None]
                s = s.masked_fill(~seen, -math.inf)
                if S == 0:
                    continue
                p = torch.softmax(s, -1)
                p = torch.where(seen.any(-1, keepdim=True), p, torch.zeros_like(p))
                out[q0:q0 + L, h] = p @ V
                mass[q0:q0 + L, h] = p @ torch.maximum(V.abs(), (V - M).abs())
                r = (qr.abs() @ K.abs().t() * scale).masked_fill(~seen, 0.0)
                reach[q0:q0 + L, h] = r.amax(-1, keepdim=True)
    return out, mass, reach


def norm_rotary(x, weight, eps, cos, sin, rot, neox):
    """x [T, heads, D] normalised and turned by cos / sin [T, rot / 2]; the second
    result is what a rounding error of an element is relative to."""
    f = x.double()
    y = f / torch.sqrt((f * f).mean(-1, keepdim=True) + eps) * weight.double()
    half, c, s = rot // 2, cos.double()[:, None], sin.double()[:, None]
    one = slice(0, half) if neox else slice(0, rot, 2)
    two = slice(half, rot) if neox else slice(1, rot, 2)
    out, size = y.clone(), y.abs()
    out[..., one] = y[..., one] * c - y[..., two] * s
    out[..., two] = y[..., two] * c + y[..., one] * s
    size[..., one] = y[..., one].abs() + y[..., two].abs()
    size[..., two] = size[..., one]
    return out, size


def weights(codes, scales, zeros, group):
    n = codes.double().view(codes.shape[0], -1, group)
    z = 8.0 if zeros is None else zeros.double()[..., None]
    return ((n - z) * scales.double()[..., None]).flatten(1)


def check(got, ref, bound, what=""):
    """|got - ref| <= bound, element by element; where ref is no number, got the same."""
    got = got.detach().cpu().double()
    bound = torch.as_tensor(bound, dtype=torch.float64).expand_as(ref)
    fine = torch.isfinite(ref)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    err = torch.where(fine, (got - ref).abs(), torch.zeros_like(ref))
    over = torch.where(fine, err - bound, torch.zeros_like(ref))
    if over.numel() and (over > 0).any():
        i = int(over.argmax())
        raise AssertionError(f"{what}: {int((over > 0).sum())} of {over.numel()} off; worst at {i}: got "
                             f"{got.flatten()[i]} for {ref.flatten()[i]}, bound {bound.flatten()[i]:.3e}")
