"""The e4m3 projection, rotary and cross-attention operators in 64 bits on the host, with bounds on what a correct
kernel may be off by.  Every bound is a sum of roundings: half a step of the output's type (finfo.eps / 2 of the value,
and half a subnormal step), and counted f32 roundings of 2^-24 (2^-23 where a sum may be truncated)."""
import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SUBNORMAL = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
F32 = 2.0 ** -24
GROUP = 128
KINDS = {"f16": torch.float16, "bf16": torch.bfloat16}


def groups(width):
    return -(-width // GROUP)


def f64(t):
    return t.detach().cpu().to(torch.float64) if t.dtype != torch.float8_e4m3fn else t.detach().cpu().to(torch.float32).to(torch.float64)


def spread(scale, width):
    """[rows][groups] -> [rows][width]"""
    return scale.repeat_interleave(GROUP, 1)[:, :width]


# ------------------------------------------------------------------ codes
def norm_rows(x, residual, weight, eps, offset):
    """(the rows the codes are taken of, the sum in x's type or None), from the kernel's own inputs."""
    total = None
    if residual is not None:
        # x + residual in f32, rounded to the type: the one f32 rounding in front of it is part of the definition
        total = (x.detach().cpu().float() + residual.detach().cpu().float()).to(x.dtype)
        x = total
    y = f64(x)
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
    factor = offset + (f64(weight) if weight is not None else torch.zeros(x.shape[1], dtype=torch.float64))
    return y * factor, total


def check_codes(q, q_scale, y, roundings):
    """q, q_scale against rows y (f64) that the kernel computed with at most that many f32 roundings.

    scale is off by `roundings` + 1, the quotient code's argument by that, `roundings` of y, one reciprocal and one
    product; so the code lies between the roundings of the exact quotient made that much smaller and larger."""
    rows, width = y.shape
    padded = torch.nn.functional.pad(y, (0, groups(width) * GROUP - width)).view(rows, -1, GROUP)
    scale = (padded.abs().amax(-1) / 448.0).clamp_min(2.0 ** -126)
    got = f64(q_scale)
    assert torch.all((got - scale).abs() <= (roundings + 1) * F32 * scale), float(((got - scale).abs() / scale).max() / F32)
    quotient = y / spread(scale, width)
    slack = (2 * roundings + 4) * F32
    low, high = ((quotient * (1.0 + s)).clamp(-448.0, 448.0).to(torch.float32).to(torch.float8_e4m3fn).float() for s in (-slack, slack))
    codes = q.detach().cpu().float()
    inside = (codes >= torch.minimum(low, high)) & (codes <= torch.maximum(low, high))
    assert bool(inside.all()), (int((~inside).sum()), codes[~inside][:4], quotient[~inside][:4])


# ------------------------------------------------------------------ product
def product(a, a_scale, w, w_scale):
    """(c in f64, the sum of the magnitudes of its terms)"""
    m, k = a.shape
    n = w.shape[0]
    left = f64(a) * spread(f64(a_scale), k)
    right = f64(w) * spread(f64(w_scale), k).repeat_interleave(GROUP, 0)[:n]
    return left @ right.t(), left.abs() @ right.abs().t()


def check_product(c, a, a_scale, w, w_scale):
    exact, magnitude = product(a, a_scale, w, w_scale)
    # products of codes are exact in f32; a block's 128 are added, scaled (two roundings) and added to the others
    bound = HALF_STEP[c.dtype] * exact.abs() + SUBNORMAL[c.dtype] + (GROUP + groups(a.shape[1]) + 4) * 2 * F32 * magnitude
    got, top = f64(c), torch.finfo(c.dtype).max
    finite = exact.abs() + bound < top
    off = (got - exact).abs()
    assert bool((off[finite] <= bound[finite]).all()), float((off[finite] / bound[finite]).max())


# ------------------------------------------------------------------ rotary
def rotary(x, positions, frequencies, magnitude, layout, inverse):
    """(x turned in f64, |a| + |b| of each channel's pair times the magnitude, 0 for channels left as they are)"""
    half = frequencies.numel()
    y, reach = f64(x).clone(), torch.zeros(x.shape, dtype=torch.float64)
    angle = (positions.to(torch.float64)[:, None] * frequencies.cpu()[None])[:, None, :]
    cosine, sine = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude * (-1.0 if inverse else 1.0)
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if layout == "interleaved" else (slice(0, half), slice(half, 2 * half))
    a, b = f64(x)[..., first], f64(x)[..., second]
    y[..., first], y[..., second] = a * cosine - b * sine, b * cosine + a * sine
    reach[..., first] = reach[..., second] = (a.abs() + b.abs()) * abs(magnitude)
    return y, reach


def check_rotary(out, x, positions, frequencies, magnitude, layout, inverse):
    exact, reach = rotary(x, positions, frequencies, magnitude, layout, inverse)
    # the remainder of the turns in f32: 2^-26 turns = 1.6 * 2^-24 radians; sincospif: 2 ulp; the product with the
    # magnitude (and its own rounding to f32), two products and a sum: under 10 roundings of the pair's values
    bound = HALF_STEP[out.dtype] * exact.abs() + SUBNORMAL[out.dtype] + 10 * F32 * reach
    off = (f64(out) - exact).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    kept = reach == 0
    assert torch.equal(out.detach().cpu()[kept & (f64(x) != 0)], x.detach().cpu()[kept & (f64(x) != 0)])


# ------------------------------------------------------------------ cross attention
def check_cross(out, q, k, v, scale, kv_lengths=None, key_mask=None):
    batch, q_len, q_heads, d = q.shape
    kv_len, kv_heads = k.shape[1], k.shape[2]
    u = HALF_STEP[out.dtype]
    worst = 0.0
    for b in range(batch):
        counts = torch.ones(kv_len, dtype=torch.bool)
        if kv_lengths is not None:
            counts[max(0, int(kv_lengths[b])):] = False
        if key_mask is not None:
            counts &= key_mask[b].cpu() != 0
        if not bool(counts.any()):
            assert not bool(f64(out[b]).any()), "rows without a counting key must be zero"
            continue
        for h in range(q_heads):
            queries, keys, values = f64(q[b, :, h]), f64(k[b, :, h * kv_heads // q_heads])[counts], f64(v[b, :, h * kv_heads // q_heads])[counts]
            scores = queries @ keys.t() * scale
            p = torch.softmax(scores, -1)
            exact, magnitude = p @ values, p @ values.abs()
            # a score is off by d + 3 roundings of the sum of its terms' magnitudes (twice: weight and weights' sum);
            # a weight by that, the exponential's 2^-21 and, before it meets the values, half a step of the type; the
            # sum over the keys by one rounding a key (and one for each tile of 128 that moves the maximum)
            reach = (queries.abs() @ keys.abs().t() * scale).amax(-1, keepdim=True)
            counted = float(counts.sum())
            relative = u + 2 * ((d + 3) * 2 * F32 * reach) + 2.0 ** -20 + 2 * (counted + counted / 64 + 8) * F32
            bound = u * exact.abs() + relative * magnitude * (1 + u) + SUBNORMAL[out.dtype] + 2.0 ** -24 * values.abs().amax() * (out.dtype == torch.float16)
            off = (f64(out[b, :, h]) - exact).abs()
            assert bool((off <= bound).all()), (b, h, float((off / bound).max()))
            worst = max(worst, float((off / bound).max()))
    return worst


def frequencies_of(rotary_dim, base, scaling, factor, trained, slow, fast):
    """Plain Python restatement of rotary_frequencies."""
    if scaling == "base":
        base = base * factor ** (rotary_dim / (rotary_dim - 2 if rotary_dim > 2 else 1))
    out = []
    for i in range(rotary_dim // 2):
        f = base ** (-2.0 * i / rotary_dim)
        if scaling == "linear":
            f /= factor
        if scaling == "parts":
            kept = min(1.0, max(0.0, (trained * f / (2 * math.pi) - slow) / (fast - slow)))
            f = f * kept + f / factor * (1 - kept)
        out.append(f)
    return out, (0.1 * math.log(factor) + 1.0) if scaling == "parts" else 1.0
