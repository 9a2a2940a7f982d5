"""Attention over latent vectors and its rotations by their definitions, in 64 bits, a request and a token at a time (torch, on the CPU)."""
import math

import torch

# A rounding to a type: at most half a step, relative to the value.
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# The smallest value's half step, where a rounding is not relative any more.
LEAST = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def frequencies(n_dims, base, freq_scale=1.0, ext_factor=0.0, corr_dims=(0.0, 0.0), freq_factors=None):
    out = []
    for p in range(n_dims // 2):
        far = base ** (-2.0 * p / n_dims) / (1.0 if freq_factors is None else float(torch.tensor(freq_factors[p], dtype=torch.float32)))
        f = far * freq_scale
        if ext_factor != 0.0:
            mix = ext_factor * (1.0 - min(1.0, max(0.0, (p - corr_dims[0]) / max(0.001, corr_dims[1] - corr_dims[0]))))
            f = f * (1.0 - mix) + far * mix
        out.append(f)
    return torch.tensor(out, dtype=torch.float64)


def rotate(x, positions, freqs, layout, magnitude=1.0, inverse=False):
    """The last axis of x [tokens, ..., 2 * pairs], in 64 bits."""
    pairs = freqs.numel()
    x = x.double()
    angle = positions.double()[:, None] * freqs
    angle = (-angle if inverse else angle).view((x.shape[0],) + (1,) * (x.dim() - 2) + (pairs,))
    cos, sin = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude
    a, b = (x[..., :pairs], x[..., pairs:]) if layout == "half" else (x[..., 0::2], x[..., 1::2])
    u, v = a * cos - b * sin, a * sin + b * cos
    return torch.cat([u, v], -1) if layout == "half" else torch.stack([u, v], -1).flatten(-2)


E4M3 = torch.tensor([(m & 7) * 2.0 ** -9 if m < 8 else (8 + (m & 7)) * 2.0 ** ((m >> 3) - 10) for m in range(127)] + [math.nan], dtype=torch.float64)


def code_values(codes, scales):
    """What E4M3 codes uint8 [..., width] and E8M0 scales uint8 [...] stand for."""
    c = codes.long()
    return torch.where(c >= 128, -1.0, 1.0) * E4M3[c & 127] * torch.exp2(scales.double() - 127.0)[..., None]


def encode(x):
    """float32 rows as (codes, scales): the smallest power of two that holds the largest finite or infinite value, 448 at most."""
    codes = torch.zeros(x.shape, dtype=torch.uint8)
    scales = torch.zeros(x.shape[:-1], dtype=torch.uint8)
    for i, row in enumerate(x.reshape(-1, x.shape[-1])):
        most = float(torch.nan_to_num(row.abs(), nan=0.0, posinf=math.inf).max())
        e = 0
        while e < 253 and most > 448.0 * 2.0 ** (e - 127):
            e += 1
        y = (row.double() * 2.0 ** (127 - e)).clamp(-448.0, 448.0)
        distance = (y.abs()[:, None] - E4M3[:127][None, :]).abs()
        best = distance.amin(1, keepdim=True)
        near = distance == best  # one code, or two and the even one of them
        code = torch.arange(127)[None, :].expand_as(near)
        code = torch.where(near & ((near.sum(1, keepdim=True) == 1) | (code % 2 == 0)), code, 0).amax(1)
        code = torch.where(torch.isnan(row), 127, code)
        codes.view(-1, x.shape[-1])[i] = (code + torch.where(torch.signbit(row), 128, 0)).to(torch.uint8)
        scales.view(-1)[i] = e
    return codes, scales


def attention(q, k, v, scale, position, kept):
    """Rows of q [rows, d] at positions [rows] over k [keys, d] and v [keys, w], key j at position j where kept[j]; a row that sees nothing
    is zero. Returns (out, the same sum over |v|, the largest sum of |q k| of a row's logits)."""
    sees = (torch.arange(k.shape[0])[None, :] <= position[:, None]) & kept[None, :]
    k, v = torch.where(kept[:, None], k, 0.0), torch.where(kept[:, None], v, 0.0)
    out, size, logits = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64), torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64), torch.zeros(q.shape[0], dtype=torch.float64)
    for i in range(q.shape[0]):
        j = sees[i].nonzero()[:, 0]
        if not len(j):
            continue
        p = torch.softmax(k[j] @ q[i] * scale, 0)
        out[i], size[i] = p @ v[j], p @ v[j].abs()
        logits[i] = (k[j].abs() @ q[i].abs()).max() * abs(scale)
    return out, size, logits


def close(got, want, size, logits, dtype, dims, keys):
    """What an attention's stated roundings leave: a logit's products summed in F32 (dims steps of 2^-24 of the sum of magnitudes) and
    an exponential off by 2^-21, in the weights and, once more, in their sum (keys steps of 2^-24); a weight's rounding, of itself, or of F16's least
    step under the row's largest (2^-33); the products' sum in F32 (keys steps); the result's own rounding."""
    got = got.double().cpu()
    logit = logits[:, None] * dims * 2.0 ** -24 * 1.01 + 2.0 ** -21
    weight = HALF[dtype] + (2.0 ** -33 * keys if dtype is torch.float16 else 0.0)
    bound = size * (2.0 * logit + weight + 3.0 * keys * 2.0 ** -24) * 1.01
    bound = bound + (want.abs() + bound) * HALF[dtype] + LEAST[dtype]
    worst = ((got - want).abs() / bound.clamp(min=1e-300)).nan_to_num(nan=math.inf)
    worst = torch.where(got == want, 0.0, worst)
    assert worst.numel() == 0 or worst.max() <= 1.0, f"{float(worst.max()):.3g} of the bound at {torch.nonzero(worst == worst.max())[0].tolist()}"
