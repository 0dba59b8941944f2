"""Plain 64-bit forms of the sequence operators and the error bounds their
results are held to."""
import math

import torch

# unit roundoff of each type: half the spacing at 1
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}  # half the spacing of subnormals


def norm_rope(x, w, pos, table, rot, interleaved, eps):
    """The operator in 64 bits, and per element |a| + |b| of what was rotated."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    out, size = y.clone(), y.abs()
    if rot:
        i = torch.arange(rot // 2, device=x.device)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, s = (table[pos.long()].double()[:, None, k * (rot // 2):(k + 1) * (rot // 2)] for k in (0, 1))
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
        size[..., a] = size[..., b] = y[..., a].abs() + y[..., b].abs()
    return out, size


def check_norm_rope(got, want, size):
    """One rounding of the result, and the f32 arithmetic before it: the mean
    of up to 512 squares in lanes of 16 (relative error under 24 roundings),
    its root, two products each and a sum: under 64 roundings of |a| + |b|."""
    dt = got.dtype
    err = (got.double() - want).abs()
    limit = UNIT[dt] * want.abs() + TINY[dt] + 64 * 2.0 ** -24 * size
    assert bool((err <= limit).all()), f"off by {float((err / limit.clamp(min=1e-300)).max()):.3g} of the bound"


def attend(q, k, v, seen, scale, dt):
    """softmax(scale q k^T) v over the first seen[i] keys for row i of one head,
    in 64 bits, and the bound of a result in dt: the output's rounding, the
    weights' rounding to dt, and the scores' error (products summed in f32,
    in the worst order) together with the exponential's (under 2^-20)."""
    q, k, v = q.double(), k.double(), v.double()
    if k.shape[0] == 0:
        z = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        return z, z
    mask = torch.arange(k.shape[0], device=q.device) < seen[:, None]
    s = torch.where(mask, scale * (q @ k.T), -math.inf)
    w = torch.nan_to_num(torch.softmax(s, -1)) * mask
    out = w @ v
    size = w @ v.abs()
    ds = (q.shape[-1] + 8) * 2.0 ** -24 * abs(scale) * torch.where(mask, q.abs() @ k.abs().T, 0.0).amax(-1, keepdim=True)
    low = TINY[dt] * seen[:, None].double() * v.abs().max()
    return out, UNIT[dt] * out.abs() + (UNIT[dt] + 2 * ds + 2.0 ** -19) * size + low + TINY[dt]


def check(got, want, limit):
    err = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all()), "not finite"
    assert bool((err <= limit).all()), f"off by {float((err / limit.clamp(min=1e-300)).max()):.3g} of the bound"
