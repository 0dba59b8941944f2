"""Plain 64-bit forms of attention to frames' states and of the 4-bit cache."""
import math

import torch

from tests import _seq


def starts(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def cross(q, k, v, q_lens, k_lens, scale=None):
    """Each sequence's tokens over its states: the result and its bound."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    group = q.shape[1] // k.shape[1]
    want = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    limit = want.clone()
    row = key = 0
    for m, n in zip(q_lens, k_lens):
        seen = torch.full((m,), n, device=q.device)
        for h in range(q.shape[1]):
            want[row:row + m, h], limit[row:row + m, h] = _seq.attend(
                q[row:row + m, h], k[key:key + n, h // group], v[key:key + n, h // group], seen, scale, q.dtype)
        row, key = row + m, key + n
    return want, limit


def quantise(x):
    """Codes, scale and lowest value of groups of 32, in 64 bits."""
    y = x.double().clamp(-65504, 65504).unflatten(-1, (-1, 32))
    lo = y.amin(-1).float().half()
    s = ((y.amax(-1) - lo.double()) / 15).clamp(min=0).float().half()
    code = torch.where((s > 0)[..., None], torch.round((y - lo.double()[..., None]) / torch.where(s > 0, s, 1).double()[..., None]), 0)
    return code.clamp(0, 15), s, lo


def values(x):
    """What the cache gives back for x, in 64 bits."""
    code, s, lo = quantise(x)
    return (lo.double()[..., None] + code * s.double()[..., None]).flatten(-2)


def read_cache(cache, head_dim):
    """All values [pages, heads, places, head_dim] of one half of a cache, in 64 bits."""
    p, h, n, _ = cache.shape
    flat = cache.reshape(p, h, -1)
    code, pair = flat[..., :n * head_dim // 2], flat[..., n * head_dim // 2:].contiguous().view(torch.float16).double()
    code = torch.stack([code & 15, code >> 4], -1).double().view(p, h, n, head_dim // 32, 32)
    pair = pair.view(p, h, n, head_dim // 32, 1, 2)
    return (pair[..., 1] + code * pair[..., 0]).flatten(-2)


def kv4_attend(q, kp, vp, table, lens, scale=None):
    """One token of each stream over a 4-bit cache: the result and its bound.
    Beyond _seq.attend's: queries in f16 with the largest at 2^8 or more, odd ones
    a 16th of that (an element loses at most 2^-29 of the largest); the scores as
    a sum over codes and one over lowest values, in f32 and with the queries' sums
    to 2^-22, so that each counts at its own size; weights in f16, then times
    scales in f16 (2^-11 twice), over codes and lowest values that may cancel,
    and their subnormals, which lose 2^-25 beside a largest weight of 2^4."""
    b, hq, d = q.shape
    hk, size = kp.shape[1], kp.shape[2]
    scale = d ** -0.5 if scale is None else scale
    ks, vs = read_cache(kp, d), read_cache(vp, d)
    want = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    limit = want.clone()
    for i, n in enumerate(lens):
        n = max(n, 0)
        pages = table[i, : -(-n // size)].long()
        for h in range(hk if n else 0):
            k, v = (x[pages, h].reshape(-1, d)[:n] for x in (ks, vs))
            rows = slice(h * (hq // hk), (h + 1) * (hq // hk))
            seen = torch.full((hq // hk,), n, device=q.device)
            w, e = _seq.attend(q[i, rows], k, v, seen, scale, q.dtype)
            def parts(cache):  # 15 s and |lo| of each group of each place
                pair = cache.reshape(*cache.shape[:2], -1)[pages, h][:, size * d // 2:].contiguous().view(torch.float16).double()
                pair = pair.reshape(-1, d // 32, 2)[:n]
                return 15 * pair[..., 0] + pair[..., 1].abs()
            qsum = q[i, rows].double().abs().unflatten(-1, (-1, 32)).sum(-1)
            ds = abs(scale) * (34 * 2.0 ** -24 * (qsum @ parts(kp).T).amax(-1, keepdim=True)
                               + 2.0 ** -29 * q[i, rows].double().abs().amax(-1, keepdim=True) * k.abs().sum(-1).max())
            size_ = parts(vp).amax(0).repeat_interleave(32)
            want[i, rows], limit[i, rows] = w, e + (2 * ds + 2.0 ** -10) * size_ + n * 2.0 ** -28 * size_.max()
    return want, limit
