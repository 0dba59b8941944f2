"""A narrower bound for the one-token attention over a 4-bit cache than
``_read.kv4_attend``'s, in which every place counts by its weight.  Runs on any
device, so that the bound can itself be tested without a GPU."""
import torch

from tests import _read, _seq


def _pairs(cache, head_dim):
    """(s, lo) of all groups [pages, heads, places, head_dim / 32, 2], in 64 bits."""
    p, h, n, _ = cache.shape
    flat = cache.reshape(p, h, -1)[..., n * head_dim // 2:]
    return flat.contiguous().view(torch.float16).double().view(p, h, n, head_dim // 32, 2)


def one_stream(q, k, v, ks, kl, vs, vl, scale, dt):
    """softmax(scale q k^T) v of a key head's queries [rows, d] over all places,
    in 64 bits, and the bound of the kernel's result in dt.  ks, kl, vs, vl: the
    groups' scales and lowest values, a place a row.  With w the weights, x = lo +
    code s the values, p = w l the kernel's weights (the largest is 2^7 or more):

      result      rounded once
      scores      queries in f16, the largest at 2^8 or more, odd ones a 16th of it:
                  2^-29 of the largest is lost; a sum over codes and one over
                  lowest values in f32, 34 roundings of what each adds up to
      weights     exponent (s - m) scale and its power of two in f32: 2^-23 of the
                  exponent and 2^-20; then to f16: 2^-11, or 2^-25 where subnormal
      p s         to f16: 2^-11 of code s, or 2^-25 where subnormal (times 2^-8
                  where all scales are below 2^-8: they are held larger then).  Where
                  a tile's 32 places have a scale of 16 or more in a group, all of it
                  are held 2^lift times smaller, and the largest is 2^(lift + 2) or
                  more: 32 places of 15 2^(lift - 25), of a sum of 2^7 or more, are no
                  more than 2^-29 of 15 times that scale; and scales that are subnormal
                  then are off by 2^(lift - 25), 2^-27 of the largest, which counts by
                  the tile's weight.  f16 results have what it lost put back times 7.5, the middle code:
                  code times the loss becomes code - 7.5 times it
      sums        in f32: 2^-23 for each 16 places
    """
    q, n = q.double(), k.shape[0]
    ks, kl, vs, vl = (x.repeat_interleave(32, -1) for x in (ks, kl, vs, vl))
    s = scale * (q @ k.T)
    w = torch.softmax(s, -1)
    out = w @ v
    ds = abs(scale) * (34 * 2.0 ** -24 * (q.abs() @ (15 * ks + kl.abs()).T)
                       + 2.0 ** -29 * q.abs().amax(-1, keepdim=True) * k.abs().sum(-1))
    ds = ds + 2.0 ** -23 * (s.amax(-1, keepdim=True) - s) * 1.5 + 2.0 ** -20
    wd = w * (ds + (w * ds).sum(-1, keepdim=True))
    size, whole = w @ v.abs(), w @ (15 * vs + vl.abs())
    codes = v - vl - (7.5 * vs if dt == torch.float16 else 0)  # times s
    limit = _seq.UNIT[dt] * out.abs() + _seq.TINY[dt] + wd @ v.abs() + 2.0 ** -11 * (size + w @ codes.abs())
    limit = limit + (8 + n / 16) * 2.0 ** -23 * whole + (2.0 ** -32 + 2.0 ** -29) * (15 * vs + vl.abs()).sum(0)
    tile = torch.nn.functional.pad(vs, (0, 0, 0, -n % 32)).view(-1, 32, vs.shape[1]).amax(1)
    share = torch.nn.functional.pad(w, (0, -n % 32)).view(w.shape[0], -1, 32).sum(-1)
    limit = limit + 2.0 ** -27 * share @ (15 * tile * (tile >= 16))
    return out, limit + n * 15 * 2.0 ** -32 * (2.0 ** -8 if float(vs.max()) < 2.0 ** -8 else 1.0)


def attend(q, kp, vp, table, lens, scale=None):
    """One token of each stream: the result in 64 bits and its bound."""
    b, hq, d = q.shape
    hk, size = kp.shape[1], kp.shape[2]
    scale = d ** -0.5 if scale is None else scale
    want = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    limit = want.clone()
    ks, vs, kpair, vpair = _read.read_cache(kp, d), _read.read_cache(vp, d), _pairs(kp, d), _pairs(vp, d)
    for i, n in enumerate(lens):
        pages = table[i, : -(-max(n, 0) // size)].long()
        for h in range(hk if n > 0 else 0):
            def of(x):
                return x[pages, h].flatten(0, 1)[:n]
            rows = slice(h * (hq // hk), (h + 1) * (hq // hk))
            want[i, rows], limit[i, rows] = one_stream(q[i, rows], of(ks), of(vs), of(kpair)[..., 0], of(kpair)[..., 1], of(vpair)[..., 0],
                                                       of(vpair)[..., 1], scale, q.dtype)
    return want, limit


def block(x):
    """[pages, heads, places, d] in the cache's layout, by its definition (on any device)."""
    code, s, lo = _read.quantise(x)
    code = code.to(torch.uint8).flatten(-2)
    pair = torch.stack([s, lo], -1).flatten(-2).contiguous().view(torch.uint8)
    return torch.cat([(code[..., 0::2] | code[..., 1::2] << 4).flatten(-2), pair.flatten(-2)], -1).view(*x.shape[:3], -1)


def streams(k, v, lens, size, gap=0, device="cuda"):
    """A cache of streams one after the other: k, v [places, heads, d] in 64 or 32
    bits, lens[i] places of stream i; pages in an order of their own."""
    need = [-(-max(n, 0) // size) for n in lens]
    total = sum(need) + gap
    order = torch.randperm(total, generator=torch.Generator().manual_seed(total)).to(device)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32, device=device)
    caches = []
    for x in (k, v):
        h, d = x.shape[1:]
        pages = torch.zeros(total, size, h, d, dtype=x.dtype, device=device)
        first = at = 0
        for i, (n, m) in enumerate(zip(lens, need)):
            if m:
                table[i, :m] = order[first:first + m]
                padded = torch.zeros(m * size, h, d, dtype=x.dtype, device=device)
                padded[:n] = x[at:at + n]
                pages[order[first:first + m]] = padded.view(m, size, h, d)
                first, at = first + m, at + n
        caches.append(block(pages.transpose(1, 2).contiguous()))
    return caches[0], caches[1], table


def markers(lens, heads, d, tile=32):
    """Values that tell which tiles a result counts, and how often: those of a
    stream's tile i are 1 in element (7 i) % d and 0 elsewhere."""
    rows = []
    for n in lens:
        i = torch.arange(max(n, 0)) // tile
        rows.append(torch.nn.functional.one_hot(7 * i % d, d))
    return torch.cat(rows).double()[:, None].expand(-1, heads, -1)
