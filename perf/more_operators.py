"""Operators of streams that read frames, as measured cases.

What a decoder over video needs beside the attention that is there: the norm
and rotation of heads by positions along several axes (time, height, width),
attention of text tokens to the frames' states, which have a length of their
own, and a paged cache held in 4 bits, with its filing, its reading back and
the one-token attention over it.

A place of the 4-bit cache is, per head, groups of 32 elements with a scale s
and a lowest value lo in 16 bits each: value = lo + code * s, codes 0 to 15.
The block of a page and head holds all places' codes (two to a byte, the even
element low), then all places' (s, lo) pairs.

``own`` False: plain torch forms in 32 bits, rounded once at the end (the
quantisation in 64 bits, where its borders count).  ``own`` True: the
framework's entry points.  ``exact`` gives the operators' definitions in 64
bits, written apart from both.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


# ------------------------------------------------------------------ cases ---

def listed():
    return [
        # one decode step of eight streams that have reached different moments of a clip: latency
        dict(name="axes_step_8", op="axes", frames=0, height=10, width=18, text=8, q_heads=16, kv_heads=4, dim=64, sections="8,12,12",
             turns=False, interleaved=False, dtype="f16", cached=True, page=16),
        # seven 160x288 frames at stride 16 and a question behind them, half of a head rotated, axes taking turns
        dict(name="axes_frames_1297", op="axes", frames=7, height=10, width=18, text=37, q_heads=20, kv_heads=5, dim=96,
             sections="8,8,8", turns=True, interleaved=True, dtype="bf16", cached=False, page=16),
        # a clip of 90 such frames entering the cache: memory-bound
        dict(name="axes_clip_16350", op="axes", frames=90, height=10, width=18, text=150, q_heads=32, kv_heads=8, dim=128,
             sections="16,24,24", turns=False, interleaved=False, dtype="bf16", cached=True, page=64),
        # one token of each of eight streams looks at its own frame of 180 states: latency
        dict(name="cross_step_8x180", op="cross", q_lens="", k_lens=",".join(["180"] * 8), q_heads=8, kv_heads=2, dim=64,
             dtype="f16"),
        # a batch of streams, each with its own clip of up to 16 frames, some of odd lengths, one without any: memory-bound
        dict(name="cross_step_96", op="cross", q_lens="", k_lens=",".join(str((i * 1171) % 2881) for i in range(96)), q_heads=32,
             kv_heads=8, dim=128, dtype="bf16"),
        # short questions about long clips: few rows over a long axis
        dict(name="cross_question_52", op="cross", q_lens="32,1,19", k_lens="16200,5401,0", q_heads=32, kv_heads=8, dim=128,
             dtype="bf16"),
        # whole texts over clips: bound by the matrix products
        dict(name="cross_text_5095", op="cross", q_lens="4096,999", k_lens="8192,5041", q_heads=32, kv_heads=8, dim=128,
             dtype="bf16"),
        # the new token of eight streams goes into the 4-bit cache: latency
        dict(name="kv4_file_8", op="file", tokens=8, kv_heads=4, dim=64, page=16, dtype="f16"),
        # a batch of prompts enters it: memory-bound
        dict(name="kv4_file_16384", op="file", tokens=16384, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # a few streams with short contexts: latency
        dict(name="kv4_4x240", op="kv4", batch=4, longest=240, q_heads=8, kv_heads=2, dim=64, page=16, dtype="f16"),
        # an ordinary batch, odd in size, one stream without places
        dict(name="kv4_33x4501", op="kv4", batch=33, longest=4501, q_heads=32, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # many long contexts, which is what 4 bits are for: memory-bound
        dict(name="kv4_64x16384", op="kv4", batch=64, longest=16384, q_heads=32, kv_heads=8, dim=128, page=64, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op, dtype = rng.choice(["axes", "cross", "cross", "file", "kv4"]), rng.choice(["bf16", "f16"])
    kv, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 4, 7, 8])
    if kv * group > 32:
        group = 4
    page = rng.choice([16, 32, 64])
    if op == "axes":
        dim = rng.choice([64, 80, 96, 128])
        height, width = rng.choice([(10, 18), (9, 16), (5, 9), (20, 36)])
        pairs = rng.choice([dim // 2, dim // 4])
        cut = sorted(rng.sample(range(1, pairs), 2))
        frames = rng.choice([0, _log(rng, 1, 16000 // (height * width))])
        return dict(op=op, frames=frames, height=height, width=width, text=_log(rng, 1, 300 if frames else 16000), q_heads=kv * group, kv_heads=kv, dim=dim,
                    sections="%d,%d,%d" % (cut[0], cut[1] - cut[0], pairs - cut[1]), turns=rng.random() < 0.3,
                    interleaved=rng.random() < 0.3, dtype=dtype, cached=rng.random() < 0.6, page=page)
    if op == "cross":
        n, top = _log(rng, 1, 96), _log(rng, 8, 16384)
        dim = rng.choice([64, 80, 128])
        if rng.random() < 0.5:  # one token of each
            top = min(top, max(8, 130_000 // n))
            k_lens = [top] + [rng.choice([0, _log(rng, 1, top), _log(rng, 1, top)]) for _ in range(n - 1)]
            q_lens = ""
        else:
            # the plain form pads both sides to the longest
            n, q_top = min(n, 16), _log(rng, 1, 4096)
            top = max(1, min(top, 33_000_000 // (n * q_top)))
            k_lens = [top] + [rng.choice([0, _log(rng, 1, top), _log(rng, 1, top)]) for _ in range(n - 1)]
            q_lens = ",".join(str(x) for x in [q_top] + [rng.randint(0, q_top) for _ in range(n - 1)])
        return dict(op=op, q_lens=q_lens, k_lens=",".join(map(str, k_lens)), q_heads=kv * group, kv_heads=kv, dim=dim, dtype=dtype)
    dim = rng.choice([64, 96, 128])
    if op == "file":
        return dict(op=op, tokens=_log(rng, 1, 16384), kv_heads=kv, dim=dim, page=page, dtype=dtype)
    batch = _log(rng, 1, 128)
    return dict(op=op, batch=batch, longest=min(_log(rng, 1, 32768), 500_000 // batch), q_heads=kv * group, kv_heads=kv, dim=dim,
                page=page, dtype=dtype)


def _ints(text):
    return [int(x) for x in text.split(",")] if text else []


def _tokens(case):
    return case["frames"] * case["height"] * case["width"] + case["text"]


def _stream_lens(case):
    """Places of each stream of a kv4 case: 1 to `longest`, none for one stream."""
    return [0 if b == 5 else case["longest"] - (b * 7919 * case["longest"] // 10007) % (case["longest"] + 1) for b in range(case["batch"])]


# ----------------------------------------------------------------- inputs ---

def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed))
    return dict({"axes": _prepare_axes, "cross": _prepare_cross, "file": _prepare_file, "kv4": _prepare_kv4}[case["op"]](case, g),
                case=case)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return _int32(cu)


def _prepare_axes(case, g):
    t, hq, hk, d, dt = _tokens(case), case["q_heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    sections = _ints(case["sections"])
    pairs = sum(sections)
    qkv = (2.0 * _randn(g, t, hq + 2 * hk, d)).to(dt)
    # frames first: (time, row, column); then text, one step on all axes per token (alone: streams at moments of their own)
    h, w, patches = case["height"], case["width"], t - case["text"]
    i = torch.arange(patches, device="cuda")
    grid = torch.stack([i // (h * w), i // w % h, i % w], 1)
    after = max(case["frames"], h, w) if patches else 0
    n = torch.arange(case["text"], device="cuda") + after if patches or case["text"] > 64 else \
        torch.randint(0, 4000, (case["text"],), generator=g, device="cuda")
    pos = torch.cat([grid, n[:, None].expand(-1, 3)]).to(torch.int32).contiguous()
    axis = torch.repeat_interleave(torch.arange(3, device="cuda"), torch.tensor(sections, device="cuda"))
    if case["turns"]:
        axis = torch.arange(pairs, device="cuda") % 3
    top = 16384
    freq = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    ang = torch.arange(top, dtype=torch.float64, device="cuda")[:, None] * freq
    s = dict(q=qkv[:, :hq], k=qkv[:, hq:hq + hk], v=qkv[:, hq + hk:], pos=pos, axis=axis.to(torch.uint8),
             table=torch.cat([ang.cos(), ang.sin()], 1).float().contiguous(), wq=1.0 + 0.2 * _randn(g, d),
             wk=1.0 + 0.2 * _randn(g, d))
    if case["cached"]:
        pages = -(-t // case["page"]) + 3
        s["kp"] = torch.zeros(pages, case["page"], hk, d, dtype=dt, device="cuda")
        s["vp"] = torch.zeros_like(s["kp"])
        s["slots"] = _slots(t, pages, case["page"], g)
    return s


def _slots(t, pages, page, g):
    """Tokens side by side in pages of a random order; the last of several is not filed."""
    at = torch.arange(t, device="cuda")
    slots = torch.randperm(pages, generator=g, device="cuda")[at // page] * page + at % page
    if t > 1:
        slots[-1] = -1
    return slots


def _key_gain(d):
    """A few key channels stand out, as they do behind a norm with a weight."""
    gain = torch.ones(d, device="cuda")
    gain[:: max(1, d // 4)] = 3.0
    return gain


def _prepare_cross(case, g):
    k_lens, q_lens = _ints(case["k_lens"]), _ints(case["q_lens"])
    hq, hk, d, dt = case["q_heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    t = sum(q_lens) if q_lens else len(k_lens)
    kv = _randn(g, sum(k_lens), 2, hk, d)  # a projection of the states: keys and values of a state side by side
    kv[:, 0] *= _key_gain(d)
    kv = kv.to(dt)
    return dict(q=_randn(g, t, hq, d).to(dt), k=kv[:, 0], v=kv[:, 1], cu_k=_starts(k_lens), cu_q=_starts(q_lens) if q_lens else None)


def _prepare_file(case, g):
    t, hk, d, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
    kv = _randn(g, t, 2, hk, d)
    kv[:, 0] *= _key_gain(d)
    kv = kv.to(DTYPES[case["dtype"]])
    pages = -(-t // page) + 3
    kp, vp = torch.zeros(2, pages, hk, page, d * 5 // 8, dtype=torch.uint8, device="cuda")
    return dict(k=kv[:, 0], v=kv[:, 1], kp=kp, vp=vp, slots=_slots(t, pages, page, g))


def _prepare_kv4(case, g):
    b, hq, hk, d, page, dt = case["batch"], case["q_heads"], case["kv_heads"], case["dim"], case["page"], DTYPES[case["dtype"]]
    lens = _stream_lens(case)
    need = [-(-n // page) for n in lens]
    pages, width = sum(need) + 5, -(-case["longest"] // page)
    kp = _blocks((_randn(g, pages, hk, page, d) * _key_gain(d)).to(dt))
    vp = _blocks(_randn(g, pages, hk, page, d).to(dt))
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    first, at = _starts(need)[:-1, None], torch.arange(width, device="cuda")
    table = torch.where(at < _int32(need)[:, None], order[(first + at).clamp(max=pages - 1).long()], -1)
    return dict(q=_randn(g, b, hq, d).to(dt), kp=kp, vp=vp, table=table.to(torch.int32).contiguous(), lens=_int32(lens))


# -------------------------------------------------------- the 4-bit cache ---

def _quantise(x):
    """Codes (uint8) and scale, lowest value (float16) of groups of 32 along the last dimension, in 64 bits."""
    y = x.float().clamp(-65504.0, 65504.0).unflatten(-1, (-1, 32)).double()
    lo = y.amin(-1).to(torch.float16)
    s = ((y.amax(-1) - lo.double()) / 15.0).clamp(min=0.0).to(torch.float16)
    step = torch.where(s == 0, 1.0, s.double())
    code = torch.round((y - lo.double()[..., None]) / step[..., None]).clamp(0.0, 15.0)
    return torch.where((s == 0)[..., None], 0.0, code).to(torch.uint8).flatten(-2), s, lo


def _bytes(code, s, lo):
    """Packed codes, and (s, lo) pairs as bytes."""
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.stack([s, lo], -1).flatten(-2).contiguous().view(torch.uint8)


def _blocks(x):
    """[pages, heads, places, d] as blocks of the cache, which keep that shape but for the last size."""
    code, pair = _bytes(*_quantise(x))
    return torch.cat([code.flatten(-2), pair.flatten(-2)], -1).view(*x.shape[:3], -1)


def _planes(cache, d):
    """The codes [pages, heads, places, d / 2] and the pairs' bytes [pages, heads, places, d / 8], as views."""
    p, h, n, _ = cache.shape
    flat = cache.view(p, h, -1)
    return flat[..., :n * d // 2].unflatten(-1, (n, d // 2)), flat[..., n * d // 2:].unflatten(-1, (n, d // 8))


def _values(code, pair):
    """Values in 32 bits of packed codes and pairs' bytes."""
    c = torch.stack([code & 15, code >> 4], -1).flatten(-2).float().unflatten(-1, (-1, 32))
    m = pair.contiguous().view(torch.float16).float().unflatten(-1, (-1, 2))
    return (m[..., 1:] + c * m[..., :1]).flatten(-2)


# ---------------------------------------------------------------- a pass ---

def run(state):
    return {"axes": _run_axes, "cross": _run_cross, "file": _run_file, "kv4": _run_kv4}[state["case"]["op"]](state)


def _run_axes(s):
    case = s["case"]
    if own:
        from ai_engine_b200 import attention
        q, k = attention.qk_norm_rope(s["q"], s["k"], s["pos"], s["table"], pair_axis=s["axis"], q_weight=s["wq"], k_weight=s["wk"],
                                      eps=EPS, interleaved=case["interleaved"], v=s["v"] if case["cached"] else None,
                                      k_pages=s.get("kp"), v_pages=s.get("vp"), slots=s.get("slots"))
    else:
        q, k = _plain_axes(s["q"], s["wq"], s), _plain_axes(s["k"], s["wk"], s)
        if case["cached"]:
            keep = s["slots"] >= 0
            at = s["slots"][keep]
            s["kp"].view(-1, case["kv_heads"], case["dim"])[at] = k[keep]
            s["vp"].view(-1, case["kv_heads"], case["dim"])[at] = s["v"][keep]
    return (q, k, s["kp"], s["vp"]) if case["cached"] else (q, k)


def _plain_axes(x, w, s):
    half = s["axis"].shape[0]
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w
    at = s["pos"].long()[:, s["axis"].long()]  # each pair's position
    i = torch.arange(half, device=x.device)
    cos, sin = s["table"][at, i][:, None], s["table"][at, i + half][:, None]
    if s["case"]["interleaved"]:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, y[..., 2 * half:]], -1).to(x.dtype)


def _run_cross(s):
    if own:
        from ai_engine_b200 import attention
        return attention.cross_attention(s["q"], s["k"], s["v"], s["cu_k"], cu_q=s["cu_q"])
    q, k, v, cu_k = s["q"], s["k"], s["v"], s["cu_k"].long()
    k_lens, q_lens = _ints(s["case"]["k_lens"]), _ints(s["case"]["q_lens"])
    t, hq, d = q.shape
    hk, n = k.shape[1], len(k_lens)
    cu_q = s["cu_q"].long() if q_lens else torch.arange(n + 1, device=q.device)
    rows, keys = max(q_lens or [1]), max(k_lens)
    if keys == 0 or t == 0:
        return torch.zeros_like(q)
    # packed to [sequence, place], padded to the longest
    place = torch.arange(keys, device=q.device)
    real = place < (cu_k[1:] - cu_k[:-1])[:, None]
    at = (cu_k[:-1, None] + place).clamp(max=k.shape[0] - 1)
    kf, vf = k[at].float().transpose(1, 2), v[at].float().transpose(1, 2)
    row = torch.arange(rows, device=q.device)
    qf = q[(cu_q[:-1, None] + row).clamp(max=t - 1)].float().view(n, rows, hk, -1, d).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, d)
    p = torch.matmul(qf, kf.transpose(-1, -2)).mul_(d ** -0.5).masked_fill_(~real[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()  # rows without keys: all 0
    o = torch.matmul(p, vf) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.view(n, hk, hq // hk, rows, d).permute(0, 3, 1, 2, 4).reshape(n * rows, hq, d)
    token = torch.arange(t, device=q.device)
    seq = torch.searchsorted(cu_q[1:], token, right=True)
    return o[seq * rows + token - cu_q[seq]].to(q.dtype)


def _run_file(s):
    if own:
        from ai_engine_b200 import attention
        attention.kv4_file(s["k"], s["v"], s["kp"], s["vp"], s["slots"])
        return attention.kv4_load(s["kp"], s["vp"], s["slots"], dtype=s["k"].dtype)
    return _plain_file(s["k"], s["kp"], s["slots"]), _plain_file(s["v"], s["vp"], s["slots"])


def _plain_file(x, cache, slots):
    n, d = cache.shape[2], x.shape[2]
    codes, pairs = _planes(cache, d)
    keep = slots >= 0
    page, place = slots[keep] // n, slots[keep] % n
    code, pair = _bytes(*_quantise(x[keep]))
    codes[page, :, place], pairs[page, :, place] = code, pair
    # back out of the cache; what was not filed is zeros
    page, place = slots.clamp(min=0) // n, slots.clamp(min=0) % n
    return torch.where(keep[:, None, None], _values(codes[page, :, place], pairs[page, :, place]), 0.0).to(x.dtype)


def _run_kv4(s):
    q, kp, vp, table, lens, case = s["q"], s["kp"], s["vp"], s["table"], s["lens"], s["case"]
    if own:
        from ai_engine_b200 import attention
        return attention.kv4_attention(q, kp, vp, table, lens, max_len=case["longest"])
    b, hq, d = q.shape
    hk, n = kp.shape[1], kp.shape[2]
    qf = q.float().view(b, hk, hq // hk, d)
    row = table.long().clamp(min=0)
    # [stream, page, head, place, d] -> [stream, head, places, d]
    kf, vf = (_values(*(x[row] for x in _planes(c, d))).transpose(1, 2).flatten(2, 3) for c in (kp, vp))
    sc = torch.matmul(qf, kf.transpose(-1, -2)) * d ** -0.5
    sc.masked_fill_(torch.arange(kf.shape[2], device=q.device) >= lens[:, None, None, None], -math.inf)
    p = (sc - sc.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    return (torch.matmul(p, vf) / p.sum(-1, keepdim=True).clamp(min=1e-30)).reshape(b, hq, d).to(q.dtype)


# ------------------------------------------------------------------- work ---

def work(case):
    op, hk, d = case["op"], case["kv_heads"], case["dim"]
    if op == "axes":
        t, hq, pairs = _tokens(case), case["q_heads"], sum(_ints(case["sections"]))
        elems = 2 * t * (hq + hk) * d + (t * hk * d * 3 if case["cached"] else 0)
        rows = min(t, case["frames"] + case["height"] + case["width"] + case["text"])  # of the table, each read once
        return {"bytes": 2 * elems + t * (12 + (8 if case["cached"] else 0)) + 8 * pairs * rows, "flops": 8 * t * (hq + hk) * d}
    if op == "cross":
        k_lens, q_lens, hq = _ints(case["k_lens"]), _ints(case["q_lens"]), case["q_heads"]
        q_lens = q_lens or [1] * len(k_lens)
        pairs = sum(a * b for a, b in zip(q_lens, k_lens))
        return {"bytes": 2 * (sum(q_lens) * 2 * hq + sum(k_lens) * 2 * hk) * d, "flops": 4 * pairs * hq * d}
    if op == "file":  # in 16 bits, into the cache's 5 an element, out of it and in 16 bits again
        return {"bytes": case["tokens"] * (2 * hk * d * (2 + 0.625 + 0.625 + 2) + 16), "flops": 6 * case["tokens"] * 2 * hk * d}
    places = sum(_stream_lens(case))
    return {"bytes": places * 2 * hk * d * 0.625 + 4 * case["batch"] * case["q_heads"] * d, "flops": 4 * places * case["q_heads"] * d}


# ------------------------------------------------------------------ exact ---

def exact(case, seed):
    s = prepare(case, seed)
    return {"axes": _exact_axes, "cross": _exact_cross, "file": _exact_file, "kv4": _exact_kv4}[case["op"]](case, s)


def _exact_axes(case, s):
    axis = s["axis"].tolist()
    half = len(axis)

    def turn(x, w):
        x = x.double()
        y = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
        out = y.clone()
        for i, ax in enumerate(axis):
            j, k = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
            c, sn = (s["table"][s["pos"][:, ax].long(), i + m].double()[:, None] for m in (0, half))
            out[..., j] = c * y[..., j] - sn * y[..., k]
            out[..., k] = sn * y[..., j] + c * y[..., k]
        return out

    q, k = turn(s["q"], s["wq"]), turn(s["k"], s["wk"])
    if not case["cached"]:
        return q, k
    kp, vp = s["kp"].double(), s["vp"].double()
    keep = s["slots"] >= 0
    page, at = s["slots"][keep] // case["page"], s["slots"][keep] % case["page"]
    kp[page, at], vp[page, at] = k[keep], s["v"][keep].double()
    return q, k, kp, vp


def _attend(q, k, v):
    """softmax(q k^T / sqrt(d)) v of one key head's queries [rows, d], in 64 bits; zeros without keys."""
    return torch.softmax(q @ k.T / math.sqrt(q.shape[-1]), -1) @ v if k.shape[0] else torch.zeros_like(q)


def _exact_cross(case, s):
    k_lens, q_lens = _ints(case["k_lens"]), _ints(case["q_lens"])
    group, out = case["q_heads"] // case["kv_heads"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    row = key = 0
    for m, n in zip(q_lens or [1] * len(k_lens), k_lens):
        for h in range(case["q_heads"]):
            k, v = (x[key:key + n, h // group].double() for x in (s["k"], s["v"]))
            out[row:row + m, h] = _attend(s["q"][row:row + m, h].double(), k, v)
        row, key = row + m, key + n
    return out


def _exact_file(case, s):
    def stored(x):
        x = x.double().reshape(*x.shape[:2], -1, 32)
        lo = x.min(-1, keepdim=True).values.half().double()
        s_ = ((x.max(-1, keepdim=True).values - lo) / 15).half().double()
        code = torch.where(s_ > 0, (x - lo) / s_, 0).round().clip(0, 15)
        return (lo + s_ * code).flatten(-2) * (s["slots"] >= 0)[:, None, None]

    return stored(s["k"]), stored(s["v"])


def _exact_kv4(case, s):
    d, page, group = case["dim"], case["page"], case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")

    def read(cache, pages, h, n):
        block = cache[pages, h].reshape(len(pages), -1)
        code, meta = block[:, :page * d // 2].reshape(-1, d // 2)[:n].int(), block[:, page * d // 2:].contiguous().view(torch.float16)
        meta = meta.reshape(-1, d // 32, 2)[:n].double()
        x = torch.zeros(n, d, dtype=torch.float64, device="cuda")
        x[:, 0::2], x[:, 1::2] = (code % 16).double(), (code // 16).double()
        return (x.view(n, -1, 32) * meta[..., :1] + meta[..., 1:]).view(n, d)

    for b, n in enumerate(_stream_lens(case)):
        pages = s["table"][b, : -(-n // page)].long()
        for h in range(case["kv_heads"] if n else 0):
            rows = slice(h * group, (h + 1) * group)
            out[b, rows] = _attend(s["q"][b, rows].double(), read(s["kp"], pages, h, n), read(s["vp"], pages, h, n))
    return out
