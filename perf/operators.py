"""Sequence operators of a serving loop over video streams, as measured cases.

Four operators that belong together: the norm of queries and keys with the
position rotation (which also files keys and values into the paged cache),
attention over whole packed prompts, one-token attention for a batch of
streams that share a long prefix, and the upkeep of the cache's pages (fork,
copy, free, compact).

``own`` False: plain torch forms in 32 bits, rounded once at the end.
``own`` True: the framework's entry points.  ``exact`` gives the operators'
definitions in 64 bits, written apart from both.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------ cases ---

def listed():
    return [
        # one decode step of eight small streams: the call's latency
        dict(name="rope_step_8", op="rope", lens="1," * 7 + "1", q_heads=16, kv_heads=4, dim=64, rot=64, interleaved=False,
             dtype="f16", cached=True, page=16),
        # ragged prompts, half of each head rotated, neighbouring pairs, nothing cached
        dict(name="rope_ragged_1237", op="rope", lens="1,701,35,500", q_heads=20, kv_heads=5, dim=96, rot=48, interleaved=True,
             dtype="bf16", cached=False, page=16),
        # a batch of long prompts entering the cache: memory-bound
        dict(name="rope_fill_16384", op="rope", lens="8192,4096,4000,96", q_heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, dtype="bf16", cached=True, page=64),
        # one 160x288 frame at stride 16 (10 x 18 tokens), every token sees every other: latency
        dict(name="prompt_frame_180", op="prompt", lens="180", q_heads=8, kv_heads=8, dim=64, causal=False, dtype="f16"),
        # packed prompts of many lengths, one token to a few hundred
        dict(name="prompt_packed_40", op="prompt", lens=",".join(str(1 + (i * 311) % 719) for i in range(40)), q_heads=32,
             kv_heads=8, dim=128, causal=True, dtype="bf16"),
        # two long prompts, the second of an odd length: matrix-product bound
        dict(name="prompt_long_14193", op="prompt", lens="8192,6001", q_heads=32, kv_heads=8, dim=128, causal=True,
             dtype="bf16"),
        # four streams behind a short instruction that ends inside a page: latency
        dict(name="prefix_4x200", op="prefix", batch=4, q_heads=8, kv_heads=2, dim=64, page=16, prefix=200, suffix=40,
             dtype="f16"),
        # an ordinary batch, odd in size, behind a prompt of a few thousand tokens
        dict(name="prefix_33x4001", op="prefix", batch=33, q_heads=32, kv_heads=8, dim=128, page=16, prefix=4001, suffix=500,
             dtype="bf16"),
        # a full batch behind a long document
        dict(name="prefix_256x32768", op="prefix", batch=256, q_heads=32, kv_heads=4, dim=128, page=64, prefix=32768,
             suffix=1000, dtype="bf16"),
        # a short prompt forked for four streams: latency
        dict(name="fork_4", op="pages", kind="fork", layers=2, pages=64, page=16, kv_heads=2, dim=64, rows=8, sources=1,
             take=4, longest=200, dtype="f16"),
        # several prompts forked for many streams over a deep cache
        dict(name="fork_96", op="pages", kind="fork", layers=24, pages=1024, page=16, kv_heads=8, dim=64, rows=128, sources=12,
             take=96, longest=900, dtype="bf16"),
        # half of the streams end, the rest move to the front of the cache: memory-bound
        dict(name="compact_1024", op="pages", kind="compact", layers=32, pages=1024, page=16, kv_heads=8, dim=128, rows=64,
             sources=64, take=32, longest=250, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "prompt", "prefix", "pages"])
    dtype = rng.choice(["bf16", "f16"])
    kv, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 4, 7, 8])
    if kv * group > 32:
        group = 4
    page = rng.choice([16, 32, 64])
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128])
        lens, total = [], _log(rng, 1, 16384)
        while sum(lens) < total:
            lens.append(min(total - sum(lens), _log(rng, 1, 8192)))
            if len(lens) == 200:
                lens[-1] = max(1, total - sum(lens[:-1]))
                break
        return dict(op=op, lens=",".join(map(str, lens)), q_heads=kv * group, kv_heads=kv, dim=dim,
                    rot=rng.choice([dim, dim // 2]), interleaved=rng.random() < 0.3, dtype=rng.choice([dtype, dtype, "f32"]),
                    cached=rng.random() < 0.6, page=page)
    if op == "prompt":
        dim = rng.choice([64, 80, 128])
        n, top = _log(rng, 1, 64), _log(rng, 8, 8192)
        # the plain form pads to the longest prompt
        top = min(top, int(math.sqrt(0.75 * 8192 * 8192 / n)))
        lens = [top] + [_log(rng, 1, top) for _ in range(n - 1)]
        return dict(op=op, lens=",".join(map(str, lens)), q_heads=kv * group, kv_heads=kv, dim=dim,
                    causal=rng.random() < 0.8, dtype=dtype)
    if op == "prefix":
        return dict(op=op, batch=_log(rng, 1, 256), q_heads=kv * group, kv_heads=kv, dim=rng.choice([64, 128]), page=page,
                    prefix=rng.choice([0, _log(rng, 16, 32768), _log(rng, 16, 32768)]), suffix=_log(rng, 1, 1000), dtype=dtype)
    kind = rng.choice(["fork", "copy", "compact"])
    rows, longest = _log(rng, 4, 128), _log(rng, 16, 500)
    pages = rows * (-(-longest // page)) + 8
    layers = min(rng.choice([1, 4, 12, 32]), max(1, 2_000_000_000 // (pages * page * kv * 64 * 4)))
    sources = rows if kind == "compact" else max(1, rows // 4)
    return dict(op=op, kind=kind, layers=layers, pages=pages, page=page, kv_heads=kv, dim=64, rows=rows, sources=sources,
                take=rows // 2, longest=longest, dtype=dtype)


def _lens(case):
    return [int(x) for x in case["lens"].split(",")]


def _suffix_lens(case):
    """What each stream of a prefix case has said of its own: 0 to `suffix` tokens, none for some."""
    return [(b * 7919 + 13) % (case["suffix"] + 1) for b in range(case["batch"])]


def _row_lens(case):
    """Tokens of the rows in use in a pages case: 1 to `longest`, whole pages now and then."""
    return [1 + (r * 389 + case["longest"] - 1) % case["longest"] for r in range(case["sources"])]


# ----------------------------------------------------------------- inputs ---

def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed))
    return dict({"rope": _prepare_rope, "prompt": _prepare_prompt, "prefix": _prepare_prefix, "pages": _prepare_pages}[
        case["op"]](case, g), case=case)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def _prepare_rope(case, g):
    lens, dt = _lens(case), DTYPES[case["dtype"]]
    t, hq, hk, d, rot = sum(lens), case["q_heads"], case["kv_heads"], case["dim"], case["rot"]
    # the projection's output: one buffer with all heads of a token side by side
    qkv = (2.0 * _randn(g, t, hq + 2 * hk, d)).to(dt)
    top = 8192 + 64
    freq = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") / max(1, rot // 2))
    ang = torch.arange(top, dtype=torch.float64, device="cuda")[:, None] * freq
    first = torch.randint(0, 64, (len(lens),), generator=g, device="cuda", dtype=torch.int32)
    n = torch.tensor(lens, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), n)
    cu = _cu(lens)
    pos = torch.arange(t, device="cuda", dtype=torch.int32) - cu[seq] + first[seq]
    s = dict(q=qkv[:, :hq], k=qkv[:, hq:hq + hk], v=qkv[:, hq + hk:], pos=pos,
             table=torch.cat([ang.cos(), ang.sin()], 1).float().contiguous(),
             wq=1.0 + 0.2 * _randn(g, d), wk=1.0 + 0.2 * _randn(g, d))
    if case["cached"]:
        pages = -(-t // case["page"]) + 3
        s["kp"] = torch.zeros(pages, case["page"], hk, d, dtype=dt, device="cuda")
        s["vp"] = torch.zeros_like(s["kp"])
        # every prompt's tokens side by side in pages of a random order; the last token is not filed
        perm = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(t, device="cuda")
        s["slots"] = perm[at // case["page"]] * case["page"] + at % case["page"]
        if t > 1:
            s["slots"][-1] = -1
    return s


def _qkv(g, t, hq, hk, d, dt):
    """Normed and rotated heads: rows of unit variance, a few key channels that stand out."""
    x = _randn(g, t, hq + 2 * hk, d)
    gain = torch.ones(d, device="cuda")
    gain[:: max(1, d // 4)] = 3.0
    x[:, hq:hq + hk] *= gain
    return x.to(dt)


def _prepare_prompt(case, g):
    lens = _lens(case)
    hq, hk = case["q_heads"], case["kv_heads"]
    x = _qkv(g, sum(lens), hq, hk, case["dim"], DTYPES[case["dtype"]])
    return dict(q=x[:, :hq], k=x[:, hq:hq + hk], v=x[:, hq + hk:], cu=_cu(lens))


def _prepare_prefix(case, g):
    b, hq, hk, d, page = case["batch"], case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    dt, pre = DTYPES[case["dtype"]], case["prefix"]
    own_lens = _suffix_lens(case)
    shared = pre // page                                  # whole pages that every stream has in common
    width = -(-(pre + case["suffix"]) // page) + 1
    need = -(-pre // page) + b * (width - shared)
    kv = torch.empty(2, need + 5, page, hk, d, dtype=dt, device="cuda")
    for half in kv:
        half.copy_(_randn(g, *half.shape))
    kv[0, :, :, :, :: max(1, d // 4)] *= 3.0
    order = torch.randperm(need + 5, generator=g, device="cuda").to(torch.int32)
    prefix = order[: -(-pre // page)].contiguous()
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    table[:, :shared] = prefix[:shared]
    table[:, shared:] = order[prefix.numel(): prefix.numel() + b * (width - shared)].view(b, -1)
    lens = torch.tensor(own_lens, dtype=torch.int32, device="cuda") + pre
    return dict(q=_randn(g, b, hq, d).to(dt), kp=kv[0], vp=kv[1], prefix=prefix, table=table, lens=lens)


def _prepare_pages(case, g):
    page, rows, pages = case["page"], case["rows"], case["pages"]
    kv = torch.empty(case["layers"], 2, pages, page, case["kv_heads"], case["dim"], dtype=DTYPES[case["dtype"]], device="cuda")
    for layer in kv:
        layer.copy_(_randn(g, *layer.shape))
    lens = _row_lens(case)
    width = -(-case["longest"] // page) + 1
    counts = [-(-n // page) for n in lens]
    # the rows' integers in one buffer, so that one copy sets a pass's state: refs, lens, table, status
    ints = torch.zeros(pages + rows + rows * width + 1, dtype=torch.int32, device="cuda")
    refs, row_lens, table = ints[:pages], ints[pages:pages + rows], ints[pages + rows:-1].view(rows, width)
    table.fill_(-1)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    used = 0
    for r, (n, c) in enumerate(zip(lens, counts)):
        table[r, :c] = order[used:used + c]
        used += c
    refs[order[:used].long()] = 1
    row_lens[: len(lens)] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s = dict(kv=kv, ints=ints, ints0=ints.clone())
    if case["kind"] == "fork":
        s["src"] = torch.tensor([i % case["sources"] for i in range(_forks(case))], dtype=torch.int32, device="cuda")
        s["dst"] = torch.arange(case["sources"], case["sources"] + _forks(case), dtype=torch.int32, device="cuda")
    elif case["kind"] == "copy":
        n = min(used, pages - used)
        s["src"], s["dst"] = order[:n].contiguous(), order[pages - n:].contiguous()
    else:
        pick = torch.randperm(case["sources"], generator=g, device="cuda")[: case["take"]]
        s["gone"] = pick.to(torch.int32)
    return s


def _forks(case):
    return min(case["take"], case["rows"] - case["sources"])


def _ints(case, ints):
    p, r = case["pages"], case["rows"]
    return ints[:p], ints[p:p + r], ints[p + r:-1].view(r, -1), ints[-1:]


# ---------------------------------------------------------------- a pass ---

def run(state):
    return {"rope": _run_rope, "prompt": _run_prompt, "prefix": _run_prefix, "pages": _run_pages}[state["case"]["op"]](state)


def _run_rope(s):
    case = s["case"]
    if own:
        from ai_engine_b200 import attention
        q, k = attention.qk_norm_rope(s["q"], s["k"], s["pos"], s["table"], q_weight=s["wq"], k_weight=s["wk"], eps=EPS,
                                      interleaved=case["interleaved"], v=s["v"] if case["cached"] else None,
                                      k_pages=s.get("kp"), v_pages=s.get("vp"), slots=s.get("slots"))
    else:
        q = _plain_norm_rope(s["q"], s["wq"], s["pos"], s["table"], case)
        k = _plain_norm_rope(s["k"], s["wk"], s["pos"], s["table"], case)
        if case["cached"]:
            keep = s["slots"] >= 0
            at = s["slots"][keep]
            s["kp"].view(-1, case["kv_heads"], case["dim"])[at] = k[keep]
            s["vp"].view(-1, case["kv_heads"], case["dim"])[at] = s["v"][keep]
    return (q, k, s["kp"], s["vp"]) if case["cached"] else (q, k)


def _plain_norm_rope(x, w, pos, table, case):
    rot = case["rot"]
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w
    cs = table[pos.long()][:, None]
    cos, sin = cs[..., :rot // 2], cs[..., rot // 2:]
    if case["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _run_prompt(s):
    case = s["case"]
    if own:
        from ai_engine_b200 import attention
        return attention.prompt_attention(s["q"], s["k"], s["v"], s["cu"], causal=case["causal"])
    q, k, v, cu = s["q"], s["k"], s["v"], s["cu"].long()
    t, hq, d = q.shape
    hk = k.shape[1]
    lens = _lens(case)
    n, top = len(lens), max(lens)
    # packed tokens to [sequence, place], padded to the longest
    at = cu[:-1, None] + torch.arange(top, device=q.device)
    real = at < cu[1:, None]
    at = at.clamp(max=t - 1)
    qf = q[at].float().view(n, top, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, hq // hk * top, d)
    kf, vf = k[at].float().transpose(1, 2), v[at].float().transpose(1, 2)
    p = torch.matmul(qf, kf.transpose(-1, -2)).view(n, hk, hq // hk, top, top)
    p.mul_(d ** -0.5).masked_fill_(~real[:, None, None, None], -math.inf)
    if case["causal"]:
        place = torch.arange(top, device=q.device)
        p.masked_fill_(place > place[:, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    norm = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, hk, -1, top), vf).view(n, hk, hq // hk, top, d) / norm
    o = o.permute(0, 3, 1, 2, 4).reshape(n * top, hq, d)
    # back to packed: token i of sequence b stands at b * top + i
    seq = torch.searchsorted(cu[1:], torch.arange(t, device=q.device), right=True)
    return o[seq * top + torch.arange(t, device=q.device) - cu[seq]].to(q.dtype)


def _run_prefix(s):
    case = s["case"]
    q, kp, vp, table, lens, pre = s["q"], s["kp"], s["vp"], s["table"], s["lens"], case["prefix"]
    if own:
        from ai_engine_b200 import attention
        return attention.prefix_attention(q, kp, vp, s["prefix"], pre, table, lens, max_len=pre + case["suffix"])
    b, hq, d = q.shape
    page, hk = kp.shape[1], kp.shape[2]
    qf = q.float().view(b, hk, hq // hk, d)
    # the shared part, read once for all
    kf, vf = (x[s["prefix"].long()].reshape(-1, hk, d)[:pre].float() for x in (kp, vp))
    sp = torch.einsum("bhgd,lhd->bhgl", qf, kf) * d ** -0.5
    # each stream's own part, from the page in which the prefix ends
    own_pages = table[:, pre // page:].long().clamp(min=0)
    ks, vs = (x[own_pages].flatten(1, 2).float() for x in (kp, vp))
    place = pre // page * page + torch.arange(ks.shape[1], device=q.device)
    real = (place >= pre) & (place < lens[:, None])
    so = torch.einsum("bhgd,blhd->bhgl", qf, ks) * d ** -0.5
    so.masked_fill_(~real[:, None, None], -math.inf)
    top = torch.maximum(so.amax(-1), sp.amax(-1) if pre else so.new_tensor(-math.inf)).clamp(min=-1e30)[..., None]
    sp, so = (sp - top).exp(), (so - top).exp()
    norm = sp.sum(-1) + so.sum(-1)
    o = torch.einsum("bhgl,lhd->bhgd", sp, vf) + torch.einsum("bhgl,blhd->bhgd", so, vs)
    return (o / norm.clamp(min=1e-30)[..., None]).reshape(b, hq, d).to(q.dtype)


def _run_pages(s):
    case, kv, ints = s["case"], s["kv"], s["ints"]
    ints.copy_(s["ints0"])  # the integers of the state at the start of the pass
    refs, lens, table, status = _ints(case, ints)
    if own:
        from ai_engine_b200 import pages
        st = pages.PageState(refs, lens, table, status)
        if case["kind"] == "fork":
            pages.fork(kv, st, s["src"], s["dst"])
        elif case["kind"] == "copy":
            pages.copy(kv, s["src"], s["dst"])
        else:
            pages.free(st, s["gone"])
            return kv, ints, pages.compact(kv, st)
        return kv, ints
    page = case["page"]
    if case["kind"] == "fork":
        src, dst = s["src"].long(), s["dst"].long()
        n = lens[src]
        whole, tail = n // page, n % page > 0
        # the lowest free pages, one for each prompt that ends inside a page
        fresh = torch.nonzero(refs == 0).view(-1)
        mine = fresh[(torch.cumsum(tail, 0) - 1).clamp(min=0)].to(torch.int32)
        row = table[src]
        at = torch.arange(table.shape[1], device=kv.device)
        last = row.gather(1, whole.long()[:, None].clamp(max=table.shape[1] - 1))[:, 0]
        kv[:, :, mine[tail].long()] = kv[:, :, last[tail].long()]
        shared = at < whole[:, None]
        refs.index_add_(0, row[shared].long(), torch.ones_like(row[shared]))
        refs[mine[tail].long()] = 1
        end = (at == whole[:, None]) & tail[:, None]
        table[dst] = torch.where(shared, row, torch.where(end, mine[:, None], -1))
        lens[dst] = n
    elif case["kind"] == "copy":
        kv[:, :, s["dst"].long()] = kv[:, :, s["src"].long()]
    else:
        gone = s["gone"].long()
        row = table[gone]
        refs.index_add_(0, row[row >= 0].long(), -torch.ones_like(row[row >= 0]))
        table[gone], lens[gone] = -1, 0
        live = refs > 0
        front = torch.arange(case["pages"], device=kv.device) < live.sum()
        hole, late = torch.nonzero(front & ~live).view(-1), torch.nonzero(live & ~front).view(-1)
        kv[:, :, hole] = kv[:, :, late]
        refs[hole], refs[late] = refs[late], 0
        moved = torch.where(live, torch.arange(case["pages"], dtype=torch.int32, device=kv.device), -1)
        moved[late] = hole.to(torch.int32)
        table.copy_(torch.where(table >= 0, moved[table.long().clamp(min=0)], -1))
        return kv, ints, moved
    return kv, ints


# ------------------------------------------------------------------- work ---

def work(case):
    size, op = BYTES[case["dtype"]], case["op"]
    if op == "rope":
        t, hq, hk, d = sum(_lens(case)), case["q_heads"], case["kv_heads"], case["dim"]
        elems = 2 * t * (hq + hk) * d + (t * hk * d * 3 if case["cached"] else 0)
        return {"bytes": elems * size + t * (4 + 4 * case["rot"] + (8 if case["cached"] else 0)), "flops": 8 * t * (hq + hk) * d}
    if op == "prompt":
        lens, hq, hk, d = _lens(case), case["q_heads"], case["kv_heads"], case["dim"]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        return {"bytes": sum(lens) * (2 * hq + 2 * hk) * d * size, "flops": 4 * pairs * hq * d}
    if op == "prefix":
        b, hq, hk, d = case["batch"], case["q_heads"], case["kv_heads"], case["dim"]
        mine = sum(_suffix_lens(case))
        return {"bytes": ((case["prefix"] + mine) * hk * 2 * d + 2 * b * hq * d) * size,
                "flops": 4 * (b * case["prefix"] + mine) * hq * d}
    one = 2 * case["layers"] * case["page"] * case["kv_heads"] * case["dim"] * size
    ints = 4 * (case["pages"] + case["rows"] * (-(-case["longest"] // case["page"]) + 2) + 1)
    return {"bytes": 2 * one * _moved(case) + 4 * ints, "flops": 0}


def _moved(case):
    """Pages whose contents move, at the least (which rows end is left to chance: the mean of it)."""
    lens, page = _row_lens(case), case["page"]
    used = sum(-(-n // page) for n in lens)
    if case["kind"] == "fork":
        return sum(lens[i % case["sources"]] % page > 0 for i in range(_forks(case)))
    if case["kind"] == "copy":
        return min(used, case["pages"] - used)
    live = used * (1 - case["take"] / case["sources"])
    return max(1, int(live * (1 - live / case["pages"])))


# ------------------------------------------------------------------ exact ---

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "prompt": _exact_prompt, "prefix": _exact_prefix, "pages": _exact_pages}[case["op"]](case, s)


def _exact_rope(case, s):
    rot = case["rot"]

    def turn(x, w):
        x = x.double()
        y = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
        out = y.clone()
        for i in range(rot // 2):
            j, k = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
            c = s["table"][s["pos"].long(), i].double()[:, None]
            sn = s["table"][s["pos"].long(), i + rot // 2].double()[:, None]
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


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(d)) v of one head over the first seen[i] keys for row i, in 64 bits."""
    s = q @ k.T / math.sqrt(q.shape[-1])
    s = torch.where(torch.arange(k.shape[0], device=q.device) < seen[:, None], s, -math.inf)
    return torch.softmax(s, -1) @ v


def _exact_prompt(case, s):
    lens, group = _lens(case), case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for n in lens:
        seen = torch.arange(1, n + 1, device="cuda") if case["causal"] else torch.full((n,), n, device="cuda")
        for h in range(case["q_heads"]):
            q, k, v = s["q"][at:at + n, h], s["k"][at:at + n, h // group], s["v"][at:at + n, h // group]
            out[at:at + n, h] = _attend(q.double(), k.double(), v.double(), seen)
        at += n
    return out


def _exact_prefix(case, s):
    page, pre, group = case["page"], case["prefix"], case["q_heads"] // case["kv_heads"]
    lens = [pre + n for n in _suffix_lens(case)]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    kp, vp = (x.flatten(0, 1) for x in (s["kp"], s["vp"]))
    place = torch.arange(max(lens + [1]), device="cuda")
    for b, n in enumerate(lens):
        if n == 0:
            continue  # nothing to attend to: zeros
        pages = s["table"][b].long().clone()
        pages[: s["prefix"].numel()][: -(-pre // page)] = s["prefix"].long()
        at = pages[place[:n] // page] * page + place[:n] % page
        if pre % page:  # past the prefix, the page in which it ends is the stream's own
            at[pre:] = s["table"][b].long()[place[pre:n] // page] * page + place[pre:n] % page
        k, v = kp[at].double().transpose(0, 1), vp[at].double().transpose(0, 1)
        q = s["q"][b].double().view(case["kv_heads"], group, -1)
        w = torch.softmax(q @ k.transpose(1, 2) / math.sqrt(q.shape[-1]), -1)
        out[b] = (w @ v).reshape(-1, q.shape[-1])
    return out


def _exact_pages(case, s):
    refs, lens, table, _ = (x.tolist() for x in _ints(case, s["ints0"]))
    page, kv, moves, moved = case["page"], s["kv"], [], None
    if case["kind"] == "fork":
        free = [p for p, n in enumerate(refs) if n == 0]
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            lens[b] = lens[a]
            for i in range(lens[a] // page):
                table[b][i] = table[a][i]
                refs[table[a][i]] += 1
            if lens[a] % page:
                p = free.pop(0)
                refs[p], table[b][lens[a] // page] = 1, p
                moves.append((table[a][lens[a] // page], p))
    elif case["kind"] == "copy":
        moves = list(zip(s["src"].tolist(), s["dst"].tolist()))
    else:
        for r in s["gone"].tolist():
            for p in table[r]:
                if p >= 0:
                    refs[p] -= 1
            table[r], lens[r] = [-1] * len(table[r]), 0
        live = [p for p, n in enumerate(refs) if n > 0]
        holes = [p for p in range(len(live)) if refs[p] == 0]
        moves = list(zip([p for p in live if p >= len(live)], holes))
        moved = [p if refs[p] > 0 else -1 for p in range(case["pages"])]
        for a, b in moves:
            moved[a], refs[b], refs[a] = b, refs[a], 0
        table = [[moved[p] if p >= 0 else -1 for p in row] for row in table]
    kv = kv.clone()
    if moves:
        a, b = (torch.tensor(x, device="cuda") for x in zip(*moves))
        kv[:, :, b] = s["kv"][:, :, a]
    ints = torch.tensor(refs + lens + [p for row in table for p in row] + [0], dtype=torch.int32)
    out = kv.double(), ints
    return out if moved is None else (*out, torch.tensor(moved, dtype=torch.int32))
