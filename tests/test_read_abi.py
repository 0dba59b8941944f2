"""The C ABI of axes, attention to states and the 4-bit cache without a GPU:
argument layouts and refusals, all of which come before any CUDA call."""
import os
import subprocess

import pytest
import torch

from ai_engine_b200 import _lib, attention, pages
from ai_engine_b200.build import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # stands for a device pointer; never followed
F16, F32 = _lib.DT_F16, _lib.DT_F32


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


def test_packed_arguments_match_the_header(tmp_path):
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include "aie_seq.h"\nint main(void) {'
                   'printf("%zu %zu %zu %zu %zu %zu", sizeof(aie_cross), offsetof(aie_cross, scale), sizeof(aie_kv4_rows),'
                   'offsetof(aie_kv4_rows, dtype), sizeof(aie_kv4_step), offsetof(aie_kv4_step, scale)); return 0; }')
    exe = tmp_path / "p"
    subprocess.run(["gcc", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [_lib.CROSS.size, _lib.CROSS.size - 4, _lib.KV4_ROWS.size, _lib.KV4_ROWS.size - 4, _lib.KV4_STEP.size,
                   _lib.KV4_STEP.size - 4]


def axes(lib, axis=P, axes_=3, tokens=3, rot=64, pos=P, ko=(P, 256, 64)):
    p = _lib.QK_ROPE.pack(P, 256, 64, P, 256, 64, 0, 0, 0, P, 256, 64, *ko, *(0,) * 7, P, P, P, pos, 0, tokens, 4, 2, 64, rot, 100,
                          F16, 0, 1e-6, 0)
    return lib.aie_qk_norm_rope_axes(p, axis, axes_, None)


def test_axes_refuse(lib):
    assert axes(lib, tokens=0) == 0
    for kw, status in [(dict(axes_=0), -2), (dict(axes_=256), -2), (dict(axis=None), -2), (dict(rot=66), -2), (dict(pos=0), -2),
                       (dict(ko=(0, 0, 0)), -2)]:
        assert axes(lib, **kw) == status and _lib.last_error()
    assert lib.aie_qk_norm_rope_axes(None, P, 3, None) == -2


def cross_args(q=(P, 256, 64), k=(P, 256, 64), v=(P, 256, 64), out=(P, 256, 64), cu_q=P, cu_k=P, ws=P, wb=1 << 40, tokens=5, keys=9,
               seqs=2, hq=4, hk=2, d=64, dt=F16, scale=1.0):
    return _lib.CROSS.pack(*q, *k, *v, *out, cu_q, cu_k, ws, wb, tokens, keys, seqs, hq, hk, d, dt, scale)


@pytest.mark.parametrize("kw, status", [
    (dict(dt=9), -2), (dict(hq=5), -2), (dict(hk=0), -2), (dict(d=0), -2), (dict(d=257), -3), (dict(cu_k=0), -2), (dict(cu_q=0), -2),
    (dict(v=(0, 0, 0)), -2), (dict(out=(0, 0, 0)), -2), (dict(out=(P + 1, 256, 64)), -5), (dict(scale=float("nan")), -2),
    (dict(tokens=1 << 31), -2), (dict(keys=1 << 31), -2), (dict(q=(P, 256, -64)), -2), (dict(hq=8192, hk=1), -3), (dict(ws=0), -2),
    (dict(wb=0), -2), (dict(ws=P + 8), -2),
])
def test_cross_refuses(lib, kw, status):
    assert lib.aie_cross_attn(cross_args(**kw), None) == status
    assert _lib.last_error()


def test_nothing_to_do_is_no_error(lib):
    assert lib.aie_cross_attn(cross_args(tokens=0), None) == 0 and lib.aie_cross_attn(cross_args(seqs=0), None) == 0
    assert lib.aie_kv4_file(rows(tokens=0), None) == 0 and lib.aie_kv4_load(rows(tokens=0), None) == 0
    assert lib.aie_kv4_attn(step(batch=0), None) == 0
    assert lib.aie_cross_attn_workspace(cross_args(hq=5)) == 0 and lib.aie_kv4_attn_workspace(step(hq=5)) == 0
    assert lib.aie_cross_attn_workspace(cross_args()) > 0 and lib.aie_kv4_attn_workspace(step()) > 0


# k v page_stride pages page_size kv_heads head_dim
CACHE = (P, P, 2 * 16 * 40, 8, 16, 2, 64)


def rows(cache=CACHE, k=(P, 128, 64), v=(P, 128, 64), slots=P, tokens=3, dt=F16):
    return _lib.KV4_ROWS.pack(*cache, *k, *v, slots, tokens, dt)


def step(cache=CACHE, q=(P, 256, 64), out=(P, 256, 64), table=P, lens=P, ws=P, wb=1 << 40, batch=3, hq=4, top=64, width=4, dt=F16,
         scale=1.0):
    return _lib.KV4_STEP.pack(*cache, *q, *out, table, lens, ws, wb, batch, hq, top, width, dt, scale)


BAD_CACHES = [((0, P, 1280, 8, 16, 2, 64), -2), ((P, 0, 1280, 8, 16, 2, 64), -2), ((P + 8, P, 1280, 8, 16, 2, 64), -5),
              ((P, P, 1288, 8, 16, 2, 64), -5), ((P, P, 1264, 8, 16, 2, 64), -2), ((P, P, 1280, 0, 16, 2, 64), -2),
              ((P, P, 1280, 8, 12, 2, 64), -2), ((P, P, 1280, 8, 0, 2, 64), -2), ((P, P, 1280, 8, 16, 0, 64), -2),
              ((P, P, 1280, 8, 16, 2, 48), -2), ((P, P, 1280, 8, 16, 2, 0), -2), ((P, P, 1 << 20, 8, 16, 2, 288), -3),
              ((P, P, -1280, 8, 16, 2, 64), -2)]


@pytest.mark.parametrize("kw, status", [(dict(cache=c), s) for c, s in BAD_CACHES] + [
    (dict(dt=7), -2), (dict(k=(0, 0, 0)), -2), (dict(v=(0, 0, 0)), -2), (dict(k=(P + 1, 128, 64)), -5), (dict(slots=0), -2),
    (dict(tokens=1 << 31), -3)])
def test_filing_and_reading_refuse(lib, kw, status):
    for call in (lib.aie_kv4_file, lib.aie_kv4_load):
        assert call(rows(**kw), None) == status
        assert _lib.last_error()


@pytest.mark.parametrize("kw, status", [(dict(cache=c), s) for c, s in BAD_CACHES] + [
    (dict(dt=F32), -3), (dict(dt=7), -3), (dict(hq=5), -2), (dict(batch=65536), -3), (dict(top=1 << 31), -2), (dict(lens=0), -2),
    (dict(table=0), -2), (dict(width=3), -2), (dict(q=(0, 0, 0)), -2), (dict(out=(P + 1, 256, 64)), -5), (dict(ws=0), -2),
    (dict(wb=8), -2), (dict(ws=P + 8), -2), (dict(scale=float("nan")), -2)])
def test_attention_over_4_bits_refuses(lib, kw, status):
    assert lib.aie_kv4_attn(step(**kw), None) == status
    assert _lib.last_error()


def test_python_refuses_host_tensors(lib):
    q, i = torch.zeros(3, 4, 64, dtype=torch.float16), torch.zeros(4, dtype=torch.int32)
    kv = pages.new_cache4(1, 8, 16, 4, 64, device="cpu")
    with pytest.raises(TypeError):
        attention.cross_attention(q, q, q, i)
    with pytest.raises(TypeError):
        attention.kv4_file(q, q, kv[0, 0], kv[0, 1], torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError):
        attention.kv4_load(kv[0, 0], kv[0, 1], torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError):
        attention.kv4_attention(q, kv[0, 0], kv[0, 1], i.view(1, 4), i[:1])
    with pytest.raises(TypeError):
        attention.qk_norm_rope(q, q, i, torch.zeros(4, 64), pair_axis=torch.zeros(32, dtype=torch.uint8))


def test_grid_of_a_clip():
    from ai_engine_b200 import decoder
    p = decoder.grid(2, 2, 3, device="cpu")
    assert p.dtype == torch.int32 and p.tolist() == [[t, r, c] for t in range(2) for r in range(2) for c in range(3)]
