"""The sequence operators' C ABI without a GPU: symbols, argument layouts and
refusals, all of which come before any CUDA call."""
import os
import re
import subprocess

import pytest
import torch

from ai_engine_b200 import _lib, attention, pages
from ai_engine_b200.build import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # stands for a device pointer; never followed
F16 = _lib.DT_F16


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


def test_header_declares_the_binding(lib):
    src = open(os.path.join(ROOT, "include", "aie_seq.h")).read()
    names = sorted(set(re.findall(r"AIE_API\s+[\w\s\*]*?\b(aie_\w+)\s*\(", src)))
    assert names == sorted(_lib.SEQ_SIGNATURES)
    for n in names:
        assert hasattr(lib, n)


def test_packed_arguments_match_the_header(tmp_path):
    # the header as C: each struct's size, and the offset of its last field
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include "aie_seq.h"\nint main(void) {'
                   'printf("%zu %zu %zu %zu %zu %zu", sizeof(aie_qk_rope), offsetof(aie_qk_rope, eps), sizeof(aie_prompt),'
                   'sizeof(aie_prefix), offsetof(aie_prefix, scale), sizeof(aie_pages)); return 0; }')
    exe = tmp_path / "p"
    subprocess.run(["gcc", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [_lib.QK_ROPE.size, _lib.QK_ROPE.size - 8, _lib.PROMPT.size, _lib.PREFIX.size, _lib.PREFIX.size - 8,
                   _lib.PAGES.size]


def rope(lib, q=(P, 256, 64), k=(P, 256, 64), v=(0, 0, 0), qo=(P, 256, 64), ko=(P, 256, 64), cache=(0,) * 7, wq=P, wk=P,
         cs=P, pos=P, slots=0, tokens=3, hq=4, hk=2, d=64, rot=64, top=100, dt=F16):
    return lib.aie_qk_norm_rope(_lib.QK_ROPE.pack(*q, *k, *v, *qo, *ko, *cache, wq, wk, cs, pos, slots, tokens, hq, hk, d,
                                                  rot, top, dt, 0, 1e-6, 0), None)


@pytest.mark.parametrize("kw, status", [
    (dict(dt=3), -2), (dict(dt=-1), -2), (dict(hq=3), -2), (dict(hk=0), -2), (dict(d=0, rot=0), -2), (dict(d=514), -3),
    (dict(rot=66), -2), (dict(rot=7), -2), (dict(k=(0, 0, 0)), -2), (dict(q=(P + 1, 256, 64)), -5),
    (dict(q=(0, 0, 0)), -2), (dict(qo=(0, 0, 0)), -2), (dict(pos=0), -2), (dict(cs=0), -2), (dict(ko=(0, 0, 0)), -2),
    (dict(k=(P, -256, 64)), -2), (dict(cache=(P, P, 64, 64, 64, 8, 16)), -2),
    (dict(cache=(P, P, 64, 64, 64, 8, 16), v=(P, 64, 64)), -2),
    (dict(cache=(P, 0, 64, 64, 64, 8, 16), v=(P, 64, 64), slots=P), -2),
    (dict(cache=(P, P, 64, 64, 64, 0, 16), v=(P, 64, 64), slots=P), -2),
])
def test_norm_rope_refuses(lib, kw, status):
    assert rope(lib, **kw) == status
    assert _lib.last_error()


def test_nothing_to_do_is_no_error(lib):
    assert rope(lib, tokens=0) == 0
    assert prompt(lib, tokens=0) == 0 and prompt(lib, seqs=0) == 0
    assert prefix(lib, batch=0) == 0
    assert lib.aie_pages_fork(page_args(), None, None, 0, None) == 0
    assert lib.aie_pages_free(page_args(), None, 0, None) == 0
    assert lib.aie_pages_grow(page_args(), None, None, 0, None, 0, None) == 0


def prompt(lib, q=(P, 256, 64), k=(P, 256, 64), v=(P, 256, 64), out=(P, 256, 64), cu=P, tokens=5, seqs=1, hq=4, hk=2, d=64,
           dt=F16, scale=1.0):
    return lib.aie_prompt_attn(_lib.PROMPT.pack(*q, *k, *v, *out, cu, tokens, seqs, hq, hk, d, dt, 1, scale), None)


@pytest.mark.parametrize("kw, status", [
    (dict(dt=9), -2), (dict(hq=5), -2), (dict(hk=0), -2), (dict(d=0), -2), (dict(d=257), -3), (dict(cu=0), -2),
    (dict(v=(0, 0, 0)), -2), (dict(out=(0, 0, 0)), -2), (dict(out=(P + 1, 256, 64)), -5), (dict(scale=float("nan")), -2),
    (dict(tokens=1 << 31), -2), (dict(q=(P, 256, -64)), -2), (dict(hq=8192, hk=1), -3),
])
def test_prompt_refuses(lib, kw, status):
    assert prompt(lib, **kw) == status
    assert _lib.last_error()


def prefix(lib, q=(P, 256, 64), out=(P, 256, 64), cache=(P, P, 2048, 128, 64, 8, 16), pre=P, table=P, lens=P, ws=P, wb=1 << 30,
           batch=3, hq=4, hk=2, d=64, shared=20, top=64, width=4, dt=F16, scale=1.0):
    return lib.aie_prefix_attn(_lib.PREFIX.pack(*q, *out, *cache, pre, table, lens, ws, wb, batch, hq, hk, d, shared, top,
                                                width, dt, scale, 0), None)


@pytest.mark.parametrize("kw, status", [
    (dict(dt=9), -2), (dict(hq=5), -2), (dict(d=257), -3), (dict(batch=65536), -3), (dict(lens=0), -2), (dict(pre=0), -2),
    (dict(table=0), -2), (dict(width=3), -2), (dict(ws=0), -2), (dict(wb=0), -2), (dict(ws=P + 8), -2),
    (dict(q=(0, 0, 0)), -2), (dict(cache=(0, P, 2048, 128, 64, 8, 16)), -2), (dict(cache=(P, P, 2048, 128, 64, 8, 0)), -2),
    (dict(cache=(P + 1, P, 2048, 128, 64, 8, 16)), -5), (dict(scale=float("nan")), -2), (dict(top=1 << 31), -2),
])
def test_prefix_refuses(lib, kw, status):
    assert prefix(lib, **kw) == status
    assert _lib.last_error()


def page_args(kv=P, refs=P, lens=P, table=P, status=P, ws=P, nbytes=4096, layers=2, pages=8, size=16, rows=4, width=3):
    return _lib.PAGES.pack(kv, refs, lens, table, status, ws, nbytes, layers, pages, size, rows, width, 0)


@pytest.mark.parametrize("kw, status", [
    (dict(kv=0), -2), (dict(kv=P + 8), -5), (dict(nbytes=4100), -5), (dict(layers=0), -2), (dict(pages=0), -2),
    (dict(refs=0), -2), (dict(table=0), -2), (dict(status=0), -2), (dict(size=0), -2), (dict(rows=0), -2), (dict(width=0), -2),
    (dict(rows=(1 << 18) + 1), -3), (dict(width=1 << 28), -3), (dict(ws=0), -2), (dict(ws=P + 4), -2),
])
def test_fork_refuses(lib, kw, status):
    assert lib.aie_pages_fork(page_args(**kw), P, P, 1, None) == status
    assert _lib.last_error()


def test_page_lists_are_checked(lib):
    assert lib.aie_pages_fork(page_args(), None, P, 1, None) == -2
    assert lib.aie_pages_fork(page_args(), P, P, (1 << 20) + 1, None) == -3
    assert lib.aie_pages_copy(page_args(), P, None, 1, None) == -2
    assert lib.aie_pages_free(page_args(), None, 1, None) == -2
    assert lib.aie_pages_grow(page_args(), P, None, 1, P, 4, None) == -2
    assert lib.aie_pages_grow(page_args(), P, P, 1, None, 4, None) == -2
    assert lib.aie_pages_compact(page_args(), None, None) == -2


def test_python_refuses_host_tensors(lib):
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(TypeError):
        attention.prompt_attention(q, q, q, i)
    with pytest.raises(TypeError):
        attention.qk_norm_rope(q, q, i, torch.zeros(4, 64))
    with pytest.raises(TypeError):
        attention.prefix_attention(q, q, q, None, 0, i, i)
    st = pages.new_state(8, 4, 3, device="cpu")
    kv = pages.new_cache(1, 8, 16, 2, 64, device="cpu")
    with pytest.raises((TypeError, ValueError)):
        pages.fork(kv, st, i, i)
    with pytest.raises(TypeError):
        pages.copy(kv, i, i)
