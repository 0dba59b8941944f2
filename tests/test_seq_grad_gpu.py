"""The sequence operators have no backward pass: a call that would drop a
gradient is refused, and what a call writes in place counts as changed."""
import pytest
import torch

from ai_engine_b200 import attention, pages

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _calls():
    """Every call by its float arguments' names; each takes them as keywords."""
    def rand(*shape):
        return torch.randn(*shape, device="cuda").half()
    pos, table, cu = torch.arange(6, dtype=torch.int32, device="cuda"), torch.rand(8, 64, device="cuda"), _i32([0, 6])
    w = torch.ones(64, device="cuda")
    slots = torch.arange(6, device="cuda")
    row, one, src, dst = _i32([[0, 1]]), _i32([6]), _i32([0]), _i32([2])
    st = pages.new_state(3, 2, 2)
    return [
        (lambda q, k, v, cos_sin, q_weight, k_weight, k_pages, v_pages, q_out, k_out: attention.qk_norm_rope(
            q, k, pos, cos_sin, q_weight=q_weight, k_weight=k_weight, v=v, k_pages=k_pages, v_pages=v_pages, slots=slots,
            q_out=q_out, k_out=k_out),
         dict(q=rand(6, 2, 64), k=rand(6, 1, 64), v=rand(6, 1, 64), cos_sin=table, q_weight=w, k_weight=w.clone(),
              k_pages=rand(3, 8, 1, 64), v_pages=rand(3, 8, 1, 64), q_out=rand(6, 2, 64), k_out=rand(6, 1, 64)),
         ("k_pages", "v_pages", "q_out", "k_out")),
        (lambda q, k, v, out: attention.prompt_attention(q, k, v, cu, out=out),
         dict(q=rand(6, 2, 64), k=rand(6, 1, 64), v=rand(6, 1, 64), out=rand(6, 2, 64)), ("out",)),
        (lambda q, k_pages, v_pages, out: attention.prefix_attention(q, k_pages, v_pages, None, 0, row, one, out=out),
         dict(q=rand(1, 2, 64), k_pages=rand(3, 8, 1, 64), v_pages=rand(3, 8, 1, 64), out=rand(1, 2, 64)), ("out",)),
        (lambda kv: pages.copy(kv, src, dst), dict(kv=rand(1, 2, 3, 8, 1, 64)), ("kv",)),
        (lambda kv: pages.fork(kv, st, _i32([0]), _i32([1])), dict(kv=rand(1, 2, 3, 8, 1, 64)), ("kv",)),
        (lambda kv: pages.compact(kv, st), dict(kv=rand(1, 2, 3, 8, 1, 64)), ("kv",)),
    ]


@pytest.mark.parametrize("which", range(6))
def test_gradients_are_refused(cuda_ok, which):
    call, args, _ = _calls()[which]
    call(**args)
    for name in args:
        wants = dict(args, **{name: args[name].clone().requires_grad_()})
        with pytest.raises(ValueError, match="grad"):
            call(**wants)
        with torch.no_grad():
            call(**wants)
        call(**dict(args, **{name: wants[name].detach()}))
    with torch.inference_mode():
        call(**{name: t.clone() for name, t in args.items()})


@pytest.mark.parametrize("which", range(6))
def test_what_is_written_counts_as_changed(cuda_ok, which):
    call, args, written = _calls()[which]
    before = {name: t._version for name, t in args.items()}
    call(**args)
    for name, t in args.items():
        assert (t._version > before[name]) == (name in written), name


def test_a_saved_tensor_written_in_place_is_noticed(cuda_ok):
    """A product saved k; the call overwrites it; the product's backward says so."""
    x = torch.randn(6, 1, 64, device="cuda", dtype=torch.float32).requires_grad_()
    k = torch.randn(6, 1, 64, device="cuda")
    y = x * k
    pos, table = torch.arange(6, dtype=torch.int32, device="cuda"), torch.rand(8, 64, device="cuda")
    attention.qk_norm_rope(k.clone(), k, pos, table, k_out=k)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_state_counts_as_changed(cuda_ok):
    st = pages.new_state(4, 2, 2)
    kv = pages.new_cache(1, 4, 8, 1, 64, torch.float16)
    for call in (lambda: pages.grow(st, 8, _i32([0]), _i32([3]), 3), lambda: pages.fork(kv, st, _i32([0]), _i32([1])),
                 lambda: pages.free(st, _i32([0])), lambda: pages.compact(kv, st)):
        before = [t._version for t in st]
        call()
        assert all(t._version > n for t, n in zip(st, before))
