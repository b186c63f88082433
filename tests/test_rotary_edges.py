"""Edges of apply_rotary: inputs of which only some need a gradient, heads that are not there, positions of any size."""
import pytest
import torch

import helpers as H
from sageattention_rdna3_b200 import PagedKV, apply_rotary, check_status, paged_kv_append, rotary_axes


def allocations(fn):
    """Result of fn() and how many blocks of device memory it asked for."""
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    got = fn()
    return got, torch.cuda.memory_stats()["allocation.all.allocated"] - before


@pytest.mark.gpu
@pytest.mark.parametrize("strided", [False, True])
def test_only_what_needs_a_gradient_gets_one(strided):
    """q trained and k frozen, or the other way round: the other result needs no gradient (the cache would refuse it)."""
    dev = torch.device("cuda", 0)
    rope, pos = rotary_axes(64, 64), torch.arange(30, device=dev)

    def leaf(heads, seed, grad):
        t = H.randn((1, heads, 30, 66 if strided else 64), seed, torch.bfloat16, dev)[..., :64]   # (66: by the way through Python)
        return t.requires_grad_(grad)

    full = [leaf(h, s, True) for h, s in ((4, 1), (2, 2))]
    gq, gk = H.randn((1, 4, 30, 64), 3, torch.bfloat16, dev), H.randn((1, 2, 30, 64), 4, torch.bfloat16, dev)
    outs = apply_rotary(*full, pos, rope)
    want = torch.autograd.grad(outs, full, (gq, gk), retain_graph=True)
    for i in range(2):
        args = [leaf(h, s, i == n) for n, (h, s) in enumerate(((4, 1), (2, 2)))]
        got = apply_rotary(*args, pos, rope)
        assert [t.requires_grad for t in got] == [i == 0, i == 1]
        assert torch.equal(got[0], outs[0]) and torch.equal(got[1], outs[1])
        (grad,) = torch.autograd.grad(got[i], (args[i],), ((gq, gk)[i],))
        assert torch.equal(grad, want[i])
        # both results have a gradient behind them, one of them is asked for: one tensor is made
        (one,), made = allocations(lambda: torch.autograd.grad(outs, (full[i],), (gq, gk), retain_graph=True))
        assert torch.equal(one, want[i])
        _, both = allocations(lambda: torch.autograd.grad(outs, full, (gq, gk), retain_graph=True))
        assert both == made + 1
    # a frozen k goes on into the cache
    cache = PagedKV.allocate(4, 16, 2, 64)
    q, k = leaf(4, 1, True), leaf(2, 2, False)
    _, rk = apply_rotary(q, k, pos, rope)
    i32 = dict(dtype=torch.int32, device=dev)
    rows = rk[0].transpose(0, 1)
    paged_kv_append(cache, rows, rows, torch.arange(4, **i32)[None], torch.full((1,), 30, **i32), cu_q=torch.tensor([0, 30], **i32))
    check_status(dev)
    assert torch.equal(cache.k_pages.view(64, 2, 64)[:30], rows)


@pytest.mark.gpu
def test_second_derivatives_of_a_frozen_input():
    """The gradient's own gradient: with respect to what came in."""
    dev = torch.device("cuda", 0)
    rope, pos = rotary_axes(64, 64), torch.arange(9, device=dev)
    q = H.randn((1, 2, 9, 64), 1, torch.float32, dev).requires_grad_()
    k = H.randn((1, 2, 9, 64), 2, torch.float32, dev)
    g = H.randn((1, 2, 9, 64), 3, torch.float32, dev).requires_grad_()
    rq, _ = apply_rotary(q, k, pos, rope)
    (dq,) = torch.autograd.grad(rq, (q,), (g,), create_graph=True)
    w = H.randn((1, 2, 9, 64), 4, torch.float32, dev)
    (dg,) = torch.autograd.grad(dq, (g,), (w,))
    assert torch.equal(dg, apply_rotary(w, None, pos, rope))


@pytest.mark.gpu
def test_dispatch_modes_see_the_rotation():
    """... forward and backward, not only what it allocates."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Names(TorchDispatchMode):
        seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            Names.seen.append(func.__name__)
            return func(*args, **(kwargs or {}))

    dev = torch.device("cuda", 0)
    rope, pos = rotary_axes(64, 64), torch.arange(9, device=dev)
    x = H.randn((1, 2, 9, 64), 1, torch.float32, dev)
    want = apply_rotary(x, None, pos, rope)
    leaf = x.clone().requires_grad_()
    (dwant,) = torch.autograd.grad(apply_rotary(leaf, None, pos, rope), (leaf,), (x,))
    with Names():
        assert torch.equal(apply_rotary(x, None, pos, rope), want)
        assert Names.seen.count("rotary.default") == 1
        (got,) = torch.autograd.grad(apply_rotary(leaf, None, pos, rope), (leaf,), (x,))
        assert Names.seen.count("rotary.default") == 3
    assert torch.equal(got, dwant)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_heads_that_are_not_there(layout):
    dev = torch.device("cuda", 0)
    rope, pos = rotary_axes(64, 64), torch.arange(9, device=dev)
    q = H.randn((2, 9, 9, 64), 1, torch.float16, dev)
    none = torch.empty((2, 0, 9, 64) if layout == "HND" else (2, 9, 0, 64), dtype=torch.float16, device=dev)
    want = apply_rotary(q, None, pos, rope, tensor_layout=layout)
    rq, rk = apply_rotary(q, none, pos, rope, tensor_layout=layout)
    assert torch.equal(rq, want) and rk.shape == none.shape
    rq, rk = apply_rotary(none, q, pos, rope, tensor_layout=layout)
    assert torch.equal(rk, want) and rq.shape == none.shape
