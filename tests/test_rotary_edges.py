"""Edges of apply_rotary: inputs of which only some need a gradient, heads that are not there, positions of any size."""
from fractions import Fraction

import pytest
import torch

import helpers as H
from sageattention_rdna3_b200 import PagedKV, apply_rotary, check_status, paged_kv_append, rotary_axes
from test_rotary import partner_sum, rotate64, tolerance

DIGITS = 400                                          # binary digits behind the point
PI_DIGITS = 1200                                      # ... of pi: 2^997 radians are still to be known to 2^-64 turns


def _pi():
    """pi by Machin's formula, 16 arctan(1/5) - 4 arctan(1/239), within 2^-PI_DIGITS."""
    one = 1 << (PI_DIGITS + 20)

    def arctan_inverse(n):
        total, power, k = 0, one // n, 0
        while power:
            total += (power if k % 2 == 0 else -power) // (2 * k + 1)
            power //= n * n
            k += 1
        return total
    return Fraction(16 * arctan_inverse(5) - 4 * arctan_inverse(239), one)


PI = _pi()


def _root(x, n):
    """x ** (1/n) of a fraction, within 2^-DIGITS, by bisection on integers."""
    scaled = (x.numerator << (n * DIGITS)) // x.denominator
    lo, hi = 0, 1 << (DIGITS + max(1, x.numerator.bit_length()))
    while hi - lo > 1:
        mid = (lo + hi) // 2
        if mid ** n <= scaled:
            lo = mid
        else:
            hi = mid
    return Fraction(lo, 1 << DIGITS)


def frequencies(base, width):
    """base ** (-2 i / width), i < width / 2, as fractions."""
    step = _root(Fraction(base), width // 2)          # base ** (2 / width)
    return [1 / step ** i for i in range(width // 2)]


def units_off(stored, radians):
    """How far a stored frequency is from the true one, in units of 2^-64 turns."""
    d = (Fraction(int(stored) % 2 ** 64) - radians / (2 * PI) * 2 ** 64) % 2 ** 64
    return float(min(d, 2 ** 64 - d))


def test_frequencies_keep_64_bits():
    """A stored frequency is the nearest of its 2^64 values to the formula's: half a unit."""
    rope = rotary_axes(128, (32, 48, 48), base=(10000.0, 500000.0, 100.0), device="cpu")
    want = frequencies(10000, 32) + frequencies(500000, 48) + frequencies(100, 48)
    assert max(units_off(f, w) for f, w in zip(rope.freq, want)) <= 0.500001
    rope = rotary_axes(128, 128, device="cpu")
    assert max(units_off(f, w) for f, w in zip(rope.freq, frequencies(10000, 128))) <= 0.500001
    own = [0.1, -0.1, 1e-7, -1e-7, 3.0, 1234.5, -2.0 ** -70, 0.0, 1e18, 2.0 ** -64, 1.0, -1.0, 0.7, 1e-19, 6.283185307179586, 1e300]
    rope = rotary_axes(64, 32, inv_freq=own, device="cpu")
    assert max(units_off(f, Fraction(w)) for f, w in zip(rope.freq, own)) <= 0.500001


@pytest.mark.gpu
@pytest.mark.parametrize("top", [2 ** 31, 2 ** 40])
def test_positions_far_from_zero(top):
    """The kernel's angle is within 2^-32 turns of position times stored frequency, and that is half a unit of 2^-64 turns
    off: 2 pi (2^-32 + position 2^-65) radians beyond what fp32 does to every angle."""
    dev = torch.device("cuda", 0)
    pos = [top - 1, top // 2 + 7, top - 12345, -top + 1, top // 3]
    freqs = frequencies(10000, 64)
    turns = [[(p * f / (2 * PI)) % 1 for f in freqs] for p in pos]
    phase = torch.tensor([[float(t * 2 * PI if t < Fraction(1, 2) else (t - 1) * 2 * PI) for t in row] for row in turns], dtype=torch.float64)
    x = H.randn((1, 2, len(pos), 64), 5, torch.float32, dev)
    y = apply_rotary(x, None, torch.tensor(pos, dtype=torch.int64, device=dev), rotary_axes(64, 64)).cpu().double()
    want = rotate64(x.cpu(), phase[None, None], False)
    tol = tolerance(x.cpu(), want, 32, False, torch.float32) + 6.2832 * (2.0 ** -32 + top * 2.0 ** -65) * partner_sum(x.cpu(), 32, False)
    assert ((y - want).abs() - tol).max() <= 0


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
