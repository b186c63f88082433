"""Rotary positions (apply_rotary): against the rotation in 64 bits, its gradient, and what it refuses."""
import ctypes
import math

import pytest
import torch

import helpers as H
from sageattention_rdna3_b200 import _native, apply_rotary, rotary_axes, sageattn



def phases(positions, axes, base=10000.0, inv_freq=None):
    """Angles in 64 bits, [.., pairs]; positions [.., n_axes]."""
    cols = []
    i0 = 0
    for a, w in enumerate(axes):
        for i in range(w // 2):
            f = base ** (-2.0 * i / w) if inv_freq is None else inv_freq[i0]
            # whole turns are taken off in integers where a double would lose them: positions here stay below 2^31
            cols.append(torch.remainder(positions[..., a].double() * f, 2 * math.pi))
            i0 += 1
    return torch.stack(cols, dim=-1)


def rotate64(x, phase, interleaved, inverse=False):
    """x [.., D] in 64 bits; phase broadcasts against [.., pairs]."""
    x = x.double()
    n = phase.size(-1)
    c, s = torch.cos(phase), torch.sin(phase) * (-1 if inverse else 1)
    out = x.clone()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])
    ya, yb = a * c - b * s, a * s + b * c
    if interleaved:
        out[..., 0:2 * n:2], out[..., 1:2 * n:2] = ya, yb
    else:
        out[..., :n], out[..., n:2 * n] = ya, yb
    return out


def partner_sum(x, n, interleaved):
    """|x| + |y| of the pair that every value belongs to (0 behind the pairs)."""
    x = x.double().abs()
    out = torch.zeros_like(x)
    if interleaved:
        t = x[..., 0:2 * n:2] + x[..., 1:2 * n:2]
        out[..., 0:2 * n:2] = out[..., 1:2 * n:2] = t
    else:
        t = x[..., :n] + x[..., n:2 * n]
        out[..., :n] = out[..., n:2 * n] = t
    return out


def tolerance(x, exact, n, interleaved, dtype):
    """cos and sin: the angle, at most pi, rounded to fp32 (pi 2^-25) and 2 ulp of the function (2^-23): below 2.2e-7.
    The two products and their sum in fp32: 2^-23 of |x| + |y|.  Together below 4e-7 of |x| + |y|.  Then one rounding to the
    output type, half a step of it (fp16: or of its smallest numbers, 2^-25)."""
    err = 4e-7 * partner_sum(x, n, interleaved)
    return err + (exact.abs() + err) * torch.finfo(dtype).eps / 2 + (2.0 ** -25 if dtype == torch.float16 else 1e-38)


def make(shape, seed, dtype, device):
    return H.randn(shape, seed, dtype, device)


CASES = [
    # B, S, Hq, Hkv, D, layout, axes, interleaved, dtype
    (1, 1, 1, 1, 64, "HND", (64,), False, torch.float16),
    (2, 7, 3, 1, 64, "NHD", (16, 24, 24), True, torch.bfloat16),
    (1, 117, 12, 4, 128, "NHD", (128,), False, torch.bfloat16),
    (3, 33, 5, 5, 128, "HND", (32, 48, 48), True, torch.float16),
    (1, 1000, 9, 3, 128, "HND", (44, 42, 42), False, torch.float32),
    (2, 129, 4, 2, 64, "NHD", (32,), True, torch.float32),           # half of the head is left alone
    (1, 65, 2, 2, 128, "HND", (16, 16, 16, 16), False, torch.bfloat16),
    (2, 4213, 16, 4, 128, "NHD", (64, 64), False, torch.float16),     # slices of eight heads
    (1, 16, 17, 1, 64, "HND", (62, 2), True, torch.float16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("per_batch", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_matches_the_rotation_in_64_bits(case, per_batch):
    B, S, Hq, Hkv, D, layout, axes, inter, dtype = case
    dev = torch.device("cuda")
    g = torch.Generator().manual_seed(S)
    shape = (B, S, len(axes)) if per_batch else (S, len(axes))
    pos = torch.randint(-50, 100000, shape, generator=g)
    shp = (lambda h: (B, h, S, D)) if layout == "HND" else (lambda h: (B, S, h, D))
    q, k = make(shp(Hq), 1, dtype, dev), make(shp(Hkv), 2, dtype, dev)
    rope = rotary_axes(D, axes, interleaved=inter)
    for dt in (torch.int32, torch.int64):
        rq, rk = apply_rotary(q, k, pos.to(dt).to(dev), rope, tensor_layout=layout)
        ph = phases(pos, axes)
        if not per_batch:
            ph = ph.unsqueeze(0)
        ph = ph.unsqueeze(1 if layout == "HND" else 2)
        for x, y in ((q, rq), (k, rk)):
            want = rotate64(x.cpu(), ph, inter)
            bad = (y.cpu().double() - want).abs() - tolerance(x.cpu(), want, ph.size(-1), inter, dtype)
            assert bad.max() <= 0, float(bad.max())
            assert y.dtype == dtype and y.shape == x.shape
    only_q = apply_rotary(q, None, pos.to(dev), rope, tensor_layout=layout)
    assert torch.equal(only_q, rq)


@pytest.mark.gpu
def test_far_positions_lose_nothing():
    """Frequency 1 at positions up to 2^31: an fp32 angle would be off by whole turns."""
    dev = torch.device("cuda")
    pos = torch.tensor([2 ** 31 - 1, 2 ** 30 + 7, 10 ** 9 + 1, 123456789, -2 ** 31, 2 ** 20 + 3], dtype=torch.int32)
    x = make((1, 1, 6, 64), 5, torch.float32, dev)
    rope = rotary_axes(64, 64)
    y = apply_rotary(x, None, pos.to(dev), rope).cpu().double()
    # the frequency has 2^-53 of itself as a double, times 2^31 positions: 2^-22 radians more than the usual tolerance
    ph = torch.tensor([[math.remainder(p * 10000.0 ** (-2.0 * i / 64), 2 * math.pi) for i in range(32)] for p in pos.tolist()],
                      dtype=torch.float64)
    want = rotate64(x.cpu(), ph[None, None], False)
    tol = tolerance(x.cpu(), want, 32, False, torch.float32) + 4 * 2.0 ** -22 * partner_sum(x.cpu(), 32, False)
    assert ((y - want).abs() - tol).max() <= 0


@pytest.mark.gpu
def test_own_frequencies_and_bases():
    dev = torch.device("cuda")
    x = make((2, 3, 20, 128), 7, torch.float32, dev)
    pos = torch.arange(20, device=dev)
    freqs = [0.5 + 0.01 * i for i in range(32)]
    rope = rotary_axes(128, (64,), inv_freq=freqs)
    ph = phases(pos.cpu()[:, None], (64,), inv_freq=freqs)[None, None]
    want = rotate64(x.cpu(), ph, False)
    assert ((apply_rotary(x, None, pos, rope).cpu().double() - want).abs() - tolerance(x.cpu(), want, 32, False, torch.float32)).max() <= 0
    two = rotary_axes(128, (64, 64), base=(100.0, 10000.0))
    pos2 = torch.stack([pos, 3 * pos], dim=1)
    ph = torch.cat([phases(pos2.cpu()[:, :1], (64,), base=100.0), phases(pos2.cpu()[:, 1:], (64,))], dim=-1)[None, None]
    want = rotate64(x.cpu(), ph, False)
    assert ((apply_rotary(x, None, pos2, two).cpu().double() - want).abs() - tolerance(x.cpu(), want, 64, False, torch.float32)).max() <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients(dtype, inter):
    """Against the formula (the rotation the other way), with upstream gradients in strides of their own, and differences."""
    dev = torch.device("cuda")
    B, S, Hq, Hkv, D, axes = 2, 37, 6, 2, 64, (16, 24, 24)
    q, k = make((B, S, Hq, D), 1, dtype, dev).requires_grad_(), make((B, S, Hkv, D), 2, dtype, dev).requires_grad_()
    pos = torch.randint(0, 500, (S, 3), generator=torch.Generator().manual_seed(3))
    rope = rotary_axes(D, axes, interleaved=inter)
    rq, rk = apply_rotary(q, k, pos.to(dev), rope, tensor_layout="NHD")
    gq = make((B, Hq, S, D), 4, dtype, dev).transpose(1, 2)
    gk = make((B, S, Hkv, D), 5, dtype, dev)
    dq, dk = torch.autograd.grad((rq, rk), (q, k), (gq, gk), retain_graph=True)
    ph = phases(pos, axes)[None, :, None]
    for g, d in ((gq, dq), (gk, dk)):
        want = rotate64(g.cpu(), ph, inter, inverse=True)
        assert ((d.cpu().double() - want).abs() - tolerance(g.cpu(), want, 32, inter, dtype)).max() <= 0
    # one of the two results unused; a gradient that is one number expanded
    (dk2,) = torch.autograd.grad(rk.sum(), (k,), retain_graph=True)
    want = rotate64(torch.ones(B, S, Hkv, D), ph, inter, inverse=True)
    assert ((dk2.cpu().double() - want).abs() - tolerance(torch.ones(B, S, Hkv, D), want, 32, inter, dtype)).max() <= 0
    (dq2,) = torch.autograd.grad(rq, (q,), (gq,))
    assert torch.equal(dq2, dq)
    if dtype == torch.float32:
        # differences: the rotation is linear, f(q + h d) - f(q) = h * (R d); <g, R d> = <R^T g, d>
        d = make((B, S, Hq, D), 6, dtype, dev)
        rd = apply_rotary(d, None, pos.to(dev), rope, tensor_layout="NHD")
        lhs, rhs = (gq.double() * rd.double()).sum().item(), (dq.double() * d.double()).sum().item()
        # each side: sums of N(0,1) products with errors below 2e-6 of |x| + |y| each
        assert abs(lhs - rhs) <= 2e-6 * 4 * d.numel()


@pytest.mark.gpu
def test_gradient_of_a_broadcast_input():
    """k of one batch entry expanded over the batch: its gradient is the sum."""
    dev = torch.device("cuda")
    k = make((1, 2, 9, 64), 1, torch.float32, dev).requires_grad_()
    pos = torch.arange(9, device=dev)
    rope = rotary_axes(64, 64)
    q = make((3, 4, 9, 64), 2, torch.float32, dev)
    _, rk = apply_rotary(q, k.expand(3, 2, 9, 64), pos, rope)
    g = make((3, 2, 9, 64), 3, torch.float32, dev)
    (dk,) = torch.autograd.grad(rk, (k,), (g,))
    ph = phases(pos.cpu()[:, None], (64,))[None, None]
    want = rotate64(g.cpu(), ph, False, inverse=True).sum(0, keepdim=True)
    tol = tolerance(g.cpu(), rotate64(g.cpu(), ph, False, True), 32, False, torch.float32).sum(0, keepdim=True)
    # and three fp32 additions
    assert ((dk.cpu().double() - want).abs() - tol - 3 * 2.0 ** -24 * g.cpu().double().abs().sum(0, keepdim=True)).max() <= 0


@pytest.mark.gpu
def test_strides_streams_and_graphs():
    dev = torch.device("cuda")
    rope = rotary_axes(128, (32, 48, 48), interleaved=True)
    pos = torch.randint(0, 99, (50, 3), device=dev)
    qkv = make((2, 50, 3, 4, 128), 1, torch.bfloat16, dev)
    want = apply_rotary(qkv[:, :, 0].contiguous(), qkv[:, :, 1].contiguous(), pos, rope, tensor_layout="NHD")
    got = apply_rotary(qkv[:, :, 0], qkv[:, :, 1], pos, rope, tensor_layout="NHD")       # slices of a joint projection
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.empty(2, 50, 4, 129, dtype=torch.bfloat16, device=dev)[..., 1:]           # no 16-byte loads: copied first
    odd.copy_(qkv[:, :, 0])
    assert torch.equal(apply_rotary(odd, None, pos, rope, tensor_layout="NHD"), want[0])
    swapped = pos.t().contiguous().t()                                                    # axes not neighbours in memory
    assert torch.equal(apply_rotary(qkv[:, :, 0], None, swapped, rope, tensor_layout="NHD"), want[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = apply_rotary(qkv[:, :, 0], qkv[:, :, 1], pos, rope, tensor_layout="NHD")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other[0], want[0])
    x = make((2, 50, 4, 128), 9, torch.bfloat16, dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = apply_rotary(x, None, pos, rope, tensor_layout="NHD")
    x.copy_(qkv[:, :, 0])
    graph.replay()
    assert torch.equal(y, want[0])


@pytest.mark.gpu
def test_captured_backward():
    dev = torch.device("cuda")
    rope = rotary_axes(64, 64)
    pos = torch.arange(30, device=dev)
    q = make((1, 2, 30, 64), 1, torch.float32, dev)
    g = make((1, 2, 30, 64), 2, torch.float32, dev)
    leaf = q.clone().requires_grad_()
    (want,) = torch.autograd.grad(apply_rotary(leaf, None, pos, rope), (leaf,), (g,))
    del leaf
    static = q.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(apply_rotary(static, None, pos, rope), (static,), (g,))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_empty_and_in_front_of_attention():
    dev = torch.device("cuda")
    rope = rotary_axes(64, (16, 24, 24))
    empty = apply_rotary(torch.empty(2, 4, 0, 64, device=dev), None, torch.empty(0, 3, dtype=torch.int32, device=dev), rope)
    assert empty.shape == (2, 4, 0, 64)
    # attention sees differences of positions: a common offset changes nothing
    q, k, v = (make((1, 4, 200, 64), s, torch.float16, dev) for s in (1, 2, 3))
    pos = torch.randint(0, 30, (200, 3), device=dev)
    outs = []
    for off in (0, 977):
        rq, rk = apply_rotary(q, k, pos + off, rope)
        outs.append(sageattn(rq, rk, v).float())
    # q and k are each rounded to fp16 twice differently: scores of up to ~6 differ by at most 2^-10 of their terms
    assert (outs[0] - outs[1]).abs().max() <= 0.02


# ---------------------------------------------------------------- without a GPU

def test_table():
    rope = rotary_axes(64, (16, 24, 24), device="cpu")
    assert rope.n_axes == 3 and rope.rotary_dim == 64 and rope.freq.dtype == torch.int64
    assert rope.axis.tolist() == [0] * 8 + [1] * 12 + [2] * 12
    for i, f in zip((0, 1, 8, 20), (1.0, 10000.0 ** (-2 / 16), 1.0, 1.0)):
        turns = (int(rope.freq[i]) % 2 ** 64) / 2.0 ** 64
        assert abs(turns - f / (2 * math.pi)) < 2.0 ** -52
    negative = rotary_axes(64, (16,), inv_freq=[-1.0] * 8, device="cpu")
    assert abs((int(negative.freq[0]) % 2 ** 64) / 2.0 ** 64 - (1 - 1 / (2 * math.pi))) < 2.0 ** -52


@pytest.mark.parametrize("kwargs", [
    dict(head_dim=96, axes=(96,)), dict(head_dim=64, axes=()), dict(head_dim=64, axes=(8,) * 8), dict(head_dim=64, axes=(15, 17)),
    dict(head_dim=64, axes=(24,)), dict(head_dim=64, axes=(128,)), dict(head_dim=64, axes=(64, 0)),
    dict(head_dim=64, axes=(32, 32), base=(1.0,)), dict(head_dim=64, axes=(64,), base=-1.0),
    dict(head_dim=64, axes=(64,), inv_freq=[1.0]), dict(head_dim=64, axes=(16,), inv_freq=[float("nan")] * 8)])
def test_refused_tables(kwargs):
    with pytest.raises(AssertionError):
        rotary_axes(device="cpu", **kwargs)


def test_refused_calls():
    rope = rotary_axes(64, (32, 32), device="cpu")
    q = torch.zeros(2, 4, 8, 64)
    pos = torch.zeros(8, 2, dtype=torch.int32)
    for args in ((q, None, pos, "rope"), (q.double(), None, pos, rope), (q[0], None, pos, rope), (torch.zeros(2, 4, 8, 128), None, pos, rope),
                 (q, q[:1], pos, rope), (q, q.half(), pos, rope), (q, q[:, :, :4], pos, rope), (q, None, pos.float(), rope),
                 (q, None, pos[:4], rope), (q, None, pos[:, 0], rope), (q, None, pos.expand(3, 8, 2), rope)):
        with pytest.raises(AssertionError):
            apply_rotary(*args)
    with pytest.raises(AssertionError):
        apply_rotary(q, None, pos, rope, tensor_layout="BSHD")
    with pytest.raises(AssertionError, match="CUDA device"):
        apply_rotary(q, None, pos, rope)


class SageRotary(ctypes.Structure):
    _fields_ = [("freq", ctypes.c_void_p), ("axis", ctypes.c_void_p), ("pairs", ctypes.c_int), ("n_axes", ctypes.c_int),
                ("interleaved", ctypes.c_int), ("positions", ctypes.c_void_p), ("positions_64", ctypes.c_int),
                ("stride_b", ctypes.c_int64), ("stride_s", ctypes.c_int64)]


def test_c_entry_refuses_before_cuda():
    lib = _native.load_abi()
    lib.sage_apply_rotary.restype = ctypes.c_int

    def call(q=(0x1000, 4096, 1024, 64), out=(0x2000, 4096, 1024, 64), dtype=0, D=64, pairs=32, axes=1, freq=0x100, pos=0x200, B=1, Hq=4):
        qs, os_ = H.SageStrided(*q), H.SageStrided(*out)
        r = SageRotary(freq, 0x300, pairs, axes, 0, pos, 0, 0, 1)
        return lib.sage_apply_rotary(ctypes.byref(qs), ctypes.byref(os_), None, None, ctypes.byref(r), dtype, B, Hq, 0, 16, D, 0, None)

    assert call(D=96) == 1 and b"head_dim" in lib.sage_last_error()
    assert call(dtype=3) == 1
    assert call(pairs=40) == 1 and b"pairs" in lib.sage_last_error()
    assert call(pairs=12) == 1
    assert call(axes=5) == 1 and call(axes=0) == 1
    assert call(freq=None) == 1 and call(pos=None) == 1
    assert call(q=(0x1008, 4096, 1024, 64)) == 1 and call(out=(0x2000, 4096, 1024, 60)) == 1
    assert call(B=-1) == 1
    assert call(B=0) == 0                                     # nothing to do, nothing touched
