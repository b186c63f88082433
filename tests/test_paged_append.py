"""paged_kv_append: what is in the pages afterwards, value by value, and the turned q."""
import ctypes

import pytest
import torch

import helpers as H
from paged_helpers import PagedBatch
from sageattention_rdna3_b200 import PagedKV, _native, check_status, paged_kv_append, rotary_axes
from test_rotary import SageRotary, phases, rotate64, tolerance


def token_positions(batch):
    return torch.cat([torch.arange(n - m, n) for m, n in zip(batch.q_lens, batch.kv_lens)] + [torch.empty(0, dtype=torch.int64)])


def append_and_check(batch, k, v, q, rope, inter, positions=None, with_cu=True, pad=0):
    """Runs the call on `pad` more rows than there are tokens and compares the whole cache, NaN for NaN."""
    dev, T = batch.dev, batch.T
    cache = batch.cache()
    table, lens = batch.args()
    out = paged_kv_append(cache, k.to(dev), v.to(dev), table, lens, cu_q=batch.cu_q() if with_cu else None, rotary=rope,
                          positions=None if positions is None else positions.to(dev), q=None if q is None else q.to(dev))
    check_status(dev)
    want_v, want_k = batch.v_pages.clone(), batch.k_pages.double()
    tol_k = torch.zeros_like(want_k)
    pos = token_positions(batch)
    if rope is not None:
        ph = phases(pos[:, None].expand(T, rope.n_axes) if positions is None else positions.reshape(positions.size(0), -1)[:T], rope.axes)[:, None]
        rows = rotate64(k[:T], ph, inter)
        tol = tolerance(k[:T], rows, ph.size(-1), inter, batch.dtype)
    else:
        rows, tol = k[:T].double(), torch.zeros(T, batch.Hkv, batch.D, dtype=torch.float64)
    t = 0
    for b, m in enumerate(batch.q_lens):
        for _ in range(m):
            j = int(pos[t])
            pid, slot = batch.page_of(b, j), j % batch.page
            at = (pid, slice(None), slot) if batch.layout == "HND" else (pid, slot)
            want_k[at], tol_k[at], want_v[at] = rows[t], tol[t], v[t]
            t += 1
    got_k, got_v = cache.k_pages.cpu(), cache.v_pages.cpu()
    assert torch.equal(got_v.view(torch.int16), want_v.view(torch.int16))
    untouched = torch.isnan(want_k)
    assert torch.equal(torch.isnan(got_k), untouched)
    assert ((got_k.double() - want_k).abs() - tol_k)[~untouched].max() <= 0
    if q is not None:
        want = rotate64(q[:T], ph, inter)
        assert ((out[:T].cpu().double() - want).abs() - tolerance(q[:T], want, ph.size(-1), inter, batch.dtype)).max() <= 0
        assert torch.equal(out[T:].cpu(), torch.zeros_like(q[T:]))
    else:
        assert out is None


CASES = [
    # q_lens, kv_lens, Hq, Hkv, D, page, layout, dtype, interleaved
    ([1], [1], 4, 1, 64, 16, "NHD", torch.bfloat16, False),
    ([1] * 5, [16, 17, 1, 333, 32], 12, 4, 128, 16, "HND", torch.float16, True),
    ([3, 0, 40, 1], [3, 20, 55, 129], 8, 2, 128, 32, "NHD", torch.bfloat16, True),
    ([130, 7], [130, 300], 2, 2, 64, 256, "HND", torch.float16, False),
    ([700, 900, 1], [700, 1900, 64], 16, 8, 128, 64, "NHD", torch.bfloat16, False),
    ([1] * 1300, [1 + i % 40 for i in range(1300)], 2, 1, 64, 16, "NHD", torch.float16, False),    # cu_q searched in memory
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("joint", [False, True])
def test_pages_hold_what_was_appended(case, joint):
    q_lens, kv_lens, Hq, Hkv, D, page, layout, dtype, inter = case
    dev = torch.device("cuda")
    batch = PagedBatch(q_lens, kv_lens, Hq, Hkv, D, page, layout, dtype, dev, seed=len(q_lens), joint=joint)
    T, pad = batch.T, 3
    # one projection gives q, k and v of a token side by side
    qkv = H.randn((T + pad, Hq + 2 * Hkv, D), 5, dtype)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    rope = rotary_axes(D, D, interleaved=inter)
    append_and_check(batch, k, v, q, rope, inter, pad=pad)
    append_and_check(batch, k, v, None, None, inter, pad=pad)
    append_and_check(batch, k, v, None, rotary_axes(D, 32, interleaved=inter), inter, pad=pad)
    if all(m == 1 for m in q_lens):
        append_and_check(batch, k[:T], v[:T], q[:T], rope, inter, with_cu=False)


@pytest.mark.gpu
@pytest.mark.parametrize("int64", [False, True])
def test_positions_of_their_own(int64):
    dev = torch.device("cuda")
    batch = PagedBatch([5, 9], [30, 9], 6, 2, 64, 16, "NHD", torch.float16, dev)
    k, v, q = (H.randn((14, h, 64), s, torch.float16) for h, s in ((2, 1), (2, 2), (6, 3)))
    pos = torch.randint(-9, 70000, (14, 3), generator=torch.Generator().manual_seed(1)).to(torch.int64 if int64 else torch.int32)
    append_and_check(batch, k, v, q, rotary_axes(64, (16, 24, 24)), False, positions=pos)
    append_and_check(batch, k, v, q, rotary_axes(64, 64), False, positions=pos[:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["page", "negative_page", "table", "negative_position"])
def test_bad_pages_and_lengths_are_reported_and_not_stored(what):
    dev = torch.device("cuda")
    batch = PagedBatch([2, 2], [20, 40], 2, 2, 64, 16, "NHD", torch.float16, dev)
    cache = batch.cache()
    table, lens = batch.args()
    code = 3
    if what == "page":
        table[1, 2] = batch.n_pages
    elif what == "negative_page":
        table[1, 2] = -1
    else:
        code = 4
        lens[1] = table.size(1) * 16 + 2 if what == "table" else 1
    k, v = H.randn((4, 2, 64), 1, torch.float16, dev), H.randn((4, 2, 64), 2, torch.float16, dev)
    paged_kv_append(cache, k, v, table, lens, cu_q=batch.cu_q())
    with pytest.raises(RuntimeError, match=f"device status {code}"):
        check_status(dev)
    check_status(dev)
    # the tokens of the first sequence are in their places all the same, and nothing else has changed but ...
    want = batch.k_pages.clone()
    for t, j in ((0, 18), (1, 19)):
        want[batch.page_of(0, j), j % 16] = k[t].cpu()
    if what == "negative_position":       # ... the new token of the second that does have a place
        want[batch.page_of(1, 0), 0] = k[3].cpu()
    assert torch.equal(cache.k_pages.cpu().view(torch.int16), want.view(torch.int16))


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    dev = torch.device("cuda")
    batch = PagedBatch([1] * 3, [5, 17, 33], 4, 2, 128, 16, "HND", torch.bfloat16, dev)
    table, lens = batch.args()
    rope = rotary_axes(128, 128)
    q, k, v = (H.randn((3, h, 128), s, torch.bfloat16, dev) for h, s in ((4, 1), (2, 2), (2, 3)))
    plain = batch.cache()
    want = paged_kv_append(plain, k, v, table, lens, rotary=rope, q=q)
    captured = batch.cache()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged_kv_append(captured, k, v, table, lens, rotary=rope, q=q)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(captured.k_pages.view(torch.int16), plain.k_pages.view(torch.int16))
    other = batch.cache()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_kv_append(other, k, v, table, lens, rotary=rope, q=q)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(other.v_pages.view(torch.int16), plain.v_pages.view(torch.int16))
    check_status(dev)


# ---------------------------------------------------------------- without a GPU

def test_refused_calls():
    cache = PagedKV.allocate(4, 16, 2, 64, dtype=torch.float16, device="cpu")
    k, v, q = (torch.zeros(3, h, 64, dtype=torch.float16) for h in (2, 2, 4))
    table, lens = torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    rope = rotary_axes(64, 64, device="cpu")
    bad = [dict(k=k[:, :1]), dict(k=k.float()), dict(v=v[:2]), dict(page_table=table.long()), dict(page_table=table[:2]),
           dict(kv_lens=lens.long()), dict(kv_lens=lens[:2]), dict(cu_q=lens), dict(k=k[:2], v=v[:2]), dict(q=q),
           dict(q=q[:2], rotary=rope), dict(positions=torch.zeros(3, dtype=torch.int32)),
           dict(rotary=rope, positions=torch.zeros(4, dtype=torch.int32)), dict(rotary=rope, positions=torch.zeros(3)),
           dict(rotary=rotary_axes(128, 128, device="cpu")), dict(rotary="rope"), dict(k=k.clone().requires_grad_())]
    for change in bad:
        args = dict(k=k, v=v, page_table=table, kv_lens=lens)
        args.update(change)
        with pytest.raises(AssertionError):
            paged_kv_append(cache, **args)
    with pytest.raises(AssertionError, match="CUDA device"):
        paged_kv_append(cache, k, v, table, lens)
    with pytest.raises(AssertionError):
        paged_kv_append("cache", k, v, table, lens)


def test_refused_caches():
    ok = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    assert PagedKV(ok, ok).page_size == 16 and PagedKV(ok, ok).num_kv_heads == 2 and PagedKV(ok, ok).num_pages == 4
    hnd = PagedKV.allocate(3, 32, 5, 128, tensor_layout="HND", device="cpu")
    assert (hnd.page_size, hnd.num_kv_heads, hnd.head_dim) == (32, 5, 128)
    for k, v in ((ok, ok[:2]), (ok, ok.bfloat16()), (ok.float(), ok.float()), (ok[0], ok[0]), (torch.zeros(4, 24, 2, 64).half(),) * 2,
                 (torch.zeros(4, 16, 2, 96).half(),) * 2, (torch.zeros(4, 16, 2, 128).half()[..., ::2],) * 2,
                 (torch.zeros(4, 16, 2, 65).half()[..., :64],) * 2, (torch.zeros(0, 16, 2, 64).half(),) * 2):
        with pytest.raises(AssertionError):
            PagedKV(k, v)
    with pytest.raises(AssertionError):
        PagedKV(ok, ok, "BSHD")
    with pytest.raises(AssertionError, match="gradient"):
        PagedKV(ok, ok.clone().requires_grad_())


class SagePagedKV(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in "kp ks kh vp vs vh".split()] + \
               [(n, ctypes.c_int) for n in ("num_pages", "page_size", "Hkv", "D", "dtype")]


class SagePagedBatch(ctypes.Structure):
    _fields_ = [("page_table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("table_width", ctypes.c_int),
                ("kv_lens", ctypes.c_void_p), ("cu_q", ctypes.c_void_p), ("B", ctypes.c_int), ("T", ctypes.c_int)]


class SageRows(ctypes.Structure):
    _fields_ = [("ptr", ctypes.c_void_p), ("stride_t", ctypes.c_int64), ("stride_h", ctypes.c_int64)]


def test_c_entry_refuses_before_cuda():
    lib = _native.load_abi()

    def call(page=16, D=64, dtype=0, pages=4, k=0x1000, ks=64, rows=0x4000, B=2, T=2, table=0x100, cu=None, with_q=False, rotary=False):
        c = SagePagedKV(k, 0x2000, 2048, ks, 1024, 2048, 64, 1024, pages, page, 2, D, dtype)
        b = SagePagedBatch(table, 8, 8, 0x200, cu, B, T)
        r = SageRows(rows, 128, 64)
        rope = SageRotary(0x300, 0x400, 32, 1, 0, None, 0, 0, 0)
        qp = ctypes.byref(r) if with_q else None
        return lib.sage_paged_append(ctypes.byref(c), ctypes.byref(b), ctypes.byref(r), ctypes.byref(r), qp, qp, 4 if with_q else 0,
                                     ctypes.byref(rope) if rotary else None, None, None)

    assert call(page=24) == 1 and b"page_size" in lib.sage_last_error()
    assert call(page=8) == 1 and call(page=512) == 1
    assert call(D=96) == 1 and call(dtype=2) == 1 and call(pages=0) == 1
    assert call(k=0x1008) == 1 and call(k=None) == 1 and call(ks=60) == 1 and call(ks=0) == 1
    assert call(rows=0x4004) == 1 and call(table=None) == 1
    assert call(T=3) == 1 and b"T must be B" in lib.sage_last_error()
    assert call(with_q=True) == 1 and b"rotary" in lib.sage_last_error()
    assert call(B=-1, T=-1) == 1
    assert call(B=0, T=0) == 0 and call(T=0, cu=0x500) == 0
