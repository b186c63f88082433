"""Edges of the operators around a growing cache: what one call leaves for another, rows that see nothing, slots that are not in
use, results that overlap, and calls that come with more of autograd than the cache has."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import helpers as H
from paged_helpers import PagedBatch
from sageattention_rdna3_b200 import (PagedKV, _native, apply_rotary, check_status, core, paged_kv_append, rotary_axes, sageattn,
                                      sageattn_paged)
from test_paged_attention import compare

F16, BF16 = torch.float16, torch.bfloat16


def clear_status(dev):
    torch.cuda.synchronize()
    core._status_word(dev).zero_()
    core._status_mirror(dev)[1][0] = 0
    torch.cuda.synchronize()


# ---------------------------------------------------------------- what one call leaves for another

# head_dim, heads, length, kernel: plain, persistent and paired launches of both kernels
SAGEATTN_CALLS = [(64, 2, 200, "int8"), (128, 2, 200, "direct"), (128, 20, 4000, "int8"), (64, 10, 4096, "int8"), (128, 148, 1280, "direct")]


@pytest.mark.gpu
@pytest.mark.parametrize("code", [3, 4])
@pytest.mark.parametrize("case", SAGEATTN_CALLS, ids=[str(i) for i in range(len(SAGEATTN_CALLS))])
def test_a_page_code_stops_no_other_call(case, code):
    """A bad page of one call (the host has not seen it yet) leaves what runs behind it alone."""
    D, heads, n, kernel = case
    dev = torch.device("cuda", 0)
    q, k, v = (H.randn((1, heads, n, D), s, F16, dev) for s in (1, 2, 3))
    want = torch.empty_like(q)
    sageattn(q, k, v, kernel=kernel, out=want)
    check_status(dev)
    got = torch.full_like(q, 7.0)
    core._status_word(dev).fill_(code)
    try:
        sageattn(q, k, v, kernel=kernel, out=got)
        torch.cuda.synchronize()
        assert int(core._status_word(dev)) == code and int(core._status_mirror(dev)[1][0]) == 0
    finally:
        clear_status(dev)
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_sageattn_behind_a_bad_page():
    """As a program meets it: the append and the call behind it are both in the stream before the first has run."""
    dev = torch.device("cuda", 0)
    cache = PagedKV.allocate(4, 16, 2, 64, dtype=F16)
    table, lens = torch.full((3, 1), 99, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)
    rows = torch.ones(3, 2, 64, dtype=F16, device=dev)
    q = H.randn((1, 2, 300, 64), 1, F16, dev)
    want = torch.empty_like(q)
    sageattn(q, q, q, out=want, kernel="int8")
    check_status(dev)
    got = torch.full_like(q, 7.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_kv_append(cache, rows, rows, table, lens)
        sageattn(q, q, q, out=got, kernel="int8")
    got.fill_(7.0)
    graph.replay()
    with pytest.raises(RuntimeError, match="device status 3"):
        check_status(dev)
    assert torch.equal(got, want)
    check_status(dev)


@pytest.fixture
def dropped_load():
    """A wait that runs out, by the library's test hook."""
    lib = _native.load_abi()
    lib.sage_test_set_wait_limit_us(20000)
    lib.sage_test_drop_v_load(1)
    yield
    lib.sage_test_drop_v_load(0)
    lib.sage_test_set_wait_limit_us(0)


@pytest.mark.gpu
@pytest.mark.parametrize("what", [1, 60, "sageattn"])
def test_a_wait_that_runs_out_is_not_hidden_by_a_page_code(what, dropped_load):
    """The word keeps the more serious code, the mirror what the word holds, and the launch behind does nothing."""
    dev = torch.device("cuda", 0)
    word, mirror = core._status_word(dev), core._status_mirror(dev)[1]
    if what == "sageattn":
        q = H.randn((1, 2, 300, 128), 1, F16, dev)
        call = lambda: sageattn(q, q, q, kernel="int8")                     # noqa: E731
    else:
        batch = PagedBatch([what] * 2, [what + 500] * 2, 4, 2, 128, 16, "NHD", F16, dev)
        table, lens = batch.args()
        args = (batch.q.to(dev), batch.cache(), table, lens)
        call = lambda: sageattn_paged(*args, cu_q=batch.cu_q(), max_q=what)  # noqa: E731
    torch.cuda.synchronize()
    word.fill_(3)
    try:
        call()
        torch.cuda.synchronize()
        first = int(word)
        assert first % 16 == 2 and int(mirror[0]) == first
        mirror[0] = 0                                                        # (or the next call would raise before its launch)
        call()
        torch.cuda.synchronize()
        assert int(word) == first
    finally:
        clear_status(dev)


@pytest.mark.gpu
def test_a_page_code_does_not_replace_a_wait():
    """... nor is a wait's code taken for the page's, whichever is reported first."""
    dev = torch.device("cuda", 0)
    batch = PagedBatch([1, 1], [20, 40], 2, 2, 64, 16, "NHD", F16, dev)
    table, lens = batch.args()
    table[1, 2] = -1
    k = H.randn((2, 2, 64), 1, F16, dev)
    cache = batch.cache()
    core._prepare_status(dev)
    word, mirror = core._status_word(dev), core._status_mirror(dev)[1]
    try:
        word.fill_(2 + 16 * 20)
        paged_kv_append(cache, k, k, table, lens)
        torch.cuda.synchronize()
        assert int(word) == 2 + 16 * 20 and int(mirror[0]) == 2 + 16 * 20
    finally:
        clear_status(dev)


# ---------------------------------------------------------------- rows that belong to no token

def fill_shared_memory(value, D, dtype, dev):
    """A call that leaves `value` in the places of Q of every SM."""
    heads = 320
    cache = PagedKV.allocate(16, 16, heads, D, dtype=dtype)
    q = torch.full((256, heads, D), value, dtype=dtype, device=dev)
    i32 = dict(dtype=torch.int32, device=dev)
    sageattn_paged(q, cache, torch.arange(16, **i32)[None], torch.full((1,), 256, **i32), cu_q=torch.tensor([0, 256], **i32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group, D", [(3, 128), (5, 64), (12, 128), (1, 64)])
def test_rows_without_a_token_change_nothing(group, D, dtype):
    """Groups that do not divide a row tile, and a tile that reaches behind the last sequence: what stands in those rows (of an earlier
    kernel, of the padding, of the next sequence) does not change a bit of the others."""
    dev = torch.device("cuda", 0)
    batch = PagedBatch([61, 75], [900, 333], 2 * group, 2, D, 16, "NHD", dtype, dev, seed=group)
    table, lens = batch.args()
    cache, cu = batch.cache(), batch.cu_q()
    results = []
    for filler in (0.0, float("nan"), 300.0, float("inf")):
        for pad in (0.0, float("nan")):
            q = torch.cat([batch.q, torch.full((200, 2 * group, D), pad, dtype=dtype)]).to(dev)
            fill_shared_memory(filler, D, dtype, dev)
            results.append(sageattn_paged(q, cache, table, lens, cu_q=cu, return_lse=True))
    check_status(dev)
    for o, lse in results:
        compare(batch, o[:batch.T], lse[:batch.T])
        assert torch.equal(o, results[0][0]) and torch.equal(lse, results[0][1])
    # a neighbour that is not a number
    sick = batch.q.clone()
    sick[61:] = float("nan")
    o, lse = sageattn_paged(sick.to(dev), cache, table, lens, cu_q=cu, return_lse=True)
    assert torch.equal(o[:61], results[0][0][:61]) and torch.equal(lse[:61], results[0][1][:61])


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("q_lens, kv_lens", [([6, 1], [2, 50]), ([100, 1], [30, 50]), ([700], [500])])
def test_a_row_without_keys_is_zero_whatever_v_holds(q_lens, kv_lens, value):
    dev = torch.device("cuda", 0)
    batch = PagedBatch(q_lens, kv_lens, 8, 2, 64, 16, "HND", F16, dev)
    batch.v[0][:] = value
    batch._put(0, 0, kv_lens[0], batch.k[0], batch.v[0])
    table, lens = batch.args()
    for max_q in (None, 1):
        o, lse = sageattn_paged(batch.q.to(dev), batch.cache(), table, lens, cu_q=batch.cu_q(), max_q=max_q, return_lse=True)
        check_status(dev)
        blind = q_lens[0] - kv_lens[0]
        assert (lse[:blind] == float("-inf")).all() and torch.isfinite(lse[blind:]).all()
        assert torch.equal(o[:blind], torch.zeros_like(o[:blind]))
        assert not torch.isfinite(o[blind:q_lens[0]]).any() and torch.isfinite(o[q_lens[0]:]).all()


# ---------------------------------------------------------------- lengths that change too early

@pytest.mark.gpu
@pytest.mark.parametrize("q_len, shared", [(1, 0), (60, 0), (1, 64)])
def test_lengths_that_change_during_a_call(q_len, shared):
    """A program's mistake, which gives numbers without a meaning: the calls end all the same, write their own rows only, and those
    behind them are right."""
    dev = torch.device("cuda", 0)
    n = 40
    batch = PagedBatch([q_len] * n, [shared + q_len + (173 * i) % 900 for i in range(n)], 4, 2, 64, 16, "NHD", F16, dev, shared=shared)
    table, lens = batch.args()
    table[:, :shared // 16] = 0
    table.clamp_(0, batch.n_pages - 1)                        # (any length up to the width of the table finds pages)
    cache, cu, room = batch.cache(), batch.cu_q(), torch.full((batch.T + 8, 4, 64), 7.0, dtype=F16, device=dev)
    args = dict(cu_q=cu, max_q=q_len, shared_pages=batch.shared_pages())
    q = batch.q.to(dev)
    want = sageattn_paged(q, cache, table, lens, **args)
    good, good_cu = lens.clone(), cu.clone()
    g = torch.Generator(device=dev).manual_seed(1)
    other = torch.randint(0, table.size(1) * 16, (64, n), generator=g, device=dev, dtype=torch.int32)
    rows = torch.randint(0, batch.T + 1, (64, n + 1), generator=g, device=dev, dtype=torch.int32).sort(dim=1).values.to(torch.int32)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(200):
        with torch.cuda.stream(side):
            lens.copy_(other[i % 64])
            cu.copy_(rows[(i * 7) % 64])
        sageattn_paged(q, cache, table, lens, out=room[4:-4], **args)
    torch.cuda.synchronize()
    assert (room[:4] == 7.0).all() and (room[-4:] == 7.0).all()
    check_status(dev)
    lens.copy_(good)
    cu.copy_(good_cu)
    assert torch.equal(sageattn_paged(q, cache, table, lens, **args), want)


# ---------------------------------------------------------------- slots that are not in use

@pytest.mark.gpu
@pytest.mark.parametrize("aligned", [True, False])
def test_slots_that_are_not_in_use(aligned):
    """Without cu_q a sequence of length 0 is a slot that is not in use: nothing stored, nothing reported, its rows zero."""
    dev = torch.device("cuda", 0)
    batch = PagedBatch([1] * 5, [20, 1, 33, 1, 16], 4, 2, 64, 16, "NHD", F16, dev)
    table, lens = batch.args()
    lens[1] = lens[3] = 0
    rope = rotary_axes(64, 64)
    joint = torch.randn(5, 8, 64 if aligned else 68, device=dev).to(F16)[..., :64]       # (else copied, by the way through Python)
    q, k, v = joint[:, :4], joint[:, 4:6], joint[:, 6:]
    cache, plain = batch.cache(), batch.cache()
    used = [0, 2, 4]
    want = paged_kv_append(plain, k[used], v[used], table[used], lens[used], rotary=rope, q=q[used])
    for positions in (None, torch.arange(5, device=dev)):
        got = paged_kv_append(cache, k, v, table, lens, rotary=rope, q=q, positions=positions)
        check_status(dev)
        assert torch.equal(got[[1, 3]], torch.zeros_like(got[[1, 3]]))
        if positions is None:
            assert torch.equal(got[used], want)
            for x, y in ((cache.k_pages, plain.k_pages), (cache.v_pages, plain.v_pages)):
                assert torch.equal(x.view(torch.int16), y.view(torch.int16))
            o, lse = sageattn_paged(got, cache, table, lens, return_lse=True)
            assert torch.equal(o[[1, 3]], torch.zeros_like(o[[1, 3]])) and (lse[[1, 3]] == float("-inf")).all()
            assert torch.equal(o[used], sageattn_paged(want, plain, table[used], lens[used]))
    check_status(dev)
    # a negative length is no slot
    lens[1] = -1
    paged_kv_append(cache, k, v, table, lens)
    with pytest.raises(RuntimeError, match="device status 4"):
        check_status(dev)


# ---------------------------------------------------------------- results that overlap

@pytest.mark.gpu
def test_overlaps_of_strided_results_are_refused():
    """q and out as slices of one joint projection: heads that another block still reads must not be written."""
    dev = torch.device("cuda", 0)
    batch = PagedBatch([1, 1, 1], [20, 300, 5], 4, 2, 64, 16, "NHD", F16, dev)
    table, lens = batch.args()
    cache = batch.cache()
    want = sageattn_paged(batch.q.to(dev), cache, table, lens)
    joint = torch.zeros(4, 12, 64, dtype=F16, device=dev)
    by_head = torch.zeros(12, 4, 64, dtype=F16, device=dev).transpose(0, 1)
    pairs = torch.zeros(3, 4, 2, 64, dtype=F16, device=dev)
    for q, out in ((joint[:3, :4], joint[:3, 1:5]), (joint[:3, :4], joint[1:, :4]), (joint[:3, :4], joint[1:, 3:7]),
                   (by_head[:3, :4], by_head[:3, 2:6]), (by_head[:3, :4], by_head[1:, :4]),
                   (joint[:3, :4], joint.view(-1, 64)[:12].view(3, 4, 64))):
        with pytest.raises(RuntimeError, match="overlap|memory"):
            sageattn_paged(q, cache, table, lens, out=out)
    both = torch.zeros(6, 2, 16, 2, 64, dtype=F16, device=dev)
    pool = PagedKV(both[:, 0], both[:, 1])
    with pytest.raises(RuntimeError, match="overlap|memory"):
        sageattn_paged(batch.q[:, :2].to(dev), pool, table, lens, out=both[0, 0, 4:7])
    # neighbours that only lie between each other are none
    for q, out in ((joint[:3, :4], joint[:3, 4:8]), (joint[:3, 8:], joint[1:, :4]), (by_head[:3, :4], by_head[:3, 4:8]),
                   (by_head[:3, :4], by_head[1:, 8:]), (pairs[:, :, 0], pairs[:, :, 1]), (joint[:3, :4], joint[:3, :4])):
        q.copy_(batch.q)
        assert torch.equal(sageattn_paged(q, cache, table, lens, out=out), want)
    check_status(dev)


# ---------------------------------------------------------------- versions, tangents, modes, subclasses

@pytest.mark.gpu
@pytest.mark.parametrize("aligned", [True, False])
def test_what_is_written_counts_as_changed(aligned):
    """Autograd refuses a backward pass whose saved tensors were written: the pages and `out` count their versions."""
    dev = torch.device("cuda", 0)
    cache = PagedKV.allocate(4, 16, 2, 64, dtype=F16)
    table, lens = torch.arange(3, dtype=torch.int32, device=dev)[:, None], torch.ones(3, dtype=torch.int32, device=dev)
    rows = torch.ones(3, 2, 64 if aligned else 68, dtype=F16, device=dev)[..., :64]
    for _ in range(2):                                       # the second call on a device may take the short way
        versions = cache.k_pages._version, cache.v_pages._version
        paged_kv_append(cache, rows, rows, table, lens)
        assert cache.k_pages._version > versions[0] and cache.v_pages._version > versions[1]
    q = torch.ones(3, 4, 64, dtype=F16, device=dev, requires_grad=True)
    x = q * 1.0
    y = x * x                                                # keeps x
    sageattn_paged(x.detach(), cache, table, lens, out=x.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        pages = PagedKV.allocate(4, 16, 2, 64, dtype=F16)
    paged_kv_append(pages, rows, rows, table, lens)          # a cache made for inference may be used outside of it
    sageattn_paged(torch.ones(3, 4, 64, dtype=F16, device=dev), pages, table, lens)
    check_status(dev)


def refused(fn, *args, match="gradient|tangent", **kwargs):
    with pytest.raises(AssertionError, match=match):
        fn(*args, **kwargs)


def test_tangents_are_refused():
    """The cache has no derivative in either mode: a dual tensor is refused, not stripped of its tangent."""
    cache = PagedKV.allocate(4, 16, 2, 64, dtype=F16, device="cpu")
    table, lens = torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    q, k = torch.zeros(3, 4, 64, dtype=F16), torch.zeros(3, 2, 64, dtype=F16)
    with fwAD.dual_level():
        dq, dk = fwAD.make_dual(q, torch.ones_like(q)), fwAD.make_dual(k, torch.ones_like(k))
        refused(sageattn_paged, dq, cache, table, lens)
        refused(paged_kv_append, cache, dk, k, table, lens)
        refused(paged_kv_append, cache, k, dk, table, lens)
        refused(paged_kv_append, cache, k, k, table, lens, q=dq, rotary=rotary_axes(64, 64, device="cpu"))


def test_a_result_that_needs_a_gradient_is_refused():
    cache = PagedKV.allocate(4, 16, 2, 64, dtype=F16, device="cpu")
    table, lens = torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    q = torch.zeros(3, 4, 64, dtype=F16)
    out = torch.zeros(3, 4, 64, dtype=F16, requires_grad=True)
    refused(sageattn_paged, q, cache, table, lens, out=out)


class Marked(torch.Tensor):
    """A subclass that sees every function called on it."""
    seen = 0

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        Marked.seen += 1
        return super().__torch_function__(func, types, args, kwargs or {})


@pytest.mark.gpu
def test_the_short_ways_leave_what_is_not_plain():
    """Modes, subclasses, dual tensors, vmap: none of them is passed by."""
    import sageattention_rdna3_b200._C as C
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode
    dev = torch.device("cuda", 0)
    batch = PagedBatch([1, 1], [20, 40], 4, 2, 64, 16, "NHD", F16, dev)
    table, lens = batch.args()
    cache, q = batch.cache(), batch.q.to(dev)
    k = H.randn((2, 2, 64), 1, F16, dev)
    rope = rotary_axes(64, 64)
    x, pos = H.randn((1, 2, 8, 64), 2, torch.float32, dev), torch.arange(8, device=dev)
    want, turned = sageattn_paged(q, cache, table, lens), apply_rotary(x, None, pos, rope)
    table_args = (rope.freq, rope.axis, 1, False)

    def attn(q):
        return C.paged_attn_plain(q, cache.k_pages, cache.v_pages, "NHD", table, lens, None, None, True, None, False, None)

    def append(k):
        return C.paged_append_plain(cache.k_pages, cache.v_pages, "NHD", k, k, table, lens, None, None, None, None, 0, False, None)

    def rotary(x):
        return C.rotary_plain(x, None, pos, *table_args, 64, "HND")

    assert torch.equal(attn(q), want) and append(k) is True and torch.equal(rotary(x), turned)
    want = sageattn_paged(q, cache, table, lens)

    class Functions(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    class Dispatched(TorchDispatchMode):
        names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            Dispatched.names.append(func.__name__)
            return func(*args, **(kwargs or {}))

    for mode in (Functions, Dispatched):
        with mode():
            assert attn(q) is None and append(k) is None and rotary(x) is None
            assert torch.equal(sageattn_paged(q, cache, table, lens), want)
            paged_kv_append(cache, k, k, table, lens)
            assert torch.equal(apply_rotary(x, None, pos, rope), turned)
    assert {"paged_attn.default", "paged_append.default", "rotary.default"} <= set(Dispatched.names)
    marked = [t.as_subclass(Marked) for t in (q, k, x)]
    assert attn(marked[0]) is None and append(marked[1]) is None and rotary(marked[2]) is None
    # a parameter is a tensor that needs a gradient: refused by the cache, turned with a gradient behind it
    assert attn(torch.nn.Parameter(q)) is None and append(torch.nn.Parameter(k)) is None
    assert rotary(torch.nn.Parameter(x)).requires_grad and torch.equal(rotary(torch.nn.Parameter(x)), turned)
    with fwAD.dual_level():
        dual = [fwAD.make_dual(t, torch.ones_like(t)) for t in (q, k, x)]
        assert attn(dual[0]) is None and append(dual[1]) is None and rotary(dual[2]) is None
        refused(sageattn_paged, dual[0], cache, table, lens)
        refused(paged_kv_append, cache, dual[1], k, table, lens)
        with pytest.raises(RuntimeError):                                    # no forward derivative either
            apply_rotary(dual[2], None, pos, rope)
    with pytest.raises(RuntimeError):                                        # no batching rule
        torch.func.vmap(lambda t: sageattn_paged(t, cache, table, lens))(q[None].repeat(2, 1, 1, 1))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: apply_rotary(t, None, pos, rope))(x[None].repeat(2, 1, 1, 1, 1))
    check_status(dev)


# ---------------------------------------------------------------- bounds and schemas

@pytest.mark.gpu
@pytest.mark.parametrize("max_q", [2 ** 31 - 1, 2 ** 31, 2 ** 40, 2 ** 80])
def test_an_upper_bound_may_be_any_number(max_q):
    dev = torch.device("cuda", 0)
    batch = PagedBatch([3, 1], [20, 40], 4, 2, 64, 16, "NHD", F16, dev)
    table, lens = batch.args()
    args = (batch.q.to(dev), batch.cache(), table, lens)
    assert torch.equal(sageattn_paged(*args, cu_q=batch.cu_q(), max_q=max_q), sageattn_paged(*args, cu_q=batch.cu_q()))


def test_schemas_say_what_is_written():
    ops = _native.load_ops()
    for op, names in ((ops.paged_append, {"k_pages", "v_pages", "status"}), (ops.paged_attn, {"output", "lse", "status"})):
        schema = op.default._schema
        assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == names
        assert schema.is_mutable
