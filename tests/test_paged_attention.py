"""sageattn_paged against attention in 64 bits: lengths, groups, pages, masks, shared prefixes, and what it refuses."""
import ctypes

import pytest
import torch

import helpers as H
from paged_helpers import PagedBatch
from sageattention_rdna3_b200 import (PagedKV, _native, check_status, paged_kv_append, rotary_axes, sageattn,
                                      sageattn_paged)
from test_paged_append import SagePagedBatch, SagePagedKV, SageRows

F16, BF16 = torch.float16, torch.bfloat16


def compare(batch, o, lse, causal=True, sm_scale=None):
    want, want_lse, bound, bound_lse = batch.attention(causal, sm_scale, dev=batch.dev)
    got = o.cpu().double()
    assert not torch.isnan(got).any()
    worst = (got - want).abs() - bound
    assert worst.max() <= 0, f"off by {float(worst.max())} more than allowed, at {torch.nonzero(worst == worst.max())[0].tolist()}"
    if lse is not None:
        got = lse.cpu().double()
        empty = want_lse == float("-inf")
        assert torch.equal(got == float("-inf"), empty)
        if (~empty).any():
            assert ((got - want_lse).abs() - bound_lse)[~empty].max() <= 0
        assert torch.equal(o.cpu()[empty], torch.zeros_like(o.cpu()[empty]))


def run(batch, causal=True, sm_scale=None, lse=True, **kwargs):
    table, lens = batch.args()
    single = all(m == 1 for m in batch.q_lens)
    kwargs.setdefault("cu_q", None if single else batch.cu_q())
    out = sageattn_paged(batch.q.to(batch.dev), batch.cache(), table, lens, is_causal=causal, sm_scale=sm_scale, return_lse=lse,
                         shared_pages=batch.shared_pages(), **kwargs)
    check_status(batch.dev)
    return out


SINGLE = [
    # kv_lens, Hq, Hkv, D, page, layout, dtype: one token per sequence
    ([1], 1, 1, 64, 16, "NHD", F16),
    ([1, 2, 3], 4, 4, 128, 16, "HND", BF16),
    ([15, 16, 17, 31, 32, 33], 8, 2, 64, 16, "NHD", BF16),
    ([127, 128, 129, 255, 256, 257], 12, 4, 128, 32, "HND", F16),
    ([0, 5, 0, 700, 1], 6, 2, 128, 64, "NHD", F16),                # sequences without keys
    ([4213], 48, 12, 128, 16, "NHD", BF16),
    ([9000, 3], 16, 1, 64, 256, "HND", BF16),                      # 16 rows, long next to short
    ([333, 1000], 24, 1, 128, 128, "NHD", F16),                    # 24 rows: two of 16
    ([640], 32, 1, 64, 16, "HND", F16),
    ([500, 77], 40, 1, 128, 16, "NHD", BF16),                      # more than 32 rows
    ([300], 128, 1, 64, 32, "NHD", F16),
    ([20000], 8, 8, 64, 16, "HND", F16),
    ([1 + 37 * i % 900 for i in range(200)], 4, 2, 64, 16, "NHD", BF16),      # more sequences than threads
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", SINGLE, ids=[str(i) for i in range(len(SINGLE))])
def test_single_tokens(case):
    kv_lens, Hq, Hkv, D, page, layout, dtype = case
    batch = PagedBatch([1] * len(kv_lens), kv_lens, Hq, Hkv, D, page, layout, dtype, torch.device("cuda"), seed=len(kv_lens) + Hq)
    o, lse = run(batch)
    compare(batch, o, lse)
    o2, lse2 = run(batch, cu_q=batch.cu_q(), max_q=1)              # the same batch said in another way
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    o2, lse2 = run(batch, cu_q=batch.cu_q())                       # ... and so that it may take the other kernel
    compare(batch, o2, lse2)
    assert torch.equal(run(batch, lse=False), o)                   # and the same again


SEVERAL = [
    # q_lens, kv_lens, Hq, Hkv, D, page, layout, dtype
    ([3, 5, 1], [3, 100, 1], 4, 1, 128, 16, "NHD", BF16),
    ([4, 0, 2, 7], [129, 50, 2, 640], 8, 2, 64, 32, "HND", F16),
    ([5] * 9, [5 + 71 * i for i in range(9)], 32, 8, 128, 32, "HND", BF16),
    ([16, 17], [16, 400], 3, 3, 64, 16, "NHD", F16),
    ([33, 1, 130], [33, 2000, 700], 8, 2, 128, 64, "NHD", BF16),
    ([200], [200], 4, 4, 64, 128, "HND", F16),
    ([129, 64], [1000, 64], 12, 4, 128, 16, "NHD", F16),
    ([700, 1, 40], [2100, 999, 41], 16, 2, 64, 256, "HND", BF16),
    ([9, 2], [4, 1], 4, 2, 128, 16, "NHD", F16),                   # more tokens than keys: the first rows see nothing
    ([257], [1300], 10, 10, 128, 64, "HND", BF16),
    ([20, 3], [60, 500], 40, 1, 128, 16, "NHD", BF16),             # groups that do not divide a row tile
    ([11], [300], 96, 1, 64, 32, "HND", F16),
    ([6, 5], [800, 5], 128, 1, 128, 64, "NHD", F16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", SEVERAL, ids=[str(i) for i in range(len(SEVERAL))])
def test_several_tokens(case, causal):
    q_lens, kv_lens, Hq, Hkv, D, page, layout, dtype = case
    batch = PagedBatch(q_lens, kv_lens, Hq, Hkv, D, page, layout, dtype, torch.device("cuda"), seed=sum(q_lens))
    o, lse = run(batch, causal)
    compare(batch, o, lse, causal)
    # the bound of the new tokens chooses the kernel, not the result; one that is too small is no error
    for max_q in (max(q_lens), 1):
        o2, lse2 = run(batch, causal, max_q=max_q)
        compare(batch, o2, lse2, causal)


SHARED = [
    # shared, own lengths behind it, q_lens, Hq, Hkv, D, page, layout, dtype
    (16, [1, 5, 17], [1, 1, 1], 4, 2, 64, 16, "NHD", F16),
    (512, [1] * 8, [1] * 8, 16, 16, 64, 16, "HND", BF16),
    (2048, [1, 300, 64, 129, 7], [1, 1, 1, 1, 1], 32, 8, 128, 64, "NHD", BF16),
    (384, [5, 3, 200], [4, 3, 2], 12, 4, 128, 128, "HND", F16),
    (4096, [1 + i for i in range(40)], [1] * 40, 8, 1, 128, 32, "NHD", F16),
    (256, [30, 1], [30, 1], 8, 2, 64, 256, "HND", BF16),
    (1024, [3 + i for i in range(130)], [1] * 130, 8, 2, 64, 16, "NHD", F16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", SHARED, ids=[str(i) for i in range(len(SHARED))])
def test_shared_prefix(case):
    shared, own, q_lens, Hq, Hkv, D, page, layout, dtype = case
    batch = PagedBatch(q_lens, [shared + n for n in own], Hq, Hkv, D, page, layout, dtype, torch.device("cuda"), seed=len(own), shared=shared)
    for causal in (True, False):
        o, lse = run(batch, causal)
        compare(batch, o, lse, causal)
    # the same keys through the table give the same, within the same bound
    table, lens = batch.args()
    table[:, :shared // page] = batch.shared_ids.to(batch.dev)
    o, lse = sageattn_paged(batch.q.to(batch.dev), batch.cache(), table, lens, cu_q=batch.cu_q(), return_lse=True)
    check_status(batch.dev)
    compare(batch, o, lse)


@pytest.mark.gpu
def test_shared_prefix_with_sequences_that_end_inside_it():
    """kv_lens below the shared length: such a sequence sees the part of the prefix that it has, or nothing at all."""
    dev = torch.device("cuda")
    batch = PagedBatch([1, 2, 1, 3, 0], [300, 100, 0, 2, 0], 8, 2, 128, 32, "NHD", BF16, dev, shared=256)
    for causal in (True, False):
        o, lse = run(batch, causal)
        compare(batch, o, lse, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kind", ["sharp", "flat", "sink", "large"])
def test_distributions(dtype, kind):
    dev = torch.device("cuda")
    for q_lens, kv_lens in (([1, 1], [3000, 500]), ([90], [1500])):
        batch = PagedBatch(q_lens, kv_lens, 8, 2, 128, 16, "NHD", dtype, dev, seed=3, q_scale=8.0 if kind == "sharp" else 1.0)
        if kind == "flat":
            batch.q.zero_()
        if kind == "sink":          # one key far above the rest, whose weights are then about 2^-18
            for b in range(len(kv_lens)):
                batch.k[b][0] = 1.25
                batch._put(b, 0, kv_lens[b], batch.k[b], batch.v[b])
            batch.q.copy_((batch.q.float() * 0.2 + 0.9).to(dtype))
        if kind == "large":
            for b in range(len(kv_lens)):
                batch.v[b].mul_(3000.0)
                batch._put(b, 0, kv_lens[b], batch.k[b], batch.v[b])
        o, lse = run(batch)
        compare(batch, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("sm_scale", [0.0, 0.5, -0.25])
def test_scales(sm_scale):
    batch = PagedBatch([1, 6, 70], [200, 300, 70], 4, 2, 64, 16, "HND", F16, torch.device("cuda"))
    o, lse = run(batch, sm_scale=sm_scale)
    compare(batch, o, lse, sm_scale=sm_scale)


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [3, 70, 2]])
def test_a_row_that_is_not_a_number_stays_one(q_lens):
    """NaN or infinity among a sequence's own keys reach its rows, in one piece or cut into parts, and no other's."""
    dev = torch.device("cuda")
    for value in (float("nan"), float("inf")):
        batch = PagedBatch(q_lens, [900, 800, 20000], 4, 2, 64, 16, "NHD", F16, dev)
        batch.k[2][5, 0] = value
        batch._put(2, 0, 20000, batch.k[2], batch.v[2])
        o, lse = run(batch)
        sick, first = slice(batch.cu[2], batch.cu[3]), slice(0, batch.cu[2])
        if value != value:
            assert torch.isnan(o[sick][:, :2]).all() and torch.isnan(lse[sick][:, :2]).all()
        assert not torch.isnan(o[sick][:, 2:]).any()
        assert not torch.isnan(o[first]).any() and not torch.isnan(lse[first]).any()


@pytest.mark.gpu
def test_rows_of_no_sequence():
    dev = torch.device("cuda")
    for q_lens in ([1, 2], [50, 2]):
        batch = PagedBatch(q_lens, [80, 30], 4, 2, 64, 16, "NHD", F16, dev)
        table, lens = batch.args()
        T = batch.T
        q = torch.cat([torch.randn(3, 4, 64).half(), batch.q, torch.randn(5, 4, 64).half()]).to(dev)
        cu = batch.cu_q() + 3
        o, lse = sageattn_paged(q, batch.cache(), table, lens, cu_q=cu, return_lse=True)
        check_status(dev)
        compare(batch, o[3:3 + T], lse[3:3 + T])
        rest = torch.cat([o[:3], o[3 + T:]])
        assert torch.equal(rest, torch.zeros_like(rest))
        assert (torch.cat([lse[:3], lse[3 + T:]]) == float("-inf")).all()
        wide = torch.full((T + 8, 4, 2, 64), 7.0, dtype=F16, device=dev)        # rows of a larger tensor
        given = wide[:, :, 1]
        o2, lse2 = sageattn_paged(q, batch.cache(), table, lens, cu_q=cu, out=given, return_lse=True)
        assert o2.data_ptr() == given.data_ptr() and torch.equal(o2[3:3 + T], o[3:3 + T])
        assert (given[:3] == 7.0).all() and (given[3 + T:] == 7.0).all() and (wide[:, :, 0] == 7.0).all()
        assert torch.equal(lse2, lse)


@pytest.mark.gpu
def test_rows_of_no_sequence_behind_a_shared_prefix():
    dev = torch.device("cuda")
    batch = PagedBatch([1, 2], [80, 100], 4, 2, 64, 16, "NHD", F16, dev, shared=64)
    table, lens = batch.args()
    q = torch.cat([batch.q, torch.randn(5, 4, 64).half()]).to(dev)
    o, lse = sageattn_paged(q, batch.cache(), table, lens, cu_q=batch.cu_q(), return_lse=True, shared_pages=batch.shared_pages())
    compare(batch, o[:3], lse[:3])
    assert torch.equal(o[3:], torch.zeros_like(o[3:])) and (lse[3:] == float("-inf")).all()
    given = torch.full_like(q, 7.0)
    sageattn_paged(q, batch.cache(), table, lens, cu_q=batch.cu_q(), shared_pages=batch.shared_pages(), out=given)
    assert torch.equal(given[:3], o[:3]) and (given[3:] == 7.0).all()
    check_status(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [1, 40])
def test_strides_streams_graphs_and_joint_pages(q_len):
    dev = torch.device("cuda")
    batch = PagedBatch([q_len] * 3, [40, 600, 2000], 8, 2, 128, 32, "NHD", BF16, dev, joint=True)
    table, lens = batch.args()
    cu = batch.cu_q()
    cache, q = batch.cache(), batch.q.to(dev)
    want = sageattn_paged(q, cache, table, lens, cu_q=cu)
    compare(batch, want, None)
    joint = torch.randn(batch.T, 12, 128, device=dev).to(BF16)
    joint[:, :8] = q
    assert torch.equal(sageattn_paged(joint[:, :8], cache, table, lens, cu_q=cu), want)
    odd = torch.empty(batch.T, 8, 129, dtype=BF16, device=dev)[..., 1:]
    odd.copy_(q)
    assert torch.equal(sageattn_paged(odd, cache, table, lens, cu_q=cu), want)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(sageattn_paged(by_head, cache, table, lens, cu_q=cu), want)
    wide = torch.full((3, table.size(1) + 5), 0x7ffffff0, dtype=torch.int32, device=dev)
    wide[:, :table.size(1)] = table
    assert torch.equal(sageattn_paged(q, cache, wide[:, :table.size(1)], lens, cu_q=cu), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = sageattn_paged(q, cache, table, lens, cu_q=cu)
    torch.cuda.synchronize()
    assert torch.equal(other, want)
    # two graphs captured one after the other, replayed at the same time on two streams
    static = torch.zeros_like(q)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(sageattn_paged(static, cache, table, lens, cu_q=cu))
        graphs.append(graph)
    static.copy_(q)
    torch.cuda.synchronize()
    for _ in range(5):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    # lengths change between replays, the launches do not
    lens.copy_(torch.tensor([q_len, 128, 1999], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], sageattn_paged(q, cache, table, lens, cu_q=cu))
    check_status(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [1, 40])
def test_bad_pages_and_lengths_are_reported(q_len):
    dev = torch.device("cuda")
    batch = PagedBatch([q_len] * 2, [200, 100], 4, 2, 64, 16, "NHD", F16, dev)
    cache, q = batch.cache(), batch.q.to(dev)
    good, lens = batch.args()
    want = sageattn_paged(q, cache, good, lens, cu_q=batch.cu_q())
    check_status(dev)
    for bad in (batch.n_pages, -1, 0x7fffffff, -0x80000000):
        table = good.clone()
        table[1, 3] = bad
        o = sageattn_paged(q, cache, table, lens, cu_q=batch.cu_q())
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="device status 3.*call after"):
            sageattn_paged(q, cache, good, lens, cu_q=batch.cu_q())
        assert torch.equal(o[:q_len], want[:q_len])
    long = lens.clone()
    long[0] = good.size(1) * 16 + 1
    good[0, :] = good[0, 0]
    sageattn_paged(q, cache, good, long, cu_q=batch.cu_q())
    with pytest.raises(RuntimeError, match="device status 4"):
        check_status(dev)
    check_status(dev)


@pytest.mark.gpu
def test_wild_cu_q_stays_inside_the_rows():
    """cu_q that leaves [0, T] or falls is clipped: nothing is read or written outside the rows."""
    dev = torch.device("cuda")
    batch = PagedBatch([2, 2], [40, 60], 4, 2, 64, 16, "NHD", F16, dev)
    table, lens = batch.args()
    for cu in ([0, 2, 900], [-5, 2, 4], [0, 4, 2], [3, 1, 4], [7, 8, 9]):
        room = torch.full((12, 4, 64), 7.0, dtype=F16, device=dev)
        sageattn_paged(batch.q.to(dev), batch.cache(), table, lens, cu_q=torch.tensor(cu, dtype=torch.int32, device=dev), out=room[4:8])
        torch.cuda.synchronize()
        assert (room[:4] == 7.0).all() and (room[8:] == 7.0).all()
    check_status(dev)


@pytest.mark.gpu
def test_empty_batches():
    dev = torch.device("cuda")
    cache = PagedKV.allocate(2, 16, 2, 64, dtype=F16)
    none = torch.empty(0, 4, 64, dtype=F16, device=dev)
    i32 = dict(dtype=torch.int32, device=dev)
    assert sageattn_paged(none, cache, torch.zeros(0, 3, **i32), torch.zeros(0, **i32)).shape == (0, 4, 64)
    assert sageattn_paged(none, cache, torch.zeros(2, 3, **i32), torch.ones(2, **i32), cu_q=torch.zeros(3, **i32)).shape == (0, 4, 64)
    q = torch.ones(3, 4, 64, dtype=F16, device=dev)
    o, lse = sageattn_paged(q, cache, torch.zeros(0, 3, **i32), torch.zeros(0, **i32), cu_q=torch.zeros(1, **i32), return_lse=True)
    assert (o == 0).all() and (lse == float("-inf")).all()
    o = sageattn_paged(q, cache, torch.zeros(3, 0, **i32), torch.zeros(3, **i32))          # a table without columns
    assert (o == 0).all()
    check_status(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_a_prompt_and_its_answer(layout):
    """As used together: a prompt enters in two chunks, then tokens one by one; every output against attention over the
    turned keys in one piece, by sageattn's own causal kernel for the prompt and in 64 bits for the tokens."""
    dev = torch.device("cuda")
    Hq, Hkv, D, n_prompt, n_new, page = 8, 2, 128, 200, 5, 16
    rope = rotary_axes(D, D)
    lens = [n_prompt, 77]
    total = [n + n_new for n in lens]
    g = torch.Generator().manual_seed(0)
    q, k, v = ([torch.randn(n, h, D, generator=g).to(BF16).to(dev) for n in total] for h in (Hq, Hkv, Hkv))
    cache = PagedKV.allocate(40, page, Hkv, D, tensor_layout=layout)
    table = torch.randperm(40, generator=g)[:28].to(torch.int32).view(2, 14).to(dev)
    done = [0, 0]
    outs = [[], []]
    chunks = [[120, 77], [80, 0]] + [[1, 1]] * n_new
    turned = [[], []]
    for step in chunks:
        at = [slice(d, d + c) for d, c in zip(done, step)]
        done = [d + c for d, c in zip(done, step)]
        kv_lens = torch.tensor(done, dtype=torch.int32, device=dev)
        cu = torch.tensor([0, step[0], sum(step)], dtype=torch.int32, device=dev)
        rows = [torch.cat([x[0][at[0]], x[1][at[1]]]) for x in (q, k, v)]
        qr = paged_kv_append(cache, rows[1], rows[2], table, kv_lens, cu_q=cu, rotary=rope, q=rows[0])
        o = sageattn_paged(qr, cache, table, kv_lens, cu_q=cu, max_q=max(step))
        for b, part in enumerate(o.split(step)):
            outs[b].append(part)
            turned[b].append(qr.split(step)[b])
    check_status(dev)
    # the cache's keys in one piece
    for b in range(2):
        ids = table[b].long()
        pages = [(x[ids].transpose(1, 2) if layout == "HND" else x[ids]).reshape(-1, Hkv, D)[:total[b]] for x in (cache.k_pages, cache.v_pages)]
        assert torch.equal(pages[1], v[b])
        qr = torch.cat(turned[b])
        batch = PagedBatch([total[b]], [total[b]], Hq, Hkv, D, page, layout, BF16, dev)
        batch.q, batch.k, batch.v = qr.cpu(), [pages[0].cpu()], [pages[1].cpu()]
        compare(batch, torch.cat(outs[b]), None)
        one = sageattn(qr[None], pages[0][None], pages[1][None], tensor_layout="NHD", is_causal=True, kernel="direct")[0]
        _, _, bound, _ = batch.attention(dev=dev)
        assert ((one.float() - torch.cat(outs[b]).float()).abs().cpu() <= 2 * bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [1, 60])
def test_many_sequences(q_len):
    """More sequences than a block has threads, some of them without new tokens or without keys."""
    dev = torch.device("cuda")
    n = 700
    q_lens = [q_len if i == 300 else (i % 3 if q_len > 1 else 1) for i in range(n)]
    kv_lens = [m + (7 * i) % 61 if i % 11 else m for i, m in enumerate(q_lens)]
    batch = PagedBatch(q_lens, kv_lens, 4, 1, 64, 16, "NHD", F16, dev)
    o, lse = run(batch)
    compare(batch, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [1, 5, 150])
def test_result_over_q_and_a_cache_of_one_page(q_len):
    """out may be q itself: a row of it is read by the CTAs that write it, and only before they do."""
    dev = torch.device("cuda")
    batch = PagedBatch([q_len] * 4, [q_len + 900 * i for i in range(4)], 8, 2, 128, 16, "HND", BF16, dev)
    table, lens = batch.args()
    cu = batch.cu_q()
    want = sageattn_paged(batch.q.to(dev), batch.cache(), table, lens, cu_q=cu)
    q = batch.q.to(dev)
    assert sageattn_paged(q, batch.cache(), table, lens, cu_q=cu, out=q) is q
    assert torch.equal(q, want)
    for Hkv in (1, 2):
        one = PagedBatch([min(q_len, 200)], [200], 4, Hkv, 64, 256, "NHD", F16, dev, spare=0)
        assert one.n_pages == 1
        o, lse = run(one)
        compare(one, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("short_way", [True, False])
def test_lengths_that_are_a_column(short_way):
    dev = torch.device("cuda")
    cache = PagedKV(*(torch.randn(4, 16, 2, 64, device=dev).to(F16) for _ in range(2)))
    q = torch.randn(1, 4, 64, device=dev).to(F16)
    table = torch.arange(4, dtype=torch.int32, device=dev)[None]
    lens = torch.tensor([[50, 7]], dtype=torch.int32, device=dev)
    out = None if short_way else torch.empty_like(q)
    got = sageattn_paged(q, cache, table, lens[:, 0], out=out)          # one element, a stride of two
    assert torch.equal(got, sageattn_paged(q, cache, table, lens[:, 0].contiguous()))


@pytest.mark.gpu
def test_results_that_overlap_are_refused():
    dev = torch.device("cuda")
    cache = PagedKV.allocate(4, 16, 2, 64, dtype=F16)
    table, lens = torch.zeros(3, 2, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)
    rows = torch.zeros(4, 4, 64, dtype=F16, device=dev)
    for q, out in ((rows[:3], rows[1:]), (rows[:3], cache.k_pages.view(-1, 4, 64)[:3]), (rows[:3], cache.v_pages.view(-1, 4, 64)[5:8])):
        with pytest.raises(RuntimeError, match="memory"):
            sageattn_paged(q, cache, table, lens, out=out)
    with pytest.raises(AssertionError, match="every row"):
        sageattn_paged(rows[:3], cache, table, lens, out=rows[:1].expand(3, 4, 64))
    check_status(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_offsets_beyond_32_bits(layout):
    """A cache of more than 2^31 values, the sequences in its last pages."""
    dev = torch.device("cuda")
    page, Hkv, D = 256, 8, 128
    n_pages = 2 ** 31 // (page * Hkv * D) + 40
    shape = (n_pages, Hkv, page, D) if layout == "HND" else (n_pages, page, Hkv, D)
    k_pages, v_pages = (torch.empty(shape, dtype=BF16, device=dev) for _ in range(2))
    cache = PagedKV(k_pages, v_pages, layout)
    batch = PagedBatch([1, 70], [600, 1000], 16, Hkv, D, page, layout, BF16, dev)
    table, lens = batch.args()
    moved = table.clone()
    used = batch.n_pages
    for b, c in enumerate(batch.counts):
        moved[b, :c] += n_pages - used
    k_pages[n_pages - used:], v_pages[n_pages - used:] = batch.k_pages.to(dev), batch.v_pages.to(dev)
    o, lse = sageattn_paged(batch.q.to(dev), cache, moved, lens, cu_q=batch.cu_q(), return_lse=True)
    check_status(dev)
    compare(batch, o, lse)
    # and what is appended goes there too
    k, v = (H.randn((71, Hkv, D), s, BF16, dev) for s in (1, 2))
    paged_kv_append(cache, k, v, moved, lens, cu_q=batch.cu_q())
    check_status(dev)
    t = 0
    for b, m in enumerate(batch.q_lens):
        for j in range(batch.kv_lens[b] - m, batch.kv_lens[b]):
            pid, slot = int(moved[b, j // page]), j % page
            at = (pid, slice(None), slot) if layout == "HND" else (pid, slot)
            if t % 10 == 0:
                assert torch.equal(k_pages[at], k[t]) and torch.equal(v_pages[at], v[t])
            t += 1


@pytest.mark.gpu
@pytest.mark.parametrize("q_len", [1, 7, 60])
def test_a_wait_that_runs_out_is_reported(q_len):
    """A load that never comes (the test hook leaves it out): the kernel ends after its bound with a status, the next call says
    so, and the one after that works."""
    lib = _native.load_abi()
    dev = torch.device("cuda")
    batch = PagedBatch([q_len] * 3, [q_len + 500] * 3, 4, 2, 128, 16, "NHD", F16, dev)
    table, lens = batch.args()
    args = (batch.q.to(dev), batch.cache(), table, lens)
    want = sageattn_paged(*args, cu_q=batch.cu_q(), max_q=q_len)
    check_status(dev)
    lib.sage_test_set_wait_limit_us(20000)
    lib.sage_test_drop_v_load(1)
    try:
        sageattn_paged(*args, cu_q=batch.cu_q(), max_q=q_len)
        torch.cuda.synchronize()
    finally:
        lib.sage_test_drop_v_load(0)
        lib.sage_test_set_wait_limit_us(0)
    with pytest.raises(RuntimeError, match="device status.*call after"):
        sageattn_paged(*args, cu_q=batch.cu_q(), max_q=q_len)
    assert torch.equal(sageattn_paged(*args, cu_q=batch.cu_q(), max_q=q_len), want)
    check_status(dev)


@pytest.mark.gpu
def test_checked_at_once_if_asked(monkeypatch):
    monkeypatch.setenv("SAGEATTN_B200_CHECK_STATUS", "1")
    dev = torch.device("cuda")
    batch = PagedBatch([1, 1], [20, 30], 4, 2, 64, 16, "NHD", F16, dev)
    cache, (table, lens) = batch.cache(), batch.args()
    o, lse = run(batch)
    compare(batch, o, lse)
    table[0, 0] = -1
    with pytest.raises(RuntimeError, match="device status 3"):
        sageattn_paged(batch.q.to(dev), cache, table, lens)
    k = H.randn((2, 2, 64), 1, F16, dev)
    table[0, 1] = -1
    with pytest.raises(RuntimeError, match="device status 3"):
        paged_kv_append(cache, k, k, table, lens)
    check_status(dev)


@pytest.mark.gpu
def test_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs a second GPU")
    dev = torch.device("cuda", 1)
    batch = PagedBatch([1, 40], [300, 100], 4, 2, 64, 16, "NHD", F16, dev)
    o, lse = run(batch)
    compare(batch, o, lse)


# ---------------------------------------------------------------- without a GPU

def test_refused_calls():
    cache = PagedKV.allocate(4, 16, 2, 64, dtype=F16, device="cpu")
    q = torch.zeros(3, 4, 64, dtype=F16)
    table, lens = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    bad = [dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[:2]), dict(q=q[..., :32]), dict(q=q[:, :0]), dict(page_table=table.long()),
           dict(page_table=table[:2]), dict(kv_lens=lens.long()), dict(cu_q=lens), dict(max_q=-1), dict(q=q.expand(3, 4, 64).clone().requires_grad_()),
           dict(shared_pages=lens.long()), dict(shared_pages=table), dict(shared_pages=torch.zeros(3, dtype=torch.int32)),
           dict(out=q.float()), dict(out=q[:2]), dict(out=torch.zeros(3, 4, 65, dtype=F16)[..., :64]),
           dict(q=torch.zeros(3, 2 * 129, 64, dtype=F16))]
    for change in bad:
        args = dict(q=q, cache=cache, page_table=table, kv_lens=lens)
        args.update(change)
        with pytest.raises(AssertionError):
            sageattn_paged(**args)
    with pytest.raises(AssertionError, match="CUDA device"):
        sageattn_paged(q, cache, table, lens)


def test_c_entry_refuses_before_cuda():
    lib = _native.load_abi()
    lib.sage_paged_workspace_bytes.restype = ctypes.c_int64

    def call(Hq=4, max_q=0, n_shared=0, D=64, page=16, q=0x4000, o=0x5000, width=8, T=2, cu=None, ws=0x8000, ws_bytes=1 << 40, shared=0x900):
        c = SagePagedKV(0x1000, 0x2000, 2048, 64, 1024, 2048, 64, 1024, 4, page, 2, D, 0)
        b = SagePagedBatch(0x100, width, width, 0x200, cu, 2, T)
        r, w = SageRows(q, 256, 64), SageRows(o, 256, 64)
        return lib.sage_paged_attn(ctypes.byref(c), ctypes.byref(b), ctypes.byref(r), ctypes.byref(w), Hq, max_q, 1, ctypes.c_float(0.1), None,
                                   ctypes.c_void_p(shared), n_shared, 0, None, ctypes.c_void_p(ws), ctypes.c_int64(ws_bytes), None)

    assert call(Hq=3) == 1 and b"multiple" in lib.sage_last_error()
    assert call(Hq=2 * 129) == 1 and call(Hq=0) == 1
    assert call(D=80) == 1 and call(page=48) == 1 and call(max_q=-1) == 1 and call(n_shared=-1) == 1
    assert call(n_shared=9) == 1 and b"columns" in lib.sage_last_error()
    assert call(q=0x4008) == 1 and call(o=0x5002) == 1 and call(q=None) == 1
    assert call(T=3) == 1
    assert call(width=1 << 27) == 1 and b"2^30" in lib.sage_last_error()
    assert call(T=0, cu=0x700) == 0                           # nothing to do, nothing touched
