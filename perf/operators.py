"""The operators around a growing cache that are timed: rotary positions with several axes, the append to a
paged cache, attention that reads such a cache, and the same for a batch that shares a prefix.

Listed are calls over the range that a program makes: one odd prompt up to the tokens of a video for the rotation,
one token per sequence up to a chunk of a prompt for the cache.  Head counts and head sizes are those of the
repository's benchmark shapes (48 query heads on 12, 16 on 16) and generic ones (32 on 8, 16 on 2).  ``draw`` gives further
cases of the same families.  Lengths inside a ragged batch follow from the case itself (``mix``), values from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


# ---------------------------------------------------------------- cases ----------------------------------------

def _rotary(name, batch, tokens, heads, kv_heads, head_dim, dtype, layout, axes, interleaved, train, far=0):
    """axes: widths as "32-48-48"; far: the first position (long prompts continue far from zero)."""
    case = dict(op="rotary", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype,
                layout=layout, axes=axes, interleaved=interleaved, train=train, far=far)
    if name is not None:
        case["name"] = name
    return case


def _paged(name, op, batch, q_min, q_max, kv_min, kv_max, heads, kv_heads, head_dim, dtype, layout, page, mix,
           interleaved=False, lse=False, shared=0, causal=True):
    """q_min..q_max new tokens and kv_min..kv_max cached ones (new ones not counted, the shared prefix neither) in each of
    `batch` sequences, spread over their logarithm; shared: keys of the common prefix."""
    case = dict(op=op, batch=batch, q_min=q_min, q_max=q_max, kv_min=kv_min, kv_max=kv_max, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, dtype=dtype, layout=layout, page=page, mix=mix, interleaved=interleaved, lse=lse,
                shared=shared, causal=causal)
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # The prompt of a GQA text encoder: one short odd sequence, one axis; the latency of a call.
        _rotary("rotary_text_117", 1, 117, 48, 12, 128, "bf16", "NHD", "128", False, False, far=100000),
        # The tokens of a picture and its prompt in one sequence: three axes (frame, row, column), neighbouring pairs.
        _rotary("rotary_image_4213", 1, 4213, 48, 12, 128, "bf16", "NHD", "32-48-48", True, False),
        # Training on video tokens: forward and the gradients of q and k.
        _rotary("rotary_video_24576", 1, 24576, 16, 16, 64, "fp16", "HND", "16-24-24", False, True),
        # One decoding step of a batch: a token per sequence is rotated and put in its page.
        _paged("append_step_64", "append", 64, 1, 1, 100, 8000, 32, 8, 128, "bf16", "NHD", 16, 1),
        # Chunks of prompts of different lengths enter the cache.
        _paged("append_chunk_6", "append", 6, 300, 2500, 0, 9000, 48, 12, 128, "fp16", "HND", 64, 2, interleaved=True),
        # One user's next token after a prompt with a picture: few keys, the latency of a call; with the log-sum-exp.
        _paged("decode_one_4213", "attend", 1, 1, 1, 4212, 4212, 48, 12, 128, "bf16", "NHD", 16, 3, lse=True),
        # A serving batch in the middle of its answers: lengths all over the range.
        _paged("decode_batch_64", "attend", 64, 1, 1, 60, 16000, 32, 8, 128, "bf16", "NHD", 16, 4),
        # A few very long documents, few kv heads of 64, large pages.
        _paged("decode_long_4", "attend", 4, 1, 1, 90000, 131000, 16, 2, 64, "fp16", "HND", 128, 5),
        # Drafted tokens are checked: some new tokens per sequence at once.
        _paged("verify_32x5", "attend", 32, 3, 5, 500, 6000, 32, 8, 128, "bf16", "HND", 32, 6),
        # Chunks of long prompts attend to what the cache has of them, next to sequences that take single tokens.
        _paged("chunk_mixed_9", "attend", 9, 1, 1500, 900, 30000, 32, 8, 128, "bf16", "NHD", 64, 7),
        # A few answers to one question, many heads of 64 without groups; with the log-sum-exp.
        _paged("shared_few_8", "shared", 8, 1, 1, 0, 200, 16, 16, 64, "fp16", "NHD", 16, 8, lse=True, shared=2048),
        # Many users behind one long system prompt.
        _paged("shared_many_128", "shared", 128, 1, 1, 1, 1000, 32, 8, 128, "bf16", "HND", 32, 9, shared=16384),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads = rng.choice([(48, 12), (16, 16), (32, 8), (16, 2), (8, 1), (10, 10), (20, 4), (12, 4)])
    dtype, layout = rng.choice(["fp16", "bf16"]), rng.choice(["NHD", "HND"])
    head_dim = rng.choice([64, 128])
    op = rng.choice(["rotary", "append", "attend", "attend", "shared"])
    mix = rng.randrange(1 << 30)
    # No more than the largest listed case of the family: values rotated, cached values read, products made.
    if op == "rotary":
        dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
        most = 24576 * 32 * 64 * 2 // ((heads + kv_heads) * head_dim * _BYTES[dtype])
        tokens = _log_int(rng, 1, most)
        axes = rng.choice(["64", "16-24-24", "32-32", "20-22-22", "32"] if head_dim == 64
                          else ["128", "32-48-48", "44-42-42", "64-64", "64", "16-16-32-32"])
        return _rotary(None, rng.randint(1, max(1, min(4, most // tokens))), tokens, heads, kv_heads, head_dim, dtype, layout,
                       axes, rng.random() < 0.5, rng.random() < 0.5, far=rng.choice([0, 0, 1000, 1000000]))
    page = rng.choice([16, 32, 64, 128, 256])
    inter = rng.random() < 0.5
    lse = rng.random() < 0.3
    cached = 160000000 // (kv_heads * head_dim)               # keys in all
    if op == "append":
        batch = _log_int(rng, 1, 128)
        q_max = _log_int(rng, 1, max(1, min(2500, 4000 // batch)))
        return _paged(None, op, batch, rng.randint(1, q_max), q_max, 0, _log_int(rng, 1, 2000), heads, kv_heads, head_dim,
                      dtype, layout, page, mix, interleaved=inter)
    if op == "shared":
        batch = _log_int(rng, 2, 128)
        q_max = rng.choice([1, 1, 1, 3])
        most = min(16384, 128 * 16384 * 8 * 128 // (batch * q_max * kv_heads * head_dim), cached - 1000 * batch)
        return _paged(None, op, batch, 1, q_max, rng.choice([0, 1]), _log_int(rng, 1, 700), heads, kv_heads, head_dim, dtype,
                      layout, page, mix, lse=lse, shared=page * max(1, _log_int(rng, 256, max(300, most)) // page))
    kind = rng.choice(["one", "batch", "batch", "several", "chunk"])
    if kind == "one":
        batch = rng.randint(1, 4)
        kv = _log_int(rng, 1, min(131000, cached // batch))
        return _paged(None, op, batch, 1, 1, kv, kv, heads, kv_heads, head_dim, dtype, layout, page, mix, lse=lse)
    if kind == "batch":
        batch = _log_int(rng, 2, 128)
        return _paged(None, op, batch, 1, 1, rng.randint(0, 60), _log_int(rng, 61, min(60000, cached // batch)), heads, kv_heads,
                      head_dim, dtype, layout, page, mix, lse=lse)
    if kind == "several":
        batch = _log_int(rng, 1, 64)
        return _paged(None, op, batch, 1, rng.randint(2, 12), rng.randint(0, 60), _log_int(rng, 61, min(6000, cached // batch)),
                      heads, kv_heads, head_dim, dtype, layout, page, mix, lse=lse, causal=rng.random() < 0.8)
    batch = rng.randint(1, 9)
    q_max = _log_int(rng, 20, 1500)
    most = min(12000, cached // batch, 8000000 * 32 * 128 // (batch * q_max * heads * head_dim))
    return _paged(None, op, batch, rng.randint(1, q_max), q_max, rng.randint(0, 300), max(301, _log_int(rng, 301, max(302, most))),
                  heads, kv_heads, head_dim, dtype, layout, page, mix, lse=lse, causal=rng.random() < 0.8)


def _lengths(case):
    """(new tokens, keys in all without the shared prefix) of every sequence: fixed by the case."""
    rng = random.Random(case["mix"])
    q = [_log_int(rng, case["q_min"], case["q_max"]) for _ in range(case["batch"])]
    kv = [_log_int(rng, case["kv_min"] + 1, case["kv_max"] + 1) - 1 for _ in range(case["batch"])]
    if case["op"] == "attend" and case["q_max"] > 1000:      # chunks of prompts next to single tokens
        q[0], q[-1] = case["q_max"], case["q_min"]
    return q, [a + b for a, b in zip(q, kv)]


def work(case):
    size = _BYTES[case["dtype"]]
    d, hq, hkv = case["head_dim"], case["heads"], case["kv_heads"]
    if case["op"] == "rotary":
        rows = case["batch"] * case["tokens"] * (hq + hkv)
        axes = case["axes"].count("-") + 1
        passes = 2 if case["train"] else 1
        pairs = sum(int(a) for a in case["axes"].split("-")) // 2
        return {"bytes": passes * (2 * rows * d * size + 4 * axes * case["tokens"]), "flops": passes * 6 * rows * pairs}
    q_lens, kv_lens = _lengths(case)
    tokens = sum(q_lens)
    if case["op"] == "append":
        return {"bytes": 2 * tokens * (hq + 2 * hkv) * d * size, "flops": 6 * tokens * (hq + hkv) * d // 2}
    keys = sum(kv_lens) + case["shared"]
    visible = 0
    for nq, nk in zip(q_lens, kv_lens):
        visible += nq * (nk + case["shared"]) - (nq * (nq - 1) // 2 if case["causal"] else 0)
    nbytes = 2 * keys * hkv * d * size + 2 * tokens * hq * d * size + (4 * tokens * hq if case["lse"] else 0)
    return {"bytes": nbytes, "flops": 4 * hq * d * visible}


# ---------------------------------------------------------------- inputs ---------------------------------------

def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, dtype=torch.float32, device="cuda") * scale).to(dtype)


def _widths(case):
    if case["op"] == "rotary":
        return tuple(int(a) for a in case["axes"].split("-"))
    return (case["head_dim"],)


def _prepare_rotary(case, gen):
    dt = _DTYPES[case["dtype"]]
    b, s, d, widths = case["batch"], case["tokens"], case["head_dim"], _widths(case)

    def heads(n):
        return (b, n, s, d) if case["layout"] == "HND" else (b, s, n, d)

    state = dict(case=case, widths=widths)
    state["q"], state["k"] = _randn(gen, heads(case["heads"]), dt), _randn(gen, heads(case["kv_heads"]), dt)
    if len(widths) == 1:
        pos = torch.arange(s, device="cuda") + case["far"] + torch.randint(0, 50, (1,), generator=gen, device="cuda")
    else:                                     # a picture or film: slow axes first, the last one counts columns
        side = max(1, int(round(math.sqrt(s / 2))))
        i = torch.arange(s, device="cuda") + torch.randint(0, 50, (1,), generator=gen, device="cuda")
        parts = [i // (side * side), i // side % side, i % side] + [i % 7]
        pos = torch.stack(parts[3 - len(widths):3] if len(widths) <= 3 else parts, dim=1) + case["far"]
    state["positions"] = pos.to(torch.int32)
    if case["train"]:
        state["grad_q"], state["grad_k"] = _randn(gen, heads(case["heads"]), dt), _randn(gen, heads(case["kv_heads"]), dt)
        if own:
            state["q"].requires_grad_()
            state["k"].requires_grad_()
    return state


def _prepare_paged(case, gen):
    dt = _DTYPES[case["dtype"]]
    d, hq, hkv, page, b = case["head_dim"], case["heads"], case["kv_heads"], case["page"], case["batch"]
    q_lens, own_lens = _lengths(case)
    n_shared = case["shared"] // page
    counts = [-(-n // page) for n in own_lens]
    n_pages = n_shared + sum(counts) + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)      # as an allocator leaves them
    table = torch.zeros(b, n_shared + max(counts), dtype=torch.int32, device="cuda")
    first = n_shared
    for i, n in enumerate(counts):
        table[i, :n_shared] = order[:n_shared]
        table[i, n_shared:n_shared + n] = order[first:first + n]
        first += n
    tokens = sum(q_lens)
    shape = (n_pages, hkv, page, d) if case["layout"] == "HND" else (n_pages, page, hkv, d)
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    kv_lens = [n + case["shared"] for n in own_lens]
    state = dict(case=case, widths=_widths(case), q_lens=q_lens, lens=kv_lens, cu=cu, table=table,
                 k_pages=_randn(gen, shape, dt), v_pages=_randn(gen, shape, dt),
                 kv_lens=torch.tensor(kv_lens, dtype=torch.int32, device="cuda"),
                 cu_q=None if case["q_max"] == 1 else torch.tensor(cu, dtype=torch.int32, device="cuda"),
                 max_q=max(q_lens), shared_pages=order[:n_shared].clone() if n_shared else None)
    # one projection gives q, k and v of a token side by side
    qkv = _randn(gen, (tokens, hq + 2 * hkv, d), dt)
    state["q"], state["k"], state["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = _prepare_rotary(case, gen) if case["op"] == "rotary" else _prepare_paged(case, gen)
    inv = []
    for w in state["widths"]:
        inv += [10000.0 ** (-2.0 * i / w) for i in range(w // 2)]
    state["inv_freq"] = torch.tensor(inv, dtype=torch.float64, device="cuda")
    state["axis"] = torch.tensor([a for a, w in enumerate(state["widths"]) for _ in range(w // 2)], device="cuda")
    if own:
        from sageattention_rdna3_b200 import PagedKV, rotary_axes
        state["rotary"] = rotary_axes(case["head_dim"], state["widths"], interleaved=case["interleaved"])
        if case["op"] != "rotary":
            state["cache"] = PagedKV(state["k_pages"], state["v_pages"], case["layout"])
    return state


# ---------------------------------------------------------------- plain forms ----------------------------------

def _angles(state, positions):
    """cos and sin of every token and pair, [T, pairs]; the angle in 64 bits, as positions may be far from zero."""
    if positions.dim() == 1:
        positions = positions[:, None]
    angle = positions.double()[:, state["axis"]] * state["inv_freq"]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _rotate(x, cos, sin, interleaved):
    """x [.., pairs of D], cos / sin broadcast to [.., pairs]; 32 bits."""
    n = cos.size(-1)
    x = x.float()
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        out[..., 0:2 * n:2] = a * cos - b * sin
        out[..., 1:2 * n:2] = a * sin + b * cos
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        out[..., :n] = a * cos - b * sin
        out[..., n:2 * n] = a * sin + b * cos
    return out


def _plain_rotary(state):
    case = state["case"]
    cos, sin = _angles(state, state["positions"])
    if case["layout"] == "NHD":
        cos, sin = cos[:, None], sin[:, None]
    dt = state["q"].dtype
    outs = [_rotate(state[n].detach(), cos, sin, case["interleaved"]).to(dt) for n in ("q", "k")]
    if case["train"]:
        outs += [_rotate(state[n], cos, -sin, case["interleaved"]).to(dt) for n in ("grad_q", "grad_k")]
    return tuple(outs)


def _plain_append(state):
    case = state["case"]
    page = case["page"]
    pos = torch.cat([torch.arange(n - m, n, device="cuda") for m, n in zip(state["q_lens"], state["lens"])])
    seq = torch.repeat_interleave(torch.arange(case["batch"], device="cuda"),
                                  torch.tensor(state["q_lens"], device="cuda"), output_size=pos.numel())
    cos, sin = _angles(state, pos)
    cos, sin = cos[:, None], sin[:, None]
    dt = state["q"].dtype
    q = _rotate(state["q"], cos, sin, case["interleaved"]).to(dt)
    k = _rotate(state["k"], cos, sin, case["interleaved"]).to(dt)
    pid, slot = state["table"][seq, pos // page].long(), pos % page
    for pages, rows in ((state["k_pages"], k), (state["v_pages"], state["v"])):
        if case["layout"] == "NHD":
            pages[pid, slot] = rows
        else:
            pages[pid, :, slot] = rows
    return q, state["k_pages"], state["v_pages"]


def _gather(pages, ids, layout, count):
    """Keys or values of the pages `ids`, [Hkv, count, D] in 32 bits."""
    x = pages[ids.long()].float()
    if layout == "NHD":
        x = x.permute(2, 0, 1, 3)
    else:
        x = x.permute(1, 0, 2, 3)
    return x.reshape(x.size(0), -1, x.size(3))[:, :count]


def _plain_attend(state):
    # (one sequence after the other: padded to the longest one, the batch would be several times the work)
    case = state["case"]
    d, hq, hkv, page = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    rep = hq // hkv
    out = torch.empty(state["cu"][-1], hq, d, dtype=state["q"].dtype, device="cuda")
    lse = torch.empty(state["cu"][-1], hq, dtype=torch.float32, device="cuda")
    for i, (m, n) in enumerate(zip(state["q_lens"], state["lens"])):
        t0, t1 = state["cu"][i], state["cu"][i + 1]
        ids = state["table"][i, :-(-n // page)]
        k, v = _gather(state["k_pages"], ids, case["layout"], n), _gather(state["v_pages"], ids, case["layout"], n)
        # [Hkv, group * m, D]: the heads of a group stand one after the other
        q = state["q"][t0:t1].float().reshape(m, hkv, rep, d).permute(1, 2, 0, 3).reshape(hkv, rep * m, d)
        s = torch.matmul(q, k.transpose(1, 2)) * d ** -0.5
        if case["causal"] and m > 1:
            row = torch.arange(m, device="cuda").repeat(rep)[:, None]
            s = s.masked_fill(torch.arange(n, device="cuda")[None, :] > row + (n - m), float("-inf"))
        top = s.amax(dim=-1, keepdim=True)
        p = torch.exp(s - top)
        total = p.sum(dim=-1, keepdim=True)
        o = torch.matmul(p, v) / total
        out[t0:t1] = o.reshape(hkv, rep, m, d).permute(2, 0, 1, 3).reshape(m, hq, d).to(out.dtype)
        if case["lse"]:
            lse[t0:t1] = (top + torch.log(total)).reshape(hkv, rep, m).permute(2, 0, 1).reshape(m, hq)
    return (out, lse) if case["lse"] else out


def run(state):
    case = state["case"]
    if not own:
        return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend, "shared": _plain_attend}[case["op"]](state)
    from sageattention_rdna3_b200 import apply_rotary, paged_kv_append, sageattn_paged
    if case["op"] == "rotary":
        q, k = apply_rotary(state["q"], state["k"], state["positions"], state["rotary"], tensor_layout=case["layout"])
        if not case["train"]:
            return q, k
        dq, dk = torch.autograd.grad((q, k), (state["q"], state["k"]), (state["grad_q"], state["grad_k"]))
        return q.detach(), k.detach(), dq, dk
    if case["op"] == "append":
        q = paged_kv_append(state["cache"], state["k"], state["v"], state["table"], state["kv_lens"], cu_q=state["cu_q"],
                            rotary=state["rotary"], q=state["q"])
        return q, state["k_pages"], state["v_pages"]
    return sageattn_paged(state["q"], state["cache"], state["table"], state["kv_lens"], cu_q=state["cu_q"],
                          max_q=state["max_q"], is_causal=case["causal"], return_lse=case["lse"],
                          shared_pages=state["shared_pages"])


# ---------------------------------------------------------------- in 64 bits -----------------------------------

def _exact_rotation(x, phase, interleaved):
    """x times exp(i phase), pair by pair, as complex numbers in 64 bits."""
    n = phase.size(-1)
    y = x.double().clone()
    if interleaved:
        z = torch.view_as_complex(y[..., :2 * n].reshape(*y.shape[:-1], n, 2).contiguous())
    else:
        z = torch.complex(y[..., :n].contiguous(), y[..., n:2 * n].contiguous())
    z = z * torch.polar(torch.ones_like(phase), phase)
    if interleaved:
        y[..., :2 * n] = torch.view_as_real(z).reshape(*y.shape[:-1], 2 * n)
    else:
        y[..., :n], y[..., n:2 * n] = z.real, z.imag
    return y


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        pos = state["positions"].double().reshape(case["tokens"], -1)
        phase = torch.stack([pos[:, a] * f for a, f in zip(state["axis"].tolist(), state["inv_freq"].tolist())], dim=1)
        if case["layout"] == "NHD":
            phase = phase.unsqueeze(1)
        names = [("q", 1), ("k", 1)] + ([("grad_q", -1), ("grad_k", -1)] if case["train"] else [])
        return tuple(_exact_rotation(state[n].detach(), sign * phase, case["interleaved"]) for n, sign in names)
    d, page, rep = case["head_dim"], case["page"], case["heads"] // case["kv_heads"]
    by_head = case["layout"] == "HND"
    if case["op"] == "append":
        k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
        rotated = []
        table = state["table"].tolist()
        for i, (m, n) in enumerate(zip(state["q_lens"], state["lens"])):
            t0 = state["cu"][i]
            pos = torch.arange(n - m, n, dtype=torch.float64, device="cuda")
            phase = (pos[:, None] * state["inv_freq"]).unsqueeze(1)
            rotated.append(_exact_rotation(state["q"][t0:t0 + m], phase, case["interleaved"]))
            k = _exact_rotation(state["k"][t0:t0 + m], phase, case["interleaved"])
            v = state["v"][t0:t0 + m].double()
            j = n - m
            while j < n:                              # page by page
                stop = min(n, (j // page + 1) * page)
                at, rows = slice(j % page, j % page + stop - j), slice(j - (n - m), stop - (n - m))
                for pages, x in ((k_pages, k), (v_pages, v)):
                    if by_head:
                        pages[table[i][j // page], :, at] = x[rows].transpose(0, 1)
                    else:
                        pages[table[i][j // page], at] = x[rows]
                j = stop
        return torch.cat(rotated), k_pages, v_pages
    outs, sums = [], []
    for i, (m, n) in enumerate(zip(state["q_lens"], state["lens"])):
        q = state["q"][state["cu"][i]:state["cu"][i] + m].double()
        ids = state["table"][i, :(n + page - 1) // page].long()
        o = torch.empty(m, case["heads"], d, dtype=torch.float64, device="cuda")
        z = torch.empty(m, case["heads"], dtype=torch.float64, device="cuda")
        hidden = None
        if case["causal"]:
            hidden = torch.ones(m, n, dtype=torch.bool, device="cuda").triu(n - m + 1)
        for h in range(case["kv_heads"]):
            k, v = [(p[ids, h] if by_head else p[ids][:, :, h]).double().reshape(-1, d)[:n]
                    for p in (state["k_pages"], state["v_pages"])]
            for g in range(h * rep, (h + 1) * rep):
                score = q[:, g] @ k.t() / math.sqrt(d)
                if hidden is not None:
                    score[hidden] = float("-inf")
                z[:, g] = torch.logsumexp(score, dim=1)
                o[:, g] = torch.exp(score - z[:, g:g + 1]) @ v
        outs.append(o)
        sums.append(z)
    return (torch.cat(outs), torch.cat(sums)) if case["lse"] else torch.cat(outs)
