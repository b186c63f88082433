"""Batches over a paged cache for the tests: pages in shuffled order, NaN wherever no token stands, and attention in 64 bits."""
from __future__ import annotations

import torch

import helpers as H
from sageattention_rdna3_b200 import PagedKV


class PagedBatch:
    """Sequences of kv_lens[b] keys, the last q_lens[b] of which are new.  Values ~ N(0,1); whatever the cache holds besides
    them is NaN, and page indices behind the last key are wild."""

    def __init__(self, q_lens, kv_lens, Hq, Hkv, D, page, layout, dtype, dev, seed=0, shared=0, spare=2, q_scale=1.0, joint=False):
        self.q_lens, self.kv_lens, self.Hq, self.Hkv, self.D, self.page = list(q_lens), list(kv_lens), Hq, Hkv, D, page
        self.layout, self.dtype, self.dev, self.shared = layout, dtype, dev, shared
        g = torch.Generator().manual_seed(seed)
        n_shared = shared // page
        assert shared % page == 0
        counts = [max(0, -(-n // page) - n_shared) for n in kv_lens]
        n_pages = n_shared + sum(counts) + spare
        order = torch.randperm(n_pages, generator=g, dtype=torch.int64).to(torch.int32)
        width = n_shared + max(counts + [0]) + 1
        table = torch.full((len(kv_lens), width), 0x7ffffff0, dtype=torch.int32)
        at = n_shared
        for b, c in enumerate(counts):
            table[b, n_shared:n_shared + c] = order[at:at + c]
            if not shared:
                assert n_shared == 0
            at += c
        self.shared_ids = order[:n_shared]
        self.counts, self.n_pages = counts, n_pages
        self.table = table
        shape = (n_pages, Hkv, page, D) if layout == "HND" else (n_pages, page, Hkv, D)
        if joint:                                     # keys and values of a page side by side in one tensor
            both = torch.full((n_pages, 2) + shape[1:], float("nan"), dtype=dtype)
            self.k_pages, self.v_pages = both[:, 0], both[:, 1]
            self._both = both
        else:
            self.k_pages, self.v_pages = (torch.full(shape, float("nan"), dtype=dtype) for _ in range(2))
        shared_kv = [torch.randn(shared, Hkv, D, generator=g).to(dtype) for _ in range(2)]
        self.k, self.v = [], []
        for b, n in enumerate(kv_lens):
            k, v = (torch.randn(n, Hkv, D, generator=g).to(dtype) for _ in range(2))
            m = min(n, shared)
            k[:m], v[:m] = shared_kv[0][:m], shared_kv[1][:m]
            self.k.append(k)
            self.v.append(v)
            self._put(b, 0, n, k, v)
        if shared:
            for j in range(shared):
                self._slot(int(self.shared_ids[j // page]), j % page, shared_kv[0][j], shared_kv[1][j])
        T = sum(q_lens)
        self.T = T
        self.q = (torch.randn(T, Hq, D, generator=g) * q_scale).to(dtype)
        cu = [0]
        for m in q_lens:
            cu.append(cu[-1] + m)
        self.cu = cu

    def _slot(self, page_id, slot, k, v):
        if self.layout == "HND":
            self.k_pages[page_id, :, slot], self.v_pages[page_id, :, slot] = k, v
        else:
            self.k_pages[page_id, slot], self.v_pages[page_id, slot] = k, v

    def page_of(self, b, j):
        p = j // self.page
        return int(self.shared_ids[p]) if p < len(self.shared_ids) else int(self.table[b, p])

    def _put(self, b, first, last, k, v):
        """Keys [first, last) of sequence b, given as rows 0.. of k and v (the shared ones are left out)."""
        j = max(first, self.shared)
        while j < last:
            stop = min(last, (j // self.page + 1) * self.page)
            pid, at, rows = self.page_of(b, j), slice(j % self.page, j % self.page + stop - j), slice(j - first, stop - first)
            for pages, x in ((self.k_pages, k), (self.v_pages, v)):
                if self.layout == "HND":
                    pages[pid, :, at] = x[rows].transpose(0, 1)
                else:
                    pages[pid, at] = x[rows]
            j = stop

    # ---- what the calls take
    def cache(self):
        if hasattr(self, "_both"):
            both = self._both.to(self.dev)
            return PagedKV(both[:, 0], both[:, 1], self.layout)
        return PagedKV(self.k_pages.to(self.dev), self.v_pages.to(self.dev), self.layout)

    def args(self):
        return self.table.to(self.dev), torch.tensor(self.kv_lens, dtype=torch.int32, device=self.dev)

    def cu_q(self):
        return torch.tensor(self.cu, dtype=torch.int32, device=self.dev)

    def shared_pages(self):
        return self.shared_ids.to(self.dev) if self.shared else None

    # ---- in 64 bits
    def attention(self, causal=True, sm_scale=None, dev="cpu"):
        """(o, lse, bound): bound is what rounding P to the type of V, and the output to its own, may take from o, and
        bound_lse from lse."""
        D, rep = self.D, self.Hq // self.Hkv
        scale = D ** -0.5 if sm_scale is None else sm_scale
        o = torch.zeros(self.T, self.Hq, D, dtype=torch.float64)
        lse = torch.full((self.T, self.Hq), float("-inf"), dtype=torch.float64)
        mag = torch.zeros(self.T, self.Hq, D, dtype=torch.float64)
        dot = torch.zeros(self.T, self.Hq, dtype=torch.float64)
        for b, (m, n) in enumerate(zip(self.q_lens, self.kv_lens)):
            if m == 0 or n == 0:
                continue
            rows = slice(self.cu[b], self.cu[b] + m)
            k = self.k[b].to(dev).double().repeat_interleave(rep, dim=1)
            v = self.v[b].to(dev).double().repeat_interleave(rep, dim=1)
            q = self.q[rows].to(dev).double()
            s = torch.einsum("qhd,khd->hqk", q, k) * scale
            # |q| . |k| bounds the fp32 sums of the scores
            dot[rows] = (torch.einsum("qhd,khd->hqk", q.abs(), k.abs()).amax(-1) * abs(scale)).t().cpu()
            if causal:
                i = torch.arange(m, device=dev)[:, None]
                s = s.masked_fill(torch.arange(n, device=dev)[None] > i + (n - m), float("-inf"))
            seen = (s > float("-inf")).any(-1)
            z = torch.logsumexp(s, -1)
            p = torch.exp(s - torch.where(seen, z, torch.zeros_like(z))[..., None])
            p = torch.where(seen[..., None], p, torch.zeros_like(p))
            o[rows] = torch.einsum("hqk,khd->qhd", p, v).cpu()
            mag[rows] = torch.einsum("hqk,khd->qhd", p, v.abs()).cpu()
            lse[rows] = z.t().cpu()
        # Scores: D products summed in fp32 and a scale, within (D + 3) 2^-24 of |q|.|k| scale; an error e of a score is a
        # factor 1 + e of its p, and of the sum.  exp2 to 2^-22, fp32 sums of up to 2^17 terms in parts: below 2^-18 of
        # sum p |v| in all.  P rounded to the 16-bit type: eps / 2 of every p |v|.  One rounding of the result.
        eps = torch.finfo(self.dtype).eps
        score = (D + 3) * 2.0 ** -24 * dot
        bound = mag * (eps / 2 + 2 * score[..., None] + 2.0 ** -18)
        bound = bound + (o.abs() + bound) * eps / 2 + (2.0 ** -24 if self.dtype == torch.float16 else 1e-38)
        bound_lse = score + 2.0 ** -18 + 2.0 ** -23 * torch.where(torch.isfinite(lse), lse.abs(), torch.zeros_like(lse))
        return o, lse, bound, bound_lse


def randn(shape, seed, dtype, dev):
    return H.randn(shape, seed, dtype, dev)
