"""Helpers of the paged-cache tests: a pool whose every element that no sequence owns is NaN, the attention in 64 bits, and the
error that the kernels' roundings allow."""
import math

import torch

from mycaffe_b200 import paged

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


class Setup:
    """seqs: (new tokens, positions) of each sequence.  drop: (sequence, page index) pairs that are not held."""

    def __init__(self, seqs, heads, kv, hs, page, act, cache, seed=0, drop=(), pad=0, stride_pages=0, max_new=None, max_len=None):
        self.seqs, self.heads, self.kv, self.hs, self.page = seqs, heads, kv, hs, page
        g = torch.Generator("cuda").manual_seed(seed)
        self.act, self.cache_t = DT[act], DT[cache]
        need = [-(-n // page) for _, n in seqs]
        n_pages, stride = sum(need) + 2, max(need + [1]) + 2
        order = torch.randperm(n_pages, generator=g, device="cuda").tolist()
        size = page * kv * hs
        pools = []
        for _ in range(2):
            raw = torch.full((n_pages, size + stride_pages), math.nan, device="cuda", dtype=self.cache_t)
            pools.append(raw[:, :size].unflatten(1, (page, kv, hs)))
        self.k_pages, self.v_pages = pools
        table = torch.full((len(seqs), stride), -1, dtype=torch.int32)
        self.k, self.v = [], []
        at = 0
        for b, (_, n) in enumerate(seqs):
            k, v = (torch.randn(n, kv, hs, generator=g, device="cuda").to(self.cache_t) for _ in range(2))
            self.k.append(k)
            self.v.append(v)
            for i in range(need[b]):
                table[b, i] = order[at]
                lo, hi = i * page, min(n, (i + 1) * page)
                self.k_pages[order[at], : hi - lo] = k[lo:hi]
                self.v_pages[order[at], : hi - lo] = v[lo:hi]
                at += 1
        self.held = [torch.ones(n, dtype=torch.bool, device="cuda") for _, n in seqs]
        for b, i in drop:
            table[b, i] = -1
            self.held[b][i * page:(i + 1) * page] = False
        self.table = table.cuda()
        self.starts = torch.tensor([0] + [n for n, _ in seqs]).cumsum(0).to(torch.int32).cuda()
        self.lengths = torch.tensor([n for _, n in seqs], dtype=torch.int32).cuda()
        self.used = sum(n for n, _ in seqs)
        self.n_tokens = self.used + pad
        self.q = torch.randn(self.n_tokens, heads, hs, generator=g, device="cuda").to(self.act)
        self.out = torch.full_like(self.q, 7.0)
        self.max_new = max_new or max(max(n for n, _ in seqs), 1)
        self.max_len = max_len or max(max(n for _, n in seqs), 1)
        self.cache = paged.PagedCache(self.k_pages, self.v_pages, heads)
        self.batch = self.cache.batch(self.starts, self.lengths, self.table, self.n_tokens, self.max_new, self.max_len)

    def exact(self, q=None, scale=None):
        """Attention in 64 bits and, for each output element, what the kernels' roundings may move it by.

        Logits: sums of D products in fp32 (D 2^-23 of the sum of magnitudes, doubled for the scaling), fp32 queries over bf16 pages
        as two bf16 halves (2^-8 2^-8 of the sum of magnitudes); the exponential's argument and the exponential (2^-21).  A logit off
        by d moves a probability by d and the row's sum by as much: 2 d of the mean magnitude A = sum p |v|.  Probabilities are rounded
        to bf16 (bf16 queries: 2^-8) or two halves (2^-16), sums of n products in fp32 (n 2^-23), the output to its type."""
        q = (self.q if q is None else q).double()
        scale = scale or 1.0 / math.sqrt(self.hs)
        group = self.heads // self.kv
        out, tol = torch.full_like(q, 7.0), torch.zeros_like(q)
        bf16 = self.act == torch.bfloat16
        halves = not bf16 and self.cache_t == torch.bfloat16
        row = 0
        for b, (new, n) in enumerate(self.seqs):
            k, v = self.k[b].double(), self.v[b].double()
            for i in range(new):
                keep = self.held[b][: n - new + i + 1]
                m = int(keep.sum())
                kk, vv = k[: n - new + i + 1][keep], v[: n - new + i + 1][keep]
                if m == 0:
                    out[row] = 0
                else:
                    qq = q[row].view(self.kv, group, self.hs)
                    s = torch.einsum("hgd,nhd->hgn", qq, kk) * scale
                    mag = (torch.einsum("hgd,nhd->hgn", qq.abs(), kk.abs()) * scale).amax(-1)
                    p = torch.softmax(s, -1)
                    o = torch.einsum("hgn,nhd->hgd", p, vv)
                    a = torch.einsum("hgn,nhd->hgd", p, vv.abs())
                    d = mag * (2 * self.hs * 2.0 ** -23 + (2.0 ** -16 if halves else 0)) + 2.0 ** -21
                    r = 2 * d + (2.0 ** -8 if bf16 else (2.0 ** -16 if halves else 0)) + (m + 64) * 2.0 ** -23
                    out[row] = o.reshape(self.heads, self.hs)
                    tol[row] = (a * r[..., None] + o.abs() * (2.0 ** -8 if bf16 else 2.0 ** -22)).reshape(self.heads, self.hs)
                row += 1
        return out, tol + 1e-30

    def check(self, scale=None):
        ref, tol = self.exact(scale=scale)
        assert torch.isfinite(self.out.double()).all()
        over = ((self.out.double() - ref).abs() / tol).amax().item() if ref.numel() else 0.0
        assert over <= 1.0, over
        return over
