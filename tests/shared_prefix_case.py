"""Batches whose requests share their first positions in groups, and their attention in 64 bits."""

from __future__ import annotations

import torch


class Case:
    """`groups`: a list of (prefix, [(own cached positions, new tokens), ...]).  The cache holds NaN wherever
    no position of a request lies; pages are shuffled; a page that the prefix fills only in part is
    each member's own.  `loose`: requests behind the groups, in none of them, as (cached, new)."""

    def __init__(self, nq, nkv, hd, page, groups, dtype, seed=0, loose=(), extra_columns=0, rows_in_front=0,
                 rows_behind=0, spare_pages=2, scale=None, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.nq, self.nkv, self.hd, self.page, self.dtype = nq, nkv, hd, page, dtype
        self.scale = hd ** -0.5 if scale is None else scale
        requests, off, prefix = [], [0], []
        for P, members in groups:
            requests += [(P, own, new) for own, new in members]
            off.append(len(requests))
            prefix.append(P)
        requests += [(0, cached, new) for cached, new in loose]
        self.requests = requests
        R = len(requests)
        total = [P + own + new for P, own, new in requests]
        blocks = [-(-t // page) for t in total]
        shared = [P // page for P, _ in groups]
        n_pages = sum(shared) + sum(blocks) - sum(s * len(m) for s, (_, m) in zip(shared, groups)) + spare_pages
        ids = torch.randperm(n_pages, generator=g).tolist()
        table = torch.full((R, max(blocks) + 1), -1, dtype=torch.int32)
        keys = torch.full((n_pages, nkv, page, hd), float("nan"), dtype=dtype)
        values = torch.full((n_pages, nkv, page, hd), float("nan"), dtype=dtype)
        self.k, self.v = [], []                         # of every request, [positions, nkv, hd]
        at = 0

        def draw(n):
            return [torch.randn((n, nkv, hd), generator=g).to(dtype) for _ in range(2)]

        r = 0
        for gi, members in enumerate([m for _, m in groups] + [[m] for m in loose]):
            P = prefix[gi] if gi < len(groups) else 0
            kp, vp = draw(P)
            first = ids[at:at + P // page]
            at += P // page
            for own, new in members:
                ko, vo = draw(own + new)
                k, v = torch.cat([kp, ko]), torch.cat([vp, vo])
                mine = first + ids[at:at + blocks[r] - len(first)]
                at += blocks[r] - len(first)
                table[r, :blocks[r]] = torch.tensor(mine, dtype=torch.int32)
                pos = torch.arange(total[r])
                where = torch.tensor(mine)[pos // page]
                keys[where, :, pos % page], values[where, :, pos % page] = k, v
                self.k.append(k)
                self.v.append(v)
                r += 1
        new = [n for _, _, n in requests]
        cu = torch.tensor([rows_in_front] + new).cumsum(0)
        T = int(cu[-1]) + rows_behind
        width = nq * hd + extra_columns
        self.rows = torch.randn((T, width), generator=g).to(dtype)
        self.cu = cu.tolist()

        def ints(x):
            return torch.as_tensor(x, dtype=torch.int32).contiguous().to(device)

        self.table, self.cu_q = ints(table), ints(cu)
        self.ctx_len = ints([P + own for P, own, _ in requests])
        self.prefix_len, self.group_off = ints(prefix), ints(off)
        self.keys, self.values = keys.to(device), values.to(device)
        self.qkv = self.rows.to(device)
        self.out = torch.full((T, nq * hd), 7.0, dtype=dtype, device=device)
        self.single = all(n == 1 for n in new) and rows_in_front == rows_behind == 0

    def call(self, ops, cu_q="as needed", out=None):
        cu = (None if self.single else self.cu_q) if cu_q == "as needed" else cu_q
        out = self.out if out is None else out
        ops.shared_prefix_attention(self.qkv, self.keys, self.values, self.table, self.ctx_len, self.prefix_len,
                                    self.group_off, self.nq, self.nkv, self.hd, self.scale, out, cu_q=cu)
        return out

    def check(self, got, sums):
        """`got` [T, nq * hd] against 64 bits.

        A probability is a rounding of `sums` ("bfloat16": 2^-8, as the tensor cores take it) or none; a
        score s = scale q.k has hd products and sums of relative error 2^-23 each of |q|.|k| at most, which
        moves the probability by as much as the score; the hardware's 2^x and the product with log2(e) are off by 2^-21;
        sums over n keys are off by 2^-23 a term; joining parts twice 2^-21; the output is rounded once.
        All bounds are on sum p |v|."""
        got = got.double().cpu()
        half = torch.finfo(self.dtype).eps / 2
        per = self.nq // self.nkv
        for r, (P, own, new) in enumerate(self.requests):
            k, v = self.k[r].double(), self.v[r].double()
            q = self.rows[self.cu[r]:self.cu[r + 1], :self.nq * self.hd].double().view(new, self.nkv, per, self.hd)
            n = P + own + new
            s = torch.einsum("tkpd,nkd->tkpn", q, k) * self.scale
            size = torch.einsum("tkpd,nkd->tkpn", q.abs(), k.abs()).amax(-1, keepdim=True) * self.scale
            seen = torch.arange(n)[None] <= (P + own + torch.arange(new))[:, None]
            s = s.masked_fill(~seen[:, None, None], float("-inf"))
            w = torch.softmax(s, -1)
            want = torch.einsum("tkpn,nkd->tkpd", w, v)
            span = torch.einsum("tkpn,nkd->tkpd", w, v.abs())
            off = size * (self.hd + 4) * 2.0 ** -23 + s.masked_fill(~seen[:, None, None], 0).abs().amax(-1, keepdim=True) * 2.0 ** -22
            tol = span * ((2.0 ** -8 if sums == "bfloat16" else 0.0) + 2 * off + (n + 64) * 2.0 ** -23) + want.abs() * half
            have = got[self.cu[r]:self.cu[r + 1]].view_as(want)
            bad = (have - want).abs() > tol
            assert torch.isfinite(have).all() and not bad.any(), (
                r, (P, own, new), int(bad.sum()), float(((have - want).abs() / tol).max()))
        # rows of no request are as they were
        for a, b in ((0, self.cu[0]), (self.cu[-1], got.shape[0])):
            assert (got[a:b] == 7.0).all()
