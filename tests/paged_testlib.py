"""Paged-cache test helpers: ragged batches over a pool whose unneeded places
hold NaN, and the operators' definitions in 64 bits (numpy, no library code)."""
from __future__ import annotations

import math

import numpy as np

EPS_HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative


def torch_dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def sees(p, j, window, sinks):
    """Which keys j the token with index p sees (arrays broadcast)."""
    return (j <= p) & ((window == 0) | (j < sinks) | (j > p - window))


class Case:
    """A ragged batch on the host, its pool on the device.  q_len/kv_len per
    sequence; `prefix` shared tokens in front of every sequence's own.  Places
    that no token of the call needs hold NaN, pages that none needs are -1 in
    the table.  layout: "heads" [page, head, slot, dim], "slots" [page, slot,
    head, dim], "pair" (keys and values of a page side by side)."""

    def __init__(self, V, torch, dtype="bf16", heads=8, kv_heads=2, dim=64, page=16, q_len=(1,), kv_len=(5,),
                 window=0, sinks=0, prefix=0, layout="heads", seed=0, device="cuda", spare_tokens=0, q_scale=1.5,
                 poison=True, max_kv=None, max_q=None):
        rng = np.random.default_rng(seed)
        self.V, self.torch, self.dtype, self.device = V, torch, dtype, device
        self.heads, self.kv_heads, self.dim, self.page = heads, kv_heads, dim, page
        self.q_len, self.kv_len, self.window, self.sinks, self.prefix = list(q_len), list(kv_len), window, sinks, prefix
        self.n = len(self.q_len)
        self.tokens = sum(self.q_len) + spare_tokens
        td = torch_dtype(dtype)
        n_pre = -(-prefix // page)
        width = max([1] + [-(-x // page) for x in self.kv_len])
        table = np.full((self.n, width), -1, np.int64)
        used = n_pre
        for s in range(self.n):
            for t in range(self.kv_len[s]):
                if table[s, t // page] < 0 and self.needed(s, prefix + t):
                    table[s, t // page] = used
                    used += 1
        self.n_pages = used + 2
        order = rng.permutation(self.n_pages)
        self.table = np.where(table >= 0, order[np.maximum(table, 0)], -1).astype(np.int32)
        pre = order[:n_pre].astype(np.int32)
        for i in range(n_pre):  # prefix pages that no query's window reaches
            if not any(self.needed(s, t) for s in range(self.n) for t in range(i * page, min(prefix, (i + 1) * page))):
                pre[i] = -1
        self.pre = pre
        rnd = lambda *sh: torch.from_numpy(rng.standard_normal(sh).astype(np.float32)).to(td)  # noqa: E731
        q = rnd(self.tokens, heads, dim) * q_scale
        # logical keys and values, rounded to the dtype: [prefix + own tokens of each sequence]
        self.pk, self.pv = rnd(prefix, kv_heads, dim), rnd(prefix, kv_heads, dim)
        self.k = [rnd(x, kv_heads, dim) for x in self.kv_len]
        self.v = [rnd(x, kv_heads, dim) for x in self.kv_len]
        fill = math.nan if poison else 0.0
        shape = (self.n_pages, kv_heads, page, dim)
        kp, vp = torch.full(shape, fill, dtype=td), torch.full(shape, fill, dtype=td)
        for i in range(prefix):
            if pre[i // page] >= 0 and any(self.needed(s, i) for s in range(self.n)):
                kp[pre[i // page], :, i % page] = self.pk[i]
                vp[pre[i // page], :, i % page] = self.pv[i]
        for s in range(self.n):
            for t in range(self.kv_len[s]):
                if self.table[s, t // page] >= 0 and self.needed(s, prefix + t):
                    kp[self.table[s, t // page], :, t % page] = self.k[s][t]
                    vp[self.table[s, t // page], :, t % page] = self.v[s][t]
        if layout == "heads":
            self.kp, self.vp = kp.to(device), vp.to(device)
        elif layout == "slots":
            self.kp, self.vp = (x.transpose(1, 2).contiguous().to(device).transpose(1, 2) for x in (kp, vp))
        else:
            both = torch.stack((kp, vp), 1).to(device)
            self.kp, self.vp = both[:, 0], both[:, 1]
        self.q = q.to(device)
        self.q_host = q
        i32 = dict(dtype=torch.int32, device=device)
        self.q_start = torch.tensor([0] + list(np.cumsum(self.q_len)), **i32)
        self.kv = torch.tensor(self.kv_len, **i32)
        self.table_dev = torch.from_numpy(self.table).to(device)
        self.pre_dev = torch.from_numpy(pre).to(device)
        self.pre_len = torch.tensor([prefix], **i32)
        self.status = torch.zeros(1, **i32)
        if device == "cuda":
            self.cache = V.PagedKvCache(self.kp, self.vp)
            self.batch = V.PagedBatch(self.q_start, self.kv, self.table_dev, self.tokens,
                                      max_q or max([1] + self.q_len), max_kv, status=self.status)

    def needed(self, s, j):
        """Whether some token of the call's sequence s sees key j (prefix first)."""
        last = self.prefix + self.kv_len[s] - 1
        first = last - self.q_len[s] + 1
        if self.q_len[s] == 0 or j > last:
            return False
        return self.window == 0 or j < self.sinks or j > first - self.window

    def run(self, q=None, **kw):
        V = self.V
        q = self.q if q is None else q
        if self.prefix:
            return V.paged_prefix_attention(self.cache, self.batch, self.pre_dev, self.pre_len,
                                            len(self.pre) * self.page, q, sliding_window=self.window,
                                            n_sinks=self.sinks, **kw)
        return V.paged_attention(self.cache, self.batch, q, sliding_window=self.window, n_sinks=self.sinks, **kw)

    def expected(self, scale=None):
        """(out, tolerance) [tokens, heads, dim] in 64 bits; rows of no sequence are NaN.

        Tolerance, all steps relative: scores are sums of `dim` exact products
        in 32 bits (f32 tensors: products of split operands, 2^-20), so a score
        is off by d = scale * sum|q||k| * (dim 2^-24 [+ 2^-20]), a weight by 2d
        plus 2^-11 of the exponential's approximation (2^-21 for f32) plus its
        rounding to the type; a result moves by that share of sum p|v|, and is
        rounded once."""
        scale = scale or 1.0 / math.sqrt(self.dim)
        u = EPS_HALF[self.dtype]
        g = self.heads // self.kv_heads
        out = np.full((self.tokens, self.heads, self.dim), np.nan)
        tol = np.zeros_like(out)
        at = 0
        f64 = lambda t: t.float().numpy().astype(np.float64)  # noqa: E731
        qh, pk, pv = f64(self.q_host), f64(self.pk), f64(self.pv)
        for s in range(self.n):
            k, v = (np.concatenate((a, f64(b))) for a, b in ((pk, self.k[s]), (pv, self.v[s])))
            j = np.arange(k.shape[0])
            for i in range(self.q_len[s]):
                p = self.prefix + self.kv_len[s] - self.q_len[s] + i
                seen = sees(p, j, self.window, self.sinks)
                kk, vv = np.repeat(k[seen], g, 1), np.repeat(v[seen], g, 1)  # [keys, heads, dim]
                if not seen.any():
                    out[at + i] = 0.0
                    continue
                q = qh[at + i]
                with np.errstate(invalid="ignore", over="ignore"):
                    sc = np.einsum("hd,jhd->hj", q, kk) * scale
                    w = np.exp(sc - sc.max(-1, keepdims=True))
                    w /= w.sum(-1, keepdims=True)
                    out[at + i] = np.einsum("hj,jhd->hd", w, vv)
                    size = np.einsum("hj,jhd->hd", w, np.abs(vv))
                    d = np.einsum("hd,jhd->hj", np.abs(q), np.abs(kk)).max(-1) * scale
                d = d * (self.dim * 2.0 ** -24 + (2.0 ** -20 if self.dtype == "f32" else 0))
                loose = 2.0 ** -20 if self.dtype == "f32" else 2.0 ** -11
                tol[at + i] = u * np.abs(out[at + i]) + (2 * d[:, None] + u + loose) * size + 1e-30
            at += self.q_len[s]
        return out, tol

    def check(self, got, scale=None):
        want, tol = self.expected(scale)
        got = got.detach().cpu().float().numpy().astype(np.float64)
        mine = ~np.isnan(want)
        assert np.array_equal(np.isnan(got[:sum(self.q_len)]), ~mine[:sum(self.q_len)]), "NaN where there should be none"
        worst = np.max(np.where(mine, np.abs(got - want) - tol, -1.0))
        assert worst <= 0, f"off by {np.nanmax(np.abs(got - want)):.3e}, {worst:.3e} over the tolerance"
        return want
