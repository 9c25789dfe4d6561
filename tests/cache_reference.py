"""Problems for the tests of the cache on pages, and the plain definitions in 64 bits on the CPU they are held against,
with the error that each rounding may leave, worked out per element.

Attention, per result element, with p_j the probabilities, A = sum_j p_j |v_j|, n positions seen:
  scores     a product of dh terms in fp32 and two multiplications are off by at most (dh + 2) 2^-24 scale sum |q k| =: d;
             a probability and the sum of all by exp(+-2 d): 2 d each on both sides of the quotient -> 4 d A;
  exp2, sums every exp2, its scaled argument (|s| log2 e 2^-24 absolute, twice for the shift), rescaling and addition:
             n + 64 roundings of 2^-24, and 4 |s|max 2^-24 -> (n + 64 + 4 smax) 2^-24 A;
  half       probabilities, of 2^8 at most before they are divided, rounded to half: 2^-11 A, or 2^-25 each where they are below the
             normal range: 2^-25 sum |v_j| (the sum they are divided by is at least 1). That sum may be the exact or the rounded
             ones': in the second case it is off by 2^-11 of itself and n 2^-25, so the result by (2^-11 + n 2^-25) |out| more.
             The result: 2^-11 |out|, 2^-25 at least.
"""
import math

import numpy as np
import torch


class Problem:
    """A cache on pages with everything that is no sequence's position filled with NaN, and a batch over it."""

    def __init__(self, lens, new, heads, kv, dh, page, half, seed, layout="rows", prefix=0, uniform=False, slack=2, spare=3,
                 max_length=None, pad_tokens=0, spread=1.0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.heads, self.kv, self.dh, self.page, self.half = list(lens), list(new), heads, kv, dh, page, half
        dt = torch.float16 if half else torch.float32
        n = len(lens)
        shared = prefix // page
        need = [-(-a // page) for a in lens]
        own = [max(0, a - shared) for a in need]
        pages = shared + sum(own) + spare
        perm = torch.randperm(pages, generator=g).tolist()
        width = max(max(need), 1) + slack
        table = torch.full((n, width), -7, dtype=torch.int32)
        at = shared
        for i in range(n):
            table[i, :min(shared, need[i])] = torch.tensor(perm[:min(shared, need[i])], dtype=torch.int32)
            table[i, shared:shared + own[i]] = torch.tensor(perm[at:at + own[i]], dtype=torch.int32)
            at += own[i]
        if prefix:
            table[0, :shared] = torch.tensor(perm[:shared], dtype=torch.int32)
        self.table = table
        nan = lambda: torch.full((pages, page, kv, dh), float("nan"), dtype=dt)     # noqa: E731
        self.k, self.v = nan(), nan()
        for i in range(n):
            for b in range(need[i]):
                used = min(page, lens[i] - b * page)
                if b < shared and i > 0:
                    continue
                self.k[table[i, b], :used] = (torch.randn((used, kv, dh), generator=g) * spread).to(dt)
                self.v[table[i, b], :used] = torch.randn((used, kv, dh), generator=g).to(dt)
        if prefix and lens[0] < prefix:                 # the prefix stands whole on row 0 of the table
            for b in range(shared):
                self.k[table[0, b]] = (torch.randn((page, kv, dh), generator=g) * spread).to(dt)
                self.v[table[0, b]] = torch.randn((page, kv, dh), generator=g).to(dt)
        self.starts = [0]
        for a in new:
            self.starts.append(self.starts[-1] + a)
        self.tokens = self.starts[-1] + pad_tokens
        self.q = (torch.randn((self.tokens, heads, dh), generator=g) * spread).to(dt)
        self.scale = dh ** -0.5
        self.max_new = max(max(new), 1)
        self.max_length = max_length if max_length is not None else max(max(lens), 1)
        self.uniform = uniform
        self.layout = layout
        self.device = device

    def pool(self, x):
        if self.layout == "heads":
            return x.transpose(1, 2).contiguous().to(self.device).transpose(1, 2)
        return x.to(self.device)

    def place(self, nt):
        """The problem on the device: (cache, batch, q, out), out full of a mark."""
        d = self.device
        self.kd, self.vd = self.pool(self.k), self.pool(self.v)
        cache = nt.KVCache(self.kd, self.vd)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=d)                # noqa: E731
        self.lengths_d, self.table_d = i32(self.lens), self.table.to(d)
        self.starts_d = None if self.uniform else i32(self.starts)
        batch = nt.CacheBatch(self.lengths_d, self.table_d, starts=self.starts_d, tokens=self.tokens, max_new=self.max_new,
                              max_length=self.max_length)
        return cache, batch, self.q.to(d), torch.full_like(self.q, 77.0, device=d)

    def row(self, i, p):
        """Page and row of position p of sequence i."""
        return int(self.table[i, p // self.page]), p % self.page

    def attention(self, causal, absent=()):
        """(expected, tolerance) in 64 bits; rows that belong to nobody expect the mark. absent: page numbers left out."""
        want = torch.full(self.q.shape, 77.0, dtype=torch.float64)
        tol = torch.zeros(self.q.shape, dtype=torch.float64)
        per = self.heads // self.kv
        for i, (size, n) in enumerate(zip(self.lens, self.new)):
            if n == 0:
                continue
            rows = [(p, *self.row(i, p)) for p in range(size)]
            rows = [(p, a, b) for p, a, b in rows if 0 <= a < self.k.shape[0] and a not in absent]
            pos = torch.tensor([p for p, _, _ in rows], dtype=torch.long)
            pg = torch.tensor([a for _, a, _ in rows], dtype=torch.long)
            rw = torch.tensor([b for _, _, b in rows], dtype=torch.long)
            k, v = self.k[pg, rw].double(), self.v[pg, rw].double()                 # [positions, kv, dh]
            q = self.q[self.starts[i]:self.starts[i] + n].double()
            seen = torch.arange(size - n + 1, size + 1) if causal else torch.full((n,), size)
            for h in range(self.heads):
                kh, vh, qh = k[:, h // per], v[:, h // per], q[:, h]
                s = qh @ kh.T * self.scale
                hide = pos[None] >= seen[:, None]
                s = s.masked_fill(hide, -math.inf)
                m = s.amax(-1, keepdim=True) if s.shape[1] else torch.zeros((n, 1), dtype=torch.float64)
                m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
                e = torch.exp(s - m)
                total = e.sum(-1, keepdim=True)
                p = torch.where(total > 0, e / total.clamp(min=1e-300), torch.zeros_like(e))
                vs = torch.where(torch.isfinite(vh), vh, torch.zeros_like(vh))
                o = p @ vs
                a = p @ vs.abs()
                d = ((self.dh + 2) * 2.0 ** -24 * abs(self.scale) * (qh.abs() @ kh.abs().T)).masked_fill(hide, 0.0)
                d = d.amax(-1, keepdim=True) if s.shape[1] else torch.zeros((n, 1), dtype=torch.float64)
                smax = (qh @ kh.T * self.scale).abs().masked_fill(hide, 0.0)
                smax = smax.amax(-1, keepdim=True) if s.shape[1] else torch.zeros((n, 1), dtype=torch.float64)
                t = (4 * d + (len(rows) + 64 + 4 * smax) * 2.0 ** -24) * a + 2.0 ** -126
                if self.half:
                    t = t + 2.0 ** -11 * a + 2.0 ** -25 * ((~hide).double() @ vs.abs()) + torch.maximum(2.0 ** -11 * o.abs(), torch.tensor(2.0 ** -25))
                    t = t + (2.0 ** -11 + 2.0 ** -25 * seen[:, None]) * o.abs()
                    t = t * (1 + 2.0 ** -10)            # the bounds on each other's results
                want[self.starts[i]:self.starts[i] + n, h], tol[self.starts[i]:self.starts[i] + n, h] = o, t
        return want, tol


def assert_within(got, want, tol, what=""):
    got = got.detach().cpu().double()
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        at = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError("%s: %d of %d elements beyond their tolerance, the first at %s: got %r, expected %r within %.3g" % (
            what, int(bad.sum()), bad.numel(), at, float(got[at]), float(want[at]), float(tol[at])))


def rotation_table(positions, rotated, base=10000.0):
    """float [positions][rotated / 2][2] of cosine and sine, the angles in 64 bits."""
    j = np.arange(rotated // 2, dtype=np.float64)
    ang = np.arange(positions, dtype=np.float64)[:, None] * base ** (-2.0 * j / max(rotated, 1))
    return torch.from_numpy(np.stack((np.cos(ang), np.sin(ang)), -1).astype(np.float32))


def rotated_rows(x, cs, pairs):
    """x [tokens, heads, dh] in 64 bits turned by cs [tokens, columns / 2, 2], and what fp32 and one rounding may leave:
    two products, a sum (2^-24 each of its result, the products at most |x c| + |y s| together) and the last rounding."""
    h = cs.shape[1]
    c, s = cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    y = x.double().clone()
    err = torch.zeros_like(y)
    first, second = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if pairs else (slice(0, h), slice(h, 2 * h))
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    fp32 = 2.0 ** -23 * 1.001
    err[..., first], err[..., second] = fp32 * ((a * c).abs() + (b * s).abs()), fp32 * ((b * c).abs() + (a * s).abs())
    if x.dtype == torch.float16:
        last = torch.maximum(2.0 ** -11 * (y.abs() + err), torch.tensor(2.0 ** -25, dtype=torch.float64))
        last[..., 2 * h:] = 0.0
        err = err + last
    return y, err
