"""Plain implementations of the paged cache's operators for its tests: request by request and page by
page in Python lists, attention in float64, and the bounds that the attention's outputs are held to."""
import math

import torch


class PageState:
    """resize_pages on Python lists: the free pages a stack, all or nothing."""

    def __init__(self, requests, width, pages, page):
        self.page, self.width, self.pages = page, width, pages
        self.lens = [0] * requests
        self.table = [[-1] * width for _ in range(requests)]
        self.free = list(range(pages))[::-1]

    def resize(self, new, tokens):
        """(slots, pos, cu, status)"""
        need = lambda n: -(-n // self.page)  # noqa: E731
        cap = self.width * self.page
        refused = lambda s: ([-1] * tokens, [0] * tokens, [0] * (len(new) + 1), s)  # noqa: E731
        if any(not 0 <= n <= cap for n in new):
            return refused(-1)
        if sum(max(0, n - o) for o, n in zip(self.lens, new)) > tokens:
            return refused(-2)
        lack = sum(max(0, need(n) - need(o)) for o, n in zip(self.lens, new)) - len(self.free)
        if lack > 0:
            return refused(lack)
        slots, pos, cu = [], [], [0]
        for b, (o, n) in enumerate(zip(self.lens, new)):
            for e in range(need(o), need(n)):
                self.table[b][e] = self.free.pop()
            for j in range(o, n):
                slots.append(self.table[b][j // self.page] * self.page + j % self.page)
                pos.append(j)
            cu.append(len(slots))
        back = []
        for b, (o, n) in enumerate(zip(self.lens, new)):
            for e in range(need(n), need(o)):
                back.append(self.table[b][e])
                self.table[b][e] = -1
        self.free += back[::-1]
        self.lens = list(new)
        spare = tokens - len(slots)
        return slots + [-1] * spare, pos + [0] * spare, cu, 0


def gather(pool, row, n):
    """The first n tokens of a request with table row `row`: (Hkv, n, d) float64 on the CPU."""
    page = pool.shape[2]
    ids = row[:-(-n // page)].long()
    x = pool[ids].double().cpu()  # (pages, Hkv, page, d)
    return x.transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]


def attend(q, kpool, vpool, table, lens, scale, window=0):
    """(out, lse, tol_out, tol_lse) in float64 on the CPU.

    The bounds are sums of what the arithmetic may be off by, u = 2^-24:
      a score        its d products are exact or one rounding, added in fp32 in any order, then scaled:
                     |ds| <= (d + 3) u scale sum |q_i k_i|
      a weight       exp2 of (score - maximum) in fp32: relative |ds| of its own score, and of the
                     maximum's, plus 4 u for exp2 and u times the exponent's size (at most 150)
      the 16-bit products' weights are the sum of two 16-bit parts, 2^-14 off at most (bf16: the second
                     part holds at least 8 bits below the first's 7)
      the sums       n terms in fp32 in any order: n u of the sum of their sizes, numerator and
                     denominator, and as much again for the joins of partial sums (fewer than n)
    so an output is off by at most A (2 (2 ds + 160 u) + 2^-14 + 4 n u), A = sum w |v| / sum w, and by
    the rounding to its type, half a step of the value, or of the smallest normal number's."""
    B, hq, d = q.shape
    hkv, G = kpool.shape[1], hq // kpool.shape[1]
    u = 2.0 ** -24
    out = torch.zeros(B, hq, d, dtype=torch.float64)
    lse = torch.full((B, hq), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    fi = torch.finfo(q.dtype)
    for b, n in enumerate(lens.tolist()):
        if n == 0:
            continue
        first = max(0, n - window) if window else 0
        k, v = gather(kpool, table[b], n)[:, first:], gather(vpool, table[b], n)[:, first:]
        for h in range(hq):
            x = q[b, h].double().cpu()
            kh, vh = k[h // G], v[h // G]
            s = kh @ x * scale
            ds = float((kh.abs() @ x.abs()).max()) * abs(scale) * (d + 3) * u
            w = torch.softmax(s, 0)
            out[b, h] = w @ vh
            lse[b, h] = torch.logsumexp(s, 0)
            rel = 2 * (2 * ds + 160 * u) + 4 * (n - first) * u
            split = 0.0 if q.dtype == torch.float32 else 2.0 ** -14
            tol[b, h] = (w @ vh.abs()) * (rel + split) * (1 + fi.eps)
            tol[b, h] += fi.eps / 2 * out[b, h].abs() + fi.tiny * fi.eps
            # the log of a sum that is off by `rel`, and the roundings of log2, of the sum with the
            # maximum and of the change of base
            ltol[b, h] = rel + 8 * u * (float(s.abs().max()) + math.log(n) + 1)
    return out, lse, tol, ltol


def close(got, want, tol):
    """Every finite value within its bound, infinities and NaN in the same places."""
    got = got.double().cpu()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)])
    off = (got - want).abs()[fin] - tol[fin]
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())
