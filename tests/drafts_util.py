"""Plain implementations of the drafted tokens' and shared pages' operators for their tests: token by
token and page by page in Python lists, attention in float64 with the bounds its outputs are held to."""
import math

import torch

from tests import paged_util as U


def random_parents(rng, n, reach=9):
    """A tree of n drafted tokens: each continues one of the few before it, or the context."""
    return [t - 1 if rng.random() < 0.4 else max(-1, t - 1 - rng.randrange(reach)) for t in range(n)]


def ancestors(parents):
    """Per token the set of drafted tokens it attends; None where a parent on its way does not fit."""
    seen = []
    for t, p in enumerate(parents):
        up = set() if p == -1 else seen[p] if 0 <= p < t else None
        seen.append(None if up is None else up | {t})
    return seen


def masks_and_pos(parents, n, lens, words, N):
    """(masks, pos) as lists, of requests with n[b] tokens; parents a list over all of them."""
    masks, pos, at = [], [], 0
    for count, total in zip(n, lens):
        fits = count <= total and count <= 32 * words
        for seen in ancestors(parents[at:at + count]):
            if seen is None or not fits:
                masks.append([0] * words)
                pos.append(-1)
                continue
            bits = sum(1 << i for i in seen)
            row = [bits >> 32 * w & 0xffffffff for w in range(words)]
            masks.append([x - (1 << 32) if x >> 31 else x for x in row])
            pos.append(total - count + len(seen) - 1)
        at += count
    pad = N - len(pos)
    return masks + [[0] * words] * pad, pos + [0] * pad


def bit(masks, row, i):
    return masks[row][i // 32] >> i % 32 & 1


def attended(n, ctx, window, masks=None, pos=None):
    """(n, ctx + n) booleans: which keys the drafted tokens of a request attend (masks, pos its rows)."""
    if masks is None:
        t, j = ctx + torch.arange(n)[:, None], torch.arange(ctx + n)
        return (j <= t) & (j > t - window) if window else j <= t
    at = pos
    out = torch.zeros(n, ctx + n, dtype=torch.bool)
    for t in range(n):
        low = at[t] - window if window else -1
        out[t, max(0, min(ctx, low + 1)):ctx] = True
        for i in range(n):
            out[t, ctx + i] = bool(bit(masks, t, i)) and (not window or at[i] > low)
    return out


def attend(q, kpool, vpool, table, lens, cu, scale, window=0, masks=None, pos=None):
    """(out, lse, tol_out, tol_lse) in float64 on the CPU; rows behind the last request's 0 and -inf.

    The bounds are paged_util.attend's, u = 2^-24, over the keys a row attends:
      a score        |ds| <= (d + 3) u scale sum |q_i k_i|
      a weight       exp2 of (score - maximum): its own |ds| and the maximum's, 4 u for exp2 and u times
                     the exponent's size (at most 150)
      its parts      bf16: two, each rounded to 8 bits, leave 2^-9 of 2^-9 of it (three hold it exactly).
                     fp16: two, cut to 11 bits, leave 2^-10 of 2^-10 of it, or 2^-38 of the largest
                     weight where the second falls below fp16's least number (weights are taken up to
                     2^14)
      the sums       the parts' products add up in any order: 3 n terms, the later parts' 2^-7 of the
                     first's or less, so 2 n u of the sum of sizes, the weights' own sum n u, and as much
                     again for the joins of partial sums
    so an output is off by at most A (2 (2 ds + 160 u) + 2^-18 or 2^-20 + 6 n u) + n 2^-37 max |v|
    (fp16), and by half a step of its type."""
    N, hq, d = q.shape
    hkv, G = kpool.shape[1], hq // kpool.shape[1]
    u = 2.0 ** -24
    out = torch.zeros(N, hq, d, dtype=torch.float64)
    lse = torch.full((N, hq), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    fi = torch.finfo(q.dtype)
    cu, lens = cu.tolist(), lens.tolist()
    masks = None if masks is None else masks.tolist()
    pos = None if pos is None else pos.tolist()
    qd = q.double().cpu()
    for b, total in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        rows = slice(cu[b], cu[b + 1])
        see = attended(n, total - n, window, None if masks is None else masks[rows],
                       None if pos is None else pos[rows])
        k, v = U.gather(kpool, table[b], total), U.gather(vpool, table[b], total)
        some = see.any(1)
        count = see.sum(1).double()[:, None]
        kz = torch.where(torch.isfinite(k), k, 0.0)
        vz = torch.where(torch.isfinite(v), v, 0.0)
        for h in range(hq):
            x = qd[rows, h]
            kh, vh = k[h // G], v[h // G]
            s = (x @ kz[h // G].T * scale).masked_fill(~see, -math.inf)
            odd = ~torch.isfinite(kh).all(1)
            if odd.any():
                s[:, odd] = torch.stack([x @ kh[j] for j in odd.nonzero()[:, 0]], 1) * scale
                s = s.masked_fill(~see, -math.inf)
            w = torch.softmax(s, 1)
            w = torch.where(see, w, 0.0)
            o = w @ vz[h // G]
            odd = ~torch.isfinite(vh).all(1)
            for j in odd.nonzero()[:, 0].tolist():  # to the rows that attend it only
                o[see[:, j]] += w[see[:, j], j, None] * (vh[j] - vz[h // G][j])
            ds = ((x.abs() @ kz[h // G].abs().T).masked_fill(~see, 0.0).amax(1, keepdim=True)
                  * abs(scale) * (d + 3) * u)
            rel = 2 * (2 * ds + 160 * u) + 6 * count * u
            part = {torch.bfloat16: 2.0 ** -18, torch.float16: 2.0 ** -20}.get(q.dtype, 0.0)
            lost = count * 2.0 ** -37 * vz[h // G].abs().max() if q.dtype == torch.float16 else 0.0
            out[rows, h] = torch.where(some[:, None], o, 0.0)
            lse[rows, h] = torch.where(some, torch.logsumexp(s, 1), -math.inf)
            t = ((w @ vz[h // G].abs()) * (rel + part) + lost) * (1 + fi.eps)
            tol[rows, h] = t + fi.eps / 2 * o.abs() + fi.tiny * fi.eps
            big = s.masked_fill(~see, 0.0).abs().amax(1)
            ltol[rows, h] = rel[:, 0] + 8 * u * (big + math.log(total) + 1)
    return out, lse, tol, ltol


class ForkState(U.PageState):
    """fork_pages on Python lists, beside resize."""

    def fork(self, src, new):
        """(source, target, tokens, status)"""
        B = len(new)
        need = lambda n: -(-n // self.page)  # noqa: E731
        refused = lambda s: ([-1] * B, [-1] * B, [0] * B, s)  # noqa: E731
        src = list(range(B)) if src is None else src
        for a, n in zip(src, new):
            if n < 0 or n > 0 and not (0 <= a < B and n <= self.lens[a]):
                return refused(-1)
        old = [row[:need(n)] for row, n in zip(self.table, self.lens)]
        rows = [old[a][:need(n)] if n else [] for a, n in zip(src, new)]
        part = [row[-1] if n % self.page else None for row, n in zip(rows, new)]
        whole = {x for row, p in zip(rows, part) for x in (row if p is None else row[:-1])}
        first = {}
        for b, p in enumerate(part):
            first.setdefault(p, b)
        copies = [b for b, p in enumerate(part) if p is not None and (p in whole or first[p] != b)]
        if len(copies) > len(self.free):
            return refused(len(copies) - len(self.free))
        source, target, tokens = [-1] * B, [-1] * B, [0] * B
        for b in copies:
            source[b], target[b], tokens[b] = part[b], self.free.pop(), new[b] % self.page
            rows[b][-1] = target[b]
        held = {x for row in rows for x in row}
        back = []
        for row in old:
            for x in row:
                if x not in held and x not in back:
                    back.append(x)
        self.free += back[::-1]
        self.table = [row + [-1] * (self.width - len(row)) for row in rows]
        self.lens = list(new)
        return source, target, tokens, 0


# A key of score 0 and value 1 and three of score -3 WEIGHT_SCALE and values that add up to -1 / w, w their
# weight: nothing is left of the sum but what the weights lack. w = 0.5051 loses 2^-17.2 of itself in two
# bf16 parts and 2^-10.6 in one fp16 part. Every other key's score is so low that its weight is 0.
WEIGHT_SCALE = 1865 / 8192
WEIGHT_KEYS = {0: 0.0, 20: -3.0, 77: -3.0, 131: -3.0}


def cancelling(dtype):
    """Of each of WEIGHT_KEYS the value, the output's exact value and what it may be off by.

    u = 2^-24: the weight's exp2 4 u, its exponent (scale, log2 e, their product and the score's) 3 u of
    0.69; at most 10 products that are not zero, of sizes that add up to 2.01, added in fp32: 10 u of
    that; fp16's two parts 2^-20 of the weight, whose products' sizes add up to 1.01."""
    u = 2.0 ** -24
    w = math.exp(-3.0 * WEIGHT_SCALE)
    left, values = -1.0 / w, []
    for _ in range(3):
        values.append(torch.tensor(left, dtype=torch.float64).to(dtype).double().item())
        left -= values[-1]
    total = 1.0 + 3.0 * w
    want = (1.0 + w * sum(values)) / total
    off = 7 * u + 10 * u * 2.01 + (2.0 ** -20 * 1.01 if dtype == torch.float16 else 0.0)
    return dict(zip(WEIGHT_KEYS, [1.0] + values)), want, off / total + torch.finfo(dtype).eps / 2 * abs(want)


def in_parts(w, dtype, parts):
    """A weight (fp32) as the sum of its first 16-bit parts, in float64."""
    left, total = w.double(), torch.zeros_like(w.double())
    for _ in range(parts):
        x = left.float().to(dtype).double()
        total, left = total + x, left - x
    return total


def rows_of(cu, N):
    """Of a call's rows: (first row, offsets, requests) of the requests whose offsets lie among them, and the
    row from which they are behind the last request's (N: none are). Every other row does not fit."""
    if any(b < a for a, b in zip(cu, cu[1:])):
        return 0, [0], [], N
    held = [b for b in range(len(cu) - 1) if cu[b] >= 0 and cu[b + 1] <= N]
    behind = cu[-1] if 0 <= cu[-1] <= N else N
    if not held:
        return 0, [0], [], behind
    first = cu[held[0]]
    return first, [cu[b] - first for b in held] + [cu[held[-1] + 1] - first], held, behind
