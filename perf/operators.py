"""The paged key-value cache's operators as they are measured: cases, plain forms, exact values.

A case is a dict of plain values; its "op" says which operator it takes:

  attend   paged.attend_pages: one new token of each request over its pages of the cache
  resize   paged.resize_pages: block tables and slot maps from the requests' lengths
  append   paged.append_pages: keys and values of new tokens into their slots

With `own` false a pass computes the plain form in elementary torch operations.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one request at the 1M-token cache that the routed decode is timed on: a layer left dense
        dict(name="attend_bf16_1m", op="attend", dtype="bf16", requests=1, hq=14, hkv=2, d=64,
             page=128, lo=1048577, hi=1048577, idle=0, window=0, new=True, token_major=False,
             mix=1),
        # the same layer early in one conversation: latency
        dict(name="attend_bf16_4k", op="attend", dtype="bf16", requests=1, hq=14, hkv=2, d=64,
             page=128, lo=4097, hi=4097, idle=0, window=0, new=True, token_major=False, mix=2),
        # a serving batch of mixed lengths, a fifth of the rows idle, small pages, tokens outermost
        dict(name="attend_fp16_mixed64", op="attend", dtype="fp16", requests=64, hq=32, hkv=8,
             d=128, page=16, lo=64, hi=32768, idle=5, window=0, new=True, token_major=True, mix=3),
        # the sliding layers of a hybrid model: wide heads, the last 1024 keys of long requests
        dict(name="attend_bf16_sliding", op="attend", dtype="bf16", requests=32, hq=8, hkv=4,
             d=256, page=64, lo=300, hi=16384, idle=0, window=1024, new=False, token_major=False,
             mix=4),
        # full precision, a key head for every query head
        dict(name="attend_fp32_8", op="attend", dtype="fp32", requests=8, hq=12, hkv=12, d=64,
             page=32, lo=1000, hi=30000, idle=0, window=0, new=False, token_major=False, mix=5),
        # many query heads on one key head, a large batch at ordinary lengths
        dict(name="attend_bf16_shared", op="attend", dtype="bf16", requests=128, hq=20, hkv=1,
             d=128, page=256, lo=2000, hi=9000, idle=0, window=0, new=False, token_major=False,
             mix=6),
        # head dim 80 and pages of 48 tokens: sizes that fill neither tiles nor powers of two
        dict(name="attend_fp16_d80", op="attend", dtype="fp16", requests=24, hq=10, hkv=5, d=80,
             page=48, lo=1, hi=5000, idle=7, window=0, new=True, token_major=False, mix=7),
        # a decode step of 256 requests: one token each, taken back
        dict(name="resize_step256", op="resize", requests=256, page=16, lo=1, hi=20000, grow_lo=1,
             grow_hi=1, idle=9, mix=8),
        # prompts admitted and, at the end, released: about 200K tokens
        dict(name="resize_prompts", op="resize", requests=64, page=16, lo=0, hi=0, grow_lo=500,
             grow_hi=8000, idle=0, mix=9),
        # a decode step's keys and values, a row each, as views of a fused projection
        dict(name="append_bf16_step", op="append", dtype="bf16", tokens=256, pad=19, run=1, hq=32,
             hkv=8, d=128, page=16, token_major=True, mix=10),
        # a prompt of 64K tokens
        dict(name="append_bf16_prompt", op="append", dtype="bf16", tokens=65536, pad=100,
             run=65000, hq=14, hkv=2, d=64, page=128, token_major=False, mix=11),
        # chunks of several prompts, full precision, an odd page
        dict(name="append_fp32_chunks", op="append", dtype="fp32", tokens=8191, pad=7, run=1000,
             hq=5, hkv=5, d=80, page=48, token_major=False, mix=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "resize", "append"])
    mix = rng.randrange(1 << 30)
    if op == "resize":
        requests = _log(rng, 1, 1024)
        lo = rng.randrange(0, 50)
        top = _log(rng, 2, min(8000, 400000 // requests)) if rng.random() < 0.5 else 1
        return dict(op=op, requests=requests, page=rng.choice([16, 32, 48, 64, 128, 256]), lo=lo,
                    hi=lo + _log(rng, 1, 20000), grow_lo=rng.randrange(1, top + 1),
                    grow_hi=top, idle=rng.choice([0, 2, 3, 7]),
                    mix=mix)
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    d = rng.choice([64, 64, 80, 96, 128, 128, 192, 256, 512])
    hkv = rng.choice([1, 2, 3, 4, 5, 8])
    page = rng.choice([16, 16, 32, 48, 64, 128, 256])
    token_major = rng.random() < 0.4
    if op == "append":
        tokens = _log(rng, 1, max(2, (1 << 23) // (hkv * d)))
        return dict(op=op, dtype=dtype, tokens=tokens, pad=rng.randrange(0, max(1, tokens // 3)),
                    run=_log(rng, 1, tokens + 1), hq=hkv * rng.choice([1, 2, 7]), hkv=hkv, d=d,
                    page=page, token_major=token_major, mix=mix)
    requests = _log(rng, 1, 128)
    most = max(2, (1 << 26) // (requests * hkv * d))
    hi = _log(rng, 2, most)
    return dict(op=op, dtype=dtype, requests=requests, hq=hkv * rng.choice([1, 2, 4, 7, 16, 20]),
                hkv=hkv, d=d, page=page, lo=_log(rng, 1, hi), hi=hi, idle=rng.choice([0, 0, 3, 6]),
                window=rng.choice([0, 0, 0, 1, 100, 1024]), new=rng.random() < 0.5,
                token_major=token_major, mix=mix)


def lengths(case, lo, hi, salt):
    """The requests' lengths, log-uniform in lo..hi; every idle-th row has none."""
    rng = random.Random(case["mix"] * 7 + salt)
    every = case["idle"]
    out = []
    for b in range(case["requests"]):
        x = _log(rng, max(lo, 1), max(hi, lo, 1)) if hi > 0 else 0
        out.append(0 if every and b % every == every - 1 else x)
    return out


def attended(case):
    """Keys each request attends."""
    lens = lengths(case, case["lo"], case["hi"], 0)
    return [min(n, case["window"]) if case["window"] else n for n in lens]


def grown(case):
    """(before, after) of a resize: idle requests stay as they are."""
    before = lengths(case, case["lo"], case["hi"], 0)
    add = lengths(case, case["grow_lo"], case["grow_hi"], 1)
    return before, [a + b for a, b in zip(before, add)]


def work(case):
    if case["op"] == "resize":
        before, after = grown(case)
        page, B = case["page"], case["requests"]
        taken = sum(-(-b // page) - -(-a // page) for a, b in zip(before, after))
        new = sum(after) - sum(before)
        # lengths read and written twice; a page's id moved to the table and back; slot and position
        return dict(bytes=2 * 12 * B + 16 * taken + 12 * new + 4 * (B + 1), flops=2 * B)
    es = 4 if case["dtype"] == "fp32" else 2
    row = case["hkv"] * case["d"] * es
    if case["op"] == "append":
        return dict(bytes=4 * (case["tokens"] - case["pad"]) * row + 8 * case["tokens"],
                    flops=0)
    keys, B = attended(case), case["requests"]
    entries = sum(-(-n // case["page"]) for n in keys)
    new = 2 * B * row if case["new"] else 0
    return dict(bytes=2 * sum(keys) * row + 2 * B * case["hq"] * case["d"] * es
                + 4 * B * case["hq"] + 4 * entries + 4 * B + new,
                flops=4 * sum(keys) * case["hq"] * case["d"])


def _pool(case, pages, g):
    """A pool of pages (pages, hkv, page, d): heads or tokens outermost within a page."""
    hkv, page, d = case["hkv"], case["page"], case["d"]
    shape = (pages, page, hkv, d) if case["token_major"] else (pages, hkv, page, d)
    x = torch.empty(shape, device="cuda", dtype=DTYPES[case["dtype"]])
    step = max(1, (1 << 26) // (hkv * page * d))
    for i in range(0, pages, step):  # in pieces: no fp32 copy of the whole pool
        part = x[i:i + step]
        part.copy_(torch.randn(part.shape, device="cuda", generator=g))
    return x.transpose(1, 2) if case["token_major"] else x


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    page = case["page"]
    i32 = dict(device="cuda", dtype=torch.int32)
    if case["op"] == "resize":
        before, after = grown(case)
        B, width = case["requests"], max(1, max(-(-n // page) for n in after)) + 1
        have = [-(-n // page) for n in before]
        pages = sum(-(-n // page) for n in after) + 37
        ids = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        table = torch.full((B, width), -1, **i32)
        col = torch.arange(width, device="cuda")
        table[col < torch.tensor(have, device="cuda")[:, None]] = ids[:sum(have)]
        free = torch.full((pages,), -1, **i32)
        free[:pages - sum(have)] = ids[sum(have):]
        return dict(op="resize", page=page, tokens=sum(after) - sum(before) + 5, table=table,
                    free=free, nfree=torch.tensor([pages - sum(have)], **i32),
                    lens=torch.tensor(before, **i32), before=torch.tensor(before, **i32),
                    after=torch.tensor(after, **i32))
    dtype = DTYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "append":
        live = case["tokens"] - case["pad"]
        run = min(case["run"], live)
        rng = random.Random(seed)
        per = -(-(run + page - 1) // page)  # pages of one run, from any offset in its first
        runs = -(-live // run)
        ids = torch.randperm(runs * per + 3, device="cuda", generator=g)[:runs * per]
        start = torch.tensor([rng.randrange(page) for _ in range(runs)], device="cuda")
        at = start[:, None] + torch.arange(run, device="cuda")
        slots = ids.view(runs, per).gather(1, at // page) * page + at % page
        slots = torch.cat([slots.flatten()[:live],
                           torch.full((case["pad"],), -1, device="cuda", dtype=torch.int64)])
        qkv = torch.randn(case["tokens"], (hq + 2 * hkv) * d, device="cuda",
                          generator=g).to(dtype)
        k = qkv[:, hq * d:(hq + hkv) * d].view(-1, hkv, d)
        v = qkv[:, (hq + hkv) * d:].view(-1, hkv, d)
        return dict(op="append", page=page, k=k, v=v, slots=slots,
                    kpool=_pool(case, runs * per + 3, g), vpool=_pool(case, runs * per + 3, g))
    lens = lengths(case, case["lo"], case["hi"], 0)
    need = [-(-n // page) for n in lens]
    B, width, total = case["requests"], max(1, max(need)), sum(need)
    ids = torch.randperm(total + 1, device="cuda", generator=g).to(torch.int32)
    table = torch.full((B, width), -1, **i32)
    table[torch.arange(width, device="cuda")
          < torch.tensor(need, device="cuda")[:, None]] = ids[:total]
    qkv = torch.randn(B, (hq + 2 * hkv) * d, device="cuda", generator=g)
    qkv[:, :hq * d] *= 2.0  # scores of standard deviation 2: a few keys carry a row
    qkv = qkv.to(dtype)
    new = case["new"]
    return dict(op="attend", page=page, window=case["window"], table=table,
                q=qkv[:, :hq * d].view(B, hq, d),
                k_new=qkv[:, hq * d:(hq + hkv) * d].view(B, hkv, d) if new else None,
                v_new=qkv[:, (hq + hkv) * d:].view(B, hkv, d) if new else None,
                lens=torch.tensor(lens, **i32), kpool=_pool(case, total + 1, g),
                vpool=_pool(case, total + 1, g))


# ---- plain forms ------------------------------------------------------------------------------

def _plain_resize(s, new, tokens):
    lens, table, free, nfree, page = s["lens"], s["table"], s["free"], s["nfree"], s["page"]
    B, width = table.shape
    P = free.numel()
    old, new = lens.long(), new.long()
    have, need = (old + page - 1) // page, (new + page - 1) // page
    take, give = (need - have).clamp(min=0), (have - need).clamp(min=0)
    add = (new - old).clamp(min=0)
    fits = ((old >= 0) & (new >= 0) & (old <= width * page) & (new <= width * page)).all()
    lack = (take.sum() - nfree).clamp(min=0)[0]
    over = add.sum() > tokens
    status = torch.where(~fits, -1, torch.where(over, -2, lack))
    ok = status == 0
    take, give, add = take * ok, give * ok, add * ok
    col = torch.arange(width, device=table.device)
    taking = (col >= have[:, None]) & (col < (have + take)[:, None])
    giving = (col >= (have - give)[:, None]) & (col < have[:, None])
    nth = lambda m: (torch.cumsum(m.flatten().long(), 0) - 1).view(B, width)  # noqa: E731
    top = nfree.long() - take.sum()
    left = top + give.sum()
    back = torch.where(giving, left - 1 - nth(giving), P)
    room = torch.cat([free, free.new_zeros(1)])  # the last place takes what is not given back
    fresh = free[(nfree.long() - 1 - nth(taking)).clamp(0, P - 1)]
    room[back.flatten()] = table.flatten()
    table.copy_(torch.where(giving, -1, torch.where(taking, fresh, table)))
    free.copy_(room[:P])
    nfree.copy_(left)
    lens.copy_(torch.where(ok, new, old))
    cu = torch.cat([add.new_zeros(1), torch.cumsum(add, 0)])
    t = torch.arange(tokens, device=table.device)
    b = torch.searchsorted(cu[1:], t, right=True).clamp(max=B - 1)
    pos = old[b] + t - cu[b]
    live = t < cu[B]
    pos = torch.where(live, pos, 0)
    slots = table[b, pos // page].long() * page + pos % page
    i32 = torch.int32
    return (torch.where(live, slots, -1), pos.to(i32), cu.to(i32), status.to(i32).view(1))


def _plain_append(s):
    slots, page = s["slots"], s["page"]
    keep = slots >= 0
    # padded rows write the first row's values to the first row's slot again
    at = torch.where(keep, slots, slots[0])
    row = torch.where(keep, torch.arange(slots.numel(), device=slots.device), 0)
    for pool, x in ((s["kpool"], s["k"]), (s["vpool"], s["v"])):
        pool[at // page, :, at % page] = x[row]
    return s["kpool"], s["vpool"]


def _plain_attend(s):
    q, table, page = s["q"], s["table"], s["page"]
    lens = s["lens"].long()
    B, hq, d = q.shape
    hkv, width = s["kpool"].shape[1], table.shape[1]
    if s["k_new"] is not None:
        # rows without a token write nothing: they repeat the longest row's write
        lead = lens.argmax()
        row = torch.where(lens > 0, torch.arange(B, device=q.device), lead)
        last = lens[row] - 1
        at = table[row, last // page].long()
        s["kpool"][at, :, last % page] = s["k_new"][row]
        s["vpool"][at, :, last % page] = s["v_new"][row]
    n = width * page
    span = min(s["window"], n) if s["window"] else n
    start = (lens - span).clamp(min=0) if s["window"] else torch.zeros_like(lens)
    pos = start[:, None] + torch.arange(span, device=q.device)
    pid = table.gather(1, (pos // page).clamp(max=width - 1)).long().clamp(min=0)
    mask = pos < lens[:, None]
    k = s["kpool"][pid, :, pos % page].float()  # (B, keys, hkv, d)
    qg = q.float().view(B, hkv, hq // hkv, d)
    score = torch.matmul(qg, k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(d)
    del k
    score = score.masked_fill(~mask[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (score - top).exp()
    del score
    total = p.sum(-1, keepdim=True)
    v = s["vpool"][pid, :, pos % page].float().masked_fill(~mask[..., None, None], 0.0)
    out = torch.matmul(p, v.transpose(1, 2).contiguous())
    lse = (top + total.log()).view(B, hq)
    empty = (lens == 0)[:, None, None, None]
    out = torch.where(empty, 0.0, out / total).to(q.dtype).view(B, hq, d)
    return out, lse


def run(state):
    s = state
    if s["op"] == "resize":
        # a step's tokens get their pages and slots, and the requests go back to where they were
        if own:
            from ssa_amd import paged
            args = (s["table"], s["free"], s["nfree"], s["page"])
            r = paged.resize_pages(s["lens"], s["after"], *args, s["tokens"])
            b = paged.resize_pages(s["lens"], s["before"], *args, 0)
            got, back = (r.slots, r.pos, r.cu, r.status), b.status
        else:
            got = _plain_resize(s, s["after"], s["tokens"])
            back = _plain_resize(s, s["before"], 0)[3]
        return dict(slots=got[0], pos=got[1], cu=got[2], status=got[3], back=back, lens=s["lens"],
                    table=s["table"], free=s["free"], nfree=s["nfree"])
    if s["op"] == "append":
        if own:
            from ssa_amd import paged
            paged.append_pages(s["k"], s["v"], s["kpool"], s["vpool"], s["slots"])
        else:
            _plain_append(s)
        return dict(kpool=s["kpool"], vpool=s["vpool"])
    if own:
        from ssa_amd import paged
        out, lse = paged.attend_pages(s["q"], s["kpool"], s["vpool"], s["table"], s["lens"],
                                      k_new=s["k_new"], v_new=s["v_new"], window=s["window"],
                                      return_lse=True)
    else:
        out, lse = _plain_attend(s)
    if s["k_new"] is None:
        return dict(out=out, lse=lse)
    return dict(out=out, lse=lse, kpool=s["kpool"], vpool=s["vpool"])


# ---- exact values -----------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    page = s["page"]
    if s["op"] == "resize":
        return _exact_resize(case, s)
    if s["op"] == "append":
        k, v = s["kpool"].double(), s["vpool"].double()
        order = [(t, x) for t, x in enumerate(s["slots"].tolist()) if x >= 0]
        rows = torch.tensor([t for t, _ in order], device="cuda")
        pid = torch.tensor([x // page for _, x in order], device="cuda")
        off = torch.tensor([x % page for _, x in order], device="cuda")
        for h in range(case["hkv"]):
            k[pid, h, off] = s["k"][rows, h].double()
            v[pid, h, off] = s["v"][rows, h].double()
        return dict(kpool=k, vpool=v)
    B, hq, d = s["q"].shape
    hkv = case["hkv"]
    G = hq // hkv
    out = torch.zeros(B, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((B, hq), float("-inf"), dtype=torch.float64, device="cuda")
    table = s["table"].tolist()
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        first = max(0, n - case["window"]) if case["window"] else 0
        if s["k_new"] is not None:
            at = table[b][(n - 1) // page]
            s["kpool"][at, :, (n - 1) % page] = s["k_new"][b]
            s["vpool"][at, :, (n - 1) % page] = s["v_new"][b]
        used = torch.tensor(table[b][first // page:(n - 1) // page + 1], device="cuda")
        skip = first % page
        for h in range(hkv):
            k = s["kpool"][used, h].reshape(-1, d)[skip:skip + n - first].double()
            v = s["vpool"][used, h].reshape(-1, d)[skip:skip + n - first].double()
            x = s["q"][b, h * G:(h + 1) * G].double() @ k.T * d ** -0.5
            lse[b, h * G:(h + 1) * G] = torch.logsumexp(x, -1)
            out[b, h * G:(h + 1) * G] = torch.softmax(x, -1) @ v
    if s["k_new"] is None:
        return dict(out=out, lse=lse)
    return dict(out=out, lse=lse, kpool=s["kpool"].double(), vpool=s["vpool"].double())


def _exact_resize(case, s):
    """Request by request, page by page; taken and given back, the state is what it was."""
    page, before, after = case["page"], *grown(case)
    table, stack = s["table"].tolist(), s["free"].tolist()[:int(s["nfree"])]
    slots, pos, cu = [], [], [0]
    for b, (old, new) in enumerate(zip(before, after)):
        for j in range(old, new):
            if j % page == 0:
                table[b][j // page] = stack.pop()
            slots.append(table[b][j // page] * page + j % page)
            pos.append(j)
        cu.append(len(slots))
    spare = s["tokens"] - len(slots)
    put = lambda x, t: torch.tensor(x, dtype=t, device="cuda")  # noqa: E731
    return dict(slots=put(slots + [-1] * spare, torch.int64),
                pos=put(pos + [0] * spare, torch.int32), cu=put(cu, torch.int32),
                status=put([0], torch.int32), back=put([0], torch.int32), lens=s["lens"],
                table=s["table"], free=s["free"], nfree=s["nfree"])
