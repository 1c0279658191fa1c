"""Drafted tokens and shared pages over the paged key-value cache: cases, plain forms, exact values.

A case is a dict of plain values; its "op" says which operator it takes:

  attend   paged.attend_drafts: the drafted tokens of each request over its pages, each token over
           the context and those of the drafted tokens that its mask lists
  masks    paged.draft_masks: the masks and positions of drafted tokens from their parents
  keep     paged.keep_drafts: the accepted tokens of each request moved together, in every layer
  fork     paged.fork_pages and copy_pages: requests that share another's pages, and their end

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
        # one conversation early on, a small tree of drafted tokens: latency
        dict(name="attend_bf16_4k", op="attend", dtype="bf16", requests=1, hq=14, hkv=2, d=64,
             page=128, lo=4097, hi=4097, nlo=8, nhi=8, idle=0, pad=0, window=0, tree=True,
             token_major=False, mix=1),
        # a layer left dense at the 1M-token cache that the routed decode is timed on
        dict(name="attend_bf16_1m", op="attend", dtype="bf16", requests=1, hq=14, hkv=2, d=64,
             page=128, lo=1048561, hi=1048561, nlo=16, nhi=16, idle=0, pad=0, window=0, tree=True,
             token_major=False, mix=2),
        # a serving batch of mixed lengths and trees, some requests without drafted tokens, padded
        dict(name="attend_fp16_mixed64", op="attend", dtype="fp16", requests=64, hq=32, hkv=8,
             d=128, page=16, lo=64, hi=32768, nlo=1, nhi=32, idle=5, pad=37, window=0, tree=True,
             token_major=True, mix=3),
        # large trees: as much to compute as to read
        dict(name="attend_bf16_trees64", op="attend", dtype="bf16", requests=16, hq=32, hkv=8,
             d=128, page=64, lo=2000, hi=9000, nlo=64, nhi=64, idle=0, pad=0, window=0, tree=True,
             token_major=False, mix=4),
        # the sliding layers of a hybrid model: wide heads, the last 1024 positions
        dict(name="attend_bf16_sliding", op="attend", dtype="bf16", requests=32, hq=8, hkv=4,
             d=256, page=64, lo=300, hi=16384, nlo=2, nhi=24, idle=0, pad=0, window=1024,
             tree=True, token_major=False, mix=5),
        # chains of up to 200 tokens (the next piece of a prompt), full precision, sizes that fill
        # neither tiles nor powers of two
        dict(name="attend_fp32_chain", op="attend", dtype="fp32", requests=6, hq=10, hkv=5, d=80,
             page=48, lo=1, hi=5000, nlo=3, nhi=200, idle=0, pad=5, window=0, tree=False,
             token_major=False, mix=6),
        # the trees of a serving batch
        dict(name="masks_64x64", op="masks", requests=64, most=64, lo=300, hi=16384, nlo=7, nhi=64,
             idle=6, pad=11, mix=7),
        # the largest trees
        dict(name="masks_8x1024", op="masks", requests=8, most=1024, lo=300, hi=16384, nlo=900,
             nhi=1024, idle=0, pad=0, mix=8),
        # a few accepted tokens of every request, in all layers of a small model
        dict(name="keep_bf16_step", op="keep", dtype="bf16", layers=24, requests=64, hkv=2, d=64,
             page=16, lo=100, hi=2000, nlo=16, nhi=64, most=8, idle=7, token_major=False, mix=9),
        # long chains of which about half stays, full precision, an odd page
        dict(name="keep_fp32_long", op="keep", dtype="fp32", layers=8, requests=24, hkv=5, d=80,
             page=48, lo=1, hi=3000, nlo=400, nhi=800, most=400, idle=0, token_major=False,
             mix=10),
        # several answers sampled for each prompt: every page shared, the last one copied
        dict(name="fork_bf16_samples", op="fork", dtype="bf16", layers=24, requests=16, copies=3,
             hkv=2, d=64, page=16, lo=500, hi=8000, whole=True, token_major=False, mix=11),
        # requests that continue another's prefix, large pages: up to a page is copied for each
        dict(name="fork_fp16_prefix", op="fork", dtype="fp16", layers=4, requests=32, copies=3,
             hkv=8, d=128, page=128, lo=1000, hi=6000, whole=False, token_major=True, mix=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "masks", "keep", "fork"])
    mix = rng.randrange(1 << 30)
    if op == "masks":
        most = _log(rng, 1, 1024)
        return dict(op=op, requests=_log(rng, 1, min(256, 8192 // most)), most=most, lo=1,
                    hi=_log(rng, 1, 20000), nlo=rng.randrange(1, most + 1), nhi=most,
                    idle=rng.choice([0, 2, 5]), pad=rng.choice([0, 0, 3, 50]), mix=mix)
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    d = rng.choice([64, 64, 80, 96, 128, 128, 192, 256, 512])
    hkv = rng.choice([1, 2, 3, 4, 5, 8])
    page = rng.choice([16, 16, 32, 48, 64, 128, 256])
    token_major = rng.random() < 0.4
    base = dict(op=op, dtype=dtype, hkv=hkv, d=d, page=page, token_major=token_major, mix=mix)
    if op == "keep":
        nhi = _log(rng, 1, 800)
        layers = _log(rng, 1, 32)
        requests = _log(rng, 1, max(1, min(128, (1 << 26) // (layers * hkv * d * nhi))))
        hi = _log(rng, 1, max(1, (1 << 27) // (requests * layers * hkv * d)))
        return dict(base, layers=layers, requests=requests, lo=_log(rng, 1, hi), hi=hi,
                    nlo=rng.randrange(1, nhi + 1), nhi=nhi, most=rng.randrange(1, nhi + 1),
                    idle=rng.choice([0, 0, 3]))
    if op == "fork":
        copies = rng.choice([1, 1, 2, 3, 7])
        requests = _log(rng, 1, max(1, min(64, (1 << 25) // ((copies + 2) * hkv * page * d))))
        layers = _log(rng, 1, max(1, min(32, (1 << 26) // (requests * (copies + 2) * hkv * page * d))))
        hi = _log(rng, 1, max(1, (1 << 27) // (requests * layers * hkv * d)))
        return dict(base, layers=layers, requests=requests, copies=copies, lo=_log(rng, 1, hi),
                    hi=hi, whole=rng.random() < 0.5)
    G = rng.choice([1, 2, 4, 7, 16])
    requests = _log(rng, 1, 64)
    nhi = _log(rng, 1, max(1, min(256, (1 << 18) // (requests * hkv * G))))
    most = max(2, min((1 << 26) // (requests * hkv * d), (1 << 34) // (requests * nhi * hkv * G * d)))
    hi = _log(rng, 2, most)
    return dict(base, requests=requests, hq=hkv * G, lo=_log(rng, 1, hi), hi=hi,
                nlo=rng.randrange(1, nhi + 1), nhi=nhi, idle=rng.choice([0, 0, 4]),
                pad=rng.choice([0, 0, 1, 20]), window=rng.choice([0, 0, 0, 5, 100, 1024]),
                tree=rng.random() < 0.7)


def shape(case):
    """(tokens of the cache before the drafted ones, drafted tokens) of each request, log-uniform in
    their ranges; every idle-th request has no drafted tokens."""
    rng = random.Random(case["mix"])
    ctx, n = [], []
    for b in range(case["requests"]):
        ctx.append(_log(rng, case["lo"], case["hi"]) - 1)
        x = _log(rng, case["nlo"], case["nhi"])
        every = case["idle"]
        n.append(0 if every and b % every == every - 1 else x)
    return ctx, n


def grown(case, n):
    """The parents of each request's drafted tokens: a token mostly continues the one before it or one
    of a few before that, now and then the context."""
    rng = random.Random(case["mix"] + 1)
    out = []
    for count in n:
        out.append([t - 1 if rng.random() < 0.4 else max(-1, t - 1 - rng.randrange(9))
                    for t in range(count)])
    return out


def ancestors(parents):
    """Of each token the bits of itself and its ancestors, as a whole number."""
    bits = []
    for t, p in enumerate(parents):
        bits.append(1 << t | (bits[p] if p >= 0 else 0))
    return bits


def accepted(case, n):
    """The accepted tokens of each request, ascending: some first ones, then some past the places that
    are written, so that a second pass moves the same tokens again."""
    rng = random.Random(case["mix"] + 2)
    out = []
    for count in n:
        keep = rng.randrange(0, min(case["most"], count) + 1)
        stay = rng.randrange(max(0, 2 * keep - count), keep + 1)
        out.append(list(range(stay)) + sorted(rng.sample(range(keep, count), keep - stay)))
    return out


def forked(case):
    """(lengths before, source rows, lengths after): the requests, then their copies' rows."""
    rng = random.Random(case["mix"])
    R = case["requests"]
    lens = [_log(rng, case["lo"], case["hi"]) for _ in range(R)]
    src = list(range(R)) + [i for i in range(R) for _ in range(case["copies"])]
    after = lens + [lens[i] if case["whole"] else rng.randrange(1, lens[i] + 1) for i in src[R:]]
    return lens + [0] * (len(src) - R), src, after


def work(case):
    op = case["op"]
    if op == "fork":
        before, src, after = forked(case)
        page = case["page"]
        es = 4 if case["dtype"] == "fp32" else 2
        R = case["requests"]
        entries = sum(-(-x // page) for x in before)
        fresh = sum(-(-x // page) for x in after[R:])
        tokens = sum(x % page for x in after[R:])  # at the most: a request's own last page stays
        B = len(src)
        # page ids read, listed for the copies and taken out; lengths; the copied tokens
        return dict(bytes=4 * (2 * entries + 3 * fresh) + 2 * 16 * B
                    + 4 * tokens * case["layers"] * case["hkv"] * case["d"] * es, flops=2 * B)
    ctx, n = shape(case)
    B, N = len(n), sum(n)
    if op == "masks":
        words = -(-case["most"] // 32)
        return dict(bytes=4 * N + (N + case["pad"]) * (4 * words + 4) + 4 * (2 * B + 1), flops=N)
    es = 4 if case["dtype"] == "fp32" else 2
    row = case["hkv"] * case["d"] * es
    if op == "keep":
        moved = sum(sum(i != x for i, x in enumerate(path)) for path in accepted(case, n))
        return dict(bytes=4 * moved * row * case["layers"] + 4 * (3 * B + 1 + N), flops=0)
    parents = grown(case, n) if case["tree"] else [list(range(-1, c - 1)) for c in n]
    pairs = keys = 0
    for c, count, par in zip(ctx, n, parents):
        if count == 0:
            continue
        w = case["window"]
        keys += min(c, w - 1) + count if w else c + count
        for bits in ancestors(par):
            depth = bin(bits).count("1")
            pairs += min(c + depth, w) if w else c + depth
    rows = (N + case["pad"]) * case["hq"]
    words = -(-case["nhi"] // 32) + 1 if case["tree"] else 0
    return dict(bytes=2 * keys * row + 2 * N * case["hq"] * case["d"] * es
                + case["pad"] * case["hq"] * case["d"] * es + 4 * rows + 4 * N * words
                + 4 * (keys // case["page"] + 2 * B + 1),
                flops=4 * pairs * case["hq"] * case["d"])


def _pool(case, layers, pages, g):
    """Pools (layers, pages, hkv, page, d), heads or tokens outermost within a page."""
    hkv, page, d = case["hkv"], case["page"], case["d"]
    form = (page, hkv, d) if case["token_major"] else (hkv, page, d)
    x = torch.empty(layers * pages, *form, device="cuda", dtype=DTYPES[case["dtype"]])
    step = max(1, (1 << 26) // (hkv * page * d))
    for i in range(0, x.shape[0], step):  # in pieces: no fp32 copy of the whole pool
        part = x[i:i + step]
        part.copy_(torch.randn(part.shape, device="cuda", generator=g))
    x = x.view(layers, pages, *form)
    return x.transpose(2, 3) if case["token_major"] else x


def _tables(lens, page, g, spare=1, wider=0):
    """(table, ids): pages scattered over the pool, the spare ones last in ids."""
    need = [-(-x // page) for x in lens]
    width, total = max(1, max(need)) + wider, sum(need)
    ids = torch.randperm(total + spare, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(lens), width), -1, device="cuda", dtype=torch.int32)
    table[torch.arange(width, device="cuda")
          < torch.tensor(need, device="cuda")[:, None]] = ids[:total]
    return table, ids


def _words(bits, words):
    """Whole numbers as rows of 32-bit words, the lowest bits first."""
    raw = b"".join(x.to_bytes(4 * words, "little") for x in bits)
    return torch.frombuffer(bytearray(raw), dtype=torch.int32).view(-1, words) if raw \
        else torch.empty(0, words, dtype=torch.int32)


def _cumulative(n):
    cu = [0]
    for x in n:
        cu.append(cu[-1] + x)
    return cu


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    put = lambda x: torch.tensor(x, device="cuda", dtype=torch.int32)  # noqa: E731
    op = case["op"]
    if op == "fork":
        before, src, after = forked(case)
        page = case["page"]
        spare = len(src) + 3
        table, ids = _tables(before, page, g, spare)
        total = ids.numel() - spare
        free = torch.full((ids.numel(),), -1, device="cuda", dtype=torch.int32)
        free[:spare] = ids[total:]
        return dict(op=op, page=page, table=table, free=free, nfree=put([spare]),
                    lens=put(before), before=put(before), after=put(after), src=put(src),
                    same=put(list(range(len(src)))),
                    kpool=_pool(case, case["layers"], ids.numel(), g),
                    vpool=_pool(case, case["layers"], ids.numel(), g))
    ctx, n = shape(case)
    lens = [c + x for c, x in zip(ctx, n)]
    cu = _cumulative(n)
    if op == "masks":
        # which token continues which, and where, differs from seed to seed
        lens = [x + seed % 997 for x in lens]
        parents = sum(grown(dict(mix=case["mix"] + seed), n), [])
        return dict(op=op, parents=put(parents + [0] * case["pad"]), cu=put(cu), lens=put(lens),
                    most=case["most"])
    page = case["page"]
    table, ids = _tables(lens, page, g)
    if op == "keep":
        paths = accepted(case, n)
        width = max(1, max(map(len, paths)))
        return dict(op=op, page=page, table=table, lens=put(lens), cu=put(cu),
                    path=put([p + [-1] * (width - len(p)) for p in paths]),
                    counts=put([len(p) for p in paths]),
                    kpool=_pool(case, case["layers"], ids.numel(), g),
                    vpool=_pool(case, case["layers"], ids.numel(), g))
    N, hq, d = sum(n) + case["pad"], case["hq"], case["d"]
    # scores of standard deviation 2: a few keys carry a row
    qkv = torch.randn(N, (hq + 2 * case["hkv"]) * d, device="cuda", generator=g) * 2.0
    qkv = qkv.to(DTYPES[case["dtype"]])
    masks = pos = None
    if case["tree"]:
        words = -(-max(1, max(n)) // 32)
        bits = [ancestors(p) for p in grown(case, n)]
        at = [c + bin(x).count("1") - 1 for c, of in zip(ctx, bits) for x in of]
        masks = _words(sum(bits, []) + [0] * case["pad"], words).to("cuda")
        pos = put(at + [0] * case["pad"])
    return dict(op=op, page=page, window=case["window"], table=table, lens=put(lens), cu=put(cu),
                q=qkv[:, :hq * d].view(N, hq, d), masks=masks, pos=pos, most=max(1, max(n)),
                kpool=_pool(case, 1, ids.numel(), g)[0], vpool=_pool(case, 1, ids.numel(), g)[0])


# ---- plain forms ------------------------------------------------------------------------------

def _plain_attend(s):
    q, table, page, window, most = s["q"], s["table"], s["page"], s["window"], s["most"]
    lens, cu = s["lens"].long(), s["cu"].long()
    N, hq, d = q.shape
    B, width = table.shape
    hkv = s["kpool"].shape[1]
    G = hq // hkv
    n = cu[1:] - cu[:-1]
    ctx = lens - n
    t = torch.arange(most, device=q.device)
    live = t < n[:, None]
    row = (cu[:-1, None] + t).clamp(max=N - 1)  # of each request's tokens, as many for all
    pos = ctx[:, None] + t if s["pos"] is None else s["pos"][row].long()
    span = min(window - 1 + most, width * page) if window else width * page
    start = (ctx - window + 1).clamp(min=0) if window else torch.zeros_like(ctx)
    at = start[:, None] + torch.arange(span, device=q.device)
    inside = at < lens[:, None]
    i = (at - ctx[:, None]).clamp(min=0, max=most - 1)  # a key's place among the drafted tokens
    if s["masks"] is None:
        listed_ = i[:, None] <= t[None, :, None]
    else:
        words = s["masks"][row].long()  # (B, most, W)
        word = words.gather(2, (i // 32)[:, None].expand(B, most, span))
        listed_ = (word >> (i % 32)[:, None]) & 1 == 1
    drafted = at >= ctx[:, None]
    mask = inside[:, None] & (~drafted[:, None] | listed_)
    if window:
        keypos = torch.where(drafted, pos.gather(1, i), at)
        mask &= keypos[:, None] > pos[..., None] - window
    mask &= live[..., None]
    pid = table.gather(1, (at // page).clamp(max=width - 1)).long().clamp(min=0)
    k = s["kpool"][pid, :, at % page].float()  # (B, keys, hkv, d)
    qg = q[row].float().view(B, most, hkv, G, d).transpose(1, 2).reshape(B, hkv, most * G, d)
    score = torch.matmul(qg, k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(d)
    del k
    score = score.view(B, hkv, most, G, span)
    score.masked_fill_(~mask[:, None, :, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (score - top).exp()
    del score
    total = p.sum(-1, keepdim=True)
    v = s["vpool"][pid, :, at % page].float().masked_fill(~inside[..., None, None], 0.0)
    out = torch.matmul(p.view(B, hkv, most * G, span), v.transpose(1, 2).contiguous())
    out = out.view(B, hkv, most, G, d) / total
    out = torch.where(total > 0, out, 0.0).transpose(1, 2).reshape(B, most, hq, d)
    lse = (top + total.log())[..., 0].transpose(1, 2).reshape(B, most, hq)
    # back to the tokens in a row: behind the last one zeros
    tok = torch.arange(N, device=q.device)
    b = torch.searchsorted(cu[1:], tok, right=True).clamp(max=B - 1)
    at = (b, (tok - cu[b]).clamp(max=most - 1))
    real = (tok < cu[B])[:, None]
    return (torch.where(real[..., None], out[at], 0.0).to(q.dtype),
            torch.where(real, lse[at], float("-inf")))


def _plain_masks(s):
    parents, cu, lens, most = s["parents"].long(), s["cu"].long(), s["lens"].long(), s["most"]
    N, B = parents.numel(), lens.numel()
    dev = parents.device
    n = cu[1:] - cu[:-1]
    tok = torch.arange(N, device=dev)
    b = torch.searchsorted(cu[1:], tok, right=True).clamp(max=B - 1)
    real = tok < cu[B]
    words = -(-most // 32)
    t = torch.arange(most, device=dev)
    row = (cu[:-1, None] + t).clamp(max=max(N - 1, 0))
    par = torch.where(t < n[:, None], parents[row], -1)
    # reach: a token to itself and its parent, then as far again each time
    reach = (t == par[..., None]).float() + torch.eye(most, device=dev)
    for _ in range(max(1, (most - 1).bit_length())):
        reach = (torch.matmul(reach, reach) > 0).float()
    at = (b, (tok - cu[b]).clamp(max=most - 1))
    bits = torch.zeros(N, words * 32, device=dev, dtype=torch.int64)
    bits[:, :most] = (reach[at] * real[:, None]).long()
    depth = bits.sum(1)
    value = (bits.view(N, words, 32) << torch.arange(32, device=dev)).sum(-1)
    masks = torch.where(value >= 1 << 31, value - (1 << 32), value).to(torch.int32)
    pos = torch.where(real, (lens - n)[b] + depth - 1, 0)
    return masks, pos.to(torch.int32)


def _plain_keep(s):
    lens, cu, path, counts = (s[x].long() for x in ("lens", "cu", "path", "counts"))
    page, table = s["page"], s["table"]
    ctx = lens - (cu[1:] - cu[:-1])
    i = torch.arange(path.shape[1], device=path.device).expand_as(path)
    b = torch.arange(path.shape[0], device=path.device)[:, None].expand_as(path)
    # where nothing moves the first move of the request with the most is made again, or a token to
    # its own place
    live, lead = i < counts[:, None], counts.argmax()
    b = torch.where(live, b, lead)
    src = torch.where(live, path, torch.where(counts[lead] > 0, path[lead, 0], 0)) + ctx[b]
    dst = torch.where(live, i, 0) + ctx[b]
    a, c = table[b, src // page].long(), table[b, dst // page].long()
    for pool in (s["kpool"], s["vpool"]):
        pool[:, c, :, dst % page] = pool[:, a, :, src % page]
    return (ctx + counts).to(torch.int32)


def _plain_fork(s, src, new):
    lens, table, free, nfree, page = s["lens"], s["table"], s["free"], s["nfree"], s["page"]
    B, width = table.shape
    P = free.numel()
    dev = table.device
    old, src, new = lens.long(), src.long(), new.long()
    me = torch.arange(B, device=dev)
    ok = ((src >= 0) & (src < B)).all()
    src = src.clamp(0, B - 1)
    ok = ok & ((new >= 0) & (new <= old[src])).all()
    have, full = (old + page - 1) // page, new // page
    part = new % page > 0
    col = torch.arange(width, device=dev)
    held = col < have[:, None]
    source = table[src].long()
    whole = torch.zeros(P + 1, device=dev, dtype=torch.bool)  # the last place takes what is not meant
    whole[torch.where(col < full[:, None], source, P).flatten()] = True
    whole[P] = False
    last = source.gather(1, full.clamp(max=width - 1)[:, None])[:, 0]
    last = torch.where(part, last, P)
    first = torch.full((P + 1,), B, device=dev).scatter_reduce_(0, last, me, "amin")
    copy = part & (whole[last] | (first[last] != me))
    stays = whole | (first < B)
    ids = torch.where(held, table.long(), P)
    holder = torch.full((P + 1,), B, device=dev).scatter_reduce_(
        0, ids.flatten(), me[:, None].expand(B, width).flatten(), "amin")
    gone = held & ~stays[ids] & (holder[ids] == me[:, None])
    taken, given = copy.sum(), gone.sum()
    lack = (taken - nfree).clamp(min=0)[0]
    status = torch.where(~ok, -1, lack)
    ok = status == 0
    copy, gone = copy & ok, gone & ok
    nth = torch.cumsum(copy.long(), 0) - 1
    fresh = free[(nfree.long() - 1 - nth).clamp(0, P - 1)].long()
    left = nfree.long() - copy.sum() + gone.sum()
    order = (torch.cumsum(gone.flatten().long(), 0) - 1).view(B, width)
    room = torch.cat([free, free.new_zeros(1)])
    room[torch.where(gone, left - 1 - order, P).flatten()] = table.flatten()
    need = full + part.long()
    rows = torch.where(col < need[:, None], source, -1)
    rows = torch.where((col == full[:, None]) & copy[:, None], fresh[:, None], rows)
    i32 = torch.int32
    table.copy_(torch.where(ok, rows, table.long()).to(i32))
    free.copy_(room[:P])
    nfree.copy_(left.to(i32))
    lens.copy_(torch.where(ok, new, old).to(i32))
    return (torch.where(copy, last, -1).to(i32), torch.where(copy, fresh, -1).to(i32),
            torch.where(copy, new % page, 0).to(i32), status.to(i32).view(1))


def _plain_copy(s, source, target, tokens):
    page = s["page"]
    # rows without a copy make that of the row with the most tokens again, or a page's into itself
    lead = tokens.argmax()
    row = torch.where(source >= 0, torch.arange(source.numel(), device=source.device), lead)
    a, c = source.long().clamp(min=0)[row], target.long().clamp(min=0)[row]
    slot = torch.arange(page, device=source.device)
    slot = torch.where(slot < tokens[row][:, None], slot, 0)
    for pool in (s["kpool"], s["vpool"]):
        pool[:, c[:, None], :, slot] = pool[:, a[:, None], :, slot]


def run(state):
    s = state
    if own:
        from ssa_amd import paged
    if s["op"] == "masks":
        if own:
            d = paged.draft_masks(s["parents"], s["cu"], s["lens"], s["most"])
            return dict(masks=d.masks, pos=d.pos)
        masks, pos = _plain_masks(s)
        return dict(masks=masks, pos=pos)
    if s["op"] == "keep":
        if own:
            lens = paged.keep_drafts(s["kpool"], s["vpool"], s["table"], s["lens"], s["cu"],
                                     s["path"], s["counts"])
        else:
            lens = _plain_keep(s)
        return dict(lens=lens, kpool=s["kpool"], vpool=s["vpool"])
    if s["op"] == "fork":
        # the copies are made, and at their end give back what is theirs alone
        if own:
            rest = (s["lens"], s["table"], s["free"], s["nfree"], s["page"])
            f = paged.fork_pages(s["src"], s["after"], *rest)
            paged.copy_pages(s["kpool"], s["vpool"], f.source, f.target, f.tokens)
            f = tuple(f)
            back = paged.fork_pages(s["same"], s["before"], *rest).status
        else:
            f = _plain_fork(s, s["src"], s["after"])
            _plain_copy(s, *f[:3])
            back = _plain_fork(s, s["same"], s["before"])[3]
        return dict(source=f[0], target=f[1], tokens=f[2], status=f[3], back=back,
                    lens=s["lens"], table=s["table"], free=s["free"], nfree=s["nfree"],
                    kpool=s["kpool"], vpool=s["vpool"])
    if own:
        drafts = None if s["masks"] is None else paged.Drafts(s["masks"], s["pos"])
        out, lse = paged.attend_drafts(s["q"], s["kpool"], s["vpool"], s["table"], s["lens"],
                                       s["cu"], drafts, window=s["window"], return_lse=True)
    else:
        out, lse = _plain_attend(s)
    return dict(out=out, lse=lse)


# ---- exact values -----------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    put = lambda x: torch.tensor(x, device="cuda", dtype=torch.int32)  # noqa: E731
    if op == "fork":
        return _exact_fork(case, s)
    ctx, n = shape(case)
    if op == "masks":
        parents, words = s["parents"].tolist(), -(-case["most"] // 32)
        cu = _cumulative(n)
        bits, pos = [], []
        for b, count in enumerate(n):
            for t in range(count):
                x, m, depth = t, 0, 0
                while x >= 0:  # token by token up to the context
                    m, depth, x = m | 1 << x, depth + 1, parents[cu[b] + x]
                bits.append(m)
                pos.append(ctx[b] + seed % 997 + depth - 1)
        bits, pos = bits + [0] * case["pad"], pos + [0] * case["pad"]
        return dict(masks=_words(bits, words).to("cuda"), pos=put(pos))
    page = s["page"]
    if op == "keep":
        k, v = s["kpool"].double(), s["vpool"].double()
        table, lens = s["table"].tolist(), []
        for b, path in enumerate(accepted(case, n)):
            where = lambda j: (table[b][j // page], j % page)  # noqa: E731
            a = [where(ctx[b] + x) for x in path]
            c = [where(ctx[b] + i) for i in range(len(path))]
            lens.append(ctx[b] + len(path))
            if path:
                (ap, ao), (cp, co) = (map(list, zip(*z)) for z in (a, c))
                for new, pool in ((k, s["kpool"]), (v, s["vpool"])):
                    for layer in range(case["layers"]):
                        new[layer][cp, :, co] = pool[layer][ap, :, ao].double()
        return dict(lens=put(lens), kpool=k, vpool=v)
    N, hq, d = s["q"].shape
    hkv, window = case["hkv"], case["window"]
    G = hq // hkv
    out = torch.zeros(N, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((N, hq), float("-inf"), dtype=torch.float64, device="cuda")
    table, cu = s["table"].tolist(), _cumulative(n)
    par = grown(case, n) if case["tree"] else [list(range(-1, c - 1)) for c in n]
    for b, count in enumerate(n):
        if count == 0:
            continue
        c, total = ctx[b], ctx[b] + count
        bits = ancestors(par[b])
        at = torch.tensor([c + bin(x).count("1") - 1 for x in bits], device="cuda")
        first = max(0, c - window + 1) if window else 0
        seen = torch.tensor([[x >> i & 1 for i in range(count)] for x in bits], device="cuda") == 1
        mask = torch.cat([torch.ones(count, c - first, device="cuda", dtype=torch.bool), seen], 1)
        if window:
            keypos = torch.cat([torch.arange(first, c, device="cuda"), at])
            mask &= keypos > at[:, None] - window
        used = torch.tensor(table[b][first // page:(total - 1) // page + 1], device="cuda")
        skip = first % page
        rows = slice(cu[b], cu[b] + count)
        for h in range(hkv):
            k = s["kpool"][used, h].reshape(-1, d)[skip:skip + total - first].double()
            v = s["vpool"][used, h].reshape(-1, d)[skip:skip + total - first].double()
            for j in range(h * G, (h + 1) * G):
                x = (s["q"][rows, j].double() @ k.T * d ** -0.5).masked_fill(~mask, float("-inf"))
                lse[rows, j] = torch.logsumexp(x, -1)
                out[rows, j] = torch.softmax(x, -1) @ v
    return dict(out=out, lse=lse)


def _exact_fork(case, s):
    """Row by row in Python lists; forked and ended, the state is what it was."""
    page = case["page"]
    _, src, after = forked(case)
    table, stack = s["table"].tolist(), s["free"].tolist()[:int(s["nfree"])]
    k, v = s["kpool"].double(), s["vpool"].double()
    keeper, source, target, tokens = set(), [], [], []
    whole = {table[a][e] for a, x in zip(src, after) for e in range(x // page)}
    for a, x in zip(src, after):
        part = table[a][x // page] if x % page else None
        if part is None or part not in whole and part not in keeper:
            keeper.add(part)
            source.append(-1)
            target.append(-1)
            tokens.append(0)
            continue
        fresh = stack.pop()
        for pool in (k, v):
            pool[:, fresh, :, :x % page] = pool[:, part, :, :x % page]
        source.append(part)
        target.append(fresh)
        tokens.append(x % page)
    put = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(source=put(source), target=put(target), tokens=put(tokens), status=put([0]),
                back=put([0]), lens=s["lens"], table=s["table"], free=s["free"], nfree=s["nfree"],
                kpool=k, vpool=v)
