"""Drafted tokens and shared pages over the paged cache on the GPU: masks, positions, tables and moved rows
equal to plain lists, attention within the bounds of its arithmetic (drafts_util.attend)."""
import math
import random

import pytest
import torch

from ssa_amd import _lib
from ssa_amd import paged as P
from tests import drafts_util as D
from tests import paged_util as U

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def int32(x, dev):
    return torch.tensor(x, device=dev, dtype=torch.int32)


def offsets(n):
    cu = [0]
    for x in n:
        cu.append(cu[-1] + x)
    return cu


# ---- masks and positions ------------------------------------------------------------------------

@pytest.mark.parametrize("most", [1, 2, 31, 32, 33, 64, 65, 200, 256, 257, 1000, 1024])
def test_masks_equal_sets(cuda, most):
    rng = random.Random(most)
    n = [most, 0, 1, max(1, most // 2), most, max(1, most - 1)]
    lens = [most, 5, 1, 4000, 70000, 2 ** 31 - 2000]
    parents = []
    for b, count in enumerate(n):
        parents += [list(range(-1, count - 1)),  # a chain
                    D.random_parents(rng, count), [-1] * count][b % 3]
    N = len(parents) + 7
    words = -(-most // 32)
    print(most, N, flush=True)
    d = P.draft_masks(int32(parents + [3] * 7, cuda), int32(offsets(n), cuda), int32(lens, cuda),
                      most)
    masks, pos = D.masks_and_pos(parents, n, lens, words, N)
    assert d.masks.tolist() == masks and d.pos.tolist() == pos


def test_masks_of_parents_that_do_not_fit(cuda):
    parents = [-1, 0, 2, 2, 1, -2, 5, 3, 4, 2 ** 31 - 1, -2 ** 31, 0]
    n, lens = [12, 3, 5, 40], [20, 2, 5, 100]  # 3 of a length of 2, 40 in a mask of 32 bits
    parents += [-1, 0, 1] + [-1, 0, 1, 2, 3] + list(range(-1, 39))
    d = P.draft_masks(int32(parents, cuda), int32(offsets(n), cuda), int32(lens, cuda), 20)
    masks, pos = D.masks_and_pos(parents, n, lens, 1, len(parents))
    assert d.masks.tolist() == masks and d.pos.tolist() == pos
    assert pos[:12] == [8, 9, -1, -1, 10, -1, -1, -1, 11, -1, -1, 9] and pos[12:15] == [-1] * 3


def test_masks_of_offsets_that_do_not_fit(cuda):
    """Offsets that descend, are negative or pass N make a request none; nothing is read through them."""
    parents = int32([-1, 0, 1, 2], cuda)
    for cu in ([0, 5, 4], [0, -1, 4], [2 ** 31 - 1, 0, 4], [-2 ** 31, 2 ** 31 - 1, 4]):
        d = P.draft_masks(parents, int32(cu, cuda), int32([50, 50], cuda), 8)
        torch.cuda.synchronize()
        assert d.masks.shape == (4, 1) and d.pos.shape == (4,)
    assert P.draft_masks(parents[:0], int32([0], cuda), parents[:0], 8).masks.shape == (0, 1)
    assert P.draft_masks(parents, int32([0], cuda), parents[:0], 8).pos.tolist() == [0] * 4


# ---- attention ----------------------------------------------------------------------------------

def make(dev, dtype, ctx, n, hq, hkv, d, page, token_major=False, seed=0, spread=1.0, extra=0,
         pad=0):
    """(q, cache, cu) with the requests' pages scattered over the pool; unused slots hold NaN."""
    g = torch.Generator(device=dev).manual_seed(seed)
    lens = [c + x for c, x in zip(ctx, n)]
    need = [-(-x // page) for x in lens]
    pages, width = sum(need) + 2, max(max(need), 1) + extra
    cache = P.PagedCache(len(lens), width * page, pages, hkv, d, page=page, dtype=dtype,
                         device=dev, token_major=token_major)
    ids = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    cache.k.fill_(math.nan)
    cache.v.fill_(math.nan)
    at = 0
    for b, total in enumerate(lens):
        cache.table[b, :need[b]] = ids[at:at + need[b]]
        for e in range(need[b]):
            m = min(page, total - e * page)
            pid = int(ids[at + e])
            cache.k[0, pid, :, :m] = torch.randn(hkv, m, d, device=dev, generator=g).to(dtype)
            cache.v[0, pid, :, :m] = torch.randn(hkv, m, d, device=dev, generator=g).to(dtype)
        at += need[b]
    cache.lens.copy_(int32(lens, dev))
    q = (torch.randn(sum(n) + pad, hq, d, device=dev, generator=g) * spread).to(dtype)
    return q, cache, int32(offsets(n), dev)


def check(cache, q, cu, drafts=None, scale=None, window=0, **kw):
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    out, lse = cache.attend_drafts(0, q, cu, drafts, scale=scale, window=window, return_lse=True,
                                   **kw)
    torch.cuda.synchronize()
    masks, pos = (None, None) if drafts is None else drafts
    want, wlse, tol, ltol = D.attend(q, cache.k[0], cache.v[0], cache.table, cache.lens, cu, scale,
                                     window, masks, pos)
    U.close(out, want, tol)
    U.close(lse, wlse, ltol)
    return out, lse


def tree(cache, cu, n, seed=0):
    rng = random.Random(seed)
    parents = sum((D.random_parents(rng, x) for x in n), [])
    return P.draft_masks(int32(parents, cu.device), cu, cache.lens, max(1, max(n)))


CTX = [0, 0, 1, 15, 16, 17, 31, 32, 33, 63, 100, 127, 128, 129, 257, 500, 1000, 7, 0, 90]
DRAFTED = [1, 33, 1, 2, 16, 17, 5, 0, 31, 1, 28, 1, 8, 3, 15, 20, 9, 0, 0, 64]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page,token_major", [
    (14, 2, 64, 128, False), (4, 4, 64, 16, True), (32, 8, 128, 16, True), (20, 1, 128, 64, False),
    (10, 5, 80, 48, False), (8, 4, 256, 32, True), (3, 1, 8, 16, False), (33, 1, 96, 80, False),
    (6, 2, 512, 64, False), (2, 2, 192, 16, True), (2, 1, 328, 16, False), (16, 1, 40, 256, False)])
def test_attend_at_every_edge(cuda, dtype, hq, hkv, d, page, token_major):
    q, cache, cu = make(cuda, dtype, CTX, DRAFTED, hq, hkv, d, page, token_major, seed=d,
                        spread=2.0, extra=1, pad=3)
    drafts = tree(cache, cu, DRAFTED, d)
    drafts = P.Drafts(torch.cat([drafts.masks, drafts.masks[:3]]),
                      torch.cat([drafts.pos, drafts.pos[:3]]))
    for window in (0, 1, 16, 33, 200):
        print(dtype, hq, hkv, d, page, window, flush=True)
        check(cache, q, cu, drafts, window=window)
        check(cache, q, cu, None, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ctx,n,hq,hkv,d,page", [
    ([20000], [9], 14, 2, 64, 128), ([9001, 3, 0, 20000, 1, 700], [5, 40, 3, 1, 0, 64], 8, 2, 128, 16),
    ([0], [1], 4, 4, 64, 16), ([0, 0, 0], [0, 0, 1], 4, 2, 64, 16), ([9000], [20], 2, 1, 512, 64),
    ([6345, 6300], [33, 70], 6, 1, 256, 48), ([5000], [300], 2, 1, 128, 32)])
def test_attend_long_and_uneven(cuda, dtype, ctx, n, hq, hkv, d, page):
    q, cache, cu = make(cuda, dtype, ctx, n, hq, hkv, d, page, seed=1, spread=2.0)
    drafts = tree(cache, cu, n, 1)
    for window in (0, 3000):
        print(dtype, ctx, n, hq, hkv, d, page, window, flush=True)
        check(cache, q, cu, drafts, window=window)
        check(cache, q, cu, None, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_many_requests(cuda, dtype):
    """More requests than a wave has lanes, most without drafted tokens."""
    rng = random.Random(2)
    ctx = [rng.choice([0, 1, rng.randrange(1, 60), rng.randrange(1, 700)]) for _ in range(300)]
    n = [rng.choice([0, 0, 0, 1, 3, 20]) for _ in ctx]
    q, cache, cu = make(cuda, dtype, ctx, n, 4, 2, 64, 16, seed=3, extra=200)
    print(dtype, sum(n), flush=True)
    check(cache, q, cu, tree(cache, cu, n))


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_token_equals_attend_pages(cuda, dtype):
    """A drafted token a request, alone, is the decode step; both are within the bounds of the same."""
    ctx = [0, 5, 700, 15, 16, 4000]
    q, cache, cu = make(cuda, dtype, ctx, [1] * 6, 8, 2, 128, 16, seed=4)
    out, lse = check(cache, q, cu)
    ref, rlse = cache.attend(0, q, return_lse=True)
    _, _, tol, ltol = D.attend(q, cache.k[0], cache.v[0], cache.table, cache.lens, cu,
                               1 / math.sqrt(128))
    U.close(out, ref.double().cpu(), 2 * tol)
    U.close(lse, rlse.double().cpu(), 2 * ltol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256, 512])
def test_any_masks_and_empty_rows(cuda, dtype, d):
    """Masks that are no tree's: later tokens, not itself, none at all. A row without a key is 0 and
    -inf."""
    rng = random.Random(d)
    ctx, n = [0, 40, 3, 0], [37, 12, 33, 1]
    q, cache, cu = make(cuda, dtype, ctx, n, 4, 2, d, 16, seed=5)
    bits = [[rng.getrandbits(count) if rng.random() < 0.7 else 0 for _ in range(count)] for count in n]
    bits[3] = [0]
    rows = [x for of in bits for x in of]
    masks = [[x >> 32 * w & 0xffffffff for w in range(2)] for x in rows]
    masks = int32([[x - (1 << 32) if x >> 31 else x for x in r] for r in masks], cuda)
    pos = [c + rng.randrange(count) for c, count in zip(ctx, n) for _ in range(count)]
    drafts = P.Drafts(masks, int32(pos, cuda))
    for window in (0, 1, 5, 1000):
        print(dtype, d, window, flush=True)
        out, lse = check(cache, q, cu, drafts, window=window)
        assert (out[-1] == 0).all() and (lse[-1] == -math.inf).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,hq,n", [(64, 4, 21), (128, 8, 30), (256, 2, 21), (512, 2, 21),
                                    (64, 1, 3), (128, 1, 7)])
def test_infinities_and_nan_in_masked_places(cuda, dtype, d, hq, n):
    """Values and keys that are infinite or NaN reach the rows that attend them and no other."""
    ctx = 37
    q, cache, cu = make(cuda, dtype, [ctx], [n], hq, 1, d, 16, seed=6)
    place = lambda j: (int(cache.table[0, j // 16]), slice(None), j % 16)  # noqa: E731
    drafts = tree(cache, cu, [n], 3)
    bad = {ctx + 1: math.inf, ctx + 2: -math.inf, ctx + n - 1: math.nan}
    for j, x in bad.items():
        at = place(j)
        cache.v[0][at][:, 1::3] = x
    print(dtype, d, "values", flush=True)
    out, _ = check(cache, q, cu, drafts)
    assert torch.isfinite(out[0]).all() and not torch.isfinite(out[1]).all()
    q[0].zero_()
    check(cache, q, cu, drafts, window=3)  # keys of the context outside a window too
    for j in (2, 20, ctx + n - 1):
        cache.v[0][place(j)][:] = math.nan
        cache.k[0][place(j)][:] = math.nan
    print(dtype, d, "keys", flush=True)
    check(cache, q, cu, drafts, window=5)
    check(cache, q, cu, None, window=9)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_minus_infinity(cuda, dtype):
    """A row whose attended keys all score -inf is NaN, as softmax has it, next to rows that are not."""
    q, cache, cu = make(cuda, dtype, [0], [5], 2, 1, 64, 16, seed=7)
    q.fill_(1.0)
    cache.k[0][int(cache.table[0, 0]), :, 1] = -math.inf
    masks, pos = int32([[1], [2], [3], [12], [0]], cuda), int32([0, 1, 2, 3, 4], cuda)
    out, lse = cache.attend_drafts(0, q, cu, P.Drafts(masks, pos), return_lse=True)
    assert torch.isnan(out[1]).all() and (lse[1] == -math.inf).all()
    assert torch.isfinite(out[[0, 2, 3]]).all() and (out[4] == 0).all()
    assert torch.equal(out[0], out[2]) and (lse[4] == -math.inf).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_behind_the_last_and_given_out(cuda, dtype):
    ctx, n = [100, 0, 9], [4, 7, 0]
    q, cache, cu = make(cuda, dtype, ctx, n, 4, 2, 64, 16, seed=8, pad=9)
    out, lse = check(cache, q, cu)
    assert (out[11:] == 0).all() and (lse[11:] == -math.inf).all()
    room = torch.full((20, 8, 64), 7.0, device=cuda, dtype=dtype)[:, ::2]
    got, lse2 = cache.attend_drafts(0, q, cu, out=room, return_lse=True)
    assert got is room and torch.equal(got[:11], out[:11]) and (got[11:] == 7).all()
    assert torch.equal(lse2, lse)
    wide = torch.randn(20, 4, 65, device=cuda).to(dtype)[..., 1:]  # off a multiple of 16 bytes
    a = cache.attend_drafts(0, wide, cu)
    assert torch.equal(a, cache.attend_drafts(0, wide.contiguous(), cu))
    with pytest.raises(ValueError, match="broadcast"):
        cache.attend_drafts(0, q, cu, out=room[:, :1].expand(-1, 4, -1))
    with pytest.raises(ValueError, match="out must be"):
        cache.attend_drafts(0, q, cu, out=room[1:])


def test_what_does_not_fit_is_nan(cuda):
    """Lengths, offsets, parents and page ids that do not fit: their rows NaN, the others right."""
    ctx, n = [50, 20, 33, 64], [6, 3, 9, 2]
    q, cache, cu = make(cuda, torch.float16, ctx, n, 4, 2, 64, 16, seed=9)
    good = cache.attend_drafts(0, q, cu)
    lens = cache.lens.clone()
    for value in (-1, 2, 10 ** 6, 2 ** 31 - 1, -2 ** 31):  # 2: shorter than its drafted tokens
        cache.lens[2] = value
        out, lse = cache.attend_drafts(0, q, cu, return_lse=True)
        assert torch.isnan(out[9:18]).all() and torch.isnan(lse[9:18]).all()
        assert torch.equal(out[:9], good[:9]) and torch.equal(out[18:], good[18:])
    cache.lens.copy_(lens)
    held = cache.table.clone()
    for value in (-1, cache.k.shape[1], 2 ** 31 - 1):
        cache.table[0, 2] = value
        out = cache.attend_drafts(0, q, cu)
        assert torch.isnan(out[:6]).all() and torch.equal(out[6:], good[6:])
    cache.table.copy_(held)
    parents = [0, 5, -1] + [-1] * 17
    d = P.draft_masks(int32(parents, cuda), cu, cache.lens, 9)
    out = cache.attend_drafts(0, q, cu, d)
    assert torch.isnan(out[:2]).all() and torch.isfinite(out[2:]).all()
    d.pos[12] = 32  # before the context's end
    out = cache.attend_drafts(0, q, cu, d)
    assert torch.isnan(out[12]).all() and torch.isfinite(out[13:]).all()
    for bad in ([0, 6, 4, 18, 20], [0, -5, 9, 18, 20], [0, 6, 9, 21, 20], [5, 0, 5, 0, 2 ** 31 - 1]):
        cache.attend_drafts(0, q, int32(bad, cuda))
        torch.cuda.synchronize()
    cache.status.fill_(3)  # a refused resize
    out, lse = cache.attend_drafts(0, q, cu, return_lse=True)
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    room = torch.zeros_like(q)
    assert torch.isnan(cache.attend_drafts(0, q, cu * 0, out=room)).all()


def test_no_tokens_and_no_requests(cuda):
    q, cache, cu = make(cuda, torch.bfloat16, [10, 20], [0, 0], 4, 2, 64, 16, pad=3)
    out, lse = cache.attend_drafts(0, q, cu, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = cache.attend_drafts(0, q[:0], cu, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    out, lse = P.attend_drafts(q, cache.k[0], cache.v[0], cache.table[:0], cache.lens[:0], cu[:1],
                               return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


# ---- accepted tokens ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layers,hkv,d,page,token_major,most", [
    (1, 1, 8, 16, False, 40), (3, 2, 64, 16, True, 70), (2, 5, 80, 48, False, 300),
    (24, 2, 64, 128, False, 9), (2, 1, 512, 32, True, 600)])
def test_keep_equals_indexing(cuda, dtype, layers, hkv, d, page, token_major, most):
    rng = random.Random(most)
    ctx = [0, 5, 300, 15, 16, 47, 1]
    n = [most, 1, most // 2 + 1, 0, most, 3, 2]
    lens = [c + x for c, x in zip(ctx, n)]
    need = [-(-x // page) for x in lens]
    g = torch.Generator(device=cuda).manual_seed(most)
    cache = P.PagedCache(7, max(need) * page, sum(need) + 1, hkv, d, page=page, layers=layers,
                         dtype=dtype, device=cuda, token_major=token_major)
    cache.resize(int32(lens, cuda), sum(lens))
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    paths = [sorted(rng.sample(range(x), rng.randrange(x + 1))) for x in n]
    paths[0], paths[4] = list(range(n[0])), list(range(n[4]))[1:]  # all stay; all move by one
    K = max(map(len, paths))
    path = int32([x + [rng.randrange(-9, 9)] * (K - len(x)) for x in paths], cuda)
    counts = int32([len(x) for x in paths], cuda)
    want = [x.clone() for x in (cache.k, cache.v)]
    for b, x in enumerate(paths):
        where = lambda j: (int(cache.table[b, j // page]), j % page)  # noqa: E731
        for i, t in enumerate(x):
            (a, s), (c, r) = where(ctx[b] + t), where(ctx[b] + i)
            for new, pool in zip(want, (cache.k, cache.v)):
                new[:, c, :, r] = pool[:, a, :, s]
    print(dtype, layers, hkv, d, page, most, flush=True)
    cu = int32(offsets(n), cuda)
    got = P.keep_drafts(cache.k, cache.v, cache.table, cache.lens, cu, path, counts)
    assert got.tolist() == [c + len(x) for c, x in zip(ctx, paths)]
    assert torch.equal(cache.k, want[0]) and torch.equal(cache.v, want[1])


def test_keep_refuses_what_does_not_fit(cuda):
    """A path, count, length, offset or page id that does not fit: -1, nothing moved; the others kept."""
    cache = P.PagedCache(2, 64, 8, 1, 64, page=16, device=cuda)
    cache.resize(int32([30, 30], cuda), 60)
    cache.k.normal_()
    cache.v.normal_()
    cu, held = int32([0, 10, 20], cuda), (cache.k.clone(), cache.v.clone())
    good = [3, 5, 9]

    def keep(path, count, cu=cu, lens=cache.lens, table=cache.table):
        return P.keep_drafts(cache.k, cache.v, table, lens, cu,
                             int32([path, [0, 1, 2]], cuda), int32([count, 3], cuda)).tolist()
    bad_table = cache.table.clone()
    bad_table[0, 1] = 8
    for got in (keep([5, 3, 9], 3), keep([3, 3, 9], 3), keep([3, 5, 10], 3), keep([-1, 5, 9], 3),
                keep(good, 4), keep(good, -1), keep(good, 3, table=bad_table),
                keep(good, 3, lens=int32([9, 30], cuda)), keep(good, 3, lens=int32([65, 30], cuda)),
                keep(good, 3, lens=int32([-1, 30], cuda))):
        assert got == [-1, 23]
    assert keep(good, 3, cu=int32([-1, 10, 20], cuda)) == [-1, 23]
    assert keep(good, 3, cu=int32([11, 10, 20], cuda)) == [-1, 23]
    assert torch.equal(cache.k, held[0]) and torch.equal(cache.v, held[1])
    assert keep([9, 9, 9], 0) == [20, 23]  # nothing accepted: the path is not read
    assert P.keep_drafts(cache.k, cache.v, cache.table, cache.lens, cu,
                         torch.zeros(2, 0, device=cuda, dtype=torch.int32),
                         int32([0, 0], cuda)).tolist() == [20, 20]
    assert torch.equal(cache.k, held[0])
    shared = int32([[2, 4, 6]], cuda).expand(2, 3)  # the same path for all
    P.keep_drafts(cache.k[0], cache.v[0], cache.table, cache.lens, cu, shared, int32([3, 3], cuda))
    assert torch.equal(cache.k[0, cache.table[1, 1].item(), :, 4 + 2],
                       held[0][0, cache.table[1, 1].item(), :, 4 + 6])


# ---- shared pages -------------------------------------------------------------------------------

def check_state(cache, ref, f, want):
    assert f.status.item() == want[3]
    assert [x.tolist() for x in f[:3]] == list(want[:3])
    assert cache.lens.tolist() == ref.lens and cache.nfree.item() == len(ref.free)
    assert cache.table.tolist() == ref.table
    assert cache.free[:len(ref.free)].tolist() == ref.free


@pytest.mark.parametrize("requests,page,max_len", [(1, 16, 300), (2, 48, 700), (16, 16, 900),
                                                   (64, 16, 300), (65, 32, 300), (300, 16, 200),
                                                   (5, 16, 40000), (90, 16, 18000),
                                                   (1100, 64, 500)])
def test_fork_equals_lists(cuda, requests, page, max_len):
    rng = random.Random(requests)
    width = -(-max_len // page)
    pages = max(3, min(requests * width * 2 // 3, 6000) + 3)
    cache = P.PagedCache(requests, max_len, pages, 1, 8, page=page, device=cuda)
    ref = D.ForkState(requests, width, pages, page)
    statuses = set()
    for step in range(16):
        print(requests, page, step, flush=True)
        if step % 2 == 0:  # some grow; shared pages never shrink here
            room = pages // max(1, requests) + 1
            new = [min(width * page, x + (rng.randrange(page * room) if rng.random() < 0.6 else 0))
                   for x in ref.lens]
            if step == 0:
                new[0] = min(width * page, pages // 2 * page)
            total = sum(x - o for x, o in zip(new, ref.lens))
            ref.resize(new, total)
            cache.resize(int32(new, cuda), total)
            continue
        kind = rng.choice(["beams", "cut", "end", "mixed", "all"])
        src = [b if kind in ("cut", "end") else 0 if kind == "all"
               else rng.randrange(requests) if rng.random() < 0.6 else b for b in range(requests)]
        new = [rng.randrange(ref.lens[a] + 1) if kind in ("cut", "mixed") and rng.random() < 0.5
               else 0 if kind == "end" and rng.random() < 0.5 else ref.lens[a] for a in src]
        if step == 7:
            new[-1] = ref.lens[src[-1]] + 1
        if step == 11:
            src[0], new[0] = requests, 1
        want = ref.fork(src, new)
        f = P.fork_pages(int32(src, cuda), int32(new, cuda), cache.lens, cache.table, cache.free,
                         cache.nfree, page)
        check_state(cache, ref, f, want)
        statuses.add(min(want[3], 1))
    assert {0, -1} <= statuses


@pytest.mark.parametrize("requests", [3, 200])
def test_forked_and_ended_restores_the_state(cuda, requests):
    cache = P.PagedCache(2 * requests, 600, 60 * requests, 1, 8, page=16, device=cuda)
    rng = random.Random(requests)
    lens = [rng.randrange(1, 500) for _ in range(requests)] + [0] * requests
    cache.free.copy_(cache.free[torch.randperm(60 * requests, device=cuda)])
    cache.resize(int32(lens, cuda), sum(lens))
    held = [x.clone() for x in (cache.lens, cache.table, cache.free, cache.nfree)]
    src = list(range(requests)) * 2
    f = cache.fork(int32(src, cuda), int32([lens[a] for a in src], cuda))
    cache.check()
    assert (f.source[requests:] >= 0).sum() == sum(x % 16 != 0 for x in lens)
    cache.fork(None, held[0].clone())
    cache.check()
    for x, y in zip((cache.lens, cache.table, cache.free, cache.nfree), held):
        assert torch.equal(x, y)


def test_fork_refuses_what_does_not_fit(cuda):
    cache = P.PagedCache(3, 100, 8, 1, 8, page=16, device=cuda)
    cache.resize(int32([40, 33, 0], cuda), 80)
    state = lambda: [x.clone() for x in (cache.lens, cache.table, cache.free, cache.nfree)]  # noqa: E731
    held = state()

    def fork(src, new):
        f = cache.fork(None if src is None else int32(src, cuda), int32(new, cuda))
        return f.status.item(), f.source.tolist(), f.target.tolist(), f.tokens.tolist()
    none = [-1] * 3, [-1] * 3, [0] * 3
    for src, new in (([0, 3, 0], [40, 1, 0]), ([0, -1, 0], [40, 1, 0]), (None, [41, 33, 0]),
                     (None, [40, 33, 1]), (None, [-1, 33, 0]), (None, [40, 33, 2 ** 31 - 1])):
        assert fork(src, new) == (-1, *none)
        assert all(torch.equal(x, y) for x, y in zip(state(), held))
        with pytest.raises(RuntimeError, match="fork"):
            cache.check()
    for value in (-1, 8, 2 ** 31 - 1):
        cache.table[1, 1] = value
        assert fork(None, [40, 33, 0])[0] == -1
        cache.table[1, 1] = held[1][1, 1]
    for value in (-1, 101, 2 ** 31 - 1):
        cache.lens[1] = value
        assert fork(None, [40, 0, 0])[0] == -1
        cache.lens[1] = 33
    for value in (-1, 9):
        cache.nfree.fill_(value)
        assert fork(None, [40, 33, 0])[0] == -1
    cache.nfree.fill_(0)
    assert fork([0, 0, 0], [40, 40, 39])[0] == 2  # two copies, no page
    cache.nfree.copy_(held[3])
    assert all(torch.equal(x, y) for x, y in zip(state(), held))
    assert fork([7, -3, 9], [0, 0, 0])[0] == 0  # empty rows have no source
    assert cache.nfree.item() == 8 and (cache.table == -1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layers,hkv,d,page,token_major", [
    (1, 1, 8, 16, False), (3, 2, 64, 16, True), (2, 5, 80, 48, False), (5, 8, 128, 256, True)])
def test_copy_equals_indexing(cuda, dtype, layers, hkv, d, page, token_major):
    g = torch.Generator(device=cuda).manual_seed(d)
    cache = P.PagedCache(1, 16, 40, hkv, d, page=page, layers=layers, dtype=dtype, device=cuda,
                         token_major=token_major)
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    source = [3, -1, 3, 7, 40, 5, 9, 11, 2 ** 31 - 1, 12]
    target = [20, 21, 22, 23, 24, 25, 40, -5, 26, 12]
    tokens = [1, 3, page, page - 1, 5, 0, 4, 4, 4, 4]
    for given in (tokens, None):
        want = [x.clone() for x in (cache.k, cache.v)]
        for a, c, t in zip(source, target, given or [page] * 10):
            if 0 <= a < 40 and 0 <= c < 40:
                for x in want:
                    x[:, c, :, :t] = x[:, a, :, :t]
        print(dtype, layers, hkv, d, page, given is None, flush=True)
        P.copy_pages(cache.k, cache.v, int32(source, cuda), int32(target, cuda),
                     None if given is None else int32(given, cuda))
        assert torch.equal(cache.k, want[0]) and torch.equal(cache.v, want[1])
    P.copy_pages(cache.k[0], cache.v[0], int32([1], cuda), int32([2], cuda))
    assert torch.equal(cache.k[0, 2], cache.k[0, 1]) and torch.equal(cache.v[0, 2], cache.v[0, 1])
    P.copy_pages(cache.k, cache.v, int32([], cuda), int32([], cuda))
