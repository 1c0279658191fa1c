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
@pytest.mark.parametrize("hq,hkv,d", [(2, 1, 64), (1, 1, 128), (3, 1, 256), (1, 1, 512)])
def test_attend_long_chains(cuda, dtype, hq, hkv, d):
    """Prompts' pieces longer than masks can tell, from an empty cache on and behind a context: row tiles
    that end among the drafted tokens."""
    ctx, n = [0, 77, 0, 300], [1500, 1100, 1, 17]
    q, cache, cu = make(cuda, dtype, ctx, n, hq, hkv, d, 16, seed=17, spread=2.0, pad=2)
    for window in (0, 100):
        print(dtype, hq, d, window, flush=True)
        check(cache, q, cu, window=window)
    cache.v[0][cache.table[0, 20].long(), :, 3:] = math.inf  # later tokens' values reach no earlier one
    cache.k[0][cache.table[0, 30].long(), :, 3:] = math.nan
    out, _ = check(cache, q, cu)
    assert torch.isfinite(out[:323]).all()


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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq", [1, 20, 130])
def test_attend_at_the_longest_lengths(cuda, dtype, hq):
    """Positions up to 2^31 - 17, the last a table row can hold, through a window (every page but the last
    is the same), for few, more and many rows."""
    page, d, n = 16, 64, 3
    cap = 2 ** 31 - 16
    g = torch.Generator(device=cuda).manual_seed(1)
    k, v = (torch.randn(2, 1, page, d, device=cuda, generator=g).to(dtype) for _ in range(2))
    table = torch.zeros(1, cap // page, device=cuda, dtype=torch.int32)
    q = torch.randn(n, hq, d, device=cuda, generator=g).to(dtype)
    cu = int32([0, n], cuda)
    parents = int32([-1, 0, 0], cuda)
    for total, window in ((cap, 40), (cap - 1, 1), (cap - 15, 200), (cap - 16, 17), (cap - 13, 3000)):
        table[0, (total - 1) // page] = 1
        print(dtype, hq, total, window, flush=True)
        lens = int32([total], cuda)
        for tree in (None, P.draft_masks(parents, cu, lens, n)):
            out, lse = P.attend_drafts(q, k, v, table, lens, cu, tree, window=window, return_lse=True)
            torch.cuda.synchronize()
            # the same keys at the start of a short row: a length that agrees modulo the page
            m = window + 48 - (window - total) % page
            assert (m - total) % page == 0
            short = torch.zeros(1, m // page + 2, dtype=torch.int32)
            short[0, (m - 1) // page] = 1
            at = None if tree is None else tree.pos.cpu() - (total - m)
            want, wlse, tol, ltol = D.attend(q, k, v, short, int32([m], "cpu"), cu, d ** -0.5, window,
                                             None if tree is None else tree.masks, at)
            U.close(out, want, tol)
            U.close(lse, wlse, ltol)
        table[0, (total - 1) // page] = 0


@pytest.mark.parametrize("hq", [4, 16, 64])
def test_pool_beyond_32_bit_offsets(cuda, hq):
    """Pages whose elements lie past 2^32 bytes and 2^31 elements into the pool: attended, copied, kept."""
    page, d, hkv = 256, 256, 2
    pages = 2 ** 31 // (page * d * hkv) + 300
    k = torch.empty(pages, hkv, page, d, device=cuda, dtype=torch.bfloat16)
    v = torch.empty_like(k)
    table, used = int32([[pages - 1, 3, pages - 5]], cuda), [pages - 1, 3, pages - 5]
    for pid in used:
        k[pid].normal_()
        v[pid].normal_()
    lens, cu = int32([600], cuda), int32([0, 4], cuda)
    q = torch.randn(4, hq, d, device=cuda).to(torch.bfloat16)
    print(hq, flush=True)
    out = P.attend_drafts(q, k, v, table, lens, cu)
    want, _, tol, _ = D.attend(q, k, v, table, lens, cu, 1 / math.sqrt(d))
    U.close(out, want, tol)
    P.copy_pages(k, v, int32([pages - 1, 3], cuda), int32([pages - 9, pages - 7], cuda))
    assert torch.equal(k[pages - 9], k[pages - 1]) and torch.equal(v[pages - 7], v[3])
    moved = k[pages - 5, :, 599 % page].clone()
    got = P.keep_drafts(k, v, table, lens, cu, int32([[1, 3]], cuda), int32([2], cuda))
    assert got.tolist() == [598] and torch.equal(k[pages - 5, :, 597 % page], moved)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,n", [(64, 4, 8), (64, 14, 24), (128, 8, 4), (128, 16, 5), (128, 32, 32),
                                    (256, 8, 30)])
def test_scores_that_climb_and_fall(cuda, dtype, d, hq, n):
    """Rows whose scores rise by hundreds past those of their first keys (so that weights by an early maximum
    would pass the type's range), fall by as much, or stay level, with small and large values."""
    ctx = 1500
    q, cache, cu = make(cuda, dtype, [ctx, 0], [n, 3], hq, 1, d, 64, seed=11, spread=1.0)
    key = torch.zeros(d, device=cuda)
    key[0] = 1.0
    for shape, (a, b) in (("up", (-40.0, 40.0)), ("down", (40.0, -40.0)), ("late", (0.0, 0.0))):
        for j in range(ctx + n):
            size = a + (b - a) * j / (ctx + n)
            if shape == "late":
                size = 60.0 if j == ctx - 3 else -60.0
            cache.k[0][int(cache.table[0, j // 64]), 0, j % 64] = (key * size).to(dtype)
        q.zero_()
        q[..., 0] = torch.linspace(0.0, 8.0 * math.sqrt(d), q.shape[0] * hq,
                                   device=cuda).view(q.shape[:2]).to(dtype)
        print(dtype, d, hq, n, shape, flush=True)
        check(cache, q, cu, tree(cache, cu, [n, 3], 2))
        check(cache, q, cu, None, scale=-0.11)
        check(cache, q, cu, None, scale=0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hq,n", [(64, 4, 4), (64, 8, 8), (64, 16, 16), (128, 16, 5), (128, 32, 8),
                                    (256, 16, 8)])
def test_weights_keep_their_bits(cuda, dtype, d, hq, n):
    """Every key of equal weight and values of both signs: what is left of a mean shows bits that the
    weights lose. Within the bound of the parts and sums, before the rounding."""
    q, cache, cu = make(cuda, dtype, [4000], [n], hq, 1, d, 64, seed=12, spread=0.5)
    check(cache, q, cu)
    out, lse = cache.attend_drafts(0, q, cu, return_lse=True)
    again, lse2 = cache.attend_drafts(0, q, cu, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)  # bit for bit


def test_pools_of_other_layouts_and_shared_pages(cuda):
    """Strided pools, a table that is a view, requests that share their first pages."""
    q, cache, cu = make(cuda, torch.float16, [160, 160, 40], [5, 9, 2], 8, 2, 64, 16, seed=13)
    big = torch.full((2, cache.k.shape[1], 3, 16, 128), math.nan, device=cuda, dtype=torch.float16)
    k, v = big[0][:, :2, :, :64], big[1][:, 1:, :, 64:]
    k.copy_(cache.k[0])
    v.copy_(cache.v[0])
    table = torch.full((3, 20), -1, device=cuda, dtype=torch.int32)[:, 3:14]
    table[:, :11] = cache.table[:, :11]
    table[1, :9] = table[0, :9]
    out, lse = P.attend_drafts(q, k, v, table, cache.lens, cu, return_lse=True)
    want, wlse, tol, ltol = D.attend(q, k, v, table, cache.lens, cu, 1 / 8)
    U.close(out, want, tol)
    U.close(lse, wlse, ltol)


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


# ---- the run of them ----------------------------------------------------------------------------

class Told:
    """What the requests of a cache hold, token by token and layer by layer, kept beside it."""

    def __init__(self, cache):
        self.cache, self.rows = cache, [[] for _ in range(cache.lens.numel())]

    def check(self):
        c = self.cache
        c.check()
        assert c.lens.tolist() == [len(x) for x in self.rows]
        page, held = c.page, []
        for b, row in enumerate(self.rows):
            ids = c.table[b].tolist()
            need = -(-len(row) // page)
            assert all(x == -1 for x in ids[need:])
            held.append(ids[:need])
            if row:
                at = torch.tensor([ids[j // page] for j in range(len(row))], device=c.k.device)
                off = torch.arange(len(row), device=c.k.device) % page
                want = torch.stack(row)  # (n, 2, layers, hkv, d)
                for i, pool in enumerate((c.k, c.v)):
                    got = pool.permute(1, 3, 0, 2, 4)[at, off]
                    assert torch.equal(got, want[:, i])
        free = c.free[:c.nfree.item()].tolist()
        every = set(sum(held, []))
        assert len(set(free)) == len(free) and not every & set(free)
        assert len(every) + len(free) == c.k.shape[1]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("token_major,hq,d", [(False, 4, 64), (True, 16, 128)])
def test_drafts_verified_kept_and_forked(cuda, dtype, token_major, hq, d):
    """Prompts, steps of drafted trees of which a part is accepted, requests forked and ended: after each
    the cache holds what it should, attention is that of the plain form, pages are free or listed."""
    rng = random.Random(d)
    B, layers, hkv, page = 6, 2, 2, 16
    cache = P.PagedCache(B, 400, 120, hkv, d, page=page, layers=layers, dtype=dtype, device=cuda,
                         token_major=token_major)
    told = Told(cache)
    cache.k.fill_(math.nan)
    cache.v.fill_(math.nan)
    for step in range(14):
        print(dtype, token_major, step, flush=True)
        lens = cache.lens.tolist()
        if step in (0, 7):  # prompts
            grow = [rng.randrange(1, 60) if n == 0 else 0 for n in lens]
            r = cache.resize(cache.lens + int32(grow, cuda), sum(grow))
        elif step in (3, 9):  # a request's answers
            src = [0, 0, 0, 3, 4, 3]
            if step == 9:
                src = [5, 4, 2, 2, 1, 1]
            new = [rng.randrange(1, lens[a] + 1) if rng.random() < 0.5 else lens[a] for a in src]
            cache.fork(int32(src, cuda), int32(new, cuda))
            told.rows = [told.rows[a][:n] for a, n in zip(src, new)]
            told.check()
            continue
        elif step in (6, 13):  # some end
            new = [0 if step == 13 or b % 2 else n for b, n in enumerate(lens)]
            cache.fork(None, int32(new, cuda))
            told.rows = [row[:n] for row, n in zip(told.rows, new)]
            told.check()
            continue
        else:
            grow = [rng.choice([0, 1, rng.randrange(1, 20)]) if n else 0 for n in lens]
            r = cache.resize(cache.lens + int32(grow, cuda), sum(grow) + 3)
        N = r.slots.numel()
        x = torch.randn(N, 2, layers, hkv, d, device=cuda).to(dtype)
        for layer in range(layers):
            cache.append(layer, x[:, 0, layer], x[:, 1, layer], r.slots)
        at = offsets(grow)
        for b in range(B):
            told.rows[b] = told.rows[b] + list(x[at[b]:at[b + 1]])
        told.check()
        q = torch.randn(N, hq, d, device=cuda).to(dtype)
        if step in (0, 7):
            check(cache, q, r.cu)
            continue
        parents = sum((D.random_parents(rng, n) for n in grow), []) + [0] * 3
        drafts = P.draft_masks(int32(parents, cuda), r.cu, cache.lens, 20)
        check(cache, q, r.cu, drafts, window=rng.choice([0, 30]))
        path = []
        for b, n in enumerate(grow):  # a way down the tree, by the parents
            way, t = [], rng.randrange(-1, n)
            while t >= 0:
                way.append(t)
                t = parents[at[b] + t]
            path.append(way[::-1])
        K = max(map(len, path)) + 1
        cache.accept(r.cu, int32([p + [-5] * (K - len(p)) for p in path], cuda),
                     int32([len(p) for p in path], cuda))
        for b, p in enumerate(path):
            first = len(told.rows[b]) - grow[b]
            told.rows[b] = told.rows[b][:first] + [told.rows[b][first + t] for t in p]
        told.check()
    assert cache.nfree.item() == 120


def test_a_path_that_does_not_fit_refuses_the_resize(cuda):
    cache = P.PagedCache(2, 64, 8, 1, 64, page=16, device=cuda)
    r = cache.resize(int32([20, 9], cuda), 29)
    cache.accept(r.cu, int32([[3, 2], [0, 1]], cuda), int32([2, 2], cuda))
    assert cache.status.item() == -1 and cache.lens.tolist() == [20, 9]
    with pytest.raises(RuntimeError, match="resize"):
        cache.check()
    cache.accept(r.cu, int32([[2, 3], [0, 1]], cuda), int32([2, 2], cuda))
    cache.check()
    assert cache.lens.tolist() == [2, 2]


def test_a_refused_resize_leaves_no_drafts(cuda):
    """After a resize that does not fit: no masks, NaN rows, nothing kept, until one fits."""
    cache = P.PagedCache(2, 64, 4, 1, 64, page=16, device=cuda)
    x = torch.randn(40, 1, 64, device=cuda).to(torch.bfloat16)
    r = cache.resize(int32([20, 9], cuda), 40)
    cache.append(0, x, x, r.slots)
    held = cache.k.clone()
    r = cache.resize(int32([60, 20], cuda), 60)
    assert r.status.item() > 0
    drafts = P.draft_masks(torch.zeros(60, device=cuda, dtype=torch.int32), r.cu, cache.lens, 60)
    assert (drafts.masks == 0).all() and (drafts.pos == 0).all()
    q = torch.randn(60, 2, 64, device=cuda).to(torch.bfloat16)
    assert cache.attend_drafts(0, q, r.cu, drafts).isnan().all()
    got = P.keep_drafts(cache.k, cache.v, cache.table, cache.lens, r.cu, int32([[0], [0]], cuda),
                        int32([0, 0], cuda))
    assert got.tolist() == [20, 9] and torch.equal(cache.k, held)
    f = cache.fork(None, int32([20, 0], cuda))
    assert f.status.item() == 0 and not cache.attend(0, q[:2]).isnan().any()


def test_captured_run_replayed(cuda):
    """A step of drafted tokens (room, masks, stored, attended, some kept) in a graph, replayed as requests
    grow, with eager work between: equal to an eager cache beside it at every replay."""
    B, hq, hkv, d, page = 5, 8, 2, 64, 16
    a, b = (P.PagedCache(B, 500, 160, hkv, d, page=page, layers=2, dtype=torch.float16, device=cuda)
            for _ in range(2))
    start = int32([30, 1, 100, 64, 7], cuda)
    x = torch.randn(202, hkv, d, device=cuda).to(torch.float16)
    for c in (a, b):
        r = c.resize(start, 202)
        for layer in range(2):
            c.append(layer, x, x, r.slots)
    grow, N = int32([4, 1, 8, 2, 5], cuda), 23
    parents = int32([0] * N, cuda)
    path, counts = int32([[0, 1, 3]] * B, cuda), int32([0] * B, cuda)
    q = torch.randn(N, hq, d, device=cuda).to(torch.float16)
    k, v = (torch.randn(N, hkv, d, device=cuda).to(torch.float16) for _ in range(2))
    src, give = torch.arange(B, device=cuda, dtype=torch.int32), int32([0] * B, cuda)

    def step(c):
        r = c.resize(c.lens + grow, N)
        drafts = P.draft_masks(parents, r.cu, c.lens, 8)
        outs = []
        for layer in range(2):
            c.append(layer, k, v, r.slots)
            outs += c.attend_drafts(layer, q, r.cu, drafts, window=40 * layer, return_lse=True)
        c.accept(r.cu, path, counts)
        f = c.fork(src, c.lens - give)
        return outs, drafts, f
    parents.copy_(int32(sum((D.random_parents(random.Random(1), n) for n in grow.tolist()), [])
                        + [0] * 3, cuda))
    for c in (a, b):
        step(c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs, drafts, f = step(a)
    for rep in range(20):
        rng = random.Random(rep)
        grow.copy_(int32([rng.randrange(5) for _ in range(B)], cuda))
        n = grow.tolist()
        ways = sum((D.random_parents(rng, m) for m in n), [])
        parents.copy_(int32(ways + [0] * (N - len(ways)), cuda))
        keep = [sorted(rng.sample(range(m), rng.randrange(min(m, 3) + 1))) for m in n]
        path.copy_(int32([p + [0] * (3 - len(p)) for p in keep], cuda))
        counts.copy_(int32([len(p) for p in keep], cuda))
        src.copy_(int32([rng.choice([i, i, rng.randrange(B)]) for i in range(B)], cuda))
        give.zero_()
        low = torch.minimum(a.lens + counts, (a.lens + counts)[src.long()])
        give.copy_(a.lens + counts - low)  # at most what the source holds
        for t in (q, k, v):
            t.normal_()
        graph.replay()
        torch.empty(1 << 20, device=cuda).normal_().sum().item()
        torch.cuda.synchronize()
        want, wdrafts, wf = step(b)
        assert all(torch.equal(x, y) for x, y in zip(outs, want)), rep
        assert all(torch.equal(x, y) for x, y in zip(drafts, wdrafts)), rep
        assert all(torch.equal(x, y) for x, y in zip(f, wf)) and f.status.item() == 0, rep
        for x, y in ((a.lens, b.lens), (a.table, b.table), (a.free, b.free), (a.nfree, b.nfree),
                     (a.k, b.k), (a.v, b.v)):
            assert torch.equal(x, y), rep


def test_two_graphs_with_one_memory_pool(cuda):
    """Two captured calls whose workspaces share a pool, replayed in turn with eager calls between."""
    q, cache, cu = make(cuda, torch.bfloat16, [7000, 300], [9, 4], 8, 2, 64, 16, seed=14)
    q2, other, cu2 = make(cuda, torch.bfloat16, [50, 9000], [3, 17], 8, 2, 64, 16, seed=15)
    want, want2 = cache.attend_drafts(0, q, cu), other.attend_drafts(0, q2, cu2)
    torch.cuda.synchronize()
    a, b = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(a):
        out = cache.attend_drafts(0, q, cu)
    with torch.cuda.graph(b, pool=a.pool()):
        out2 = other.attend_drafts(0, q2, cu2)
    for _ in range(4):
        a.replay()
        assert torch.equal(out, want)
        b.replay()
        assert torch.equal(out2, want2)
        torch.empty(1 << 20, device=cuda).normal_().sum().item()
        assert torch.equal(cache.attend_drafts(0, q, cu), want)


def test_other_streams(cuda):
    q, cache, cu = make(cuda, torch.bfloat16, [7000, 50], [9, 30], 8, 2, 64, 16, seed=16)
    drafts = tree(cache, cu, [9, 30])
    want = cache.attend_drafts(0, q, cu, drafts)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(cache.attend_drafts(0, q, cu, tree(cache, cu, [9, 30])))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_compiled_run_equals_eager(cuda):
    caches = []
    for _ in range(2):
        c = P.PagedCache(3, 200, 40, 2, 64, page=16, layers=2, dtype=torch.float16, device=cuda)
        torch.manual_seed(3)
        x = torch.randn(90, 2, 64, device=cuda).to(torch.float16)
        r = c.resize(int32([50, 7, 33], cuda), 90)
        for layer in range(2):
            c.append(layer, x, x, r.slots)
        caches.append(c)
    q, x = torch.randn(9, 4, 64, device=cuda).half(), torch.randn(9, 2, 64, device=cuda).half()
    parents, grow = int32([-1, 0, 0, -1, 0, 1, 1, 9, 9], cuda), int32([3, 0, 4], cuda)
    path, counts = int32([[0, 2], [0, 0], [0, 3]], cuda), int32([2, 0, 2], cuda)
    src = int32([0, 0, 2], cuda)

    def run(c, out):
        r = c.resize(c.lens + grow, 9)
        drafts = P.draft_masks(parents, r.cu, c.lens, 40)
        c.append(0, x, x, r.slots)
        a, lse = c.attend_drafts(0, q, r.cu, drafts, window=20, return_lse=True)
        b = c.attend_drafts(0, q, r.cu, out=out)
        c.accept(r.cu, path, counts)
        f = c.fork(src, c.lens)
        return a, lse, b, tuple(f), tuple(drafts)
    outs = [torch.full((9, 4, 64), 7.0, device=cuda, dtype=torch.float16) for _ in range(2)]
    want = run(caches[0], outs[0])
    got = torch.compile(run, backend="aot_eager")(caches[1], outs[1])
    flat = lambda t: [y for x in t for y in (flat(x) if isinstance(x, tuple) else [x])]  # noqa: E731
    for x, y in zip(flat(want), flat(got)):
        assert torch.equal(x, y)
    assert (outs[0][7:] == 7).all() and torch.equal(outs[0], outs[1])
    for x in ("lens", "table", "free", "nfree", "status", "k", "v"):
        assert torch.equal(getattr(caches[0], x), getattr(caches[1], x)), x


# ---- the bits of the weights ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,hq,n", [(64, 2, 3), (64, 8, 4), (64, 16, 16), (128, 2, 2), (128, 16, 4),
                                    (128, 32, 8), (256, 1, 3), (256, 16, 4), (512, 2, 3)])
def test_weights_hold_all_their_bits(cuda, dtype, d, hq, n):
    """Values that cancel but for what a weight lacks (drafts_util.cancelling), at every tile size."""
    q, cache, cu = make(cuda, dtype, [150], [n], hq, 1, d, 16)
    values, want, off = D.cancelling(dtype)
    q.zero_()
    q[..., 0] = 1.0
    for j in range(150 + n):
        at = (int(cache.table[0, j // 16]), 0, j % 16)
        cache.k[0][at].zero_()
        cache.k[0][at][0] = D.WEIGHT_KEYS.get(j, -2000.0)
        if j in values:
            cache.v[0][at].fill_(values[j])
    print(dtype, d, hq, n, flush=True)
    out = cache.attend_drafts(0, q, cu, scale=D.WEIGHT_SCALE).double().cpu()
    worst = (out - want).abs().max().item()
    assert worst <= off, (worst, off, want)


# ---- rows that no request holds -----------------------------------------------------------------

BAD_OFFSETS = [[0, 6, 25], [3, 6, 20], [3, 6, 17], [0, 0, 21], [0, 20, 2 ** 31 - 1], [-2, 5, 20], [-2, 5, 18],
               [-2 ** 31, -1, 7], [20, 20, 20], [25, 30, 30], [-9, -5, -3], [-2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1],
               [0, 12, 6], [5, 0, 20], [20, 4, 4], [2 ** 31 - 1, 0, 4]]


def poison(dev, *shapes):
    """Memory of these sizes that the next allocations of them get, full of sevens."""
    held = [torch.full(shape, 7, device=dev, dtype=dtype) for shape, dtype in shapes]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("requests", [2, 70, 1500])
def test_masks_of_rows_that_no_request_holds(cuda, requests):
    """Written whatever the offsets: 0 and -1 where they do not fit, 0 and 0 behind the last request."""
    N, most = 20, 40
    rng = random.Random(1)
    parents = D.random_parents(rng, N)
    for bad in BAD_OFFSETS:
        cu = bad[:1] * (requests - 2) + bad
        lens = [2 ** 31 - 1 - b for b in range(requests)]
        first, own, held, behind = D.rows_of(cu, N)
        masks, pos = [[0, 0] for _ in range(N)], [-1] * behind + [0] * (N - behind)
        ways = []  # parents of a request's tokens count from its first
        for a, b in zip(own, own[1:]):
            ways += D.random_parents(rng, b - a)
        given = parents[:first] + ways + parents[first + len(ways):]
        m, at = D.masks_and_pos(ways, [b - a for a, b in zip(own, own[1:])], [lens[b] for b in held], 2,
                                len(ways))
        masks[first:first + len(ways)], pos[first:first + len(ways)] = m, at
        print(requests, bad, flush=True)
        args = [int32(x, cuda) for x in (given, cu, lens)]
        poison(cuda, ((N, 2), torch.int32), ((N,), torch.int32))
        d = P.draft_masks(*args, most)
        assert d.masks.tolist() == masks and d.pos.tolist() == pos, bad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ctx,requests,hq,d", [(40, 2, 4, 64), (9000, 2, 2, 64), (9000, 2, 8, 128),
                                               (5000, 2, 32, 64), (700, 70, 4, 256), (40, 70, 2, 512)])
def test_attention_of_rows_that_no_request_holds(cuda, dtype, ctx, requests, hq, d):
    """NaN where the offsets do not fit, whatever the memory held before, the other requests right; rows
    behind the last request zeros, or as they were."""
    N, page = 20, 64
    q, cache, _ = make(cuda, dtype, [ctx], [N], hq, 2, d, page, seed=21)
    table = cache.table.expand(requests, -1).contiguous()
    lens = int32([ctx + N - b % 3 for b in range(requests)], cuda)
    for bad in BAD_OFFSETS:
        cu = bad[:1] * (requests - 2) + bad
        first, own, held, behind = D.rows_of(cu, N)
        rows = slice(first, first + own[-1])
        print(dtype, ctx, requests, hq, d, bad, flush=True)
        args = (q, cache.k[0], cache.v[0], table, lens, int32(cu, cuda))
        poison(cuda, ((N, hq, d), dtype), ((N, hq), torch.float32))
        out, lse = P.attend_drafts(*args, return_lse=True)
        given = torch.full_like(q, 7.0)
        got, glse = P.attend_drafts(*args, return_lse=True, out=given)
        torch.cuda.synchronize()
        if held:
            want, wlse, tol, ltol = D.attend(q[rows], cache.k[0], cache.v[0], table[held], lens[held],
                                             torch.tensor(own), 1 / math.sqrt(d))
            U.close(out[rows], want, tol)
            U.close(lse[rows], wlse, ltol)
        misfit = torch.ones(N, dtype=torch.bool, device=cuda)
        misfit[rows] = False
        misfit[behind:] = False
        assert out[misfit].isnan().all() and lse[misfit].isnan().all(), bad
        assert (out[behind:] == 0).all() and (lse[behind:] == -math.inf).all(), bad
        assert torch.equal(got[:behind].nan_to_num(5.0), out[:behind].nan_to_num(5.0)), bad
        assert (got[behind:] == 7).all() and torch.equal(glse.nan_to_num(5.0), lse.nan_to_num(5.0)), bad


# ---- accepted for all requests or none ----------------------------------------------------------

@pytest.mark.parametrize("requests", [2, 70])
@pytest.mark.parametrize("wrong", ["order", "range", "count", "page"])
def test_accept_is_all_or_nothing_and_can_be_made_again(cuda, requests, wrong):
    """One path that does not fit: nothing is moved for any request; corrected and accepted again, every
    request holds what its path says."""
    page, layers, n = 16, 3, 9
    ctx = [(7 * b) % 40 for b in range(requests)]
    cache = P.PagedCache(requests, 80, 6 * requests, 2, 64, page=page, layers=layers, device=cuda)
    cache.resize(int32(ctx, cuda), sum(ctx))
    r = cache.resize(int32([c + n for c in ctx], cuda), n * requests)
    cache.k.normal_()
    cache.v.normal_()
    held = cache.k.clone(), cache.v.clone()
    paths = [sorted(random.Random(b).sample(range(n), 1 + b % 5)) for b in range(requests)]
    paths[0], last = [1, 2, 4], requests - 1
    paths[last] = [2, 5, 8]
    width = max(map(len, paths))
    path = int32([p + [-1] * (width - len(p)) for p in paths], cuda)
    counts = int32([len(p) for p in paths], cuda)
    bad_path, bad_counts, table = path.clone(), counts.clone(), cache.table.clone()
    if wrong == "order":
        bad_path[last, 2] = 3
    elif wrong == "range":
        bad_path[last, 2] = n
    elif wrong == "count":
        bad_counts[last] = -1
    else:
        cache.table[last, (ctx[last] + 8) // page] = 6 * requests
    print(requests, wrong, flush=True)
    cache.accept(r.cu, bad_path, bad_counts)
    with pytest.raises(RuntimeError, match="resize"):
        cache.check()
    assert cache.lens.tolist() == [c + n for c in ctx]
    assert torch.equal(cache.k, held[0]) and torch.equal(cache.v, held[1])
    new = P.keep_drafts(cache.k, cache.v, cache.table, cache.lens, r.cu, bad_path, bad_counts,
                        all_or_none=True).tolist()
    assert new == [c + len(p) for c, p in zip(ctx[:-1], paths[:-1])] + [-1]
    assert torch.equal(cache.k, held[0]) and torch.equal(cache.v, held[1])
    cache.table.copy_(table)
    want = held[0].clone(), held[1].clone()
    for b, p in enumerate(paths):
        for i, t in enumerate(p):
            (a, s), (c, at) = (divmod(ctx[b] + x, page) for x in (t, i))
            for x, y in zip(want, held):
                x[:, table[b, c], :, at] = y[:, table[b, a], :, s]
    cache.accept(r.cu, path, counts)
    cache.check()
    assert cache.lens.tolist() == [c + len(p) for c, p in zip(ctx, paths)]
    assert torch.equal(cache.k, want[0]) and torch.equal(cache.v, want[1])


# ---- rows that list a page more than once -------------------------------------------------------

@pytest.mark.parametrize("page,width", [(16, 12), (16, 2600)])
def test_pages_that_a_row_lists_twice_go_back_once(cuda, page, width):
    """Rows set by the caller, a page at several places of a row and in several rows: forked, cut and ended as
    in lists; every page is free once in the end."""
    rng = random.Random(width)
    B, pages = 4, 40
    cache = P.PagedCache(B, width * page, pages, 1, 8, page=page, device=cuda)
    ref = D.ForkState(B, width, pages, page)
    for rep in range(6):
        ref.table = [[-1] * width for _ in range(B)]
        ref.lens = [rng.randrange(1, width * page + 1) if b else width * page for b in range(B)]
        some = rng.sample(range(pages), 14)
        for b, n in enumerate(ref.lens):
            need = -(-n // page)
            ref.table[b][:need] = [rng.choice(some[:11] if b else some[3:]) for _ in range(need)]
        listed = set(sum(ref.table, [])) - {-1}
        ref.free = [x for x in range(pages) if x not in listed]
        rng.shuffle(ref.free)
        cache.table.copy_(int32(ref.table, cuda))
        cache.lens.copy_(int32(ref.lens, cuda))
        cache.free[:len(ref.free)] = int32(ref.free, cuda)
        cache.nfree.fill_(len(ref.free))
        for kind in ("fork", "cut", "some end", "end"):
            lens = ref.lens
            src = [rng.randrange(B) for _ in range(B)] if kind == "fork" else list(range(B))
            new = [0 if kind == "end" or kind == "some end" and b % 2 else
                   lens[a] if kind == "some end" else rng.randrange(lens[a] + 1) for b, a in enumerate(src)]
            print(page, width, rep, kind, flush=True)
            want = ref.fork(src, new)
            f = P.fork_pages(int32(src, cuda), int32(new, cuda), cache.lens, cache.table, cache.free,
                             cache.nfree, page)
            check_state(cache, ref, f, want)
        assert sorted(cache.free.tolist()) == list(range(pages)) and cache.nfree.item() == pages


# ---- positions below 0 --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,hq", [(64, 2), (64, 16), (128, 8), (256, 2), (512, 2)])
def test_windows_over_keys_at_positions_below_zero(cuda, dtype, d, hq):
    """With any masks and positions a drafted key counts if it lies past its row's position less the window,
    whatever its sign."""
    ctx, n = [0, 5, 40], [9, 20, 33]
    q, cache, cu = make(cuda, dtype, ctx, n, hq, 1, d, 16, seed=22)
    rng = random.Random(d)
    masks, pos = [], []
    for c, count in zip(ctx, n):
        for t in range(count):
            low = t % 3 == 1  # a key only: its own row does not fit
            bits = rng.getrandbits(count) | 1 << t
            masks.append([bits >> 32 * w & 0xffffffff for w in range(2)])
            pos.append(-rng.randrange(1, 12) if low else c + rng.randrange(count))
    words = int32([[x - (1 << 32) if x >> 31 else x for x in m] for m in masks], cuda)
    drafts = P.Drafts(words, int32(pos, cuda))
    fits = torch.tensor([p >= 0 for p in pos])
    for window in (1, 4, 10, 20, 70, 2 ** 31 - 1):
        print(dtype, d, hq, window, flush=True)
        out, lse = cache.attend_drafts(0, q, cu, drafts, window=window, return_lse=True)
        torch.cuda.synchronize()
        want, wlse, tol, ltol = D.attend(q, cache.k[0], cache.v[0], cache.table, cache.lens, cu, d ** -0.5,
                                         window, *drafts)
        U.close(out[fits], want[fits], tol[fits])
        U.close(lse[fits], wlse[fits], ltol[fits])
        assert out[~fits].isnan().all() and lse[~fits].isnan().all()


# ---- pages that only a request's last tokens read -----------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,d,ctx", [(2, 64, 0), (2, 64, 9000), (1, 128, 77), (1, 256, 300), (1, 512, 0)])
def test_a_bad_page_past_a_tile_makes_the_whole_request_nan(cuda, dtype, hq, d, ctx):
    """A chain of many row tiles, of which the first do not read the last pages: NaN in every row all the
    same, the request beside it right."""
    page, n = 16, [900, 40]
    q, cache, cu = make(cuda, dtype, [ctx, 20], n, hq, 1, d, page, seed=23)
    good = cache.attend_drafts(0, q, cu)
    assert good.isfinite().all()
    held = cache.table.clone()
    for at in (ctx + 899, ctx + 450, ctx + 16, ctx // 2):
        for value in (-1, cache.k.shape[1], 2 ** 31 - 1):
            cache.table[0, at // page] = value
            print(dtype, hq, d, ctx, at, value, flush=True)
            out, lse = cache.attend_drafts(0, q, cu, return_lse=True)
            assert out[:900].isnan().all() and lse[:900].isnan().all()
            assert torch.equal(out[900:], good[900:])
        cache.table.copy_(held)
    assert torch.equal(cache.attend_drafts(0, q, cu), good)
