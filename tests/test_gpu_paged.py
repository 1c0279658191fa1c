"""The paged key-value cache on the GPU: pages, slots and positions equal to plain lists, appended rows
bit for bit, attention within the bounds of its arithmetic (paged_util.attend)."""
import math
import random

import pytest
import torch

from ssa_amd import _lib
from ssa_amd import paged as P
from tests import paged_util as U

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def int32(x, dev):
    return torch.tensor(x, device=dev, dtype=torch.int32)


# ---- pages, slots, positions --------------------------------------------------------------------

def check_state(cache, ref, r, want):
    slots, pos, cu, status = want
    assert r.status.item() == status
    assert r.slots.tolist() == slots and r.pos.tolist() == pos and r.cu.tolist() == cu
    assert cache.lens.tolist() == ref.lens and cache.nfree.item() == len(ref.free)
    assert cache.table.tolist() == ref.table
    assert cache.free[:len(ref.free)].tolist() == ref.free


@pytest.mark.parametrize("requests,page,max_len", [(1, 16, 5000), (3, 48, 700), (64, 16, 900),
                                                   (1000, 32, 300), (1024, 16, 200),
                                                   (1025, 64, 500), (2500, 16, 100)])
def test_resize_equals_lists(cuda, requests, page, max_len):
    rng = random.Random(requests)
    width = -(-max_len // page)
    pages = requests * width * 2 // 3 + 3  # growth is refused now and then
    cache = P.PagedCache(requests, max_len, pages, 1, 8, page=page, device=cuda)
    ref = U.PageState(requests, width, pages, page)
    statuses = set()
    for step in range(14):
        kind = rng.choice(["grow", "shrink", "mixed", "end"])
        new = []
        for n in ref.lens:
            up = min(width * page, n + rng.choice([0, 1, 1, page, rng.randrange(max_len)]))
            new.append(up if kind == "grow" or kind == "mixed" and rng.random() < 0.5
                       else 0 if kind == "end" and rng.random() < 0.5 else rng.randrange(n + 1))
        if step == 5:
            new[-1] = width * page + 1
        if step == 9:
            new[0] = -1
        total = sum(max(0, n - o) for o, n in zip(ref.lens, new))
        tokens = max(0, total + rng.choice([0, 0, 5, 300, -1]))
        print(requests, page, step, kind, total, tokens, flush=True)
        before = cache.free.clone()
        want = ref.resize(new, tokens)
        r = cache.resize(int32(new, cuda), tokens)
        check_state(cache, ref, r, want)
        statuses.add(min(want[3], 1))
        if want[3]:
            assert torch.equal(cache.free, before)
            with pytest.raises(RuntimeError, match="resize"):
                cache.check()
        else:
            cache.check()
    assert {0, -1} <= statuses


@pytest.mark.parametrize("requests,pages", [(1, 4), (64, 150), (300, 400), (1024, 2000)])
def test_resize_by_single_tokens(cuda, requests, pages):
    """Steps in which no request changes by more than a token or a page: decode steps, tokens taken back,
    requests that end; now and then refused."""
    rng = random.Random(pages)
    page = 16
    cache = P.PagedCache(requests, 320, pages, 1, 8, page=page, device=cuda)
    ref = U.PageState(requests, 20, pages, page)
    lens = [rng.randrange(1 if pages < 500 else 33) for _ in range(requests)]
    ref.resize(lens, sum(lens))
    cache.resize(int32(lens, cuda), sum(lens))
    statuses = set()
    for step in range(60):
        move = rng.choice(["grow", "grow", "all", "back", "mixed"])
        new = [min(n + 1, 320) if move == "all" or move in ("grow", "mixed") and rng.random() < 0.7
               else max(0, n - rng.randrange(page)) if move in ("back", "mixed") else n
               for n in ref.lens]
        room = requests + rng.choice([0, 3]) - (step % 20 == 7) * requests
        want = ref.resize(new, room)
        r = cache.resize(int32(new, cuda), room)
        check_state(cache, ref, r, want)
        statuses.add(min(want[3], 1))
    assert -2 in statuses and 0 in statuses


def test_resize_grown_and_shrunk_back_restores_the_state(cuda):
    cache = P.PagedCache(40, 1000, 800, 1, 8, page=16, device=cuda)
    rng = random.Random(4)
    cache.resize(int32([rng.randrange(300) for _ in range(40)], cuda), 20000)
    cache.check()
    held = [x.clone() for x in (cache.lens, cache.table, cache.free, cache.nfree)]
    cache.resize(cache.lens + int32([rng.randrange(2, 180) for _ in range(40)], cuda), 9000)
    cache.check()
    assert not torch.equal(cache.table, held[1])
    cache.resize(held[0].clone(), 0)
    cache.check()
    for x, y in zip((cache.lens, cache.table, cache.free, cache.nfree), held):
        assert torch.equal(x, y)


@pytest.mark.parametrize("requests", [3, 1100])
def test_resize_sums_past_31_bits(cuda, requests):
    """Lengths whose pages or tokens add up past 2^31 are counted, not wrapped; a request of more than a
    million pages is served."""
    i32 = dict(device=cuda, dtype=torch.int32)
    width, pages = 2 ** 27 - 1, 1200000
    table = torch.full((1, width), -1, **i32).expand(requests, width)  # refused before it is written
    lens, free = torch.zeros(requests, **i32), torch.arange(pages, **i32)
    nfree, new = torch.full((1,), pages, **i32), torch.full((requests,), width * 16, **i32)
    ptr = lambda t: t.data_ptr()  # noqa: E731
    out = torch.empty(8, device=cuda, dtype=torch.int64), torch.empty(requests + 1, **i32)
    status = torch.empty(1, **i32)

    # 2^31 - 16 tokens each, room for 8: the table is neither read nor written
    _lib.call("ssa_paged_resize", ptr(lens), ptr(new), ptr(table), width, requests, width, 16,
              ptr(free), pages, ptr(nfree), ptr(out[0]), None, 8, ptr(out[1]), ptr(status),
              _lib.stream_of(lens))
    assert status.item() == -2 and (out[0] == -1).all() and (out[1] == 0).all()
    assert (lens == 0).all() and nfree.item() == pages
    new.zero_()
    new[0] = 17 * 10 ** 6
    cache = P.PagedCache(requests, 17 * 10 ** 6, pages, 1, 8, page=16, dtype=torch.float16,
                         device=cuda)
    r = cache.resize(new, 17 * 10 ** 6 + 5)
    assert r.status.item() == 0 and cache.nfree.item() == pages - 1062500
    assert torch.equal(cache.table[0, :1062500], torch.arange(1062500, **i32))
    at = torch.arange(17 * 10 ** 6, device=cuda)
    assert torch.equal(r.slots[:-5], at) and (r.slots[-5:] == -1).all()
    assert torch.equal(r.pos[:-5], at.to(torch.int32)) and r.cu[1].item() == 17 * 10 ** 6
    cache.resize(torch.zeros_like(new), 0)
    cache.check()
    assert torch.equal(cache.free, torch.arange(pages, **i32).flip(0))
    assert (cache.table == -1).all() and cache.nfree.item() == pages


def test_resize_into_its_own_lengths_changes_nothing(cuda):
    cache = P.PagedCache(5, 100, 40, 1, 8, page=16, device=cuda)
    cache.resize(int32([3, 0, 16, 17, 99], cuda), 200)
    held = cache.table.clone()
    r = cache.resize(cache.lens, 4)
    assert r.status.item() == 0 and r.slots.tolist() == [-1] * 4 and r.cu.tolist() == [0] * 6
    assert torch.equal(cache.table, held) and cache.lens.tolist() == [3, 0, 16, 17, 99]


def test_empty_batch_through_the_run(cuda):
    """No requests: resize, append and attend all answer an empty batch and leave the pool alone."""
    cache = P.PagedCache(2, 64, 6, 1, 64, page=16, device=cuda)
    lens, table = cache.lens[:0], cache.table[:0]
    r = P.resize_pages(lens, lens.clone(), table, cache.free, cache.nfree, 16, 5)
    assert r.slots.tolist() == [-1] * 5 and r.pos.tolist() == [0] * 5
    assert r.cu.tolist() == [0] and r.status.tolist() == [0]
    assert cache.nfree.item() == 6 and sorted(cache.free.tolist()) == list(range(6))
    x = torch.ones(5, 1, 64, device=cuda, dtype=torch.bfloat16)
    cache.append(0, x, x, r.slots)
    out, lse = P.attend_pages(x[:0], cache.k[0], cache.v[0], table, lens, return_lse=True)
    assert out.shape == (0, 1, 64) and lse.shape == (0, 1) and (cache.k == 0).all()


def test_resize_refuses_a_bad_free_count(cuda):
    cache = P.PagedCache(2, 100, 10, 1, 8, page=16, device=cuda)
    for n in (-1, 11, 2 ** 31 - 1):
        cache.nfree.fill_(n)
        assert cache.resize(int32([20, 0], cuda), 20).status.item() == -1
        assert cache.lens.tolist() == [0, 0] and cache.nfree.item() == n
    cache.nfree.fill_(10)
    cache.resize(int32([20, 0], cuda), 20)
    cache.nfree.fill_(10)  # two pages too many: giving back would pass the stack's end
    assert cache.resize(int32([0, 0], cuda), 0).status.item() == -1
    assert cache.lens.tolist() == [20, 0]


# ---- keys and values into their slots -----------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,hkv,d,page,token_major", [
    (1, 1, 8, 16, False), (7, 2, 64, 16, True), (300, 5, 80, 48, False), (1000, 8, 128, 128, True),
    (33, 3, 512, 32, False), (5000, 2, 64, 16, False)])
def test_append_equals_indexing(cuda, dtype, T, hkv, d, page, token_major):
    g = torch.Generator(device=cuda).manual_seed(T + d)
    pages = T // page + 7
    cache = P.PagedCache(1, 16, pages, hkv, d, page=page, dtype=dtype, device=cuda, layers=2,
                         token_major=token_major)
    cache.k[1].normal_(generator=g)
    cache.v[1].normal_(generator=g)
    kw, vw = cache.k.clone(), cache.v.clone()
    slots = torch.randperm(pages * page, device=cuda, generator=g)[:T]
    slots[torch.arange(T, device=cuda) % 5 == 3] = -1
    if T > 20:  # outside the pool on the other side
        slots[8], slots[13] = pages * page, 2 ** 62
    qkv = torch.randn(T, (4 + 2 * hkv) * d, device=cuda, generator=g).to(dtype)
    k, v = (qkv[:, (4 + i * hkv) * d:(4 + (i + 1) * hkv) * d].view(T, hkv, d) for i in (0, 1))
    print(dtype, T, hkv, d, page, flush=True)
    cache.append(1, k, v, slots)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            kw[1, s // page, :, s % page] = k[t]
            vw[1, s // page, :, s % page] = v[t]
    assert torch.equal(cache.k, kw) and torch.equal(cache.v, vw)


def test_append_copies_unaligned_rows(cuda):
    """Rows that start off a multiple of 16 bytes are copied first; the pools' own must not."""
    x = torch.randn(5, 2 * 64 + 1, device=cuda).to(torch.float16)
    k = x[:, 1:].view(5, 2, 64)
    cache = P.PagedCache(1, 16, 2, 2, 64, page=16, dtype=torch.float16, device=cuda)
    cache.append(0, k, k, torch.arange(5, device=cuda))
    assert torch.equal(cache.k[0, 0, :, :5], k.transpose(0, 1))
    odd = torch.zeros(2 * 2 * 16 * 64 + 1, device=cuda, dtype=torch.float16)[1:].view(2, 2, 16, 64)
    with pytest.raises(_lib.SSAError, match="16 bytes"):
        P.append_pages(k, k, odd, odd, torch.arange(5, device=cuda))


# ---- attention ----------------------------------------------------------------------------------

def make(dev, dtype, lens, hq, hkv, d, page, token_major=False, seed=0, spread=1.0, extra=0):
    """(q, cache) with the requests' pages scattered over the pool; unused slots hold NaN."""
    g = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages, width = sum(need) + 2, max(max(need), 1) + extra
    cache = P.PagedCache(len(lens), width * page, pages, hkv, d, page=page, dtype=dtype,
                         device=dev, token_major=token_major)
    ids = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    cache.k.fill_(math.nan)
    cache.v.fill_(math.nan)
    at = 0
    for b, n in enumerate(lens):
        cache.table[b, :need[b]] = ids[at:at + need[b]]
        for e in range(need[b]):
            m = min(page, n - e * page)
            pid = int(ids[at + e])
            cache.k[0, pid, :, :m] = torch.randn(hkv, m, d, device=dev, generator=g).to(dtype)
            cache.v[0, pid, :, :m] = torch.randn(hkv, m, d, device=dev, generator=g).to(dtype)
        at += need[b]
    cache.lens.copy_(int32(lens, dev))
    q = (torch.randn(len(lens), hq, d, device=dev, generator=g) * spread).to(dtype)
    return q, cache


def check_attend(cache, q, scale=None, window=0, **kw):
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    out, lse = cache.attend(0, q, scale=scale, window=window, return_lse=True, **kw)
    torch.cuda.synchronize()
    want, wlse, tol, ltol = U.attend(q, cache.k[0], cache.v[0], cache.table, cache.lens, scale,
                                     window)
    U.close(out, want, tol)
    U.close(lse, wlse, ltol)
    return out, lse


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513, 1000]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page,token_major", [
    (14, 2, 64, 128, False), (4, 4, 64, 16, True), (32, 8, 128, 16, True), (20, 1, 128, 64, False),
    (10, 5, 80, 48, False), (8, 4, 256, 32, True), (3, 1, 8, 16, False), (33, 1, 96, 80, False),
    (6, 2, 512, 64, False), (2, 2, 192, 16, True), (2, 1, 328, 16, False), (16, 1, 40, 256, False)])
def test_attend_at_every_edge(cuda, dtype, hq, hkv, d, page, token_major):
    q, cache = make(cuda, dtype, EDGES, hq, hkv, d, page, token_major, seed=d, spread=2.0, extra=1)
    for window in (0, 1, 16, 33, 200):
        print(dtype, hq, hkv, d, page, window, flush=True)
        check_attend(cache, q, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,hq,hkv,d,page", [
    ([20000], 14, 2, 64, 128), ([9001, 3, 0, 30000, 1, 700], 8, 2, 128, 16),
    ([1], 4, 4, 64, 16), ([0, 0, 0], 4, 2, 64, 16), ([40000], 2, 1, 512, 64),
    ([12345, 12345], 24, 1, 256, 48)])
def test_attend_long_and_uneven(cuda, dtype, lens, hq, hkv, d, page):
    print(dtype, lens, hq, hkv, d, page, flush=True)
    q, cache = make(cuda, dtype, lens, hq, hkv, d, page, seed=1, spread=2.0)
    check_attend(cache, q)
    check_attend(cache, q, window=5000)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(17, 1, 64), (32, 1, 128), (66, 2, 128), (100, 2, 72)])
def test_attend_many_heads_on_one_key_head(cuda, dtype, hq, hkv, d):
    """More than 16 query heads a key head, with room for more keys than the caches hold (a wide table)
    and without: the two ways to serve them."""
    lens = [1, 33, 0, 2500, 700, 128]
    page = 256
    q, cache = make(cuda, dtype, lens, hq, hkv, d, page, seed=hq)
    narrow = cache.table
    wide = torch.full((6, (1 << 28) // (6 * page * d * hkv)), -1, device=cuda, dtype=torch.int32)
    wide[:, :narrow.shape[1]] = narrow
    for table in (narrow, wide):
        cache.table = table
        for window in (0, 100):
            print(dtype, hq, hkv, d, table.shape[1], window, flush=True)
            check_attend(cache, q, window=window)
    x = torch.randn(6, 2 * hkv * d, device=cuda).to(dtype)
    k_new, v_new = (x[:, i * hkv * d:(i + 1) * hkv * d].view(6, hkv, d) for i in (0, 1))
    out = cache.step(0, q, k_new, v_new)
    want, _, tol, _ = U.attend(q, cache.k[0], cache.v[0], narrow, cache.lens, 1 / math.sqrt(d))
    U.close(out, want, tol)
    assert torch.equal(cache.k[0, int(narrow[3, 9]), :, 2499 % page], k_new[3])


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_many_requests(cuda, dtype):
    rng = random.Random(2)
    lens = [rng.choice([0, 1, rng.randrange(1, 60), rng.randrange(1, 400)]) for _ in range(700)]
    q, cache = make(cuda, dtype, lens, 4, 2, 64, 16, seed=3)
    check_attend(cache, q)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page,token_major", [(14, 2, 64, 128, False),
                                                       (8, 8, 80, 16, True), (40, 2, 128, 48, False),
                                                       (4, 2, 512, 16, False)])
def test_step_stores_the_newest_token_and_attends_it(cuda, dtype, hq, hkv, d, page, token_major):
    q, cache = make(cuda, dtype, EDGES + [5000], hq, hkv, d, page, token_major, seed=5)
    B = len(EDGES) + 1
    x = torch.randn(B, 2 * hkv * d, device=cuda).to(dtype)
    k_new, v_new = (x[:, i * hkv * d:(i + 1) * hkv * d].view(B, hkv, d) for i in (0, 1))
    kw, vw = cache.k.clone(), cache.v.clone()
    for b, n in enumerate(EDGES + [5000]):
        if n:
            pid = int(cache.table[b, (n - 1) // page])
            kw[0, pid, :, (n - 1) % page] = k_new[b]
            vw[0, pid, :, (n - 1) % page] = v_new[b]
    print(dtype, hq, hkv, d, page, flush=True)
    for window in (0, 1, 40):
        out, lse = cache.step(0, q, k_new, v_new, window=window, return_lse=True)
        torch.cuda.synchronize()
        assert torch.equal(cache.k.view(torch.uint8), kw.view(torch.uint8))
        assert torch.equal(cache.v.view(torch.uint8), vw.view(torch.uint8))
        want, wlse, tol, ltol = U.attend(q, cache.k[0], cache.v[0], cache.table, cache.lens,
                                         1 / math.sqrt(d), window)
        U.close(out, want, tol)
        U.close(lse, wlse, ltol)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_scores_of_every_size(cuda, dtype):
    """Large scores: one key carries the row, or keys that grow along the row move the maximum at every
    step; a scale of zero or below."""
    lens = [1, 40, 3000]
    for d, page in ((64, 16), (128, 64), (512, 32)):
        q, cache = make(cuda, dtype, lens, 4, 2, d, page, seed=d, spread=30.0)
        print(dtype, d, page, flush=True)
        check_attend(cache, q)
        check_attend(cache, q, scale=0.0)
        check_attend(cache, q, scale=-0.1)
        for b, n in enumerate(lens):
            for e in range(-(-n // page)):
                cache.k[0, int(cache.table[b, e])] *= 0.02 * (e + 1)
        check_attend(cache, q)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256, 512])
def test_attend_infinities_and_nan(cuda, dtype, d):
    """What the formula gives: a key that scores -inf counts for nothing, an attended infinite value
    makes its column infinite, a NaN key its whole row NaN; all keys at -inf: 0 / 0."""
    lens = [70, 70, 70, 70, 2000]
    q, cache = make(cuda, dtype, lens, 2, 1, d, 16, seed=9)
    q = q.abs() + 1
    at = lambda b, j: (int(cache.table[b, j // 16]), 0, j % 16)  # noqa: E731
    for b, j in ((0, 69), (0, 3), (0, 40), (4, 1999), (4, 0), (4, 700)):
        cache.k[0][at(b, j)] = -math.inf
    for b, j, x in ((1, 69, math.inf), (1, 20, -math.inf), (4, 1998, math.inf)):
        cache.v[0][at(b, j)][1 + (x < 0)] = x
    cache.k[0][at(2, 68)][0] = math.nan
    for j in range(70):
        cache.k[0][at(3, j)] = -math.inf
    out, lse = cache.attend(0, q, return_lse=True)
    torch.cuda.synchronize()
    o = out.double().cpu()
    assert o[2].isnan().all() and lse[2].isnan().all()
    assert o[3].isnan().all() and (lse[3] == -math.inf).all()
    assert (o[1, :, 1] == math.inf).all() and (o[1, :, 2] == -math.inf).all()
    assert (o[4, :, 1] == math.inf).all()
    cols = torch.tensor([c for c in range(d) if c not in (1, 2)])
    # keys at -inf: the reference over the other keys
    for b in (0, 1, 4):
        n = lens[b]
        k, v = U.gather(cache.k[0], cache.table[b], n)[0], U.gather(cache.v[0], cache.table[b], n)[0]
        s = (q[b].double().cpu() @ torch.where(k.isinf(), 0.0, k).T) / math.sqrt(d)
        s[:, k.isinf().any(1)] = -math.inf
        want = torch.softmax(s, 1) @ v[:, cols]
        assert (o[b][:, cols] - want).abs().max() < 2e-2
        assert (lse[b].double().cpu() - torch.logsumexp(s, 1)).abs().max() < 1e-3


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,d", [(2, 64), (20, 64), (2, 128), (20, 128), (2, 256), (2, 512)])
def test_attend_infinite_values_far_below_the_maximum(cuda, dtype, hq, d):
    """A value that is infinite makes its column infinite however small its key's weight: the score lies
    `gap` below the row's largest, up to 2^-37 of it in fp16 and 2^-120 in the others (a weight below 2^-126
    is zero in fp32, below 2^-38 in fp16). The other columns hold ones: 1, off by the additions of up to 40
    terms of three parts (2 u each, u = 2^-24), 40 u for the denominator's, 8 u for joins and division, 4 u
    for a weight's parts (300 u in all), and half a step of the type."""
    gaps = [0.5, 6.0, 13.0, 17.0, 19.0, 21.0, 23.0, 25.0]
    gaps += [25.6] if dtype == torch.float16 else [30.0, 50.0, 70.0, 83.0]
    page, n = 16, 40
    cache = P.PagedCache(len(gaps), 4000, 3 * len(gaps), 1, d, page=page, dtype=dtype, device=cuda)
    cache.resize(int32([n] * len(gaps), cuda), n * len(gaps))
    q = torch.zeros(len(gaps), hq, d, device=cuda, dtype=dtype)
    q[:, :, 0] = 1.0
    cache.v.fill_(1.0)
    at = lambda b, j: (0, int(cache.table[b, j // page]), 0, j % page)  # noqa: E731
    for b, gap in enumerate(gaps):
        for j in range(n):
            cache.k[at(b, j)][0] = -gap
        for j in (3, 37):  # the largest score is 0
            cache.k[at(b, j)][0] = 0.0
        cache.v[at(b, 5)][1] = math.inf
        cache.v[at(b, 20)][2] = -math.inf
        cache.v[at(b, 39)][d - 1] = math.inf
    out = cache.attend(0, q, scale=1.0).double().cpu()
    for b, gap in enumerate(gaps):
        print(dtype, hq, d, gap, flush=True)
        assert (out[b, :, 1] == math.inf).all() and (out[b, :, 2] == -math.inf).all()
        assert (out[b, :, d - 1] == math.inf).all()
        cols = [c for c in range(d) if c not in (1, 2, d - 1)]
        assert (out[b][:, cols] - 1).abs().max() <= 300 * 2.0**-24 + torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 512])
def test_attend_infinite_keys_per_head(cuda, dtype, d):
    """Keys that score -inf for one head and +inf for another, all through the first tiles: the first
    head's row is that of its other keys, the second's NaN."""
    lens = [96, 3000]
    q, cache = make(cuda, dtype, lens, 2, 1, d, 16, seed=11)
    q = q.abs() + 1
    q[:, 1] *= -1
    for b, n in enumerate(lens):
        for j in range(n - 30):
            cache.k[0][int(cache.table[b, j // 16]), 0, j % 16, 0] = -math.inf
    out, lse = cache.attend(0, q, return_lse=True)
    torch.cuda.synchronize()
    assert out[:, 1].isnan().all() and lse[:, 1].isnan().all()
    for b, n in enumerate(lens):
        k, v = (U.gather(x[0], cache.table[b], n)[0, n - 30:] for x in (cache.k, cache.v))
        s = (k @ q[b, 0].double().cpu()) / math.sqrt(d)
        assert (out[b, 0].double().cpu() - torch.softmax(s, 0) @ v).abs().max() < 2e-2
        assert abs(float(lse[b, 0]) - float(torch.logsumexp(s, 0))) < 1e-3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d,width,token_major", [
    (4, 4, 64, 1, False), (2, 1, 128, 1, False), (4, 2, 256, 1, False), (2, 2, 512, 1, False),
    (20, 1, 64, 2000, False), (20, 1, 128, 2000, False), (4, 4, 64, 2000, True),
    (4, 4, 128, 2000, True), (4, 2, 80, 300, False)])
def test_attend_weights_keep_their_bits(cuda, dtype, hq, hkv, d, width, token_major):
    """Outputs round as fp32 weights make them round. Three keys a request, a score the product of two
    16-bit numbers below 1 (exact), so that little but the weights' own bits is off, u = 2^-24:
      a weight    2 u |score| for the scale in log2 units, 0.7 u |exponent| for its difference from the
                  maximum (up to 3, in fp16 17 with the shift by 14), 2 u for exp2: 7 u, in fp16 16 u;
                  its parts: bf16 three of 8 bits, 2 u at most for the last one's rounding; fp16 two
                  of 11, 4 u, and 2^-38: 9 u, in fp16 21 u
      numerator   three terms of up to three parts, 2 u each: 18 u, and 4 u for the joins' factors
      quotient    3 u for the denominator's sum, 4 u for its joins, 2 u for division and product
    with the weights' counted for numerator and denominator: 18 + 31 = 49 u, in fp16 42 + 31 = 73 u, times
    A = sum w |v| / sum w. A weight of 16 bits (2^-16 of it off) left 0.2 % of the outputs outside."""
    B, page, u = 256, 16, 2.0**-24
    g = torch.Generator(device=cuda).manual_seed(d + hq)
    cache = P.PagedCache(B, width * page, B, hkv, d, page=page, dtype=dtype, device=cuda,
                         token_major=token_major)
    cache.table[:, 0] = torch.randperm(B, device=cuda, generator=g).to(torch.int32)
    cache.lens.fill_(3)
    rows = cache.table[:, 0].long()
    q = torch.zeros(B, hq, d, device=cuda, dtype=dtype)
    q[..., 0] = (torch.rand(B, hq, device=cuda, generator=g) * 2 - 1).to(dtype)
    k = (torch.rand(B, hkv, 3, device=cuda, generator=g) * 2 - 1).to(dtype)
    v = torch.randn(B, hkv, 3, d, device=cuda, generator=g).to(dtype)
    cache.k[0, rows, :, :3, 0] = k
    cache.v[0, rows, :, :3] = v
    out = cache.attend(0, q, scale=1.0)
    s = q[..., 0].double().view(B, hkv, -1, 1) * k.double()[:, :, None]  # (B, hkv, group, 3)
    w = torch.softmax(s, 3)[..., None]
    v = v.double()[:, :, None]
    want, size = ((w * x).sum(3).view(B, hq, d) for x in (v, v.abs()))
    # and u of the value, as the bounds below pass through fp32 on their way to the type
    t = size * (49 if dtype == torch.bfloat16 else 73) * u + want.abs() * 2 * u
    wrong = (out < (want - t).to(dtype)) | (out > (want + t).to(dtype))
    assert int(wrong.sum()) == 0, f"{int(wrong.sum())} of {wrong.numel()}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attend_subnormal_values(cuda, dtype):
    """Keys and values below the type's smallest normal number count as what they are."""
    q, cache = make(cuda, dtype, [50, 700], 4, 2, 64, 16, seed=12)
    tiny = torch.finfo(dtype).tiny
    cache.v.mul_(tiny / 4)
    cache.k.mul_(tiny / 4)
    assert 0 < float(cache.v[cache.v > 0].min()) < tiny
    check_attend(cache, q, scale=1.0 / tiny if dtype == torch.float16 else 1.0)


@pytest.mark.parametrize("d,chain", [(64, 32), (128, 32), (256, 64), (512, 128)])
def test_attend_adds_fp32_products_in_chains(cuda, d, chain):
    """fp32 products are added in chains shorter than the head: one of 2^24 hides the products of 1 in
    its own chain only (2^24 + 1 rounds back), the others' sum counts. Key 0 has the ones and key 1 has
    none, so its weight is 1 / (1 + exp(-(d - 1) 2^-17)), of slope 1/4: off by the chain's chain - 1
    products, 2 for joining the chains and 2 for the two scores of 185 in log2 units (half of 2^-16
    each), in units of 2^-17, over 4. One chain would lose all d - 1."""
    q, cache = make(cuda, torch.float32, [2], 2, 1, d, 16)
    q.fill_(1.0)
    page = int(cache.table[0, 0])
    cache.k[0, page, 0, :2] = 0.0
    cache.k[0, page, 0, :2, 0] = 2.0**24
    cache.k[0, page, 0, 0, 1:] = 1.0
    cache.v[0, page, 0, 0] = 1.0
    cache.v[0, page, 0, 1] = 0.0
    out = cache.attend(0, q, scale=2.0**-17)
    want = 1 / (1 + math.exp(-(d - 1) * 2.0**-17))
    tol = (chain - 1 + 4) * 2.0**-17 / 4
    assert tol < (want - 0.5) * 0.6
    assert float((out.double() - want).abs().max()) <= tol


@pytest.mark.parametrize("B", [63, 64, 65, 129])
def test_attend_batch_sizes(cuda, B):
    rng = random.Random(B)
    lens = [rng.choice([0, 1, 500, rng.randrange(1, 3000)]) for _ in range(B)]
    q, cache = make(cuda, torch.bfloat16, lens, 2, 1, 64, 16, seed=B)
    check_attend(cache, q)
    check_attend(cache, q, window=600)


def test_attend_bad_lengths_and_pages_give_nan(cuda):
    """A length outside the table, a page id outside the pool: NaN for that row, nothing stored, the
    other rows as they were."""
    lens = [100, 50, 200, 33, 64]
    q, cache = make(cuda, torch.bfloat16, lens, 4, 2, 64, 16, seed=2)
    good = cache.attend(0, q)
    k_new = torch.randn(5, 2, 64, device=cuda).to(torch.bfloat16)
    table, lens_ok = cache.table.clone(), cache.lens.clone()
    cap = cache.table.shape[1] * 16
    for b, n in ((0, -1), (1, cap + 1), (2, 2 ** 31 - 1), (3, -2 ** 31)):
        cache.lens.copy_(lens_ok)
        cache.lens[b] = n
        out, lse = cache.attend(0, q, return_lse=True)
        assert out[b].isnan().all() and lse[b].isnan().all()
        rest = [r for r in range(5) if r != b]
        U.close(out[rest], good[rest].double().cpu(), good[rest].double().cpu().abs() * 2 ** -7)
        held = cache.k.clone()
        cache.lens[rest] = 0
        cache.step(0, q, k_new, k_new)
        assert torch.equal(cache.k.view(torch.int16), held.view(torch.int16))
    cache.lens.copy_(lens_ok)
    for b, e, pid in ((0, 6, -1), (2, 0, cache.k.shape[1]), (4, 3, 2 ** 31 - 1), (3, 1, -2 ** 31)):
        cache.table.copy_(table)
        cache.table[b, e] = pid
        out, lse = cache.attend(0, q, return_lse=True)
        assert out[b].isnan().all() and lse[b].isnan().all()
        rest = [r for r in range(5) if r != b]
        assert not out[rest].isnan().any()
    # a bad page that the window leaves out does not matter
    cache.table.copy_(table)
    cache.table[2, 0] = -1
    assert not cache.attend(0, q, window=100).isnan().any()


def test_attend_repeats_bit_for_bit(cuda):
    lens = [5000, 17, 0, 12000, 900]
    for dtype in DTYPES:
        q, cache = make(cuda, dtype, lens, 8, 2, 128, 16, seed=6)
        first = cache.attend(0, q, return_lse=True)
        for _ in range(5):
            again = cache.attend(0, q, return_lse=True)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_attend_layouts_and_shared_pages(cuda):
    """Strided queries, a strided output, a column slice of a wider table, requests that share their
    first pages."""
    lens = [300, 310, 64]
    q, cache = make(cuda, torch.float16, lens, 8, 2, 64, 16, seed=8, extra=3)
    cache.table[1, :10] = cache.table[0, :10]
    wide = torch.zeros(3, 8, 3 * 64, device=cuda, dtype=torch.float16)
    wide[..., 64:128] = q
    q2 = wide[..., 64:128]
    out = torch.full((3, 8, 128), 7.0, device=cuda, dtype=torch.float16)
    cache.table = cache.table[:, :20]
    o = cache.attend(0, q2, out=out[..., 64:])
    assert o.data_ptr() == out[..., 64:].data_ptr() and (out[..., :64] == 7).all()
    want, _, tol, _ = U.attend(q, cache.k[0], cache.v[0], cache.table, cache.lens, 0.125)
    U.close(out[..., 64:], want, tol)
    U.close(cache.attend(0, q2.transpose(0, 1).contiguous().transpose(0, 1)), want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (2, 1, 128), (20, 1, 128), (2, 1, 256)])
def test_attend_more_than_the_caches_hold(cuda, dtype, hq, hkv, d):
    """Calls that read past the last-level cache load with another hint: the requests share their pages,
    so that the pool is small."""
    n = 12000
    row = 2 * n * hkv * d * (4 if dtype == torch.float32 else 2)
    B = (200 << 20) // row + 1
    q, cache = make(cuda, dtype, [n], hq, hkv, d, 16, seed=d, spread=2.0)
    q = torch.cat([q * (1 + b % 3) * 0.5 for b in range(B)]).to(dtype)
    cache.table = cache.table.expand(B, -1).contiguous()
    cache.lens = int32([n - b % 40 for b in range(B)], cuda)
    print(dtype, hq, hkv, d, B, flush=True)
    pick = list(range(0, B, max(1, B // 6)))
    for window in (0, n - 100):
        out, lse = cache.attend(0, q, window=window, return_lse=True)
        torch.cuda.synchronize()
        want, wlse, tol, ltol = U.attend(q[pick], cache.k[0], cache.v[0], cache.table[pick],
                                         cache.lens[pick], 1 / math.sqrt(d), window)
        U.close(out[pick], want, tol)
        U.close(lse[pick], wlse, ltol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,d,page", [(32, 8, 128, 16), (4, 4, 64, 48), (16, 8, 80, 16),
                                           (16, 16, 40, 256)])
def test_attend_heads_side_by_side(cuda, dtype, hq, hkv, d, page):
    """Token-major pools with room for many keys: a wave serves a key head of its own."""
    lens = EDGES + [3000, 129]
    q, cache = make(cuda, dtype, lens, hq, hkv, d, page, token_major=True, seed=d, spread=2.0)
    B = len(lens)
    wide = torch.full((B, (1 << 25) // (B * page * d * hkv) + 200), -1, device=cuda,
                      dtype=torch.int32)
    wide[:, :cache.table.shape[1]] = cache.table
    cache.table = wide
    for window in (0, 20, 2500):
        print(dtype, hq, hkv, d, page, window, flush=True)
        check_attend(cache, q, window=window)
    x = torch.randn(B, 2 * hkv * d, device=cuda).to(dtype)
    k_new, v_new = (x[:, i * hkv * d:(i + 1) * hkv * d].view(B, hkv, d) for i in (0, 1))
    check_attend(cache, q, k_new=k_new, v_new=v_new)
    for b, n in enumerate(lens):
        if n:
            at = int(cache.table[b, (n - 1) // page]), slice(None), (n - 1) % page
            assert torch.equal(cache.k[0][at], k_new[b]) and torch.equal(cache.v[0][at], v_new[b])
    cache.table = cache.table.clone()
    cache.table[B - 2, 3] = -1  # a bad page: this row and no other
    out = cache.attend(0, q)
    assert out[B - 2].isnan().all() and not out[[b for b in range(B) if b != B - 2]].isnan().any()


def test_attend_wide_batch_of_short_windows(cuda):
    """The one-launch form with that hint: many (request, key head) pairs, a window of 1,000 keys."""
    q, cache = make(cuda, torch.float16, [1500], 8, 8, 128, 64, seed=2)
    B = 128
    q = torch.cat([q * (1 + b % 3) * 0.5 for b in range(B)])
    cache.table = cache.table.expand(B, -1).contiguous()
    cache.lens = int32([1500 - 7 * b for b in range(B)], cuda)
    out = cache.attend(0, q, window=1000)
    pick = [0, 1, 63, 100, 127]
    want, _, tol, _ = U.attend(q[pick], cache.k[0], cache.v[0], cache.table[pick],
                               cache.lens[pick], 1 / math.sqrt(128), 1000)
    U.close(out[pick], want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_at_the_longest_lengths(cuda, dtype):
    """Positions up to 2^31 - 17, the last a table row can hold, through a window (every page but the last
    is the same)."""
    page, d = 16, 8
    cap = 2 ** 31 - 16
    g = torch.Generator(device=cuda).manual_seed(1)
    k, v = (torch.randn(2, 1, page, d, device=cuda, generator=g).to(dtype) for _ in range(2))
    table = torch.zeros(1, cap // page, device=cuda, dtype=torch.int32)
    q = torch.randn(1, 2, d, device=cuda, generator=g).to(dtype)
    new = torch.randn(1, 1, d, device=cuda, generator=g).to(dtype)
    for n, window in ((cap, 40), (cap - 1, 1), (cap - 15, 200), (cap - 16, 17), (cap - 17, 3000)):
        table[0, (n - 1) // page] = 1
        out, lse = P.attend_pages(q, k, v, table, int32([n], cuda), window=window, k_new=new,
                                  v_new=new, return_lse=True)
        torch.cuda.synchronize()
        table[0, (n - 1) // page] = 0
        assert torch.equal(k[1, 0, (n - 1) % page], new[0, 0])
        # the same keys at the start of a short row: n and its stand-in agree modulo the page
        m = window + 32 - (window - n) % page
        assert (m - n) % page == 0
        short = torch.zeros(1, m // page + 2, dtype=torch.int32)
        short[0, (m - 1) // page] = 1
        want, wlse, tol, ltol = U.attend(q, k, v, short, int32([m], "cpu"), 1 / math.sqrt(d),
                                         window)
        U.close(out, want, tol)
        U.close(lse, wlse, ltol)
    # all 2^31 - 16 keys, of equal weight: the mean of the page's values
    q.zero_()
    out = P.attend_pages(q, k, v, table, int32([cap], cuda))
    mean = v[0, 0].double().mean(0)
    assert (out[0].double() - mean).abs().max() < 2e-2
    bad = P.attend_pages(q, k, v, table, int32([cap + 1], cuda))
    assert bad.isnan().all()


def test_pool_beyond_32_bit_offsets(cuda):
    """Pages whose elements lie past 2^32 bytes and 2^31 elements into the pool."""
    page, d, hkv = 256, 512, 2
    pages = 2 ** 31 // (page * d * hkv) + 300
    k = torch.empty(pages, hkv, page, d, device=cuda, dtype=torch.bfloat16)
    v = torch.empty_like(k)
    table = int32([[pages - 1, 3, pages - 5]], cuda)
    for pid in (pages - 1, 3, pages - 5):
        k[pid].normal_()
        v[pid].normal_()
    lens = int32([600], cuda)
    q = torch.randn(1, 4, d, device=cuda).to(torch.bfloat16)
    new = torch.randn(1, hkv, d, device=cuda).to(torch.bfloat16)
    out = P.attend_pages(q, k, v, table, lens, k_new=new, v_new=new)
    assert torch.equal(k[pages - 5, :, 599 % page], new[0])
    want, _, tol, _ = U.attend(q, k, v, table, lens, 1 / math.sqrt(d))
    U.close(out, want, tol)
    slot = torch.tensor([(pages - 1) * page + 7], device=cuda)
    P.append_pages(new, new, k, v, slot)
    assert torch.equal(v[pages - 1, :, 7], new[0])


# ---- the run of them ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("token_major", [False, True])
def test_prompts_then_steps_then_ends(cuda, dtype, token_major):
    """Two layers: prompts admitted and appended, decode steps, a request ended and its pages taken by
    another -- every step's attention against each request's own contiguous keys and values."""
    hq, hkv, d, page, layers = 6, 2, 64, 16, 2
    g = torch.Generator(device=cuda).manual_seed(1)
    cache = P.PagedCache(4, 400, 44, hkv, d, page=page, layers=layers, dtype=dtype, device=cuda,
                         token_major=token_major)
    own = [[([], []) for _ in range(4)] for _ in range(layers)]
    lens = [0, 0, 0, 0]

    def extend(r, add, lay, k, v):
        cu = r.cu.tolist()
        for b in range(4):
            own[lay][b][0].append(k[cu[b]:cu[b + 1]].double().cpu())
            own[lay][b][1].append(v[cu[b]:cu[b + 1]].double().cpu())
            assert cu[b + 1] - cu[b] == add[b]

    def grow(add):
        for b in range(4):
            lens[b] += add[b]
        r = cache.resize(int32(lens, cuda), sum(add) + 3)
        cache.check()
        return r

    def prompts(add):
        r = grow(add)
        for lay in range(layers):
            k, v = (torch.randn(sum(add) + 3, hkv, d, device=cuda, generator=g).to(dtype)
                    for _ in range(2))
            cache.append(lay, k, v, r.slots)
            extend(r, add, lay, k, v)

    def step():
        add = [int(n > 0) for n in lens]
        grow(add)
        for lay in range(layers):
            q = torch.randn(4, hq, d, device=cuda, generator=g).to(dtype)
            kn, vn = (torch.randn(4, hkv, d, device=cuda, generator=g).to(dtype)
                      for _ in range(2))
            out = cache.step(lay, q, kn, vn)
            for b in range(4):
                if not lens[b]:
                    assert (out[b] == 0).all()
                    continue
                own[lay][b][0].append(kn[b:b + 1].double().cpu())
                own[lay][b][1].append(vn[b:b + 1].double().cpu())
                # the request's own keys and values as one long page
                k, v = (torch.cat(own[lay][b][i]).transpose(0, 1)[None] for i in (0, 1))
                assert k.shape[2] == lens[b]
                want, _, tol, _ = U.attend(q[b:b + 1], k, v, torch.tensor([[0]]),
                                           torch.tensor([lens[b]]), 1 / math.sqrt(d))
                U.close(out[b:b + 1], want, tol)

    prompts([33, 0, 200, 1])
    for _ in range(3):
        step()
    lens[2] = 0  # ends: its pages serve the next prompt
    cache.resize(int32(lens, cuda), 0)
    cache.check()
    for lay in range(layers):
        own[lay][2] = ([], [])
    prompts([0, 380, 0, 16])
    for _ in range(17):
        step()


def test_requests_that_share_a_prefix(cuda):
    """A prefix of two pages held by three requests, as resize_pages describes: they grow on pages of their
    own, attend the shared ones, end one by one, and every page is free exactly once at the end."""
    page, hkv, d = 16, 2, 64
    g = torch.Generator(device=cuda).manual_seed(2)
    cache = P.PagedCache(3, 200, 14, hkv, d, page=page, dtype=torch.float16, device=cuda)
    x = torch.randn(32, hkv, d, device=cuda, generator=g).to(torch.float16)
    r = cache.resize(int32([32, 0, 0], cuda), 32)
    cache.append(0, x, x, r.slots)
    for b in (1, 2):  # the caller's part
        cache.table[b, :2] = cache.table[0, :2]
        cache.lens[b] = 32
    y = torch.randn(40, hkv, d, device=cuda, generator=g).to(torch.float16)
    r = cache.resize(int32([37, 50, 32 + 17], cuda), 40)
    cache.check()
    cache.append(0, y, y, r.slots)
    q = torch.randn(3, 4, d, device=cuda, generator=g).to(torch.float16)
    new = torch.randn(3, hkv, d, device=cuda, generator=g).to(torch.float16)
    cache.resize(cache.lens + 1, 3)
    shared = cache.table[0, :2].tolist()
    out = cache.step(0, q, new, new)
    cu = [0, 5, 23, 40]
    for b in range(3):
        own = torch.cat([x, y[cu[b]:cu[b + 1]], new[b:b + 1]]).transpose(0, 1)[None]
        want, _, tol, _ = U.attend(q[b:b + 1], own, own, torch.tensor([[0]]),
                                   torch.tensor([own.shape[2]]), 1 / math.sqrt(d))
        U.close(out[b:b + 1], want, tol)
    for b in (1, 0):
        new_lens = cache.lens.clone()
        new_lens[b] = 32  # its own pages back
        cache.resize(new_lens, 0)
        cache.check()
        cache.table[b, :2] = -1  # the caller's part again
        cache.lens[b] = 0
    held = cache.table[2, :4].tolist()
    assert held[:2] == shared and cache.nfree.item() == 10
    assert sorted(cache.free[:10].tolist() + held) == list(range(14))
    cache.resize(torch.zeros_like(cache.lens), 0)  # the last holder
    cache.check()
    assert sorted(cache.free.tolist()) == list(range(14)) and (cache.table == -1).all()


def test_refused_resize_stores_nothing(cuda):
    """After a resize that did not fit, step and append leave the cache as it is and the rows are NaN."""
    cache = P.PagedCache(3, 100, 6, 2, 64, page=16, dtype=torch.float16, device=cuda)
    x = torch.randn(60, 2, 64, device=cuda).to(torch.float16)
    q = torch.randn(3, 4, 64, device=cuda).to(torch.float16)
    r = cache.resize(int32([40, 16, 0], cuda), 56)
    cache.append(0, x[:56], x[:56], r.slots)
    good = cache.attend(0, q)
    held = cache.k.clone(), cache.v.clone()
    r = cache.resize(cache.lens + int32([1, 1, 33], cuda), 60)  # 1 + 3 pages, 2 are free
    assert r.status.item() == 2
    cache.append(0, x, x, r.slots)
    out, lse = cache.step(0, q, x[:3], x[:3], return_lse=True)
    assert out.isnan().all() and lse.isnan().all()
    assert cache.attend(0, q, window=20).isnan().all()
    assert torch.equal(cache.k, held[0]) and torch.equal(cache.v, held[1])
    cache.resize(cache.lens.clone(), 0)
    assert torch.equal(cache.attend(0, q), good) and (good[2] == 0).all()


def test_captured_step_replayed(cuda):
    """resize, step and attend captured in one graph and replayed with eager work between: each replay
    grows every live request by a token, as the eager cache beside it does."""
    dtype, hq, hkv, d, page = torch.bfloat16, 14, 2, 64, 16
    lens = [300, 0, 47, 5000]
    q, a = make(cuda, dtype, lens, hq, hkv, d, page, seed=3, extra=2)
    _, b = make(cuda, dtype, lens, hq, hkv, d, page, seed=3, extra=2)
    pages = a.k.shape[1]
    for c in (a, b):  # spare pages at the pool's end
        c.k, c.v = (torch.cat([x, x.new_zeros(1, 8, hkv, page, d)], 1) for x in (c.k, c.v))
        c.free = torch.arange(pages, pages + 8, device=cuda, dtype=torch.int32)
        c.free = torch.cat([c.free, c.free.new_zeros(pages)])
        c.nfree.fill_(8)
    grow = int32([1, 0, 1, 1], cuda)
    k_new = torch.randn(4, hkv, d, device=cuda).to(dtype)
    v_new = torch.randn(4, hkv, d, device=cuda).to(dtype)
    out, lse, r = torch.empty_like(q), None, None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new = a.lens + grow
        r = a.resize(new, 4)
        a.step(0, q, k_new, v_new, out=out)
        lse = a.attend(0, q, window=64, return_lse=True)[1]
    for rep in range(40):
        k_new.normal_()
        v_new.normal_()
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        rb = b.resize(b.lens + grow, 4)
        want = b.step(0, q, k_new, v_new)
        wlse = b.attend(0, q, window=64, return_lse=True)[1]
        assert r.status.item() == rb.status.item() == 0, rep
        assert torch.equal(r.slots, rb.slots) and torch.equal(a.table, b.table), rep
        assert torch.equal(out, want) and torch.equal(lse, wlse), rep
        assert torch.equal(a.lens, b.lens) and torch.equal(a.free, b.free)
        torch.empty(1 << 20, device=cuda).normal_().sum().item()


def test_captured_step_between_eager_resizes(cuda):
    """step alone captured, resizes run eagerly between its replays with other small tensors made where
    an earlier status lay: each replay equals the eager cache beside it, a refused resize's replay stores
    nothing and gives NaN, and the next that fits serves again."""
    hq, hkv, d, page = 4, 2, 64, 16
    a, b = (P.PagedCache(3, 200, 12, hkv, d, page=page, dtype=torch.float16, device=cuda)
            for _ in range(2))
    x = torch.randn(60, hkv, d, device=cuda).to(torch.float16)
    q = torch.randn(3, hq, d, device=cuda).to(torch.float16)
    kn, vn = (torch.randn(3, hkv, d, device=cuda).to(torch.float16) for _ in range(2))
    for c in (a, b):
        r = c.resize(int32([40, 0, 20], cuda), 60)
        c.append(0, x, x, r.slots)
    one = int32([1, 0, 1], cuda)
    a.resize(a.lens + one, 2)
    b.resize(b.lens + one, 2)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(0, q, kn, vn, out=out)
    graph.replay()
    assert torch.equal(out, b.step(0, q, kn, vn))
    kept = []
    for rep in range(12):
        grow = int32([1, 500, 1] if rep % 4 == 2 else [1, 0, 1], cuda)  # 500: past the table
        for c in (a, b):
            r = c.resize(c.lens + grow, 600)
            assert r.status.item() == (-1 if rep % 4 == 2 else 0)
            if rep % 2:
                kept.append(r)  # its status is kept as well as dropped
        junk = [torch.full((n,), 7, device=cuda, dtype=torch.int32) for n in (1, 1, 1, 3, 60, 128)]
        for t in (q, kn, vn):
            t.normal_()
        held = a.k.clone(), a.v.clone()
        graph.replay()
        torch.cuda.synchronize()
        want = b.step(0, q, kn, vn)
        if rep % 4 == 2:
            assert out.isnan().all() and want.isnan().all(), rep
            assert torch.equal(a.k, held[0]) and torch.equal(a.v, held[1]), rep
            with pytest.raises(RuntimeError, match="does not fit the table"):
                a.check()
        else:
            assert torch.equal(out, want) and not out.isnan().any(), rep
            assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v), rep
            a.check()
        del junk


def test_captured_resize_refused_on_replay(cuda):
    """A captured resize replayed after an eager one: its refusal is what check, an eager step and an eager
    attend go by, and the next eager resize that fits ends it."""
    cache = P.PagedCache(2, 100, 5, 2, 64, page=16, dtype=torch.bfloat16, device=cuda)
    x = torch.randn(40, 2, 64, device=cuda).to(torch.bfloat16)
    q = torch.randn(2, 4, 64, device=cuda).to(torch.bfloat16)
    grow = int32([1, 1], cuda)
    r = cache.resize(int32([20, 20], cuda), 40)
    cache.append(0, x, x, r.slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = cache.resize(cache.lens + grow, 60)
    for rep in range(3):
        cache.resize(int32([20, 20], cuda), 0)
        cache.check()
        good = cache.attend(0, q)
        grow.fill_(1)
        graph.replay()
        torch.empty(1 << 20, device=cuda).normal_().sum().item()
        cache.check()
        assert cache.lens.tolist() == [21, 21] and not cache.attend(0, q).isnan().any()
        cache.resize(int32([20, 20], cuda), 0)
        grow.fill_(28)  # two pages more, one is free
        held = cache.k.clone(), cache.v.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert inside.status.item() == 1 and cache.lens.tolist() == [20, 20], rep
        with pytest.raises(RuntimeError, match="1 pages lacking"):
            cache.check()
        assert cache.step(0, q, x[:2], x[:2]).isnan().all() and cache.attend(0, q).isnan().all()
        assert torch.equal(cache.k, held[0]) and torch.equal(cache.v, held[1]), rep
        cache.resize(cache.lens.clone(), 0)
        cache.check()
        assert torch.equal(cache.attend(0, q), good), rep


def test_two_graphs_with_one_memory_pool(cuda):
    """Two captured attentions whose workspaces may share memory, replayed in turn."""
    q, a = make(cuda, torch.float16, [9000, 3], 8, 2, 128, 16, seed=3)
    q2, b = make(cuda, torch.float16, [40, 7000, 600], 8, 2, 128, 16, seed=4)
    want, want2 = a.attend(0, q), b.attend(0, q2)
    pool = torch.cuda.graph_pool_handle()
    outs, graphs = [torch.empty_like(q), torch.empty_like(q2)], []
    for c, x, o in ((a, q, outs[0]), (b, q2, outs[1])):
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            c.attend(0, x, out=o)
    for _ in range(4):
        for o in outs:
            o.zero_()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)


def test_other_streams(cuda):
    q, cache = make(cuda, torch.bfloat16, [7000, 50], 8, 2, 64, 16, seed=3)
    want = cache.attend(0, q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(cache.attend(0, q))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_compiled_step_equals_eager(cuda):
    q, a = make(cuda, torch.bfloat16, [100, 33], 4, 2, 64, 16, seed=3)
    _, b = make(cuda, torch.bfloat16, [100, 33], 4, 2, 64, 16, seed=3)
    x = torch.randn(2, 2, 64, device=cuda).to(torch.bfloat16)

    def f(c, q, x):
        P.append_pages(x, x, c["k"], c["v"], c["slots"])
        o = P.attend_pages(q, c["k"], c["v"], c["table"], c["lens"], k_new=x, v_new=x, window=50)
        return o + P.attend_pages(q, c["k"], c["v"], c["table"], c["lens"])

    slots = torch.tensor([int(a.table[0, 0]) * 16 + 3, -1], device=cuda)
    args = [dict(k=c.k[0], v=c.v[0], table=c.table, lens=c.lens, slots=slots) for c in (a, b)]
    def resize(c, new):
        return P.resize_pages(c["lens"], new, c["table"], c["free"], c["nfree"], 16, 3)

    want = f(args[0], q, x)
    got = torch.compile(f, backend="aot_eager")(args[1], q, x)
    assert torch.equal(got, want) and torch.equal(a.k.view(torch.int16), b.k.view(torch.int16))
    state = [dict(lens=c.lens, table=c.table, free=c.free, nfree=c.nfree.fill_(0)) for c in (a, b)]
    r = resize(state[0], int32([99, 35], cuda))
    rc = torch.compile(resize, backend="aot_eager")(state[1], int32([99, 35], cuda))
    assert r.status.item() == 0 and all(torch.equal(x, y) for x, y in zip(r, rc))
    assert all(torch.equal(state[0][x], state[1][x]) for x in state[0])


def test_compiled_cache_equals_eager(cuda):
    """PagedCache's own calls traced: a step that grows every request, one that is refused (the status kept
    in place, nothing stored) and one into a given Resized."""
    lens = [100, 33, 0]
    q, a = make(cuda, torch.float16, lens, 4, 2, 64, 16, seed=4)
    _, b = make(cuda, torch.float16, lens, 4, 2, 64, 16, seed=4)
    spare = set(range(a.k.shape[1])) - set(a.table.flatten().tolist())
    for c in (a, b):
        c.free[:len(spare)] = int32(sorted(spare), cuda)
        c.nfree.fill_(len(spare))
    x = torch.randn(3, 2, 64, device=cuda).to(torch.float16)

    def step(c, grow, x, out):
        r = c.resize(c.lens + grow, 4, out)
        return r, c.step(0, q, x, x, window=50)

    held = b.status.data_ptr()
    compiled = torch.compile(step, backend="aot_eager")
    out = [None, None]
    for i, grow in enumerate(([1, 1, 0], [0, 5, 0], [1, 1, 1], [1, 1, 0])):
        grow = int32(grow, cuda)
        r, want = step(a, grow, x, out[0])
        rc, got = compiled(b, grow, x, out[1])
        assert r.status.item() == rc.status.item() == b.status.item() == (-2 if i == 1 else 0)
        assert b.status.data_ptr() == held and all(torch.equal(s, t) for s, t in zip(r, rc))
        assert torch.equal(got.isnan(), want.isnan()) and want.isnan().all() == (i == 1)
        assert torch.equal(got.nan_to_num(), want.nan_to_num())
        assert torch.equal(a.lens, b.lens) and torch.equal(a.table, b.table)
        assert torch.equal(a.k.view(torch.int16), b.k.view(torch.int16))
        out = [r, rc] if i == 2 else [None, None]


# ---- refusals -----------------------------------------------------------------------------------

def test_arguments_are_refused(cuda):
    q, c = make(cuda, torch.bfloat16, [20, 5], 4, 2, 64, 16)
    k, v, table, lens = c.k[0], c.v[0], c.table, c.lens
    new = torch.zeros(2, 2, 64, device=cuda, dtype=torch.bfloat16)
    A = P.attend_pages
    bad = [
        (TypeError, lambda: A(q.float(), k, v, table, lens)),
        (TypeError, lambda: A(q, k, v.float(), table, lens)),
        (TypeError, lambda: A(q, k, v, table.long(), lens)),
        (TypeError, lambda: A(q, k, v, table, lens.long())),
        (ValueError, lambda: A(q[:1], k, v, table, lens)),
        (ValueError, lambda: A(q[..., :32], k, v, table, lens)),
        (ValueError, lambda: A(q, k, v[:1], table, lens)),
        (ValueError, lambda: A(q, k, v, table.t().contiguous().t(), lens)),
        (ValueError, lambda: A(q, k, v, table, lens[:1])),
        (ValueError, lambda: A(q, k, v, table, lens, k_new=new)),
        (ValueError, lambda: A(q, k, v, table, lens, k_new=new, v_new=new[:, :1])),
        (TypeError, lambda: A(q, k, v, table, lens, k_new=new, v_new=new.float())),
        (ValueError, lambda: A(q, k, v, table, lens, out=torch.empty_like(q)[:1])),
        (ValueError, lambda: A(q, k, v, table, lens, out=torch.empty_like(q.float()))),
        (ValueError, lambda: A(q, k, v, table, lens, out=torch.empty_like(q[:1]).expand_as(q))),
        (ValueError, lambda: A(q, k[:, :1].expand_as(k), v, table, lens, k_new=new, v_new=new)),
        (TypeError, lambda: A(q, k, v, table, lens, status=lens[:1].long())),
        (ValueError, lambda: A(q, k, v, table, lens, status=lens)),
        (ValueError, lambda: P.append_pages(new, new, k, v[:1].expand_as(v), lens.long())),
        (ValueError, lambda: P.resize_pages(lens, lens, table[:1].expand_as(table), c.free, c.nfree,
                                            16, 0)),
        (_lib.SSAError, lambda: A(q, k, v, table, lens, window=-1)),
        (_lib.SSAError, lambda: A(q[:, :3].contiguous(), k, v, table, lens)),
        (_lib.SSAError, lambda: A(q, k[:, :, :8], v[:, :, :8], table, lens)),
        (RuntimeError, lambda: A(q.cpu(), k, v, table, lens)),
        (RuntimeError, lambda: A(q, k, v, table.cpu(), lens)),
        (TypeError, lambda: P.append_pages(new.float(), new, k, v, lens.long())),
        (ValueError, lambda: P.append_pages(new[:1], new, k, v, lens.long())),
        (ValueError, lambda: P.append_pages(new, new, k, v, lens)),
        (TypeError, lambda: P.resize_pages(lens.long(), lens, table, c.free, c.nfree, 16, 0)),
        (ValueError, lambda: P.resize_pages(lens[:1], lens, table, c.free, c.nfree, 16, 0)),
        (ValueError, lambda: P.resize_pages(lens, lens, table, c.free, c.nfree, 16, -1)),
        (_lib.SSAError, lambda: P.resize_pages(lens, lens, table, c.free, c.nfree, 24, 0)),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail(f"case {i} was not refused")
    odd = torch.zeros(2, 4, 60, device=cuda, dtype=torch.bfloat16)  # rows that no copy can align
    pool = torch.zeros(3, 2, 16, 60, device=cuda, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="head dim 60"):
        A(odd, pool, pool, table, lens)
    with pytest.raises(ValueError, match="head dim 60"):
        P.append_pages(odd[:, :2], odd[:, :2], pool, pool, lens.long())
    assert A(q[:0], k, v, table[:0], lens[:0]).shape == (0, 4, 64)
    P.append_pages(new[:0], new[:0], k, v, lens[:0].long())
