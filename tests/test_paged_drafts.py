"""Drafted tokens and shared pages over the paged cache without a GPU: arguments refused at the C ABI and in
Python, shapes of the registered operators, and the plain restatements that the GPU tests compare with."""
import ctypes
import random

import pytest
import torch

from ssa_amd import _lib
from ssa_amd import paged as P
from tests import drafts_util as D
from tests.test_paged import FAKE, NULL, status

ODD = ctypes.c_void_p((1 << 20) + 8)
INVALID, UNSUPPORTED, SPACE = _lib.SSA_ERR_INVALID, _lib.SSA_ERR_UNSUPPORTED, _lib.SSA_ERR_WORKSPACE


def attend(**kw):
    a = dict(q=FAKE, kpool=FAKE, vpool=FAKE, out=FAKE, lse=NULL, dtype=_lib.BF16, B=2, N=9, Hq=4,
             Hkv=2, d=64, pages=10, page=16, table=FAKE, table_stride=8, W=8, lens=FAKE, cu=FAKE,
             masks=FAKE, pos=FAKE, words=1,
             strides=_lib.i64_array([256, 64, 2048, 1024, 64, 2048, 1024, 64, 256, 64]),
             scale=0.125, window=0, status=NULL, clear=1, ws=FAKE, ws_bytes=1 << 40)
    a.update(kw)
    return status("ssa_paged_attend_drafts", *a.values(), None)


WIDE = dict(W=1000, table_stride=1000)


@pytest.mark.parametrize("change,code", [
    (dict(q=NULL), INVALID), (dict(lens=NULL), INVALID), (dict(cu=NULL), INVALID),
    (dict(masks=NULL), INVALID), (dict(pos=NULL), INVALID), (dict(words=0), INVALID),
    (dict(masks=NULL, pos=NULL), INVALID), (dict(words=33), UNSUPPORTED),
    (dict(words=-1), UNSUPPORTED), (dict(dtype=7), UNSUPPORTED), (dict(d=60), UNSUPPORTED),
    (dict(d=520), UNSUPPORTED), (dict(page=24), UNSUPPORTED), (dict(Hq=3), INVALID),
    (dict(B=0), INVALID), (dict(B=65536), INVALID), (dict(N=0), INVALID), (dict(N=2 ** 31), INVALID),
    (dict(pages=0), INVALID), (dict(W=0), INVALID), (dict(W=9), INVALID),
    (dict(W=2 ** 27, table_stride=2 ** 27), INVALID), (dict(window=-1), INVALID),
    (dict(window=2 ** 31), INVALID), (dict(q=ODD), INVALID), (dict(out=ODD), INVALID),
    (dict(strides=_lib.i64_array([256, 64, 2048, 1024, 60] + [64] * 5)), INVALID),
    (dict(strides=_lib.i64_array([64] * 4 + [-64] + [64] * 5)), INVALID),
    (dict(strides=_lib.i64_array([64] * 4 + [2 ** 24] + [64] * 5)), UNSUPPORTED),
    (dict(strides=_lib.i64_array([64] * 7 + [2 ** 24] + [64] * 2)), UNSUPPORTED),
    (dict(N=2 ** 31 - 1, Hq=64, Hkv=64), UNSUPPORTED),
    (dict(ws_bytes=1000, **WIDE), SPACE), (dict(ws=NULL, **WIDE), SPACE), (dict(ws=ODD, **WIDE), SPACE),
])
def test_attend_refuses(change, code):
    assert attend(**change) == code
    assert b"ssa_paged_attend_drafts" in _lib.lib().ssa_last_error()


def test_masks_refuse():
    f = lambda parents=FAKE, cu=FAKE, B=2, N=9, words=1: status(  # noqa: E731
        "ssa_paged_draft_masks", parents, cu, FAKE, B, N, words, FAKE, FAKE, None)
    assert f(parents=NULL) == INVALID and f(cu=NULL) == INVALID
    assert f(B=0) == INVALID and f(N=-1) == INVALID and f(N=2 ** 31) == INVALID
    assert f(words=0) == UNSUPPORTED and f(words=33) == UNSUPPORTED
    assert f(B=2 ** 30) == UNSUPPORTED
    assert f(parents=NULL, N=0) == _lib.SSA_OK  # nothing to do, nothing launched
    with pytest.raises(ValueError, match="most=0"):
        P.draft_masks(None, None, None, 0)
    with pytest.raises(ValueError, match="most=1025"):
        P.draft_masks(None, None, None, 1025)


S8 = _lib.i64_array([20480, 2048, 1024, 64] * 2)


def test_keep_refuses():
    def f(kpool=FAKE, dtype=_lib.F16, layers=1, hkv=2, d=64, pages=10, page=16, st=S8, W=8, B=2,
          path=FAKE, stride=3, width=3, vpool=ctypes.c_void_p(1 << 30)):
        return status("ssa_paged_keep", kpool, vpool, dtype, layers, hkv, d, pages, page, st, FAKE, 8,
                      W, FAKE, FAKE, B, path, stride, width, FAKE, FAKE, None)
    assert f(kpool=NULL) == INVALID and f(path=NULL) == INVALID and f(B=0) == INVALID
    assert f(B=65536) == INVALID and f(layers=0) == INVALID and f(width=-1) == INVALID
    assert f(stride=-3) == INVALID and f(W=9) == INVALID and f(kpool=ODD) == INVALID
    assert f(dtype=5) == UNSUPPORTED and f(d=20) == UNSUPPORTED and f(page=20) == UNSUPPORTED
    assert f(layers=2 ** 30) == UNSUPPORTED and f(layers=2 ** 20, B=65535) == UNSUPPORTED
    assert f(st=_lib.i64_array([64, 64, 64, 60] * 2)) == INVALID
    assert f(vpool=FAKE) == INVALID and b"same memory" in _lib.lib().ssa_last_error()


def test_fork_and_copy_refuse():
    def f(new=FAKE, stride=8, B=2, W=8, page=16, pages=10, ws=FAKE, n=1 << 40):
        return status("ssa_paged_fork", NULL, new, FAKE, FAKE, stride, B, W, page, FAKE, pages,
                      FAKE, FAKE, FAKE, FAKE, FAKE, ws, n, None)
    assert f(new=NULL) == INVALID and f(B=0) == INVALID and f(stride=7) == INVALID
    assert f(pages=0) == INVALID and f(pages=2 ** 31) == INVALID
    assert f(page=17) == UNSUPPORTED and f(W=2 ** 27, stride=2 ** 27) == UNSUPPORTED
    assert f(B=2 ** 30, W=2 ** 13, stride=2 ** 13) == UNSUPPORTED
    assert f(ws=NULL) == SPACE and f(ws=ODD) == SPACE and f(n=100) == SPACE
    assert _lib.query("ssa_paged_fork_workspace_size", 0, 1, 1) == 0

    def c(kpool=FAKE, dtype=_lib.F16, layers=1, d=64, page=16, st=S8, n=3):
        return status("ssa_paged_copy", kpool, FAKE, dtype, layers, 2, d, 10, page, st, FAKE, FAKE,
                      NULL, n, None)
    assert c(kpool=NULL) == INVALID and c(n=-1) == INVALID and c(n=65536) == INVALID
    assert c(layers=0) == INVALID and c(kpool=ODD) == INVALID
    assert c(dtype=5) == UNSUPPORTED and c(d=20) == UNSUPPORTED and c(page=20) == UNSUPPORTED
    assert c(layers=2 ** 30) == UNSUPPORTED
    assert c(n=0) == _lib.SSA_OK


def test_python_refuses(monkeypatch):
    """Shapes and types are refused before anything is launched (on tensors of one device)."""
    monkeypatch.setattr(P, "_one_device", lambda *a: None)
    monkeypatch.setattr(P, "_launch", lambda *a: pytest.fail("launched"))
    i32 = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    pool, q = torch.zeros(9, 2, 16, 64), torch.zeros(5, 4, 64)
    lens, cu, table = i32(3), i32(4), i32(3, 2)
    good = dict(q=q, kpool=pool, vpool=pool, table=table, lens=lens, cu=cu, drafts=None)
    for kw in (dict(q=q[0]), dict(q=q[..., :32]), dict(q=q.half()), dict(lens=lens[:2]),
               dict(cu=lens), dict(cu=cu.long()), dict(table=table.float()),
               dict(drafts=P.Drafts(i32(4, 1), i32(5))), dict(drafts=P.Drafts(i32(5, 1), i32(4))),
               dict(drafts=P.Drafts(i32(5, 33), i32(5))), dict(drafts=P.Drafts(i32(5), i32(5))),
               dict(drafts=P.Drafts(i32(5, 1).long(), i32(5))),
               dict(drafts=P.Drafts(i32(1, 5).t(), i32(5))[:1] + (i32(5).long(),)),
               dict(drafts=P.Drafts(i32(2, 5).t(), i32(5))), dict(vpool=pool[:8]),
               dict(q=q[:1], drafts=P.Drafts(i32(1, 8)[:, ::2], i32(1))),
               dict(out=q.half()), dict(out=q[:4]), dict(out=q[:1].expand(5, 4, 64))):
        with pytest.raises((ValueError, TypeError)):
            P.attend_drafts(**{**good, **kw})
    for parents, c, n in ((i32(5, 1)[:, 0].long(), cu, lens), (i32(5), lens, lens),
                          (i32(5), cu.long(), lens)):
        with pytest.raises((ValueError, TypeError)):
            P.draft_masks(parents, c, n, 5)
    path, layers = i32(3, 2), torch.zeros(2, 9, 2, 16, 64)
    for kw in (dict(path=path.long()), dict(path=path[:2]), dict(path=i32(3)), dict(counts=cu),
               dict(path=i32(2, 3).t()), dict(kpool=layers), dict(kpool=layers[0].half()),
               dict(kpool=layers[0, :1].expand(9, 2, 16, 64)), dict(cu=lens)):
        a = dict(kpool=pool, vpool=pool, table=table, lens=lens, cu=cu, path=path, counts=lens)
        with pytest.raises((ValueError, TypeError)):
            P.keep_drafts(**{**a, **kw})
    for kw in (dict(src=cu), dict(src=lens.long()), dict(new_lens=cu), dict(lens=lens[:2]),
               dict(table=i32(3, 1).expand(3, 2)), dict(nfree=cu), dict(free=i32(2, 9).t())):
        a = dict(src=lens, new_lens=lens, lens=lens, table=table, free=i32(9), nfree=i32(1), page=16)
        with pytest.raises((ValueError, TypeError)):
            P.fork_pages(**{**a, **kw})
    for args in ((cu, lens, None), (lens, lens.long(), None), (lens, lens, cu)):
        with pytest.raises((ValueError, TypeError)):
            P.copy_pages(layers, layers.clone(), *args)
    empty = P.fork_pages(None, i32(0), i32(0), i32(0, 2), i32(9), i32(1), 16)
    assert [x.tolist() for x in empty] == [[], [], [], [0]]


def test_cpu_tensors_raise():
    i = torch.zeros(1, dtype=torch.int32)
    pool, q, cu = torch.zeros(2, 2, 16, 64), torch.zeros(1, 2, 64), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: P.attend_drafts(q, pool, pool, i.view(1, 1), i, cu),
                 lambda: P.draft_masks(i, cu, i, 4),
                 lambda: P.keep_drafts(pool, pool, i.view(1, 1), i, cu, i.view(1, 1), i),
                 lambda: P.fork_pages(i, i, i, i.view(1, 1), i, i, 16),
                 lambda: P.copy_pages(pool, pool, i, i)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_registered_operators_give_shapes():
    import ssa_amd  # noqa: F401  (registers the ops)
    ops = torch.ops.ssa_amd
    m = dict(device="meta")
    i32 = lambda *n: torch.empty(n, dtype=torch.int32, **m)  # noqa: E731
    q = torch.empty(5, 4, 64, dtype=torch.float16, **m)
    pool = torch.empty(9, 2, 16, 64, dtype=torch.float16, **m)
    masks, pos = ops.paged_draft_masks(i32(5), i32(4), i32(3), 40)
    assert masks.shape == (5, 2) and pos.shape == (5,) and masks.dtype == torch.int32
    for a in ((None, None), (masks, pos)):
        out, lse = ops.paged_attend_drafts(q, pool, pool, i32(3, 2), i32(3), i32(4), *a, 0.1, 0, None)
        assert out.shape == q.shape and out.dtype == q.dtype
        assert lse.shape == (5, 4) and lse.dtype == torch.float32
        lse = ops.paged_attend_drafts_into(q, pool, pool, i32(3, 2), i32(3), i32(4), *a, 0.1, 0,
                                           None, torch.empty_like(q))
        assert lse.shape == (5, 4)
    new = ops.paged_keep(pool, pool.clone(), i32(3, 2), i32(3), i32(4), i32(3, 2), i32(3))
    assert new.shape == (3,) and new.dtype == torch.int32
    for src in (None, i32(3)):
        f = ops.paged_fork(src, i32(3), i32(3), i32(3, 2), i32(9), i32(1), 16)
        assert [tuple(x.shape) for x in f] == [(3,), (3,), (3,), (1,)]
    assert ops.paged_copy(pool, pool.clone(), i32(3), i32(3), None) is None


def test_compiled_calls_refuse_what_eager_ones_refuse(monkeypatch):
    monkeypatch.setattr(torch.compiler, "is_compiling", lambda: True)
    m = dict(device="meta")
    i32 = lambda *n: torch.empty(n, dtype=torch.int32, **m)  # noqa: E731
    q = torch.empty(5, 4, 64, dtype=torch.float16, **m)
    pool = torch.empty(9, 2, 16, 64, dtype=torch.float16, **m)
    call = lambda out: P.attend_drafts(q, pool, pool, i32(2, 4), i32(2), i32(3), out=out)  # noqa: E731
    out = torch.empty_like(q)
    assert call(out) is out and call(None).shape == q.shape
    for bad in (q.float(), q[:4], torch.empty(3, 5, 4, 64, dtype=q.dtype, **m)):
        with pytest.raises(ValueError, match="out must be"):
            call(bad)
    with pytest.raises(ValueError, match="most=0"):
        P.draft_masks(i32(5), i32(3), i32(2), 0)


def test_plain_fork_keeps_every_page_once():
    """After any run of resizes and forks a page is free or listed, the last partly filled ones by one
    row each."""
    rng = random.Random(0)
    s = D.ForkState(6, 10, 40, 16)
    for step in range(300):
        if step % 2:
            new = [min(160, n + rng.randrange(40)) for n in s.lens]
            s.resize(new, 2000)
        else:
            src = [rng.randrange(6) for _ in range(6)]
            s.fork(src, [rng.choice([s.lens[a], rng.randrange(s.lens[a] + 1), 0]) for a in src])
        held = [row[:-(-n // 16)] for row, n in zip(s.table, s.lens)]
        assert sorted(set(sum(held, [])) | set(s.free)) == list(range(40))
        assert len(set(s.free)) == len(s.free) and not set(s.free) & set(sum(held, []))
        last = [row[-1] for row, n in zip(held, s.lens) if n % 16]
        assert all(sum(x in row for row in held) == 1 for x in last)


def test_plain_attention_is_the_softmax_of_the_attended_keys():
    """The restatement against a loop over rows, with what is not attended left out."""
    torch.manual_seed(0)
    pool = torch.randn(4, 1, 16, 8)
    table, lens = torch.tensor([[2, 0], [3, -1]]), torch.tensor([21, 9])
    cu, q = torch.tensor([0, 5, 8]), torch.randn(8, 2, 8)
    parents = [-1, 0, 0, -1, 2, -1, 0, 0]
    masks, pos = D.masks_and_pos(parents, [5, 3], [21, 9], 1, 8)
    for window in (0, 3):
        out, lse, _, _ = D.attend(q, pool, pool, table, lens, cu, 0.3, window,
                                  torch.tensor(masks), torch.tensor(pos))
        for row, (b, see) in enumerate([(0, x) for x in D.ancestors(parents[:5])]
                                       + [(1, x) for x in D.ancestors(parents[5:])]):
            ctx = (16, 6)[b]
            keys = [j for j in range(ctx) if not window or j > pos[row] - window]
            keys += [ctx + i for i in see if not window or pos[cu[b] + i] > pos[row] - window]
            k = torch.stack([pool[table[b, j // 16], 0, j % 16] for j in keys]).double()
            for h in range(2):
                s = k @ q[row, h].double() * 0.3
                torch.testing.assert_close(out[row, h], torch.softmax(s, 0) @ k)
                torch.testing.assert_close(lse[row, h], torch.logsumexp(s, 0))


def test_drafts_are_cut_to_fit(tmp_path):
    """csrc/paged_index.h compiled for the host: requests that do not fit are answered there, row tiles
    and items are no more than a call's launch and workspace hold, and every key lies in one item."""
    import shutil
    import subprocess
    from pathlib import Path
    root = Path(__file__).resolve().parents[1]
    cxx = shutil.which("g++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no host compiler")
    exe = tmp_path / "check"
    subprocess.run([cxx, "-std=c++17", "-O1", f"-I{root / 'ssa_amd' / 'csrc'}",
                    str(root / "tests/paged_drafts_check.cpp"), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert res.returncode == 0 and res.stdout.strip() == "ok", res.stdout + res.stderr


def test_weights_that_lack_bits_are_seen():
    """The bound that the GPU's outputs are held to tells weights of all their bits from those of fewer."""
    for dtype, enough in ((torch.bfloat16, 3), (torch.float16, 2)):
        values, want, off = D.cancelling(dtype)
        w = torch.tensor([1.0] + [torch.tensor(-3.0 * D.WEIGHT_SCALE, dtype=torch.float64).exp()] * 3,
                         dtype=torch.float64).float()
        v = torch.tensor(list(values.values()), dtype=torch.float64)
        for parts in range(1, 4):
            got = (D.in_parts(w, dtype, parts) * v).sum() / w.double().sum()
            assert (abs(got - want) <= off) == (parts >= enough), (dtype, parts, got, want, off)


def test_rows_of_offsets():
    assert D.rows_of([0, 6, 25], 20) == (0, [0, 6], [0], 20)
    assert D.rows_of([3, 6, 17], 20) == (3, [0, 3, 14], [0, 1], 17)
    assert D.rows_of([-2, 5, 20], 20) == (5, [0, 15], [1], 20)
    assert D.rows_of([0, 6, 4, 20], 20) == (0, [0], [], 20)
    assert D.rows_of([25, 30], 20) == (0, [0], [], 20) and D.rows_of([-5, -3], 20)[3] == 20


def test_keep_all_refuses_what_keep_refuses():
    def f(name, kpool=FAKE, vpool=ctypes.c_void_p(1 << 30), dtype=_lib.F16, d=64, W=8, B=2, path=FAKE):
        return status(name, kpool, vpool, dtype, 1, 2, d, 10, 16, S8, FAKE, 8, W, FAKE, FAKE, B, path, 3, 3,
                      FAKE, FAKE, None)
    for kw in (dict(kpool=NULL), dict(vpool=FAKE), dict(dtype=5), dict(d=20), dict(W=9), dict(B=0),
               dict(path=NULL)):
        code = f("ssa_paged_keep_all", **kw)
        assert code == f("ssa_paged_keep", **kw) and code in (INVALID, UNSUPPORTED)
    f("ssa_paged_keep_all", W=9)
    assert b"ssa_paged_keep_all" in _lib.lib().ssa_last_error()


def test_outputs_over_inputs_are_refused():
    """Workgroups of a request read what the first of them would overwrite."""
    at = lambda i: ctypes.c_void_p((1 << 32) + 4 * i)  # noqa: E731
    lens, cu, path, counts, table = at(0), at(100), at(200), at(300), at(400)

    def keep(name, new):
        return status(name, FAKE, ctypes.c_void_p(1 << 40), _lib.F16, 1, 2, 64, 10, 16, S8, table, 8, 8, lens,
                      cu, 5, path, 3, 3, counts, new, None)
    for name in ("ssa_paged_keep", "ssa_paged_keep_all"):
        for new in (0, 4, 96, 105, 196, 214, 300, 304, 439):  # 5 ints from there on
            assert keep(name, at(new)) == INVALID, new
            assert b"new_lens lies over an input" in _lib.lib().ssa_last_error()
    parents = at(500)

    def masks(out, pos, words=2):
        return status("ssa_paged_draft_masks", parents, cu, lens, 5, 9, words, out, pos, None)
    far = at(10000)
    for x in (500, 508, 492, 105, 83, 4):
        assert masks(at(x), far) == INVALID, x
    for x in (500, 508, 492, 105, 92, 4):
        assert masks(far, at(x)) == INVALID


def test_work_of_many_requests_is_covered(tmp_path):
    """csrc/paged_index.h compiled for the host: the units per item cover the work of up to 65,535 requests
    whatever the fp32 sum of it loses."""
    import shutil
    import subprocess
    from pathlib import Path
    root = Path(__file__).resolve().parents[1]
    cxx = shutil.which("g++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no host compiler")
    exe = tmp_path / "check"
    subprocess.run([cxx, "-std=c++17", "-O1", f"-I{root / 'ssa_amd' / 'csrc'}",
                    str(root / "tests/paged_drafts_work_check.cpp"), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert res.returncode == 0 and res.stdout.strip() == "ok", res.stdout + res.stderr


@pytest.mark.parametrize("sizes,match", [((65536, 16, 4, 1, 8), "65536 pages"), ((2, 16, 4, 1, 8), None),
                                         ((65535, 16, 4, 1, 8), None)])
def test_a_fork_that_cannot_be_copied_changes_nothing(monkeypatch, sizes, match):
    """The copy's limits are looked at before the table is written."""
    steps = []
    fork = P.Forked(*(torch.zeros(1, dtype=torch.int32) for _ in range(4)))
    monkeypatch.setattr(P, "fork_pages", lambda *a: steps.append("fork") or fork)
    monkeypatch.setattr(P, "copy_pages", lambda *a: steps.append("copy"))
    cache = P.PagedCache(*sizes, page=16, device="cpu")
    if match:
        with pytest.raises(ValueError, match=match):
            cache.fork(None, cache.lens)
        assert steps == []
    else:
        cache.fork(None, cache.lens)
        assert steps == ["fork", "copy"]


@pytest.mark.parametrize("layers,hkv,page,d,dtype", [
    (64, 8, 65536, 256, torch.bfloat16), (64, 8, 65536, 264, torch.bfloat16),
    (65, 8, 65536, 128, torch.float32), (32, 8, 65536, 256, torch.float32), (1 << 13, 1, 65536, 16, torch.float16)])
def test_the_limits_of_a_copy_are_the_entry_points(layers, hkv, page, d, dtype):
    """_copy_limits refuses what ssa_paged_copy refuses, and nothing else (no page is copied)."""
    pool = torch.empty(layers, 1, hkv, page, d, dtype=dtype, device="meta")
    code = status("ssa_paged_copy", FAKE, FAKE, _lib.dtype_code(dtype), layers, hkv, d, 1, page,
                  _lib.i64_array(list(pool.stride()[:4]) * 2), FAKE, FAKE, NULL, 0, None)
    assert code in (_lib.SSA_OK, UNSUPPORTED)
    if code == _lib.SSA_OK:
        P._copy_limits(65535, pool)
    else:
        with pytest.raises(ValueError, match="over all layers"):
            P._copy_limits(1, pool)
    with pytest.raises(ValueError, match="65536 pages"):
        P._copy_limits(65536, pool)
