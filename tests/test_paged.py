"""The paged cache without a GPU: arguments refused at the C ABI, shapes of the registered operators,
and the plain restatement that the GPU tests compare with."""
import ctypes

import pytest
import torch

from ssa_amd import _lib
from ssa_amd import paged as P
from tests import paged_util as U

FAKE = ctypes.c_void_p(1 << 20)  # never dereferenced: validation fails first
NULL = None


def status(name, *args):
    return getattr(_lib.lib(), name)(*args)


def attend(**kw):
    """ssa_paged_attend with one argument changed."""
    a = dict(q=FAKE, kpool=FAKE, vpool=FAKE, out=FAKE, lse=NULL, dtype=_lib.BF16, B=2, Hq=4, Hkv=2,
             d=64, pages=10, page=16, table=FAKE, table_stride=8, W=8, lens=FAKE, k_new=NULL,
             v_new=NULL, strides=_lib.i64_array([256, 64, 2048, 1024, 64, 2048, 1024, 64, 256, 64,
                                                 128, 64, 128, 64]),
             scale=0.125, window=0, status=NULL, ws=FAKE, ws_bytes=1 << 30)
    a.update(kw)
    return status("ssa_paged_attend", *a.values(), None)


@pytest.mark.parametrize("change,code", [
    (dict(q=NULL), _lib.SSA_ERR_INVALID), (dict(lens=NULL), _lib.SSA_ERR_INVALID),
    (dict(table=NULL), _lib.SSA_ERR_INVALID), (dict(k_new=FAKE), _lib.SSA_ERR_INVALID),
    (dict(dtype=7), _lib.SSA_ERR_UNSUPPORTED), (dict(d=60), _lib.SSA_ERR_UNSUPPORTED),
    (dict(d=520), _lib.SSA_ERR_UNSUPPORTED), (dict(page=24), _lib.SSA_ERR_UNSUPPORTED),
    (dict(page=8), _lib.SSA_ERR_UNSUPPORTED), (dict(page=65552), _lib.SSA_ERR_UNSUPPORTED),
    (dict(Hq=3), _lib.SSA_ERR_INVALID), (dict(B=0), _lib.SSA_ERR_INVALID),
    (dict(pages=0), _lib.SSA_ERR_INVALID), (dict(pages=2 ** 31), _lib.SSA_ERR_INVALID),
    (dict(W=0), _lib.SSA_ERR_INVALID), (dict(W=9), _lib.SSA_ERR_INVALID),
    (dict(W=2 ** 27, table_stride=2 ** 27), _lib.SSA_ERR_INVALID),
    (dict(window=-1), _lib.SSA_ERR_INVALID), (dict(window=2 ** 31), _lib.SSA_ERR_INVALID),
    (dict(q=ctypes.c_void_p((1 << 20) + 8)), _lib.SSA_ERR_INVALID),
    (dict(strides=_lib.i64_array([256, 64, 2048, 1024, 60] + [64] * 9)), _lib.SSA_ERR_INVALID),
    (dict(strides=_lib.i64_array([64] * 4 + [2 ** 24] + [64] * 9)), _lib.SSA_ERR_UNSUPPORTED),
    (dict(strides=_lib.i64_array([64] * 7 + [2 ** 24] + [64] * 6)), _lib.SSA_ERR_UNSUPPORTED),
    (dict(strides=_lib.i64_array([64] * 4 + [-64] + [64] * 9)), _lib.SSA_ERR_INVALID),
    (dict(B=65536), _lib.SSA_ERR_INVALID), (dict(Hq=65536, Hkv=1), _lib.SSA_ERR_INVALID),
    (dict(B=65535, W=2 ** 22, table_stride=2 ** 22), _lib.SSA_ERR_UNSUPPORTED),
    (dict(W=1000, table_stride=1000, ws_bytes=1000), _lib.SSA_ERR_WORKSPACE),
    (dict(W=1000, table_stride=1000, ws=NULL), _lib.SSA_ERR_WORKSPACE),
    (dict(W=1000, table_stride=1000, ws=ctypes.c_void_p((1 << 20) + 8)), _lib.SSA_ERR_WORKSPACE),
])
def test_attend_refuses(change, code):
    assert attend(**change) == code
    assert b"ssa_paged_attend" in _lib.lib().ssa_last_error()


def test_launches_past_32_bits_are_refused():
    """A launch counts its threads in 32 bits: calls with more are refused by name, and the largest that
    fits is left to the launch (which fails without a GPU)."""
    if torch.cuda.is_available():
        pytest.skip("would launch")
    wide = dict(B=65535, d=8, W=1, table_stride=1, ws_bytes=1 << 40)
    assert attend(Hq=256, Hkv=256, **wide) == _lib.SSA_ERR_HIP  # 65,535 x 256 workgroups
    assert attend(Hq=257, Hkv=257, **wide) == _lib.SSA_ERR_UNSUPPORTED
    assert b"too many rows" in _lib.lib().ssa_last_error()
    st = _lib.i64_array([0, 0, 0, 0] + [1 << 20] * 6)
    ap = lambda T: status("ssa_paged_append", FAKE, FAKE, FAKE, FAKE, _lib.F32, T, 1,  # noqa: E731
                          512, 10, 16, st, FAKE, None)
    assert ap((1 << 25) - 2) == _lib.SSA_ERR_HIP  # 128 threads a token
    assert ap(1 << 25) == _lib.SSA_ERR_UNSUPPORTED
    assert b"tokens in one call" in _lib.lib().ssa_last_error()


def test_append_and_resize_refuse():
    st = _lib.i64_array([128, 64, 128, 64, 2048, 1024, 64, 2048, 1024, 64])
    ap = lambda k, dt, T, d, page, s=st: status(  # noqa: E731
        "ssa_paged_append", k, FAKE, FAKE, FAKE, dt, T, 2, d, 10, page, s, FAKE, None)
    assert ap(NULL, _lib.F16, 4, 64, 16) == _lib.SSA_ERR_INVALID
    assert ap(FAKE, 9, 4, 64, 16) == _lib.SSA_ERR_UNSUPPORTED
    assert ap(FAKE, _lib.F16, 4, 20, 16) == _lib.SSA_ERR_UNSUPPORTED
    assert ap(FAKE, _lib.F16, 4, 64, 20) == _lib.SSA_ERR_UNSUPPORTED
    assert ap(FAKE, _lib.F16, -1, 64, 16) == _lib.SSA_ERR_INVALID
    assert ap(FAKE, _lib.F16, 4, 64, 16, _lib.i64_array([65] + [64] * 9)) == _lib.SSA_ERR_INVALID
    assert ap(FAKE, _lib.F16, 0, 64, 16) == _lib.SSA_OK  # nothing to store, nothing launched

    def rs(lens=FAKE, stride=8, B=2, W=8, page=16, pages=10, slots=FAKE, T=4):
        return status("ssa_paged_resize", lens, FAKE, FAKE, stride, B, W, page, FAKE, pages, FAKE,
                      slots, NULL, T, FAKE, FAKE, None)
    assert rs(lens=NULL) == _lib.SSA_ERR_INVALID
    assert rs(B=0) == _lib.SSA_ERR_INVALID
    assert rs(stride=7) == _lib.SSA_ERR_INVALID
    assert rs(pages=0) == _lib.SSA_ERR_INVALID
    assert rs(page=17) == _lib.SSA_ERR_UNSUPPORTED
    assert rs(W=2 ** 27, stride=2 ** 27) == _lib.SSA_ERR_UNSUPPORTED
    assert rs(T=-1) == _lib.SSA_ERR_INVALID
    assert rs(slots=NULL) == _lib.SSA_ERR_INVALID


def test_cpu_tensors_raise():
    x = torch.zeros(1, 2, 64)
    pool = torch.zeros(2, 2, 16, 64)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        P.attend_pages(x, pool, pool, i.view(1, 1), i)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        P.append_pages(x, x, pool, pool, i.long())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        P.resize_pages(i, i, i.view(1, 1), i, i, 16, 1)
    for kw in (dict(page=24), dict(d=60), dict(d=520), dict(pages=0), dict(dtype=torch.int8)):
        with pytest.raises((ValueError, TypeError)):
            P.PagedCache(**{**dict(requests=1, max_len=10, pages=2, hkv=1, d=64, device="cpu"),
                            **kw})


def test_cache_keeps_its_tensors(monkeypatch):
    """A captured step holds the addresses of the cache's tensors: resizes write them in place, the
    status among them, and a Resized given to another cache as `out` leaves this one's alone."""
    outcome = []

    def resize(lens, new_lens, table, free, nfree, page, tokens, out=None):
        if out is None:
            out = P.Resized(torch.zeros(tokens, dtype=torch.int64),
                            *(torch.zeros(n, dtype=torch.int32) for n in (tokens, 4, 1)))
        out.status.fill_(outcome.pop(0))
        return out

    monkeypatch.setattr(P, "resize_pages", resize)
    a, b = (P.PagedCache(3, 40, 9, 1, 8, page=16, device="cpu") for _ in range(2))
    state = lambda c: [t.data_ptr() for t in (c.k, c.v, c.lens, c.table, c.free,  # noqa: E731
                                              c.nfree, c.status)]
    held = state(a)
    outcome += [0, 2, 5, -1, 0, 0]
    r = a.resize(a.lens, 5)
    first = a.resize(a.lens, 5)
    assert state(a) == held and a.status.item() == 2 and r.status.item() == 0
    with pytest.raises(RuntimeError, match="2 pages lacking"):
        a.check()
    b.resize(b.lens, 5, out=first)
    assert a.status.item() == 2 and b.status.item() == first.status.item() == 5
    assert a.resize(a.lens, 5, out=r) is r
    assert state(a) == held and a.status.item() == r.status.item() == -1
    b.resize(b.lens, 5)
    a.resize(a.lens, 5)
    assert state(a) == held and a.status.item() == b.status.item() == 0
    a.check()


@pytest.mark.parametrize("made", [False, True])
@pytest.mark.parametrize("used", [False, True])
def test_cache_in_and_out_of_inference_mode(monkeypatch, made, used):
    i32 = lambda n: torch.full((n,), 3, dtype=torch.int32)  # noqa: E731
    monkeypatch.setattr(P, "resize_pages",
                        lambda *a: a[7] or P.Resized(i32(5).long(), i32(5), i32(3), i32(1)))
    with torch.inference_mode(made):
        cache = P.PagedCache(2, 40, 9, 1, 8, page=16, device="cpu")
        given = P.Resized(i32(5).long(), i32(5), i32(3), i32(1))
    with torch.inference_mode(used):
        for out in (None, given):
            cache.status.zero_()
            cache.resize(cache.lens, 5, out)
            assert cache.status.item() == 3


@pytest.mark.parametrize("tokens,given", [(0, False), (3, False), (3, True)])
def test_resize_of_no_requests(monkeypatch, tokens, given):
    """An empty batch is resized as it is appended and attended: nothing changes, every slot is padding."""
    monkeypatch.setattr(P, "_one_device", lambda *a: None)
    monkeypatch.setattr(P, "_launch", lambda *a: pytest.fail("launched"))
    i32 = lambda *n: torch.full(n, 7, dtype=torch.int32)  # noqa: E731
    lens, table, free, nfree = i32(0), i32(0, 4), i32(9), i32(1)
    out = P.Resized(i32(tokens).long(), i32(tokens), i32(1), i32(1)) if given else None
    r = P.resize_pages(lens, lens.clone(), table, free, nfree, 16, tokens, out)
    assert out is None or r is out
    assert r.slots.tolist() == [-1] * tokens and r.pos.tolist() == [0] * tokens
    assert r.cu.tolist() == [0] and r.status.tolist() == [0]
    assert nfree.item() == 7 and (free == 7).all()


def test_another_device_is_made_current(monkeypatch):
    """A call for tensors of a device that is not the current one runs with that device current."""
    from types import SimpleNamespace as NS
    seen = []

    class Device:
        def __init__(self, i):
            self.i = i

        def __enter__(self):
            seen.append(("in", self.i))

        def __exit__(self, *a):
            seen.append(("out", self.i))

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 40 + t.device.index)
    monkeypatch.setattr(_lib, "call", lambda *a: seen.append(a))
    P._launch("x", NS(device=NS(index=0)), 1)
    P._launch("y", NS(device=NS(index=1)), 2)
    assert seen == [("x", 1, 40), ("in", 1), ("y", 2, 41), ("out", 1)]
    a, b = (NS(device=NS(index=i), is_cuda=True, get_device=lambda i=i: i) for i in (0, 1))
    with pytest.raises(ValueError, match="tensors on"):
        P._one_device(a, None, b)


def test_registered_operators_give_shapes():
    import ssa_amd  # noqa: F401  (registers the ops)
    ops = torch.ops.ssa_amd
    m = dict(device="meta")
    q = torch.empty(3, 8, 64, dtype=torch.float16, **m)
    pool = torch.empty(9, 2, 16, 64, dtype=torch.float16, **m)
    new = torch.empty(3, 2, 64, dtype=torch.float16, **m)
    lens = torch.empty(3, dtype=torch.int32, **m)
    table = torch.empty(3, 4, dtype=torch.int32, **m)
    for out, lse in (ops.paged_attend(q, pool, pool, table, lens, 0.1, 0),
                     ops.paged_step(q, pool, pool.clone(), table, lens, new, new, 0.1, 5)):
        assert out.shape == q.shape and out.dtype == q.dtype
        assert lse.shape == (3, 8) and lse.dtype == torch.float32
    free, nfree = torch.empty(9, dtype=torch.int32, **m), torch.empty(1, dtype=torch.int32, **m)
    slots, pos, cu, st = ops.paged_resize(lens, lens.clone(), table, free, nfree, 16, 7)
    assert slots.shape == pos.shape == (7,) and cu.shape == (4,) and st.shape == (1,)
    assert slots.dtype == torch.int64 and pos.dtype == cu.dtype == st.dtype == torch.int32
    assert ops.paged_append(new, new, pool, pool.clone(), slots[:3]) is None


def test_compiled_calls_refuse_what_eager_ones_refuse(monkeypatch):
    """A given `out` of another size or type is refused when traced too: copies into it would broadcast and
    convert."""
    monkeypatch.setattr(torch.compiler, "is_compiling", lambda: True)
    m = dict(device="meta")
    i32 = lambda *n: torch.empty(n, dtype=torch.int32, **m)  # noqa: E731
    q = torch.empty(2, 4, 64, dtype=torch.float16, **m)
    pool = torch.empty(9, 2, 16, 64, dtype=torch.float16, **m)
    lens, table, free, nfree = i32(2), i32(2, 4), i32(9), i32(1)
    resize = lambda n, out: P.resize_pages(lens, lens.clone(), table, free, nfree, 16,  # noqa: E731
                                           n, out)
    good = [torch.empty(1, dtype=torch.int64, **m), i32(1), i32(3), i32(1)]
    assert resize(1, P.Resized(*good)).slots is good[0]
    for i, bad in ((0, torch.empty(5, dtype=torch.int64, **m)), (0, i32(1)), (1, i32(4)),
                   (2, i32(4)), (2, torch.empty(3, **m)), (3, i32(2))):
        with pytest.raises((ValueError, TypeError)):
            resize(1, P.Resized(*good[:i], bad, *good[i + 1:]))
    with pytest.raises(ValueError, match="tokens=-1"):
        resize(-1, None)
    new = torch.empty(2, 2, 64, dtype=torch.float16, **m)
    for kw in ({}, dict(k_new=new, v_new=new)):
        out = torch.empty_like(q)
        assert P.attend_pages(q, pool, pool.clone(), table, lens, out=out, **kw) is out
        for bad in (q.float(), torch.empty(3, 2, 4, 64, dtype=q.dtype, **m)):
            with pytest.raises(ValueError, match="out must be"):
                P.attend_pages(q, pool, pool.clone(), table, lens, out=bad, **kw)
        for k, v in ((new, None), (None, new)):
            with pytest.raises(ValueError, match="come together"):
                P.attend_pages(q, pool, pool.clone(), table, lens, k_new=k, v_new=v)


def test_plain_state_keeps_every_page_once():
    import random
    rng = random.Random(0)
    s = U.PageState(6, 10, 40, 16)
    for _ in range(200):
        new = [rng.randrange(161) if rng.random() < 0.5 else n for n in s.lens]
        s.resize(new, 2000)
        used = [x for row, n in zip(s.table, s.lens) for x in row[:-(-n // 16)]]
        assert sorted(used + s.free) == list(range(40))
        assert all(x == -1 for row, n in zip(s.table, s.lens) for x in row[-(-n // 16):])


def test_items_cover_every_key_once(tmp_path):
    """csrc/paged_index.h compiled for the host: lengths and page tables that do not fit are answered
    there, items cover the attended keys exactly and fit the workspace."""
    import shutil
    import subprocess
    from pathlib import Path
    root = Path(__file__).resolve().parents[1]
    cxx = shutil.which("g++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no host compiler")
    exe = tmp_path / "check"
    subprocess.run([cxx, "-std=c++17", "-O1", f"-I{root / 'ssa_amd' / 'csrc'}",
                    str(root / "tests/paged_index_check.cpp"), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert res.returncode == 0 and res.stdout.strip() == "ok", res.stdout + res.stderr
