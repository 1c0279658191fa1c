"""A paged key-value cache: many requests of different lengths in one pool of pages.

    resize_pages(lens, new_lens, table, free, nfree, page, tokens)   pages taken and given back
    append_pages(k, v, kpool, vpool, slots)                          new tokens into their slots
    attend_pages(q, kpool, vpool, table, lens, ...)                  one new token per request
    PagedCache                                                       the state these work on

A pool is a (pages, Hkv, page, d) tensor (any strides with a contiguous last dimension, so a
token-major (pages, page, Hkv, d) pool is passed transposed); token j of request b lies in page
table[b, j // page] at slot j % page, and its slot number is table[b, j // page] * page + j % page.
The lengths live on the device: every call is asynchronous on the current stream of the tensors'
device, works under graph capture and synchronises with nothing. What a call can only find out on
the device (a length beyond the table, too few free pages, a page id outside the pool) is answered
there: resize_pages changes nothing and writes a status, append_pages skips the row, attend_pages
returns NaN for the row; no call follows a bad length or page id.

attend_pages is the dense counterpart of attend_rows and dense_decode (ivf_decode) for batches of
requests: the decode of the layers that a routed model leaves dense or sliding. It is not
differentiable. The reference has no paged cache.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch

from . import _lib

RESIZE_ERRORS = {-1: "a length, the free count or the pool does not fit the table",
                 -2: "more new tokens than slots"}


class Resized(NamedTuple):
    """What resize_pages returns: of every new token (request by request, in order) its slot and
    position, the first token of each request (B + 1 offsets), and the status (1,)."""
    slots: torch.Tensor   # (tokens,) int64, -1 past the last new token
    pos: torch.Tensor     # (tokens,) int32, 0 past the last new token
    cu: torch.Tensor      # (B + 1,) int32
    status: torch.Tensor  # (1,) int32: 0, the number of pages lacking, or a key of RESIZE_ERRORS


def _launch(name, t, *args):
    """Calls an entry point on the current stream of t's device."""
    index = t.device.index
    if index == torch.cuda.current_device():
        _lib.call(name, *args, _lib.stream_of(t))
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args, _lib.stream_of(t))


def _one_device(first, *others):
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            _lib.require_device(first, *others)
            raise ValueError(f"tensors on {first.device} and {t.device}")
    if index < 0:
        _lib.require_device(first)


# The checks of shapes, strides and types depend on nothing else, and a serving loop makes the same
# call again and again: what they give is kept by those (22 us a call on the host without, 12 with).

def _int32(name, shape, stride, dtype, want):
    if dtype != torch.int32:
        raise TypeError(f"{name} is {dtype}, expected torch.int32")
    if tuple(shape) != want or (len(want) and want[0] > 1 and stride != (1,)):
        raise ValueError(f"{name} must be a contiguous {want} tensor, got {tuple(shape)}")


def _table(shape, stride, dtype):
    """(B, W, elements a row)"""
    if dtype != torch.int32:
        raise TypeError(f"table is {dtype}, expected torch.int32")
    if len(shape) != 2 or shape[1] > 1 and stride[1] != 1:
        raise ValueError("table must be (B, W) with a contiguous last dimension")
    B, W = shape
    return B, W, stride[0] if B > 1 else W


def _meta(t):
    return (t.shape, t.stride(), t.dtype)


def _pools(k, v):
    (kshape, kstride, kdtype), (vshape, vstride, vdtype) = k, v
    if len(kshape) != 4 or kshape != vshape:
        raise ValueError(f"kpool and vpool must share a (pages, Hkv, page, d) shape, got "
                         f"{tuple(kshape)} and {tuple(vshape)}")
    if kdtype != vdtype:
        raise TypeError("kpool and vpool must share a dtype")
    if kstride[3] != 1 or vstride[3] != 1:
        raise ValueError("the head dimension must be contiguous")
    if kshape[3] % 8 or kshape[3] > 512:
        raise ValueError(f"head dim {kshape[3]}: a multiple of 8 up to 512 is wanted")
    return kshape


def _written(name, meta):
    """Refuses a broadcast tensor (a stride of 0) where rows are written."""
    if any(n > 1 and st == 0 for n, st in zip(*meta[:2])):
        raise ValueError(f"{name} is written and must not be broadcast")


def _rows16(meta):
    """Whether rows (the last dimension) start at multiples of 16 bytes, given an aligned base."""
    shape, stride, dtype = meta
    vec = 4 if dtype == torch.float32 else 8
    return stride[-1] == 1 and all(s % vec == 0 for s in stride[:-1])


def _given(out, tokens, B):
    """Refuses an `out` of resize_pages that is not what a call of these sizes returns."""
    if out.slots.dtype != torch.int64 or out.slots.shape != (tokens,) \
            or not out.slots.is_contiguous():
        raise ValueError(f"out.slots must be a contiguous ({tokens},) int64 tensor")
    for name, n in (("pos", tokens), ("cu", B + 1), ("status", 1)):
        _int32("out." + name, *_meta(getattr(out, name)), (n,))


@functools.lru_cache(maxsize=1024)
def _resize_plan(lens, new_lens, table, free, nfree):
    B, W, row = _table(*table)
    _int32("lens", *lens, (B,))
    _int32("new_lens", *new_lens, (B,))
    _int32("nfree", *nfree, (1,))
    _int32("free", *free, (free[0].numel(),))
    _written("table", table)
    return B, W, row, free[0].numel()


@functools.lru_cache(maxsize=1024)
def _append_plan(k, v, kpool, vpool, slots):
    """(constants of the call, whether k or v needs a copy)"""
    pages, hkv, page, d = _pools(kpool, vpool)
    dtype = kpool[2]
    if k[2] != dtype or v[2] != dtype:
        raise TypeError(f"k is {k[2]} and v {v[2]}, the cache holds {dtype}")
    if slots[2] != torch.int64 or len(slots[0]) != 1 or slots[0][0] > 1 and slots[1] != (1,):
        raise ValueError("slots must be a contiguous (T,) int64 tensor")
    _written("kpool", kpool)
    _written("vpool", vpool)
    T = slots[0][0]
    if k[0] != (T, hkv, d) or v[0] != (T, hkv, d):
        raise ValueError(f"k and v must be ({T}, {hkv}, {d}), got {tuple(k[0])} and "
                         f"{tuple(v[0])}")
    strides = _lib.i64_array((*k[1][:2], *v[1][:2], *kpool[1][:3], *vpool[1][:3]))
    return (_lib.dtype_code(dtype), T, hkv, d, pages, page, strides), \
        not (_rows16(k) and _rows16(v))


@functools.lru_cache(maxsize=1024)
def _attend_plan(q, kpool, vpool, table, lens, out, k_new, v_new, window):
    """(sizes of the call, table's, strides, workspace bytes, whether an input needs a copy)"""
    pages, hkv, page, d = _pools(kpool, vpool)
    dtype = kpool[2]
    if len(q[0]) != 3 or q[0][2] != d:
        raise ValueError(f"q must be (B, Hq, {d}), got {tuple(q[0])}")
    B, hq, _ = q[0]
    if q[2] != dtype:
        raise TypeError(f"q is {q[2]}, the cache holds {dtype}")
    copy = not _rows16(q)
    new = (0, 0, 0, 0)
    if k_new is not None:
        if k_new[2] != dtype or v_new[2] != dtype:
            raise TypeError(f"k_new is {k_new[2]} and v_new {v_new[2]}, the cache holds {dtype}")
        if k_new[0] != (B, hkv, d) or v_new[0] != (B, hkv, d):
            raise ValueError(f"k_new and v_new must be ({B}, {hkv}, {d})")
        _written("kpool", kpool)
        _written("vpool", vpool)
        copy = copy or not (_rows16(k_new) and _rows16(v_new))
        new = (*k_new[1][:2], *v_new[1][:2])
    rows, W, row = _table(*table)
    if rows != B:
        raise ValueError(f"table has {rows} rows for {B} requests")
    _int32("lens", *lens, (B,))
    to = (hq * d, d)
    if out is not None:
        if out[2] != dtype or out[0] != (B, hq, d) or not _rows16(out):
            raise ValueError(f"out must be a ({B}, {hq}, {d}) {dtype} tensor with rows of 16-byte "
                             "pieces")
        _written("out", out)
        to = out[1][:2]
    strides = _lib.i64_array((*q[1][:2], *kpool[1][:3], *vpool[1][:3], *to, *new))
    ws_bytes = _lib.query("ssa_paged_attend_workspace_size", B, hq, hkv, d, W, page, window)
    return (_lib.dtype_code(dtype), B, hq, hkv, d, pages, page), (row, W), strides, ws_bytes, copy


def resize_pages(lens: torch.Tensor, new_lens: torch.Tensor, table: torch.Tensor,
                 free: torch.Tensor, nfree: torch.Tensor, page: int, tokens: int,
                 out: Resized | None = None) -> Resized:
    """Brings the requests to new lengths, on the device.

    lens, new_lens (B,) int32; table (B, W) int32; free (pages,) int32, a stack of the free page
    ids of which the first nfree (1,) int32 are valid. lens, table, free and nfree are updated: a
    request that grows takes pages from the top of the stack (requests in order), one that shrinks
    gives its last pages back (their table entries become -1), lens becomes new_lens. Pages given
    back in a call can be taken from the next call on. Growing and then shrinking back restores
    table and free exactly.

    tokens: room for the new tokens (at least the sum of the growths; more is padding). Returns a
    Resized; `out` takes an earlier one of the same sizes to write into. All or nothing: if the
    growth does not fit the free pages or `tokens`, or a length its table row, nothing changes, all
    slots are -1 and status says why.

    A page given back is free: nothing counts how many rows list it. Pages that requests share (a common
    prefix, set by the caller in their table rows and lengths; attend_pages reads them as any others) go
    back once, by the last request that holds them. Any other is brought to the length of its shared
    pages here, which gives back its own, and taken out by the caller: its row to -1, its length to 0."""
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError(f"tokens={tokens}")
    if torch.compiler.is_compiling():
        from . import torch_ops as T
        if out is not None:
            _given(out, tokens, lens.shape[0])
        r = T.paged_resize(lens, new_lens, table, free, nfree, int(page), tokens)
        if out is not None:
            for to, x in zip(out, r):
                to.copy_(x)
            return out
        return Resized(*r)
    _one_device(lens, new_lens, table, free, nfree)
    B, W, row, pages = _resize_plan(_meta(lens), _meta(new_lens), _meta(table), _meta(free),
                                    _meta(nfree))
    if out is None:
        dev = lens.device
        out = Resized(torch.empty(tokens, device=dev, dtype=torch.int64),
                      torch.empty(tokens, device=dev, dtype=torch.int32),
                      torch.empty(B + 1, device=dev, dtype=torch.int32),
                      torch.empty(1, device=dev, dtype=torch.int32))
    else:
        _one_device(lens, *out)
        _given(out, tokens, B)
    if B == 0:  # no requests, no new tokens
        out.slots.fill_(-1)
        for x in out[1:]:
            x.zero_()
        return out
    _launch("ssa_paged_resize", lens, lens.data_ptr(), new_lens.data_ptr(), table.data_ptr(),
            row, B, W, int(page), free.data_ptr(), pages, nfree.data_ptr(),
            out.slots.data_ptr() if tokens else None, out.pos.data_ptr() if tokens else None,
            tokens, out.cu.data_ptr(), out.status.data_ptr())
    return out


def append_pages(k: torch.Tensor, v: torch.Tensor, kpool: torch.Tensor, vpool: torch.Tensor,
                 slots: torch.Tensor) -> None:
    """Stores the tokens' keys and values k, v (T, Hkv, d) into the pools at slots (T,) int64
    (slot = page id * page + offset; rows whose slot lies outside the pool, as -1, are skipped).
    The slots of a call must be distinct."""
    if torch.compiler.is_compiling():
        from . import torch_ops as T
        T.paged_append(k, v, kpool, vpool, slots)
    else:
        _append_pages_impl(k, v, kpool, vpool, slots)


def _append_pages_impl(k, v, kpool, vpool, slots):
    _one_device(kpool, vpool, k, v, slots)
    sizes, copy = _append_plan(_meta(k), _meta(v), _meta(kpool), _meta(vpool), _meta(slots))
    kp, vp = k.data_ptr(), v.data_ptr()
    if copy or (kp | vp) & 15:
        return _append_pages_impl(*(_own(t) for t in (k, v)), kpool, vpool, slots)
    if sizes[1]:
        _launch("ssa_paged_append", kpool, kp, vp, kpool.data_ptr(), vpool.data_ptr(), *sizes,
                slots.data_ptr())


def _own(t):
    """A contiguous copy (allocations start at multiples of 16 bytes)."""
    return t.clone(memory_format=torch.contiguous_format)


def attend_pages(q: torch.Tensor, kpool: torch.Tensor, vpool: torch.Tensor, table: torch.Tensor,
                 lens: torch.Tensor, k_new: torch.Tensor | None = None,
                 v_new: torch.Tensor | None = None, scale: float | None = None, window: int = 0,
                 return_lse: bool = False, out: torch.Tensor | None = None,
                 status: torch.Tensor | None = None):
    """Attention of one token per request over its cached keys: q (B, Hq, d), out (B, Hq, d) in
    q's dtype; request b attends its keys j < lens[b] (with a window, the last `window` of them),
    softmax(scale * q.k) in fp32, query head h reading key head h // (Hq / Hkv). A request of
    length 0 (an idle row of the batch) gets zeros and a log-sum of -inf.

    k_new, v_new (B, Hkv, d): the token at position lens[b] - 1, stored into the cache by this
    call and attended with the rest (the page that holds that position must be the request's own;
    earlier pages may be shared between requests). status (1,) int32: a resize's; if that resize was
    refused, nothing is stored (lens[b] - 1 is then an older token's position) and every row is NaN.
    return_lse: also the natural log of each row's sum of exponentials (B, Hq) fp32, with which
    partial results can be joined. Under torch.compile `out` costs a copy."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new come together")
    if torch.compiler.is_compiling():
        from . import torch_ops as T
        if out is not None and (out.dtype != q.dtype or out.shape != q.shape):
            raise ValueError(f"out must be a {tuple(q.shape)} {q.dtype} tensor")
        if k_new is None:
            o, lse = T.paged_attend(q, kpool, vpool, table, lens, float(scale), int(window),
                                    status)
        else:
            o, lse = T.paged_step(q, kpool, vpool, table, lens, k_new, v_new, float(scale),
                                  int(window), status)
        if out is not None:
            out.copy_(o)
            o = out
        return (o, lse) if return_lse else o
    return _attend_pages_impl(q, kpool, vpool, table, lens, k_new, v_new, scale, window,
                              return_lse, out, status)


def _attend_pages_impl(q, kpool, vpool, table, lens, k_new, v_new, scale, window, return_lse,
                       out=None, status=None):
    _one_device(q, kpool, vpool, table, lens, k_new, v_new, out, status)
    window = int(window)
    sizes, rows, strides, ws_bytes, copy = _attend_plan(
        _meta(q), _meta(kpool), _meta(vpool), _meta(table), _meta(lens),
        None if out is None else _meta(out), None if k_new is None else _meta(k_new),
        None if v_new is None else _meta(v_new), window)
    qp = q.data_ptr()
    kp, vp = (None, None) if k_new is None else (k_new.data_ptr(), v_new.data_ptr())
    if copy or (qp if kp is None else qp | kp | vp) & 15:
        k_new, v_new = (None if t is None else _own(t) for t in (k_new, v_new))
        return _attend_pages_impl(_own(q), kpool, vpool, table, lens, k_new, v_new, scale, window,
                                  return_lse, out, status)
    _, B, hq, _, d, _, _ = sizes
    dev = q.device
    if out is None:
        out = torch.empty(B, hq, d, device=dev, dtype=q.dtype)
    lse = torch.empty(B, hq, device=dev, dtype=torch.float32) if return_lse else None
    if status is not None:
        _int32("status", *_meta(status), (1,))
    if B:
        ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8) if ws_bytes else None
        _launch("ssa_paged_attend", q, qp, kpool.data_ptr(), vpool.data_ptr(), out.data_ptr(),
                _lib.ptr(lse), *sizes, table.data_ptr(), *rows, lens.data_ptr(), kp, vp, strides,
                float(scale), window, _lib.ptr(status), _lib.ptr(ws), ws_bytes)
    return (out, lse) if return_lse else out


class PagedCache:
    """The keys and values of up to `requests` requests in `pages` pages per layer.

    Every layer has a pool of its own; the table and the lengths are shared by the layers, so a
    step resizes once and then appends and attends layer by layer:

        r = cache.resize(cache.lens + grow, tokens)       # grow (requests,) int32 on the device
        cache.append(layer, k, v, r.slots)                # a prompt's tokens, or
        o = cache.step(layer, q, k_new, v_new)            # one token of every request

    A request ends by a resize to length 0 (one that shares pages: as resize_pages says); q, k_new and
    v_new have a row for every request, idle ones included. After a resize that did not fit, append and step store nothing and attend and step give
    NaN, until a resize fits; `check` raises then (it synchronises; a caller that keeps count of the
    pages need not call it)."""

    def __init__(self, requests, max_len, pages, hkv, d, page=64, layers=1, dtype=torch.bfloat16,
                 device="cuda", token_major=False):
        if min(requests, max_len, pages, hkv, d, page, layers) < 1:
            raise ValueError("PagedCache: sizes must be positive")
        if page % 16 or d % 8 or d > 512:
            raise ValueError(f"PagedCache: pages of a multiple of 16 tokens and head dims of a "
                             f"multiple of 8 up to 512, got page={page}, d={d}")
        _lib.dtype_code(dtype)
        dev = torch.device(device)
        i32 = dict(device=dev, dtype=torch.int32)
        self.page = int(page)
        shape = (layers, pages, page, hkv, d) if token_major else (layers, pages, hkv, page, d)
        pool = torch.zeros(2, *shape, device=dev, dtype=dtype)
        if token_major:
            pool = pool.transpose(3, 4)
        self.k, self.v = pool[0], pool[1]
        self.table = torch.full((requests, -(-max_len // page)), -1, **i32)
        self.lens = torch.zeros(requests, **i32)
        self.free = torch.arange(pages, **i32).flip(0).contiguous()  # page 0 on top
        self.nfree = torch.full((1,), pages, **i32)
        with torch.inference_mode(False):  # torch writes it, inside and outside inference mode
            self.status = torch.zeros(1, **i32)

    @torch.no_grad()
    def resize(self, new_lens: torch.Tensor, tokens: int, out: Resized | None = None) -> Resized:
        """resize_pages on this cache's state. The status that attend, step and check go by is
        the cache's own tensor, like its lengths: a captured call finds the last resize's there,
        whether that one ran eagerly or in a replay."""
        r = resize_pages(self.lens, new_lens, self.table, self.free, self.nfree, self.page,
                         tokens, out)
        # r's own may be written by another cache's resize; added, not copied: a kernel in a graph too
        torch.add(r.status, 0, out=self.status)
        return r

    def check(self) -> None:
        """Raises if the last resize changed nothing because it did not fit. Synchronises."""
        status = int(self.status)
        if status:
            raise RuntimeError("resize: " + RESIZE_ERRORS.get(status, f"{status} pages lacking"))

    @torch.no_grad()
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """append_pages into a layer's pools."""
        append_pages(k, v, self.k[layer], self.v[layer], slots)

    @torch.no_grad()
    def attend(self, layer: int, q: torch.Tensor, **kwargs):
        """attend_pages over a layer's pools (scale, window, return_lse, out as there)."""
        return attend_pages(q, self.k[layer], self.v[layer], self.table, self.lens,
                            status=self.status, **kwargs)

    @torch.no_grad()
    def step(self, layer: int, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
             **kwargs):
        """attend with the newest token of every request stored first."""
        return self.attend(layer, q, k_new=k_new, v_new=v_new, **kwargs)


__all__ = ["resize_pages", "append_pages", "attend_pages", "PagedCache", "Resized"]
