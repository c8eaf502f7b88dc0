"""A key/value cache in pages: its layout, the checks of its calls and the native bodies (``csrc/paged.cu``, ``csrc/paged_pieces.cu``).

A cache is two tensors (``PagedKV``) of pages of 16 to 128 tokens; a table says which page each stretch of a sequence is in, so
sequences of any lengths share one pool and may share pages that they only read.  New tokens come as pieces, packed one after another:
rows ``starts[b] .. starts[b + 1]`` are sequence b's, at the positions from ``pos[b]`` on.  Table, starts and positions live on the
device and are never read by the host.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from . import _lib as L
from . import COUNTS
from .kv8 import HEAD_DIMS, MAX_LEN, _bf16, _table
from .logprobs import has_tangent

PAGES = (16, 32, 64, 128)              # tokens of a page
SHIFT = 32.0                           # largest |scale| * head_dim: the kernels' soft-max has this fixed shift, and its smallest weights, exp(-2 * 32), stay normal in fp32
MOST_ROWS = (1 << 31) - 256             # rows of [D] in a cache
MOST_WINDOW = 1 << 24                   # tiles of 128 tokens that hide none of any cache's
# Pieces of up to this many tokens go by tiles of 16 rows, longer ones by tiles of 128: a second tile of 16 reads the keys again.  us by tiles of 16 / of 128, 10 heads of 128, sequences
# of n tokens each: 8 behind up to 1500, n = 8 18.1 / 20.8, 16 21.2 / 21.2, 17 23.2 / 21.2, 64 35.5 / 22.6; 32 behind up to 1500, n = 1 30.0 / 35.8, 16 37.2 / 37.2, 17 48.8 / 36.9,
# 64 97 / 40; 4 behind up to 32768, n = 1 71.7 / 77.5, 16 76.5 / 77.5, 17 134 / 78; one behind 1500, n = 1 11.3 / 15.4, 16 16.4 / 15.4, 64 19.5 / 16.4.
FEW = 16


class PagedKV(NamedTuple):
    k: torch.Tensor           # [pages, H, P, D], keys behind RoPE and norm
    v: torch.Tensor           # [pages, H, P, D]

    @property
    def page(self) -> int:
        return self.k.shape[2]


def cache(pages: int, n_head: int, head_dim: int, page: int, device, dtype) -> PagedKV:
    if head_dim not in HEAD_DIMS or page not in PAGES:
        raise ValueError(f"paged cache: head_dim {head_dim} (supported: {HEAD_DIMS}), {page} tokens a page (supported: {PAGES})")
    if pages < 1 or not 1 <= n_head <= 65535 or pages * n_head * page > MOST_ROWS:
        raise ValueError(f"paged cache: {pages} pages, {n_head} heads")
    k, v = (torch.zeros(pages, n_head, page, head_dim, dtype=dtype, device=device) for _ in range(2))
    return PagedKV(k, v)


def _check(c: PagedKV, table, starts, pos):
    """``(B, M, H, P, D, device index)`` of a cache, and of a table, starts and positions of pieces, that the kernels can go by."""
    if len(c) != 2 or c[0].dim() != 4 or table.dim() != 2:
        raise ValueError("paged cache: two tensors [pages, H, P, D] and a table [B, pages of a sequence]")
    (pages, h, page, d), (b, m) = c[0].shape, table.shape
    k, v = c
    dev = k.get_device()
    if d not in HEAD_DIMS or page not in PAGES or not (
            k.dtype is v.dtype and k.is_floating_point() and v.shape == k.shape and v.get_device() == dev and k.is_contiguous() and v.is_contiguous()
            and (k.data_ptr() | v.data_ptr()) % 32 == 0 and 1 <= pages and 1 <= h <= 65535 and pages * h * page <= MOST_ROWS):
        raise ValueError(f"paged cache: k {k.dtype} {tuple(k.shape)}, v {v.dtype} {tuple(v.shape)}: not two contiguous tensors of one cache on one device, each on 32 bytes")
    if not (table.dtype is torch.int32 and table.get_device() == dev and table.stride(1) == 1 and 1 <= b <= 65534 and 1 <= m and m * page <= MAX_LEN
            and (b == 1 or table.stride(0) >= m)):
        raise ValueError(f"paged cache: table {table.dtype} {tuple(table.shape)} on {table.device}, expected int32 [B, pages] with rows of consecutive values on {k.device}")
    if not (starts.dtype is torch.int32 and starts.shape == (b + 1,) and starts.get_device() == dev and starts.is_contiguous() and pos.dtype is torch.int32
            and pos.shape == (b,) and pos.get_device() == dev and pos.is_contiguous()):
        raise ValueError(f"paged cache: starts {starts.dtype} {tuple(starts.shape)}, pos {pos.dtype} {tuple(pos.shape)}, expected contiguous int32 [{b + 1}] and [{b}] on {k.device}")
    return b, m, h, page, d, dev


def _rows(x, n_cols, dev, what):
    if x.dim() != 2 or x.shape[1] != n_cols or x.get_device() != dev or not x.is_floating_point() or x.shape[0] >= 1 << 26:
        raise ValueError(f"paged cache: {what} {x.dtype} {tuple(x.shape)} on {x.device}, expected [N, {n_cols}] on the cache's device, of fewer than 2^26 rows")


def check_append(qkv, cos, sin, c, table, starts, pos):
    dims = _, _, h, _, d, dev = _check(c, table, starts, pos)
    _rows(qkv, 3 * h * d, dev, "qkv")
    if (cos.dim() != 2 or cos.shape[1] != d // 2 or sin.shape != cos.shape or cos.get_device() != dev or sin.get_device() != dev or not cos.is_floating_point()
            or not sin.is_floating_point()):
        raise ValueError(f"paged cache: rotary tables {tuple(cos.shape)}, {tuple(sin.shape)}, expected [positions, {d // 2}]")
    return dims


def check_attention(q, c, table, starts, pos, scale, doc_start, window, longest):
    dims = b, _, h, _, d, dev = _check(c, table, starts, pos)
    _rows(q, h * d, dev, "queries")
    if q.dtype is not c[0].dtype:
        raise ValueError(f"paged attention: queries of {q.dtype}, a cache of {c[0].dtype}")
    if doc_start is not None and (doc_start.dtype is not torch.int32 or doc_start.shape != (q.shape[0],) or doc_start.get_device() != dev or not doc_start.is_contiguous()):
        raise ValueError(f"paged attention: doc_start is contiguous int32 [{q.shape[0]}] on {q.device}")
    if window < 0 or window % 128:
        raise ValueError(f"paged attention: window {window} is not a multiple of 128")
    if longest is not None and longest < 0:
        raise ValueError(f"paged attention: longest piece {longest}")
    if not abs(scale) < float("inf"):
        raise ValueError(f"paged attention: scale {scale}")
    return dims


def no_gradient(*xs):
    if torch.is_grad_enabled() and any(x.requires_grad for x in xs):
        raise ValueError("paged cache: its operators have no gradient; call them under torch.no_grad()")
    if has_tangent(*xs):
        raise ValueError("paged cache: its operators have no forward-mode differentiation")


# -- native bodies -----------------------------------------------------------------------------------------------------
def short_append(*args):
    """The call by the short way (``csrc/calls.cpp``), or None where its tensors are not as the kernel wants them."""
    q = L.calls().paged_append(*args)
    if q is not None:
        L.LAUNCHES[0] += 1
        COUNTS["paged_append"] += 1
    return q


def short_attention(q, c, table, starts, pos, scale, doc_start, window, longest):
    y = L.calls().paged_attention(q, c, table, starts, pos, scale, doc_start, window, longest, FEW, SHIFT)
    if y is not None:
        L.LAUNCHES[0] += 2
        COUNTS["paged_attention"] += 1
    return y


def _rows_on(x, by):
    """``x [N, C]`` as the kernels read it, and its address: consecutive values, rows that begin on ``by`` bytes."""
    at = x.data_ptr()
    if x.stride(1) != 1 or at % by or (x.shape[0] > 1 and x.stride(0) * 2 % by):
        x = x.contiguous() if not x.is_contiguous() else x.clone()
        at = x.data_ptr()
    return x, at


def append(dims, qkv, cos, sin, c, table, starts, pos):
    _bf16(qkv, "qkv")
    b, m, h, page, d, dev = dims
    k, v = c
    _bf16(k, "a cache")
    qkv, at = _rows_on(qkv, 16)
    cos, sin = _table(cos), _table(sin)
    n = qkv.shape[0]
    q = qkv.new_empty((n, h * d))
    if n:
        with L.device(dev):
            L.call("bones_paged_append", at, qkv.stride(0), cos.data_ptr(), sin.data_ptr(), cos.shape[0], k.data_ptr(), v.data_ptr(), k.shape[0], table.data_ptr(),
                   table.stride(0) if b > 1 else m, starts.data_ptr(), pos.data_ptr(), b, n, m, h, d, page.bit_length() - 1, q.data_ptr(), L.raw_stream())
        COUNTS["paged_append"] += 1
    return q


def attention(dims, q, c, table, starts, pos, scale, doc_start, window, longest):
    _bf16(q, "queries")
    b, m, h, page, d, dev = dims
    k, v = c
    if abs(scale) * d > SHIFT:
        raise ValueError(f"native paged attention does not cover this call: scale {scale} (at most {SHIFT / d} for heads of {d})")
    n = q.shape[0]
    if n > 1 and q.stride(0) != h * d:
        q = q.contiguous()
    q, at = _rows_on(q, 32)
    y = torch.empty_like(q)
    if n:
        if longest is None:
            longest = -(-n // b)
        tiles = min(window // 128, MOST_WINDOW)
        with L.device(dev):
            room = _room(b, n, m * page, h, d, tiles, longest > FEW, dev)
            work = torch.empty(room, dtype=torch.uint8, device=q.device)
            L.call("bones_paged_attention", at, k.data_ptr(), v.data_ptr(), k.shape[0], table.data_ptr(), table.stride(0) if b > 1 else m, starts.data_ptr(),
                   pos.data_ptr(), 0 if doc_start is None else doc_start.data_ptr(), y.data_ptr(), b, n, m, h, d, page.bit_length() - 1, scale, tiles,
                   longest > FEW, work.data_ptr(), room, L.raw_stream(), launches=2)
        COUNTS["paged_attention"] += 1
    return y


@functools.lru_cache(maxsize=4096)
def _room(b, n, capacity, h, d, window_tiles, long, dev) -> int:
    """Bytes that ``bones_paged_attention`` works with."""
    with L.device(dev):
        return L.load().bones_paged_room(b, n, capacity, h, d, window_tiles, long, 0)
