"""A key/value cache in 8 bits: its layout, the checks of its calls and the native bodies (``csrc/kv8.cu``).

Per layer six tensors (``KV8``).  Blocks of 64 tokens; a block becomes int8 codes and one fp32 scale a head when its last
token comes, from the bf16 values of all of its tokens, so what a cache holds does not depend on how they came: one by one,
in one run or in pieces.  Until then the tokens of the open block are in bf16.  The values of a block are stored transposed:
a lane that multiplies probabilities with them reads consecutive tokens of one dimension.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib as L
from . import COUNTS
from .logprobs import has_tangent

BLOCK = 64
HEAD_DIMS = (128, 64)
MAX_LEN = (1 << 31) - 2 * BLOCK        # positions are 32-bit
LONG, PARTS = 16384, 1024              # capacity from which the attention gets room for parts of its result, and for how many (it takes no more)


class KV8(NamedTuple):
    """One layer's keys and values: codes, scales (a minus sign marks a block that holds a value that is not finite) and the
    open block.  Capacity ``T`` is a multiple of 64."""
    k: torch.Tensor           # int8 [B, H, T, D]
    v: torch.Tensor           # int8 [B, H, T / 64, D, 64]
    k_scale: torch.Tensor     # fp32 [B, H, T / 64]
    v_scale: torch.Tensor     # fp32 [B, H, T / 64]
    k_open: torch.Tensor      # bf16 [B, H, 64, D]
    v_open: torch.Tensor      # bf16 [B, H, 64, D]

    @property
    def capacity(self) -> int:
        return self.k.shape[2]


def cache(batch: int, max_len: int, n_head: int, head_dim: int, device=None) -> KV8:
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"8-bit cache: head_dim {head_dim} (supported: {HEAD_DIMS})")
    if batch < 1 or n_head < 1 or max_len < 1 or max_len > MAX_LEN or batch > 65535 or n_head > 65535:
        raise ValueError(f"8-bit cache: batch {batch}, heads {n_head}, length {max_len}")
    nb = -(-max_len // BLOCK)
    z = lambda dt, *shape: torch.zeros(*shape, dtype=dt, device=device)  # noqa: E731
    return KV8(z(torch.int8, batch, n_head, nb * BLOCK, head_dim), z(torch.int8, batch, n_head, nb, head_dim, BLOCK),
               z(torch.float32, batch, n_head, nb), z(torch.float32, batch, n_head, nb),
               z(torch.bfloat16, batch, n_head, BLOCK, head_dim), z(torch.bfloat16, batch, n_head, BLOCK, head_dim))


def check_cache(c: KV8):
    """``(B, H, T, D, device index, addresses)`` of a cache whose tensors are what the kernels take them for."""
    if len(c) != 6 or c[0].dim() != 4:
        raise ValueError("8-bit cache: six tensors, the first [B, H, T, D]")
    b, h, t, d = c[0].shape
    nb = t // BLOCK
    if d not in HEAD_DIMS or t < BLOCK or t % BLOCK or t > MAX_LEN + BLOCK or not 1 <= b <= 65535 or not 1 <= h <= 65535:
        raise ValueError(f"8-bit cache: shape {tuple(c[0].shape)}")
    k, v, ks, vs, kt, vt = c
    dev, scales, open_ = k.get_device(), (b, h, nb), (b, h, BLOCK, d)
    at = k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), kt.data_ptr(), vt.data_ptr()
    # one expression: a loop over the six would be a fifth of a call's host time
    if not (k.dtype is torch.int8 and v.dtype is torch.int8 and ks.dtype is torch.float32 and vs.dtype is torch.float32 and kt.dtype is torch.bfloat16
            and vt.dtype is torch.bfloat16 and v.shape == (b, h, nb, d, BLOCK) and ks.shape == scales and vs.shape == scales and kt.shape == open_
            and vt.shape == open_ and v.get_device() == dev and ks.get_device() == dev and vs.get_device() == dev and kt.get_device() == dev
            and vt.get_device() == dev and k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous() and kt.is_contiguous()
            and vt.is_contiguous() and (at[0] | at[1] | at[2] | at[3] | at[4] | at[5]) % 16 == 0):
        have = ", ".join(f"{n} {x.dtype} {tuple(x.shape)}" for n, x in zip(KV8._fields, c))
        raise ValueError(f"8-bit cache: {have}: not six contiguous tensors of one cache on one device, each on 16 bytes")
    return b, h, t, d, dev, at


def check_per_sequence(x, b: int, name: str, device):
    """An int, or int32 of one value or of one for each sequence on the cache's device (an index, -1 for the host)."""
    if type(x) is int:
        return
    n = x.numel() if isinstance(x, torch.Tensor) else 0
    if (n != b and n != 1) or x.dtype is not torch.int32 or x.get_device() != device or x.dim() > 1 or not x.is_contiguous():
        raise ValueError(f"8-bit cache: {name} is an int or contiguous int32 of 1 or {b} values on the cache's device")


def check_append(c: KV8, k, v, pos, lens):
    dims = b, h, t, d, dev, _ = check_cache(c)
    if k.dim() != 4 or v.shape != k.shape or k.shape[0] != b or k.shape[2] != h or k.shape[3] != d:
        raise ValueError(f"8-bit cache: keys {tuple(k.shape)}, values {tuple(v.shape)}, cache {tuple(c[0].shape)}")
    if k.get_device() != dev or v.get_device() != dev or k.dtype is not v.dtype or not k.is_floating_point():
        raise ValueError("8-bit cache: keys and values of one floating type on the cache's device")
    check_per_sequence(pos, b, "pos", dev)
    if lens is not None:
        check_per_sequence(lens, b, "lens", dev)
    if isinstance(lens, int) and not 0 <= lens <= k.shape[1]:
        raise ValueError(f"8-bit cache: {lens} of {k.shape[1]} tokens")
    if isinstance(pos, int) and (lens is None or isinstance(lens, int)):
        n = k.shape[1] if lens is None else lens
        if pos < 0 or pos + n > t:
            raise ValueError(f"8-bit cache: {n} of {k.shape[1]} tokens at {pos} into a capacity of {t}")
    return dims


def check_read(c: KV8, held, length):
    dims = check_cache(c)
    check_per_sequence(held, dims[0], "held", dims[4])
    if length < 0 or length > MAX_LEN or (isinstance(held, int) and not 0 <= held <= dims[2]):
        raise ValueError(f"8-bit cache: {length} positions of {held} tokens, capacity {dims[2]}")
    return dims


def check_attention(qkv, cos, sin, c: KV8, pos, doc_start, window):
    dims = b, h, t, d, dev, _ = check_cache(c)
    if qkv.shape != (b, 3 * h * d) or qkv.get_device() != dev or not qkv.is_floating_point():
        raise ValueError(f"8-bit attention: qkv {qkv.dtype} {tuple(qkv.shape)} on {qkv.device}, expected {(b, 3 * h * d)} on {c[0].device}")
    shape = cos.shape
    if (len(shape) != 2 or shape[1] != d // 2 or sin.shape != shape or cos.get_device() != dev or sin.get_device() != dev or not cos.is_floating_point()
            or not sin.is_floating_point()):
        raise ValueError(f"8-bit attention: rotary tables {tuple(cos.shape)}, {tuple(sin.shape)}, expected [positions, {d // 2}]")
    check_per_sequence(pos, b, "pos", dev)
    if type(pos) is int and not 0 <= pos < min(t, shape[0]):
        raise ValueError(f"8-bit attention: position {pos}, capacity {t}, rotary tables of {cos.shape[0]}")
    if doc_start is not None and (doc_start.dtype is not torch.int32 or doc_start.shape != (b,) or doc_start.get_device() != dev or not doc_start.is_contiguous()):
        raise ValueError(f"8-bit attention: doc_start is contiguous int32 [{b}] on {c[0].device}")
    if window < 0 or window % 128:
        raise ValueError(f"8-bit attention: window {window} is not a multiple of 128")
    return dims


def no_gradient(x, y=None):
    if (x.requires_grad or (y is not None and y.requires_grad)) and torch.is_grad_enabled():
        raise ValueError("8-bit cache: its operators have no gradient; call them under torch.no_grad()")
    if has_tangent(x, y):
        raise ValueError("8-bit cache: its operators have no forward-mode differentiation")


def numbers(x, b: int):
    """``x`` of ``check_per_sequence`` as a list of ``b`` ints."""
    v = [x] if isinstance(x, int) else x.reshape(-1).tolist()
    return v * b if len(v) == 1 else v


# -- native bodies -----------------------------------------------------------------------------------------------------
def _per(x):
    """Address, distance from one sequence's value to the next's and the value itself where there is no address."""
    return (0, 0, x) if type(x) is int else (x.data_ptr(), 0 if x.numel() == 1 else 1, 0)


def _rows16(x):
    """``x [B, t, H, D]`` as the append kernel reads it: heads of consecutive values that begin on 16 bytes."""
    if x.stride(3) != 1 or any(x.stride(i) % 8 for i in range(3) if x.shape[i] > 1) or x.data_ptr() % 16:
        x = x.contiguous() if not x.is_contiguous() else x.clone()
    return x


def _bf16(x, what):
    if x.dtype != torch.bfloat16:
        raise ValueError(f"native 8-bit cache does not cover this call: {what} of {x.dtype} (bf16 only)")


def append(dims, k, v, pos, lens):
    _bf16(k, "keys and values")
    b, h, t, d, dev, at = dims
    n = k.shape[1]
    if n == 0:
        return
    k, v = _rows16(k), _rows16(v)
    (pa, ps, p0), (la, ls, l0) = _per(pos), _per(n if lens is None else lens)
    with L.device(dev):
        L.call("bones_kv8_append", at[0], at[1], at[2], at[3], at[4], at[5], k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.stride(0),
               v.stride(1), v.stride(2), b, h, d, t, n, pa, ps, p0, la, ls, l0, L.raw_stream())
    COUNTS["kv8_append"] += 1


def read(dims, held, length):
    b, h, t, d, dev, at = dims
    k, v = (torch.empty(b, length, h, d, dtype=torch.bfloat16, device=f"cuda:{dev}") for _ in range(2))
    if length:
        ha, hs, h0 = _per(held)
        with L.device(dev):
            L.call("bones_kv8_read", at[0], at[1], at[2], at[3], at[4], at[5], k.data_ptr(), v.data_ptr(), b, h, d, t, length, ha, hs, h0, L.raw_stream())
        COUNTS["kv8_read"] += 1
    return k, v


def _table(x):
    return x if x.dtype is torch.float32 and x.is_contiguous() else x.to(torch.float32).contiguous()


def attention(qkv, cos, sin, dims, pos, scale, doc_start, window):
    _bf16(qkv, "qkv")
    b, h, t, d, dev, _ = dims
    if qkv.stride(1) != 1 or (b > 1 and qkv.stride(0) % 8) or qkv.data_ptr() % 16:
        qkv = qkv.contiguous() if not qkv.is_contiguous() else qkv.clone()
    y = qkv.new_empty((b, h * d))
    with L.device(dev):
        launch(qkv, _table(cos), _table(sin), dims, pos, scale, doc_start, window, y)
    COUNTS["kv8_attention"] += 1
    return y


def launch(qkv, cos, sin, dims, pos, scale, doc_start, window, y, pdl=0):
    """The kernel alone, on operands that ``attention`` has checked.  ``pdl``: it may begin while the kernel before it on the stream
    still runs; what that kernel writes is not read before its end."""
    b, h, t, d, _, at = dims
    pa, ps, p0 = _per(pos)
    parts = torch.empty(PARTS * (d + 4), dtype=torch.float32, device=y.device) if t >= LONG and b <= 32 else None
    L.call("bones_kv8_attention", qkv.data_ptr(), qkv.stride(0), cos.data_ptr(), sin.data_ptr(), cos.shape[0], at[0], at[1], at[2], at[3], at[4], at[5], pa, ps,
           p0, 0 if doc_start is None else doc_start.data_ptr(), y.data_ptr(), b, h, d, t, scale, window // 128, pdl, 0 if parts is None else parts.data_ptr(), PARTS,
           L.raw_stream())
