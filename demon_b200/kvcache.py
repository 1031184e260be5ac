"""Paged 8-bit K/V cache: quantising tokens as they are written, reading them back, and
attention over the cache (``demon_kv_append`` / ``demon_kv_read`` / ``demon_kv_attention`` in
include/demon_b200.h).

A :class:`KVCache` holds E4M3 codes in pages of ``page_size`` tokens, ``[pages, heads,
page_size, 128]`` for K and for V, with one power-of-two fp32 scale per page and head; a value
is ``code * scale`` and is exact in bf16.  Which pages a sequence has is the caller's: a page
table ``[B, W]`` (int32, -1 where there is no page) lists them in order, and the same page may
stand in several rows that are only read, so that sequences share a condition's keys.

    cache = KVCache.empty(pages, heads=8, page_size=64, device="cuda")
    append(cache, k, v, table, start)              # k / v [B, S, 8, 128] bf16 -> positions start[b] ..
    o = attention(q, cache, table, lens, causal=True)   # q [B, Sq, Hq, 128] -> o, lens: keys per sequence
    k, v = read(cache, table, lens, max_len)       # back to bf16 [B, max_len, 8, 128]

It stands in for the bf16 K / V that the reference recomputes for its cross attention
(acestep/models/modeling_acestep_v15_turbo.py:320-345); :meth:`demon_b200.dit.DemonDiT.encoder_kv`
writes one with ``cache="e4m3"``.

``table``, ``start``, ``count``, ``lens`` and ``q_lens`` are device tensors and are read by the
kernels: nothing here synchronises, and every call can be captured in a CUDA graph and replayed
with other contents.  A value out of range there (a length beyond the table, a page id that does
not exist) is reported in :func:`demon_b200._native.device_status` and touches nothing.  No
PyTorch fallback: every call goes to libdemon_b200.so.
"""
from __future__ import annotations

import contextlib
import ctypes
from dataclasses import dataclass

import torch

from . import _native as nat

HEAD_DIM = 128
PAGE_SIZES = (16, 32, 64, 128)


@dataclass
class KVCache:
    """E4M3 codes ``k`` / ``v`` [pages, heads, page_size, 128] and scales [pages, heads]."""
    k: torch.Tensor        # float8_e4m3fn [pages, heads, page_size, 128], contiguous
    v: torch.Tensor
    k_scale: torch.Tensor  # float32 [pages, heads], powers of two
    v_scale: torch.Tensor

    def __post_init__(self):
        k, v = self.k, self.v
        for t, n in ((k, "k"), (v, "v")):
            if t.dtype != torch.float8_e4m3fn or t.dim() != 4 or not t.is_contiguous():
                raise ValueError(f"cache {n} must be a contiguous float8_e4m3fn tensor [pages, heads, page_size, 128]")
        if v.shape != k.shape or k.shape[3] != HEAD_DIM or k.shape[2] not in PAGE_SIZES:
            raise ValueError(f"cache k {tuple(k.shape)} and v {tuple(v.shape)} must be equal, head_dim 128, "
                             f"page_size one of {PAGE_SIZES}")
        for t, n in ((self.k_scale, "k_scale"), (self.v_scale, "v_scale")):
            if t.dtype != torch.float32 or t.shape != k.shape[:2] or not t.is_contiguous():
                raise ValueError(f"cache {n} must be a contiguous float32 tensor [pages, heads]")
        if not k.is_cuda or any(t.device != k.device for t in (v, self.k_scale, self.v_scale)):
            raise ValueError("the cache's tensors must be on one CUDA device (demon_b200 has no CPU path)")
        self._c = nat.DemonKvCache(nat.ptr(k), nat.ptr(v), nat.ptr(self.k_scale), nat.ptr(self.v_scale), k.shape[0],
                                   k.shape[1], k.shape[2], HEAD_DIM, 0)

    @classmethod
    def empty(cls, pages: int, heads: int, page_size: int = 64, device="cuda") -> "KVCache":
        """A cache of ``pages`` pages, every value zero."""
        shape = (pages, heads, page_size, HEAD_DIM)
        codes = [torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
        scales = [torch.full(shape[:2], 2.0 ** -120, dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*codes, *scales)

    @property
    def pages(self) -> int:
        return self.k.shape[0]

    @property
    def heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]


def _launch(device: torch.device, stream):
    """The context a call launches in: the tensors' device current, and, when the caller names a
    stream, that stream current too (so that outputs are allocated for it)."""
    if stream is not None:
        return torch.cuda.stream(stream)
    if device.index != torch.cuda.current_device():
        return torch.cuda.device(device)
    return contextlib.nullcontext()


def _bf16_rows(t: torch.Tensor, name: str, device: torch.device) -> None:
    if t.dtype != torch.bfloat16 or t.dim() != 4 or t.device != device:
        raise ValueError(f"{name} must be a 4-D bf16 tensor [B, rows, heads, 128] on {device}")
    if t.shape[3] != HEAD_DIM or (t.stride(3) != 1 and t.numel()):
        raise ValueError(f"{name}: head_dim must be 128 with unit stride (shape {tuple(t.shape)}, strides {t.stride()})")


def _strides(t: torch.Tensor) -> tuple:
    """(sequence, row, head) strides, 0 along dimensions of one entry (where a stride means nothing)."""
    return tuple(0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3]))


def _int32(t: torch.Tensor, name: str, B: int, device: torch.device) -> None:
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != B or t.device != device or (B > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous int32 tensor [{B}] on {device}")


def _table(t: torch.Tensor, B: int, device: torch.device) -> int:
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != B or t.device != device or \
            (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"table must be an int32 tensor [{B}, W] with unit column stride on {device}")
    return t.stride(0) if B > 1 else t.shape[1]


def append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor,
           count: torch.Tensor | None = None, stream=None) -> None:
    """Quantise ``k`` / ``v`` [B, S, heads, 128] bf16 into the cache, in place.

    Token i < ``count[b]`` (default S) of sequence b goes to position ``start[b] + i``.  Per page
    and head the scale is the smallest power of two that covers every token written since the
    page was empty; when it grows, the page's earlier tokens are rounded again.  k and v are read
    through their strides (multiples of 8 elements; columns of a fused projection work as they
    are).  The pages a call writes must belong to one sequence each.
    """
    dev = cache.k.device
    _bf16_rows(k, "k", dev)
    _bf16_rows(v, "v", dev)
    B, S, H, _ = k.shape
    if v.shape != k.shape or H != cache.heads:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be equal, with the cache's {cache.heads} heads")
    ld = _table(table, B, dev)
    _int32(start, "start", B, dev)
    if count is not None:
        _int32(count, "count", B, dev)
    a = nat.DemonKvAppendArgs(cache._c, nat.ptr(k), *_strides(k), nat.ptr(v), *_strides(v), nat.ptr(table), ld,
                              nat.ptr(start), nat.ptr(count), B, S, table.shape[1], 0)
    with _launch(dev, stream):
        nat.check(nat.load().demon_kv_append(ctypes.byref(a), nat.stream_ptr(stream)))


def read(cache: KVCache, table: torch.Tensor, lens: torch.Tensor, max_len: int, out=None, stream=None):
    """The cached values back in bf16: (k, v), each [B, max_len, heads, 128], positions
    0 .. ``lens[b]`` - 1 of sequence b and zeros from there.  ``out``: a (k, v) pair to write
    into (heads contiguous within a row)."""
    dev = cache.k.device
    B = table.shape[0]
    ld = _table(table, B, dev)
    _int32(lens, "lens", B, dev)
    shape = (B, int(max_len), cache.heads, HEAD_DIM)
    with _launch(dev, stream):
        if out is None:
            out = tuple(torch.empty(shape, dtype=torch.bfloat16, device=dev) for _ in range(2))
        else:
            for t, n in zip(out, ("out k", "out v")):
                _bf16_rows(t, n, dev)
                if tuple(t.shape) != shape or (cache.heads > 1 and t.stride(2) != HEAD_DIM):
                    raise ValueError(f"{n} must be {list(shape)} with contiguous heads, got {tuple(t.shape)}, "
                                     f"strides {t.stride()}")
        ko, vo = out
        pitch = [(t.stride(0), t.stride(1) if max_len > 1 else cache.heads * HEAD_DIM) for t in out]
        a = nat.DemonKvReadArgs(cache._c, nat.ptr(ko), *pitch[0], nat.ptr(vo), *pitch[1], nat.ptr(table), ld,
                                nat.ptr(lens), B, int(max_len), table.shape[1], 0)
        nat.check(nat.load().demon_kv_read(ctypes.byref(a), nat.stream_ptr(stream)))
    return ko, vo


def attention(q: torch.Tensor, cache: KVCache, table: torch.Tensor, lens: torch.Tensor, causal: bool = False,
              window: int | None = None, scale: float | None = None, q_lens: torch.Tensor | None = None,
              out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """softmax(scale q k^T) v of ``q`` [B, Sq, Hq, 128] bf16 over the cached keys -> [B, Sq, Hq, 128].

    ``lens[b]``: keys of sequence b (its new tokens among them, already appended).  Query i of
    its ``q_lens[b]`` (default Sq) stands at position ``lens[b] - q_lens[b] + i``; ``causal``
    hides the keys after that position, ``window`` those farther than ``window`` from it.  Rows
    that see no key, and rows i >= ``q_lens[b]``, are zero.  ``scale`` defaults to 1 / sqrt(128).
    """
    dev = cache.k.device
    _bf16_rows(q, "q", dev)
    B, Sq, Hq, _ = q.shape
    ld = _table(table, B, dev)
    _int32(lens, "lens", B, dev)
    if q_lens is not None:
        _int32(q_lens, "q_lens", B, dev)
    with _launch(dev, stream):
        if out is None:
            out = torch.empty(B, Sq, Hq, HEAD_DIM, dtype=torch.bfloat16, device=dev)
        else:
            _bf16_rows(out, "out", dev)
            if out.shape != q.shape:
                raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
        a = nat.DemonKvAttnArgs(cache._c, nat.ptr(q), *_strides(q), nat.ptr(out), *_strides(out), nat.ptr(table), ld,
                                nat.ptr(lens), nat.ptr(q_lens), B, Sq, Hq, table.shape[1], 1 if causal else 0,
                                -1 if window is None else int(window),
                                float(HEAD_DIM ** -0.5 if scale is None else scale), 0)
        nat.check(nat.load().demon_kv_attention(ctypes.byref(a), nat.stream_ptr(stream)))
    return out
