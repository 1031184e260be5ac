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
import struct
from dataclasses import dataclass

import torch

from . import _native as nat

HEAD_DIM = 128
PAGE_SIZES = (16, 32, 64, 128)


@dataclass(frozen=True, eq=False)
class KVCache:
    """E4M3 codes ``k`` / ``v`` [pages, heads, page_size, 128] and scales [pages, heads].

    The tensors are checked once and cannot be replaced (their contents are what append changes).
    """
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
        # what every call needs of them (frozen: set past the dataclass)
        self.__dict__.update(
            _device=k.device, _index=k.get_device(), _heads=k.shape[1],
            _c=(k.data_ptr(), v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr(), k.shape[0], k.shape[1],
                k.shape[2], HEAD_DIM, 0))

    def __reduce__(self):  # a copy or an unpickled cache has pointers of its own
        return _from_bytes, (self.k.view(torch.uint8), self.v.view(torch.uint8), self.k_scale, self.v_scale)

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


def _from_bytes(k, v, k_scale, v_scale) -> KVCache:
    """A cache whose codes come as bytes (torch pickles those; its 8-bit floats it does not read back)."""
    return KVCache(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), k_scale, v_scale)


# The argument blocks of include/demon_b200.h as struct formats (native sizes, no implicit padding:
# every 8-byte field lies at a multiple of 8).  Packing one takes a fraction of a microsecond where a
# ctypes structure of as many fields takes several, and a call for one token is bound by the host.
_CACHE = "4Pq4i"
_APPEND = struct.Struct("@" + _CACHE + "P3qP3qPqPP4i")
_READ = struct.Struct("@" + _CACHE + "P2qP2qPqP4i")
_ATTN = struct.Struct("@" + _CACHE + "P3qP3qPqPP4i2ifiPq")
for _s, _c in ((_APPEND, nat.DemonKvAppendArgs), (_READ, nat.DemonKvReadArgs), (_ATTN, nat.DemonKvAttnArgs)):
    assert _s.size == nat.ctypes.sizeof(_c)

_NO_CONTEXT = contextlib.nullcontext()
_DEFAULT_SCALE = HEAD_DIM ** -0.5


def _launch(index: int, stream):
    """The context a call launches in: the tensors' device current, and, when the caller names a
    stream, that stream current too (so that outputs are allocated for it)."""
    if stream is not None:
        if stream.device_index != index:
            raise ValueError(f"stream is on cuda:{stream.device_index}, the tensors on cuda:{index}")
        return torch.cuda.stream(stream)
    if index != torch._C._cuda_getDevice():
        return torch.cuda.device(index)
    return _NO_CONTEXT


def _bf16_rows(t: torch.Tensor, name: str, index: int) -> tuple:
    """Checks a [B, rows, heads, 128] bf16 tensor; its shape and (sequence, row, head) strides, 0
    along dimensions of one entry (where a stride means nothing)."""
    shape = t.shape
    if t.dtype is not torch.bfloat16 or len(shape) != 4 or t.get_device() != index:
        raise ValueError(f"{name} must be a 4-D bf16 tensor [B, rows, heads, 128] on cuda:{index}")
    st = t.stride()
    if shape[3] != HEAD_DIM or (st[3] != 1 and t.numel()):
        raise ValueError(f"{name}: head_dim must be 128 with unit stride (shape {tuple(shape)}, strides {st})")
    return shape, (0 if shape[0] == 1 else st[0], 0 if shape[1] == 1 else st[1], 0 if shape[2] == 1 else st[2])


def _int32(t: torch.Tensor, name: str, B: int, index: int) -> int:
    if t.dtype is not torch.int32 or t.shape != (B,) or t.get_device() != index or (B > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous int32 tensor [{B}] on cuda:{index}")
    return t.data_ptr()


def _table(t: torch.Tensor, B: int, index: int) -> tuple:
    """(pointer, row pitch, width) of a page table."""
    if t.dtype is not torch.int32 or t.dim() != 2 or t.shape[0] != B or t.get_device() != index or \
            (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"table must be an int32 tensor [{B}, W] with unit column stride on cuda:{index}")
    W = t.shape[1]
    return t.data_ptr(), t.stride(0) if B > 1 else W, W


def append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor,
           count: torch.Tensor | None = None, stream=None) -> None:
    """Quantise ``k`` / ``v`` [B, S, heads, 128] bf16 into the cache, in place.

    Token i < ``count[b]`` (default S) of sequence b goes to position ``start[b] + i``.  Per page
    and head the scale is the smallest power of two that covers every token written since the
    page was empty; when it grows, the page's earlier tokens are rounded again.  k and v are read
    through their strides (multiples of 8 elements; columns of a fused projection work as they
    are).  The pages a call writes must belong to one sequence each and stand in its table once.
    """
    dev = cache._index
    shape, ks = _bf16_rows(k, "k", dev)
    vshape, vs = _bf16_rows(v, "v", dev)
    B, S = shape[0], shape[1]
    if vshape != shape or shape[2] != cache._heads:
        raise ValueError(f"k {tuple(shape)} and v {tuple(vshape)} must be equal, with the cache's {cache._heads} heads")
    tp, ld, W = _table(table, B, dev)
    args = _APPEND.pack(*cache._c, k.data_ptr(), *ks, v.data_ptr(), *vs, tp, ld, _int32(start, "start", B, dev),
                        0 if count is None else _int32(count, "count", B, dev), B, S, W, 0)
    with _launch(dev, stream):
        nat.check(nat.load().demon_kv_append(args, nat.raw_stream(dev)))


def read(cache: KVCache, table: torch.Tensor, lens: torch.Tensor, max_len: int, out=None, stream=None):
    """The cached values back in bf16: (k, v), each [B, max_len, heads, 128], positions
    0 .. ``lens[b]`` - 1 of sequence b and zeros from there.  ``out``: a (k, v) pair to write
    into (heads contiguous within a row)."""
    dev, H, max_len = cache._index, cache._heads, int(max_len)
    B = table.shape[0]
    tp, ld, W = _table(table, B, dev)
    lp = _int32(lens, "lens", B, dev)
    with _launch(dev, stream):
        if out is None:
            out = torch.empty((2, B, max_len, H, HEAD_DIM), dtype=torch.bfloat16, device=cache._device).unbind(0)
            row = H * HEAD_DIM
            pitch = ((max_len * row, row),) * 2
        else:
            pitch = []
            for t, n in zip(out, ("out k", "out v")):
                shape, st = _bf16_rows(t, n, dev)
                if tuple(shape) != (B, max_len, H, HEAD_DIM) or (H > 1 and st[2] != HEAD_DIM):
                    raise ValueError(f"{n} must be {[B, max_len, H, HEAD_DIM]} with contiguous heads, got "
                                     f"{tuple(shape)}, strides {t.stride()}")
                pitch.append((st[0], st[1] if max_len > 1 else H * HEAD_DIM))
        ko, vo = out
        args = _READ.pack(*cache._c, ko.data_ptr(), *pitch[0], vo.data_ptr(), *pitch[1], tp, ld, lp, B, max_len, W, 0)
        nat.check(nat.load().demon_kv_read(args, nat.raw_stream(dev)))
    return ko, vo


def attention(q: torch.Tensor, cache: KVCache, table: torch.Tensor, lens: torch.Tensor, causal: bool = False,
              window: int | None = None, scale: float | None = None, q_lens: torch.Tensor | None = None,
              out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """softmax(scale q k^T) v of ``q`` [B, Sq, Hq, 128] bf16 over the cached keys -> [B, Sq, Hq, 128].

    ``lens[b]``: keys of sequence b (its new tokens among them, already appended).  Query i of
    its ``q_lens[b]`` (default Sq) stands at position ``lens[b] - q_lens[b] + i``; ``causal``
    hides the keys after that position, ``window`` those farther than ``window`` from it.  Rows
    that see no key, and rows i >= ``q_lens[b]``, are zero.  ``scale`` defaults to 1 / sqrt(128).
    ``out`` may be ``q`` itself; it must not overlap other rows of it.
    """
    dev = cache._index
    if window is not None and window < 0:  # (-1 is the C struct's word for none)
        raise nat.DemonError(nat.DEMON_ERR_INVALID, f"kv_attention: window must be None or at least 0 (got {window})")
    shape, qs = _bf16_rows(q, "q", dev)
    B, Sq, Hq, _ = shape
    tp, ld, W = _table(table, B, dev)
    lp = _int32(lens, "lens", B, dev)
    qp = 0 if q_lens is None else _int32(q_lens, "q_lens", B, dev)
    with _launch(dev, stream):
        if 0 in qs and any(n > 1 and st == 0 for n, st in zip(shape, qs)):
            q = q.contiguous()  # broadcast queries, copied on the call's own stream
            qs = _bf16_rows(q, "q", dev)[1]
        if out is None:
            out = torch.empty(shape, dtype=torch.bfloat16, device=cache._device)
            os = (Sq * Hq * HEAD_DIM, Hq * HEAD_DIM, HEAD_DIM)
        else:
            oshape, os = _bf16_rows(out, "out", dev)
            if oshape != shape or any(n > 1 and st == 0 for n, st in zip(shape, os)):
                raise ValueError(f"out must be {tuple(shape)} without overlap, got {tuple(oshape)}, strides {out.stride()}")
        fields = (*cache._c, q.data_ptr(), *qs, out.data_ptr(), *os, tp, ld, lp, qp, B, Sq, Hq, W,
                  1 if causal else 0, -1 if window is None else min(int(window), 1 << 30),
                  _DEFAULT_SCALE if scale is None else float(scale), 0)
        args = _ATTN.pack(*fields, 0, 0)
        if W * cache._c[6] > (8_128 if Sq * Hq <= 16 * cache._heads else 896):  # shorter tables take no workspace
            n = nat.load().demon_kv_attention_workspace(args)
            if n:
                ws = torch.empty(n, dtype=torch.uint8, device=cache._device)
                args = _ATTN.pack(*fields, ws.data_ptr(), n)
        nat.check(nat.load().demon_kv_attention(args, nat.raw_stream(dev)))
    return out
