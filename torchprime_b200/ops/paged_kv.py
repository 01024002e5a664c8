"""Paged key/value cache of a decoder: rows written and read back (csrc/paged_kv.cu) and attention of one new token per
sequence over the pages (csrc/paged_decode.cu).

A cache is a pool of pages of ``page`` tokens each.  Which pages hold a sequence, in which order, is the caller's
``block_table``; token ``i`` of sequence ``b`` lies at offset ``i % page`` of page ``block_table[b, i // page]``, and its
*slot* is ``block_table[b, i // page] * page + i % page``.  Pools are bf16, or e4m3 with one power of two (e8m0) for each
token and head: the smallest under which the row's finite values fit into +-448, at least 2^-100.

On CUDA/bf16 these run as sm_100a kernels; elsewhere, under a trace and where a gradient is recorded the same math runs in plain
PyTorch (``reference.py``).
"""

from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p
from typing import NamedTuple

import torch

from . import _debug, _lib, functional, reference as ref
from ._lib import check, lib, ptr, stream_ptr
from .functional import unobserved, use_kernels

P, I, LL, F = c_void_p, c_int, c_longlong, c_float
_lib.register_signature("tpb_paged_rows", [I, P, P, P, P, P, P, P, LL, I, I, I, I, I, P, P, P])
_lib.register_signature("tpb_paged_decode_scratch", [I, I, I, I, I, I, I])
_lib.register_signature("tpb_paged_decode", [P, LL, LL, P, P, P, P, P, P, LL, I, P, P, P, I, I, I, I, I, I, I, I, F, F, P])

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


class PagedKV(NamedTuple):
  """Pools of keys [P, page, H, Dk] and values [P, page, H, Dv]; ``k_scale`` and ``v_scale`` [P, page, H] where they are
  e4m3.  Any strides over contiguous rows; :meth:`allocate` puts a page's rows of one head back to back, which is what
  reads them fastest."""
  k: torch.Tensor
  v: torch.Tensor
  k_scale: torch.Tensor | None = None
  v_scale: torch.Tensor | None = None

  @classmethod
  def allocate(cls, pages: int, page: int, heads: int, dk: int, dv: int | None = None, dtype=torch.bfloat16,
               device=None) -> "PagedKV":
    mk = lambda d: torch.zeros(pages, heads, page, d, dtype=dtype, device=device).transpose(1, 2)  # noqa: E731
    sc = lambda: torch.ones(pages, heads, page, device=device).to(E8M0).transpose(1, 2) if dtype == E4M3 else None  # noqa: E731
    return cls(mk(dk), mk(dv if dv is not None else dk), sc(), sc())

  @property
  def page(self) -> int:
    return self.k.shape[1]

  def nbytes(self) -> int:
    return sum(t.numel() * t.element_size() for t in self if t is not None)


def _check_cache(c: PagedKV):
  if c.k.dim() != 4 or c.v.dim() != 4 or 0 in c.k.shape or 0 in c.v.shape:
    raise ValueError(f"pools are [pages, page, heads, columns], got {tuple(c.k.shape)} and {tuple(c.v.shape)}")
  pages, page, h, _ = c.k.shape
  if c.v.shape[:3] != c.k.shape[:3] or c.v.dtype != c.k.dtype:
    raise ValueError(f"pools of keys {tuple(c.k.shape)} {c.k.dtype} and values {tuple(c.v.shape)} {c.v.dtype} differ")
  if (c.k.dtype == E4M3) != (c.k_scale is not None) or (c.k_scale is None) != (c.v_scale is None):
    raise ValueError("e4m3 pools, and only they, come with k_scale and v_scale")
  for s in (c.k_scale, c.v_scale):
    if s is not None and (s.shape != (pages, page, h) or s.dtype != E8M0):
      raise ValueError(f"scales must be {E8M0} of {(pages, page, h)}, got {s.dtype} of {tuple(s.shape)}")
  for t in c[1:]:
    if t is not None and t.device != c.k.device:
      raise ValueError("a cache lies on one device")


def _rows_ok(c: PagedKV, h: int, *ds) -> bool:
  """What the row kernels take: 16-byte vectors of rows of up to 512 values, slots that fit into 31 bits."""
  unit = 16 // c.k.element_size()
  return (c.k.dtype in (torch.bfloat16, E4M3) and c.k.is_cuda and c.k.shape[0] * c.page < 2 ** 31
          and all(d % max(8, unit) == 0 and 8 <= d <= 512 for d in ds)
          and all(t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(s % unit == 0 for s in t.stride()[:3]) for t in c[:2]))


def _recorded(*tensors) -> bool:
  """What is computed of them has a gradient, which the kernels do not give."""
  return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _c_strides(c: PagedKV):
  out = []
  for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
    out += [t.stride(0), t.stride(1), t.stride(2)] + ([s.stride(0), s.stride(1), s.stride(2)] if s is not None else [0, 0, 0])
  return (c_longlong * 12)(*out)


def _move(write: bool, k, v, c: PagedKV, slots):
  pages, page, h, dk = c.k.shape
  t = slots.shape[0]
  st = (c_longlong * 4)(k.stride(0), k.stride(1), v.stride(0), v.stride(1))
  with torch.cuda.device(c.k.device):
    rc = lib().tpb_paged_rows(int(write), ptr(k), ptr(v), ptr(c.k), ptr(c.v), ptr(c.k_scale), ptr(c.v_scale), ptr(slots), t, h, dk,
                              c.v.shape[3], pages, page, st, _c_strides(c), stream_ptr())
  check(rc, f"paged_rows T={t} H={h}")


def _check_slots(op: str, c: PagedKV, slots):
  if slots.dim() != 1 or slots.dtype != torch.int64 or slots.device != c.k.device:
    raise ValueError(f"{op}: slots must be a vector of int64 on the cache's device, got {slots.dtype} {tuple(slots.shape)}")
  _debug.check_index(op, "slots", slots, 0, c.k.shape[0] * c.page, also_allowed=-1)


def _vectors(x):
  """Rows that 16-byte vectors can be read from."""
  return x if x.stride(2) == 1 and x.stride(0) % 8 == 0 and x.stride(1) % 8 == 0 and x.data_ptr() % 16 == 0 else x.contiguous()


def append(cache: PagedKV, k, v, slots):
  """Writes keys [T, H, Dk] and values [T, H, Dv] to the rows ``slots`` [T] (int64) of the cache, quantised where it is
  e4m3; a token of slot -1 (padding) is not written, and neither is one whose slot lies outside the pool, which the kernel
  reports (``_lib.raise_on_device_timeout``).  No slot may come twice: which of its tokens a row of it holds is not defined."""
  if (nat := functional._native()) is not None and nat.paged_append(*cache, k, v, slots):
    return
  _check_cache(cache)
  _check_slots("paged_append", cache, slots)
  t, h = slots.shape[0], cache.k.shape[2]
  if k.shape != (t, h, cache.k.shape[3]) or v.shape != (t, h, cache.v.shape[3]):
    raise ValueError(f"paged_append: keys {tuple(k.shape)} and values {tuple(v.shape)} for {t} slots of {tuple(cache.k.shape)} "
                     f"and {tuple(cache.v.shape)}")
  if k.device != cache.k.device or v.device != cache.k.device:
    raise ValueError("paged_append: keys and values must be on the cache's device")
  if _debug.bounds_enabled() and not (slots.is_cuda and torch.cuda.is_current_stream_capturing()):
    used = slots[slots >= 0]
    if used.unique().numel() != used.numel():
      raise IndexError("paged_append: a slot comes twice")
  if use_kernels(k, v) and k.is_cuda and unobserved() and _rows_ok(cache, h, k.shape[2], v.shape[2]):
    _move(True, _vectors(k.detach()), _vectors(v.detach()), cache, slots.contiguous())
    torch.autograd.graph.increment_version([t for t in cache if t is not None])      # an earlier graph that saved a pool has to notice
    return
  with torch.no_grad():
    for pool, scale, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
      ref.paged_append(pool, scale, x, slots)


def read(cache: PagedKV, slots, dtype=torch.bfloat16):
  """The rows ``slots`` [T] of the cache as (keys [T, H, Dk], values [T, H, Dv]) of ``dtype``; zeros for slot -1 and, reported as in
  :func:`append`, for slots outside the pool."""
  if dtype == torch.bfloat16 and (nat := functional._native()) is not None:
    rows = nat.paged_read(*cache, slots)
    if rows is not None:
      return rows
  _check_cache(cache)
  _check_slots("paged_read", cache, slots)
  h, dk, dv = cache.k.shape[2], cache.k.shape[3], cache.v.shape[3]
  if (slots.is_cuda and dtype == torch.bfloat16 and use_kernels() and unobserved() and not _recorded(*cache)
      and _rows_ok(cache, h, dk, dv)):
    k = torch.empty(slots.shape[0], h, dk, dtype=dtype, device=slots.device)
    v = torch.empty(slots.shape[0], h, dv, dtype=dtype, device=slots.device)
    _move(False, k, v, cache, slots.contiguous())
    return k, v
  return ref.paged_read(cache.k, cache.k_scale, slots).to(dtype), ref.paged_read(cache.v, cache.v_scale, slots).to(dtype)


# ----------------------------------------------------------------------------- attention over the pages
_DECODE_DIMS = ((128, 128), (192, 128), (64, 64))


def _decode_ok(q, c: PagedKV) -> bool:
  """What the attention kernel takes: see :func:`decode_attention`."""
  return (c.page % 16 == 0 and c.k.shape[0] > 0 and (c.k.shape[3], c.v.shape[3]) in _DECODE_DIMS and q.shape[1] <= 65535 and q.shape[0] <= 1 << 24
          and _rows_ok(c, c.k.shape[2], c.k.shape[3], c.v.shape[3])
          and all(0 < s for t in c[:2] for s in t.stride()[:3])
          and (c.k.dtype != E4M3 or all(s.stride(1) == 1 and s.stride(0) % 16 == 0 and s.stride(2) % 16 == 0 and s.data_ptr() % 16 == 0
                                        for s in c[2:])))


def decode_attention(q, cache: PagedKV, block_table, lengths, scale=None, window=None, softcap=None):
  """softmax(q K^T * scale + mask) V for one token per sequence: q [B, Hq, Dk], Hq a multiple of the cache's heads, over the
  ``lengths[b]`` tokens (int32) that ``block_table[b]`` (int32 [B, pages]) names, of which ``window`` leaves the last ones;
  ``softcap`` makes scores ``softcap * tanh(score / softcap)``.  Returns [B, Hq, Dv] in q's type; a sequence of no token gives zeros.

  The kernel takes bf16 queries, pools of bf16 or e4m3 whose pages are multiples of 16 tokens, and heads of 128, 192 / 128 or
  64 columns; sequences x key heads (one for each sixteen of its query heads) x the tokens that a row of the table can name may come to
  2^35 (2^36 of 128 columns in all and fewer).  It looks only at entries of the table and pages that hold a visible token, and what a
  page holds beside them may be anything; a page outside the pool counts as zeros, a length beyond the table as the whole table, a
  negative one as none, and all three are reported (``_lib.raise_on_device_timeout``)."""
  if (nat := functional._native()) is not None:
    o = nat.paged_decode(q, *cache, block_table, lengths, scale, window, softcap)
    if o is not None:
      return o
  _check_cache(cache)
  if q.dim() != 3 or q.shape[2] != cache.k.shape[3] or q.shape[1] % cache.k.shape[2] or q.shape[1] == 0:
    raise ValueError(f"decode_attention: queries {tuple(q.shape)} over keys {tuple(cache.k.shape)}")
  b, hq, dk = q.shape
  if block_table.dim() != 2 or block_table.shape[0] != b or lengths.shape != (b,):
    raise ValueError(f"decode_attention: block_table {tuple(block_table.shape)} and lengths {tuple(lengths.shape)} for {b} sequences")
  if block_table.dtype != torch.int32 or lengths.dtype != torch.int32:
    raise ValueError("decode_attention: block_table and lengths must be int32")
  if any(t.device != cache.k.device for t in (q, block_table, lengths)):
    raise ValueError("decode_attention: queries, block_table and lengths must be on the cache's device")
  window, softcap = int(window or 0), float(softcap or 0.0)
  scale = float(scale) if scale is not None else dk ** -0.5
  if window < 0 or not 0.0 <= softcap < float("inf"):
    raise ValueError(f"decode_attention: window {window}, softcap {softcap}")
  if softcap:
    softcap = max(softcap, 2.0 ** -60)       # (no score is told from another by less, and fp32 holds what it is divided by)
  _debug.check_index("decode_attention", "lengths", lengths, 0, block_table.shape[1] * cache.page + 1)
  if (use_kernels(q) and q.is_cuda and _decode_ok(q, cache) and block_table.shape[1] * cache.page <= 0x7fffff00 and unobserved()
      and not _recorded(q, *cache) and softcap <= 2.0 ** 60):      # (quotients by more would be flushed)
    q, lengths = _vectors(q), lengths.contiguous()
    block_table = block_table if block_table.stride(1) == 1 else block_table.contiguous()
    pages, page, hkv, _ = cache.k.shape
    dv, width = cache.v.shape[3], block_table.shape[1]
    out = torch.empty(b, hq, dv, dtype=q.dtype, device=q.device)
    with torch.cuda.device(q.device):
      n = lib().tpb_paged_decode_scratch(b, hkv, hq // hkv, dk, dv, int(cache.k.dtype == E4M3), width * page)
      scratch = torch.empty(n, dtype=torch.uint8, device=q.device)
      rc = lib().tpb_paged_decode(ptr(q), q.stride(0), q.stride(1), ptr(cache.k), ptr(cache.v), ptr(cache.k_scale), ptr(cache.v_scale),
                                  _c_strides(cache), ptr(block_table), block_table.stride(0), width, ptr(lengths), ptr(out),
                                  ptr(scratch), b, hkv, hq // hkv, dk, dv, pages, page, min(window, 2 ** 31 - 1), scale, softcap, stream_ptr())
    check(rc, f"paged_decode q{tuple(q.shape)} pool{tuple(cache.k.shape)}")
    return out
  return ref.paged_attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, block_table, lengths, scale, window, softcap)
