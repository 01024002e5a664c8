"""The next token of every row of logits, drawn by given random numbers (csrc/sampling.cu)."""

from __future__ import annotations

from ctypes import c_double, c_int, c_longlong, c_void_p

import torch

from . import _lib, functional, reference as ref
from ._lib import check, lib, ptr, stream_ptr

P, I, LL, D = c_void_p, c_int, c_longlong, c_double
_lib.register_signature("tpb_sample_tokens", [P, I, LL, P, P, P, P, P, D, I, D, D, P, I, I, P])

MAX_VOCAB = 1 << 18


def _setting(name, t, b, device, dtype):
  """A number, or one for each row."""
  if not torch.is_tensor(t):
    return t
  if t.shape != (b,) or t.device != device or t.dtype != dtype:
    raise ValueError(f"sample_tokens: {name} must be a number or {dtype} [{b}] on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
  return t


def sample_tokens(logits, u, temperature=1.0, top_k=None, top_p=None, min_p=None):
  """Draws a token (int64 [B]) for every row of ``logits`` [B, V] by the numbers ``u`` [B] (fp32, in [0, 1)).

  With w_i = exp((l_i - max l) / temperature): tokens are put in the order of their logits, of equal ones the lowest index
  first, and kept are the first ``top_k`` (0 or None: all), of those the ones with w_i >= ``min_p``, of those the first ones until
  their weights add up to ``top_p`` of what is left (1 or None: all; the first always stays).  The result is the first index, in the order
  of the indices, at which the kept weights' sum exceeds u times their total.  A temperature of 0 takes the first index of the largest
  logit.  NaN counts as -inf; a row without a logit above -inf gives -1.

  The four settings are numbers or one for each row (fp32, ``top_k`` int32).  Rows of up to 2^18 logits in fp32 or bf16 run in
  one kernel, whose weights are good to 2^-34 and whose sums of them are exact: the same call draws the same tokens."""
  if (nat := functional._native()) is not None:
    y = nat.sample_tokens(logits, u, temperature, top_k, top_p, min_p)
    if y is not None:
      return y
  if logits.dim() != 2 or logits.shape[1] == 0 or not logits.is_floating_point():
    raise ValueError(f"sample_tokens: logits must be [B, V], got {logits.dtype} {tuple(logits.shape)}")
  b, v = logits.shape
  if u.shape != (b,) or u.dtype != torch.float32 or u.device != logits.device:
    raise ValueError(f"sample_tokens: u must be fp32 [{b}] on {logits.device}, got {u.dtype} {tuple(u.shape)} on {u.device}")
  temperature = _setting("temperature", temperature, b, logits.device, torch.float32)
  top_k = _setting("top_k", 0 if top_k is None else top_k, b, logits.device, torch.int32)
  top_p = _setting("top_p", 1.0 if top_p is None else top_p, b, logits.device, torch.float32)
  min_p = _setting("min_p", 0.0 if min_p is None else min_p, b, logits.device, torch.float32)
  logits = logits.detach()
  if (logits.is_cuda and functional.get_backend() != "torch" and functional.unobserved() and logits.dtype in (torch.float32, torch.bfloat16)
      and v <= MAX_VOCAB and b < 1 << 26):
    _lib.lib()
    logits = logits if logits.stride(1) == 1 else logits.contiguous()
    out = torch.empty(b, dtype=torch.int64, device=logits.device)
    # (held until the launch: a copy that is let go is the next one's memory)
    rows = [t.contiguous() if torch.is_tensor(t) else None for t in (u, temperature, top_k, top_p, min_p)]
    num = lambda t, other: other if torch.is_tensor(t) else t  # noqa: E731
    with torch.cuda.device(logits.device):
      rc = lib().tpb_sample_tokens(ptr(logits), int(logits.dtype == torch.bfloat16), logits.stride(0), *map(ptr, rows),
                                   float(num(temperature, 1.0)), min(max(int(num(top_k, 0)), 0), v), float(num(top_p, 1.0)),
                                   float(num(min_p, 0.0)), ptr(out), b, v, stream_ptr())
    check(rc, f"sample_tokens {b}x{v}")
    return out
  return ref.sample_tokens(logits, u, temperature, top_k, top_p, min_p)
