"""KV-cached inference for the DeepSeek-V3 family on top of the training model's weights.

Capability reference: torchprime/experimental/torchax_models/deepseek_v3/model.py:307-449 (MLA with
a ``naive`` cache of full keys/values or an ``absorb`` cache of the compressed latent) and
:718-773 (``Transformer.forward(tokens, start_pos)`` returning the logits of the last position).

The engine does not re-declare the network: it walks the layers of a
``DeepseekV3ForCausalLM`` and replaces only the attention core with a cached one, so a
checkpoint trained or converted for the training model serves as is.  Three cache layouts:

* ``naive``  - per layer K ``[B, S, H, dn+dr]`` and V ``[B, S, H, dv]``;
* ``absorb`` - per layer the normalised latent ``[B, S, kv_lora_rank]`` and the shared rotary
  key ``[B, S, dr]``.  The up-projection of keys is folded into the query and the
  up-projection of values is applied after the weighted sum, so a decode step reads
  ``kv_lora_rank + dr`` numbers per cached token instead of ``H * (dn + dr + dv)`` (576 against
  40960 for the 671B model) — on a bandwidth-bound decode that ratio is the speed-up.
* ``paged``  - keys and values as in ``naive``, in a pool of pages for each layer (``ops/paged_kv.py``), bf16 or, with
  ``cache_dtype=torch.float8_e4m3fn``, in 8 bits.  A sequence takes pages as it grows and sequences stand at positions of their
  own, so a batch of prompts of different lengths decodes without padding.

Prefill at position 0 with the ``naive`` layout goes through the flash-attention kernel and a bf16
decode step of the ``absorb`` layout through the kernels of ``ops/mla_decode.py``, one of the ``paged`` layout through
``ops/paged_kv.decode_attention``; everything else uses batched matrix products over the cache.
"""

from __future__ import annotations

import functools

import torch

from ...ops import functional as ops
from ...ops import mla_decode, paged_kv
from ...ops import reference as ref


class DeepseekInferenceEngine:
  def __init__(self, model, max_batch_size: int = 1, max_seq_len: int = 4096, attn_impl: str = "absorb",
               cache_dtype=None, page_size: int = 64, num_pages: int | None = None):
    """``page_size`` tokens to a page and ``num_pages`` in all (default: enough for every sequence at its longest) are the
    ``paged`` cache's."""
    assert attn_impl in ("naive", "absorb", "paged"), attn_impl
    self.model = model.eval()
    self.cfg = model.config
    self.attn_impl = attn_impl
    self.max_batch_size = max_batch_size
    self.max_seq_len = max_seq_len
    p = next(model.parameters())
    self.device, self.dtype = p.device, cache_dtype or p.dtype
    a0 = model.model.layers[0].self_attn
    h, dn, dr, dv, c = a0.num_heads, a0.qk_nope_head_dim, a0.qk_rope_head_dim, a0.v_head_dim, a0.kv_lora_rank
    n = len(model.model.layers)
    mk = lambda *shape: torch.zeros(*shape, device=self.device, dtype=self.dtype)  # noqa: E731
    if attn_impl == "naive":
      self.k_cache = [mk(max_batch_size, max_seq_len, h, dn + dr) for _ in range(n)]
      self.v_cache = [mk(max_batch_size, max_seq_len, h, dv) for _ in range(n)]
    elif attn_impl == "paged":
      width = -(-max_seq_len // page_size)
      num_pages = num_pages if num_pages is not None else max_batch_size * width
      self.page_size, self.pages = page_size, [
        paged_kv.PagedKV.allocate(num_pages, page_size, h, dn + dr, dv, dtype=self.dtype, device=self.device) for _ in range(n)]
      self._free, self._owned = list(range(num_pages))[::-1], [[] for _ in range(max_batch_size)]
      self._written = [0] * max_batch_size         # tokens of each sequence
      self._table = torch.zeros(max_batch_size, width, dtype=torch.int32)      # on the host; a step takes the rows that it needs
    else:
      self.kv_cache = [mk(max_batch_size, max_seq_len, c) for _ in range(n)]
      self.pe_cache = [mk(max_batch_size, max_seq_len, dr) for _ in range(n)]
    self.cos, self.sin = model.model.rope_tables(max_seq_len, self.device)

  def cache_bytes(self) -> int:
    if self.attn_impl == "paged":
      return sum(c.nbytes() for c in self.pages)
    bufs = (self.k_cache + self.v_cache) if self.attn_impl == "naive" else (self.kv_cache + self.pe_cache)
    return sum(t.numel() * t.element_size() for t in bufs)

  # ------------------------------------------------------------------------------------- pages
  def release(self, rows=None):
    """Gives back the pages of the sequences ``rows`` (default: of all)."""
    for r in range(self.max_batch_size) if rows is None else rows:
      self._free += self._owned[r][::-1]
      self._owned[r] = []
      self._written[r] = 0

  def _step(self, rows, starts, s: int):
    """Pages for ``s`` tokens more of each sequence, and where a step finds them: slots of the new tokens [B * s], table [B, pages]
    and lengths [B] with them."""
    p, ends = self.page_size, [st + s for st in starts]
    need = [max(0, -(-e // p) - (len(self._owned[r]) if st else 0)) for r, st, e in zip(rows, starts, ends)]
    for r, st in zip(rows, starts):
      assert st <= self._written[r], f"sequence {r} has {self._written[r]} tokens, not all in front of position {st}"
    spare = len(self._free) + sum(len(self._owned[r]) for r, st in zip(rows, starts) if not st)
    if sum(need) > spare:
      raise RuntimeError(f"the cache is full: {sum(need)} pages are needed, {spare} are free")
    self.release(r for r, st in zip(rows, starts) if not st)
    for r, n, e in zip(rows, need, ends):
      for _ in range(n):
        self._table[r, len(self._owned[r])] = self._free[-1]
        self._owned[r].append(self._free.pop())
      self._written[r] = max(self._written[r], e)
    pos = torch.tensor(starts)[:, None] + torch.arange(s)
    table = self._table[rows, : max(len(self._owned[r]) for r in rows)]
    slots = table.long().gather(1, pos // p) * p + pos % p
    to = lambda t: t.to(self.device, non_blocking=True)  # noqa: E731
    return to(slots.reshape(-1)), to(table), to(torch.tensor(ends, dtype=torch.int32))

  def _paged(self, li: int, attn, q4, k, v, starts, step):
    """Attention of the new tokens (their keys and values are written to the cache first), [B, S, H, dv]."""
    b, s, h, _ = q4.shape
    slots, table, lengths = step
    cache = self.pages[li]
    paged_kv.append(cache, k.reshape(b * s, h, -1), v.reshape(b * s, h, -1), slots)
    if s == 1:
      return paged_kv.decode_attention(q4[:, 0], cache, table, lengths, scale=attn.scaling)[:, None]
    if not any(starts):
      if q4.is_cuda and s >= 128:
        return ops.attention(q4, k.reshape(b, s, h, -1), v.reshape(b, s, h, -1), causal=True, scale=attn.scaling)
      return ref.attention(q4, k.reshape(b, s, h, -1), v.reshape(b, s, h, -1), causal=True, scale=attn.scaling)
    out = []
    for i, start in enumerate(starts):      # the part of a prompt behind what is in the cache
      pos = torch.arange(start + s, device=q4.device)
      kc, vc = paged_kv.read(cache, table[i].long()[pos // self.page_size] * self.page_size + pos % self.page_size, dtype=q4.dtype)
      kc[start:], vc[start:] = k.view(b, s, h, -1)[i], v.view(b, s, h, -1)[i]
      out.append(ref.attention(q4[i:i + 1], kc[None], vc[None], causal=True, scale=attn.scaling))
    return torch.cat(out)

  # -------------------------------------------------------------------------------------
  def _attention(self, li: int, attn, x, start: int, residual, positions, step=None):
    b, s, _ = x.shape
    end = start + s if step is None else None
    h, dn, dr, dv, c = attn.num_heads, attn.qk_nope_head_dim, attn.qk_rope_head_dim, attn.v_head_dim, attn.kv_lora_rank
    if not attn.q_lora_rank and attn.kv_a_proj_with_mqa.bias is None:
      q, ckv = ops.linear_pair(x, attn.q_proj.weight, attn.kv_a_proj_with_mqa.weight)
    else:
      q = ops.linear(x, attn.q_proj.weight) if not attn.q_lora_rank else ops.linear(
        attn.q_a_layernorm(ops.linear(x, attn.q_a_proj.weight, bias=attn.q_a_proj.bias)), attn.q_b_proj.weight)
      ckv = ops.linear(x, attn.kv_a_proj_with_mqa.weight, bias=attn.kv_a_proj_with_mqa.bias)
    norm = attn.kv_a_layernorm
    if self.attn_impl == "absorb" and mla_decode.supported(q, ckv, norm.weight, self.kv_cache[li], self.pe_cache[li],
                                                           attn.kv_b_proj.weight, h, dn, dr, dv, c):
      o = mla_decode.absorb_step(q, ckv, norm.weight, norm.variance_epsilon, self.cos, self.sin, start,
                                 self.kv_cache[li], self.pe_cache[li], attn.kv_b_proj.weight, h, dn, dv, attn.scaling,
                                 attn.rope_interleave)
      return ops.linear(o, attn.o_proj.weight, bias=attn.o_proj.bias, residual=residual)
    pos = positions()
    q = ops.rope_slices(q, self.cos, self.sin, h, dr, s, col0=dn, head_stride=dn + dr, pos=pos,
                        interleaved=attn.rope_interleave)
    latent, k_rot = ops.latent_split_rope(ckv, c, self.cos, self.sin, s, pos=pos, interleaved=attn.rope_interleave)
    latent = norm(latent)
    q4 = q.view(b, s, h, dn + dr)

    def mask(scores):          # keys after a query's own position
      if s == 1:
        return scores
      t = torch.arange(end, device=x.device)
      causal = t[None, :] > (start + torch.arange(s, device=x.device))[:, None]          # [s, end]
      return scores.masked_fill(causal[None, :, None, :], float("-inf"))

    if self.attn_impl == "paged":
      k, v = ops.mla_pack(ops.linear(latent, attn.kv_b_proj.weight), k_rot, h, dn, dv)
      o = self._paged(li, attn, q4, k, v, start, step)
    elif self.attn_impl == "naive":
      kv, k, v = ops.linear(latent, attn.kv_b_proj.weight), self.k_cache[li][:b, start:end], self.v_cache[li][:b, start:end]
      prefill = start == 0 and x.is_cuda and s >= 128
      if prefill and (b > 1 or self.dtype != x.dtype):     # the attention kernel takes rows of a batch back to back
        k, v = ops.mla_pack(kv, k_rot, h, dn, dv)
        self.k_cache[li][:b, start:end] = k
        self.v_cache[li][:b, start:end] = v
      else:
        ops.mla_pack_into(kv, k_rot, h, dn, dv, k, v)
      if prefill:
        o = ops.attention(q4, k, v, causal=True, scale=attn.scaling)
      else:
        kc, vc = self.k_cache[li][:b, :end], self.v_cache[li][:b, :end]
        scores = mask(torch.einsum("bshd,bthd->bsht", q4.float(), kc.float()) * attn.scaling)
        o = torch.einsum("bsht,bthd->bshd", scores.softmax(-1), vc.float()).to(x.dtype)
    else:
      w = attn.kv_b_proj.weight.view(h, dn + dv, c)
      self.kv_cache[li][:b, start:end] = latent
      self.pe_cache[li][:b, start:end] = k_rot
      q_abs = torch.einsum("bshd,hdc->bshc", q4[..., :dn].float(), w[:, :dn].float())
      lc, pc = self.kv_cache[li][:b, :end].float(), self.pe_cache[li][:b, :end].float()
      scores = mask((torch.einsum("bshc,btc->bsht", q_abs, lc)
                     + torch.einsum("bshr,btr->bsht", q4[..., dn:].float(), pc)) * attn.scaling)
      o_lat = torch.einsum("bsht,btc->bshc", scores.softmax(-1), lc)
      o = torch.einsum("bshc,hdc->bshd", o_lat, w[:, dn:].float()).to(x.dtype)
    o = o.reshape(b, s, h * dv)
    return ops.linear(o, attn.o_proj.weight, bias=attn.o_proj.bias, residual=residual)

  @torch.no_grad()
  def forward(self, tokens: torch.Tensor, start_pos=0, rows=None) -> torch.Tensor:
    """tokens [B, S] at positions ``start_pos .. start_pos+S-1`` -> logits [B, vocab] of the last one.  With the ``paged`` cache
    ``start_pos`` may be a list, one for each sequence, and ``rows`` says which sequences of the cache these are (default: the
    first B); one that starts at position 0 begins anew."""
    b, s = tokens.shape
    step = None
    if self.attn_impl == "paged":
      rows = list(range(b)) if rows is None else list(rows)
      start_pos = [start_pos] * b if isinstance(start_pos, int) else [int(p) for p in start_pos]
      assert len(rows) == len(start_pos) == b and len(set(rows)) == b and 0 <= min(rows) and max(rows) < self.max_batch_size, (rows, b)
      assert min(start_pos) >= 0 and max(start_pos) + s <= self.max_seq_len, (start_pos, s)
      step = self._step(rows, start_pos, s)
    else:
      assert rows is None and b <= self.max_batch_size and start_pos + s <= self.max_seq_len, (b, start_pos, s)
    m = self.model.model
    h = m.embed_tokens(tokens.to(self.device))

    @functools.cache
    def positions():       # of every token, for the layers that need them as a tensor
      if step is not None:
        return (torch.tensor(start_pos, dtype=torch.int32)[:, None] + torch.arange(s, dtype=torch.int32)).reshape(-1).to(self.device)
      return (start_pos + torch.arange(s, device=self.device, dtype=torch.int32)).repeat(b).contiguous()

    for li, layer in enumerate(m.layers):
      h = self._attention(li, layer.self_attn, layer.input_layernorm(h), start_pos, h, positions, step)
      h = layer.mlp(layer.post_attention_layernorm(h), residual=h)
    last = m.norm(h[:, -1:, :].contiguous())
    return ops.linear_f32(last[:, 0], self.model.lm_head.weight)

  __call__ = forward


def full_forward_last_logits(model, tokens: torch.Tensor) -> torch.Tensor:
  """Uncached oracle: the training model's own forward, last position (used by tests)."""
  with torch.no_grad():
    out = model(tokens)
  logits = out[0] if isinstance(out, (tuple, list)) else out
  return logits[:, -1].float()


__all__ = ["DeepseekInferenceEngine", "full_forward_last_logits", "ref"]
