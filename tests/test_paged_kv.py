"""Paged cache on the CPU: the definitions, what is refused, and pages and slots that do not exist."""

import pytest
import torch

from torchprime_b200.ops import paged_kv, reference as ref
from torchprime_b200.ops.paged_kv import E4M3, E8M0, PagedKV


def test_quantised_rows_take_the_smallest_power_of_two_that_fits():
  x = torch.tensor([[448.0, 1.0], [449.0, -1.0], [0.0, 0.0], [224.0, 0.5], [2.0 ** -120, 0.0], [1.984375 * 2.0 ** 127, 1.0]])
  q, e = ref.quantise_e4m3(x)
  assert e.dtype == E8M0 and e.view(torch.uint8).tolist() == [127, 128, 127, 126, 27, 247]
  # half a step of four significant bits, and half a step of 2^-9 below 2^-6
  held = q.float() * ref.power_of_two(e.view(torch.uint8).int() - 127)[:, None]
  scale = ref.power_of_two(e.view(torch.uint8).int() - 127)[:, None]
  assert bool(((held - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10))[:5].all())


def test_powers_of_two_are_those_of_their_type():
  """All 256 bytes of e8m0, the ends too: 2^-127 and NaN."""
  c = PagedKV.allocate(16, 16, 1, 16, dtype=E4M3)
  c.k.view(torch.uint8).fill_(0x40), c.v.view(torch.uint8).fill_(0x00)                  # 2, 0
  every = torch.arange(256, dtype=torch.uint8)
  for s in (c.k_scale, c.v_scale):
    s.view(torch.uint8).copy_(every.view(16, 16, 1))
  k, v = paged_kv.read(c, torch.arange(256), dtype=torch.float32)
  want = torch.tensor([2.0 * 2.0 ** (i - 127) for i in range(255)], dtype=torch.float64).float()      # (2^128 is infinity)
  assert torch.equal(k[:255, 0, 0], want) and bool(k[255].isnan().all())
  assert not v[:255].any() and bool(v[255].isnan().all())


def test_quantising_twice_changes_nothing():
  torch.manual_seed(0)
  x = torch.randn(200, 64) * torch.exp2(torch.randn(200, 1) * 8)
  q, e = ref.quantise_e4m3(x)
  held = q.float() * ref.power_of_two(e.view(torch.uint8).int() - 127)[:, None]
  q2, e2 = ref.quantise_e4m3(held)
  again = q2.float() * ref.power_of_two(e2.view(torch.uint8).int() - 127)[:, None]
  assert torch.equal(held, again)


def test_infinities_saturate_and_nan_stays():
  q, e = ref.quantise_e4m3(torch.tensor([[float("inf"), float("-inf"), float("nan"), 3.0]]))
  assert q.float()[0, :2].tolist() == [448.0, -448.0] and q.float()[0, 2].isnan() and q.float()[0, 3] * 2.0 ** (int(e.view(torch.uint8)) - 127) == 3.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_rows_come_back_and_others_stay(dtype):
  torch.manual_seed(1)
  c = PagedKV.allocate(5, 16, 3, 24, 16, dtype=dtype)
  slots = torch.tensor([79, 0, -1, 17, 40])
  k, v = torch.randn(5, 3, 24).bfloat16(), torch.randn(5, 3, 16).bfloat16()
  before = [t.clone() for t in c if t is not None]
  paged_kv.append(c, k, v, slots)
  gk, gv = paged_kv.read(c, slots)
  for got, x in ((gk, k), (gv, v)):
    want = x.float() if dtype == torch.bfloat16 else None
    if want is None:
      q, e = ref.quantise_e4m3(x)
      want = q.float() * ref.power_of_two(e.view(torch.uint8).int() - 127)[..., None]
    assert torch.equal(got[[0, 1, 3, 4]].float(), want[[0, 1, 3, 4]]) and not got[2].any()
  rest = torch.ones(80, dtype=torch.bool)
  rest[slots[slots >= 0]] = False
  for t, b in zip([t for t in c if t is not None], before):
    t8, b8 = t.contiguous().view(torch.uint8).reshape(80, -1), b.contiguous().view(torch.uint8).reshape(80, -1)
    assert torch.equal(t8[rest], b8[rest])


def test_slots_outside_the_pool_are_left_out():
  c = PagedKV.allocate(2, 16, 1, 8)
  x = torch.ones(3, 1, 8).bfloat16()
  paged_kv.append(c, x, x, torch.tensor([32, -7, 31]))
  assert c.k.float().sum() == 8
  k, _ = paged_kv.read(c, torch.tensor([1 << 40, 31]))
  assert not k[0].any() and bool((k[1] == 1).all())


def test_debug_mode_names_bad_and_repeated_slots(monkeypatch):
  monkeypatch.setenv("TPB_DEBUG_BOUNDS", "1")
  c = PagedKV.allocate(2, 16, 1, 8)
  x = torch.ones(2, 1, 8).bfloat16()
  with pytest.raises(IndexError, match="slots"):
    paged_kv.append(c, x, x, torch.tensor([32, 0]))
  with pytest.raises(IndexError, match="twice"):
    paged_kv.append(c, x, x, torch.tensor([3, 3]))
  with pytest.raises(IndexError, match="slots"):
    paged_kv.read(c, torch.tensor([-2]))


def test_refusals():
  c = PagedKV.allocate(2, 16, 1, 8)
  x = torch.ones(2, 1, 8).bfloat16()
  s = torch.tensor([0, 1])
  with pytest.raises(ValueError):
    paged_kv.append(c, x[:1], x, s)
  with pytest.raises(ValueError):
    paged_kv.append(c, x, x, s.int())
  with pytest.raises(ValueError):
    paged_kv.read(c, s[None])
  with pytest.raises(ValueError):
    paged_kv.append(PagedKV(c.k, c.v.to(E4M3)), x, x, s)
  with pytest.raises(ValueError):
    paged_kv.read(PagedKV(c.k.to(E4M3), c.v.to(E4M3)), s)
  for empty in (PagedKV.allocate(0, 16, 1, 8), PagedKV.allocate(2, 0, 1, 8), PagedKV(c.k[0], c.v[0])):
    with pytest.raises(ValueError):
      paged_kv.read(empty, s)
  q = PagedKV.allocate(2, 16, 1, 16, dtype=E4M3)
  with pytest.raises(ValueError):
    paged_kv.read(PagedKV(q.k, q.v, q.k_scale, q.v_scale.view(torch.uint8)), s)


def test_cache_bytes():
  c, q = PagedKV.allocate(4, 16, 2, 64), PagedKV.allocate(4, 16, 2, 64, dtype=E4M3)
  assert c.nbytes() == 4 * 16 * 2 * 128 * 2 and q.nbytes() == 4 * 16 * 2 * (128 + 2)


# ----------------------------------------------------------------------------- attention over the pages
def _dense(q, k, v, n, scale, window=0, softcap=0.0):
  """One sequence against the plain attention definition: keys [S, H, D], the query after all of them."""
  lo = max(0, n - window) if window else 0
  return ref.attention(q[None, None], k[None, lo:n], v[None, lo:n], causal=False, scale=scale, softcap=softcap or None)[0, 0]


@pytest.mark.parametrize("window,softcap", [(0, 0.0), (5, 0.0), (0, 3.0)])
def test_decode_attention_is_attention_over_the_pages(window, softcap):
  torch.manual_seed(2)
  c = PagedKV.allocate(8, 16, 2, 24, 16, dtype=torch.float32)
  c.k.fill_(float("nan"))
  c.v.fill_(float("nan"))
  lens = [40, 1, 0, 16]
  table = torch.full((4, 3), 10 ** 6, dtype=torch.int32)
  table[0], table[1, 0], table[3, 0] = torch.tensor([7, 2, 4]), 1, 6
  q = torch.randn(4, 6, 24)
  rows = {}
  for b, n in enumerate(lens):
    k, v = torch.randn(n, 2, 24), torch.randn(n, 2, 16)
    pos = torch.arange(n)
    paged_kv.append(c, k, v, table[b].long()[pos // 16] * 16 + pos % 16)
    rows[b] = k, v
  got = paged_kv.decode_attention(q, c, table, torch.tensor(lens, dtype=torch.int32), window=window, softcap=softcap)
  for b, n in enumerate(lens):
    want = _dense(q[b], *rows[b], n, 24 ** -0.5, window, softcap) if n else torch.zeros(6, 16)
    assert torch.allclose(got[b], want, atol=1e-5)


def test_decode_attention_refusals():
  c = PagedKV.allocate(4, 16, 2, 8)
  q, table, lens = torch.randn(3, 4, 8).bfloat16(), torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
  assert paged_kv.decode_attention(q, c, table, lens).shape == (3, 4, 8)
  for bad in ((q[:, :3], c, table, lens), (q[..., :4], c, table, lens), (q, c, table[:2], lens), (q, c, table, lens[:2]),
              (q, c, table.long(), lens), (q, c, table, lens.long()), (q[0], c, table, lens), (q[:, :0], c, table, lens)):
    with pytest.raises(ValueError):
      paged_kv.decode_attention(*bad)
  for kw in ({"window": -1}, {"softcap": -2.0}, {"softcap": float("nan")}):
    with pytest.raises(ValueError):
      paged_kv.decode_attention(q, c, table, lens, **kw)


def test_an_infinite_cap_is_refused():
  c = PagedKV.allocate(4, 16, 2, 8)
  with pytest.raises(ValueError, match="softcap"):
    paged_kv.decode_attention(torch.randn(1, 4, 8).bfloat16(), c, torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32),
                              softcap=float("inf"))


def test_debug_mode_names_lengths_beyond_the_table(monkeypatch):
  monkeypatch.setenv("TPB_DEBUG_BOUNDS", "1")
  c = PagedKV.allocate(4, 16, 2, 8)
  with pytest.raises(IndexError, match="lengths"):
    paged_kv.decode_attention(torch.randn(1, 4, 8).bfloat16(), c, torch.zeros(1, 2, dtype=torch.int32), torch.tensor([33], dtype=torch.int32))


# ----------------------------------------------------------------------------- in the inference engine
def _tiny():
  from torchprime_b200.config import compose
  from torchprime_b200.models.model_utils import initialize_model_class
  cfg = compose("default", ["model=deepseek-tiny"]).model
  torch.manual_seed(0)
  return cfg, initialize_model_class(cfg).eval()


def test_paged_engine_matches_the_training_model():
  from torchprime_b200.experimental.deepseek_inference.engine import DeepseekInferenceEngine, full_forward_last_logits
  cfg, model = _tiny()
  eng = DeepseekInferenceEngine(model, max_batch_size=2, max_seq_len=32, attn_impl="paged", page_size=4)
  ids = torch.randint(0, cfg.vocab_size, (2, 12))
  full = lambda n: full_forward_last_logits(model, ids[:, :n])  # noqa: E731
  assert torch.allclose(eng.forward(ids, 0), full(12), atol=2e-4)
  assert torch.allclose(eng.forward(ids[:, :5], 0), full(5), atol=2e-4)          # anew
  assert torch.allclose(eng.forward(ids[:, 5:8], 5), full(8), atol=2e-4)         # the next part of the prompts
  for t in range(8, 12):
    assert torch.allclose(eng.forward(ids[:, t:t + 1], t), full(t + 1), atol=2e-4)
  eng.forward(ids[:1, :3], 0, rows=[1])                                           # sequences at positions of their own
  got = eng.forward(torch.stack([ids[0, 3:4], ids[0, :1]]), [3, 12], rows=[1, 0])
  assert torch.allclose(got[0], full_forward_last_logits(model, ids[:1, :4])[0], atol=2e-4)


def test_paged_engine_takes_and_gives_back_pages():
  from torchprime_b200.experimental.deepseek_inference.engine import DeepseekInferenceEngine
  cfg, model = _tiny()
  eng = DeepseekInferenceEngine(model, max_batch_size=3, max_seq_len=16, attn_impl="paged", page_size=4, num_pages=5)
  ids = torch.randint(0, cfg.vocab_size, (1, 9))
  eng.forward(ids, 0, rows=[2])
  assert len(eng._free) == 2
  with pytest.raises(RuntimeError, match="full"):
    eng.forward(ids, 0, rows=[0])
  assert len(eng._free) == 2 and len(eng._owned[2]) == 3                          # a refusal changes nothing
  eng.forward(ids, 0, rows=[2])
  eng.release([2])
  assert sorted(eng._free) == list(range(5))
  with pytest.raises(AssertionError):
    eng.forward(ids[:, :1], 4, rows=[0])                                          # nothing in front of it


def test_paged_engine_refuses_positions_that_nothing_was_written_in_front_of():
  """A page holds what its last sequence left behind the tokens of this one."""
  from torchprime_b200.experimental.deepseek_inference.engine import DeepseekInferenceEngine, full_forward_last_logits
  cfg, model = _tiny()
  eng = DeepseekInferenceEngine(model, max_batch_size=2, max_seq_len=32, attn_impl="paged", page_size=16)
  ids = torch.randint(0, cfg.vocab_size, (1, 9))
  eng.forward(ids[:, :4], 0)
  with pytest.raises(AssertionError, match="position 6"):
    eng.forward(ids[:, 6:7], 6)
  eng.forward(ids[:, 4:8], 4)                                                     # (the refusal changed nothing)
  assert torch.allclose(eng.forward(ids[:, 3:4], 3), full_forward_last_logits(model, ids[:, :4]), atol=2e-4)      # back, and on again
  assert torch.allclose(eng.forward(ids[:, 8:9], 8), full_forward_last_logits(model, ids[:, :9]), atol=2e-4)
  eng.forward(ids[:, :2], 0)                                                      # anew
  with pytest.raises(AssertionError, match="position 3"):
    eng.forward(ids[:, 3:4], 3)
  eng.release()
  with pytest.raises(AssertionError, match="position 1"):
    eng.forward(ids[:, 1:2], 1)


@pytest.mark.parametrize("dtype", [None, E4M3])
def test_paged_generation(dtype):
  from torchprime_b200.experimental.deepseek_inference.engine import DeepseekInferenceEngine, full_forward_last_logits
  from torchprime_b200.experimental.deepseek_inference.generate import generate
  cfg, model = _tiny()
  eng = DeepseekInferenceEngine(model, 2, 32, "paged", cache_dtype=dtype, page_size=4)
  prompts = [[5, 9, 17, 3], [7, 2]]
  outs = generate(eng, prompts, max_new_tokens=5, eos_id=-5, temperature=0.0)
  assert [len(o) for o in outs] == [5, 5] and sorted(eng._free) == list(range(16))
  if dtype is None:
    for p, o in zip(prompts, outs):
      for i, tok in enumerate(o):
        assert tok == int(full_forward_last_logits(model, torch.tensor([p + o[:i]])).argmax())
  stop = outs[0][2]
  assert generate(eng, prompts[:1], 5, stop, 0.0)[0] == outs[0][: outs[0].index(stop)]
  g = torch.Generator().manual_seed(0)
  assert generate(eng, prompts, 5, -5, 1.0, g, top_k=1) == outs                  # one token left to draw
  assert all(0 <= t < cfg.vocab_size for o in generate(eng, prompts, 4, -5, 1.0, g, top_p=0.9, min_p=0.01) for t in o)


def test_generation_that_the_pages_do_not_suffice_for_gives_them_back():
  from torchprime_b200.experimental.deepseek_inference.engine import DeepseekInferenceEngine
  from torchprime_b200.experimental.deepseek_inference.generate import generate
  _, model = _tiny()
  eng = DeepseekInferenceEngine(model, 2, 32, "paged", page_size=4, num_pages=3)
  with pytest.raises(RuntimeError, match="full"):
    generate(eng, [[5, 9, 17, 3], [7, 2]], max_new_tokens=9, eos_id=-5, temperature=0.0)
  assert sorted(eng._free) == [0, 1, 2]
  assert len(generate(eng, [[5, 9, 17, 3]], max_new_tokens=7, eos_id=-5, temperature=0.0)[0]) == 7


def test_sequences_that_have_ended_give_their_pages_to_the_others():
  from torchprime_b200.experimental.deepseek_inference.engine import DeepseekInferenceEngine
  from torchprime_b200.experimental.deepseek_inference.generate import generate
  _, model = _tiny()
  prompts = [[5, 9, 17, 3], [7, 2]]
  outs = generate(DeepseekInferenceEngine(model, 2, 32, "paged", page_size=4), prompts, 9, -5, 0.0)
  eos = outs[1][0]                                                                # the second ends at once
  assert eos not in outs[0]
  eng = DeepseekInferenceEngine(model, 2, 32, "paged", page_size=4, num_pages=3)  # what the first takes to its end
  assert generate(eng, prompts, 9, eos, 0.0) == [outs[0], []]
  assert sorted(eng._free) == [0, 1, 2]


def test_filters_with_the_other_caches():
  from torchprime_b200.experimental.deepseek_inference.engine import DeepseekInferenceEngine
  from torchprime_b200.experimental.deepseek_inference.generate import generate
  _, model = _tiny()
  eng = DeepseekInferenceEngine(model, 2, 32, "absorb")
  prompts = [[5, 9, 17, 3], [7, 2]]
  assert generate(eng, prompts, 5, -5, 1.0, torch.Generator().manual_seed(1), top_k=1) == generate(eng, prompts, 5, -5, 0.0)


@pytest.mark.parametrize("window,softcap", [(0, 0.0), (7, 0.0), (0, 2.0)])
def test_gradients_of_attention_over_the_pages(window, softcap):
  """Of queries and pools, against the formula in 64 bits over dense rows, and along one direction against differences."""
  torch.manual_seed(4)
  lens, table = [21, 0, 5], torch.tensor([[3, 1], [0, 0], [2, 0]], dtype=torch.int32)
  c = PagedKV.allocate(4, 16, 2, 8, dtype=torch.float32)
  leaves = [torch.randn(3, 4, 8), torch.randn(4, 16, 2, 8), torch.randn(4, 16, 2, 8)]
  do = torch.randn(3, 4, 8)
  n = torch.tensor(lens, dtype=torch.int32)
  def f(q, k, v):
    return (paged_kv.decode_attention(q, c._replace(k=k, v=v), table, n, window=window, softcap=softcap) * do).sum()
  def formula(q, k, v):
    total = 0
    for b, m in enumerate(lens):
      pos = torch.arange(max(0, m - window) if window else 0, m)
      kb, vb = (t[table[b].long()[pos // 16], pos % 16].repeat_interleave(2, 1) for t in (k, v))
      s = torch.einsum("hd,shd->hs", q[b], kb) * 8 ** -0.5
      if softcap:
        s = softcap * torch.tanh(s / softcap)
      total = total + (torch.einsum("hs,shd->hd", s.softmax(-1), vb) * do[b].double()).sum()
    return total
  a, b = [t.clone().requires_grad_() for t in leaves], [t.double().requires_grad_() for t in leaves]
  got, want = torch.autograd.grad(f(*a), a), torch.autograd.grad(formula(*b), b)
  for x, y in zip(got, want):
    assert bool(y.any()) and torch.allclose(x.double(), y, atol=1e-5)                # (sums of up to 21 terms near 1 in fp32)
  way = [torch.randn_like(t) for t in leaves]
  step = 2.0 ** -7                       # rest of the series: step^2 by a third derivative along a way of length ~20; rounding 2^-24 / step
  ends = [f(*[t + s * step * w for t, w in zip(leaves, way)]) for s in (1, -1)]
  along = sum((x * w).sum() for x, w in zip(got, way))
  assert abs(float((ends[0] - ends[1]) / (2 * step) - along)) < 2.0 ** -6 * (1 + abs(float(along)))
