"""Norms of query and key heads with the rotation, the scaled embedding and dropout: definitions, gradients and refusals."""

import pytest
import torch

from torchprime_b200.models.llama4 import Llama4TextL2Norm
from torchprime_b200.ops import functional as ops
from torchprime_b200.ops import reference as ref

F64 = torch.float64


def _tables(n, half):
  angle = torch.arange(n, dtype=F64)[:, None] * 100.0 ** (-torch.arange(half, dtype=F64) / half)
  return angle.cos(), angle.sin()


def _qkv(b, s, hq, hkv, d, seed=0):
  return torch.randn(b, s, (hq + 2 * hkv) * d, dtype=F64, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [8, 4])
@pytest.mark.parametrize("positions", [False, True])
def test_qk_norm_rope_is_its_formula(interleaved, rot, positions):
  """A head at a time, its pairs as complex numbers."""
  b, s, hq, hkv, d = 2, 3, 4, 2, 8
  x, (cos, sin) = _qkv(b, s, hq, hkv, d), _tables(9, rot // 2)
  wq, wk = torch.rand(d, dtype=F64) + 0.5, torch.rand(d, dtype=F64) + 0.5
  pos = torch.tensor([[8, 0, 3], [1, 1, 7]], dtype=torch.int32) if positions else None
  q, k, v = ops.qk_norm_rope(x, cos, sin, hq, hkv, d, s, wq, wk, eps=1e-3, pos=pos, interleaved=interleaved)
  assert q.shape == (b, s, hq, d) and k.shape == v.shape == (b, s, hkv, d)
  heads = x.view(b, s, -1, d)
  assert torch.equal(v, heads[:, :, hq + hkv:])
  for i in range(b):
    for j in range(s):
      p = int(pos[i, j]) if positions else j
      for h in range(hq + hkv):
        one = heads[i, j, h] / (heads[i, j, h].square().mean() + 1e-3).sqrt() * (wq if h < hq else wk)
        at = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        z = torch.complex(one[at[0]], one[at[1]]) * torch.complex(cos[p], sin[p])
        one[at[0]], one[at[1]] = z.real, z.imag
        assert torch.allclose((q[i, j, h] if h < hq else k[i, j, h - hq]), one, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("weights", [True, False])
@pytest.mark.parametrize("interleaved", [False, True])
def test_qk_norm_rope_gradients(weights, interleaved):
  """Against differences, and the formulas against autograd's."""
  b, s, hq, hkv, d = 1, 3, 2, 1, 8
  x, (cos, sin) = _qkv(b, s, hq, hkv, d, 1).requires_grad_(), _tables(5, 3)
  ws = [(torch.rand(d, dtype=F64) + 0.5).requires_grad_() if weights else None for _ in range(2)]
  inputs = [x] + [w for w in ws if w is not None]
  fn = lambda x, wq=None, wk=None: ops.qk_norm_rope(x, cos, sin, hq, hkv, d, s, wq, wk, eps=1e-2, interleaved=interleaved)  # noqa: E731
  assert torch.autograd.gradcheck(fn, inputs) and torch.autograd.gradgradcheck(fn, inputs)
  out = fn(*inputs)
  grads = [torch.randn_like(t) for t in out]
  want = torch.autograd.grad(out, inputs, grads)
  got = ref.qk_norm_rope_grad(*grads, x, cos, sin, hq, hkv, d, s, *ws, 1e-2, None, interleaved)
  for a, w in zip([g for g in got if g is not None], want):
    assert torch.allclose(a, w, rtol=1e-10, atol=1e-12)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_qk_norm_rope_without_weights_is_the_norm_behind_the_rotation(dtype):
  """Llama-4's order: a rotation does not change a head's mean square.  (bf16: the other way rounds twice more.)"""
  b, s, hq, hkv, d = 2, 5, 4, 2, 16
  x, (cos, sin) = _qkv(b, s, hq, hkv, d, 2).to(dtype), (t.float() for t in _tables(5, 8))
  norm = Llama4TextL2Norm(1e-5)
  rotated = ops.rope_inplace(x.clone(), cos, sin, hq + hkv, d, s, interleaved=True)
  q, k, _ = ops.qk_norm_rope(x, cos, sin, hq, hkv, d, s, eps=1e-5, interleaved=True)
  got, want = torch.cat([q, k], 2), norm(rotated[..., : (hq + hkv) * d].view(b, s, -1, d))
  assert got.dtype == dtype
  # values up to 4 = sqrt(d): three roundings to bf16 and the change of the statistics by one of them
  assert (got.double() - want.double()).abs().max() <= (4 * 4 * 2.0 ** -8 if dtype == torch.bfloat16 else 1e-5)


def test_qk_norm_rope_counts_positions_outside_as_the_nearest():
  x, (cos, sin) = _qkv(1, 3, 1, 1, 8), _tables(4, 4)
  at = lambda p: ops.qk_norm_rope(x, cos, sin, 1, 1, 8, 3, pos=torch.tensor([p]))[0]  # noqa: E731
  assert torch.equal(at([-5, 1, 9]), at([0, 1, 3]))


def test_qk_norm_rope_refusals(monkeypatch):
  x, (cos, sin) = _qkv(2, 3, 2, 1, 8), _tables(5, 4)
  call = lambda x=x, cos=cos, sin=sin, hq=2, hkv=1, d=8, seq=3, **kw: ops.qk_norm_rope(x, cos, sin, hq, hkv, d, seq, **kw)  # noqa: E731
  call()
  w = torch.ones(8, dtype=F64)
  for bad in (dict(hq=3), dict(hq=4, hkv=0), dict(d=16), dict(x=x[0]), dict(cos=cos[:4]), dict(cos=cos[0], sin=sin[0]),
              dict(cos=torch.ones(5, 5), sin=torch.ones(5, 5)), dict(cos=cos[:, :0], sin=sin[:, :0]), dict(cos=cos[:0], sin=sin[:0]),
              dict(seq=6), dict(seq=0), dict(q_weight=w[:4]), dict(k_weight=w[None]), dict(eps=-1e-6), dict(eps=float("nan")),
              dict(eps=float("inf")), dict(pos=torch.zeros(5, dtype=torch.int32)), dict(pos=torch.zeros(6)),
              dict(q_weight=torch.ones(8, device="meta"))):
    with pytest.raises(ValueError):
      call(**bad)
  monkeypatch.setenv("TPB_DEBUG_BOUNDS", "1")
  with pytest.raises(IndexError, match="pos"):
    call(pos=torch.tensor([[0, 1, 2], [3, 4, 5]]))


# Published known answers of Philox4x32-10: counter, key, words.
KNOWN = [((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
         ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
         ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))]


@pytest.mark.parametrize("counter,key,words", KNOWN)
def test_generator_has_its_known_answers(counter, key, words):
  assert ref.philox(counter, key) == words
  t = lambda v: tuple(torch.tensor([x]) for x in v)  # noqa: E731
  assert tuple(int(w) for w in ref.philox(t(counter), t(key))) == words


def test_dropout_keeps_what_the_generator_says():
  """Element i by the i % 8-th 16 bits at i // 8, the low half of a word first; seeds with a sign, too."""
  for seed, step, site in ((5, 7, 0), (-3, 2 ** 33 + 1, 2 ** 32 - 1)):
    x = torch.arange(1.0, 28.0).view(3, 9)
    y = ops.dropout(x, 0.3, torch.tensor([seed, step]), site=site)
    t = round(0.3 * 65536)
    for i in range(27):
      w = ref.philox((i // 8, 0, step % 2 ** 32, site), (seed % 2 ** 32, seed % 2 ** 64 >> 32))
      keep = (w[i % 8 // 2] >> 16 * (i % 2) & 0xFFFF) >= t
      assert float(y.view(-1)[i]) == (pytest.approx((i + 1) * 65536 / (65536 - t), rel=2e-7) if keep else 0.0)


@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
def test_dropout_drops_that_many(p):
  """Of 2^18 elements within five standard deviations; other steps, sites and seeds drop others, about as many in common as chance has."""
  n = 2 ** 18
  x, seed = torch.ones(n), torch.tensor([11, 0])
  masks = [ops.dropout(x, p, s, site=k) > 0 for s, k in ((seed, 0), (seed + 1, 0), (torch.tensor([11, 1]), 0), (seed, 1))]
  for m in masks:
    assert abs(int((~m).sum()) - p * n) < 5 * (n * p * (1 - p)) ** 0.5
  for m in masks[1:]:
    both = p * p
    assert abs(int((~m & ~masks[0]).sum()) - both * n) < 5 * (n * both * (1 - both)) ** 0.5
  assert torch.equal(ops.dropout(x, p, seed) > 0, masks[0])


def test_dropout_gradients_and_ends():
  seed = torch.tensor([3, 4])
  x, r = (torch.randn(5, 7, dtype=F64).requires_grad_() for _ in range(2))
  fn = lambda x, r: ops.dropout(x, 0.4, seed, site=2, residual=r)  # noqa: E731
  assert torch.autograd.gradcheck(fn, (x, r)) and torch.autograd.gradgradcheck(fn, (x, r))
  assert torch.equal(fn(x, r), ops.dropout(x, 0.4, seed, site=2) + r)
  assert ops.dropout(x, 0.4, seed, training=False) is x and ops.dropout(x, 0.0, seed) is x
  assert torch.equal(ops.dropout(x, 0.0, seed, residual=r), x + r)
  bad = torch.full((9,), float("nan"))
  assert torch.equal(ops.dropout(bad, 1.0, seed), torch.zeros(9)) and torch.equal(ops.dropout(bad, 1.0, seed, residual=torch.ones(9)), torch.ones(9))
  kept = ops.dropout(torch.ones(100), 0.5, seed) > 0
  inf = ops.dropout(torch.full((100,), float("inf")), 0.5, seed)       # what is dropped is 0, whatever it was
  assert torch.equal(inf.isinf(), kept) and not inf[~kept].any()
  assert ops.dropout(torch.empty(0, 4), 0.5, seed).shape == (0, 4)


def test_dropout_refusals():
  x, seed = torch.randn(4, 4), torch.tensor([1, 2])
  for kw in (dict(p=-0.1), dict(p=1.1), dict(p=float("nan")), dict(seed=torch.tensor([1])), dict(seed=torch.tensor([1, 2], dtype=torch.int32)),
             dict(seed=torch.empty(2, dtype=torch.int64, device="meta")), dict(site=-1), dict(site=2 ** 32), dict(residual=torch.randn(4)),
             dict(residual=x.double()), dict(residual=torch.empty(4, 4, device="meta")), dict(x=torch.ones(4, dtype=torch.int64))):
    with pytest.raises(ValueError):
      ops.dropout(**{**dict(x=x, p=0.5, seed=seed), **kw})


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scaled_embedding(dtype):
  table, ids = torch.randn(11, 6, dtype=dtype).requires_grad_(), torch.tensor([[3, 3, 10], [0, 3, 10]])
  y = ops.embedding(ids, table, scale=6 ** 0.5)
  assert y.dtype == dtype and torch.equal(y, (table.detach()[ids].float() * 6 ** 0.5).to(dtype))
  assert torch.equal(ops.embedding(ids, table, scale=1.0), ops.embedding(ids, table)) and torch.equal(ops.embedding(ids, table), table[ids])
  dy = torch.randn(2, 3, 6).to(dtype)
  (g,) = torch.autograd.grad(y, table, dy)
  want = torch.zeros(11, 6, dtype=F64).index_add_(0, ids.view(-1), dy.double().view(-1, 6)) * 6 ** 0.5
  # an id's up to three tokens are each rounded after the product, and their sums
  assert (g.double() - want).abs().max() <= 6 * torch.finfo(dtype).eps / 2 * 6 ** 0.5 * dy.double().abs().sum((0, 1)).max()
  for bad in (float("nan"), float("inf")):
    with pytest.raises(ValueError):
      ops.embedding(ids, table, scale=bad)


def test_llama4_with_the_fused_norms():
  """The model's option gives its logits and gradients (fp32: another order of two products), and is off unless asked for."""
  from torchprime_b200.config import compose
  from torchprime_b200.models.model_utils import initialize_model_class
  size = ["model=llama-4-text-only-dummy", "model.hidden_size=128", "model.num_attention_heads=4", "model.num_key_value_heads=2", "model.head_dim=32",
          "model.intermediate_size=48", "model.intermediate_size_mlp=96", "model.num_local_experts=4", "model.vocab_size=256",
          "model.num_hidden_layers=2", "model.moe_layers=[1]", "model.no_rope_layers=[1,0]"]
  ids = torch.randint(0, 256, (2, 40), generator=torch.Generator().manual_seed(3))
  outs = []
  for extra in ([], ["+model.fused_qk_norm=true"]):
    torch.manual_seed(0)
    m = initialize_model_class(compose("default", size + extra).model)
    assert [layer.self_attn.fused_qk_norm for layer in m.model.layers] == [bool(extra), False]
    logits, loss = m(ids, labels=ids)
    loss.backward()
    outs.append([logits, *(p.grad for p in m.parameters())])
  for a, b in zip(*outs):
    assert torch.allclose(a, b, atol=1e-5)
