"""Norms of query and key heads, the embedding's gradient and dropout where offsets pass 32 bits, over large vocabularies and in
recomputed layers."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from torchprime_b200.ops import functional as ops
from torchprime_b200.ops import kernels as k
from torchprime_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HALF = 2.0 ** -8              # a rounding to bf16
AROUND = 2.0 ** -18           # fp32 around a head: see test_training_ops_gpu


def _fill(*shape, rows=16384):
  t = torch.empty(*shape, device="cuda", dtype=BF16)
  for i in range(0, t.shape[0], rows):
    t[i: i + rows].normal_()
  return t


def _tables(n, half):
  angle = torch.arange(n, device="cuda")[:, None].double() * 10000.0 ** (-torch.arange(half, device="cuda").double() / half)
  return angle.cos().float().contiguous(), angle.sin().float().contiguous()


def test_qk_norm_rope_past_32_bits(cuda_lib):
  """2^31 numbers and more in the projection, the queries and their gradients: the first, middle and last tokens."""
  tokens, hq, hkv, d, s = 209800, 80, 8, 128, 4099
  assert tokens * hq * d > 2 ** 31
  torch.manual_seed(0)
  cos, sin = _tables(s, d // 2)
  x = _fill(tokens, (hq + 2 * hkv) * d)[None].requires_grad_()
  wq, wk = ((1 + 0.3 * torch.randn(d, device="cuda")).to(BF16).requires_grad_() for _ in range(2))
  out = ops.qk_norm_rope(x, cos, sin, hq, hkv, d, s, wq, wk)
  grads = [_fill(*t.shape[1:])[None] for t in out]
  dx, dwq, dwk = torch.autograd.grad(out, (x, wq, wk), grads)
  up = lambda t: t.detach().double()  # noqa: E731
  for at in (slice(0, 40), slice(tokens // 2, tokens // 2 + 40), slice(tokens - 40, tokens)):
    args = (up(cos), up(sin), hq, hkv, d, s, up(wq), up(wk), 1e-6, torch.arange(at.start, at.stop, device="cuda") % s)
    want = ref.qk_norm_rope(up(x[:, at]), *args)
    for y, w in zip(out[:2], want):
      assert bool(((y[:, at].double() - w).abs() <= HALF * w.abs() + AROUND * 2 * w.abs().amax(-1, keepdim=True)).all())
    assert torch.equal(out[2][:, at].double(), want[2])
    want = ref.qk_norm_rope_grad(*(up(g[:, at]) for g in grads), up(x[:, at]), *args)[0].view(1, 40, -1, d)
    n = hq + hkv
    heads = up(x[:, at]).view(1, 40, -1, d)[:, :, :n]
    r = (heads.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    w = torch.cat([up(wq).expand(hq, d), up(wk).expand(hkv, d)])
    g = 2 * torch.cat([up(grads[0][:, at]), up(grads[1][:, at])], 2).abs().amax(-1, keepdim=True) * w.abs()
    size = r * g + heads.abs() * r ** 3 * (g * heads.abs()).mean(-1, keepdim=True)
    got = dx[:, at].view(1, 40, -1, d)
    assert bool(((got[:, :, :n].double() - want[:, :, :n]).abs() <= HALF * want[:, :, :n].abs() + AROUND * size).all())
    assert torch.equal(got[:, :, n:], grads[2][:, at])
  # sums over all heads, a rounding of each term and of the sum beside those of 2^16 parts (terms of both signs: relative to their sizes)
  sums, sizes = [torch.zeros(2, d, device="cuda", dtype=torch.float64) for _ in range(2)]
  for i in range(0, tokens, 4100):
    at = slice(i, min(i + 4100, tokens))
    pos = torch.arange(at.start, at.stop, device="cuda") % s
    c, sn = cos[pos][None, :, None].double(), sin[pos][None, :, None].double()
    for j, (lo, hi) in enumerate(((0, hq), (hq, hq + hkv))):
      h = x.detach()[:, at].view(1, pos.numel(), -1, d)[:, :, lo:hi].double()
      t = ref._turn(grads[j][:, at].double(), c, -sn, False) * h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
      sums[j] += t.sum((0, 1, 2))
      sizes[j] += t.abs().sum((0, 1, 2))
  for got, want, size in zip((dwq, dwk), sums, sizes):
    assert bool(((got.double() - want).abs() <= HALF * want.abs() + 2.0 ** -16 * size).all())


def test_embedding_past_32_bits(cuda_lib):
  """A table of 2^31 numbers and more; ids in its last rows, one of them for a third of the tokens."""
  vocab, dim, tokens = 530007, 4096, 9001
  assert vocab * dim > 2 ** 31
  torch.manual_seed(0)
  table = _fill(vocab, dim, rows=65536).requires_grad_()
  ids = torch.randint(0, vocab, (tokens,), device="cuda")
  ids[::3], ids[1::7] = vocab - 1, 524288
  y = ops.embedding(ids, table, scale=2.5)
  assert torch.equal(y, (table.detach()[ids].float() * 2.5).to(BF16))
  dout = _fill(tokens, dim)
  (got,) = torch.autograd.grad(y, table, dout)
  rows, at = ids.unique(return_inverse=True)
  want, size = (torch.zeros(rows.numel(), dim, device="cuda", dtype=torch.float64).index_add_(0, at, t) for t in
                (dout.double() * 2.5, dout.double().abs() * 2.5))
  count = torch.bincount(at)[:, None].double()
  assert bool(((got[rows].double() - want).abs() <= HALF * want.abs() + (count + 2) * 2.0 ** -24 * size).all())
  others = torch.ones(vocab, dtype=torch.bool, device="cuda").index_fill_(0, rows, False)
  assert int(others.sum()) == vocab - rows.numel()
  for i in range(0, vocab, 65536):
    assert not bool(got[i: i + 65536][others[i: i + 65536]].any())


@pytest.mark.parametrize("tokens", [8191, 8192, 8193, 20011])
def test_embedding_gradient_of_large_vocabularies(cuda_lib, tokens):
  """More sets of ids than multiprocessors, on both sides of 8192 tokens."""
  vocab, dim = 300007, 40
  g = torch.Generator(device="cuda").manual_seed(tokens)
  ids = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
  ids[: tokens // 2], ids[-1], ids[-2] = 299999, vocab - 1, 0
  dout = torch.randn(tokens, dim, generator=g, device="cuda").to(BF16)
  got = torch.full((vocab, dim), float("nan"), device="cuda")
  k.embedding_bwd_(dout, ids, got, overwrite=True)
  want, size = (torch.zeros(vocab, dim, device="cuda", dtype=torch.float64).index_add_(0, ids, t.double()) for t in (dout, dout.abs()))
  count = torch.bincount(ids, minlength=vocab)[:, None].double()
  assert bool(((got.double() - want).abs() <= (count + 2) * 2.0 ** -24 * size).all())


def test_dropout_past_32_bits(cuda_lib):
  """Numbers behind the 2^32-th have bits of their own; windows around the powers of two and the end."""
  n = 2 ** 32 + 8 * 1001 + 3
  x, seed, t = torch.ones(n, device="cuda", dtype=BF16), torch.tensor([7, 9], device="cuda"), 16384
  y = ops.dropout(x, 0.25, seed, site=3)
  for at in (0, 2 ** 31 - 64, 2 ** 32 - 64, n // 8 * 8 - 256):
    i = torch.arange(at // 8, min(at // 8 + 33, (n + 7) // 8), device="cuda")
    low = 0xFFFFFFFF
    words = ref.philox((i & low, i >> 32, (seed[1] & low).expand_as(i), torch.full_like(i, 3)), (seed[0] & low, seed[0] >> 32 & low))
    keep = (torch.stack([half for w in words for half in (w & 0xFFFF, w >> 16)], -1).reshape(-1) >= t)[: n - at]
    assert torch.equal(y[at: at + keep.numel()], ref.dropout(x[: keep.numel()], keep, t))


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed(cuda_lib, reentrant):
  """A layer that is recomputed in the backward pass drops the same elements and has the same gradients, to the bit."""
  g = torch.Generator(device="cuda").manual_seed(4)
  cos, sin = _tables(33, 32)
  seed, ids = torch.tensor([5, 6], device="cuda"), torch.randint(0, 50, (2, 33), generator=g, device="cuda")
  table, w = ((torch.randn(*shape, generator=g, device="cuda")).to(BF16).requires_grad_() for shape in ((50, 256), (64,)))
  x = torch.randn(2, 33, 256, generator=g, device="cuda").to(BF16).requires_grad_()

  def layer(x):
    h = ops.dropout(ops.embedding(ids, table, scale=3.0), 0.3, seed, site=1, residual=x)
    return torch.cat(ops.qk_norm_rope(h, cos, sin, 2, 1, 64, 33, w, w), 2)

  dy = torch.randn(2, 33, 4, 64, generator=g, device="cuda").to(BF16)
  results = []
  for run in (layer, lambda x: checkpoint(layer, x, use_reentrant=reentrant)):
    y = run(x)
    y.backward(dy)
    results.append([y.detach(), x.grad, table.grad, w.grad])
    x.grad = table.grad = w.grad = None
  for a, b in zip(*results):
    assert torch.equal(a, b)


def test_embedding_of_other_ids(cuda_lib):
  """int32 ids and ids that are not contiguous."""
  g = torch.Generator(device="cuda").manual_seed(5)
  table = torch.randn(50, 64, generator=g, device="cuda").to(BF16).requires_grad_()
  ids = torch.randint(0, 50, (6, 8), generator=g, device="cuda")
  dy = torch.randn(6, 8, 64, generator=g, device="cuda").to(BF16)
  want = ops.embedding(ids, table, scale=0.5)
  (dt,) = torch.autograd.grad(want, table, dy)
  for other, d in ((ids.int(), dy), (ids.t().contiguous().t(), dy), (torch.stack([ids, ids], -1)[..., 1], dy)):
    y = ops.embedding(other, table, scale=0.5)
    (got,) = torch.autograd.grad(y, table, d)
    # (sums of up to 48 rows in another order and, in torch's operator, other roundings)
    assert torch.equal(y, want) and (got.double() - dt.double()).abs().max() <= 48 * HALF * dt.double().abs().max()
