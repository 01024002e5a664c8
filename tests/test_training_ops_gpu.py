"""Norms of query and key heads with the rotation, the scaled embedding with its gradient, and dropout on the kernels, against
64-bit definitions."""

import pytest
import torch

from torchprime_b200.ops import functional as ops
from torchprime_b200.ops import kernels as k
from torchprime_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HALF = 2.0 ** -8              # a rounding to bf16


@pytest.fixture(autouse=True, params=["native", "python"])
def way(request, monkeypatch):
  """The operators as native torch functions, and their Python definitions over the same kernels."""
  if request.param == "python":
    monkeypatch.setattr(ops, "_native", lambda: None)
  return request.param


def test_plain_calls_are_native(cuda_lib, way):
  g = torch.Generator(device="cuda").manual_seed(0)
  cos, sin = _tables(9, 32)
  x, table, seed = _randn(g, 2, 9, 4 * 64), _randn(g, 50, 64), torch.tensor([1, 2], device="cuda")
  w, ids = _randn(g, 64), torch.randint(0, 50, (2, 9), generator=g, device="cuda")
  for grad in (False, True):
    for t in (x, table, w):
      t.requires_grad_(grad)
    ws = [None, w]
    outs = [ops.embedding(ids, table), ops.embedding(ids, table, scale=2.0), ops.dropout(x, 0.1, seed), ops.dropout(x, 0.1, seed, residual=x)]
    outs += [ops.qk_norm_rope(x, cos, sin, 2, 1, 64, 9, a, b)[0] for a in ws for b in ws]
    for y in outs:
      assert y.requires_grad == grad and (not grad or ("CppFunction" in type(y.grad_fn).__name__) == (way == "native"))


def _randn(g, *shape, std=1.0):
  return (torch.randn(*shape, generator=g, device="cuda") * std).to(BF16)


def _tables(n, half):
  angle = torch.arange(n, device="cuda")[:, None].double() * 10000.0 ** (-torch.arange(half, device="cuda").double() / half)
  return angle.cos().float().contiguous(), angle.sin().float().contiguous()


def _qk_exact(x, cos, sin, hq, hkv, d, s, wq, wk, eps, pos, interleaved, grads=None):
  """(results or gradients, the size of the terms that each is a sum of) in 64 bits."""
  up = lambda t: None if t is None else t.detach().double()  # noqa: E731
  args = (up(cos), up(sin), hq, hkv, d, s, up(wq), up(wk), eps, pos, interleaved)
  if grads is None:
    want = ref.qk_norm_rope(up(x), *args)[:2]
    # both terms of a turned column are at most the head's largest
    return want, [t.abs().amax(-1, keepdim=True).expand_as(t) * 2 for t in want]
  want = ref.qk_norm_rope_grad(*(up(t) for t in grads), up(x), *args)
  b, n = x.shape[0], hq + hkv
  heads = up(x).view(b, x.shape[1], -1, d)[:, :, :n]
  r = (heads.square().mean(-1, keepdim=True) + eps).rsqrt()
  dy = torch.cat([up(grads[0]), up(grads[1])], 2)
  w = torch.cat([torch.ones(m, d, device="cuda", dtype=torch.float64) if t is None else up(t).expand(m, d) for m, t in ((hq, wq), (hkv, wk))])
  g = dy.abs().amax(-1, keepdim=True) * 2
  size = r * (g * w.abs()) + heads.abs() * r ** 3 * (g * w.abs() * heads.abs()).mean(-1, keepdim=True)
  dw = (g * (heads * r).abs())
  return want, [size, dw[:, :, :hq].sum((0, 1, 2)), dw[:, :, hq:].sum((0, 1, 2))]


# fp32 around a head: sums of 16 terms a lane and five over lanes, a reciprocal root of 2^-22, its third power and a few products
AROUND = 2.0 ** -18


def _check_qk(x, cos, sin, hq, hkv, d, wq, wk, eps=1e-6, pos=None, interleaved=False, g=None):
  b, s, _ = x.shape
  leaf = x.detach().requires_grad_(g is not None)
  ws = [None if w is None else w.detach().clone().requires_grad_(g is not None) for w in (wq, wk)]
  out = ops.qk_norm_rope(leaf, cos, sin, hq, hkv, d, s, *ws, eps=eps, pos=pos, interleaved=interleaved)
  want, size = _qk_exact(x, cos, sin, hq, hkv, d, s, wq, wk, eps, pos, interleaved)
  for a, w, z in zip(out, want, size):
    assert a.dtype == BF16 and a.is_contiguous() and bool(((a.double() - w).abs() <= HALF * w.abs() + AROUND * z).all())
  assert out[2].data_ptr() == x[..., (hq + hkv) * d:].data_ptr()
  if g is None:
    return out
  grads = [_randn(g, *t.shape) for t in out]
  got = torch.autograd.grad(out, [leaf] + [w for w in ws if w is not None], grads)
  want, size = _qk_exact(x, cos, sin, hq, hkv, d, s, wq, wk, eps, pos, interleaved, grads)
  n = (hq + hkv) * d
  dqk, w = got[0][..., :n].double(), want[0][..., :n]
  assert bool(((dqk - w).abs() <= HALF * w.abs() + AROUND * size[0].reshape(b, s, n)).all())
  assert torch.equal(got[0][..., n:], grads[2].flatten(2))
  at = 1
  for i, wt in enumerate((wq, wk)):
    if wt is not None:       # (a sum over tokens and heads beside what is around each term)
      assert bool(((got[at].double() - want[1 + i]).abs() <= HALF * want[1 + i].abs() + 2.0 ** -16 * size[1 + i]).all())
      at += 1
  return out


@pytest.mark.parametrize("hq,hkv,d,rot", [(32, 8, 128, 128), (40, 8, 128, 128), (7, 1, 128, 64), (16, 4, 64, 64), (3, 3, 96, 64), (4, 2, 256, 256),
                                          (2, 1, 512, 32), (9, 5, 80, 80), (5, 1, 16, 16), (33, 2, 32, 16), (1, 1, 400, 400)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("weights", ["both", "none", "keys"])
def test_qk_norm_rope(cuda_lib, hq, hkv, d, rot, interleaved, weights):
  g = torch.Generator(device="cuda").manual_seed(hq * d)
  for b, s in ((1, 1), (2, 37), (3, 128)):
    x = _randn(g, b, s, (hq + 2 * hkv) * d) * torch.exp2(torch.randn(b, s, 1, generator=g, device="cuda")).to(BF16)
    cos, sin = _tables(300, rot // 2)
    wq, wk = (1 + _randn(g, d, std=0.3) if weights in ("both", one) else None for one in ("queries", "keys"))
    pos = torch.randint(0, 300, (b, s), generator=g, device="cuda").to(torch.int32) if b > 1 else None
    _check_qk(x, cos, sin, hq, hkv, d, wq, wk, pos=pos, interleaved=interleaved, g=g)


def test_qk_norm_rope_of_many_tokens(cuda_lib):
  """More than the grid takes at once; the weights' gradients are sums over 5003 x 40 heads."""
  g = torch.Generator(device="cuda").manual_seed(5)
  cos, sin = _tables(5003, 64)
  x = _randn(g, 1, 5003, 48 * 128)
  _check_qk(x, cos, sin, 32, 8, 128, 1 + _randn(g, 128, std=0.3), 1 + _randn(g, 128, std=0.3), g=g)


def test_qk_norm_rope_of_heads_of_zeros_and_large_ones(cuda_lib):
  """A head of zeros gives zeros and eps' gradient; NaN and infinity stay in their head."""
  g = torch.Generator(device="cuda").manual_seed(6)
  cos, sin = _tables(8, 64)
  x = _randn(g, 1, 8, 6 * 128)
  x[0, 1, :128] = 0
  x[0, 2] *= 2.0 ** 40
  x[0, 3] *= 2.0 ** -40
  _check_qk(x, cos, sin, 4, 1, 128, None, None, eps=1e-5, g=g)
  clean = ops.qk_norm_rope(x, cos, sin, 4, 1, 128, 8)
  x[0, 4, 128] = float("nan")
  x[0, 5, 256] = float("inf")
  q, kk, _ = ops.qk_norm_rope(x, cos, sin, 4, 1, 128, 8)
  bad = torch.zeros(1, 8, 4, dtype=torch.bool, device="cuda")
  bad[0, 4, 1] = bad[0, 5, 2] = True
  assert torch.equal(q.isnan().any(-1), bad) and torch.equal(q[~bad], clean[0][~bad]) and torch.equal(kk, clean[1])


@pytest.mark.parametrize("form", ["pitch", "one token of longer rows", "batches apart", "unaligned", "columns apart", "expanded"])
def test_qk_norm_rope_takes_any_strides(cuda_lib, form):
  g = torch.Generator(device="cuda").manual_seed(7)
  c = 4 * 64
  cos, sin = _tables(9, 32)
  x = {"pitch": lambda: _randn(g, 2, 9, c + 64)[..., 32: 32 + c], "one token of longer rows": lambda: _randn(g, 5, 7, c)[:, 3:4],
       "batches apart": lambda: _randn(g, 2, 12, c)[:, :9], "unaligned": lambda: _randn(g, 18 * c + 1)[1:].view(2, 9, c),
       "columns apart": lambda: _randn(g, 2, 9, 2 * c)[..., ::2], "expanded": lambda: _randn(g, 1, 1, c).expand(2, 9, c)}[form]()
  _check_qk(x, cos, sin, 2, 1, 64, 1 + _randn(g, 64, std=0.3), None, g=g)


def test_qk_norm_rope_positions(cuda_lib):
  """int64 ones, and ones outside the tables: the nearest row, and a report."""
  from torchprime_b200.ops import _lib
  g = torch.Generator(device="cuda").manual_seed(8)
  cos, sin = _tables(9, 32)
  x = _randn(g, 1, 4, 3 * 64)
  call = lambda p, t=torch.int32: ops.qk_norm_rope(x, cos, sin, 1, 1, 64, 4, pos=torch.tensor([p], dtype=t, device="cuda"))[0]  # noqa: E731
  good = call([0, 8, 3, 8])
  assert torch.equal(call([0, 8, 3, 8], torch.int64), good)
  torch.cuda.synchronize()
  _lib.raise_on_device_timeout()
  for p, t in (([0, 9, 3, 2 ** 31 - 1], torch.int32), ([-1, 8, 3, 8], torch.int32), ([-2 ** 40, 2 ** 40, 3, 2 ** 32 + 8], torch.int64)):
    got = call(p, t)
    torch.cuda.synchronize()
    with pytest.raises(_lib.KernelError, match="bad argument"):
      _lib.raise_on_device_timeout()
    assert torch.equal(got, good)


def test_qk_norm_rope_other_forms_take_the_definition(cuda_lib):
  """Types, sizes and recordings that the kernels do not take."""
  g = torch.Generator(device="cuda").manual_seed(9)
  cos, sin = _tables(9, 32)
  x = torch.randn(2, 9, 4 * 64, generator=g, device="cuda")
  for t in (torch.float32, torch.float16):
    q, _, _ = ops.qk_norm_rope(x.to(t), cos, sin, 2, 1, 64, 9)
    assert q.dtype == t and torch.equal(q, ref.qk_norm_rope(x.to(t), cos, sin, 2, 1, 64, 9)[0])
  odd = _randn(g, 2, 9, 4 * 24)
  c, s = _tables(9, 6)
  assert torch.equal(ops.qk_norm_rope(odd, c, s, 2, 1, 24, 9)[0], ref.qk_norm_rope(odd, c, s, 2, 1, 24, 9)[0])
  c = cos.clone().requires_grad_()
  q, _, _ = ops.qk_norm_rope(x.to(BF16), c, sin, 2, 1, 64, 9)
  assert torch.autograd.grad(q.float().sum(), c)[0].abs().sum() > 0


def test_qk_norm_rope_gradients_recorded_or_several_at_once(cuda_lib):
  g = torch.Generator(device="cuda").manual_seed(10)
  cos, sin = _tables(9, 32)
  x, w = _randn(g, 2, 9, 4 * 64).requires_grad_(), (1 + _randn(g, 64, std=0.3)).requires_grad_()
  out = ops.qk_norm_rope(x, cos, sin, 2, 1, 64, 9, w, w)
  dy = [_randn(g, *t.shape).requires_grad_() for t in out]
  dx, dw = torch.autograd.grad(out, (x, w), dy, create_graph=True)
  plain = torch.autograd.grad(out, (x, w), [t.detach() for t in dy], retain_graph=True)
  for a, b in zip((dx, dw), plain):       # (a rounding each; the weight's two gradients are rounded before they are added)
    assert (a - b).abs().max() <= 2 ** -6 * b.abs().max()
  ddy, ddx = torch.autograd.grad(dx.float().square().sum(), (dy[0], x))
  assert ddy.abs().sum() > 0 and ddx.abs().sum() > 0
  many = torch.autograd.grad(out, x, [torch.stack([t.detach(), 2 * t.detach()]) for t in dy], is_grads_batched=True, retain_graph=True)[0]
  assert (many[0] - plain[0]).abs().max() <= 2 ** -6 * plain[0].abs().max() and torch.equal(many[1], 2 * many[0])
  (only,) = torch.autograd.grad(out[1], x, dy[1].detach())      # one of the results used: the others' gradients are zeros
  assert not only[..., : 2 * 64].any() and not only[..., 3 * 64:].any() and torch.equal(only[..., 128: 192], plain[0][..., 128: 192])


def test_qk_norm_rope_over_a_frozen_projection(cuda_lib):
  """Only the weights learn: the values have no gradient, and what uses them does not ask for one."""
  g = torch.Generator(device="cuda").manual_seed(26)
  cos, sin = _tables(9, 32)
  x, w = _randn(g, 2, 9, 4 * 64), (1 + _randn(g, 64, std=0.3)).requires_grad_()
  q, k_, v = ops.qk_norm_rope(x, cos, sin, 2, 1, 64, 9, q_weight=w)
  assert q.requires_grad and not v.requires_grad
  dq = _randn(g, *q.shape)
  (dw,) = torch.autograd.grad(q, w, dq)
  want, size = _qk_exact(x, cos, sin, 2, 1, 64, 9, w, None, 1e-6, None, False, [dq, torch.zeros_like(k_), torch.zeros_like(v)])
  assert bool(((dw.double() - want[1]).abs() <= HALF * want[1].abs() + 2.0 ** -16 * size[1]).all())


def test_qk_norm_rope_of_small_eps(cuda_lib):
  """The third power of the factor leaves fp32, the gradient does not."""
  g = torch.Generator(device="cuda").manual_seed(27)
  cos, sin = _tables(8, 64)
  x = _randn(g, 1, 8, 6 * 128)
  x[0, 1, :128] = 0
  x[0, 2] *= 2.0 ** -48
  _check_qk(x, cos, sin, 4, 1, 128, None, 1 + _randn(g, 128, std=0.3), eps=2.0 ** -100, g=g)


def test_weights_collect_their_gradients(cuda_lib):
  """Norm weights and tables with a main_grad: overwritten first, then added to."""
  g = torch.Generator(device="cuda").manual_seed(11)
  cos, sin = _tables(9, 32)
  x = _randn(g, 2, 9, 4 * 64).requires_grad_()
  dy = [_randn(g, 2, 9, n, 64) for n in (2, 1, 1)]
  ids, dout = torch.randint(0, 50, (40,), generator=g, device="cuda"), _randn(g, 40, 64)
  for dtype in (torch.float32, BF16):
    w, table = (1 + _randn(g, 64, std=0.3)).requires_grad_(), _randn(g, 50, 64).requires_grad_()
    dw = torch.autograd.grad(ops.qk_norm_rope(x, cos, sin, 2, 1, 64, 9, q_weight=w), w, dy)[0]
    dt = torch.autograd.grad(ops.embedding(ids, table, scale=3.0), table, dout)[0]
    for t in (w, table):
      t.main_grad, t.grad_overwrite = torch.full(t.shape, 7.0, device="cuda", dtype=dtype), True
    for times in (1, 2):
      torch.autograd.backward(ops.qk_norm_rope(x, cos, sin, 2, 1, 64, 9, q_weight=w), dy)
      ops.embedding(ids, table, scale=3.0).backward(dout)
      for t, d in ((w, dw), (table, dt)):
        assert t.grad is None and (t.main_grad - times * d.float()).abs().max() <= 3 * HALF * times * d.float().abs().max()


# ------------------------------------------------------------------------------------------- embedding
def _check_table_gradient(got, ids, dout, scale, row0=0, before=None):
  """Sums of each id's rows in fp32, in an order of their own: a rounding to an addition, of terms no larger than the sum of sizes."""
  v, d = got.shape
  ids, dout = ids.view(-1), dout.view(-1, d).double() * scale
  ok = (ids >= row0) & (ids < row0 + v)
  at, rows = ids[ok] - row0, dout[ok]
  want, size = (torch.zeros(v, d, device="cuda", dtype=torch.float64).index_add_(0, at, t) for t in (rows, rows.abs()))
  count = torch.bincount(at, minlength=v)[:, None].double()
  if before is not None:
    want, size = want + before.double(), size + before.double().abs()
  half = HALF if got.dtype == BF16 else 0.0
  assert bool(((got.double() - want).abs() <= half * want.abs() + (count + 2) * 2.0 ** -24 * size).all())


@pytest.mark.parametrize("tokens,vocab,dim", [(1, 7, 8), (31, 300, 64), (32, 300, 64), (33, 1, 264), (100, 129, 1000), (1000, 32000, 136),
                                              (1025, 1000, 2048), (4099, 5, 520), (5000, 202048, 72), (40000, 700, 96), (140001, 3, 24)])
@pytest.mark.parametrize("hot", [0.0, 0.7])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_embedding_gradient_by_sorted_tokens(cuda_lib, tokens, vocab, dim, hot, dtype):
  g = torch.Generator(device="cuda").manual_seed(tokens + vocab)
  ids = torch.randint(0, vocab, (tokens,), generator=g, device="cuda")
  ids = torch.where(torch.rand(tokens, generator=g, device="cuda") < hot, vocab // 2, ids)
  dout = _randn(g, tokens, dim)
  got = torch.full((vocab, dim), float("nan"), dtype=dtype, device="cuda")
  k.embedding_bwd_(dout, ids, got, scale=1.7, overwrite=True)
  _check_table_gradient(got, ids, dout, float(torch.tensor(1.7)))
  again = torch.empty_like(got)
  assert torch.equal(k.embedding_bwd_(dout, ids, again, scale=1.7, overwrite=True), got)
  before = _randn(g, vocab, dim).to(dtype)
  added = k.embedding_bwd_(dout, ids, before.clone())
  _check_table_gradient(added, ids, dout, 1.0, before=before)
  untouched = torch.ones(vocab, dtype=torch.bool, device="cuda").index_fill_(0, ids, False)
  assert torch.equal(added[untouched], before[untouched])


def test_embedding_gradient_of_a_shard(cuda_lib):
  """Ids in front of the shard and behind it, negative ones too, have no row."""
  g = torch.Generator(device="cuda").manual_seed(3)
  ids = torch.randint(-50, 2000, (3000,), generator=g, device="cuda")
  ids[5], ids[6], ids[7] = 2 ** 40, -2 ** 62, 2 ** 62
  dout = _randn(g, 3000, 128)
  for row0, rows in ((0, 1000), (700, 300), (1999, 1), (5000, 10), (2 ** 40 - 3, 8)):
    got = torch.empty(rows, 128, device="cuda")
    k.embedding_bwd_(dout, ids, got, row0=row0, overwrite=True)
    _check_table_gradient(got, ids, dout, 1.0, row0=row0)


@pytest.mark.parametrize("shape,vocab,dim", [((1,), 9, 8), ((3, 17), 1000, 1024), ((2, 500), 128256, 1032), ((5, 1), 300, 4096), ((0,), 9, 64), ((2, 0), 9, 64)])
@pytest.mark.parametrize("scale", [None, 1.0, 45.25, 1.0 / 3])
def test_scaled_embedding(cuda_lib, shape, vocab, dim, scale):
  g = torch.Generator(device="cuda").manual_seed(vocab)
  table = _randn(g, vocab, dim).requires_grad_()
  ids = torch.randint(0, vocab, shape, generator=g, device="cuda")
  y = ops.embedding(ids, table, scale=scale)
  assert torch.equal(y, (table.detach()[ids].float() * (1.0 if scale is None else scale)).to(BF16))
  with torch.no_grad():
    assert torch.equal(ops.embedding(ids, table, scale=scale), y)
  dout = _randn(g, *shape, dim)
  (got,) = torch.autograd.grad(y, table, dout)
  assert got.dtype == BF16 and got.shape == table.shape
  _check_table_gradient(got, ids, dout, 1.0 if scale is None else float(torch.tensor(scale)))


def test_embedding_gradients_recorded_or_several_at_once(cuda_lib):
  g = torch.Generator(device="cuda").manual_seed(4)
  table, ids = _randn(g, 30, 64).requires_grad_(), torch.randint(0, 30, (3, 20), generator=g, device="cuda")
  y = ops.embedding(ids, table, scale=2.0)
  dout = _randn(g, 3, 20, 64).requires_grad_()
  (got,) = torch.autograd.grad(y, table, dout, create_graph=True)
  (back,) = torch.autograd.grad(got.float().sum(), dout)
  assert torch.equal(back, torch.full_like(back, 2.0))
  (plain,) = torch.autograd.grad(y, table, dout.detach(), retain_graph=True)
  (many,) = torch.autograd.grad(y, table, torch.stack([dout.detach(), -dout.detach()]), is_grads_batched=True)
  for a in (got, many[0], -many[1]):
    assert (a - plain).abs().max() <= 2 * HALF * plain.abs().max()


# ------------------------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9, 1), (333, 2048), (17, 1001), (3, 5, 4099), (2048, 2100)])
@pytest.mark.parametrize("p", [2.0 ** -16, 0.1, 0.5, 0.999, 1.0])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout(cuda_lib, shape, p, residual):
  """To the bit: a product and a sum in fp32, rounded once."""
  g = torch.Generator(device="cuda").manual_seed(len(shape))
  x, r = _randn(g, *shape).requires_grad_(), _randn(g, *shape).requires_grad_() if residual else None
  seed, site = torch.tensor([2 ** 62 + 12345, 2 ** 40 + 77], device="cuda"), 2 ** 32 - 5
  y = ops.dropout(x, p, seed, site=site, residual=r)
  keep, t = ref.dropout_keep(shape, round(p * 65536), seed, site), round(p * 65536)
  assert torch.equal(y, ref.dropout(x, keep, t, r)) and torch.equal(keep.cpu(), ref.dropout_keep(shape, t, seed.cpu(), site))
  with torch.no_grad():
    assert torch.equal(ops.dropout(x, p, seed, site=site, residual=r), y)
  dy = _randn(g, *shape)
  got = torch.autograd.grad(y, [x] + ([r] if residual else []), dy)
  assert torch.equal(got[0], ref.dropout(dy, keep, t)) and (not residual or torch.equal(got[1], dy))


def test_dropout_of_what_is_not_ordinary(cuda_lib):
  """Strides, alignment, small and infinite numbers, other types."""
  g = torch.Generator(device="cuda").manual_seed(1)
  seed = torch.tensor([1, 2], device="cuda")
  big = _randn(g, 50, 130)
  for x in (big[:, ::2], big.t(), big.flatten()[1:].view(-1), big[:1].expand(9, 130), big * 2.0 ** -133, big / 0, big.float(), big.half()):
    y = ops.dropout(x, 0.25, seed, residual=x)
    assert y.dtype == x.dtype and torch.equal(y.nan_to_num(3.0), ref.dropout(x, ref.dropout_keep(x.shape, 16384, seed, 0), 16384, x).nan_to_num(3.0))
  assert torch.equal(ops.dropout(big.float(), 0.25, seed) != 0, ops.dropout(big, 0.25, seed) != 0)      # the mask does not hang on the type


def test_dropout_gradients_recorded_or_several_at_once(cuda_lib):
  g = torch.Generator(device="cuda").manual_seed(2)
  seed = torch.tensor([1, 2], device="cuda")
  x = _randn(g, 20, 64).requires_grad_()
  y = ops.dropout(x, 0.3, seed)
  dy = _randn(g, 20, 64).requires_grad_()
  (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
  (back,) = torch.autograd.grad(dx, dy, torch.ones_like(dx), retain_graph=True)
  assert torch.equal(back, ops.dropout(torch.ones_like(x), 0.3, seed))
  (many,) = torch.autograd.grad(y, x, torch.stack([dy.detach(), 2 * dy.detach()]), is_grads_batched=True)
  assert torch.equal(many[0], dx) and torch.equal(many[1], 2 * dx)


def test_dropout_notices_a_seed_counted_up(cuda_lib):
  seed = torch.tensor([1, 2], device="cuda")
  x = torch.randn(20, 64, device="cuda").to(BF16).requires_grad_()
  y = ops.dropout(x, 0.3, seed)
  seed[1] += 1
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    y.sum().backward()


# ------------------------------------------------------------------------------------------- all of them
def _calls(g):
  """Each operator as a function of its floating inputs, and those inputs."""
  cos, sin = _tables(9, 32)
  seed, ids = torch.tensor([5, 6], device="cuda"), torch.randint(0, 50, (2, 9), generator=g, device="cuda")
  return {"qk": (lambda x, a, b: ops.qk_norm_rope(x, cos, sin, 2, 1, 64, 9, a, b, interleaved=True), [_randn(g, 2, 9, 256), 1 + _randn(g, 64, std=0.3), 1 + _randn(g, 64, std=0.3)]),
          "embedding": (lambda t: ops.embedding(ids, t, scale=3.0), [_randn(g, 50, 64)]),
          "dropout": (lambda x, r: ops.dropout(x, 0.3, seed, residual=r), [_randn(g, 2, 9, 64), _randn(g, 2, 9, 64)])}


NAMES = ["qk", "embedding", "dropout"]
listed = lambda t: [t] if torch.is_tensor(t) else list(t)  # noqa: E731


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("give_back", ["elsewhere", "unaligned", "wider", "columns first"])
def test_saved_tensor_hooks(cuda_lib, name, give_back):
  """Hooks may give saved tensors back in another layout, alignment or type."""
  fn, inputs = _calls(torch.Generator(device="cuda").manual_seed(20))[name]
  inputs = [t.requires_grad_() for t in inputs]

  def back(t):
    if give_back == "elsewhere":
      return t.clone()
    if give_back == "unaligned" and t.element_size() < 8:
      return torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)
    if give_back == "columns first" and t.dim() > 1:
      return t.transpose(0, 1).contiguous().transpose(0, 1)
    return t.float() if give_back == "wider" and t.dtype == BF16 else t

  out = listed(fn(*inputs))
  dy = [torch.randn_like(t) for t in out]
  want = torch.autograd.grad(out, inputs, dy)
  with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
    got = torch.autograd.grad(listed(fn(*inputs)), inputs, dy)
  for a, b in zip(got, want):      # (torch's operators where the kernels cannot go on: a rounding more or less)
    assert a.shape == b.shape and (a.float() - b.float()).abs().max() <= 4 * HALF * b.float().abs().max()


@pytest.mark.parametrize("name", NAMES)
def test_traces_follow_their_input(cuda_lib, name):
  g = torch.Generator(device="cuda").manual_seed(21)
  fn, (first, *rest) = _calls(g)[name]
  second = _randn(g, *first.shape)
  with torch.no_grad():
    traced = torch.jit.trace(lambda x: fn(x, *rest), (first,), check_trace=False)
    for x in (second, first):
      with ops.backend("torch"):
        want = listed(fn(x, *rest))
      for a, b in zip(listed(traced(x)), want):
        assert (a.float() - b.float()).abs().max() <= 2 * HALF * b.float().abs().max()


@pytest.mark.parametrize("name", NAMES)
def test_tangents_and_transforms(cuda_lib, name):
  """Forward-mode derivatives, torch.func.grad and vmap give what the definitions give."""
  import torch.autograd.forward_ad as fwd
  g = torch.Generator(device="cuda").manual_seed(22)
  fn, (first, *rest) = _calls(g)[name]
  tangent = _randn(g, *first.shape)

  def every():
    with fwd.dual_level():
      duals = [fwd.unpack_dual(t).tangent for t in listed(fn(fwd.make_dual(first, tangent), *rest))]
    grad = torch.func.grad(lambda x: sum(t.float().square().sum() for t in listed(fn(x, *rest))))(first)
    many = torch.func.vmap(lambda x: fn(x, *rest))(torch.stack([first, tangent]))
    return [*duals, grad, *listed(many)]

  got = every()
  with ops.backend("torch"):
    want = every()
  for a, b in zip(got, want):
    assert a is not None and torch.equal(a, b)


@pytest.mark.parametrize("name", NAMES)
def test_calls_of_other_streams_and_two_at_once(cuda_lib, name):
  """Two streams' calls do not meet; results and gradients are those of one after the other."""
  g = torch.Generator(device="cuda").manual_seed(23)
  fn, inputs = _calls(g)[name]
  sets = [[t.clone().requires_grad_() for t in inputs], [(2 * t).requires_grad_() for t in inputs]]

  def both(streams):
    out = []
    for s, ins in zip(streams, sets):
      with torch.cuda.stream(s):
        for _ in range(20):
          y = listed(fn(*ins))
          grads = torch.autograd.grad(y, ins, [torch.ones_like(t) for t in y])
        out += [*(t.detach() for t in y), *grads]
    torch.cuda.synchronize()
    return out

  now = torch.cuda.current_stream()
  torch.cuda.synchronize()
  for a, b in zip(both([torch.cuda.Stream(), torch.cuda.Stream()]), both([now, now])):
    assert torch.equal(a, b)


def test_empty_calls(cuda_lib):
  cos, sin = _tables(9, 32)
  w = torch.ones(64, device="cuda", dtype=BF16, requires_grad=True)
  for shape in ((0, 9, 256), (2, 0, 256)):
    x = torch.empty(shape, device="cuda", dtype=BF16, requires_grad=True)
    out = ops.qk_norm_rope(x, cos, sin, 2, 1, 64, 9, w, w)
    dx, dw = torch.autograd.grad(out, (x, w), [torch.ones_like(t) for t in out])
    assert [t.shape[2] for t in out] == [2, 1, 1] and dx.shape == shape and not dw.any()
    y = ops.dropout(x, 0.5, torch.tensor([1, 2], device="cuda"))
    assert y.shape == shape and torch.autograd.grad(y, x, torch.ones_like(y))[0].shape == shape


def test_numbers_of_numpy(cuda_lib):
  import numpy as np
  g = torch.Generator(device="cuda").manual_seed(24)
  cos, sin = _tables(9, 32)
  x, seed = _randn(g, 2, 9, 256), torch.tensor([1, 2], device="cuda")
  i = np.int64
  for a, b in zip(ops.qk_norm_rope(x, cos, sin, i(2), i(1), i(64), i(9), eps=np.float32(1e-5)), ops.qk_norm_rope(x, cos, sin, 2, 1, 64, 9, eps=float(np.float32(1e-5)))):
    assert torch.equal(a, b)
  assert torch.equal(ops.dropout(x, np.float64(0.3), seed, site=i(4)), ops.dropout(x, 0.3, seed, site=4))
  assert torch.equal(ops.embedding(torch.arange(2, device="cuda"), x[0], scale=np.float64(0.5)), x[0, :2] * 0.5)


def test_llama4_attention_with_the_fused_norms(cuda_lib):
  """The model's option: the same up to the roundings of the separate passes (three more of heads' values, which attention hands on), in
  results and gradients, with positions of packed rows."""
  from torchprime_b200.config import compose
  from torchprime_b200.models.llama4 import Llama4TextAttention
  g = torch.Generator(device="cuda").manual_seed(25)
  size = ["model=llama-4-text-only-dummy", "model.hidden_size=512", "model.num_attention_heads=4", "model.num_key_value_heads=2", "model.head_dim=128",
          "model.no_rope_layers=[1,0]"]
  cos, sin = _tables(300, 64)
  x, dy = _randn(g, 2, 150, 512).requires_grad_(), _randn(g, 2, 150, 512)
  pos = (torch.arange(300, device="cuda") % 100).to(torch.int32)
  got = []
  state = None
  for fused in (False, True):
    cfg = compose("default", size + ([f"+model.fused_qk_norm={str(fused).lower()}"] if fused else [])).model
    m = Llama4TextAttention(cfg, 0).cuda().to(BF16)
    assert m.fused_qk_norm == fused and not Llama4TextAttention(cfg, 1).fused_qk_norm
    if state is None:
      for p in m.parameters():
        torch.nn.init.normal_(p, std=0.05)
      state = m.state_dict()
    m.load_state_dict(state)
    y = m(x, cos, sin, position_ids=pos)
    got.append([y, *torch.autograd.grad(y, [x, *m.parameters()], dy)])
  for a, b in zip(*got):
    assert (a.float() - b.float()).abs().max() <= 8 * HALF * a.float().abs().max()


# ------------------------------------------------------------------------------------------- together
def _block(p, ids, cos, sin, seed, drop, o):
  """Embedding, dropout, norm, projection, normalised heads, attention, projection, dropout with the residual."""
  b, s = ids.shape
  hq, hkv, d = 4, 2, 128
  h = o.dropout(o.embedding(ids, p["table"], scale=16.0), drop, seed, site=0)
  qkv = o.linear(o.rms_norm(h, p["norm"], 1e-5), [p["qkv"]])
  q, kk, v = o.qk_norm_rope(qkv, cos, sin, hq, hkv, d, s, p["qn"], p["kn"], eps=1e-6)
  a = o.attention(q, kk, v, causal=True)
  return o.dropout(o.linear(a.reshape(b, s, hq * d), p["o"]), drop, seed, site=1, residual=h)


def _params(g):
  return {"table": _randn(g, 500, 256, std=0.06), "norm": 1 + _randn(g, 256, std=0.1), "qkv": _randn(g, 8 * 128, 256, std=0.06),
          "qn": 1 + _randn(g, 128, std=0.1), "kn": 1 + _randn(g, 128, std=0.1), "o": _randn(g, 256, 512, std=0.04)}


def test_a_layer_of_them(cuda_lib):
  """Forward and gradients against 64 bits; relative to the largest, since roundings of activations spread over a layer: about ten
  of them, each half a step of a value no larger than the largest."""
  g = torch.Generator(device="cuda").manual_seed(12)
  params = {n: t.requires_grad_() for n, t in _params(g).items()}
  ids, (cos, sin) = torch.randint(0, 500, (2, 150), generator=g, device="cuda"), _tables(150, 64)
  ids[:, 140:] = 0
  seed = torch.tensor([5, 6], device="cuda")
  y = _block(params, ids, cos, sin, seed, 0.2, ops)
  dy = _randn(g, *y.shape)
  got = torch.autograd.grad(y, list(params.values()), dy)
  wide = {n: t.detach().double().requires_grad_() for n, t in params.items()}
  with ops.backend("torch"):
    want_y = _exact_block(wide, ids, cos.double(), sin.double(), seed, 0.2)
  want = torch.autograd.grad(want_y, list(wide.values()), dy.double())
  for name, a, w in zip(["y", *params], [y, *got], [want_y, *want]):
    assert (a.double() - w).abs().max() <= 10 * HALF * w.abs().max(), name


def _exact_block(p, ids, cos, sin, seed, drop):
  b, s = ids.shape
  x = p["table"][ids] * 16.0
  t = round(drop * 65536)
  h = ref.dropout(x, ref.dropout_keep(x.shape, t, seed, 0), t)
  n = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5) * p["norm"]
  q, kk, v = ref.qk_norm_rope(n @ p["qkv"].t(), cos, sin, 4, 2, 128, s, p["qn"], p["kn"], 1e-6)
  kk, v = (u.repeat_interleave(2, 2).transpose(1, 2) for u in (kk, v))
  sc = (q.transpose(1, 2) @ kk.transpose(2, 3)) / 128 ** 0.5
  sc = sc.masked_fill(torch.ones(s, s, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
  o = (torch.softmax(sc, -1) @ v).transpose(1, 2).reshape(b, s, 512) @ p["o"].t()
  return ref.dropout(o, ref.dropout_keep(o.shape, t, seed, 1), t, h)


def test_a_layer_captured_and_replayed(cuda_lib):
  """Forward and backward in one graph: a replay with the next step's seed, other ids and other weights gives what an ordinary
  call gives, to the bit."""
  g = torch.Generator(device="cuda").manual_seed(13)
  names = list(_params(g))
  params = {n: t.requires_grad_() for n, t in _params(g).items()}
  ids, (cos, sin) = torch.randint(0, 500, (2, 150), generator=g, device="cuda"), _tables(150, 64)
  seed, dy = torch.tensor([5, 6], device="cuda"), _randn(g, 2, 150, 256)

  def step():
    y = _block(params, ids, cos, sin, seed, 0.2, ops)
    return [y.detach(), *torch.autograd.grad(y, list(params.values()), dy)]

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step()
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = step()
  for i in range(2):
    with torch.no_grad():
      seed[1] += 1
      ids.copy_(torch.randint(0, 500, (2, 150), generator=g, device="cuda"))
      for n in names:
        params[n].mul_(1.0 + 0.125 * i)
    graph.replay()
    got = [t.clone() for t in out]
    for name, a, b in zip(["y", *names], got, step()):
      if name == "norm":     # (its gradient over few rows is added up by atomics)
        assert (a - b).abs().max() <= 2 * HALF * b.abs().max()
      else:
        assert torch.equal(a, b), name
