"""Norms of query and key heads, the embedding and dropout inside autograd: recomputed layers under partial backward passes, gradients
that are collected in a ``main_grad``, numbers that are not finite."""

import contextlib

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

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


def _randn(g, *shape, std=1.0):
  return (torch.randn(*shape, generator=g, device="cuda") * std).to(BF16)


def _tables(n, half):
  angle = torch.arange(n, device="cuda")[:, None].double() * 10000.0 ** (-torch.arange(half, device="cuda").double() / half)
  return angle.cos().float().contiguous(), angle.sin().float().contiguous()


class _Rerun(torch.autograd.Function):
  """A layer that runs without a graph, and once more with one when its gradients are asked for."""

  @staticmethod
  def forward(ctx, fn, x, *weights):
    ctx.fn = fn
    ctx.save_for_backward(x, *weights)
    return fn(x, *weights)

  @staticmethod
  def backward(ctx, *dy):
    again = [t.detach().requires_grad_(need) for t, need in zip(ctx.saved_tensors, ctx.needs_input_grad[1:])]
    with torch.enable_grad():
      y = ctx.fn(*again)
    pairs = [(a, b) for a, b in zip(y, dy) if a.requires_grad]
    torch.autograd.backward([a for a, _ in pairs], [b for _, b in pairs])
    return (None, *(t.grad for t in again))


@pytest.mark.parametrize("how", ["grad", "inputs", "all"])
def test_a_layer_rerun_in_a_backward_pass_has_its_values_gradient(cuda_lib, how):
  g = torch.Generator(device="cuda").manual_seed(1)
  cos, sin = _tables(9, 32)
  x, w = _randn(g, 2, 9, 4 * 64).requires_grad_(), (1 + _randn(g, 64, std=0.3)).requires_grad_()
  dy = [_randn(g, 2, 9, n, 64) for n in (2, 1, 1)]
  layer = lambda x, w: ops.qk_norm_rope(x, cos, sin, 2, 1, 64, 9, w, w)  # noqa: E731
  want = torch.autograd.grad(layer(x, w), (x, w), dy)
  y = _Rerun.apply(layer, x, w)
  if how == "grad":
    got = torch.autograd.grad(y, (x, w), dy)
  else:
    torch.autograd.backward(y, dy, **(dict(inputs=[x, w]) if how == "inputs" else {}))
    got = (x.grad, w.grad)
  assert torch.equal(got[0][..., 3 * 64:], dy[2].view(2, 9, 64))
  for a, b in zip(got, want):
    assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------- main_grad
def _collect(t, dtype=torch.float32):
  """The same numbers as a parameter that collects its gradient."""
  p = t.detach().clone().requires_grad_()
  p.main_grad, p.grad_overwrite = torch.full(t.shape, 7.0, device="cuda", dtype=dtype), True
  return p


def _captured(step):
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step()
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    step()
  return graph


def test_a_captured_pass_adds_up_the_gradients_of_a_shared_weight(cuda_lib):
  """One weight for queries and keys; a table that is the output projection too; two microbatches in one graph."""
  g = torch.Generator(device="cuda").manual_seed(3)
  cos, sin = _tables(9, 32)
  table, w, x = _randn(g, 64, 64, std=0.1), 1 + _randn(g, 64, std=0.3), _randn(g, 2, 9, 4 * 64)
  ids, dout = torch.randint(0, 64, (40,), generator=g, device="cuda"), _randn(g, 40, 64)
  dq, dk = _randn(g, 2, 9, 2, 64), _randn(g, 2, 9, 1, 64)

  def step(table, w):
    for _ in range(2):
      q, kk, _ = ops.qk_norm_rope(x, cos, sin, 2, 1, 64, 9, w, w)
      torch.autograd.grad((q, kk), w, (dq, dk), allow_unused=True)
      torch.autograd.grad(ops.linear(ops.embedding(ids, table), [table]), table, dout, allow_unused=True)

  mine, want = ([_collect(t) for t in (table, w)] for _ in range(2))
  graph = _captured(lambda: step(*mine))
  for _ in range(2):
    graph.replay()
  step(*want)
  for a, b in zip(mine, want):
    assert torch.equal(a.main_grad, b.main_grad)


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_a_captured_pass_replaces_what_its_last_replay_collected(cuda_lib, dtype):
  """A table's and a norm's gradient, each replay with other incoming gradients."""
  g = torch.Generator(device="cuda").manual_seed(2)
  cos, sin = _tables(9, 32)
  table, w, x = _randn(g, 50, 64), 1 + _randn(g, 64, std=0.3), _randn(g, 2, 9, 4 * 64)
  ids, dout = torch.randint(0, 50, (40,), generator=g, device="cuda"), _randn(g, 40, 64)
  dq, dk = _randn(g, 2, 9, 2, 64), _randn(g, 2, 9, 1, 64)

  def step(table, w):
    assert torch.autograd.grad(ops.embedding(ids, table, scale=3.0), table, dout, allow_unused=True) == (None,)
    q, kk, _ = ops.qk_norm_rope(x, cos, sin, 2, 1, 64, 9, w)
    assert torch.autograd.grad((q, kk), w, (dq, dk), allow_unused=True) == (None,)

  mine = [_collect(t, dtype) for t in (table, w)]
  graph = _captured(lambda: step(*mine))
  for _ in range(2):
    for t in (dout, dq, dk):
      t.copy_(_randn(g, *t.shape))
    graph.replay()
    want = [_collect(t, dtype) for t in (table, w)]
    step(*want)
    for a, b in zip(mine, want):
      assert torch.equal(a.main_grad, b.main_grad)


# ------------------------------------------------------------------------------------------- definitions in place of kernels
class _Mode(TorchDispatchMode):
  def __torch_dispatch__(self, func, types, args=(), kwargs=None):
    return func(*args, **(kwargs or {}))


def test_ids_without_a_row_where_something_follows_the_operators(cuda_lib):
  """Under a dispatch mode, in a trace and as int32: what the kernels give."""
  g = torch.Generator(device="cuda").manual_seed(8)
  table = _randn(g, 50, 64).requires_grad_()
  ids, dout = torch.randint(-20, 70, (6, 40), generator=g, device="cuda"), _randn(g, 6, 40, 64)
  want = ops.embedding(ids, table, scale=0.5)
  (dt,) = torch.autograd.grad(want, table, dout)
  with _Mode():
    ys = [ops.embedding(ids, table, scale=0.5)]
  ys.append(ops.embedding(ids.int(), table, scale=0.5))
  traced = torch.jit.trace(lambda i, t: ops.embedding(i, t, scale=0.5), (ids % 50, table))
  ys.append(traced(ids, table))
  for y in ys:
    (got,) = torch.autograd.grad(y, table, dout)
    # (sums of up to 15 rows in another order and, in torch's operator, other roundings)
    assert torch.equal(y, want) and (got.double() - dt.double()).abs().max() <= 15 * HALF * dt.double().abs().max()


def test_weights_collect_their_gradients_where_something_follows_the_operators(cuda_lib):
  g = torch.Generator(device="cuda").manual_seed(9)
  cos, sin = _tables(9, 32)
  table, w, x = _randn(g, 50, 64), 1 + _randn(g, 64, std=0.3), _randn(g, 2, 9, 4 * 64).requires_grad_()
  ids, dout = torch.randint(0, 50, (40,), generator=g, device="cuda"), _randn(g, 40, 64)
  dy = [_randn(g, 2, 9, n, 64) for n in (2, 1, 1)]
  for dtype in (torch.float32, BF16):
    mine, want = ([_collect(t, dtype) for t in (table, w)] for _ in range(2))
    for ps, mode in ((mine, _Mode()), (want, contextlib.nullcontext())):
      with mode:
        for _ in range(2):
          ops.embedding(ids, ps[0], scale=3.0).backward(dout)
          torch.autograd.backward(ops.qk_norm_rope(x, cos, sin, 2, 1, 64, 9, q_weight=ps[1]), dy)
    for a, b in zip(mine, want):
      # (torch's operators round each row of the table's gradient, up to eight to an id, and the weights' sums)
      assert a.grad is None and (a.main_grad - b.main_grad).abs().max() <= 12 * HALF * b.main_grad.abs().max()


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_weights_that_collect_their_gradients_from_after_the_forward_pass_on(cuda_lib, dtype):
  g = torch.Generator(device="cuda").manual_seed(4)
  cos, sin = _tables(9, 32)
  x, dy = _randn(g, 2, 9, 4 * 64).requires_grad_(), [_randn(g, 2, 9, n, 64) for n in (2, 1, 1)]
  table, wq, wk = _randn(g, 50, 64), 1 + _randn(g, 64, std=0.3), 1 + _randn(g, 64, std=0.3)
  ids, dout = torch.randint(0, 50, (40,), generator=g, device="cuda"), _randn(g, 40, 64)
  results = []
  for late in (False, True):
    ps = [_collect(t, dtype) if not late else t.detach().clone().requires_grad_() for t in (table, wq, wk)]
    y, heads = ops.embedding(ids, ps[0], scale=3.0), ops.qk_norm_rope(x, cos, sin, 2, 1, 64, 9, *ps[1:])
    if late:
      for p in ps:
        p.main_grad, p.grad_overwrite = torch.full(p.shape, 7.0, device="cuda", dtype=dtype), True
    torch.autograd.backward([y, *heads], [dout, *dy])
    assert all(p.grad is None and not p.grad_overwrite for p in ps)
    results.append([x.grad, *(p.main_grad for p in ps)])
    x.grad = None
  for a, b in zip(*results):
    assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------- not finite
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_qk_norm_rope_gradient_of_numbers_that_are_not_finite(cuda_lib, bad, interleaved):
  """They reach what the formula says and nothing else: the head of theirs, and their columns (or all, of a head that is not
  finite itself) of the weights' sums."""
  g = torch.Generator(device="cuda").manual_seed(5)
  b, s, hq, hkv, d = 2, 33, 6, 2, 64
  cos, sin = _tables(s, d // 2)
  for where in ("dq", "dk", "dv", "q", "k"):
    x = _randn(g, b, s, (hq + 2 * hkv) * d)
    dy = [_randn(g, b, s, n, d) for n in (hq, hkv, hkv)]
    if where[0] == "d":
      dy[("dq", "dk", "dv").index(where)][1, 7, 1, 5] = bad
    else:
      x[1, 7, (0 if where == "q" else hq) * d + 5] = bad
    x.requires_grad_()
    wq, wk = ((1 + _randn(g, d, std=0.3)).requires_grad_() for _ in range(2))
    got = torch.autograd.grad(ops.qk_norm_rope(x, cos, sin, hq, hkv, d, s, wq, wk, interleaved=interleaved), (x, wq, wk), dy)
    up = [t.detach().double() for t in (*dy, x, cos, sin, wq, wk)]
    want = ref.qk_norm_rope_grad(*up[:6], hq, hkv, d, s, *up[6:], 1e-6, None, interleaved)
    for a, w in zip(got, want):
      assert torch.equal(a.isfinite(), w.isfinite()), where
      # against the largest: a rounding of the result, and fp32 sums of up to 400 terms
      ok = w.isfinite()
      assert not ok.any() or (a[ok].double() - w[ok]).abs().max() <= (HALF + 400 * 2.0 ** -23) * w[ok].abs().max()


@pytest.mark.parametrize("tokens", [40, 3000, 9000])
def test_embedding_gradient_of_numbers_that_are_not_finite(cuda_lib, tokens):
  g = torch.Generator(device="cuda").manual_seed(6)
  table, ids = _randn(g, 300, 72).requires_grad_(), torch.randint(0, 300, (tokens,), generator=g, device="cuda")
  ids[:3], ids[3:20] = 7, 9
  dout = _randn(g, tokens, 72)
  dout[0, 3], dout[1, 4], dout[2, 5], dout[3, 5], dout[4, 5] = float("nan"), float("inf"), float("-inf"), float("inf"), float("-inf")
  (got,) = torch.autograd.grad(ops.embedding(ids, table, scale=0.5), table, dout)
  want = torch.zeros(300, 72, device="cuda", dtype=torch.float64).index_add_(0, ids, dout.double() * 0.5)
  for test in (torch.isnan, torch.isposinf, torch.isneginf):
    assert torch.equal(test(got), test(want))
  ok = want.isfinite()
  assert (got[ok].double() - want[ok]).abs().max() <= (HALF + tokens * 2.0 ** -23) * want[ok].abs().max()
  added = torch.ones(300, 72, device="cuda")
  k.embedding_bwd_(dout, ids, added, scale=0.5)
  for test in (torch.isnan, torch.isposinf, torch.isneginf):
    assert torch.equal(test(added), test(want))


def test_dropout_gradient_of_numbers_that_are_not_finite(cuda_lib):
  g = torch.Generator(device="cuda").manual_seed(7)
  x, seed = _randn(g, 5, 1001).requires_grad_(), torch.tensor([3, 9], device="cuda")
  dy = _randn(g, 5, 1001)
  dy[0], dy[1], dy[2] = float("nan"), float("inf"), float("-inf")
  (dx,) = torch.autograd.grad(ops.dropout(x, 0.25, seed, site=4), x, dy)
  keep = ref.dropout_keep(dy.shape, 16384, seed, 4)
  assert bool(keep[:3].any()) and not bool(keep[:3].all()) and not bool(dx[~keep].any())
  assert torch.equal(dx.nan_to_num(1.0, 2.0, 3.0), ref.dropout(dy, keep, 16384).nan_to_num(1.0, 2.0, 3.0))
