"""Operators in torch operations, as what follows or rewrites them gets them in place of the kernels: ids without a row, weights that collect
their gradient."""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from torchprime_b200.ops import functional as ops


class _Mode(TorchDispatchMode):
  def __torch_dispatch__(self, func, types, args=(), kwargs=None):
    return func(*args, **(kwargs or {}))


@pytest.fixture
def taken(monkeypatch):
  """Tables that the kernels would take (they are on the CPU: nothing launches under a mode)."""
  monkeypatch.setattr(ops, "use_kernels", lambda *t: True)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize("scale", [None, 3.0])
def test_ids_without_a_row(taken, dtype, scale):
  table = torch.randn(5, 8).requires_grad_()
  ids = torch.tensor([[0, -1, 4], [5, 2, 2 ** 31 - 1]], dtype=dtype)
  with _Mode():
    y = ops.embedding(ids, table, scale=scale)
  s = 1.0 if scale is None else scale
  rows = table.detach() * s
  assert torch.equal(y, torch.stack([rows[0], rows[0] * 0, rows[4], rows[0] * 0, rows[2], rows[0] * 0]).view(2, 3, 8))
  dy = torch.randn(2, 3, 8)
  dy[0, 1] = float("nan")               # (of an id without a row: nobody's)
  (g,) = torch.autograd.grad(y, table, dy)
  want = torch.zeros(5, 8)
  want[0], want[4], want[2] = dy[0, 0] * s, dy[0, 2] * s, dy[1, 1] * s
  assert torch.equal(g, want)


def test_a_table_without_rows(taken):
  with _Mode():
    assert torch.equal(ops.embedding(torch.tensor([0, 3]), torch.empty(0, 8)), torch.zeros(2, 8))


def test_the_gradient_goes_where_it_is_collected(taken):
  """The first one overwritten, the next added; none in .grad; what is recorded itself or several at once is returned."""
  table, ids = torch.randn(5, 8).requires_grad_(), torch.tensor([1, 1, 7])
  dy = torch.randn(3, 8)
  want = torch.zeros(5, 8)
  want[1] = dy[0] + dy[1]
  table.main_grad, table.grad_overwrite = torch.full((5, 8), 7.0), True
  for times in (1, 2):
    with _Mode():
      ops.embedding(ids, table).backward(dy)
    assert table.grad is None and not table.grad_overwrite and torch.equal(table.main_grad, times * want)
  with _Mode():
    y = ops.embedding(ids, table)
  (many,) = torch.autograd.grad(y, table, torch.stack([dy, -dy]), is_grads_batched=True, retain_graph=True)
  (again,) = torch.autograd.grad(y, table, dy.requires_grad_(), create_graph=True)
  assert torch.equal(many, torch.stack([want, -want])) and torch.equal(again, want) and again.requires_grad
  assert torch.equal(table.main_grad, 2 * want)
  with torch.no_grad(), _Mode():
    assert not ops.embedding(ids, table).requires_grad


@pytest.mark.parametrize("shared", [False, True])
def test_heads_weights_too(taken, shared):
  x, dy = torch.randn(2, 3, 4 * 16).requires_grad_(), [torch.randn(2, 3, n, 16) for n in (2, 1, 1)]
  cos, sin = torch.rand(3, 8), torch.rand(3, 8)
  ws = [(torch.rand(16) + 0.5).requires_grad_() for _ in range(2 - shared)]
  call = lambda: ops.qk_norm_rope(x, cos, sin, 2, 1, 16, 3, ws[0], ws[-1])  # noqa: E731
  with _Mode():
    want = torch.autograd.grad(call(), [x, *ws], dy)
    for w in ws:
      w.main_grad, w.grad_overwrite = torch.full((16,), 7.0), True
    torch.autograd.backward(call(), dy)
  assert torch.equal(x.grad, want[0])
  for w, dw in zip(ws, want[1:]):
    assert w.grad is None and torch.allclose(w.main_grad, dw, atol=1e-5)     # (shared: two sums of fp32)


def test_in_a_trace(taken):
  class Rows(torch.nn.Module):
    def __init__(self):
      super().__init__()
      self.table = torch.nn.Parameter(torch.randn(5, 8))

    def forward(self, ids):
      return ops.embedding(ids, self.table, scale=2.0)

  for collected in (False, True):
    m = Rows()
    if collected:
      m.table.main_grad, m.table.grad_overwrite = torch.zeros(5, 8), True
    traced = torch.jit.trace(m, (torch.tensor([1, 2]),), check_trace=False)
    y, dy = traced(torch.tensor([4, -3])), torch.randn(2, 8)
    assert torch.equal(y, torch.stack([m.table.detach()[4] * 2, torch.zeros(8)]))
    y.backward(dy)
    want = torch.zeros(5, 8).index_put((torch.tensor([4]),), dy[:1] * 2)
    assert torch.equal(m.table.main_grad if collected else m.table.grad, want) and (m.table.grad is None) == collected


def test_forward_derivatives(taken):
  table, tangent = torch.randn(5, 8).requires_grad_(), torch.randn(5, 8)
  table.main_grad = torch.zeros(5, 8)
  with torch.autograd.forward_ad.dual_level():
    dual = torch.autograd.forward_ad.make_dual(table, tangent)
    y = ops.embedding(torch.tensor([3, 9]), dual)
    assert torch.equal(torch.autograd.forward_ad.unpack_dual(y).tangent, torch.stack([tangent[3], torch.zeros(8)]))
    y = ops.embedding(torch.tensor([3, 9]), table)
    assert torch.autograd.forward_ad.unpack_dual(y).tangent is None
  jac = torch.func.jacrev(lambda t: ops.embedding(torch.tensor([3]), t))(table.detach())
  assert torch.equal(jac[0, :, 3], torch.eye(8))
