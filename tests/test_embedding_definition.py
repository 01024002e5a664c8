"""The embedding in torch operations, as what follows or rewrites operators gets it in place of the kernels: ids without a row."""

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


def test_in_a_trace(taken):
  class Rows(torch.nn.Module):
    def __init__(self):
      super().__init__()
      self.table = torch.nn.Parameter(torch.randn(5, 8))

    def forward(self, ids):
      return ops.embedding(ids, self.table, scale=2.0)

  m = Rows()
  traced = torch.jit.trace(m, (torch.tensor([1, 2]),), check_trace=False)
  y, dy = traced(torch.tensor([4, -3])), torch.randn(2, 8)
  assert torch.equal(y, torch.stack([m.table.detach()[4] * 2, torch.zeros(8)]))
  y.backward(dy)
  assert torch.equal(m.table.grad, torch.zeros(5, 8).index_put((torch.tensor([4]),), dy[:1] * 2))


def test_forward_derivatives(taken):
  table, tangent = torch.randn(5, 8).requires_grad_(), torch.randn(5, 8)
  with torch.autograd.forward_ad.dual_level():
    dual = torch.autograd.forward_ad.make_dual(table, tangent)
    y = ops.embedding(torch.tensor([3, 9]), dual)
    assert torch.equal(torch.autograd.forward_ad.unpack_dual(y).tangent, torch.stack([tangent[3], torch.zeros(8)]))
  jac = torch.func.jacrev(lambda t: ops.embedding(torch.tensor([3]), t))(table.detach())
  assert torch.equal(jac[0, :, 3], torch.eye(8))
