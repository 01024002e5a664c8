"""Which gradient of a weight with a ``main_grad`` replaces what is there, and which adds to it."""

from types import SimpleNamespace

import pytest

from torchprime_b200.ops import functional as ops
from torchprime_b200.ops import moe


@pytest.fixture
def capture(monkeypatch):
  """The number of the capture that runs: a test sets it."""
  now = SimpleNamespace(id=0)
  monkeypatch.setattr(ops, "_capture", lambda: now.id)
  return now


def test_the_first_gradient_of_a_step_replaces(capture):
  w = SimpleNamespace(is_cuda=True, grad_overwrite=True)
  assert ops.overwrites_grad(w)
  ops.grad_delivered(w)
  assert not ops.overwrites_grad(w) and not ops.overwrites_grad(SimpleNamespace(is_cuda=True))


def test_the_first_gradient_of_a_capture_replaces(capture):
  """Whatever a warm-up pass has left in the flag; the next one in the same capture adds, and in another one replaces again."""
  w = SimpleNamespace(is_cuda=True, grad_overwrite=False)
  for capture.id in (5, 6):
    assert ops.overwrites_grad(w) and ops.overwrites_grad(w)
    ops.grad_delivered(w)
    assert not ops.overwrites_grad(w) and not ops.overwrites_grad(w)
  capture.id = 0
  assert not ops.overwrites_grad(w)
  w.grad_overwrite = True
  assert ops.overwrites_grad(w)


def test_expert_weights_too(capture):
  w = SimpleNamespace(is_cuda=True, main_grad=None)
  w.main_grad, added = "sink", []
  for capture.id in (5, 5, 6):
    assert moe._deliver_wgrad(w, lambda out, accumulate: added.append(accumulate)) is None
  assert added == [False, True, False]


def test_a_cpu_weight_has_no_capture(monkeypatch):
  monkeypatch.setattr(ops, "_capture", lambda: pytest.fail("no capture on a CPU"))
  w = SimpleNamespace(is_cuda=False, grad_overwrite=True)
  assert ops.overwrites_grad(w)
  ops.grad_delivered(w)
  assert not ops.overwrites_grad(w)


def test_a_captured_table_replaces(capture, monkeypatch):
  """A table whose warm-up pass has cleared the flag: overwritten by the first gradient of a capture, added to by the next."""
  table, how = SimpleNamespace(is_cuda=True, main_grad="sink", grad_overwrite=False), []
  monkeypatch.setattr(ops, "_embedding_collect", lambda ids, mg, dout, scale, overwrite: how.append(overwrite))
  for capture.id in (0, 7, 7, 8):
    assert ops._embedding_backward(None, table, None, 1.0) is None
  assert how == [False, True, False, True]
