"""What operators without an autograd function ask before they launch a kernel by hand."""

import torch

from torchprime_b200.ops import functional


def test_traces_dispatch_modes_and_transforms_are_seen():
  from torch.utils._python_dispatch import TorchDispatchMode
  class Watch(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
      return func(*args, **(kwargs or {}))
  seen = []
  def fn(x):
    seen.append(functional.unobserved())
    return x * 2
  x = torch.ones(3)
  fn(x)
  torch.jit.trace(fn, (x,), check_trace=False)
  with Watch():
    fn(x)
  torch.func.vmap(fn)(x[None])
  torch.func.grad(lambda t: fn(t).sum())(x)
  fn(x)
  assert seen == [True, False, False, False, False, True]


def test_forward_mode_is_seen():
  with torch.autograd.forward_ad.dual_level():
    assert not functional.unobserved()
  assert functional.unobserved()
