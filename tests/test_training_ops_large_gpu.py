"""Sizes from which the norms of heads and dropout give each thread more to do."""

import pytest
import torch

from torchprime_b200.ops import functional as ops
from torchprime_b200.ops import reference as ref
from test_training_ops_gpu import BF16, _check_qk, _randn, _tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,d,rot", [(40, 3, 64, 64), (12, 1, 96, 32), (11, 2, 256, 256), (5, 1, 128, 128), (70, 2, 16, 16), (3, 1, 400, 400)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("behind", [False, True])
def test_qk_norm_rope_on_both_sides_of_the_border(cuda_lib, hq, hkv, d, rot, interleaved, behind):
  """64 steps for each of eight warps to an SM, 512 / d heads of a token (a power of two) to a step; the last block of a token's is not a whole one."""
  group = 1
  while group * 16 < d:
    group *= 2
  steps = -(-(hq + hkv) * group // 32)
  border = -(-64 * 8 * torch.cuda.get_device_properties(0).multi_processor_count // steps)
  g = torch.Generator(device="cuda").manual_seed(hq + d)
  s = border if behind else border - 1
  cos, sin = _tables(s, rot // 2)
  x = _randn(g, 1, s, (hq + 2 * hkv) * d)
  wq, wk = (1 + _randn(g, d, std=0.3) for _ in range(2))
  _check_qk(x, cos, sin, hq, hkv, d, wq, wk, interleaved=interleaved, g=g)


@pytest.mark.parametrize("n", [2 ** 24 - 8, 2 ** 24, 2 ** 24 + 8 * 1001 + 3])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_on_both_sides_of_the_border(cuda_lib, n, residual):
  """To the bit, forward and backward."""
  g = torch.Generator(device="cuda").manual_seed(n)
  x, r = _randn(g, n).requires_grad_(), _randn(g, n).requires_grad_() if residual else None
  seed, t = torch.tensor([-9, 77], device="cuda"), 26214
  keep = ref.dropout_keep(x.shape, t, seed, 5)
  y = ops.dropout(x, 0.4, seed, site=5, residual=r)
  assert y.dtype == BF16 and torch.equal(y, ref.dropout(x.detach(), keep, t, None if r is None else r.detach()))
  dy = _randn(g, n)
  dx, *dr = torch.autograd.grad(y, (x, r) if residual else (x,), dy)
  assert torch.equal(dx, ref.dropout(dy, keep, t)) and all(torch.equal(d, dy) for d in dr)
