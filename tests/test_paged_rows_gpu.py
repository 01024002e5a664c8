"""Rows of a paged cache written and read by the kernels, bit for bit those of the definitions."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from torchprime_b200.ops import _lib, functional as ops, paged_kv
from torchprime_b200.ops.paged_kv import E4M3, PagedKV


def _bytes(t):
  return t.contiguous().view(torch.uint8)


def _same(a, b):
  return all(x is None or torch.equal(_bytes(x), _bytes(y)) for x, y in zip(a, b))


def _clone(c):
  return PagedKV(*(None if t is None else t.transpose(1, 2).clone().transpose(1, 2) for t in c))


def _cache(pages, page, h, dk, dv, dtype, g):
  c = PagedKV.allocate(pages, page, h, dk, dv, dtype=dtype, device="cuda")
  for t in c:
    if t is not None:      # what was there before, any bytes
      _fill = torch.randint(0, 120, t.transpose(1, 2).shape + ((2,) if dtype == torch.bfloat16 else ()), generator=g, device="cuda",
                            dtype=torch.uint8)
      t.transpose(1, 2).copy_(_fill.view(t.dtype).squeeze(-1) if dtype == torch.bfloat16 else _fill.view(t.dtype))
  return c


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("t,h,dk,dv,page", [(1, 1, 64, 64, 16), (48, 8, 128, 128, 64), (777, 5, 192, 128, 48), (33, 3, 16, 512, 1),
                                            (2500, 16, 192, 128, 32), (100, 2, 256, 48, 7)])
def test_append_and_read_are_the_definitions(cuda_lib, dtype, t, h, dk, dv, page):
  g = torch.Generator(device="cuda").manual_seed(t)
  pages = -(-t // page) + 2
  c = _cache(pages, page, h, dk, dv, dtype, g)
  want = _clone(c)
  slots = torch.randperm(pages * page, generator=g, device="cuda")[:t]
  slots[t // 3] = -1
  size = torch.exp2(torch.randn(t, h, 1, generator=g, device="cuda") * 6)
  k = (torch.randn(t, h, dk, generator=g, device="cuda") * size).bfloat16()
  v = (torch.randn(t, h, dv, generator=g, device="cuda") * size).bfloat16()
  k[t // 2, 0], v[-1, -1, 0], v[-1, -1, -1] = 0, float("inf"), float("nan")
  n = _lib.launch_count()
  paged_kv.append(c, k, v, slots)
  assert _lib.launch_count() == n + 1
  with ops.backend("torch"):
    paged_kv.append(want, k, v, slots)
    ek, ev = paged_kv.read(want, slots)
  assert _same(c, want)
  gk, gv = paged_kv.read(c, slots)
  for got, w in ((gk, ek), (gv, ev)):
    assert torch.equal(got.isnan(), w.isnan()) and torch.equal(got.nan_to_num(), w.nan_to_num())


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_every_finite_value_is_rounded_as_defined(cuda_lib, dtype):
  """All bf16 magnitudes, beside a value that sets the row's factor and alone."""
  bits = torch.arange(0, 0x8000, dtype=torch.int32, device="cuda")
  x = (bits << 16).view(torch.float32).bfloat16()
  x = torch.where(x.isfinite(), x, 0.0)
  for other in (0.0, 1.0, -3e38):
    k = torch.zeros(x.numel(), 1, 16, dtype=torch.bfloat16, device="cuda")
    k[:, 0, 3], k[:, 0, 11] = x, other
    c, want = (PagedKV.allocate(x.numel() // 16, 16, 1, 16, dtype=dtype, device="cuda") for _ in range(2))
    slots = torch.arange(x.numel(), device="cuda")
    paged_kv.append(c, k, -k, slots)
    with ops.backend("torch"):
      paged_kv.append(want, k, -k, slots)
      ek, _ = paged_kv.read(want, slots)
    assert _same(c, want)
    assert torch.equal(paged_kv.read(c, slots)[0], ek)


def test_every_byte_is_read_as_defined(cuda_lib):
  """All values under all powers of two, down to bf16's subnormal numbers, and the type's NaN."""
  c = PagedKV.allocate(16, 16, 1, 256, dtype=E4M3, device="cuda")
  every = torch.arange(256, dtype=torch.uint8, device="cuda")
  for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
    t.view(torch.uint8).copy_(every.expand(16, 16, 1, 256))
    s.view(torch.uint8).copy_(every.view(16, 16, 1))
  slots = torch.arange(256, device="cuda")
  with ops.backend("torch"):
    want = paged_kv.read(c, slots)
  for got, w in zip(paged_kv.read(c, slots), want):
    assert torch.equal(got.isnan(), w.isnan()) and torch.equal(got.nan_to_num(), w.nan_to_num())
  # and by arithmetic: magnitudes below NaN's, in 64 bits, rounded once
  x = c.k.reshape(256, 256).float().double() * torch.exp2(torch.arange(256, device="cuda").double() - 127)[:, None]
  assert torch.equal(want[0].view(256, 256)[:255].nan_to_num(), x[:255].float().bfloat16().nan_to_num())


def test_strided_inputs_and_pools(cuda_lib):
  torch.manual_seed(0)
  pool = torch.zeros(6, 2, 16, 4, 128, dtype=torch.bfloat16, device="cuda")      # keys and values of a page side by side
  c = PagedKV(pool[:, 0], pool[:, 1])
  qkv = torch.randn(20, 4 * 128 * 3, device="cuda").bfloat16()
  k, v = qkv[:, 512:1024].view(20, 4, 128), qkv[:, 1024:].view(20, 4, 128)
  slots = torch.randperm(96, device="cuda")[:20]
  paged_kv.append(c, k, v, slots)
  gk, gv = paged_kv.read(c, slots)
  assert torch.equal(gk, k) and torch.equal(gv, v)
  assert torch.equal(pool[:, 0].reshape(96, 4, 128)[slots], k)
  paged_kv.append(c, k.transpose(1, 2).contiguous().transpose(1, 2), v[:, :1].expand(20, 4, 128), slots)     # other orders, a shared head
  assert torch.equal(paged_kv.read(c, slots)[0], k) and torch.equal(paged_kv.read(c, slots)[1], v[:, :1].expand(20, 4, 128))


def test_slots_outside_the_pool_are_reported(cuda_lib):
  c = PagedKV.allocate(2, 16, 1, 64, device="cuda")
  x = torch.ones(3, 1, 64, device="cuda", dtype=torch.bfloat16)
  paged_kv.append(c, x, x, torch.tensor([32, 31, 1 << 33], device="cuda"))
  torch.cuda.synchronize()
  with pytest.raises(_lib.KernelError, match="bad argument"):
    _lib.raise_on_device_timeout()
  assert c.k.float().sum() == 64
  k, v = paged_kv.read(c, torch.tensor([-2, 31, -1], device="cuda"))
  torch.cuda.synchronize()
  with pytest.raises(_lib.KernelError, match="bad argument"):
    _lib.raise_on_device_timeout()
  assert not k[0].any() and bool((v[1] == 1).all()) and not v[2].any()


def test_other_types_take_the_definitions(cuda_lib):
  c = PagedKV.allocate(2, 16, 1, 24, dtype=torch.float32, device="cuda")
  x = torch.randn(2, 1, 24, device="cuda")
  paged_kv.append(c, x, x, torch.tensor([3, 30], device="cuda"))
  assert torch.equal(paged_kv.read(c, torch.tensor([30, 3], device="cuda"), dtype=torch.float32)[0], x.flip(0))


def test_no_tokens(cuda_lib):
  c = PagedKV.allocate(2, 16, 1, 64, device="cuda")
  x, s = torch.empty(0, 1, 64, device="cuda", dtype=torch.bfloat16), torch.empty(0, dtype=torch.int64, device="cuda")
  paged_kv.append(c, x, x, s)
  assert paged_kv.read(c, s)[0].shape == (0, 1, 64)


def test_captured_step_on_a_side_stream(cuda_lib):
  """Slots and rows change between replays of one graph."""
  c = PagedKV.allocate(4, 16, 2, 128, dtype=E4M3, device="cuda")
  x, s = torch.zeros(2, 2, 128, device="cuda", dtype=torch.bfloat16), torch.tensor([0, 1], device="cuda")
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    paged_kv.append(c, x, x, s)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    paged_kv.append(c, x, x, s)
    out = paged_kv.read(c, s)
  for i in range(3):
    x.fill_(float(i + 1))
    s.copy_(torch.tensor([5 + i, 40 - i]))
    graph.replay()
    assert bool((out[0] == i + 1).all()) and bool((out[1] == i + 1).all())
  assert bool((paged_kv.read(c, torch.tensor([5, 6, 7], device="cuda"))[0][:, 0, 0] == torch.tensor([1.0, 2, 3], device="cuda")).all())


def test_debug_mode_is_asked_at_every_call(cuda_lib, monkeypatch):
  c = PagedKV.allocate(2, 16, 1, 64, 64, device="cuda")
  k, slots = torch.ones(2, 1, 64, device="cuda").bfloat16(), torch.tensor([3, 3], device="cuda")
  paged_kv.append(c, k, k, slots)
  monkeypatch.setenv("TPB_DEBUG_BOUNDS", "1")
  with pytest.raises(IndexError, match="twice"):
    paged_kv.append(c, k, k, slots)
  with pytest.raises(IndexError, match="slots"):
    paged_kv.read(c, slots + 40)
  with pytest.raises(IndexError, match="lengths"):
    paged_kv.decode_attention(torch.ones(1, 1, 64, device="cuda").bfloat16(), c, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                              torch.tensor([17], dtype=torch.int32, device="cuda"))
  monkeypatch.delenv("TPB_DEBUG_BOUNDS")
  paged_kv.append(c, k, k, slots)
