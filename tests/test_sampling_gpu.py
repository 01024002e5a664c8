"""The sampling kernel draws the token of the definition (64 bits), whatever the distribution and however many CTAs share a row."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from torchprime_b200.ops import _lib, functional as ops, reference as ref
from torchprime_b200.ops.sampling import sample_tokens


def _logits(g, b, v, kind):
  x = torch.randn(b, v, generator=g, device="cuda") * 2
  if kind == "peaks":
    n = min(v, 20)
    x.scatter_add_(1, torch.randint(0, v, (b, n), generator=g, device="cuda"), torch.rand(b, n, generator=g, device="cuda") * 9)
  elif kind == "flat":
    x *= 1e-3
  elif kind == "equal":
    x.fill_(1.25)
  elif kind == "few values":
    x = torch.randint(-3, 4, (b, v), generator=g, device="cuda").float()
  elif kind == "masked":                      # a grammar that allows a few tokens, in one row none
    x[torch.rand(b, v, generator=g, device="cuda") > 3 / v] = -math.inf
    x[0] = -math.inf
  elif kind == "huge":
    x *= 1e30
  elif kind == "tiny":
    x *= 1e-42
  return x


def _same(x, u, **kw):
  got = sample_tokens(x, u, **kw)
  want = ref.sample_tokens(x, u, **{n: (kw.get(n) if kw.get(n) is not None else d) for n, d in
                                    (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))})
  assert got.dtype == torch.int64 and got.shape == want.shape
  bad = (got != want).nonzero()[:5, 0].tolist()
  assert not bad, [(i, int(got[i]), int(want[i])) for i in bad]


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=50), dict(top_p=0.9), dict(min_p=0.05),
            dict(temperature=1.5, top_p=0.99), dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.02), dict(top_k=1), dict(top_p=0.0),
            dict(top_k=3000), dict(top_k=3000, top_p=0.5), dict(temperature=2.0, top_k=2500, top_p=0.999, min_p=1e-4), dict(min_p=1.0),
            dict(top_k=10 ** 9, top_p=1.0, min_p=-1.0), dict(temperature=math.inf, top_p=0.5, min_p=1.0), dict(temperature=1e-6)]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("kind", ["normal", "peaks", "flat", "equal", "few values", "masked"])
def test_every_setting_on_every_distribution(cuda_lib, kw, kind):
  g = torch.Generator(device="cuda").manual_seed(len(kind))
  for b, v in ((6, 32000), (3, 5003)):
    x, u = _logits(g, b, v, kind), torch.rand(b, generator=g, device="cuda")
    _same(x, u, **kw)
    _same(x.bfloat16(), u, **kw)


@pytest.mark.parametrize("v", [1, 2, 3, 31, 257, 1000, 2047, 2048, 2049, 4097, 65537, 128256, 202048, 262144])
@pytest.mark.parametrize("b", [1, 5, 90])
def test_sizes(cuda_lib, b, v):
  g = torch.Generator(device="cuda").manual_seed(v + b)
  x, u = _logits(g, b, v, "peaks"), torch.rand(b, generator=g, device="cuda")
  for kw in (dict(), dict(top_p=0.95, temperature=0.8), dict(top_k=50, min_p=0.01), dict(top_p=0.98, temperature=3.0), dict(temperature=0)):
    _same(x, u, **kw)


def test_more_rows_than_the_machine_has_room_for(cuda_lib):
  g = torch.Generator(device="cuda").manual_seed(4)
  x, u = _logits(g, 1500, 8000, "peaks"), torch.rand(1500, generator=g, device="cuda")
  _same(x, u, top_p=0.9)
  _same(x, u, temperature=1.3, top_k=20)


def test_settings_for_each_row(cuda_lib):
  g = torch.Generator(device="cuda").manual_seed(6)
  b, v = 64, 50000
  x, u = _logits(g, b, v, "peaks"), torch.rand(b, generator=g, device="cuda")
  i = torch.arange(b, device="cuda")
  _same(x, u, temperature=(i % 5).float() * 0.4, top_k=((i % 7) * 700).int(), top_p=0.5 + (i % 6).float() * 0.1, min_p=(i % 3).float() * 0.03)


@pytest.mark.parametrize("b", [17, 100, 300, 513, 700, 1500])
def test_rows_of_unequal_work(cuda_lib, b):
  """Some rows take all their logits, some a few, some one; their order in the batch is no order of the work."""
  g = torch.Generator(device="cuda").manual_seed(b)
  x, u = _logits(g, b, 9001, "few values"), torch.rand(b, generator=g, device="cuda")
  i = torch.randperm(b, generator=g, device="cuda")
  kw = dict(temperature=torch.where(i % 4 == 0, 0.0, 0.9), top_k=torch.where(i % 3 == 0, 0, i % 9000 + 1).int(),
            top_p=torch.where(i % 5 == 0, 1.0, 0.93))
  _same(x, u, **kw)
  _same(x, u, **kw, min_p=torch.where(i % 2 == 0, 0.0, 0.2))


@pytest.mark.parametrize("kind", ["huge", "tiny", "normal"])
def test_extreme_logits(cuda_lib, kind):
  g = torch.Generator(device="cuda").manual_seed(8)
  x, u = _logits(g, 8, 3001, kind), torch.rand(8, generator=g, device="cuda")
  x[1, 7], x[1, 2000] = math.inf, math.inf
  x[2, ::3] = math.nan
  x[3] = math.nan
  x[4] = -math.inf
  x[5, 1:] = -math.inf
  x[6, :3000] = 0.0
  x[6, ::2] = -0.0
  for kw in SETTINGS:
    _same(x, u, **kw)


def test_temperatures_too_small_for_normal_numbers(cuda_lib):
  """Above 0 all the same: drawn among the largest logits, given for all rows or for each."""
  g = torch.Generator(device="cuda").manual_seed(16)
  x, u = _logits(g, 40, 9000, "few values"), torch.rand(40, generator=g, device="cuda")
  _same(x, u, temperature=1e-42)
  _same(x, u, temperature=torch.full((40,), 1e-42, device="cuda"))
  _same(x, u, temperature=torch.full((40,), 1e-42, device="cuda"), top_k=700, top_p=torch.full((40,), 1e-40, device="cuda"))
  tiny = _logits(g, 40, 9000, "tiny")                # of the same size as the temperature
  for kw in (dict(), dict(top_p=0.9), dict(top_k=50), dict(min_p=0.1), dict(top_k=3000, top_p=0.8, min_p=0.01)):
    _same(tiny, u, temperature=1e-42, **kw)
    _same(tiny, u, temperature=torch.full((40,), 2e-42, device="cuda"), **kw)


def test_first_and_last_numbers(cuda_lib):
  g = torch.Generator(device="cuda").manual_seed(9)
  x = _logits(g, 6, 40000, "peaks")
  u = torch.tensor([0.0, 1 - 2.0 ** -24, 0.0, 1 - 2.0 ** -24, 0.5, 2.0 ** -24], device="cuda")
  for kw in (dict(), dict(top_k=5), dict(top_p=0.7), dict(temperature=2.0, top_p=0.95)):
    _same(x, u, **kw)
  got = sample_tokens(x, torch.tensor([1.0, 7.0, -3.0, math.nan, math.inf, 0.0], device="cuda"), top_k=4)      # outside [0, 1): a kept token all the same
  kept = x.topk(4)[1]
  assert bool((kept == got[:, None]).any(1).all())


def test_strided_rows(cuda_lib):
  g = torch.Generator(device="cuda").manual_seed(10)
  wide = _logits(g, 7, 9005, "peaks")
  u = torch.rand(7, generator=g, device="cuda")
  for x in (wide[:, 1:8002], wide[::2, 3:], wide.t().contiguous().t(), wide.bfloat16()[:, 1:7000]):
    _same(x, u[: x.shape[0]], top_p=0.9)
    _same(x, u[: x.shape[0]], temperature=2.5, top_k=30)


@pytest.mark.parametrize("b,v", [(1, 32768), (1, 262144), (3, 40007), (16, 128256), (40, 8200), (70, 60000)])
def test_rows_without_a_filter_over_and_over(cuda_lib, b, v):
  """The CTAs of a row meet after the largest logits and then not before the sums: all of them work with the same largest logit,
  however far apart they are (rows whose slices weigh nothing but for one, and slices of unequal length)."""
  g = torch.Generator(device="cuda").manual_seed(v)
  x, u = _logits(g, b, v, "peaks"), torch.rand(b, generator=g, device="cuda")
  x[0, v // 2:] = -math.inf
  want = ref.sample_tokens(x, u)
  got = torch.stack([sample_tokens(x, u) for _ in range(200)])
  assert bool((got == want).all())


def test_settings_out_of_wider_tensors(cuda_lib):
  g = torch.Generator(device="cuda").manual_seed(15)
  x, u = _logits(g, 16, 9000, "peaks"), torch.rand(32, generator=g, device="cuda")[::2]
  both = torch.stack([torch.linspace(0, 2, 16, device="cuda"), torch.linspace(0.3, 1, 16, device="cuda")], 1)
  _same(x, u, temperature=both[:, 0], top_p=both[:, 1], min_p=(both * 0.01)[:, 0], top_k=torch.arange(0, 64, 2, dtype=torch.int32, device="cuda")[::2])


def test_same_token_every_time_and_from_python(cuda_lib, monkeypatch):
  g = torch.Generator(device="cuda").manual_seed(11)
  x, u = _logits(g, 40, 30000, "normal"), torch.rand(40, generator=g, device="cuda")
  kw = dict(temperature=torch.full((40,), 1.1, device="cuda"), top_k=5000, top_p=0.97)
  first = sample_tokens(x, u, **kw)
  assert all(torch.equal(first, sample_tokens(x, u, **kw)) for _ in range(3))
  monkeypatch.setattr(ops, "_native", lambda: None)
  n = _lib.launch_count()
  assert torch.equal(first, sample_tokens(x, u, **kw)) and _lib.launch_count() == n + 1


def test_captured_and_replayed(cuda_lib):
  g = torch.Generator(device="cuda").manual_seed(12)
  x, u = _logits(g, 3, 20000, "peaks"), torch.rand(3, generator=g, device="cuda")
  t = torch.ones(3, device="cuda")
  sample_tokens(x, u, t, top_p=0.9)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = sample_tokens(x, u, t, top_p=0.9)
  for _ in range(4):
    x.copy_(_logits(g, 3, 20000, "peaks"))
    u.copy_(torch.rand(3, generator=g, device="cuda"))
    t.copy_(torch.rand(3, generator=g, device="cuda") * 2)
    graph.replay()
    assert torch.equal(out, ref.sample_tokens(x, u, t, top_p=0.9))


def test_frequencies_follow_the_distribution(cuda_lib):
  g = torch.Generator(device="cuda").manual_seed(13)
  n = 40000
  x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 1.5]], device="cuda").expand(n, 5)
  f = torch.bincount(sample_tokens(x, torch.rand(n, generator=g, device="cuda"), 1.0, top_k=4), minlength=5) / n
  want = torch.softmax(torch.tensor([0.0, 1.0, 2.0, -math.inf, 1.5], device="cuda"), 0)
  assert torch.allclose(f, want, atol=5 * (0.25 / n) ** 0.5)


def test_empty_batch_and_wide_rows(cuda_lib):
  assert sample_tokens(torch.zeros(0, 9, device="cuda"), torch.zeros(0, device="cuda")).shape == (0,)
  g = torch.Generator(device="cuda").manual_seed(14)
  x, u = _logits(g, 2, (1 << 18) + 3, "peaks"), torch.rand(2, generator=g, device="cuda")
  _same(x, u, top_p=0.9)                       # (more than the kernel takes: the definition)


@pytest.mark.parametrize("order", ["random", "rising", "falling", "few finite", "equal"])
@pytest.mark.parametrize("k", [1, 50, 128, 129])
def test_long_slices_in_any_order(cuda_lib, order, k):
  """So many rows that a CTA reads its slice in pieces: what the k largest may be is known better and better, or worst at first."""
  g = torch.Generator(device="cuda").manual_seed(k)
  b, v = 160, 40003
  x, u = torch.randn(b, v, generator=g, device="cuda") * 2, torch.rand(b, generator=g, device="cuda")
  if order in ("rising", "falling"):
    x = x.sort(1, descending=order == "falling").values
  elif order == "few finite":
    x[torch.rand(b, v, generator=g, device="cuda") > 100 / v] = -math.inf
  elif order == "equal":
    x = x.round()
  x = torch.nn.functional.pad(x, (0, 5))[:, :v]      # rows that bulk copies can take
  _same(x, u, top_k=k, temperature=0.8)
  _same(x, u, top_k=k, top_p=0.9, min_p=0.01)
  _same(x.bfloat16(), u, top_k=k, top_p=0.9)
