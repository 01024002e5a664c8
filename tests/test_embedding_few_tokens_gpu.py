"""The embedding's gradient of few tokens: runs of every length around the borders between warps, CTAs and the form for many tokens."""

import pytest
import torch

from torchprime_b200.ops import kernels as k

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HALF = 2.0 ** -8              # a rounding to bf16
LENGTHS = [1, 2, 3, 8, 9, 10, 30, 31, 32, 33, 63, 64, 65, 127, 128, 129, 160, 255, 256, 257, 300]


def _check(got, ids, dout, scale, row0, before):
  """Against 64 bits: a rounding to an addition, of terms no larger than the sum of sizes, and one of the result in bf16."""
  v, d = got.shape
  scale = float(torch.tensor(scale))
  ok = (ids >= row0) & (ids < row0 + v)
  at, rows = ids[ok] - row0, dout[ok].double() * scale
  want, size = (torch.zeros(v, d, device="cuda", dtype=torch.float64).index_add_(0, at, t) for t in (rows, rows.abs()))
  count = torch.bincount(at, minlength=v)[:, None].double()
  if before is not None:
    want, size = want + before.double(), size + before.double().abs()
  half = HALF if got.dtype == BF16 else 0.0
  assert bool(((got.double() - want).abs() <= half * want.abs() + (count + 2) * 2.0 ** -24 * size).all())
  if before is not None:
    none = count[:, 0] == 0
    assert torch.equal(got[none], before[none])


def _both(ids, dout, rows, dtype, row0=0, scale=1.7, rest=None):
  """Added to a table and written over one, twice each: the same bits."""
  d = dout.shape[1]
  before = torch.randn(rows, d, generator=rest, device="cuda").to(dtype)
  added = k.embedding_bwd_(dout, ids, before.clone(), row0=row0, scale=scale)
  _check(added, ids, dout, scale, row0, before)
  assert torch.equal(k.embedding_bwd_(dout, ids, before.clone(), row0=row0, scale=scale), added)
  written = k.embedding_bwd_(dout, ids, torch.full_like(before, float("nan")), row0=row0, scale=scale, overwrite=True)
  _check(written, ids, dout, scale, row0, None)
  assert torch.equal(k.embedding_bwd_(dout, ids, torch.full_like(before, float("nan")), row0=row0, scale=scale, overwrite=True), written)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("dim", [8, 72, 264, 512, 1032])
@pytest.mark.parametrize("order", ["mixed", "together", "apart"])
def test_runs_of_every_length(cuda_lib, dtype, dim, order):
  """Tokens of one id next to one another, as far apart as they can be, and in any order; some have no row."""
  g = torch.Generator(device="cuda").manual_seed(dim)
  ids = torch.cat([torch.full((n,), 3 * i + 1, device="cuda") for i, n in enumerate(LENGTHS)] + [torch.full((40,), i, device="cuda") for i in (-7, 999)])
  if order == "mixed":
    ids = ids[torch.randperm(ids.numel(), generator=g, device="cuda")]
  elif order == "apart":
    ids = ids.view(-1, 2).t().reshape(-1) if ids.numel() % 2 == 0 else torch.cat([ids[::2], ids[1::2]])
  _both(ids, torch.randn(ids.numel(), dim, generator=g, device="cuda").to(BF16), 3 * len(LENGTHS), dtype, rest=g)


@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 15, 16, 17, 31, 32, 33, 2047, 2048, 2049, 4095, 4096, 4097])
@pytest.mark.parametrize("rows", [1, 40, 5003])
def test_numbers_of_tokens(cuda_lib, tokens, rows):
  """Around every border, of one row, of few and of many; a third of the ids in front of the shard or behind it."""
  g = torch.Generator(device="cuda").manual_seed(tokens)
  ids = torch.randint(100 - rows // 3, 100 + rows + rows // 3 + 1, (tokens,), generator=g, device="cuda")
  ids[-1] = 100 + rows - 1
  _both(ids, torch.randn(tokens, 136, generator=g, device="cuda").to(BF16), rows, torch.float32, row0=100, scale=0.5, rest=g)


@pytest.mark.parametrize("tokens", [1, 700, 4096])
def test_all_of_one_id_or_none(cuda_lib, tokens):
  g = torch.Generator(device="cuda").manual_seed(tokens)
  dout = torch.randn(tokens, 1000, generator=g, device="cuda").to(BF16)
  for i in (0, 6, -1, 7, 2 ** 40, -2 ** 63, 2 ** 63 - 1):
    for dtype in (BF16, torch.float32):
      _both(torch.full((tokens,), i, device="cuda", dtype=torch.int64), dout, 7, dtype, rest=g)


def test_past_32_bits(cuda_lib):
  """A table of more than 2^31 numbers, its last rows."""
  vocab, dim, tokens = 530007, 4096, 1500
  g = torch.Generator(device="cuda").manual_seed(1)
  ids = torch.randint(vocab - 600, vocab, (tokens,), generator=g, device="cuda")
  ids[::5] = vocab - 1
  dout = torch.randn(tokens, dim, generator=g, device="cuda").to(BF16)
  table = torch.full((vocab, dim), 2.0, device="cuda", dtype=BF16)
  for overwrite in (False, True):
    k.embedding_bwd_(dout, ids, table, overwrite=overwrite)
    _check(table[vocab - 600:], ids - (vocab - 600), dout, 1.0, 0, None if overwrite else torch.full((600, dim), 2.0, device="cuda"))
    assert all(bool((table[i: min(i + 65536, vocab - 600)] == (0.0 if overwrite else 2.0)).all()) for i in range(0, vocab - 600, 65536))


def test_two_at_once(cuda_lib):
  """On two streams, each into a table of its own: each has its own order."""
  g = torch.Generator(device="cuda").manual_seed(2)
  work = []
  for _ in range(2):
    ids = torch.randint(0, 50, (4000,), generator=g, device="cuda")
    work.append((torch.randn(4000, 256, generator=g, device="cuda").to(BF16), ids, torch.zeros(50, 256, device="cuda"), torch.cuda.Stream()))
  want = [k.embedding_bwd_(dout, ids, torch.zeros_like(table)) for dout, ids, table, _ in work]
  torch.cuda.synchronize()
  for _ in range(20):
    for dout, ids, table, stream in work:
      with torch.cuda.stream(stream):
        k.embedding_bwd_(dout, ids, table.zero_())
  torch.cuda.synchronize()
  for (_, _, table, _), w in zip(work, want):
    assert torch.equal(table, w)
