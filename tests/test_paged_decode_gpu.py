"""Attention of one new token over a paged cache (csrc/paged_decode.cu) against 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from torchprime_b200.ops import _lib, functional as ops, paged_kv, reference as ref
from torchprime_b200.ops.paged_kv import E4M3, PagedKV

BAD = (1 << 30) + 7          # a page that no pool has


def _cache(g, pages, page, h, dk, dv, dtype, token_major=False, rows=None):
  """A pool whose every row is NaN but the slots ``rows``."""
  c = PagedKV.allocate(pages, page, h, dk, dv, dtype=dtype, device="cuda")
  if token_major:
    c = PagedKV(c.k.contiguous(), c.v.contiguous(), c.k_scale, c.v_scale)
  for t in (c.k, c.v):
    t.copy_(torch.full((), float("nan"), device="cuda").to(t.dtype).expand(t.shape))
  n = rows.numel()
  size = torch.exp2(torch.randint(-3, 4, (n, h, 1), generator=g, device="cuda").float())
  paged_kv.append(c, torch.randn(n, h, dk, generator=g, device="cuda").bfloat16(),
                  (torch.randn(n, h, dv, generator=g, device="cuda") * size).bfloat16(), rows)
  return c


def _problem(lens, heads, kv_heads, dk, dv, page, dtype, seed=0, token_major=False, spare=3, width=None):
  g = torch.Generator(device="cuda").manual_seed(seed)
  need = [-(-n // page) for n in lens]
  pages = sum(need) + spare
  order = torch.randperm(pages, generator=g, device="cuda")
  width = width or max(need + [1]) + 1
  table = torch.full((len(lens), width), BAD, dtype=torch.int32, device="cuda")
  at, rows = 0, []
  for i, n in enumerate(need):
    table[i, :n] = order[at:at + n]
    at += n
    pos = torch.arange(lens[i], device="cuda")
    rows.append(table[i].long()[pos // page] * page + pos % page)
  rows = torch.cat(rows)
  c = _cache(g, pages, page, kv_heads, dk, dv, dtype, token_major, rows)
  q = (torch.randn(len(lens), heads, dk, generator=g, device="cuda") * 1.5).bfloat16()
  return q, c, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def _held(c, slots):
  return tuple(ref.paged_read(t, s, slots).double() for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)))


def _check(got, q, c, table, lengths, scale=None, window=0, softcap=0.0):
  """Within: half a step of bf16 on the result; half a step of bf16 or f16 on every weight; f16 weights below 2^-14 half a step of
  2^-24 of the largest term; 2^-20 on sums, exponentials and scores (fp32, cut by the tensor core after each 16 products)."""
  b, hq, d = q.shape
  page, hkv = c.page, c.k.shape[2]
  scale = scale if scale is not None else d ** -0.5
  assert got.shape == (b, hq, c.v.shape[3]) and got.dtype == q.dtype
  held8 = c.k.dtype == E4M3
  for i, n in enumerate(lengths.tolist()):
    if n <= 0:
      assert not got[i].any()
      continue
    pos = torch.arange(max(0, n - window) if window else 0, n, device=q.device)
    k, v = _held(c, table[i].long()[pos // page] * page + pos % page)
    q1 = q[i].double().view(hkv, hq // hkv, d)
    s = torch.einsum("hgd,shd->hgs", q1, k) * scale
    size = torch.einsum("hgd,shd->hgs", q1.abs(), k.abs()).amax(-1, keepdim=True) * scale
    if softcap:
      s = softcap * torch.tanh(s / softcap)
      size = size + softcap
    p = s.softmax(-1)
    o = torch.einsum("hgs,shd->hgd", p, v)
    a = torch.einsum("hgs,shd->hgd", p, v.abs())
    tol = 2.0 ** -8 * o.abs() + a * ((2.0 ** -11 if held8 else 2.0 ** -8) + 2.0 ** -20 * (2 * size + 2))
    if held8:
      tol = tol + pos.numel() * 2.0 ** -25 * torch.einsum("hgs,sh->hgs", p, v.abs().amax(-1)).amax(-1, keepdim=True)
    off = (got[i].double().view(o.shape) - o).abs()
    assert bool((off <= tol).all()), (i, n, (off / tol).max().item())


DIMS = [(8, 2, 128, 128), (4, 4, 192, 128), (12, 4, 64, 64), (40, 8, 128, 128), (7, 1, 128, 128), (32, 2, 128, 128), (33, 1, 64, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("heads,kv_heads,dk,dv", DIMS)
def test_ragged_batch(cuda_lib, dtype, heads, kv_heads, dk, dv):
  lens = [300, 1, 0, 16, 17, 129, 1000, 33, 0, 127, 128]
  p = _problem(lens, heads, kv_heads, dk, dv, 16, dtype)
  n = _lib.launch_count()
  got = paged_kv.decode_attention(*p)
  assert _lib.launch_count() > n
  _check(got, *p)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("lens", [[1], [2, 3], [5000], [255, 256, 257], [0, 0], [64] * 70, list(range(1, 40))])
def test_pages_and_lengths(cuda_lib, dtype, page, lens):
  p = _problem(lens, 8, 2, 128, 128, page, dtype, seed=page)
  _check(paged_kv.decode_attention(*p), *p)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("window,softcap,scale", [(1, 0, None), (16, 0, None), (100, 0, 0.3), (4096, 30.0, None), (0, 5.0, 0.5), (333, 2.0, None)])
def test_window_softcap_and_scale(cuda_lib, dtype, window, softcap, scale):
  p = _problem([1, 90, 100, 101, 2000, 0, 513], 8, 2, 128, 128, 32, dtype, seed=window)
  got = paged_kv.decode_attention(*p, scale=scale, window=window, softcap=softcap)
  _check(got, *p, scale=scale, window=window, softcap=softcap)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_more_sequences_than_threads(cuda_lib, dtype):
  g = torch.Generator().manual_seed(5)
  lens = (torch.rand(700, generator=g) ** 3 * 300).int().tolist()
  p = _problem(lens, 4, 4, 64, 64, 16, dtype)
  _check(paged_kv.decode_attention(*p), *p)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("lens", [[40000], [20000, 3, 17, 9000], [3000] * 20])
def test_long_sequences_are_joined(cuda_lib, dtype, lens):
  p = _problem(lens, 16, 4, 128, 128, 64, dtype)
  got = paged_kv.decode_attention(*p)
  _check(got, *p)
  assert torch.equal(got, paged_kv.decode_attention(*p))        # the order of every sum is fixed


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_other_layouts(cuda_lib, dtype):
  """Pools with the heads inside the tokens, queries out of a fused projection, a table that is part of a wider one."""
  q, c, table, lens = _problem([70, 200, 5], 8, 2, 128, 128, 16, dtype, token_major=True)
  fused = torch.randn(3, 12 * 128, device="cuda").bfloat16()
  fused[:, :1024] = q.reshape(3, -1)
  wide = torch.full((3, 40), BAD, dtype=torch.int32, device="cuda")
  wide[:, 3:3 + table.shape[1]] = table
  got = paged_kv.decode_attention(fused[:, :1024].view(3, 8, 128), c, wide[:, 3:3 + table.shape[1]], lens)
  _check(got, q, c, table, lens)


def test_keys_and_values_in_one_pool(cuda_lib):
  q, c, table, lens = _problem([70, 200, 5], 8, 2, 128, 128, 16, torch.bfloat16)
  both = torch.stack([c.k, c.v], 1)
  got = paged_kv.decode_attention(q, PagedKV(both[:, 0], both[:, 1]), table, lens)
  _check(got, q, c, table, lens)


def test_values_whose_sizes_differ_by_far(cuda_lib):
  """The weights of an e4m3 cache carry the values' powers of two: neither they nor the sums overflow, and a row that has the
  largest values but no weight does not take the others' bits."""
  q, c, table, lens = _problem([200, 130], 8, 2, 128, 128, 16, E4M3)
  n = int(lens[0])
  slots = table[0].long()[torch.arange(n, device="cuda") // 16] * 16 + torch.arange(n, device="cuda") % 16
  k, v = paged_kv.read(c, slots)
  v = v.float() * torch.exp2(torch.arange(n, device="cuda").float() % 41 - 20)[:, None, None] * 2.0 ** 60
  v[7] *= 2.0 ** 30                       # beside a key that every query looks away from
  k[7] = -40 * q[0].float().view(2, 4, 128).sum(1).sign().bfloat16() * 2.0
  paged_kv.append(c, k, v.bfloat16(), slots)
  _check(paged_kv.decode_attention(q, c, table, lens), q, c, table, lens)


def _check_scores(got, q, c, table, lengths, scale, softcap=0.0):
  """Within: half a step of bf16 on the result; half a step of bf16 or f16 on every weight; 2^-19 of their size on scores, capped or
  not, and 2^-20 on exponentials and sums."""
  for i, n in enumerate(lengths.tolist()):
    pos = torch.arange(n, device=q.device)
    k, v = _held(c, table[i].long()[pos // c.page] * c.page + pos % c.page)
    q1 = q[i].double().view(k.shape[1], -1, q.shape[2])
    s = torch.einsum("hgd,shd->hgs", q1, k) * scale
    size = torch.einsum("hgd,shd->hgs", q1.abs(), k.abs()).amax(-1, keepdim=True) * scale
    p = (softcap * torch.tanh(s / softcap) if softcap else s).softmax(-1)
    o, a = torch.einsum("hgs,shd->hgd", p, v), torch.einsum("hgs,shd->hgd", p, v.abs())
    tol = 2.0 ** -8 * o.abs() + a * ((2.0 ** -11 if c.k.dtype == E4M3 else 2.0 ** -8) + 2.0 ** -19 * (2 * size + 2))
    off = (got[i].double().view(o.shape) - o).abs()
    assert bool((off <= tol).all()), (i, n, (off / tol).max().item())


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("lens", [[30000], [900, 17]])
def test_many_small_weights_count(cuda_lib, dtype, lens):
  """A first token that outweighs each of the others 2^26 times, but holds nothing."""
  q, c, table, lengths = _problem(lens, 4, 1, 64, 64, 64, dtype)
  q.zero_()[:, :, 0] = 1
  first = table[:, 0].long() * 64
  every = torch.cat([table[i].long()[(r := torch.arange(n, device="cuda")) // 64] * 64 + r % 64 for i, n in enumerate(lens)])
  k = torch.zeros(every.numel(), 1, 64, device="cuda").bfloat16()
  v = torch.rand(every.numel(), 1, 64, device="cuda").bfloat16() + 1
  begins = torch.isin(every, first)
  k[begins, 0, 0] = 26
  v[begins] = 0
  paged_kv.append(c, k, v, every)
  scale = 0.6931471805599453
  _check_scores(paged_kv.decode_attention(q, c, table, lengths, scale=scale), q, c, table, lengths, scale)


@pytest.mark.parametrize("lens", [[5, 17], [2], [30], [900, 64]])
@pytest.mark.parametrize("below", [10, 22, 26, 30])
def test_small_weights_of_any_fraction(cuda_lib, lens, below):
  """As above, with an 8-bit cache, few tokens and scores at fractions of an octave: a weight below 2^-29 of the largest, each times its
  power of two of the values, is off by up to 2^-40 of that instead of 2^-11 of itself."""
  q, c, table, lengths = _problem(lens, 4, 1, 64, 64, 64, E4M3)
  q.zero_()[:, :, 0] = 1
  g = torch.Generator(device="cuda").manual_seed(below)
  scale = 0.6931471805599453             # scores in octaves
  for i, n in enumerate(lens):
    pos = torch.arange(n, device="cuda")
    slots = table[i].long()[pos // 64] * 64 + pos % 64
    k = torch.zeros(n, 1, 64, device="cuda")
    k[:, 0, 0] = -below - torch.rand(n, generator=g, device="cuda") * 2
    k[0, 0, 0] = 0
    v = torch.rand(n, 1, 64, generator=g, device="cuda") + 1
    v[0] = 0
    paged_kv.append(c, k.bfloat16(), v.bfloat16(), slots)
  got = paged_kv.decode_attention(q, c, table, lengths, scale=scale)
  for i, n in enumerate(lens):
    pos = torch.arange(n, device="cuda")
    slots = table[i].long()[pos // 64] * 64 + pos % 64
    k, v = _held(c, slots)
    power = c.v_scale[slots // 64, slots % 64].double()[:, 0]
    s = torch.einsum("hd,sd->hs", q[i].double(), k[:, 0]) * scale
    p = s.softmax(-1)
    o, a = p @ v[:, 0], p @ v[:, 0].abs()
    size = s.abs().amax()
    subnormal = 2.0 ** -40 * (p * power).amax(-1, keepdim=True) * (v[:, 0].abs() / power[:, None]).sum(0)
    tol = 2.0 ** -8 * o.abs() + a * (2.0 ** -11 + 2.0 ** -19 * (2 * size + 2)) + subnormal
    off = (got[i].double() - o).abs()
    assert bool((off <= tol).all()), (i, n, (off / tol).max().item())


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("softcap", [1.0, 50.0, 3e4, 1e7])
def test_caps_far_above_the_scores(cuda_lib, dtype, softcap):
  p = _problem([700, 33], 8, 2, 128, 128, 32, dtype, seed=3)
  _check_scores(paged_kv.decode_attention(*p, scale=0.3, softcap=softcap), *p, 0.3, softcap)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("softcap", [1e-42, 1e-37, 1e-25, 1e-6, 1e25, 1e33, 1e37, 3e38])
def test_caps_of_any_size(cuda_lib, dtype, softcap):
  """Far below the scores all tokens weigh the same, far above them they weigh as without a cap."""
  p = _problem([700, 33], 8, 2, 128, 128, 32, dtype, seed=3)
  _check_scores(paged_kv.decode_attention(*p, scale=0.3, softcap=softcap), *p, 0.3, softcap)


def test_a_window_beyond_32_bits_is_none(cuda_lib):
  p = _problem([700, 33], 8, 2, 128, 128, 32, torch.bfloat16)
  assert torch.equal(paged_kv.decode_attention(*p, window=(1 << 32) + 5), paged_kv.decode_attention(*p))


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("size", [0.0, 2.0 ** -60, 2.0 ** 30])
def test_queries_of_any_size(cuda_lib, dtype, size):
  q, c, table, lens = _problem([200, 130], 8, 2, 128, 128, 16, dtype)
  q = (q.float() * size).bfloat16()
  scale = 128 ** -0.5 / max(size, 1.0)
  _check(paged_kv.decode_attention(q, c, table, lens, scale=scale), q, c, table, lens, scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_nan_of_a_visible_row_reaches_its_sequence_alone(cuda_lib, dtype):
  q, c, table, lens = _problem([200, 130], 8, 2, 128, 128, 16, dtype)
  at = table[0, 3].long()
  (c.k.view(torch.uint8) if dtype == E4M3 else c.k)[at, 5, 1] = 0x7f if dtype == E4M3 else float("nan")
  got = paged_kv.decode_attention(q, c, table, lens)
  assert bool(got[0, 4:].isnan().all())
  assert not got[0, :4].isnan().any() and not got[1].isnan().any()


@pytest.mark.parametrize("dims", [(8, 2, 128, 128), (32, 2, 128, 128), (4, 4, 192, 128), (12, 4, 64, 64)])
@pytest.mark.parametrize("lens", [[200, 130, 90, 77], [4000, 130, 900, 61]])
def test_powers_of_two_at_the_ends_of_their_type(cuda_lib, dims, lens):
  """A NaN for a power of two reaches its sequence and head, and no other from rows that cannot be seen; 2^-127 counts as that."""
  heads, kv_heads, dk, dv = dims
  q, c, table, lengths = _problem(lens, heads, kv_heads, dk, dv, 16, E4M3)
  group = heads // kv_heads
  good = paged_kv.decode_attention(q, c, table, lengths)
  k8, v8 = c.k_scale.view(torch.uint8), c.v_scale.view(torch.uint8)
  for i in range(4):
    end = lens[i]                          # behind the last token, on its page
    if end % 16:
      page = table[i, end // 16].long()
      for s in (k8, v8):
        s[page, end % 16:] = 255
  assert torch.equal(paged_kv.decode_attention(q, c, table, lengths), good)
  k8[table[0, 3].long(), 5, 1] = 255
  v8[table[1, 2].long(), 9, 0] = 255
  got = paged_kv.decode_attention(q, c, table, lengths)
  bad = torch.zeros(4, heads, dtype=torch.bool, device="cuda")
  bad[0, group:2 * group] = True
  bad[1, :group] = True
  assert torch.equal(got.isnan().all(-1), bad) and torch.equal(got.isnan().any(-1), bad) and torch.equal(got[~bad], good[~bad])
  # the smallest power of two, under keys that huge queries see, with values of the same, then of 1
  q[2] = (q[2].float() * 2.0 ** 122).bfloat16()
  pos = torch.arange(lens[2], device="cuda")
  at = (table[2].long()[pos // 16], pos % 16)
  k8[at] = 0
  q1 = q[2].double().view(kv_heads, group, dk)
  s = torch.einsum("hgd,shd->hgs", q1, c.k[at].float().double() * 2.0 ** -127) * 2.0 ** 3
  size = torch.einsum("hgd,shd->hgs", q1.abs(), c.k[at].float().double().abs() * 2.0 ** -124).amax()
  p = s.softmax(-1)
  assert float(s.abs().max()) > 1
  for byte in (0, 127):
    v8[at] = byte
    got = paged_kv.decode_attention(q[2:3], c, table[2:3], lengths[2:3], scale=2.0 ** 3)[0]
    v = c.v[at].float().double() * 2.0 ** (byte - 127)
    o, a = torch.einsum("hgs,shd->hgd", p, v).reshape(heads, dv), torch.einsum("hgs,shd->hgd", p, v.abs()).reshape(heads, dv)
    # as in _check; results and terms below 2^-126 are flushed
    tol = 2.0 ** -8 * o.abs() + a * (2.0 ** -11 + 2.0 ** -20 * (2 * size + 2)) + pos.numel() * 2.0 ** -25 * v.abs().max() + 2.0 ** -126
    assert bool(((got.double() - o).abs() <= tol).all())


def test_addresses_past_32_bits(cuda_lib):
  c = PagedKV.allocate(70000, 16, 16, 128, dtype=E4M3, device="cuda")        # 2.3e9 values a pool
  table = torch.tensor([[69999, 0, 69998], [35000, 69997, 1]], dtype=torch.int32, device="cuda")
  lens = torch.tensor([41, 48], dtype=torch.int32, device="cuda")
  g = torch.Generator(device="cuda").manual_seed(3)
  slots = (table.long()[:, :, None] * 16 + torch.arange(16, device="cuda")).reshape(-1)
  paged_kv.append(c, *(torch.randn(96, 16, 128, generator=g, device="cuda").bfloat16() for _ in range(2)), slots)
  q = torch.randn(2, 16, 128, generator=g, device="cuda").bfloat16()
  _check(paged_kv.decode_attention(q, c, table, lens), q, c, table, lens)
  with ops.backend("torch"):
    want = paged_kv.read(c, slots)[0]
  assert torch.equal(paged_kv.read(c, slots)[0], want)


def test_pages_and_lengths_that_do_not_exist_are_reported(cuda_lib):
  q, c, table, lens = _problem([64, 40, 20], 8, 2, 128, 128, 16, torch.bfloat16, width=4)
  good = paged_kv.decode_attention(q, c, table, lens)
  for bad_table, bad_lens in ((BAD, None), (-1, None), (None, 10 ** 9), (None, -3)):
    t, n = table.clone(), lens.clone()
    if bad_table is not None:
      t[1, 1] = bad_table
    else:
      n[1] = bad_lens
      t[1] = table[0]
    got = paged_kv.decode_attention(q, c, t, n)
    torch.cuda.synchronize()
    with pytest.raises(_lib.KernelError, match="bad argument"):
      _lib.raise_on_device_timeout()
    assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])
    if bad_lens is not None:
      assert not got[1].any() if bad_lens < 0 else bool(got[1].isfinite().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("bad", [BAD, -1])
@pytest.mark.parametrize("dims", [(8, 2, 128, 128), (32, 2, 128, 128), (4, 4, 192, 128), (12, 4, 64, 64)])
def test_pages_outside_the_pool_count_as_zeros(cuda_lib, dtype, bad, dims):
  """Whatever keys, values and powers of two the places held that such a page would have come to: every other sequence has the largest
  values there are, and a warp has steps of several sequences."""
  heads, kv_heads, dk, dv = dims
  lens = [290, 130] * 500
  q, c, table, lengths = _problem(lens, heads, kv_heads, dk, dv, 16, dtype)
  pos = torch.arange(290, device="cuda")
  slots = (table[::2].long()[:, pos // 16] * 16 + pos % 16).reshape(-1)
  paged_kv.append(c, torch.zeros(slots.numel(), kv_heads, dk, device="cuda").bfloat16(),
                  torch.full((slots.numel(), kv_heads, dv), 3e38, device="cuda").bfloat16(), slots)
  good = paged_kv.decode_attention(q, c, table, lengths)
  table[1::2, 2] = bad
  table[1::4, 6:8] = bad
  got = paged_kv.decode_attention(q, c, table, lengths)
  torch.cuda.synchronize()
  with pytest.raises(_lib.KernelError, match="bad argument"):
    _lib.raise_on_device_timeout()
  assert torch.equal(got[::2], good[::2])
  few = list(range(1, 1000, 38))
  _check(got[few], q[few], c, table[few], lengths[few])


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("page", [16, 32, 48])
@pytest.mark.parametrize("heads,kv_heads,dk,dv", [(8, 2, 128, 128), (12, 4, 64, 64), (32, 2, 64, 64)])
@pytest.mark.parametrize("window", [1, 17, 40, 100])
@pytest.mark.parametrize("bad", [BAD, -1])
def test_pages_in_front_of_a_window_are_not_looked_at(cuda_lib, dtype, page, heads, kv_heads, dk, dv, window, bad):
  """They may have been given back: nothing is reported, and the result is the same."""
  lens = [1, 16, 63, 64, 65, 112, 129, 200, 333, 700]
  q, c, table, lengths = _problem(lens, heads, kv_heads, dk, dv, page, dtype, seed=window)
  want = paged_kv.decode_attention(q, c, table, lengths, window=window)
  _check(want, q, c, table, lengths, window=window)
  for i, n in enumerate(lens):
    table[i, : max(0, n - window) // page] = bad
  got = paged_kv.decode_attention(q, c, table, lengths, window=window)
  torch.cuda.synchronize()
  _lib.raise_on_device_timeout()
  assert torch.equal(got, want)


def test_streams_and_graphs_with_scratch_of_their_own(cuda_lib):
  """Two captured steps replayed on two streams at once, lengths and pages changing between replays."""
  problems = [_problem(ls, 8, 2, 128, 128, 16, dt, seed=i) for i, (ls, dt) in
              enumerate([([900, 40, 3000], torch.bfloat16), ([1500, 1, 77], E4M3)])]
  graphs, outs = [], []
  for p in problems:
    paged_kv.decode_attention(*p)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
      outs.append(paged_kv.decode_attention(*p))
    graphs.append(gr)
  streams = [torch.cuda.Stream() for _ in graphs]
  for shift in (0, 1, 7):
    for q, c, table, lens in problems:
      lens.sub_(shift).clamp_(min=0)
    torch.cuda.synchronize()
    for _ in range(5):
      for s, gr in zip(streams, graphs):
        with torch.cuda.stream(s):
          gr.replay()
    torch.cuda.synchronize()
    for o, p in zip(outs, problems):
      _check(o, *p)


def test_other_shapes_take_the_definition(cuda_lib):
  """Pages that are no multiple of 16, other head sizes, queries with a gradient."""
  for page, dk, dv in ((7, 128, 128), (16, 96, 96), (16, 24, 16)):
    q, c, table, lens = _problem([30, 1, 0], 4, 2, dk, dv, page, torch.bfloat16)
    _check(paged_kv.decode_attention(q, c, table, lens), q, c, table, lens)
  q, c, table, lens = _problem([30, 1, 0], 4, 2, 128, 128, 16, torch.bfloat16)
  q.requires_grad_()
  paged_kv.decode_attention(q, c, table, lens).float().sum().backward()
  assert bool(q.grad.isfinite().all()) and bool(q.grad[0].any())


def test_empty_batch(cuda_lib):
  q, c, table, lens = _problem([30], 4, 2, 128, 128, 16, torch.bfloat16)
  assert paged_kv.decode_attention(q[:0], c, table[:0], lens[:0]).shape == (0, 4, 128)
  assert not paged_kv.decode_attention(q, c, table[:, :0], torch.zeros_like(lens)).any()


def test_a_decode_step_writes_and_attends(cuda_lib):
  """Append, then attend: step after step equals attention over what was appended."""
  g = torch.Generator(device="cuda").manual_seed(9)
  c = PagedKV.allocate(12, 16, 2, 128, dtype=E4M3, device="cuda")
  table = torch.randperm(12, generator=g, device="cuda").int().view(2, 6)
  for n in range(1, 40):
    k, v = (torch.randn(2, 2, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
    slots = table[:, (n - 1) // 16].long() * 16 + (n - 1) % 16
    paged_kv.append(c, k, v, slots)
    lens = torch.full((2,), n, dtype=torch.int32, device="cuda")
    q = torch.randn(2, 8, 128, generator=g, device="cuda").bfloat16()
    _check(paged_kv.decode_attention(q, c, table, lens), q, c, table, lens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_native_and_python_calls_are_the_same(cuda_lib, monkeypatch, dtype):
  q, c, table, lens = _problem([200, 130, 0], 8, 2, 128, 128, 16, dtype)
  a = paged_kv.decode_attention(q, c, table, lens, window=150, softcap=20.0)
  slots = torch.arange(0, 90, 7, device="cuda")
  rows = paged_kv.read(c, slots)
  monkeypatch.setattr(ops, "_native", lambda: None)
  assert torch.equal(a, paged_kv.decode_attention(q, c, table, lens, window=150, softcap=20.0))
  for x, y in zip(rows, paged_kv.read(c, slots)):
    assert torch.equal(x.view(torch.int16), y.view(torch.int16))
  with pytest.raises(ValueError):
    paged_kv.decode_attention(q, c, table, lens.long())
