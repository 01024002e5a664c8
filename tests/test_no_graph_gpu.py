"""Operators with nothing recorded."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from torchprime_b200.ops import functional as ops


def test_operators_without_a_graph_equal_those_with_one(cuda_lib):
  """Nothing recorded: the operators skip their autograd functions; results, in-place writes and version
  counters are the same."""
  torch.manual_seed(0)
  x = torch.randn(2, 40, 256, device="cuda", dtype=torch.bfloat16)
  w = torch.randn(256, 256, device="cuda", dtype=torch.bfloat16) / 16
  g = torch.randn(512, 256, device="cuda", dtype=torch.bfloat16) / 16
  n = torch.randn(256, device="cuda", dtype=torch.bfloat16)
  ids = torch.randint(0, 256, (2, 40), device="cuda")
  cos, sin = torch.randn(40, 64, device="cuda"), torch.randn(40, 64, device="cuda")
  def every():
    qkv = torch.randn(2, 40, 6 * 128, device="cuda", dtype=torch.bfloat16, generator=torch.Generator("cuda").manual_seed(1))
    r = ops.rope_inplace(qkv * 1, cos, sin, 5, 128, 40)
    return [ops.linear(x, w), ops.linear(x, w, residual=x), ops.linear_swiglu(x, g[:256], g[256:]), ops.rms_norm(x, n, 1e-5),
            *ops.rms_norm_residual(x, n, 1e-5), r, ops.embedding(ids, w),
            ops.attention_qkv(r, 4, 1, 128)]
  with_graph = every()
  with torch.no_grad():
    without = every()
  for a, b in zip(with_graph, without):
    assert torch.equal(a, b) and not b.requires_grad
  t = torch.randn(1, 40, 256, device="cuda", dtype=torch.bfloat16)
  v = t._version
  with torch.no_grad():
    assert ops.rope_inplace(t, cos, sin, 2, 128, 40) is t and t._version == v + 1
  with torch.inference_mode():
    ops.rope_inplace(torch.randn(1, 40, 256, device="cuda", dtype=torch.bfloat16), cos, sin, 2, 128, 40)


def test_fused_projection_with_a_row_pitch(cuda_lib):
  """A projection that is a slice of wider rows gives the same result with and without a graph."""
  from torchprime_b200.ops import attention_sm100 as A
  qkv = torch.randn(2, 70, 6 * 128 + 64, device="cuda", dtype=torch.bfloat16)[..., :6 * 128]
  with_graph = A.attention_qkv(qkv, 4, 1, 128)
  with torch.no_grad():
    assert torch.equal(A.attention_qkv(qkv, 4, 1, 128), with_graph)
    assert torch.equal(A.attention_qkv(qkv.contiguous(), 4, 1, 128), with_graph)


@pytest.mark.parametrize("op", ["linear", "swiglu", "norm", "embedding", "attention", "segments", "router"])
def test_traces_follow_their_input(cuda_lib, op):
  """An operator traced with nothing recorded computes from the input of each call."""
  from torchprime_b200.ops import moe
  torch.manual_seed(0)
  w = torch.randn(128, 64, device="cuda", dtype=torch.bfloat16) / 8
  ids = torch.arange(300, device="cuda")[None] // 70
  fn, shape = {
    "linear": (lambda x: ops.linear(x, w), (30, 64)),
    "swiglu": (lambda x: ops.linear_swiglu(x, w[:64], w[64:]), (30, 64)),
    "norm": (lambda x: ops.rms_norm(x, w[0], 1e-5), (30, 64)),
    "embedding": (lambda x: ops.embedding((x[:, 0].float().abs() * 10).long().clamp(0, 127), w), (30, 64)),
    "attention": (lambda x: ops.attention_qkv(x, 4, 1, 128), (1, 40, 6 * 128)),
    "segments": (lambda x: ops.attention_qkv(x, 4, 1, 128, q_segment_ids=ids), (1, 300, 6 * 128)),
    "router": (lambda x: moe.router_topk(x.float(), 6)[0], (30, 64)),
  }[op]
  first, second = (torch.randn(*shape, device="cuda", dtype=torch.bfloat16) for _ in range(2))
  with torch.no_grad():
    traced = torch.jit.trace(fn, (first,), check_trace=False)
    assert torch.equal(traced(second), fn(second)) and torch.equal(traced(first), fn(first))


def _cache(dtype=torch.bfloat16):
  """Two sequences of 40 and 17 tokens in pages of 16."""
  from torchprime_b200.ops import paged_kv
  g = torch.Generator(device="cuda").manual_seed(0)
  c = paged_kv.PagedKV.allocate(6, 16, 2, 64, dtype=dtype, device="cuda")
  paged_kv.append(c, *(torch.randn(96, 2, 64, generator=g, device="cuda").bfloat16() for _ in range(2)), torch.arange(96, device="cuda"))
  return c, torch.tensor([[4, 0, 2], [1, 5, 3]], dtype=torch.int32, device="cuda"), torch.tensor([40, 17], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("op", ["sample", "read", "append", "decode"])
def test_traces_of_serving_operators_follow_their_input(cuda_lib, op, dtype):
  """Traced, they are their definitions."""
  from torchprime_b200.ops import paged_kv
  from torchprime_b200.ops.sampling import sample_tokens
  c, table, lens = _cache(dtype)
  u = torch.tensor([0.3, 0.8], device="cuda")
  slots = torch.tensor([7, 90, 33], device="cuda")
  pools = [t for t in c if t is not None]
  def written(x):
    paged_kv.append(c, x, -x, slots)
    return paged_kv.read(c, slots)
  g = torch.Generator(device="cuda").manual_seed(1)
  r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
  fn, first, second = {
    "sample": (lambda x: sample_tokens(x, u, 0.8, top_p=0.9), r(2, 500), r(2, 500)),
    "read": (lambda s: paged_kv.read(c, s), slots, slots - 5),
    "append": (written, r(3, 2, 64), r(3, 2, 64)),
    "decode": (lambda q: paged_kv.decode_attention(q, c, table, lens), r(2, 4, 64), r(2, 4, 64)),
  }[op]
  same = lambda a, b: torch.equal(a, b) if torch.is_tensor(a) else all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
  with torch.no_grad():
    with ops.backend("torch"):
      want = fn(second), fn(first)
    traced = torch.jit.trace(fn, (first,), check_trace=False)
    for x, w in zip((second, first) * 3, want * 3):      # (fused from the third time on)
      for t in pools:                  # (memory that was let go is what an unwritten result shows)
        t.clone()
      if op == "append":
        for t in pools:
          t.view(torch.uint8).zero_()
      assert same(traced(x), w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_tangents_pass_the_cache(cuda_lib, dtype):
  """Of queries and of bf16 pools, as the definitions give them."""
  import torch.autograd.forward_ad as fwd
  from torchprime_b200.ops import paged_kv
  c, table, lens = _cache(dtype)
  g = torch.Generator(device="cuda").manual_seed(2)
  q, tq = (torch.randn(2, 4, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
  slots = torch.tensor([7, 90, 33], device="cuda")
  tk, tv = (torch.randn(6, 2, 16, 64, generator=g, device="cuda").bfloat16().transpose(1, 2) for _ in range(2))
  def call(pools):
    with torch.no_grad(), fwd.dual_level():
      cache = c if not pools else c._replace(k=fwd.make_dual(c.k, tk), v=fwd.make_dual(c.v, tv))
      o = paged_kv.decode_attention(fwd.make_dual(q, tq), cache, table, lens)
      return [fwd.unpack_dual(t).tangent for t in (o, *paged_kv.read(cache, slots))]
  for pools in [False] + [True] * (dtype == torch.bfloat16):
    got = call(pools)
    with ops.backend("torch"):
      want = call(pools)
    assert got[0] is not None and torch.equal(got[0], want[0])
    for a, b in zip(got[1:], want[1:]):
      assert (a is None) == (b is None) == (not pools) and (a is None or torch.equal(a, b))


@pytest.mark.parametrize("which", ["k", "v", "q"])
def test_gradients_of_the_pools(cuda_lib, which):
  """Pools that require a gradient get the one of the definition, from attention and from reads."""
  from torchprime_b200.ops import paged_kv
  c, table, lens = _cache()
  g = torch.Generator(device="cuda").manual_seed(3)
  q, do = (torch.randn(2, 4, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
  slots = torch.tensor([7, 90, 33], device="cuda")
  dr = torch.randn(3, 2, 64, generator=g, device="cuda").bfloat16()
  def call():
    leaf = {"q": q, "k": c.k, "v": c.v}[which].detach().clone().requires_grad_()
    cache = c._replace(**{which: leaf}) if which != "q" else c
    o = paged_kv.decode_attention(leaf if which == "q" else q, cache, table, lens)
    assert o.requires_grad
    grads = [torch.autograd.grad(o, leaf, do)[0]]
    if which != "q":
      rows = paged_kv.read(cache, slots)["kv".index(which)]
      assert rows.requires_grad
      grads.append(torch.autograd.grad(rows, leaf, dr)[0])
      with torch.no_grad():            # nothing is recorded: the kernels
        assert not paged_kv.read(cache, slots)[0].requires_grad
        assert not paged_kv.decode_attention(q, cache, table, lens).requires_grad
    return grads
  got = call()
  with ops.backend("torch"):
    want = call()
  for a, b in zip(got, want):
    assert bool(b.any()) and torch.allclose(a, b, rtol=2.0 ** -7, atol=2.0 ** -7 * float(b.abs().max()))      # (sums by atomics, in bf16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("native", [True, False])
def test_append_counts_as_a_write(cuda_lib, monkeypatch, dtype, native):
  """A graph that saved a pool notices, as it does where the definition writes; pools made for inference have no versions."""
  from torchprime_b200.ops import paged_kv
  if not native:
    monkeypatch.setattr(ops, "_native", lambda: None)
  c, _, _ = _cache(dtype)
  x = torch.randn(2, 2, 64, device="cuda").bfloat16()
  slots = torch.tensor([3, 50], device="cuda")
  pools = [t for t in c if t is not None]
  for backend in ("torch", "auto"):
    with ops.backend(backend):
      before = [t._version for t in pools]
      paged_kv.append(c, x, x, slots)
      assert all(t._version > v for t, v in zip(pools, before))
  if dtype == torch.bfloat16:
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    loss = (c.k * w).sum()             # saves the pool
    paged_kv.append(c, x, x, slots)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
      loss.backward()
  with torch.inference_mode():
    c, _, _ = _cache(dtype)
    paged_kv.append(c, x, x, slots)
  paged_kv.append(c, x, x, slots)
  assert torch.equal(paged_kv.read(c, slots)[0][0].isnan(), torch.zeros(2, 64, dtype=torch.bool, device="cuda"))
