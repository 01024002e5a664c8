"""The inference engine over a paged cache on the GPU: append, attention over the pages and sampling as a decode step uses them."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from torchprime_b200.config import compose
from torchprime_b200.experimental.deepseek_inference.engine import DeepseekInferenceEngine
from torchprime_b200.experimental.deepseek_inference.generate import generate
from torchprime_b200.models.deepseek_v3 import DeepseekV3ForCausalLM
from torchprime_b200.models.model_utils import set_default_dtype
from torchprime_b200.ops import paged_kv


def _model():
  cfg = compose("default", ["model=deepseek-v2-lite"]).model
  cfg["num_hidden_layers"], cfg["first_k_dense_replace"] = 2, 2
  cfg["vocab_size"], cfg["hidden_size"], cfg["intermediate_size"] = 512, 256, 256
  torch.manual_seed(0)
  with set_default_dtype(torch.bfloat16), torch.device("cuda"):
    return DeepseekV3ForCausalLM(cfg).to("cuda")


def _off(a, b):
  return ((a.float() - b.float()).norm() / b.float().norm()).item()


@pytest.mark.parametrize("dtype,most", [(None, 2.0 ** -5), (torch.float8_e4m3fn, 0.25)])
def test_decode_follows_the_contiguous_cache(cuda_lib, monkeypatch, dtype, most):
  """Prefill, part of a prompt, and single steps against the ``naive`` cache's matrix products.  Two layers, each with a result
  rounded to bf16 from weights rounded to bf16 (2 x 2 x 2^-8, doubled for what the rest of a layer makes of it); 8-bit keys and
  values are half a step, 2^-4, off each, in two layers of twice that at most."""
  calls = []
  kernel = paged_kv.decode_attention
  monkeypatch.setattr(paged_kv, "decode_attention", lambda *a, **k: calls.append(1) or kernel(*a, **k))
  model = _model()
  ids = torch.randint(0, 512, (3, 200), device="cuda")
  a = DeepseekInferenceEngine(model, 3, 256, "naive")
  b = DeepseekInferenceEngine(model, 3, 256, "paged", cache_dtype=dtype, page_size=16)
  assert _off(b.forward(ids[:, :150], 0), a.forward(ids[:, :150], 0)) < most
  assert _off(b.forward(ids[:, 150:190], 150), a.forward(ids[:, 150:190], 150)) < most
  for t in range(190, 200):
    assert _off(b.forward(ids[:, t:t + 1], t), a.forward(ids[:, t:t + 1], t)) < most
  assert len(calls) == 20


def test_sequences_at_positions_of_their_own(cuda_lib):
  """A step of a ragged batch gives each sequence what it gets alone."""
  model = _model()
  ids = torch.randint(0, 512, (3, 100), device="cuda")
  lens = [1, 37, 64]
  eng = DeepseekInferenceEngine(model, 3, 128, "paged", page_size=16)
  alone = []
  for i, n in enumerate(lens):
    eng.forward(ids[i:i + 1, :n], 0, rows=[0])
    alone.append(eng.forward(ids[i:i + 1, n:n + 1], [n], rows=[0]))
  for i, n in enumerate(lens):
    eng.forward(ids[i:i + 1, :n], 0, rows=[i])
  got = eng.forward(torch.stack([ids[i, n:n + 1] for i, n in enumerate(lens)]), lens)
  assert _off(got, torch.cat(alone)) < 2.0 ** -5


@pytest.mark.parametrize("dtype", [None, torch.float8_e4m3fn])
def test_generation(cuda_lib, dtype):
  model = _model()
  eng = DeepseekInferenceEngine(model, 4, 96, "paged", cache_dtype=dtype, page_size=16)
  prompts = [torch.randint(0, 512, (n,)).tolist() for n in (3, 17, 30, 1)]
  greedy = generate(eng, prompts, 20, -5, 0.0)
  assert [len(o) for o in greedy] == [20] * 4
  g = torch.Generator(device="cuda").manual_seed(0)
  assert generate(eng, prompts, 20, -5, 0.7, g, top_k=1) == greedy
  drawn = [generate(eng, prompts, 12, -5, 1.2, torch.Generator(device="cuda").manual_seed(7), top_k=40, top_p=0.95, min_p=0.001)
           for _ in range(2)]
  assert drawn[0] == drawn[1] and all(len(o) == 12 for o in drawn[0])             # the same numbers, the same tokens
