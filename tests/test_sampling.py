"""Sampling on the CPU: the definition against a restatement in plain Python, and what is refused."""

import math
import random

import pytest
import torch

from torchprime_b200.ops.sampling import sample_tokens


def scalar(l, u, temperature, k, p, mp):
  l = [-math.inf if math.isnan(x) else x for x in l]
  top = max(l)
  if top == -math.inf:
    return -1
  if not temperature > 0:
    return l.index(top)
  w = [1.0 if x == top else 0.0 if x == -math.inf else math.exp((x - top) / temperature) for x in l]
  order = sorted(range(len(l)), key=lambda i: (-l[i], i))
  if k > 0:
    order = order[:k]
  order = [i for i in order if w[i] >= min(mp, 1.0)]
  if p < 1:
    total, c, kept = sum(w[i] for i in order), 0.0, []
    for n, i in enumerate(order):
      if n and not c < p * total:
        break
      kept.append(i)
      c += w[i]
    order = kept
  total, c = sum(w[i] for i in sorted(order)), 0.0
  for i in sorted(order):
    c += w[i]
    if c > u * total:
      return i
  return max(i for i in order if w[i] > 0)


def test_definition():
  r = random.Random(0)
  for _ in range(500):
    v = r.randint(1, 40)
    l = torch.tensor([[round(r.gauss(0, 2), 1) if r.random() < 0.9 else r.choice([-math.inf, math.nan]) for _ in range(v)]])
    u = torch.tensor([r.random()])
    args = (r.choice([0, 0.5, 1, 2.0]), r.choice([0, 1, 3, 100]), r.choice([1.0, 0.5, 0.9, 0.0]), r.choice([0, 0.1, 0.5, 1.0, 2.0]))
    assert int(sample_tokens(l, u, *args)) == scalar(l[0].double().tolist(), float(u), *args), (l, u, args)


def test_settings_for_each_row():
  l = torch.tensor([[0.0, 3.0, 1.0, 2.9]]).repeat(4, 1)
  u = torch.tensor([0.99, 0.99, 0.99, 0.0])
  got = sample_tokens(l, u, torch.tensor([0.0, 1.0, 1.0, 1.0]), torch.tensor([0, 1, 0, 0], dtype=torch.int32),
                      torch.tensor([1.0, 1.0, 0.9, 1.0]), torch.tensor([0.0, 0.0, 0.5, 0.0]))
  assert got.tolist() == [1, 1, 3, 0] and got.dtype == torch.int64


def test_frequencies_follow_the_distribution():
  g = torch.Generator().manual_seed(0)
  l = torch.tensor([[0.0, 1.0, 2.0, -1.0]]).repeat(20000, 1)
  f = torch.bincount(sample_tokens(l, torch.rand(20000, generator=g), 2.0, top_k=3), minlength=4) / 20000
  want = torch.softmax(torch.tensor([0.0, 0.5, 1.0, -math.inf]), 0)
  assert torch.allclose(f, want, atol=5 * (0.25 / 20000) ** 0.5)        # five standard deviations at most


def test_refusals():
  l, u = torch.zeros(2, 5), torch.zeros(2)
  for bad in ((l[0], u), (l, u[:1]), (l, u.double()), (l[:, :0], u), (l.long(), u)):
    with pytest.raises(ValueError):
      sample_tokens(*bad)
  for kw in ({"temperature": torch.ones(3)}, {"top_k": torch.ones(2)}, {"top_p": torch.ones(2, dtype=torch.float64)}, {"min_p": torch.ones(2, 1)}):
    with pytest.raises(ValueError):
      sample_tokens(l, u, **kw)
