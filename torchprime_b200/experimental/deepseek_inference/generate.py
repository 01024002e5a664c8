"""Batch / interactive text generation with the cached DeepSeek-V3 engine.

  python -m torchprime_b200.experimental.deepseek_inference.generate --ckpt-path <export dir> \
      --model deepseek-v2-lite [--input-file prompts.txt | --interactive] [--max-new-tokens 100] \
      [--temperature 1.0] [--top-k 50] [--top-p 0.95] [--min-p 0.05] [--attn-impl absorb] [--cache-dtype e4m3]

Capability reference: torchprime/experimental/torchax_models/deepseek_v3/generate.py:11-234
(``sample`` = Gumbel-max over temperature-scaled logits, ``generate`` = prompt-aware incremental
decode that stops at EOS, a CLI with an interactive loop and a prompts file).
"""

from __future__ import annotations

import argparse

import torch

from ...ops.sampling import sample_tokens
from .engine import DeepseekInferenceEngine


def sample(logits: torch.Tensor, temperature: float = 1.0, generator=None) -> torch.Tensor:
  """Draw one token per row: argmax(p / Exp(1)) is a sample from p (the exponential race)."""
  probs = torch.softmax(logits.float() / max(temperature, 1e-5), dim=-1)
  noise = torch.empty_like(probs).exponential_(1, generator=generator)
  return (probs / noise).argmax(dim=-1)


def next_tokens(logits, temperature, generator=None, top_k=None, top_p=None, min_p=None) -> torch.Tensor:
  """A token for every row: the largest logit at temperature 0, else drawn, among the tokens that the filters leave
  (``ops.sampling.sample_tokens``) if there are any."""
  if not temperature > 0:
    return logits.argmax(dim=-1)
  if top_k is None and top_p is None and min_p is None:
    return sample(logits, temperature, generator)
  u = torch.rand(logits.shape[0], generator=generator, device=logits.device if generator is None else generator.device)
  return sample_tokens(logits, u.to(logits.device), temperature, top_k, top_p, min_p)


def _cut(row, eos_id):
  return row[: row.index(eos_id)] if eos_id in row else row


@torch.no_grad()
def generate(engine: DeepseekInferenceEngine, prompt_tokens: list[list[int]], max_new_tokens: int, eos_id: int,
             temperature: float = 1.0, generator=None, top_k=None, top_p=None, min_p=None) -> list[list[int]]:
  """Complete every prompt by up to ``max_new_tokens`` tokens.  Prompts of different lengths
  share the batch: positions still inside a prompt keep the prompt's token, or, with the engine's paged cache, every
  sequence stands at its own position."""
  lens = [len(t) for t in prompt_tokens]
  assert prompt_tokens and min(lens) > 0 and max(lens) <= engine.max_seq_len
  draw = lambda logits: next_tokens(logits, temperature, generator, top_k, top_p, min_p)  # noqa: E731
  if engine.attn_impl == "paged":
    return _generate_paged(engine, prompt_tokens, max_new_tokens, eos_id, draw)
  total = min(engine.max_seq_len, max_new_tokens + max(lens))
  dev = engine.device
  tokens = torch.full((len(prompt_tokens), total), -1, dtype=torch.long, device=dev)
  for i, t in enumerate(prompt_tokens):
    tokens[i, : len(t)] = torch.tensor(t, dtype=torch.long, device=dev)
  prompt_mask = tokens != -1
  finished = torch.zeros(len(prompt_tokens), dtype=torch.bool, device=dev)
  prev = 0
  for cur in range(min(lens), total):
    logits = engine.forward(tokens[:, prev:cur].clamp_min(0), prev)
    nxt = draw(logits)
    nxt = torch.where(prompt_mask[:, cur], tokens[:, cur], nxt)
    tokens[:, cur] = nxt
    finished |= (~prompt_mask[:, cur]) & (nxt == eos_id)
    prev = cur
    if bool(finished.all()):
      break
  return [_cut([t for t in row[n: n + max_new_tokens] if t >= 0], eos_id) for row, n in zip(tokens.tolist(), lens)]


def _generate_paged(engine, prompt_tokens, max_new_tokens, eos_id, draw):
  """Prompts one after the other, then a step for all sequences that have not ended, each at its own position.  Sequences give back
  their pages as they end."""
  n = len(prompt_tokens)
  lens = [len(t) for t in prompt_tokens]
  most = [min(max_new_tokens, engine.max_seq_len - k) for k in lens]
  out = [[] for _ in range(n)]
  rows = [i for i in range(n) if most[i] > 0]
  try:
    if rows:
      nxt = draw(torch.cat([engine.forward(torch.tensor([prompt_tokens[i]]), 0, rows=[i]) for i in rows]))
    while rows:
      for i, t in zip(rows, nxt.tolist()):
        out[i].append(t)
      ended = [i for i in rows if out[i][-1] == eos_id or len(out[i]) == most[i]]
      engine.release(ended)   # for the others to grow
      rows = [i for i in rows if i not in ended]
      if rows:
        nxt = draw(engine.forward(torch.tensor([[out[i][-1]] for i in rows]), [lens[i] + len(out[i]) - 1 for i in rows], rows=rows))
  finally:                    # (where the pages do not suffice, too)
    engine.release(range(min(n, engine.max_batch_size)))
  return [_cut(row, eos_id) for row in out]


def main(argv=None):
  ap = argparse.ArgumentParser()
  ap.add_argument("--ckpt-path", required=True, help="directory written by model.export() or convert.py")
  ap.add_argument("--model", default="deepseek-v2-lite", help="name of a configs/model/*.yaml")
  ap.add_argument("--tokenizer", default=None, help="defaults to the checkpoint directory")
  ap.add_argument("--input-file", default="")
  ap.add_argument("--interactive", action="store_true")
  ap.add_argument("--max-new-tokens", type=int, default=100)
  ap.add_argument("--max-seq-len", type=int, default=4096)
  ap.add_argument("--temperature", type=float, default=1.0)
  ap.add_argument("--top-k", type=int, default=None, help="draw among the k largest logits")
  ap.add_argument("--top-p", type=float, default=None, help="draw among the likeliest tokens of this probability together")
  ap.add_argument("--min-p", type=float, default=None, help="draw among tokens at least this likely, the likeliest being 1")
  ap.add_argument("--attn-impl", choices=["naive", "absorb", "paged"], default="absorb")
  ap.add_argument("--cache-dtype", choices=["model", "e4m3"], default="model", help="e4m3: 8-bit keys and values (paged cache)")
  ap.add_argument("--page-size", type=int, default=64, help="tokens to a page (paged cache)")
  args = ap.parse_args(argv)
  if args.cache_dtype == "e4m3" and args.attn_impl != "paged":
    ap.error("--cache-dtype e4m3 needs --attn-impl paged")
  from transformers import AutoTokenizer

  from ...config import compose
  from ...models.model_utils import initialize_model_class
  cfg = compose("default", [f"model={args.model}"]).model
  dev = "cuda" if torch.cuda.is_available() else "cpu"
  model = initialize_model_class(cfg, device=dev, dtype=torch.bfloat16)
  model.from_pretrained(args.ckpt_path)
  tok = AutoTokenizer.from_pretrained(args.tokenizer or args.ckpt_path)
  prompts = []
  if args.input_file:
    with open(args.input_file) as f:
      prompts = [line.strip() for line in f if line.strip()]
  engine = DeepseekInferenceEngine(model, max_batch_size=max(1, len(prompts)), max_seq_len=args.max_seq_len,
                                   attn_impl=args.attn_impl, page_size=args.page_size,
                                   cache_dtype=torch.float8_e4m3fn if args.cache_dtype == "e4m3" else None)
  filters = dict(top_k=args.top_k, top_p=args.top_p, min_p=args.min_p)

  def encode(text):
    if getattr(tok, "chat_template", None):
      return tok.apply_chat_template([{"role": "user", "content": text}], add_generation_prompt=True)
    return tok.encode(text)

  if prompts:
    outs = generate(engine, [encode(p) for p in prompts], args.max_new_tokens, tok.eos_token_id, args.temperature, **filters)
    for p, o in zip(prompts, outs):
      print("Prompt:", p)
      print("Completion:", tok.decode(o, skip_special_tokens=True))
      print()
  if args.interactive or not prompts:
    while True:
      try:
        text = input(">>> ")
      except EOFError:
        break
      if text in ("/exit", "/quit"):
        break
      out = generate(engine, [encode(text)], args.max_new_tokens, tok.eos_token_id, args.temperature, **filters)[0]
      print(tok.decode(out, skip_special_tokens=True))


if __name__ == "__main__":
  main()
