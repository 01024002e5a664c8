"""Serving operators as timed cases: keys and values written to and read back from a paged cache, attention of one new
token over it, and the choice of the next token from the logits.

``run`` computes each of them in plain torch operations, or, where ``own`` is set, through ``ops.paged_kv`` and
``ops.sampling``.  ``exact`` restates them in 64 bits.
"""

import math

import torch

own = False

BF16, E4M3, E8M0 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu


# ------------------------------------------------------------------------------- the cases
def listed():
  return [
    # A decode step of 48 sequences writes one token each to an 8-bit cache (8 key heads of 128): latency.
    {"name": "append_step_e4m3", "op": "append", "tokens": 48, "kv_heads": 8, "dk": 128, "dv": 128, "page": 64, "cache": "e4m3"},
    # One prompt of odd length goes to a bf16 cache of small pages.
    {"name": "append_prompt_bf16", "op": "append", "tokens": 4099, "kv_heads": 8, "dk": 128, "dv": 128, "page": 16, "cache": "bf16"},
    # Packed prompts of a whole batch are quantised as they are written.
    {"name": "append_prompts_e4m3", "op": "append", "tokens": 30011, "kv_heads": 8, "dk": 128, "dv": 128, "page": 64, "cache": "e4m3"},
    # The cached prefix of a prompt comes back as dense bf16 rows for the attention of the prompt's next part.
    {"name": "read_prefix_e4m3", "op": "read", "tokens": 5003, "kv_heads": 8, "dk": 128, "dv": 128, "page": 64, "cache": "e4m3"},
    # The same with the latent-attention model's uncompressed heads (192 and 128 wide), kept in bf16.
    {"name": "read_wide_bf16", "op": "read", "tokens": 16384, "kv_heads": 16, "dk": 192, "dv": 128, "page": 32, "cache": "bf16"},
    # A few short chats: three sequences of up to 700 tokens, 32 query heads on 8 key heads.
    {"name": "attend_few_short", "op": "attend", "batch": 3, "longest": 700, "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
     "page": 16, "cache": "bf16", "window": 0, "softcap": 0.0},
    # One very long document: all the work is along one sequence.
    {"name": "attend_one_long", "op": "attend", "batch": 1, "longest": 65521, "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
     "page": 64, "cache": "bf16", "window": 0, "softcap": 0.0},
    # Continuous batching: sequences of very different lengths over an 8-bit cache, 64 query heads.
    {"name": "attend_batch_e4m3", "op": "attend", "batch": 64, "longest": 8192, "heads": 64, "kv_heads": 8, "dk": 128, "dv": 128,
     "page": 64, "cache": "e4m3", "window": 0, "softcap": 0.0},
    # The latent-attention model with its uncompressed cache: a key head for every query head.
    {"name": "attend_wide_e4m3", "op": "attend", "batch": 24, "longest": 3001, "heads": 16, "kv_heads": 16, "dk": 192, "dv": 128,
     "page": 32, "cache": "e4m3", "window": 0, "softcap": 0.0},
    # The largest: a full batch over a bf16 cache.
    {"name": "attend_full_batch", "op": "attend", "batch": 128, "longest": 8192, "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
     "page": 64, "cache": "bf16", "window": 0, "softcap": 0.0},
    # One sequence's next token by nucleus sampling.
    {"name": "sample_one", "op": "sample", "batch": 1, "vocab": 128256, "logits": "fp32", "temperature": 0.8, "top_k": 0,
     "top_p": 0.95, "min_p": 0.0, "each": False},
    # A batch whose requests bring settings of their own, greedy ones among them.
    {"name": "sample_batch", "op": "sample", "batch": 256, "vocab": 102400, "logits": "fp32", "temperature": 1.0, "top_k": 50,
     "top_p": 0.9, "min_p": 0.05, "each": True},
  ]


HEADS = [(32, 8, 128, 128), (64, 8, 128, 128), (40, 8, 128, 128), (128, 8, 128, 128), (8, 8, 64, 64), (16, 16, 192, 128),
         (7, 1, 128, 128), (12, 4, 64, 64)]
MOST_BYTES = 1.6e9      # of a drawn case, below the largest listed one's


def _log_int(rng, lo, hi):
  return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
  op = rng.choice(["append", "read", "attend", "attend", "attend", "sample", "sample"])
  if op == "sample":
    vocab = _log_int(rng, 250, 202048)
    return {"op": op, "batch": _log_int(rng, 1, 256), "vocab": vocab, "logits": rng.choice(["fp32", "fp32", "bf16"]),
            "temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]), "top_k": rng.choice([0, 0, 1, _log_int(rng, 2, vocab)]),
            "top_p": rng.choice([1.0, 1.0, round(rng.uniform(0.05, 0.99), 3)]),
            "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.4), 3)]), "each": rng.random() < 0.4}
  heads, kv_heads, dk, dv = rng.choice(HEADS)
  case = {"op": op, "kv_heads": kv_heads, "dk": dk, "dv": dv, "page": rng.choice([16, 32, 48, 64, 128, 256]),
          "cache": rng.choice(["bf16", "e4m3"])}
  if op != "attend":
    return {**case, "tokens": _log_int(rng, 1, 30000)}
  batch = _log_int(rng, 1, 128)
  row = kv_heads * (dk + dv) * 2
  longest = _log_int(rng, 1, max(1, min(65536, int(MOST_BYTES / row) // batch)))
  return {**case, "batch": batch, "longest": longest, "heads": heads, "window": rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]),
          "softcap": rng.choice([0.0, 0.0, 0.0, 30.0])}


def _lengths(case):
  """Lengths spread over the range, the longest first: the same for every seed, so that the work is known."""
  b, most = case["batch"], case["longest"]
  return [most if i == 0 else 1 + int(((i * 0.6180339887498949) % 1.0) ** 1.5 * (most - 1)) for i in range(b)]


# ------------------------------------------------------------------------------- inputs
def _gen(seed):
  return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0, dtype=BF16):
  return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32 if dtype != BF16 else BF16) * std).to(dtype)


def _pow2(e):
  """2^e of whole numbers, exactly."""
  return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x):
  """[..., D] as e4m3 values and one power of two for the D of them: the smallest under which they fit into +-448."""
  x = x.float()
  amax = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
  m, e = torch.frexp(amax)
  e = torch.where(m <= 0.875, e - 9, e - 8).clamp(-100, 120)
  e = torch.where(amax > 0, e, 0)
  q = (x * _pow2(-e)[..., None]).clamp(-448.0, 448.0).to(E4M3)
  return q, (e + 127).to(torch.uint8).view(E8M0)


def _pools(case, g, pages, filled):
  """Cache pools [pages, page, heads, D], head-major within a page, and their scales; with rows in them if ``filled``."""
  out = {}
  for name, d in (("k", case["dk"]), ("v", case["dv"])):
    shape = (pages, case["kv_heads"], case["page"], d)
    x = _randn(g, *shape) if filled else torch.zeros(shape, device="cuda", dtype=BF16)
    if case["cache"] == "e4m3":
      if filled:   # tokens differ in size
        x.mul_(torch.exp2(torch.randint(-2, 3, shape[:-1], generator=g, device="cuda").float())[..., None].to(BF16) * 0.5)
      parts = [_quantise(c) for c in x.split(max(1, (1 << 26) // x[0].numel()))]
      x = torch.cat([q.view(torch.uint8) for q, _ in parts]).view(E4M3)
      out[name + "_scale"] = torch.cat([e.view(torch.uint8) for _, e in parts]).view(E8M0).transpose(1, 2)
    else:
      out[name + "_scale"] = None
    out[name] = x.transpose(1, 2)
  return out


def prepare(case, seed):
  g = _gen(seed)
  st = {"case": case}
  if case["op"] == "sample":
    b, v = case["batch"], case["vocab"]
    x = torch.randn(b, v, generator=g, device="cuda") * 2.0
    peaks = min(v, 24)       # a few tokens that the context makes likely
    at = torch.randint(0, v, (b, peaks), generator=g, device="cuda")
    x.scatter_add_(1, at, torch.rand(b, peaks, generator=g, device="cuda") * 9.0)
    st["logits"] = x if case["logits"] == "fp32" else x.to(BF16)
    st["u"] = torch.rand(b, generator=g, device="cuda")
    names = ("temperature", "top_k", "top_p", "min_p")
    if case["each"]:         # a setting for every row, spread around the case's; every seventh row is greedy
      i = torch.arange(b, device="cuda")
      st["temperature"] = torch.where(i % 7 == 6, 0.0, case["temperature"] * (0.5 + 0.25 * (i % 5).float()))
      st["top_k"] = torch.where(i % 3 == 1, 0, case["top_k"] + i % 11 if case["top_k"] else 0).to(torch.int32)
      st["top_p"] = torch.where(i % 4 == 2, 1.0, torch.tensor(case["top_p"], device="cuda"))
      st["min_p"] = torch.where(i % 5 == 3, 0.0, torch.tensor(case["min_p"], device="cuda"))
    else:
      st.update({n: case[n] for n in names})
    return st
  if case["op"] == "attend":
    lens = _lengths(case)
    need = [-(-n // case["page"]) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int64)
    at = 0
    for i, n in enumerate(need):
      table[i, :n] = torch.arange(at, at + n)
      at += n
    st["block_table"] = order[table.cuda()].contiguous()
    st["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["q"] = _randn(g, case["batch"], case["heads"], case["dk"], std=1.5)
    st.update(_pools(case, g, pages, True))
    return st
  t, page = case["tokens"], case["page"]
  pages = -(-t // page) + 3
  order = torch.randperm(pages, generator=g, device="cuda")
  i = torch.arange(t, device="cuda")
  st["slots"] = order[i // page] * page + i % page       # tokens in order, pages anywhere
  st.update(_pools(case, g, pages, case["op"] == "read"))
  if case["op"] == "append":
    size = torch.exp2(torch.randn(t, 1, 1, generator=g, device="cuda"))
    st["k_new"] = (_randn(g, t, case["kv_heads"], case["dk"], dtype=torch.float32) * size).to(BF16)
    st["v_new"] = (_randn(g, t, case["kv_heads"], case["dv"], dtype=torch.float32) * size).to(BF16)
  return st


# ------------------------------------------------------------------------------- plain forms
def _write(pool, scale, x, slots):
  """In place: rows ``slots`` of a pool (as a flat list of tokens) become the rows of ``x``."""
  page = pool.shape[1]
  at = (slots // page, slots % page)
  if scale is None:
    pool[at] = x
    return
  q, e = _quantise(x)
  pool.view(torch.uint8)[at] = q.view(torch.uint8)
  scale.view(torch.uint8)[at] = e.view(torch.uint8)


def _rows(pool, scale, page_ids, offsets):
  """Rows of a pool in 32 bits."""
  if scale is None:
    return pool[page_ids, offsets].float()
  e = scale.view(torch.uint8)[page_ids, offsets].to(torch.int32) - 127
  return pool.view(torch.uint8)[page_ids, offsets].view(E4M3).float() * _pow2(e)[..., None]


def _attend(st):
  case, n = st["case"], st["lengths"].long()
  page = case["page"]
  pos = torch.arange(st["block_table"].shape[1] * page, device="cuda")
  ids = st["block_table"].long()[:, pos // page]                     # [B, S]
  off = (pos % page).expand_as(ids)
  seen = pos[None] < n[:, None]
  if case["window"]:
    seen = seen & (pos[None] >= n[:, None] - case["window"])
  b, hq, d = st["q"].shape
  hkv = case["kv_heads"]
  q = st["q"].float().view(b, hkv, hq // hkv, d)
  s = torch.einsum("bhgd,bshd->bhgs", q, _rows(st["k"], st["k_scale"], ids, off)) * (1.0 / math.sqrt(d))
  if case["softcap"]:
    s = case["softcap"] * torch.tanh(s / case["softcap"])
  s = s.masked_fill(~seen[:, None, None], float("-inf"))
  p = torch.exp(s - s.amax(-1, keepdim=True))
  p = p / p.sum(-1, keepdim=True)
  o = torch.einsum("bhgs,bshd->bhgd", p, _rows(st["v"], st["v_scale"], ids, off))
  return o.reshape(b, hq, -1).to(BF16)


def _sample(st):
  x = st["logits"].double()
  b, v = x.shape
  column = lambda t: t.double()[:, None] if torch.is_tensor(t) else torch.full((b, 1), float(t), device="cuda", dtype=torch.float64)  # noqa: E731
  temperature, top_k, top_p, min_p = (column(st[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
  i = torch.arange(v, device="cuda")
  most = x.amax(-1, keepdim=True)
  greedy = torch.where(x == most, i, v).amin(-1)
  w = torch.where(x == most, 1.0, torch.exp((x - most) / torch.where(temperature > 0, temperature, 1.0)))
  order = torch.sort(x, dim=-1, descending=True, stable=True)[1]     # of equal logits the lowest index first
  ws = w.gather(1, order)
  ws = ws * ((i < torch.where(top_k > 0, top_k, v)) & (ws >= min_p))
  c = ws.cumsum(-1)
  ws = ws * ((c - ws < top_p * c[:, -1:]) | (top_p >= 1))
  w = torch.zeros_like(w).scatter_(1, order, ws)
  c = w.cumsum(-1)
  drawn = torch.where(c > st["u"].double()[:, None] * c[:, -1:], i, v).amin(-1)
  return torch.where(temperature[:, 0] > 0, drawn, greedy)


def _own_cache(st):
  from torchprime_b200.ops.paged_kv import PagedKV
  return PagedKV(st["k"], st["v"], st["k_scale"], st["v_scale"])


def run(st):
  case = st["case"]
  op = case["op"]
  if op == "append":
    if own:
      from torchprime_b200.ops import paged_kv
      paged_kv.append(_own_cache(st), st["k_new"], st["v_new"], st["slots"])
    else:
      _write(st["k"], st["k_scale"], st["k_new"], st["slots"])
      _write(st["v"], st["v_scale"], st["v_new"], st["slots"])
    return {n: st[n] for n in ("k", "v", "k_scale", "v_scale")}
  if op == "read":
    if own:
      from torchprime_b200.ops import paged_kv
      k, v = paged_kv.read(_own_cache(st), st["slots"])
    else:
      at = (st["slots"] // case["page"], st["slots"] % case["page"])
      k, v = (_rows(st[n], st[n + "_scale"], *at).to(BF16) for n in ("k", "v"))
    return {"k": k, "v": v}
  if op == "attend":
    if own:
      from torchprime_b200.ops import paged_kv
      return paged_kv.decode_attention(st["q"], _own_cache(st), st["block_table"], st["lengths"],
                                       window=case["window"] or None, softcap=case["softcap"] or None)
    return _attend(st)
  if own:
    from torchprime_b200.ops import sampling
    return sampling.sample_tokens(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                                  min_p=st["min_p"])
  return _sample(st)


# ------------------------------------------------------------------------------- what each cannot do without
def work(case):
  if case["op"] == "sample":
    n = case["batch"] * case["vocab"]
    return {"bytes": n * (4 if case["logits"] == "fp32" else 2) + case["batch"] * 12, "flops": 4 * n}
  width = case["dk"] + case["dv"]
  held = width * 2 if case["cache"] == "bf16" else width + 2
  if case["op"] != "attend":
    rows = case["tokens"] * case["kv_heads"]
    return {"bytes": rows * (2 * width + held) + 8 * case["tokens"], "flops": rows * width}
  keys = sum(min(n, case["window"] or n) for n in _lengths(case))
  return {"bytes": keys * case["kv_heads"] * held + case["batch"] * case["heads"] * width * 2 + 4 * keys // case["page"],
          "flops": 2 * keys * case["heads"] * width}


# ------------------------------------------------------------------------------- 64 bits
def _pow2_64(e):
  """2^e of whole numbers (``**`` is not exact there)."""
  return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _quantise64(x):
  """The e4m3 values (as 64-bit numbers) by their definition: four significant bits, steps of 2^-9 below 2^-6, ties to even."""
  x = x.double()
  amax = x.abs().amax(-1, keepdim=True)
  e = torch.ceil(torch.log2(torch.where(amax > 0, amax, 448.0) / 448.0))
  e = torch.where(amax > 448.0 * _pow2_64(e), e + 1, torch.where(amax <= 448.0 * _pow2_64(e - 1), e - 1, e))
  e = torch.where(amax > 0, e.clamp(min=-100), 0.0)
  y = x * _pow2_64(-e)
  step = _pow2_64(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
  return torch.round(y / step) * step, _pow2_64(e[..., 0])


def _held64(pool, scale):
  return pool.double() if scale is None else pool.float().double() * scale.float().double()[..., None]


def exact(case, seed):
  if case["op"] == "sample":
    return None              # whole numbers
  st = prepare(case, seed)
  page = case["page"]
  if case["op"] == "append":
    out = {}
    at = (st["slots"] // page, st["slots"] % page)
    for n in ("k", "v"):
      pool = st[n].float().double()
      if case["cache"] == "bf16":
        pool[at], scale = st[n + "_new"].double(), None
      else:
        scale = st[n + "_scale"].float().double()
        pool[at], scale[at] = _quantise64(st[n + "_new"])
      out[n], out[n + "_scale"] = pool, scale
    return out
  if case["op"] == "read":
    at = (st["slots"] // page, st["slots"] % page)
    flat = {}
    for n in ("k", "v"):
      pool, scale = st[n], st[n + "_scale"]
      part = pool[at] if scale is None else pool.view(torch.uint8)[at].view(E4M3)
      flat[n] = _held64(part, None if scale is None else scale.view(torch.uint8)[at].view(E8M0))
    return flat
  group = case["heads"] // case["kv_heads"]
  rows = []
  for i, n in enumerate(_lengths(case)):
    first = max(0, n - case["window"]) if case["window"] else 0
    pos = torch.arange(first, n, device="cuda")
    at = (st["block_table"][i].long()[pos // page], pos % page)
    held = []
    for name in ("k", "v"):
      pool, scale = st[name], st[name + "_scale"]
      part = pool[at] if scale is None else pool.view(torch.uint8)[at].view(E4M3)
      held.append(_held64(part, None if scale is None else scale.view(torch.uint8)[at].view(E8M0)).transpose(0, 1))
    q = st["q"][i].double().view(case["kv_heads"], group, -1)
    s = torch.matmul(q, held[0].transpose(1, 2)) / case["dk"] ** 0.5
    if case["softcap"]:
      s = case["softcap"] * torch.tanh(s / case["softcap"])
    rows.append(torch.matmul(torch.softmax(s, -1), held[1]).reshape(case["heads"], -1))
  return torch.stack(rows)
