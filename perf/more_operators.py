"""Operators around a decoder layer's attention in training as timed cases: norms of query and key heads with the position
rotation, the scaled embedding with its gradient, and dropout with the residual sum.

``run`` computes each of them in plain torch operations, or, where ``own`` is set, through ``ops.functional``.  Cases with
``grad`` are a training step's: forward and backward.  ``exact`` restates them in 64 bits.
"""

import math

import numpy as np
import torch

own = False

BF16 = torch.bfloat16


# ------------------------------------------------------------------------------- the cases
def listed():
  return [
    # A decode step: 48 sequences, each at a position of its own; latency counts.
    {"name": "qk_step", "op": "qk", "batch": 48, "seq": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rotated": 128, "weights": True,
     "interleaved": False, "positions": True, "grad": False},
    # A prompt of odd length in the form of the model with norms without weights and rotated pairs (40 query heads on 8).
    {"name": "qk_prompt_pairs", "op": "qk", "batch": 1, "seq": 2049, "heads": 40, "kv_heads": 8, "dim": 128, "rotated": 128,
     "weights": False, "interleaved": True, "positions": False, "grad": False},
    # Fine-tuning on short sequences: a small model with narrow heads.
    {"name": "qk_train_narrow", "op": "qk", "batch": 3, "seq": 701, "heads": 16, "kv_heads": 4, "dim": 64, "rotated": 64,
     "weights": True, "interleaved": False, "positions": True, "grad": True},
    # One sequence of pre-training.
    {"name": "qk_train", "op": "qk", "batch": 1, "seq": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "rotated": 128,
     "weights": True, "interleaved": False, "positions": False, "grad": True},
    # The largest: four sequences, 64 query heads.
    {"name": "qk_train_large", "op": "qk", "batch": 4, "seq": 8192, "heads": 64, "kv_heads": 8, "dim": 128, "rotated": 128,
     "weights": True, "interleaved": False, "positions": False, "grad": True},
    # The tokens of a decode step.
    {"name": "embed_step", "op": "embed", "tokens": 48, "vocab": 128256, "dim": 4096, "repeated": 0.0, "grad": False},
    # A prompt's, from the largest table.
    {"name": "embed_prompt", "op": "embed", "tokens": 4099, "vocab": 202048, "dim": 5120, "repeated": 0.0, "grad": False},
    # One sequence of pre-training: the gradient of a large table, most of whose rows have no token.
    {"name": "embed_train", "op": "embed", "tokens": 8192, "vocab": 128256, "dim": 4096, "repeated": 0.0, "grad": True},
    # A padded batch: nearly a third of the tokens are the padding's, all in one row of the gradient.
    {"name": "embed_train_padded", "op": "embed", "tokens": 65536, "vocab": 32000, "dim": 2048, "repeated": 0.3, "grad": True},
    # Dropout behind the embedding of a short sequence, forward only (recomputed layers run it once without a gradient).
    {"name": "drop_short", "op": "drop", "rows": 333, "dim": 2048, "p": 0.1, "residual": False, "grad": False},
    # Behind the embedding in training, an odd number of rows.
    {"name": "drop_embed", "op": "drop", "rows": 8197, "dim": 5120, "p": 0.05, "residual": False, "grad": True},
    # Behind a layer's output projection, with the sum of the residual stream.
    {"name": "drop_layer", "op": "drop", "rows": 16384, "dim": 4096, "p": 0.1, "residual": True, "grad": True},
  ]


HEADS = [(32, 8, 128), (32, 8, 128), (40, 8, 128), (64, 8, 128), (16, 4, 64), (12, 4, 64), (7, 1, 128), (6, 2, 96), (4, 2, 256),
         (10, 2, 80)]


def _log_int(rng, lo, hi):
  return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
  op = rng.choice(["qk", "qk", "embed", "embed", "drop"])
  grad = rng.random() < 0.6
  if op == "qk":
    heads, kv_heads, dim = rng.choice(HEADS)
    tokens = _log_int(rng, 1, min(32768, 32768 * 80 * 128 // ((heads + 2 * kv_heads) * dim)))
    batch = _log_int(rng, 1, min(tokens, 64))
    return {"op": op, "batch": batch, "seq": max(1, tokens // batch), "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotated": rng.choice([dim, dim, dim // 32 * 16]), "weights": rng.random() < 0.7, "interleaved": rng.random() < 0.4,
            "positions": rng.random() < 0.5, "grad": grad}
  if op == "embed":
    dim = 8 * _log_int(rng, 8, 900)
    return {"op": op, "tokens": _log_int(rng, 1, min(65536, (1 << 27) // dim)), "vocab": _log_int(rng, 300, min(202048, (1 << 29) // dim)),
            "dim": dim, "repeated": rng.choice([0.0, 0.0, 0.1, 0.6]), "grad": grad}
  dim = _log_int(rng, 1, 8192)
  return {"op": op, "rows": _log_int(rng, 1, (1 << 26) // dim), "dim": dim, "p": rng.choice([0.05, 0.1, 0.2, 0.5]),
          "residual": rng.random() < 0.5, "grad": grad}


# ------------------------------------------------------------------------------- inputs
def _gen(seed):
  return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0):
  return torch.randn(*shape, generator=g, device="cuda", dtype=BF16) * std


def prepare(case, seed):
  g = _gen(seed)
  st = {"case": case}
  grad = case["grad"]
  if case["op"] == "qk":
    b, s, hq, hkv, d = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
    size = torch.exp2(torch.randn(b, s, 1, generator=g, device="cuda")).to(BF16)       # tokens differ in size
    st["qkv"] = (_randn(g, b, s, (hq + 2 * hkv) * d) * size).requires_grad_(grad)
    for n in ("q_weight", "k_weight"):
      st[n] = (1 + _randn(g, d, std=0.2)).requires_grad_(grad) if case["weights"] else None
    most = s + 1000 if case["positions"] else s
    angle = torch.arange(most, device="cuda")[:, None].double() * 500000.0 ** (
      -torch.arange(0, case["rotated"], 2, device="cuda").double() / case["rotated"])
    st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    # (every sequence begins at a position of its own)
    st["pos"] = ((torch.randint(0, 1001, (b, 1), generator=g, device="cuda") + torch.arange(s, device="cuda")).to(torch.int32)
                 if case["positions"] else None)
    if grad:
      st["dq"], st["dk"], st["dv"] = (_randn(g, b, s, h, d, std=0.02) for h in (hq, hkv, hkv))
    return st
  if case["op"] == "embed":
    v, t = case["vocab"], case["tokens"]
    ids = torch.exp(torch.rand(t, generator=g, device="cuda", dtype=torch.float64) * math.log(v)).long() - 1       # frequent tokens first
    ids = ids.clamp(0, v - 1)
    repeated = torch.rand(t, generator=g, device="cuda") < case["repeated"]
    st["ids"] = torch.where(repeated, v // 2, ids)
    st["table"] = _randn(g, v, case["dim"], std=0.02).requires_grad_(grad)
    st["scale"] = math.sqrt(case["dim"])
    if grad:
      st["dout"] = _randn(g, t, case["dim"], std=0.02)
    return st
  shape = (case["rows"], case["dim"])
  st["x"] = _randn(g, *shape).requires_grad_(grad)
  st["residual"] = _randn(g, *shape).requires_grad_(grad) if case["residual"] else None
  st["seed"] = torch.tensor([seed * 0x9E3779B97F4A7C15 % (1 << 63), 1000 + seed % 1000], dtype=torch.int64, device="cuda")
  if grad:
    st["dy"] = _randn(g, *shape, std=0.02)
  return st


# ------------------------------------------------------------------------------- plain forms
SITE = 5       # dropout's place in the model


def _rotate(x, c, s, interleaved, inverse):
  """Rotation of the leading 2 * c.shape[-1] columns, by pairs (i, i + half) or (2i, 2i + 1)."""
  n = 2 * c.shape[-1]
  if inverse:
    s = -s
  a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., : n // 2], x[..., n // 2: n])
  y = (a * c - b * s, b * c + a * s)
  y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
  return torch.cat([y, x[..., n:]], -1)


def _qk(st):
  case = st["case"]
  b, s, hq, hkv, d = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
  pos = st["pos"].long() if st["pos"] is not None else torch.arange(s, device="cuda").expand(b, s)
  c, sn = st["cos"][pos][:, :, None], st["sin"][pos][:, :, None]
  x = st["qkv"].detach().view(b, s, hq + 2 * hkv, d)
  out, grads = {}, []
  for name, first, n in (("q", 0, hq), ("k", hq, hkv)):
    xf, w = x[:, :, first: first + n].float(), st[name + "_weight"]
    r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + 1e-6)
    y = xf * r
    if w is not None:
      y = y * w.detach().float()
    out[name] = _rotate(y, c, sn, case["interleaved"], False).to(BF16)
    if case["grad"]:
      g = _rotate(st["d" + name].float(), c, sn, case["interleaved"], True)
      if w is not None:
        out["d" + name + "_weight"] = (g * (xf * r)).sum((0, 1, 2)).to(BF16)
        g = g * w.detach().float()
      grads.append((r * g - xf * (r * r * r * (g * xf).mean(-1, keepdim=True))).to(BF16))
  out["v"] = x[:, :, hq + hkv:]
  if case["grad"]:
    out["dqkv"] = torch.cat([*grads, st["dv"]], 2).view(b, s, -1)
  return out


def _embed(st):
  case, ids, table = st["case"], st["ids"], st["table"].detach()
  out = {"out": (table[ids].float() * st["scale"]).to(BF16)}
  if case["grad"]:
    sums = torch.zeros(table.shape, device="cuda")
    out["dtable"] = sums.index_add_(0, ids, st["dout"].float()).mul_(st["scale"]).to(BF16)
  return out


LOW = 0xFFFFFFFF


def _philox(c, k):
  """Ten rounds of the counter-based generator Philox4x32 (Salmon et al., 2011) on 32-bit words held in int64."""
  c0, c1, c2, c3 = c
  k0, k1 = k
  for i in range(10):
    a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57            # (the low 64 bits of a product are the same with a sign)
    c0, c1, c2, c3 = ((b >> 32) & LOW) ^ c1 ^ k0, b & LOW, ((a >> 32) & LOW) ^ c3 ^ k1, a & LOW
    if i < 9:
      k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
  return c0, c1, c2, c3


def _keep(st):
  """Whether each element stays: its 16 bits of the generator against the probability in steps of 2^-16."""
  n = st["x"].numel()
  i = torch.arange((n + 7) // 8, device="cuda")
  seed, step = st["seed"][0], st["seed"][1]
  words = _philox((i & LOW, i >> 32, (step & LOW).expand_as(i), torch.full_like(i, SITE)), (seed & LOW, (seed >> 32) & LOW))
  bits = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], -1).view(-1)[:n]
  return (bits >= _threshold(st["case"])).view(st["x"].shape)


def _threshold(case):
  return round(case["p"] * 65536)


def _drop(st):
  case = st["case"]
  keep, up = _keep(st), 65536.0 / (65536 - _threshold(case))
  y = torch.where(keep, st["x"].detach().float() * up, 0.0)
  if case["residual"]:
    y = y + st["residual"].detach().float()
  out = {"y": y.to(BF16)}
  if case["grad"]:
    out["dx"] = torch.where(keep, st["dy"].float() * up, 0.0).to(BF16)
    if case["residual"]:
      out["dresidual"] = st["dy"]
  return out


PLAIN = {"qk": _qk, "embed": _embed, "drop": _drop}


# ------------------------------------------------------------------------------- the framework's operators
def _own(st):
  """Results by name, the inputs that get a gradient by the gradient's name, and the gradients of the results."""
  from torchprime_b200.ops import functional as ops
  case = st["case"]
  if case["op"] == "qk":
    q, k, v = ops.qk_norm_rope(st["qkv"], st["cos"], st["sin"], case["heads"], case["kv_heads"], case["dim"], case["seq"],
                               q_weight=st["q_weight"], k_weight=st["k_weight"], eps=1e-6, pos=st["pos"],
                               interleaved=case["interleaved"])
    wrt = {"dqkv": st["qkv"]}
    if case["weights"]:
      wrt.update(dq_weight=st["q_weight"], dk_weight=st["k_weight"])
    return {"q": q, "k": k, "v": v}, wrt, [st.get(n) for n in ("dq", "dk", "dv")]
  if case["op"] == "embed":
    return {"out": ops.embedding(st["ids"], st["table"], scale=st["scale"])}, {"dtable": st["table"]}, [st.get("dout")]
  wrt = {"dx": st["x"]}
  if case["residual"]:
    wrt["dresidual"] = st["residual"]
  return {"y": ops.dropout(st["x"], case["p"], st["seed"], site=SITE, residual=st["residual"])}, wrt, [st.get("dy")]


def run(st):
  if not own:
    with torch.no_grad():
      return PLAIN[st["case"]["op"]](st)
  if not st["case"]["grad"]:
    with torch.no_grad():
      return _own(st)[0]
  out, wrt, grads = _own(st)
  back = torch.autograd.grad(list(out.values()), list(wrt.values()), grads)
  return {**{n: t.detach() for n, t in out.items()}, **dict(zip(wrt, back))}


# ------------------------------------------------------------------------------- what each cannot do without
def work(case):
  grad = case["grad"]
  if case["op"] == "qk":
    t, d = case["batch"] * case["seq"], case["dim"]
    qk, v = t * (case["heads"] + case["kv_heads"]) * d, t * case["kv_heads"] * d
    tables = (t if case["positions"] else case["seq"]) * case["rotated"] * 4 + (t * 4 if case["positions"] else 0)
    weights = 4 * d if case["weights"] else 0
    return {"bytes": (8 * qk + 4 * v + 2 * weights if grad else 4 * qk + weights) + tables, "flops": qk * (20 if grad else 7)}
  if case["op"] == "embed":
    n, rows = case["tokens"] * case["dim"], case["vocab"] * case["dim"]
    return {"bytes": 2 * min(n, rows) + 2 * n + 8 * case["tokens"] + (2 * n + 2 * rows if grad else 0), "flops": 3 * n if grad else n}
  n = case["rows"] * case["dim"]
  return {"bytes": n * 2 * (2 + case["residual"] + (2 if grad else 0)), "flops": n * (20 if grad else 10)}


# ------------------------------------------------------------------------------- 64 bits
def _turned(x, angle_cos, angle_sin, interleaved):
  """Each pair as a complex number times cos + i sin."""
  n = 2 * angle_cos.shape[-1]
  turn = torch.complex(angle_cos, angle_sin)
  y = x.clone()
  first, second = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
  z = torch.complex(x[..., first], x[..., second]) * turn
  y[..., first], y[..., second] = z.real, z.imag
  return y


def _exact_qk(st):
  """A head at a time, the gradient as the projection orthogonal to the normalised head."""
  case = st["case"]
  b, s, hq, hkv, d = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "dim"))
  t = b * s
  pos = st["pos"].long().view(-1) if case["positions"] else torch.arange(t, device="cuda") % s
  c, sn = st["cos"].double()[pos], st["sin"].double()[pos]
  x = st["qkv"].detach().view(t, hq + 2 * hkv, d)
  out = {"q": torch.empty(t, hq, d, device="cuda", dtype=torch.float64), "k": torch.empty(t, hkv, d, device="cuda", dtype=torch.float64)}
  dx = torch.empty(t, hq + 2 * hkv, d, device="cuda", dtype=torch.float64) if case["grad"] else None
  for name, first, n in (("q", 0, hq), ("k", hq, hkv)):
    w = st[name + "_weight"]
    w = w.detach().double() if w is not None else torch.ones(d, device="cuda", dtype=torch.float64)
    dw = torch.zeros_like(w)
    for h in range(n):
      xh = x[:, first + h].double()
      length = (xh.square().sum(-1, keepdim=True) / d + 1e-6).sqrt()
      unit = xh / length
      out[name][:, h] = _turned(unit * w, c, sn, case["interleaved"])
      if case["grad"]:
        g = _turned(st["d" + name].view(t, n, d)[:, h].double(), c, -sn, case["interleaved"])
        dw += (g * unit).sum(0)
        g = g * w
        dx[:, first + h] = (g - unit * ((g * unit).sum(-1, keepdim=True) / d)) / length
    if case["grad"] and case["weights"]:
      out["d" + name + "_weight"] = dw
  out["v"] = x[:, hq + hkv:].double().view(b, s, hkv, d)
  out["q"], out["k"] = out["q"].view(b, s, hq, d), out["k"].view(b, s, hkv, d)
  if case["grad"]:
    dx[:, hq + hkv:] = st["dv"].view(t, hkv, d).double()
    out["dqkv"] = dx.view(b, s, -1)
  return out


def _exact_embed(st):
  ids, table = st["ids"], st["table"].detach()
  out = {"out": table.index_select(0, ids).double() * st["scale"]}
  if st["case"]["grad"]:
    order = torch.argsort(ids, stable=True)
    which, counts = torch.unique_consecutive(ids[order], return_counts=True)
    ends = counts.cumsum(0)
    dtable = torch.zeros(table.shape, device="cuda", dtype=torch.float64)
    for cols in range(0, table.shape[1], 512):
      rows = st["dout"][:, cols: cols + 512].double()[order]
      dtable[which, cols: cols + 512] = torch.segment_reduce(rows, "sum", offsets=torch.cat([ends.new_zeros(1), ends])) * st["scale"]
    out["dtable"] = dtable
  return out


def _exact_keep(st):
  """The generator on the host, in 64-bit words without a sign."""
  n = st["x"].numel()
  seed, step = (int(v) for v in st["seed"].tolist())
  i = np.arange((n + 7) // 8, dtype=np.uint64)
  low, half = np.uint64(LOW), np.uint64(32)
  w = [i & low, i >> half, np.full_like(i, step & LOW), np.full_like(i, SITE)]
  key = [seed & LOW, seed >> 32 & LOW]
  for _ in range(10):
    p, q = w[0] * np.uint64(0xD2511F53), w[2] * np.uint64(0xCD9E8D57)
    w = [(q >> half) ^ w[1] ^ np.uint64(key[0]), q & low, (p >> half) ^ w[3] ^ np.uint64(key[1]), p & low]
    key = [(key[0] + 0x9E3779B9) & LOW, (key[1] + 0xBB67AE85) & LOW]
  bits = np.stack([v.astype(np.uint32) for v in w], -1).reshape(-1).view(np.uint16)[:n]        # (little-endian: the low half first)
  return torch.from_numpy(bits >= _threshold(st["case"])).cuda().view(st["x"].shape)


def _exact_drop(st):
  case = st["case"]
  stays = 1.0 - _threshold(case) / 65536
  keep = _exact_keep(st).double()
  y = st["x"].detach().double() * keep / stays
  out = {"y": y + st["residual"].detach().double() if case["residual"] else y}
  if case["grad"]:
    out["dx"] = st["dy"].double() * keep / stays
    if case["residual"]:
      out["dresidual"] = st["dy"].double()
  return out


def exact(case, seed):
  with torch.no_grad():
    return {"qk": _exact_qk, "embed": _exact_embed, "drop": _exact_drop}[case["op"]](prepare(case, seed))
