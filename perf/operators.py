"""Workloads of the operators that answer with a model: the paged key-value cache, attention over it, and sampling.

A case is a plain dict; ``kind`` names the operator that it drives:

* ``attend``  attention of one new token per sequence over the paged cache (``ops.paged_attention``)
* ``store``   new keys and values put into the pages (``ops.kv_cache_write``), in the cache's own 16-bit or 32-bit type
* ``read``    cached keys and values laid out in rows again (``ops.kv_cache_read``)
* ``chunk``   a piece of a prompt stored in 8 bits and all that is cached so far read back, as the attention of a prompt
              that arrives in pieces needs it (``ops.kv_cache_write`` then ``ops.kv_cache_read``)
* ``sample``  the next tokens from logits and given random numbers (``ops.sample``)

Where ``own`` is false a pass computes the same from elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}
ESIZE = {"bf16": 2, "f16": 2, "f32": 4, "fp8": 1}
FP8_MAX = 448.0
TINY = 2.0**-100  # rows whose largest value is below are stored as zeros
GRID = 2.0**-12  # (w + GRID) - GRID in 32 bits is a multiple of 2^-35: sums of such weights in 64 bits are exact
LOG2E = 1.4426950408889634


# ------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------
def _attend(name, B, Hq, Hkv, Dqk, Dv, lo, hi, page, dtype, cache, ragged=0, window=0, cap=0.0, slots_first=False):
  c = dict(kind="attend", B=B, Hq=Hq, Hkv=Hkv, Dqk=Dqk, Dv=Dv, lo=lo, hi=hi, page=page, dtype=dtype, cache=cache, ragged=ragged,
           window=window, cap=cap, slots_first=slots_first)  # fmt: skip
  return dict(c, name=name) if name else c


def _store(name, kind, B, S, Hkv, Dqk, Dv, lo, hi, page, dtype, cache, ragged=0, slots_first=False):
  c = dict(kind=kind, B=B, S=S, Hkv=Hkv, Dqk=Dqk, Dv=Dv, lo=lo, hi=hi, page=page, dtype=dtype, cache=cache, ragged=ragged,
           slots_first=slots_first)  # fmt: skip
  return dict(c, name=name) if name else c


def _sample(name, B, V, dtype, rows, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
  c = dict(kind="sample", B=B, V=V, dtype=dtype, rows=rows, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
  return dict(c, name=name) if name else c


def listed():
  return [
    # The first tokens of one answer after a short prompt, Llama-3-8B's heads: nothing but latency.
    _attend("attend_one_short", 1, 32, 8, 128, 128, 461, 461, 16, "bf16", "bf16"),
    # A batch of answers of very different lengths under way, Llama-3-70B's heads.
    _attend("attend_ragged_batch", 32, 64, 8, 128, 128, 7, 4096, 64, "bf16", "bf16", ragged=3),
    # One answer at the end of the longest context the configurations allow (131072 positions).
    _attend("attend_one_long", 1, 32, 8, 128, 128, 131072, 131072, 64, "bf16", "bf16"),
    # Serving at full load: many sequences, the cache in 8 bits so that they fit.
    _attend("attend_fp8_full", 128, 32, 8, 128, 128, 512, 8192, 64, "bf16", "fp8", ragged=5),
    # DeepSeek-V3's heads (192 for keys, 128 for values, one key head per query head) with odd lengths, in float16.
    _attend("attend_192_odd", 4, 128, 128, 192, 128, 3, 1537, 32, "f16", "f16", ragged=2),
    # The small fp32 configuration, as a parity run generates with it.
    _attend("attend_f32_small", 2, 8, 8, 64, 64, 77, 129, 16, "f32", "f32", ragged=1),
    # One new token of each of 64 sequences goes into the cache: a few KB, latency only.
    _store("store_step", "store", 64, 1, 8, 128, 128, 1, 255, 64, "bf16", "bf16", ragged=4),
    # The keys and values of a batch of whole prompts.
    _store("store_prompts", "store", 4, 8192, 8, 128, 128, 0, 0, 64, "bf16", "bf16"),
    # Cached prompts of different lengths laid out for the prompt attention again.
    _store("read_ragged", "read", 4, 0, 8, 128, 128, 999, 8000, 64, "bf16", "bf16", ragged=6),
    # The next piece of two long prompts, stored in 8 bits; its attention reads all that came before, too.
    _store("chunk_fp8", "chunk", 2, 2048, 8, 128, 128, 1000, 6001, 64, "bf16", "fp8", ragged=7),
    # One user's next token from Llama 3's vocabulary, with the usual settings: latency.
    _sample("sample_one", 1, 128256, "f32", False, 0.8, 50, 0.95, 0.0),
    # The next tokens of a full batch, each request with settings of its own (greedy ones and unfiltered ones among them).
    _sample("sample_batch", 256, 128256, "f32", True),
  ]


def _log_int(rng, lo, hi):
  n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
  return n + 1 if n == 3072 else n


def draw(rng):
  kind = rng.choices(["attend", "store", "read", "chunk", "sample"], [8, 2, 2, 2, 4])[0]
  page, ragged = rng.choice([8, 16, 32, 64, 128]), rng.randrange(1, 10000)
  slots_first = rng.random() < 0.3
  half = "bf16" if rng.random() < 0.7 else "f16"
  if kind == "sample":
    V = rng.choice([256, 32000, 50257, 128256, 128256])
    B = _log_int(rng, 1, 256)
    dtype = rng.choice(["f32", "f32", half])
    if rng.random() < 0.5:
      return _sample(None, B, V, dtype, True)
    return _sample(None, B, V, dtype, False, rng.choice([0.0, 0.5, 0.7, 1.0, 1.3]), rng.choice([0, 0, 1, 20, 64, 400]),
                   rng.choice([1.0, 0.9, 0.95, 0.5]), rng.choice([0.0, 0.0, 0.05]))  # fmt: skip
  Hq, Hkv, Dqk, Dv = rng.choice([(32, 8, 128, 128), (64, 8, 128, 128), (8, 8, 64, 64), (32, 8, 64, 64), (128, 128, 192, 128),
                                 (16, 16, 192, 128), (48, 3, 128, 128)])  # fmt: skip
  if kind == "attend":
    f32 = Dqk == Dv and rng.random() < 0.12
    cache = "f32" if f32 else rng.choice([half, half, "fp8"])
    # cached values of the longest sequences that the largest listed cases have, over the whole batch
    most = 131072 * 8 * 256 // (Hkv * (Dqk + Dv)) // (8 if f32 else 1)
    B = _log_int(rng, 1, 128)
    hi = _log_int(rng, 1, max(1, min(131072, most // B)))
    lo = max(1, hi // rng.choice([1, 4, 50]))
    window = _log_int(rng, 1, max(2, hi)) if rng.random() < 0.15 else 0
    return _attend(None, B, Hq, Hkv, Dqk, Dv, lo, hi, page, "f32" if f32 else half, cache, ragged, window,
                   30.0 if rng.random() < 0.15 else 0.0, slots_first)  # fmt: skip
  most = 4 * 8192 * 8 * 256 // (Hkv * (Dqk + Dv))
  B = _log_int(rng, 1, 64)
  hi = _log_int(rng, 1, max(1, min(8192, most // (2 * B))))
  lo = max(1, hi // rng.choice([1, 3, 20]))
  if kind == "read":
    f32 = rng.random() < 0.1
    return _store(None, kind, B, 0, Hkv, Dqk, Dv, lo, hi, page, "f32" if f32 else half,
                  "f32" if f32 else rng.choice([half, half, "fp8"]), ragged, slots_first)  # fmt: skip
  S = 1 if rng.random() < 0.3 else _log_int(rng, 2, max(2, min(8192, most // (2 * B))))
  cache = "fp8" if kind == "chunk" else half
  return _store(None, kind, B, S, Hkv, Dqk, Dv, lo, hi, page, half, cache, ragged, slots_first)


def _lengths(case):
  """Tokens cached of each sequence before the pass: spread over the logarithm of lo..hi, the longest first."""
  lo, hi, rng = case["lo"], case["hi"], random.Random(case["ragged"])
  return [hi] + [_log_int(rng, lo, hi) if lo < hi else hi for _ in range(case["B"] - 1)]


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _cache(gen, pages, H, page, D, dtype, slots_first):
  """A cache whose pages all hold something, as after some time of use."""
  shape = (pages, page, H, D) if slots_first else (pages, H, page, D)
  x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
  x = x.transpose(1, 2) if slots_first else x
  if dtype != torch.float8_e4m3fn:
    return x.to(dtype), None
  return _quantise(x)


def prepare(case, seed):
  gen, rng = torch.Generator(device="cuda").manual_seed(seed), random.Random(seed)
  kind, B = case["kind"], case["B"]
  dt = DTYPES[case["dtype"]]
  normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)  # noqa: E731
  st = {"case": case}
  if kind == "sample":
    V = case["V"]
    # what a language model's head gives: a wide bulk and a few dozen candidates that stand out of it
    logits = 2.0 * normal(B, V)
    best = torch.randint(V, (B, min(V, 64)), generator=gen, device="cuda")
    bump = 4.0 + 10.0 * torch.rand(best.shape, generator=gen, device="cuda") ** 3
    st["logits"] = logits.scatter_(1, best, bump).to(dt)
    st["uniform"] = torch.rand((B,), generator=gen, device="cuda")
    if case["rows"]:
      pick = lambda xs, t: torch.tensor([rng.choice(xs) for _ in range(B)], dtype=t, device="cuda")  # noqa: E731
      st["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.25], torch.float32)
      st["top_k"] = pick([0, 0, 20, 50, 200], torch.int32)
      st["top_p"] = pick([0.8, 0.95, 1.0, 1.0], torch.float32)
      st["min_p"] = pick([0.0, 0.0, 0.02, 0.1], torch.float32)
    else:
      st.update({n: case[n] for n in ("temperature", "top_k", "top_p", "min_p")})
    return st
  Hkv, Dqk, Dv, page = case["Hkv"], case["Dqk"], case["Dv"], case["page"]
  past = _lengths(case)
  new = case.get("S", 0)
  # the pages of a sequence, those of its new tokens among them, lie anywhere in the cache
  need = [max(1, -(-(n + new) // page)) for n in past]
  where = torch.randperm(sum(need) + 3, generator=gen, device="cuda").to(torch.int32)
  st["table"] = torch.full((B, max(need)), -1, dtype=torch.int32, device="cuda")
  at = 0
  for b, n in enumerate(need):
    st["table"][b, :n] = where[at : at + n]
    at += n
  st["k_cache"], st["k_scale"] = _cache(gen, sum(need) + 3, Hkv, page, Dqk, DTYPES[case["cache"]], case["slots_first"])
  st["v_cache"], st["v_scale"] = _cache(gen, sum(need) + 3, Hkv, page, Dv, DTYPES[case["cache"]], case["slots_first"])
  st["lengths"] = torch.tensor(past, dtype=torch.int32, device="cuda")
  st["longest"] = max(past) + new
  if kind == "attend":
    st["q"] = normal(B, 1, case["Hq"], Dqk).to(dt).transpose(1, 2)
  elif new:
    # as the projections leave them: views of (batch, sequence, head, dim) memory
    st["k"], st["v"] = (normal(B, new, Hkv, d).to(dt).transpose(1, 2) for d in (Dqk, Dv))
    st["total"] = st["lengths"] + new
  return st


# ------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------
def _quantise(x):
  """Rows of the last dimension in 8 bits with a scale each: x is about stored * scale."""
  x = x.float()
  top = x.abs().amax(-1)
  some = top >= TINY
  scale = torch.where(some, top / FP8_MAX, 0.0)
  back = torch.where(some, FP8_MAX / top, 0.0)
  return (x * back[..., None]).to(torch.float8_e4m3fn), scale


def _store_rows(cache, scale, x, page, slot):
  """x (batch, head, token, dim) to the places that page and slot (batch, token) name."""
  rows = x.transpose(1, 2)
  if scale is None:
    cache[page, :, slot] = rows.to(cache.dtype)
    return
  stored, s = _quantise(rows)
  cache.view(torch.uint8)[page, :, slot] = stored.view(torch.uint8)
  scale[page, :, slot] = s


def _plain_store(st):
  S, page = st["k"].shape[2], st["k_cache"].shape[2]
  at = st["lengths"][:, None].long() + torch.arange(S, device="cuda")
  pages, slots = st["table"].gather(1, at // page).long(), at % page
  _store_rows(st["k_cache"], st["k_scale"], st["k"], pages, slots)
  _store_rows(st["v_cache"], st["v_scale"], st["v"], pages, slots)


def _gathered(cache, scale, table, n):
  """The first n positions of every sequence, (batch, head, n, dim), in 32 bits."""
  pages = table.clamp(min=0).long()[:, : -(-n // cache.shape[2])]
  x = cache.view(torch.uint8)[pages].view(cache.dtype) if scale is not None else cache[pages]
  x = x.float() if scale is None else x.float() * scale[pages][..., None]
  x = x.permute(0, 2, 1, 3, 4)
  return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])[:, :, :n]


def _plain_read(st, lengths):
  n, dt = st["longest"], DTYPES[st["case"]["dtype"]]
  real = (torch.arange(n, device="cuda") < lengths[:, None])[:, None, :, None]
  return [torch.where(real, _gathered(st[f"{x}_cache"], st[f"{x}_scale"], st["table"], n), 0.0).to(dt) for x in "kv"]


def _plain_attend(st):
  case, q, n = st["case"], st["q"], st["longest"]
  B, Hq, _, D = q.shape
  at = torch.arange(n, device="cuda")
  seen = at < st["lengths"][:, None]
  if case["window"]:
    seen = seen & (at >= st["lengths"][:, None] - 1 - case["window"])
  seen = seen[:, None, None, :]
  k = _gathered(st["k_cache"], st["k_scale"], st["table"], n)
  v = torch.where(seen.transpose(2, 3), _gathered(st["v_cache"], st["v_scale"], st["table"], n), 0.0)
  s = q.float().reshape(B, k.shape[1], Hq // k.shape[1], D) @ k.transpose(2, 3) / math.sqrt(case["Dv"])
  if case["cap"]:
    s = case["cap"] * torch.tanh(s / case["cap"])
  s = torch.where(seen, s, -math.inf)
  p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
  out = (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
  return [out.reshape(B, Hq, 1, -1).to(q.dtype)]


def _settings(st):
  """The settings as (batch, 1) tensors."""
  B = st["logits"].shape[0]
  for name, t in (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32)):
    x = st[name]
    yield (x if isinstance(x, torch.Tensor) else torch.full((B,), x, dtype=t, device="cuda"))[:, None]


def _plain_sample(st):
  temperature, top_k, top_p, min_p = _settings(st)
  x = st["logits"].float()
  x = torch.where(x == x, x, -math.inf)
  V = x.shape[1]
  ranked, order = torch.sort(x, dim=-1, descending=True, stable=True)
  best = ranked[:, :1]
  # weights relative to the best, on a grid on which sums in 64 bits are exact in any order
  w = torch.exp2((ranked - best) * (LOG2E / temperature))
  w = torch.where(ranked == best, 1.0, w)
  w = ((w + GRID) - GRID).double()
  rank = torch.arange(V, device="cuda")
  greedy = ~(temperature > 0)
  w = torch.where((top_k <= 0) | (rank < top_k), w, 0.0)
  upto = w.cumsum(-1)
  kept = (upto - w < top_p.double() * upto[:, -1:]) & (w >= min_p.clamp(max=1.0)) & (w > 0)
  kept = torch.where(greedy, rank == 0, kept | (rank == 0))
  w = torch.where(kept, w, 0.0)
  mass = w.sum(-1, keepdim=True)
  # the draw goes through the kept tokens by their indices
  w = torch.zeros_like(w).scatter_(1, order, w)
  goal = st["uniform"][:, None].clamp(0.0, 1.0 - 2.0**-24).double() * mass
  token = (w.cumsum(-1) <= goal).sum(-1, keepdim=True)
  logprob = torch.log(w.gather(1, token) / mass).float()
  none = best == -math.inf
  return [torch.where(none, -1, token)[:, 0], torch.where(none, -math.inf, logprob)[:, 0]]


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(st):
  kind = st["case"]["kind"]
  if not own:
    if kind == "attend":
      return _plain_attend(st)
    if kind == "sample":
      return _plain_sample(st)
    if kind in ("store", "chunk"):
      _plain_store(st)
    return [st["k_cache"], st["v_cache"]] if kind == "store" else _plain_read(st, st["total"] if kind == "chunk" else st["lengths"])
  from torchprime_amd import ops

  if kind == "sample":
    return list(ops.sample(st["logits"], st["uniform"], st["temperature"], st["top_k"], st["top_p"], st["min_p"]))
  cache = (st["k_cache"], st["v_cache"], st["table"])
  scales = dict(k_scale=st["k_scale"], v_scale=st["v_scale"])
  case = st["case"]
  if kind == "attend":
    return [ops.paged_attention(st["q"], *cache, st["lengths"], window_left=case["window"] or None, soft_cap=case["cap"] or None, **scales)]
  if kind in ("store", "chunk"):
    ops.kv_cache_write(st["k"], st["v"], *cache, st["lengths"], **scales)
  if kind == "store":
    return [st["k_cache"], st["v_cache"]]
  return list(ops.kv_cache_read(*cache, st["total"] if kind == "chunk" else st["lengths"], st["longest"], dtype=DTYPES[case["dtype"]], **scales))


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
  kind, B, e = case["kind"], case["B"], ESIZE[case["dtype"]]
  if kind == "sample":
    return {"bytes": float(B * case["V"] * e + B * 32), "flops": 10.0 * B * case["V"]}
  Hkv, D = case["Hkv"], case["Dqk"] + case["Dv"]
  past = _lengths(case)
  row = Hkv * (D * ESIZE[case["cache"]] + (8 if case["cache"] == "fp8" else 0))  # one cached token
  if kind == "attend":
    seen = sum(min(n, case["window"] + 1) if case["window"] else n for n in past)
    return {"bytes": float(seen * row + B * case["Hq"] * D * e + seen // case["page"] * 4), "flops": 2.0 * seen * case["Hq"] * D}
  new = B * case["S"]
  if kind == "store":
    return {"bytes": float(new * (Hkv * D * e + row)), "flops": float(new * Hkv * D)}
  # the rows come out at one length, zeros where a sequence is shorter
  out = B * (max(past) + case["S"]) * Hkv * D * e
  return {"bytes": float(new * (Hkv * D * e + row) + sum(past) * row + out), "flops": float((2 * new + sum(past)) * Hkv * D)}


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------
def _e4m3(y):
  """float64 values rounded to the nearest float8_e4m3fn, halves to even: three bits behind the leading one, down to 2^-9."""
  _, e = torch.frexp(y.abs())
  step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
  return ((y / step).round() * step).clamp(-448.0, 448.0)


def _values(cache, scale, table_row, n):
  """What the first n positions of one sequence hold, (head, n, dim) in float64."""
  at = torch.arange(n, device="cuda")
  pages, slots = table_row.long()[at // cache.shape[2]], at % cache.shape[2]
  x = cache.view(torch.uint8)[pages, :, slots].view(cache.dtype) if scale is not None else cache[pages, :, slots]
  x = x.double()
  if scale is not None:
    x *= scale[pages, :, slots].double()[..., None]
  return x.transpose(0, 1)


def exact(case, seed):
  st = prepare(case, seed)
  kind, B = case["kind"], case["B"]
  if kind == "sample":
    x = st["logits"].double()
    logprobs = torch.empty((B,), dtype=torch.float64, device="cuda")
    settings = [s[:, 0] for s in _settings(st)]
    t, k, p, lo = ([float(v) for v in s.tolist()] for s in settings)
    u = st["uniform"].double().tolist()
    for b in range(B):
      row = x[b]
      if not t[b] > 0:
        logprobs[b] = 0.0
        continue
      prob = torch.softmax(row / t[b], -1)
      down = torch.argsort(row, descending=True, stable=True)
      if k[b] > 0:
        down = down[: int(k[b])]
      share = prob[down] / prob[down].sum()
      share_before = share.cumsum(0) - share
      keep = (share_before < p[b]) & (share >= lo[b] * share[0])
      chosen = down[keep]
      left = torch.zeros_like(prob)
      left[chosen] = prob[chosen] / prob[chosen].sum()
      token = torch.searchsorted(left.cumsum(0), torch.tensor(u[b], dtype=torch.float64, device="cuda"), right=True)
      logprobs[b] = left[min(int(token), case["V"] - 1)].log()
    return [None, logprobs]
  past, page = _lengths(case), case["page"]
  if kind == "attend":
    outs = []
    rep = case["Hq"] // case["Hkv"]
    for b, n in enumerate(past):
      first = max(0, n - 1 - case["window"]) if case["window"] else 0
      k = _values(st["k_cache"], st["k_scale"], st["table"][b], n)[:, first:]
      v = _values(st["v_cache"], st["v_scale"], st["table"][b], n)[:, first:]
      q = st["q"][b, :, 0].double().view(case["Hkv"], rep, -1)
      s = (q[:, :, None, :] * k[:, None]).sum(-1) / math.sqrt(case["Dv"]) if n < 4096 else torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(case["Dv"])
      if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
      outs.append(torch.bmm(torch.softmax(s, -1), v.contiguous()).reshape(case["Hq"], 1, -1))
    return [torch.stack(outs)]
  rows = {}
  for x in "kv":
    cache, scale = st[f"{x}_cache"], st[f"{x}_scale"]
    if kind == "store":
      out = cache.double()
    else:
      out = torch.zeros((B, case["Hkv"], st["longest"], cache.shape[3]), dtype=torch.float64, device="cuda")
    for b, n in enumerate(past):
      if kind != "store":
        out[b, :, :n] = _values(cache, scale, st["table"][b], n)
      if kind == "read":
        continue
      at = torch.arange(n, n + case["S"], device="cuda")
      fresh = st[x][b].double()
      if kind == "store":
        out[st["table"][b].long()[at // page], :, at % page] = fresh.transpose(0, 1)
      else:
        top = fresh.abs().amax(-1, keepdim=True)
        out[b, :, n:n + case["S"]] = _e4m3(fresh * (448.0 / top)) * (top / 448.0)
    rows[x] = out
  return [rows["k"], rows["v"]]
