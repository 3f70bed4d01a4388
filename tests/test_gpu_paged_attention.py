"""Attention of one new token per sequence over the paged cache, against the formula in 64 bits.

Bounds, element by element: an output is a mean of values v_j with weights p_j, A = sum p_j |v_j| >= |out|.  Logits that are off by e
move it by at most 2 e A, e = (D + 8) 2^-23 * scale * max_j sum |q||k_j| for sums of D products in fp32 (plus cap * 2^-20 for the
soft cap's tanh); the sums of weights and values, and weights as two 16-bit numbers, by 2^-17 A at most.  Rounding the result adds
half a step, at most 2 u |out| <= u (|out| + A) with u = 2^-9 (bfloat16), 2^-12 (float16), u |out| with u = 2^-24 (float32), or half
of the type's smallest step (2^-25 in float16) where that is more."""

import math

import pytest
import torch

from tests.test_gpu_kv_cache import BF16, DEV, F16, F32, FP8, new_cache, table_for
from tests.util import randn
from torchprime_amd import ops

pytestmark = pytest.mark.gpu
UNIT = {BF16: 2.0**-9, F16: 2.0**-12, F32: 2.0**-24}
STEP = {BF16: 1e-40, F16: 2.0**-25, F32: 1e-40}


def formula(q, kc, vc, table, lengths, sm_scale=None, window=None, cap=None, ks=None, vs=None):
  """(out, the bound of its error, lse, the bound of its), in float64 on the CPU."""
  B, Hq, _, D = q.shape
  H, page, Dv = kc.shape[1], kc.shape[2], vc.shape[3]
  scale = 1 / math.sqrt(Dv) if sm_scale is None else sm_scale
  u = UNIT[q.dtype]
  out, bound = torch.zeros((B, Hq, 1, Dv), dtype=torch.float64), torch.zeros((B, Hq, 1, Dv), dtype=torch.float64)
  lse, lse_bound = torch.full((B, Hq, 1), -math.inf, dtype=torch.float64), torch.zeros((B, Hq, 1), dtype=torch.float64)
  for b in range(B):
    n = min(int(lengths[b]), table.shape[1] * page)
    at = [t for t in range(max(0, n - 1 - window) if window is not None else 0, n) if 0 <= table[b, t // page] < kc.shape[0]]
    if not at:
      continue
    t = torch.tensor(at)
    pages, slots = table[b].long()[t // page], t % page
    k, v = kc.view(torch.uint8)[pages, :, slots].view(kc.dtype) if ks is not None else kc[pages, :, slots], None
    v = vc.view(torch.uint8)[pages, :, slots].view(vc.dtype) if vs is not None else vc[pages, :, slots]
    k, v = k.double().transpose(0, 1), v.double().transpose(0, 1)
    if ks is not None:
      k, v = k * ks[pages, :, slots].double().t()[..., None], v * vs[pages, :, slots].double().t()[..., None]
    for h in range(Hq):
      kh, vh, qh = k[h // (Hq // H)], v[h // (Hq // H)], q[b, h, 0].double()
      s = (kh @ qh) * scale
      e = (D + 8) * 2.0**-23 * scale * float((kh.abs() @ qh.abs()).max())
      if cap is not None:
        s, e = cap * torch.tanh(s / cap), e + cap * 2.0**-20
      p = torch.softmax(s, 0)
      out[b, h, 0] = p @ vh
      bound[b, h, 0] = u * (p @ vh).abs() + ((u if q.dtype != F32 else 0.0) + 2 * e + 2.0**-17) * (p @ vh.abs()) + STEP[q.dtype]
      lse[b, h, 0] = torch.logsumexp(s, 0)
      lse_bound[b, h, 0] = e + 2.0**-19 * (1 + abs(float(lse[b, h, 0])))
  return out, bound, lse, lse_bound


def check(q, kc, vc, table, lengths, sm_scale=None, window=None, cap=None, ks=None, vs=None):
  dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
  out, bound, lse, lse_bound = formula(q, kc, vc, table, lengths, sm_scale, window, cap, ks, vs)
  n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
  args = (dev(q), dev(kc), dev(vc), dev(table), n)
  got = ops.paged_attention(*args, sm_scale, window_left=window, soft_cap=cap, k_scale=dev(ks), v_scale=dev(vs))
  scale = 1 / math.sqrt(vc.shape[3]) if sm_scale is None else sm_scale
  got2, got_lse = ops.paged_attn(*args, scale, -1 if window is None else window, cap or 0.0, dev(ks), dev(vs))
  assert got.shape == out.shape and got.dtype == q.dtype and torch.equal(got, got2)
  worst = ((got.double().cpu() - out).abs() - bound).max().item()
  assert worst <= 0, f"an output exceeds its bound by {worst:.3e}"
  some = torch.isfinite(lse)
  assert torch.equal(torch.isfinite(got_lse.cpu()), some) and (got_lse.cpu()[~some] == -math.inf).all()
  assert ((got_lse.cpu().double() - lse).abs()[some] <= lse_bound[some]).all()
  return got


def problem(B, Hq, H, Dk, Dv, page, lengths, dtype, cache=None, slots_first=False, seed=1, width=None, garbage=True):
  width = width or max(1, -(-max(lengths) // page))
  pages = B * width + 2
  table = table_for(B, width, pages, seed)
  cdt = cache or dtype
  kc, vc = (new_cache(pages, H, page, d, cdt, slots_first, seed + 1 + i) for i, d in enumerate((Dk, Dv)))
  ks = vs = None
  if cdt == FP8:
    ks, vs = randn((pages, H, page), seed + 3).abs() + 0.1, randn((pages, H, page), seed + 4).abs() * 0.01
  if garbage:  # what lies in slots that no sequence has reached takes no part
    nan = float("nan")
    used = torch.zeros((pages, page), dtype=torch.bool)
    for b, n in enumerate(lengths):
      for t in range(n):
        used[table[b, t // page], t % page] = True
    for c, s in ((kc, ks), (vc, vs)):
      if cdt == FP8:
        c.view(torch.uint8)[(~used)[:, None, :, None].expand_as(c)] = 0x7F
        s[(~used)[:, None].expand_as(s)] = nan
      else:
        c[(~used)[:, None, :, None].expand_as(c)] = nan
    for b, n in enumerate(lengths):  # entries behind a sequence's pages name none, or a page of NaN
      table[b, -(-n // page):] = -1 if b % 2 else pages - 1
  q = randn((B, 1, Hq, Dk), seed + 5, dtype).transpose(1, 2)
  return dict(q=q, kc=kc, vc=vc, table=table, lengths=lengths, ks=ks, vs=vs)


HEADS = [(32, 8, 128, 128), (8, 8, 64, 64), (8, 1, 64, 64), (16, 16, 192, 128), (40, 2, 192, 128), (34, 2, 128, 128)]


@pytest.mark.parametrize("dtype,cache", [(BF16, None), (F16, None), (F32, None), (BF16, FP8), (F16, FP8)])
@pytest.mark.parametrize("Hq,H,Dk,Dv", HEADS)
@pytest.mark.parametrize("page,slots_first", [(8, False), (16, True), (64, False)])
def test_lengths_from_none_to_some_hundreds(Hq, H, Dk, Dv, page, slots_first, dtype, cache):
  check(**problem(8, Hq, H, Dk, Dv, page, [1, 0, 2, 31, 33, 64, 129, 401], dtype, cache, slots_first))


@pytest.mark.parametrize("dtype,cache", [(BF16, None), (F16, None), (F32, None), (BF16, FP8), (F16, FP8)])
@pytest.mark.parametrize("lengths", [[8191], [5000, 1, 4097, 0, 2048], [1500] * 9])
def test_long_sequences_are_split_and_joined(lengths, dtype, cache):
  check(**problem(len(lengths), 8, 2, 128, 128, 32, lengths, dtype, cache, garbage=len(lengths) == 5))


@pytest.mark.parametrize("dtype,cache", [(BF16, None), (F32, None), (BF16, FP8)])
@pytest.mark.parametrize("window", [0, 1, 30, 511, 100000])
def test_windows(window, dtype, cache):
  check(**problem(5, 8, 2, 128, 128, 16, [1, 0, 30, 700, 1900], dtype, cache), window=window)


@pytest.mark.parametrize("dtype,cache", [(BF16, None), (F16, None), (F32, None), (BF16, FP8)])
def test_soft_cap_and_scale(dtype, cache):
  p = problem(3, 8, 2, 64, 64, 16, [5, 300, 1100], dtype, cache)
  check(**p, cap=5.0)
  check(**p, cap=30.0, sm_scale=1.3, window=200)
  check(**p, sm_scale=0.01)


@pytest.mark.parametrize("Hq,H,Dk,Dv", [(8, 2, 64, 64), (8, 2, 128, 128), (4, 4, 192, 128)])
@pytest.mark.parametrize("factor", [1.0, 0.05])
@pytest.mark.parametrize("cap", [0.5, 30.0, 1000.0, 1e5])
def test_soft_cap_in_fp32(cap, factor, Hq, H, Dk, Dv):
  """fp32 has no weights in 16 bits, and the soft cap adds errors relative to the logit, however large the cap is.  With S = scale *
  max_j sum |q||k_j| >= |s_j|, a capped logit is off by (D + 8) 2^-23 S (its sum; the cap shrinks that) and by 2^-20 S: the division, a tanh of
  2 units in the last place, three products and the difference to the maximum are 8 roundings of 2^-24, of at most 2 S.  Sums of n weights
  and of weighted values, and the exponential, are off by (n + 64) 2^-24 of themselves."""
  n = 130
  p = problem(1, Hq, H, Dk, Dv, 16, [n], F32)
  p["q"] = p["q"] * factor
  out, _, lse, _ = formula(**p, cap=cap)
  A = formula(**(p | dict(vc=p["vc"].abs())), cap=cap)[0]
  t = torch.arange(n)
  k = p["kc"][p["table"][0].long()[t // 16], :, t % 16].double().abs().repeat_interleave(Hq // H, 1)  # (n, Hq, D)
  S = (k * p["q"][0, :, 0].double().abs()).sum(-1).amax(0)[:, None] / math.sqrt(Dv)  # (Hq, 1)
  e = ((Dk + 8) * 2.0**-23 + 2.0**-20) * S
  bound = 2.0**-24 * out[0].abs() + (2 * e[..., None] + (n + 64) * 2.0**-24) * A[0]
  got, got_lse = ops.paged_attn(*(p[x].to(DEV) for x in ("q", "kc", "vc", "table")), torch.tensor([n], device=DEV), 1 / math.sqrt(Dv), -1, cap)
  assert ((got[0].cpu().double() - out[0]).abs() <= bound).all()
  assert ((got_lse[0].cpu().double() - lse[0]).abs() <= e + (n + 64) * 2.0**-24 + 2.0**-21 * (1 + lse[0].abs())).all()


@pytest.mark.parametrize("dtype,cache", [(BF16, None), (F16, None), (F32, None), (BF16, FP8)])
def test_peaked_and_growing_logits(dtype, cache):
  """Logits of several hundred, and a maximum that moves with every stretch of keys: the running maximum is taken along."""
  p = problem(2, 8, 2, 64, 64, 16, [900, 333], dtype, cache)
  p["q"] = p["q"] * 20
  check(**p)
  if cache is None:
    p = problem(1, 4, 1, 64, 64, 16, [1024], dtype)
    p["q"] = torch.ones_like(p["q"])
    for t in range(1024):
      p["kc"][p["table"][0, t // 16], 0, t % 16] = (t if t < 700 else 700 - t) / 256.0
    check(**p)


def test_entries_that_name_no_page_leave_their_positions_out():
  p = problem(3, 8, 2, 128, 128, 8, [100, 64, 20], BF16, garbage=False)
  p["table"][0, 3] = -1
  p["table"][0, 7] = 2**30
  p["table"][1] = -1
  got = check(**p)
  assert (got[1] == 0).all()


def test_lengths_beyond_the_table_and_below_zero():
  p = problem(3, 8, 2, 128, 128, 8, [40, 40, 40], BF16, garbage=False)
  p["lengths"] = [2**31 - 1, -5, 41]
  check(**p)


@pytest.mark.parametrize("dtype,cache", [(BF16, None), (F16, FP8), (F32, None)])
def test_a_nan_or_infinity_in_one_row_stays_there(dtype, cache):
  """A NaN among the keys of one sequence makes that sequence's heads NaN, as in the formula, and no other's."""
  p = problem(3, 8, 2, 128, 128, 16, [50, 50, 50], dtype, cache, garbage=False)
  clean = check(**p)
  where = p["table"][1, 1]
  if cache is None:
    p["kc"][where, 0, 3, 5] = float("nan")
  else:
    p["ks"][where, 0, 3] = float("nan")
  n = torch.tensor(p["lengths"], device=DEV)
  dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
  got = ops.paged_attention(dev(p["q"]), dev(p["kc"]), dev(p["vc"]), dev(p["table"]), n, k_scale=dev(p["ks"]), v_scale=dev(p["vs"]))
  assert torch.isnan(got[1, :4]).all() and torch.equal(got[1, 4:], clean[1, 4:]) and torch.equal(got[[0, 2]], clean[[0, 2]])


def test_scales_of_very_different_size_in_8_bits():
  """Scales of the values from 1e-6 to 1e3 within one sequence: float16 weights hold no such range, the result does."""
  for dtype in (F16, BF16):
    p = problem(2, 8, 2, 128, 128, 16, [300, 1000], dtype, FP8, garbage=False)
    p["vs"] = 10.0 ** (torch.rand(p["vs"].shape, generator=torch.Generator().manual_seed(5)) * 6 - 6)
    p["ks"] = p["ks"] * 0.05
    check(**p)
    p["vs"] = torch.full_like(p["vs"], 1e-5)
    p["sm_scale"] = 0.02
    check(**p)


@pytest.mark.parametrize("dtype,cache", [(F16, None), (F16, FP8), (BF16, None), (F32, None)])
def test_one_key_far_above_many(dtype, cache):
  """60000 keys whose weights are 1.45 times float16's smallest step beside one of weight 1: each counts little, together 0.5 %."""
  n, D = 60000, 64
  p = problem(1, 4, 1, D, D, 64, [n], dtype, cache, garbage=False)
  q = torch.zeros((1, 4, 1, D))
  q[..., 0] = 1.0
  p["q"] = q.to(dtype)
  gap = 16.25
  for c, s in ((p["kc"], p["ks"]), (p["vc"], p["vs"])):
    if s is not None:
      s.fill_(1.0)
  for name, value in (("kc", 0.0), ("vc", 1.0)):
    c = p[name]
    (c.view(torch.uint8) if cache else c).copy_(torch.full(c.shape, value).to(c.dtype).view(torch.uint8) if cache else torch.full(c.shape, value))
  row = torch.zeros(D)
  row[0] = gap if cache is None else 16.0
  where = (p["table"][0, 400], 0, 17)
  (p["kc"].view(torch.uint8) if cache else p["kc"])[where] = row.to(p["kc"].dtype).view(torch.uint8) if cache else row.to(dtype)
  (p["vc"].view(torch.uint8) if cache else p["vc"])[where] = 0
  if cache:
    p["ks"][where] = gap / 16.0
  check(**p, sm_scale=1.0)


def test_pages_before_the_window_may_be_gone():
  p = problem(3, 8, 2, 128, 128, 16, [700, 130, 33], BF16)
  for b, n in enumerate(p["lengths"]):
    p["table"][b, : max(0, n - 1 - 100) // 16] = -1
  check(**p, window=100)


def test_thousands_of_sequences():
  check(**problem(4100, 1, 1, 64, 64, 8, [b % 9 for b in range(4100)], BF16, garbage=False, width=70))


def test_many_sequences_and_one_answer_for_the_same_call():
  p = problem(300, 8, 2, 64, 64, 16, [(37 * b) % 211 for b in range(300)], BF16)
  a = check(**p)
  assert torch.equal(a, check(**p))


def test_q_strides_and_other_streams():
  p = problem(3, 8, 2, 128, 128, 16, [50, 500, 3], BF16)
  want = check(**p)
  q = p["q"]
  big = torch.zeros((3, 9, 1, 136), dtype=BF16, device=DEV)
  big[:, 1:, :, :128] = q.to(DEV)
  n = torch.tensor(p["lengths"], device=DEV)
  kc, vc, tab = p["kc"].to(DEV), p["vc"].to(DEV), p["table"].to(DEV)
  assert torch.equal(ops.paged_attention(big[:, 1:, :, :128], kc, vc, tab, n), want)
  assert torch.equal(ops.paged_attention(q.to(DEV).contiguous(), kc, vc, tab, n), want)
  odd = torch.empty(3 * 8 * 128 + 1, dtype=BF16, device=DEV)[1:].view(3, 8, 1, 128).copy_(q)
  assert torch.equal(ops.paged_attention(odd, kc, vc, tab, n), want)
  torch.cuda.synchronize()
  side = torch.cuda.Stream()
  with torch.cuda.stream(side):
    got = ops.paged_attention(q.to(DEV), kc, vc, tab, n)
  side.synchronize()
  assert torch.equal(got, want)


def test_in_a_graph():
  """Captured once and replayed with lengths, pages and queries that change in between; eager work runs in between, too."""
  p = problem(4, 8, 2, 128, 128, 16, [900, 7, 64, 300], BF16, garbage=False, width=80)
  q, kc, vc, tab = (p[n].to(DEV) for n in ("q", "kc", "vc", "table"))
  n = torch.tensor(p["lengths"], dtype=torch.int32, device=DEV)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    ops.paged_attention(q, kc, vc, tab, n)
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    out = ops.paged_attention(q, kc, vc, tab, n)
  for i in range(4):
    n.copy_(torch.tensor([1200 - 300 * i, i, 64 + i, 1 + 400 * i], dtype=torch.int32))
    q.mul_(-1.0)
    tab.copy_(tab.roll(1, 0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.paged_attention(q, kc, vc, tab, n)), i


def test_a_cache_beyond_32_bit_offsets():
  """A sequence whose pages lie at both ends of a 10 GB cache."""
  H, page, D = 8, 64, 128
  pages = 10 * 2**30 // (H * page * D * 2)
  kc = torch.zeros((pages, H, page, D), dtype=BF16, device=DEV)
  n, small = 200, 4
  sk, sv = randn((small, H, page, D), 1, BF16), randn((small, H, page, D), 2, BF16)
  at = [pages - 1, 0, pages // 2 + 1, pages - 7]
  vc = torch.zeros_like(kc)
  for i, pg in enumerate(at):
    kc[pg], vc[pg] = sk[i].to(DEV), sv[i].to(DEV)
  q = randn((1, 32, 1, D), 3, BF16)
  want, bound, _, _ = formula(q, sk, sv, torch.arange(small, dtype=torch.int32)[None], [n])
  got = ops.paged_attention(q.to(DEV), kc, vc, torch.tensor([at], dtype=torch.int32, device=DEV), torch.tensor([n], device=DEV))
  assert ((got.double().cpu() - want).abs() <= bound).all()


def test_refusals():
  kc = torch.zeros((4, 2, 8, 64), dtype=BF16, device=DEV)
  f8, sc = torch.zeros((4, 2, 8, 64), dtype=torch.uint8, device=DEV).view(FP8), torch.zeros((4, 2, 8), device=DEV)
  q = torch.zeros((1, 4, 1, 64), dtype=BF16, device=DEV)
  table, n = torch.zeros((1, 2), dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
  A = ops.paged_attention
  for err, call in (
    (ValueError, lambda: A(q[:, :3], kc, kc, table, n)),
    (ValueError, lambda: A(q.expand(1, 4, 2, 64), kc, kc, table, n)),
    (ValueError, lambda: A(q[..., :32], kc, kc, table, n)),
    (ValueError, lambda: A(q, kc, kc, table, n, soft_cap=0.0)),
    (ValueError, lambda: A(q, kc, kc, table, n, -0.5)),
    (ValueError, lambda: A(q, kc, kc, table, n, window_left=-1)),
    (ValueError, lambda: A(q, kc, kc, table.expand(2, 2), n)),
    (ValueError, lambda: A(q, f8, f8, table, n)),
    (NotImplementedError, lambda: A(q.half(), kc, kc, table, n)),
    (NotImplementedError, lambda: A(q.float(), f8, f8, table, n, k_scale=sc, v_scale=sc)),
    (NotImplementedError, lambda: A(q[..., :32], kc[..., :32], kc[..., :32], table, n)),
    (RuntimeError, lambda: A(q.cpu(), kc, kc, table, n)),
    (RuntimeError, lambda: A(q.clone().requires_grad_(), kc, kc, table, n).sum().backward()),
  ):  # fmt: skip
    with pytest.raises(err):
      call()


def test_64_bit_integers_beyond_32_bits():
  """Lengths beyond the table are the table's, pages that an int32 does not hold are none."""
  p = problem(4, 8, 2, 128, 128, 8, [40, 40, 40, 40], BF16, garbage=False)
  p["table"] = p["table"].long()
  p["table"][0, 2] += 2**32
  p["table"][3] -= 2**32
  p["lengths"] = [2**32 + 1, -(2**32) + 7, 2**63 - 1, 40]
  out, bound, _, _ = formula(**p)
  got = ops.paged_attention(*(p[x].to(DEV) for x in ("q", "kc", "vc", "table")), torch.tensor(p["lengths"], device=DEV))
  assert ((got.cpu().double() - out).abs() <= bound).all() and (got[[1, 3]] == 0).all() and (got[[0, 2]] != 0).any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (128, 128), (192, 128)])
@pytest.mark.parametrize("n", [50, 3000])
@pytest.mark.parametrize("weights", ["equal", "any", "small"])
def test_an_infinite_value_makes_its_column_infinite(weights, n, Dk, Dv, dtype):
  """A positive weight times an infinity is one, also where the weight is 1 (two equal numbers split into a rounded one and no rest), or
  2^-40 of the largest; infinities of both signs add up to NaN.  Nothing else changes."""
  p = problem(1, 8, 2, Dk, Dv, 16, [n], dtype, garbage=False)
  at = lambda t: (p["table"][0, t // 16], 0, t % 16)  # noqa: E731
  if weights == "equal":
    p["q"] = torch.zeros_like(p["q"])
  if weights == "small":
    p["q"] = torch.zeros_like(p["q"])
    p["q"][..., 0] = 1.0
    p["kc"][..., 0] = 0.0
    for t in (17, 33):
      p["kc"][at(t)][0] = -28.0
  args = lambda: (*(p[x].to(DEV) for x in ("q", "kc", "vc", "table")), torch.tensor([n], device=DEV), 1.0 if weights == "small" else None)  # noqa: E731
  clean = ops.paged_attention(*args())
  inf = math.inf
  want = clean.clone()
  for t, col, x in ((17, 3, inf), (33, 7, -inf), (17, 9, inf), (33, 9, -inf), (17, Dv - 1, inf), (33, Dv - 1, inf)):
    p["vc"][at(t)][col] = x
    want[:, :4, :, col] = x if col != 9 else float("nan")
  got = ops.paged_attention(*args())
  assert torch.isfinite(clean).all()
  assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(0.5, 1e4, -1e4), want.nan_to_num(0.5, 1e4, -1e4))
