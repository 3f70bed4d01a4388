"""Sampling against the definition in 64 bits.

The definition ranks tokens by falling logit (the lower index first among equals), keeps the first top_k, of those the fewest
with top_p of their weight, of those the ones with min_p of the largest weight, and draws by cumulative weight in the order of
the indices.  A weight w = 2^x in fp32 is off by a relative 2^-20 at most (x = (l - m) c is rounded twice, |x| < 36, each by 2^-24 of
itself: 2 * 36 * 2^-24 * ln 2 < 2^-18; the exponential by 2^-22), and by 2^-36 from its grid.  Tests draw at the middle of a
token's share and cut at the middle between two cumulative weights; they assert on the definition's side that each such
middle is further than those errors from its ends, so the token has to be the same.  The log-probability is then off by
2^-17 + 2^-35 V / w at most."""

import math

import pytest
import torch

from tests.util import randn
from torchprime_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
REL = 2.0**-17


def kept_weights(row, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
  """(V,) float64: the weights of the tokens that are drawn from, 0 for the others; asserts that no cut is close."""
  l = row.double()
  l = torch.where(l == l, l, torch.full_like(l, -math.inf))
  m = l.max()
  w = torch.exp((l - m) / temperature)
  w[l == m] = 1.0
  down = torch.sort(l, descending=True, stable=True).indices
  if top_k > 0:
    down = down[:top_k]
  upto = w[down].cumsum(0)
  if top_p < 1:
    goal = top_p * upto[-1]
    n = int((upto - w[down] < goal).sum().clamp(min=1))
    assert n == 1 or (goal - (upto[n - 1] - w[down[n - 1]])) > REL * upto[-1]
    assert upto[n - 1] - goal > REL * upto[-1]
    down = down[:n]
  if min_p > 0:
    assert (((w[down] / min_p - 1).abs() > REL) | (w[down] == 1)).all()  # (the largest is exactly 1)
    down = down[w[down] >= min_p]
  out = torch.zeros_like(w)
  out[down] = w[down]
  return out


def check_draws(row, draws, dtype=F32, **settings):
  """Draws at the middle of the shares of some tokens of one row of logits."""
  row = row.to(dtype)
  w = kept_weights(row, **settings)
  share = w / w.sum()
  upto = share.cumsum(0)
  g = torch.Generator().manual_seed(len(row))
  some = torch.nonzero(share > 4 * REL)[:, 0]
  assert len(some)
  some = some[torch.randperm(len(some), generator=g)[:draws]]
  some = torch.cat([some, share.argmax()[None]])
  u = (upto[some] - share[some] / 2).to(F32)
  B = len(some)
  tokens, logprobs = ops.sample(row.to(DEV).expand(B, -1).contiguous(), u.to(DEV), **settings)
  assert tokens.dtype == torch.int64 and logprobs.dtype == F32
  assert torch.equal(tokens.cpu(), some)
  off = REL + 2.0**-35 * len(row) / w[some] + 2.0**-23 * share[some].log().abs()
  assert ((logprobs.cpu().double() - share[some].log()).abs() <= off).all()


def between(row, n, top_k=0, temperature=1.0):
  """A top_p that keeps n tokens with room on both sides."""
  l = row.double().sort(descending=True).values
  w = torch.exp((l - l[0]) / temperature)
  w = w[:top_k] if top_k else w
  upto = w.cumsum(0) / w.sum()
  return float((upto[n - 2] + upto[n - 1]) / 2) if n > 1 else float(upto[0] / 2)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [1, 2, 7, 64, 255, 1000, 32000, 50257, 128256, 2**18])
def test_all_tokens(V, dtype):
  check_draws(randn((V,), V, F32, 2.0), 20, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V,top_k", [(7, 3), (255, 255), (1000, 999), (50257, 1), (50257, 40), (128256, 1000), (128256, 100000)])
def test_top_k(V, top_k, dtype):
  check_draws(randn((V,), V + top_k, F32, 2.0), 30, dtype, top_k=top_k)


@pytest.mark.parametrize("V,n,std,temperature", [
  (100, 1, 2.0, 1.0), (100, 7, 2.0, 0.7), (50257, 40, 3.0, 1.0), (50257, 2000, 2.0, 1.3), (128256, 30, 4.0, 0.6), (128256, 300, 1.0, 1.0),
  (128256, 10000, 1.0, 1.0),
])  # fmt: skip
def test_top_p(V, n, std, temperature):
  row = randn((V,), V + n, F32, std)
  check_draws(row, 30, temperature=temperature, top_p=between(row, n, 0, temperature))


def test_filters_one_after_the_other():
  row = randn((50257,), 3, F32, 3.0)
  check_draws(row, 30, temperature=0.9, top_k=100, top_p=between(row, 31, 100, 0.9))
  check_draws(row, 30, temperature=0.9, top_k=20, top_p=between(row, 20, 20, 0.9))
  check_draws(row, 30, temperature=0.9, min_p=0.05)
  check_draws(row, 30, temperature=1.1, top_k=500, top_p=between(row, 200, 500, 1.1), min_p=0.031)
  check_draws(row, 5, min_p=1.0)
  check_draws(row, 5, top_p=0.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_equal_logits_go_by_index(dtype):
  """Cuts through equals: the lower indices stay."""
  row = torch.zeros(5000)
  check_draws(row, 20, dtype)
  check_draws(row, 20, dtype, top_k=37)
  check_draws(row, 20, dtype, top_p=(137 - 0.5) / 5000)
  row[torch.randperm(5000, generator=torch.Generator().manual_seed(1))[:900]] = 1.0
  row[7] = 2.0
  check_draws(row, 20, dtype, top_k=451)
  check_draws(row, 20, dtype, top_k=1200)
  check_draws(row, 20, dtype, top_k=1200, top_p=0.31371)
  signs = torch.where(torch.arange(300) % 2 == 0, 0.0, -0.0)  # one value, two encodings
  check_draws(signs, 10, dtype, top_k=11)


def test_ends_of_the_draw():
  """u = 0 takes the first kept token, u just below 1 (and anything from 1 up) the last; a NaN is taken for 0."""
  row = randn((1000,), 4)
  kept = torch.nonzero(kept_weights(row, top_k=50))[:, 0]
  u = torch.tensor([0.0, 1 - 2.0**-24, 1.0, 7.0, -1.0, float("nan")])
  tokens, _ = ops.sample(row.to(DEV).expand(6, -1).contiguous(), u.to(DEV), top_k=50)
  assert tokens.tolist() == [int(kept[i]) for i in (0, -1, -1, -1, 0, 0)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_greedy(dtype):
  x = randn((5, 50257), 8).to(dtype)
  x[1, 77] = x[1, 50000] = 50.0
  x[2] = 0.0
  x[3, 50256] = 60.0
  x[4, 0] = 60.0
  tokens, logprobs = ops.sample(x.to(DEV), torch.rand(5, device=DEV), 0.0)
  assert tokens.tolist() == [int(x[0].float().argmax()), 77, 0, 50256, 0] and (logprobs == 0).all()
  odd = torch.tensor([0.0, -1.0, float("nan"), -0.0, -math.inf], device=DEV)
  assert torch.equal(ops.sample(x.to(DEV), torch.rand(5, device=DEV), odd)[0], tokens)


def test_masked_and_special_logits():
  inf, nan = math.inf, math.nan
  x = torch.full((8, 300), -inf)
  x[0, 123] = 1.0                     # one token left
  x[1, 5], x[1, 9] = 2.0, 2.0         # two equals
  x[2] = nan                          # nothing
  x[4] = torch.finfo(F32).min         # the lowest value everywhere: all equal
  x[5] = 0.0
  x[5, ::2] = nan                     # NaN counts as -inf
  x[6, 17], x[6, 40] = inf, 3.0       # an infinity takes all
  x[7, :10] = torch.finfo(F32).max
  u = torch.tensor([0.5, 0.75, 0.5, 0.5, (150 + 0.5) / 300, (20 + 0.5) / 150, 0.999, 0.55])
  want = [123, 9, -1, -1, 150, 41, 17, 5]
  for settings in ({}, dict(top_k=299), dict(top_p=0.9999999), dict(min_p=0.5), dict(temperature=1e-30), dict(temperature=1e30), dict(temperature=inf)):
    tokens, logprobs = ops.sample(x.to(DEV), u.to(DEV), **settings)
    if settings.get("temperature", 0) >= 1e30:
      want = want[:7] + [int(tokens[7])]  # the largest float32 and -inf: any of the ten
    want[4] = int(float(u[4]) * settings.get("top_k", 300))
    assert tokens.tolist() == want, settings
    assert (logprobs[[2, 3]] == -inf).all() and logprobs[0] == 0 and abs(logprobs[1].item() + math.log(2)) < 1e-6
  # a top-k that reaches into what is masked
  tokens, _ = ops.sample(x[1:2].expand(2, -1).contiguous().to(DEV), torch.tensor([0.2, 0.9], device=DEV), top_k=100)
  assert tokens.tolist() == [5, 9]


def test_settings_of_each_row_and_strides():
  B, V = 37, 4001
  x = randn((B, V + 3), 9, F32, 3.0)[:, 1 : V + 1]
  g = torch.Generator().manual_seed(3)
  pick = lambda xs: torch.tensor([xs[int(torch.randint(len(xs), (1,), generator=g))] for _ in range(B)])  # noqa: E731
  t, k, p, mp = pick([0.0, 0.5, 1.0]), pick([0, 5, 50]), pick([1.0, 0.9]), pick([0.0, 0.01])
  u = torch.empty(B)
  want = torch.empty(B, dtype=torch.int64)
  for b in range(B):
    if t[b] == 0:
      u[b], want[b] = 0.3, x[b].argmax()
      continue
    if p[b] < 1:
      p[b] = between(x[b], 4, int(k[b]), float(t[b]))
    w = kept_weights(x[b], float(t[b]), int(k[b]), float(p[b]), float(mp[b]))
    share = w / w.sum()
    want[b] = torch.multinomial(share, 1, generator=g)[0]
    u[b] = share.cumsum(0)[want[b]] - share[want[b]] / 2
  dx = torch.empty((B, V + 3), device=DEV)[:, 1 : V + 1].copy_(x)
  rows = [y.to(DEV) for y in (t, k, p, mp)]
  for logits in (dx, dx.contiguous(), dx.t().contiguous().t()):
    tokens, logprobs = ops.sample(logits, u.to(DEV), *rows)
    assert torch.equal(tokens.cpu(), want)
    again, lp = ops.sample(logits, u.to(DEV).double(), rows[0].double(), rows[1].int(), rows[2], rows[3])
    assert torch.equal(again, tokens) and torch.equal(lp, logprobs)


def test_rows_of_many_and_frequencies():
  """4000 rows of one distribution with evenly spread random numbers: every token comes as often as its weight says."""
  row = torch.tensor([0.0, 1.0, 2.0, 0.5, -1.0, 1.5])
  B = 4000
  u = (torch.arange(B) + 0.5) / B
  tokens, _ = ops.sample(row.to(DEV).expand(B, -1).contiguous(), u.to(DEV))
  seen = torch.bincount(tokens.cpu(), minlength=6).double() / B
  assert ((seen - torch.softmax(row.double(), 0)).abs() <= 1.0 / B + 1e-6).all()
  empty, lp = ops.sample(row[None, :].expand(0, 6).to(DEV), u[:0].to(DEV))
  assert empty.shape == lp.shape == (0,)


@pytest.mark.parametrize("V", [50257, 128256])
def test_the_same_in_any_batch_and_graph(V):
  """A row's token is the same alone and in a batch, in 64-bit reach of every split; and in replays of a graph."""
  x = randn((70, V), 11, F32, 2.5).to(DEV)
  u = torch.rand(70, generator=torch.Generator().manual_seed(1)).to(DEV)
  for settings in (dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.8, temperature=1.2)):
    tokens, logprobs = ops.sample(x, u, **settings)
    for b in (0, 1, 33, 69):
      one, lp = ops.sample(x[b : b + 1], u[b : b + 1], **settings)
      assert torch.equal(one, tokens[b : b + 1]) and torch.equal(lp, logprobs[b : b + 1])
    few, _ = ops.sample(x[5:17], u[5:17], **settings)
    assert torch.equal(few, tokens[5:17])
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  logits, draw = x[:3].clone(), u[:3].clone()
  with torch.cuda.stream(side):
    ops.sample(logits, draw, 0.8, 50, 0.95)
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    got, got_lp = ops.sample(logits, draw, 0.8, 50, 0.95)
  for i in range(4):
    logits.copy_(x[10 * i : 10 * i + 3])
    draw.copy_(u[10 * i : 10 * i + 3])
    graph.replay()
    torch.cuda.synchronize()
    want, want_lp = ops.sample(logits, draw, 0.8, 50, 0.95)
    assert torch.equal(got, want) and torch.equal(got_lp, want_lp)


def test_refusals():
  x, u = torch.zeros((2, 5), device=DEV), torch.zeros(2, device=DEV)
  S = ops.sample
  for err, call in (
    (ValueError, lambda: S(x[0], u)),
    (ValueError, lambda: S(x, u[:1])),
    (ValueError, lambda: S(x[:, :0], u)),
    (ValueError, lambda: S(x, u, -1.0)),
    (ValueError, lambda: S(x, u, top_p=1.5)),
    (ValueError, lambda: S(x, u, top_p=float("nan"))),
    (ValueError, lambda: S(x, u, min_p=-0.1)),
    (ValueError, lambda: S(x, u, temperature=u[:1])),
    (ValueError, lambda: S(x, u, top_k=torch.ones((2, 1), dtype=torch.int32, device=DEV))),
    (TypeError, lambda: S(x, u, top_k=u)),
    (TypeError, lambda: S(x.double(), u)),
    (TypeError, lambda: S(x, u.long())),
    (NotImplementedError, lambda: S(torch.zeros((1, 2**18 + 1), device=DEV), u[:1])),
    (RuntimeError, lambda: S(x, u.cpu())),
  ):  # fmt: skip
    with pytest.raises(err):
      call()


def test_top_k_of_64_bits():
  """A top-k that an int32 does not hold keeps all, as the number does; so do those far below zero."""
  row, ks = randn((3000,), 21, F32, 1.5), [2**32 + 1, 2**32, 2**63 - 1, -(2**32) + 1, -(2**63), 3000]
  w = kept_weights(row)
  at = torch.argsort(w)[1500:].tolist()[:: 1500 // len(ks)][: len(ks)]
  share = w / w.sum()
  u = (share.cumsum(0) - share / 2)[at]
  assert (share[at] > 4 * REL).all()
  x = row.to(DEV).expand(len(ks), -1).contiguous()
  tokens, _ = ops.sample(x, u.float().to(DEV), top_k=torch.tensor(ks, device=DEV))
  assert tokens.tolist() == at
  for k, want in zip(ks, at):
    assert ops.sample(x[:1], u[at.index(want)][None].float().to(DEV), top_k=k)[0].tolist() == [want]


def special_rows(V, dtype):
  """Rows in which most tokens are masked, or the logits' range is all that the type has."""
  inf, nan, top, low = math.inf, math.nan, torch.finfo(dtype).max, torch.finfo(dtype).min
  g = torch.Generator().manual_seed(V)
  any_of = lambda n: torch.randperm(V, generator=g)[:n]  # noqa: E731
  filled = lambda *parts: _filled(V, -inf, parts)  # noqa: E731
  yield "one token", filled((any_of(1), 3.0))
  yield "thirty tokens", filled((any_of(30), 2 * randn((30,), 1)))
  yield "two thousand side by side", filled((torch.arange(V // 3, V // 3 + 2000), 2 * randn((2000,), 2)))
  yield "the last twenty", filled((torch.arange(V - 20, V), randn((20,), 3)))
  yield "between NaN", _filled(V, nan, [(any_of(V // 2), -inf), (any_of(40), randn((40,), 4))])
  yield "three infinities", _filled(V, 1.0, [(any_of(V // 2), randn((V // 2,), 5)), (any_of(3), inf)])
  yield "many infinities", _filled(V, -1.0, [(any_of(1500), inf)])
  yield "infinities and nothing else", filled((any_of(7), inf))
  yield "both ends of the range", filled((any_of(20), low), (any_of(5), top))
  yield "the lowest value", filled((any_of(400), low))
  yield "the largest value", _filled(V, low, [(any_of(1500), top)])


def _filled(V, value, parts):
  row = torch.full((V,), value)
  for at, x in parts:
    row[at] = x
  return row


SPECIAL_SETTINGS = [dict(), dict(top_k=50), dict(top_k=1000), dict(top_p=0.3713), dict(min_p=0.51), dict(top_k=300, top_p=0.3713),
                    dict(temperature=0.5, top_p=0.6171, min_p=0.051), dict(top_k=1200, top_p=0.6171)]  # fmt: skip


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [5000, 128256])
@pytest.mark.parametrize("settings", SPECIAL_SETTINGS, ids=str)
def test_masked_and_special_logits_of_large_vocabularies(settings, V, dtype):
  for name, row in special_rows(V, dtype):
    print(name, flush=True)
    check_draws(row, 8, dtype, **settings)


@pytest.mark.parametrize("V", [5000, 128256])
@pytest.mark.parametrize("settings", SPECIAL_SETTINGS + [dict(temperature=0.0)], ids=str)
def test_rows_of_nothing_in_large_vocabularies(settings, V):
  x = torch.full((3, V), -math.inf)
  x[1] = math.nan
  x[2, V - 1] = 1.0
  tokens, logprobs = ops.sample(x.to(DEV), torch.full((3,), 0.5, device=DEV), **settings)
  assert tokens.tolist() == [-1, -1, V - 1] and logprobs.tolist() == [-math.inf, -math.inf, 0.0]


@pytest.mark.parametrize("V", [1023, 1024, 1025, 1040])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=200), dict(top_k=1000), dict(top_p=0.6171), dict(min_p=0.051), dict(temperature=0.0)], ids=str)
def test_around_the_rows_that_one_launch_takes(settings, V):
  row = randn((V,), V, F32, 1.5)
  if settings.get("temperature", 1.0) > 0:
    return check_draws(row, 20, **settings)
  x = row.to(DEV).expand(300, -1).contiguous()
  assert (ops.sample(x, torch.rand(300, device=DEV), **settings)[0] == int(row.argmax())).all()
