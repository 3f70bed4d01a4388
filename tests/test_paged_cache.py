"""Which pages belong to which sequence: the host side of PagedKVCache, on the CPU."""

import random

import pytest
import torch

import torchprime_amd as tpa


def cache(**kw):
  args = dict(num_pages=12, max_batch=3, page_size=8, dtype=torch.bfloat16, device="cpu") | kw
  return tpa.PagedKVCache(2, 4, 64, **args)


def check(c):
  """Every page is free or one sequence's, the table says which, and there are enough of them."""
  pages = [p for ps in c._pages for p in ps]
  assert sorted(pages + c._free) == list(range(c.k.shape[1]))
  for b, ps in enumerate(c._pages):
    assert c.block_table[b].tolist() == ps + [-1] * (c.block_table.shape[1] - len(ps))
    assert len(ps) * c.page_size >= c.host_lengths[b] > (len(ps) - 1) * c.page_size or not ps and c.host_lengths[b] == 0
  assert c.lengths.tolist() == c.host_lengths


def test_pages_are_taken_and_given_back():
  c = cache()
  c.extend([8, 0, 1])
  assert c.positions.tolist() == [0, 0, 0] and c.free_pages == 10
  check(c)
  c.extend([1, 1, 7])
  assert c.positions.tolist() == [8, 0, 1] and c.lengths.tolist() == [9, 1, 8] and c.free_pages == 8
  check(c)
  c.release(0)
  check(c)
  c.extend([17, 0, 1])
  check(c)


def test_a_full_cache_refuses_and_stays_as_it_was():
  c = cache()
  c.extend([40, 20, 8])
  before = (c.host_lengths[:], c.lengths.tolist(), c.block_table.clone(), c.free_pages)
  with pytest.raises(RuntimeError, match="full"):
    c.extend([0, 5, 25])
  assert before[0] == c.host_lengths and before[1] == c.lengths.tolist() and torch.equal(before[2], c.block_table) and before[3] == c.free_pages
  check(c)
  c = cache(max_pages_per_sequence=2)
  with pytest.raises(RuntimeError, match="more than 2 pages"):
    c.extend([17, 0, 0])
  check(c)


def test_any_order_of_extending_and_releasing():
  rng = random.Random(1)
  c = cache(num_pages=40, max_batch=5)
  for _ in range(300):
    try:
      c.extend([rng.choice([0, 0, 1, 1, 9, 30]) for _ in range(5)])
    except RuntimeError:
      c.release(rng.randrange(5))
    check(c)


def test_refusals():
  for kw in (dict(page_size=12), dict(page_size=4), dict(num_pages=0), dict(quantized=True, dtype=torch.float32)):
    with pytest.raises(ValueError):
      cache(**kw)
  c = cache()
  for counts in ([1, 1], [1, -1, 1]):
    with pytest.raises(ValueError):
      c.extend(counts)


def test_an_8_bit_cache_has_scales():
  c = cache(quantized=True, v_head_dim=128)
  assert c.k.dtype == c.v.dtype == torch.float8_e4m3fn and c.v.shape == (2, 12, 4, 8, 128)
  assert c.k_scale.shape == c.v_scale.shape == (2, 12, 4, 8)
