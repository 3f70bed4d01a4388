"""What the cache, paged attention and sampling do without a GPU: refusals of the C entry points before any launch, CPU tensors
refused, operators traced with fake tensors and seen by function modes."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from tests.test_host import _Seen
from torchprime_amd import _lib, ops

FP8 = torch.float8_e4m3fn


def _buffer():
  buf = ctypes.create_string_buffer(1 << 16)
  p = ctypes.addressof(buf)
  return buf, p + (-p) % 16


def _cache(p, **edit):
  c = _lib.KvCache(k=p, v=p, table=p, table_stride=4, table_width=4, pages=4, page_size=16, heads=2, k_dim=64, v_dim=64, dtype=_lib.TP_BF16)
  for s in (c.k_strides, c.v_strides):
    s[:] = [2048, 1024, 64]
  for n, x in edit.items():
    if n.endswith("strides"):
      getattr(c, n)[:] = x
    else:
      setattr(c, n, x)
  return c


CACHES = [
  (dict(k=None), -1, b"null"), (dict(table=None), -1, b"null"), (dict(pages=0), -1, b"positive"), (dict(heads=0), -1, b"positive"),
  (dict(page_size=12), -2, b"power of two"), (dict(page_size=4), -2, b"power of two"), (dict(k_dim=60), -2, b"head dim"),
  (dict(v_dim=520), -2, b"head dim"), (dict(dtype=_lib.TP_F16), -2, b"does not go"), (dict(dtype=_lib.TP_FP8), -1, b"k_scale"),
  (dict(k_scale=16), -1, b"k_scale"), (dict(k_scale=20), -1, b"16-byte"), (dict(k_strides=[2048, 1024, 63]), -1, b"aligned"), (dict(v_strides=[-2048, 1024, 64]), -1, b"aligned"),
  (dict(table_width=1 << 28), -2, b"2^30"), (dict(dtype=9), -2, b"does not go"),
]  # fmt: skip


@pytest.mark.parametrize("edit,status,message", CACHES)
def test_a_cache_that_the_kernels_cannot_take(edit, status, message):
  lib = _lib.load()
  buf, p = _buffer()
  c = _cache(p, **edit)
  s3, s2 = _lib._I64x3(256, 128, 64), (ctypes.c_int64 * 2)(128, 64)
  calls = (
    lambda: lib.tp_kv_cache_write(ctypes.byref(c), p, p, p, None, 1, 2, s3, s3, _lib.TP_BF16, None),
    lambda: lib.tp_kv_cache_read(ctypes.byref(c), p, p, p, 1, 2, s3, s3, _lib.TP_BF16, None),
    lambda: lib.tp_paged_attn(ctypes.byref(c), p, p, p, None, p, 1, 2, s2, s2, 0.1, -1, 0.0, _lib.TP_BF16, None),
  )
  for call in calls:
    assert call() == status and message in lib.tp_last_error(), lib.tp_last_error()


def test_other_arguments():
  lib = _lib.load()
  buf, p = _buffer()
  c = ctypes.byref(_cache(p))
  s3, odd, s2 = _lib._I64x3(256, 128, 64), _lib._I64x3(256, 128, 63), (ctypes.c_int64 * 2)(128, 64)
  W, R, A, S = lib.tp_kv_cache_write, lib.tp_kv_cache_read, lib.tp_paged_attn, lib.tp_sample
  bf = _lib.TP_BF16
  for status, call in (
    (-1, lambda: W(c, None, p, p, None, 1, 2, s3, s3, bf, None)),
    (-1, lambda: W(c, p, p, None, None, 1, 2, s3, s3, bf, None)),
    (-1, lambda: W(c, p, p, p, None, 0, 2, s3, s3, bf, None)),
    (-1, lambda: W(c, p, p, p, None, 1, 0, s3, s3, bf, None)),
    (-1, lambda: W(c, p + 2, p, p, None, 1, 2, s3, s3, bf, None)),
    (-1, lambda: W(c, p, p, p, None, 1, 2, s3, odd, bf, None)),
    (-2, lambda: W(c, p, p, p, None, 1 << 14, 1 << 14, s3, s3, bf, None)),
    (-2, lambda: W(c, p, p, p, None, 1, 2, s3, s3, _lib.TP_FP8, None)),
    (-1, lambda: R(c, None, p, p, 1, 2, s3, s3, bf, None)),
    (-1, lambda: R(c, p, p, p, 1, 0, s3, s3, bf, None)),
    (-1, lambda: A(c, None, p, p, None, p, 1, 2, s2, s2, 0.1, -1, 0.0, bf, None)),
    (-1, lambda: A(c, p, p, p, None, p, 1, 3, s2, s2, 0.1, -1, 0.0, bf, None)),
    (-1, lambda: A(c, p, p, p, None, p, 1, 2, s2, s2, 0.0, -1, 0.0, bf, None)),
    (-1, lambda: A(c, p, p, p, None, p, 1, 2, s2, s2, 0.1, -1, -1.0, bf, None)),
    (-1, lambda: A(c, p + 2, p, p, None, p, 1, 2, s2, s2, 0.1, -1, 0.0, bf, None)),
    (-2, lambda: A(ctypes.byref(_cache(p, k_dim=32, v_dim=32)), p, p, p, None, p, 1, 2, s2, s2, 0.1, -1, 0.0, bf, None)),
    (-1, lambda: S(None, p, None, None, None, None, 1.0, 0, 1.0, 0.0, p, p, p, 1, 8, 8, 2, None)),
    (-1, lambda: S(p, p, None, None, None, None, 1.0, 0, 1.0, 0.0, p, p, p, 0, 8, 8, 2, None)),
    (-1, lambda: S(p, p, None, None, None, None, 1.0, 0, 1.0, 0.0, p, p, p, 2, 8, 7, 2, None)),
    (-1, lambda: S(p + 2, p, None, None, None, None, 1.0, 0, 1.0, 0.0, p, p, p, 2, 8, 8, 2, None)),
    (-2, lambda: S(p, p, None, None, None, None, 1.0, 0, 1.0, 0.0, p, p, p, 1, (1 << 18) + 1, 1 << 19, 2, None)),
    (-2, lambda: S(p, p, None, None, None, None, 1.0, 0, 1.0, 0.0, p, p, p, 1, 8, 8, 3, None)),
  ):  # fmt: skip
    assert call() == status, lib.tp_last_error()


def test_workspaces():
  """What fits a workgroup per segment (up to 512 keys) needs none; beyond that it is asked for, and its absence refused."""
  lib = _lib.load()
  buf, p = _buffer()
  s2 = (ctypes.c_int64 * 2)(128, 64)
  short, long = _cache(p, table_width=32), _cache(p, table_width=33)
  size = lambda c, dt=_lib.TP_BF16: lib.tp_paged_attn_workspace_bytes(ctypes.byref(c), 1, 2, dt)  # noqa: E731
  assert size(short) == 0 and 0 < size(long) < 1 << 20
  assert size(_cache(p, table_width=33, page_size=12)) == 0 and size(long, 7) == 0  # (refused anyway)
  assert lib.tp_paged_attn(ctypes.byref(long), p, p, p, None, None, 1, 2, s2, s2, 0.1, -1, 0.0, _lib.TP_BF16, None) == -1
  assert lib.tp_paged_attn(ctypes.byref(long), p, p, p, None, p + 4, 1, 2, s2, s2, 0.1, -1, 0.0, _lib.TP_BF16, None) == -1
  assert b"workspace" in lib.tp_last_error()
  huge = _cache(p, table_width=1 << 26)
  assert size(huge) < 1 << 24  # (bounded by the workgroups, not by the keys)
  assert lib.tp_paged_attn(ctypes.byref(_cache(p, table_width=1 << 26)), p, p, p, None, p, 1 << 10, 2, s2, s2, 0.1, -1, 0.0, _lib.TP_BF16, None) == -2
  assert lib.tp_sample_workspace_bytes(0, 5) == 0 and lib.tp_sample_workspace_bytes(3, (1 << 18) + 1) == 0
  assert lib.tp_sample_workspace_bytes(3, 128256) == 3 * lib.tp_sample_workspace_bytes(1, 128256) > 0
  assert lib.tp_sample(p, p, None, None, None, None, 1.0, 0, 1.0, 0.0, p, p, None, 1, 8, 8, 2, None) == -1


def _tensors(dev="cpu"):
  k = torch.zeros((2, 4, 3, 128), dtype=torch.bfloat16, device=dev)
  cache = torch.zeros((6, 4, 16, 128), dtype=torch.bfloat16, device=dev)
  table, n = torch.zeros((2, 3), dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int32, device=dev)
  return k, cache, table, n, torch.zeros((2, 50), device=dev), torch.zeros(2, device=dev)


def test_cpu_tensors_raise():
  k, cache, table, n, logits, u = _tensors()
  q = k[:, :, :1]
  for call in (lambda: ops.kv_cache_write(k, k, cache, cache, table, n), lambda: ops.kv_cache_read(cache, cache, table, n, 4),
               lambda: ops.paged_attention(q, cache, cache, table, n), lambda: ops.sample(logits, u)):  # fmt: skip
    with pytest.raises(RuntimeError, match="no CPU path"):
      call()


def test_function_modes_see_the_operators():
  k, cache, table, n, logits, u = _tensors()
  for name, call in (
    ("kv_cache_write", lambda: ops.kv_cache_write(k, k, cache, cache, table, n)), ("kv_cache_read", lambda: ops.kv_cache_read(cache, cache, table, n, 4)),
    ("paged_attn", lambda: ops.paged_attention(k[:, :, :1], cache, cache, table, n)), ("sample", lambda: ops.sample(logits, u, top_k=n)),
  ):  # fmt: skip
    with _Seen() as seen:
      call()
    assert [x for x in seen.names if "tprime" in x] == [f"tprime.{name}.default"]


def test_shapes_with_fake_tensors():
  with FakeTensorMode():
    k, cache, table, n, logits, u = _tensors("cuda")
    wide, v = torch.zeros((6, 4, 16, 192), dtype=FP8, device="cuda"), torch.zeros((6, 4, 16, 128), dtype=FP8, device="cuda")
    s = torch.zeros((6, 4, 16), device="cuda")
    assert ops.kv_cache_write_op(k, k, cache, cache, table, n) is None
    ko, vo = ops.kv_cache_read_op(wide, v, table, n, 20, torch.float16, s, s)
    assert ko.shape == (2, 4, 20, 192) and vo.shape == (2, 4, 20, 128) and ko.dtype == vo.dtype == torch.float16
    q = torch.zeros((2, 1, 8, 192), dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    out, lse = ops.paged_attn(q, wide, v, table, n, 0.1, k_scale=s, v_scale=s)
    assert out.shape == (2, 8, 1, 128) and out.dtype == q.dtype and lse.shape == (2, 8, 1) and lse.dtype == torch.float32
    tokens, logprobs = ops.sample_op(logits, u, None, None, None, None, 1.0, 0, 1.0, 0.0)
    assert tokens.shape == logprobs.shape == (2,) and tokens.dtype == torch.int64 and logprobs.dtype == torch.float32


def test_rows_that_one_launch_takes_need_next_to_no_workspace():
  """Up to 1024 logits a row never leaves its workgroup: 65535 such rows asked for 1.6 GB, of which nothing was used."""
  lib = _lib.load()
  for V in (1, 50, 1024):
    assert 0 < lib.tp_sample_workspace_bytes(65535, V) <= 64
  assert lib.tp_sample_workspace_bytes(2, 1025) == 2 * lib.tp_sample_workspace_bytes(1, 1025) > 2 * 1025
