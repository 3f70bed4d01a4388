"""Answering with a trained model: a paged key-value cache and ``generate`` for :class:`~torchprime_amd.LlamaForCausalLM`.

The reference trains only (its models have no cache and no sampling); this is the path a user takes from a checkpoint to
text: the prompt through the causal attention of training, its keys and values into pages, then token by token
``kv_cache_write`` -> ``paged_attention`` -> ``sample`` (:mod:`torchprime_amd.ops`).
"""

from __future__ import annotations

import torch

from . import ops
from .attention import AttentionModule
from .blocks import LlamaAttention, LlamaDecoderLayer, LlamaForCausalLM, LlamaModel
from .linear import _GLOBAL_HOOKS, embed, project
from .norm import LlamaRMSNorm, add_rms_norm
from .rotary import apply_rotary_pos_emb

__all__ = ["PagedKVCache", "generate"]


class PagedKVCache:
  """Keys and values of up to ``max_batch`` sequences in pages of ``page_size`` tokens, for ``num_layers`` layers.

  A page belongs to one sequence and holds the same positions in every layer.  Which pages are whose is decided on the host
  (``extend`` takes pages, ``release`` gives them back); the kernels read the table and the lengths on the device.

  ``quantized``: rows are kept in float8 (e4m3) with a float32 scale each, 132 bytes instead of 256 for a head of 128; for
  16-bit models.  ``k``, ``v``: (layers, pages, heads, page_size, dim)."""

  def __init__(
    self, num_layers: int, num_kv_heads: int, head_dim: int, *, num_pages: int, max_batch: int, page_size: int = 64,
    v_head_dim: int | None = None, max_pages_per_sequence: int | None = None, dtype: torch.dtype = torch.bfloat16,
    quantized: bool = False, device: str | torch.device = "cuda",
  ):  # fmt: skip
    if page_size < 8 or page_size & (page_size - 1):
      raise ValueError(f"page_size must be a power of two from 8 up, got {page_size}")
    if min(num_layers, num_kv_heads, head_dim, num_pages, max_batch) < 1:
      raise ValueError("sizes must be positive")
    if quantized and dtype == torch.float32:
      raise ValueError("a quantized cache goes with 16-bit models")
    self.page_size, self.dtype = page_size, dtype
    store = torch.float8_e4m3fn if quantized else dtype
    rows = (num_layers, num_pages, num_kv_heads, page_size)
    # (slots that nothing was stored in are never read; they need no clearing)
    self.k = torch.empty((*rows, head_dim), dtype=store, device=device)
    self.v = torch.empty((*rows, v_head_dim or head_dim), dtype=store, device=device)
    self.k_scale = torch.empty(rows, dtype=torch.float32, device=device) if quantized else None
    self.v_scale = torch.empty(rows, dtype=torch.float32, device=device) if quantized else None
    self.block_table = torch.full((max_batch, max_pages_per_sequence or num_pages), -1, dtype=torch.int32, device=device)
    self.positions = torch.zeros((max_batch,), dtype=torch.int32, device=device)  # where the newest tokens go
    self.lengths = torch.zeros((max_batch,), dtype=torch.int32, device=device)  # with the newest tokens
    self.host_lengths = [0] * max_batch
    self._pages: list[list[int]] = [[] for _ in range(max_batch)]
    self._free = list(range(num_pages - 1, -1, -1))

  @property
  def free_pages(self) -> int:
    return len(self._free)

  def extend(self, counts: list[int]) -> None:
    """Makes room for ``counts[b]`` new tokens of each sequence: ``positions`` are their first places, ``lengths`` count
    them.  Raises before anything is changed where the pages do not suffice."""
    if len(counts) != len(self._pages) or min(counts) < 0:
      raise ValueError(f"expected {len(self._pages)} counts that are not negative, got {counts}")
    need = [-(-(n + c) // self.page_size) - len(p) for n, c, p in zip(self.host_lengths, counts, self._pages)]
    need = [max(0, n) for n in need]
    if any(len(p) + n > self.block_table.shape[1] for p, n in zip(self._pages, need)):
      raise RuntimeError(f"a sequence needs more than {self.block_table.shape[1]} pages")
    if sum(need) > len(self._free):
      raise RuntimeError(f"the cache is full: {sum(need)} pages are needed, {len(self._free)} are free")
    at = []
    for b, n in enumerate(need):
      for _ in range(n):
        page = self._free.pop()
        at.append((b, len(self._pages[b]), page))
        self._pages[b].append(page)
    device = self.block_table.device
    if at:
      b, i, page = torch.tensor(at, dtype=torch.int64).t().to(device)
      self.block_table[b, i] = page.to(torch.int32)
    self.positions.copy_(self.lengths)
    if len(set(counts)) == 1:
      self.lengths += counts[0]
    else:
      self.lengths += torch.tensor(counts, dtype=torch.int32).to(device)
    self.host_lengths = [n + c for n, c in zip(self.host_lengths, counts)]

  def release(self, b: int) -> None:
    """Gives back the pages of sequence ``b``, whose place may be taken by another one."""
    self._free += reversed(self._pages[b])
    self._pages[b] = []
    self.block_table[b] = -1
    self.lengths[b] = 0
    self.host_lengths[b] = 0

  def _of(self, layer: int) -> tuple[tuple, dict]:
    # (no more of the table than the longest sequence needs: its width bounds the work that is planned for)
    width = max(1, max(len(p) for p in self._pages))
    scales = {} if self.k_scale is None else {"k_scale": self.k_scale[layer], "v_scale": self.v_scale[layer]}
    return (self.k[layer], self.v[layer], self.block_table[:, :width]), scales

  def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, counts: torch.Tensor | None = None) -> None:
    """Stores the newest tokens' keys and values (max_batch, heads, tokens, dim) of a layer; of sequence b, ``counts[b]``."""
    cache, scales = self._of(layer)
    ops.kv_cache_write(k, v, *cache, self.positions, counts, **scales)

  def read(self, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Everything cached of a layer as (max_batch, heads, longest, dim) keys and values, zeros behind shorter sequences."""
    cache, scales = self._of(layer)
    return ops.kv_cache_read(*cache, self.lengths, max(self.host_lengths), dtype=self.dtype, **scales)

  def attend(self, layer: int, q: torch.Tensor, sm_scale: float | None = None, **extensions) -> torch.Tensor:
    """Attention of the newest token of each sequence, (max_batch, query heads, 1, dim), over everything cached of it."""
    cache, scales = self._of(layer)
    return ops.paged_attention(q, *cache, self.lengths, sm_scale, **scales, **extensions)


# the methods that _hidden and generate stand in for
_OWN = {
  LlamaForCausalLM: ("forward", "_logits"), LlamaModel: ("forward", "deferred"), LlamaDecoderLayer: ("forward", "forward_deferred", "_one_call"),
  LlamaAttention: ("forward",), AttentionModule: ("forward",), LlamaRMSNorm: ("forward",),
}  # fmt: skip


def _check_model(model) -> None:
  """The model runs here with a cache in its attention, so some of its modules do not see a call of their own: one that has
  to (forward hooks, another ``forward``, another class) is refused rather than passed by.  Projections, the MLP, the
  embedding and the rotary module are called."""

  def check(m, cls):
    own = isinstance(m, cls) and all(getattr(type(m), n) is getattr(cls, n) and n not in m.__dict__ for n in _OWN[cls])
    if not own or m._forward_hooks or m._forward_pre_hooks:
      raise NotImplementedError(f"generate runs {cls.__name__} with a cache of its own: a {type(m).__name__} with another forward or with forward hooks would be passed by")

  if not isinstance(model, LlamaForCausalLM):
    raise TypeError(f"generate takes a LlamaForCausalLM, got {type(model).__name__}")
  if _GLOBAL_HOOKS[0] or _GLOBAL_HOOKS[1]:
    raise NotImplementedError("generate would pass by the forward hooks of all modules (torch.nn.modules.module.register_module_forward_hook)")
  check(model, LlamaForCausalLM)
  check(model.model, LlamaModel)
  for layer in model.model.layers:
    check(layer, LlamaDecoderLayer)
    check(layer.self_attn, LlamaAttention)
    check(layer.self_attn.attention_block, AttentionModule)
    check(layer.input_layernorm, LlamaRMSNorm)
    check(layer.post_attention_layernorm, LlamaRMSNorm)
    if layer.self_attn.attention_block.plain_causal(1, None) is None:
      raise NotImplementedError("generate's attention is causal, without dropout, in the order of the tokens (no load_balance_cp)")
  check(model.model.norm, LlamaRMSNorm)


def _hidden(model, ids: torch.Tensor, positions: torch.Tensor, cache: PagedKVCache, counts: torch.Tensor | None, first: int):
  """The decoder's last hidden states (before the final norm) of new tokens (batch, S) at ``positions`` (batch, S) as (x,
  residual), with their keys and values stored.  ``first``: the position of column 0 where S > 1."""
  x, residual = embed(model.embed_tokens, ids), None
  B, S = ids.shape
  cos, sin = model.rotary_emb(x, positions.float())
  for i, layer in enumerate(model.layers):
    a = layer.self_attn
    if residual is None:
      residual, h = x, layer.input_layernorm(x)
    else:
      h, residual = add_rms_norm(x, residual, layer.input_layernorm)
    q, k, v = project(h, a.q_proj, a.k_proj, a.v_proj)
    q = q.view(B, S, a.num_heads, a.head_dim).transpose(1, 2)
    k = k.view(B, S, a.num_key_value_heads, a.head_dim).transpose(1, 2)
    v = v.view(B, S, a.num_key_value_heads, a.head_dim).transpose(1, 2)
    q, k = apply_rotary_pos_emb(q, k, cos, sin)
    cache.write(i, k, v, counts)
    if S == 1:
      out = cache.attend(i, q)
    elif first == 0:
      out = ops.attention(q, k, v, causal=True)  # (what is behind a shorter prompt comes later than all of it)
    else:
      out = ops.attention(q, *cache.read(i), causal=True, causal_offset=first)
    h = project(out.transpose(1, 2).reshape(B, S, a.hidden_size), a.o_proj)[0]
    h, residual = add_rms_norm(h, residual, layer.post_attention_layernorm)
    x = layer.mlp(h)
  return x, residual


@torch.no_grad()
def generate(
  model: LlamaForCausalLM, input_ids: torch.Tensor, max_new_tokens: int, *, prompt_lengths: list[int] | None = None,
  temperature: float | torch.Tensor = 1.0, top_k: int | torch.Tensor = 0, top_p: float | torch.Tensor = 1.0,
  min_p: float | torch.Tensor = 0.0, eos_token_id: int | None = None, generator: torch.Generator | None = None,
  page_size: int = 64, quantized_cache: bool = False, prompt_chunk: int | None = None, return_logits: bool = False,
):  # fmt: skip
  """Continues each prompt by up to ``max_new_tokens`` tokens.

  ``input_ids`` (batch, S) hold the prompts from the left, ``prompt_lengths`` of them each (None: S); what is behind is not
  read.  Settings are those of :func:`torchprime_amd.ops.sample`, numbers or one per sequence; temperature 0 is greedy.  After
  ``eos_token_id`` a sequence's tokens are -1.  ``prompt_chunk``: prompts go through in pieces of that many tokens.
  ``generator``: a generator of the model's device for the draws.  A model whose decoder layers, attention or norms have forward
  hooks or a ``forward`` of their own is refused: they would not see their calls.

  Returns the new tokens (batch, n <= max_new_tokens) and their log-probabilities in the distributions that they were drawn from;
  with ``return_logits`` also the logits (batch, n, vocabulary)."""
  _check_model(model)
  if input_ids.dim() != 2 or input_ids.shape[1] < 1 or max_new_tokens < 1:
    raise ValueError("expected input_ids (batch, tokens) with at least one token, and max_new_tokens >= 1")
  B, S = input_ids.shape
  lengths = [S] * B if prompt_lengths is None else [int(n) for n in prompt_lengths]
  if len(lengths) != B or min(lengths) < 1 or max(lengths) > S:
    raise ValueError(f"prompt_lengths must be {B} numbers from 1 to {S}, got {lengths}")
  if prompt_chunk is not None and prompt_chunk < 2:
    raise ValueError("prompt_chunk must be at least 2")
  S = max(lengths)
  inner, cfg, device = model.model, model.config, input_ids.device
  weight = inner.embed_tokens.weight
  heads, dim = cfg.num_key_value_heads, cfg.hidden_size // cfg.num_attention_heads
  pages = sum(-(-(n + max_new_tokens) // page_size) for n in lengths)
  cache = PagedKVCache(len(inner.layers), heads, dim, num_pages=pages, max_batch=B, page_size=page_size, dtype=weight.dtype,
                       quantized=quantized_cache, device=device)  # fmt: skip

  # the prompts: every piece's hidden states, of which a prompt's last one is kept
  ends = torch.tensor(lengths).to(device)
  ids = input_ids[:, :S]
  if min(lengths) < S:
    # (what is behind a prompt may be no token at all: token 0 goes through the layers in its place)
    ids = torch.where(torch.arange(S, device=device) < ends[:, None], ids, 0)
  last = None
  step = prompt_chunk or S
  for first in range(0, S, step):
    n = min(step, S - first)
    counts = [min(max(length - first, 0), n) for length in lengths]
    cache.extend(counts)
    positions = torch.arange(first, first + n, device=device)[None].expand(B, n)
    x, residual = _hidden(inner, ids[:, first : first + n], positions, cache, None if min(counts) == n else torch.tensor(counts, dtype=torch.int32).to(device), first)
    h = x + residual
    row = (ends - 1 - first).clamp(0, n - 1)
    here = h[torch.arange(B, device=device), row]
    last = here if last is None else torch.where((ends > first)[:, None], here, last)

  tokens, logprobs, all_logits = [], [], []
  done = torch.zeros((B,), dtype=torch.bool, device=device)
  hidden = inner.norm(last[:, None])
  for i in range(max_new_tokens):
    logits = project(hidden, model.lm_head)[0][:, 0].float()
    token, logprob = ops.sample(logits, torch.rand((B,), generator=generator, device=device), temperature, top_k, top_p, min_p)
    tokens.append(torch.where(done, -1, token))
    logprobs.append(torch.where(done, 0.0, logprob))
    if return_logits:
      all_logits.append(logits)
    if eos_token_id is not None:
      done = done | (token == eos_token_id)
      if i % 16 == 15 and bool(done.all()):  # (asked now and then: the answer takes a synchronisation)
        break
    if i + 1 == max_new_tokens:
      break
    cache.extend([1] * B)
    x, residual = _hidden(inner, token.clamp(min=0)[:, None], cache.positions[:, None], cache, None, 0)
    hidden = add_rms_norm(x, residual, inner.norm)[0]
  out = (torch.stack(tokens, 1), torch.stack(logprobs, 1))
  return (*out, torch.stack(all_logits, 1)) if return_logits else out
