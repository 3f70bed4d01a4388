"""Generation with a small model: logits of every step against the whole sequence run through the model at once, which has no
cache, no pages and no single-token attention.

Bounds on the relative 2-norm of the logits: the two paths compute the same in another order, so 1e-4 in fp32 (a dozen products of a
few hundred terms) and 3e-2 in bfloat16, where each of them is off by as much; 0.1 with keys and values in 8 bits (e4m3 rounds by up to
2^-4 of a value, half of that on average, and the residual stream carries most of the state)."""

import pytest
import torch

import torchprime_amd as tpa
from tests.util import randn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def small_model(dtype, heads=8, kv_heads=2, hidden=512, vocab=256, layers=2, seed=1):
  cfg = tpa.Config(vocab_size=vocab, num_hidden_layers=layers, max_position_embeddings=4096, hidden_size=hidden, intermediate_size=128,
                   num_attention_heads=heads, num_key_value_heads=kv_heads, hidden_act="silu", initializer_range=0.02, rms_norm_eps=1e-5,
                   attention_dropout=False, attention_bias=False, rope_theta=500000.0, attention_kernel="splash_attention")  # fmt: skip
  model = tpa.LlamaForCausalLM(cfg)
  with torch.no_grad():
    for i, p in enumerate(model.parameters()):
      p.copy_(1 + 0.1 * randn(p.shape, seed + i) if p.dim() == 1 else 0.06 * randn(p.shape, seed + i))
  return model.to(DEV).to(dtype).eval()


def prompts(B, S, vocab, seed):
  return torch.randint(vocab, (B, S), generator=torch.Generator().manual_seed(seed)).to(DEV)


def check(model, ids, lengths, tokens, logits, limit):
  """The logits behind each token against the model's own on the prompt and the tokens before it."""
  for b, n in enumerate(lengths):
    whole = torch.cat([ids[b, :n], tokens[b, :-1].clamp(min=0)])[None]
    with torch.no_grad():
      want = model(whole)[0][0, n - 1 :].float()
    off = ((logits[b] - want).norm() / want.norm()).item()
    assert off <= limit, (b, off)


@pytest.mark.parametrize("dtype,limit", [(torch.float32, 1e-4), (torch.bfloat16, 3e-2), (torch.float16, 3e-2)])
@pytest.mark.parametrize("lengths,chunk", [([5], None), ([1, 1], None), ([70, 3, 129, 64], None), ([150, 9, 33], 32), ([130, 64], 63)])
@pytest.mark.parametrize("heads,kv_heads,hidden", [(8, 2, 512), (4, 4, 512)])
def test_every_step_sees_what_the_whole_model_sees(lengths, chunk, heads, kv_heads, hidden, dtype, limit):
  model = small_model(dtype, heads, kv_heads, hidden)
  ids = prompts(len(lengths), max(lengths) + 2, 256, 3)
  gen = torch.Generator(device=DEV).manual_seed(5)
  tokens, logprobs, logits = tpa.generate(model, ids, 20, prompt_lengths=lengths, temperature=0.8, top_k=50, generator=gen, page_size=16,
                                          prompt_chunk=chunk, return_logits=True)  # fmt: skip
  assert tokens.shape == logprobs.shape == (len(lengths), 20) and ((tokens >= 0) & (tokens < 256)).all() and (logprobs <= 0).all()
  check(model, ids, lengths, tokens, logits, limit)


def test_greedy_tokens_are_the_largest_logits():
  model = small_model(torch.float32)
  ids = prompts(3, 40, 256, 4)
  tokens, logprobs, logits = tpa.generate(model, ids, 30, temperature=0.0, return_logits=True)
  assert torch.equal(tokens, logits.argmax(-1)) and (logprobs == 0).all()
  check(model, ids, [40] * 3, tokens, logits, 1e-4)


@pytest.mark.parametrize("chunk", [None, 48])
def test_a_cache_in_8_bits(chunk):
  model = small_model(torch.bfloat16)
  lengths = [100, 17]
  ids = prompts(2, 100, 256, 6)
  tokens, _, logits = tpa.generate(model, ids, 24, prompt_lengths=lengths, temperature=0.0, quantized_cache=True, prompt_chunk=chunk, return_logits=True)
  check(model, ids, lengths, tokens, logits, 0.1)


def test_the_same_numbers_give_the_same_tokens_and_an_end_ends():
  model = small_model(torch.bfloat16)
  ids = prompts(4, 12, 256, 7)
  draw = lambda **kw: tpa.generate(model, ids, 40, generator=torch.Generator(device=DEV).manual_seed(9), **kw)  # noqa: E731
  tokens, logprobs = draw(temperature=1.0, top_p=0.9)
  again, _ = draw(temperature=1.0, top_p=0.9)
  assert torch.equal(tokens, again)
  eos = int(tokens[1, 3])
  ended, lp = draw(temperature=1.0, top_p=0.9, eos_token_id=eos)
  for b in range(4):
    hits = (tokens[b] == eos).nonzero()[:, 0].tolist()
    n = ended.shape[1]
    end = hits[0] + 1 if hits else n
    assert torch.equal(ended[b, :end], tokens[b, :end]) and (ended[b, end:] == -1).all() and (lp[b, end:] == 0).all()
  each, _ = draw(temperature=torch.tensor([0.0, 1.0, 1.0, 0.0], device=DEV), top_p=0.9)
  assert torch.equal(each[1:3], tokens[1:3])


@pytest.mark.parametrize("vocab", [256, 40000])  # (the small table's own lookup, and the library's)
@pytest.mark.parametrize("pad", [-1, -100, 2**40])
@pytest.mark.parametrize("chunk", [None, 32])
def test_what_is_behind_a_prompt_is_not_read(chunk, pad, vocab):
  """Values that are no tokens behind the prompts change nothing, bit for bit."""
  model = small_model(torch.bfloat16, vocab=vocab)
  lengths = [5, 70, 33, 64]
  ids = prompts(4, 75, vocab, 10)
  draw = lambda ids: tpa.generate(model, ids, 6, prompt_lengths=lengths, temperature=0.0, prompt_chunk=chunk, return_logits=True)  # noqa: E731
  want = draw(ids)
  for b, n in enumerate(lengths):
    ids[b, n:] = pad
  got = draw(ids)
  assert torch.isfinite(got[2]).all() and all(torch.equal(g, w) for g, w in zip(got, want))


def test_refusals():
  model = small_model(torch.bfloat16, layers=1)
  ids = prompts(2, 8, 256, 8)
  for err, call in (
    (TypeError, lambda: tpa.generate(model.model, ids, 4)),
    (ValueError, lambda: tpa.generate(model, ids[0], 4)),
    (ValueError, lambda: tpa.generate(model, ids, 0)),
    (ValueError, lambda: tpa.generate(model, ids, 4, prompt_lengths=[8])),
    (ValueError, lambda: tpa.generate(model, ids, 4, prompt_lengths=[0, 8])),
    (ValueError, lambda: tpa.generate(model, ids, 4, prompt_lengths=[9, 8])),
    (ValueError, lambda: tpa.generate(model, ids, 4, prompt_chunk=1)),
    (ValueError, lambda: tpa.generate(model, ids, 4, page_size=12)),
  ):  # fmt: skip
    with pytest.raises(err):
      call()
