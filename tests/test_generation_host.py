"""What generate does before a GPU is needed: the ids that it looks up, and the models that it refuses.  On the CPU."""

import pytest
import torch

import torchprime_amd as tpa
from torchprime_amd import generation


def small_model(**kw):
  cfg = dict(vocab_size=50, num_hidden_layers=2, max_position_embeddings=256, hidden_size=128, intermediate_size=64, num_attention_heads=2,
             num_key_value_heads=1, hidden_act="silu", initializer_range=0.02, rms_norm_eps=1e-5, attention_dropout=False, attention_bias=False,
             rope_theta=500000.0, attention_kernel="splash_attention") | kw  # fmt: skip
  return tpa.LlamaForCausalLM(tpa.Config(**cfg)).eval()


@pytest.mark.parametrize("pad", [-1, -100, 2**40])
@pytest.mark.parametrize("lengths,chunk", [([5, 1, 3], None), ([9, 4, 7], 4), ([8, 8, 8], None), ([8, 8, 8], 3)])
def test_only_ids_of_the_prompts_are_looked_up(monkeypatch, lengths, chunk, pad):
  """What is behind a prompt may be no token at all (the -1 that generate itself returns after an end)."""
  model = small_model()
  ids = torch.randint(50, (3, max(lengths) + 2), generator=torch.Generator().manual_seed(1))
  for b, n in enumerate(lengths):
    ids[b, n:] = pad
  given, seen = ids.clone(), []

  def hidden(inner, ids, positions, *_):
    seen.append(ids.clone())
    return torch.zeros((*ids.shape, 128)), torch.zeros((*ids.shape, 128))

  monkeypatch.setattr(generation, "_hidden", hidden)
  with pytest.raises(RuntimeError, match="no CPU path"):  # (the last norm)
    tpa.generate(model, ids, 2, prompt_lengths=lengths, prompt_chunk=chunk)
  seen = torch.cat(seen, 1)
  assert seen.shape == (3, max(lengths)) and ((seen >= 0) & (seen < 50)).all()
  for b, n in enumerate(lengths):
    assert torch.equal(seen[b, :n], given[b, :n])
  assert torch.equal(ids, given)
