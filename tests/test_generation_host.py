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


class OtherAttention(tpa.LlamaAttention):
  def forward(self, *args, **kw):
    return 2 * super().forward(*args, **kw)


class OtherModel(tpa.LlamaForCausalLM):
  def forward(self, *args, **kw):
    return super().forward(*args, **kw)


def _of(model, path):
  for name in path.split("."):
    model = model[int(name)] if name.isdigit() else getattr(model, name) if name else model
  return model


CALLED = ["", "model", "model.layers.1", "model.layers.1.self_attn", "model.layers.0.self_attn.attention_block", "model.layers.1.input_layernorm",
          "model.layers.0.post_attention_layernorm", "model.norm"]  # fmt: skip


@pytest.mark.parametrize("path", CALLED)
@pytest.mark.parametrize("how", ["hook", "pre_hook", "forward"])
def test_a_module_that_has_to_see_its_own_call_is_not_passed_by(path, how):
  model = small_model()
  m = _of(model, path)
  if how == "forward":
    m.forward = m.forward
  else:
    handle = m.register_forward_hook(lambda *_: None) if how == "hook" else m.register_forward_pre_hook(lambda *_: None)
  ids = torch.zeros((1, 4), dtype=torch.long)
  with pytest.raises(NotImplementedError, match=type(m).__name__):
    tpa.generate(model, ids, 2)
  if how != "forward":
    handle.remove()
    with pytest.raises(RuntimeError, match="no CPU path"):  # (taken, as far as the CPU goes)
      tpa.generate(model, ids, 2)


def test_other_classes_hooks_of_all_modules_and_other_attention_are_refused():
  ids = torch.zeros((1, 4), dtype=torch.long)
  model = small_model()
  model.model.layers[1].self_attn = OtherAttention(model.config, 1)
  with pytest.raises(NotImplementedError, match="OtherAttention"):
    tpa.generate(model, ids, 2)
  model = small_model()
  with pytest.raises(NotImplementedError, match="OtherModel"):
    tpa.generate(OtherModel(model.config), ids, 2)
  handle = torch.nn.modules.module.register_module_forward_hook(lambda *_: None)
  try:
    with pytest.raises(NotImplementedError, match="hooks"):
      tpa.generate(model, ids, 2)
  finally:
    handle.remove()
  for kw in (dict(load_balance_cp=True, context=2), dict(attention_kernel=None, attention_dropout=0.1)):
    model = small_model(**kw).train()
    with pytest.raises(NotImplementedError, match="attention"):
      tpa.generate(model, ids, 2)
  with pytest.raises(TypeError):
    tpa.generate(small_model().model, ids, 2)


def test_modules_that_generate_calls_keep_their_hooks():
  """Projections, the MLP and the embedding are called as they are; a hook of the backward has nothing to see."""
  model = small_model()
  layer = model.model.layers[0]
  for m in (layer.mlp, layer.self_attn.q_proj, model.lm_head, model.model.embed_tokens):
    m.register_forward_hook(lambda *_: None)
  model.model.layers[1].register_full_backward_hook(lambda *_: None)
  with pytest.raises(RuntimeError, match="no CPU path"):
    tpa.generate(model, torch.zeros((1, 4), dtype=torch.long), 2)


def test_a_subclass_that_runs_as_its_base_does_is_taken():
  class Named(tpa.LlamaForCausalLM):
    def name(self):
      return "named"

  with pytest.raises(RuntimeError, match="no CPU path"):
    tpa.generate(Named(small_model().config), torch.zeros((1, 4), dtype=torch.long), 2)
