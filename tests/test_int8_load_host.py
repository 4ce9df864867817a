"""Weights of 8 bits that no product takes are refused when they are loaded, by name."""
import dataclasses

import pytest
import torch

from semi_pd_b200 import llama
from semi_pd_b200.configs import get_model_config
from tests.test_int8_host import checkpoint


def model(monkeypatch=None, tp=1, **changes):
    m = llama.LlamaForCausalLM(dataclasses.replace(get_model_config("tiny-llama-test"), **changes), device="cpu", quantization="w8a8_int8")
    if tp > 1:
        monkeypatch.setattr(llama, "get_tensor_model_parallel_world_size", lambda: tp)
        monkeypatch.setattr(llama, "get_tensor_model_parallel_rank", lambda: 0)
    return m


@pytest.mark.parametrize("int8", [True, False])
def test_columns(int8):
    m = model(intermediate_size=1016)
    with pytest.raises(ValueError, match=r"model\.layers\.0\.mlp\.down_proj\.weight: a shard of \d+ x 1016 "):
        # (16-bit ones before it would be quantised, which needs a GPU)
        m.load_weights((n, w) for n, w in checkpoint(m, int8) if int8 or n.endswith("down_proj.weight"))


def test_columns_of_a_shard(monkeypatch):
    m = model(monkeypatch, tp=2, intermediate_size=1040)  # 65 x 16, 520 a rank
    with pytest.raises(ValueError, match=r"down_proj\.weight: a shard of \d+ x 520 "):
        m.load_weights(checkpoint(m))
    monkeypatch.undo()
    m.load_weights(checkpoint(m))


def test_long_rows():
    m = model(intermediate_size=32784)
    with pytest.raises(ValueError, match=r"down_proj\.weight: a shard of \d+ x 32784 .* at most 32768"):
        m.load_weights((n, w) for n, w in checkpoint(m, False) if n.endswith("down_proj.weight"))
    m.load_weights(checkpoint(m))  # as they come in 8 bits


def test_rows():
    m = model()
    name = "model.layers.1.self_attn.o_proj.weight"
    with pytest.raises(ValueError, match="o_proj.weight: a shard of 4 x "):
        m.load_weights((n, w[:4] if n == name else w) for n, w in checkpoint(m))


@pytest.mark.parametrize("name", ["model.embed_tokens.weight", "lm_head.weight", "model.norm.weight"])
def test_weights_that_are_not_products(name):
    m = model()
    with pytest.raises(ValueError, match=name + ": only the weights of products"):
        m.load_weights((n, w.to(torch.int8) if n == name else w) for n, w in checkpoint(m))
