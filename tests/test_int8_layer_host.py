"""A layer that quantises its weight: what its products may read early is behind a copy in the stream."""
import pytest
import torch

from semi_pd_b200 import layers


def test_a_copy_stands_between_the_quantisation_and_the_products(monkeypatch):
    order = []
    quantised = torch.ones(4, 16, dtype=torch.int8), torch.rand(4, 1)

    class Recorded(torch.Tensor):
        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            order.append(getattr(func, "__name__", str(func)))
            return super().__torch_function__(func, types, args, kwargs or {})

    def quant(w):
        order.append("quant")
        return quantised[0], quantised[1].as_subclass(Recorded)

    monkeypatch.setattr(layers.ops, "per_token_quant_int8", quant)
    layer = layers.LinearBase(16, 4)
    layer.weight = torch.zeros(4, 16)
    layer.quantize_weight_int8()
    assert order == ["quant", "clone"]
    assert torch.equal(layer.weight, quantised[0]) and torch.equal(layer.weight_scale.as_subclass(torch.Tensor), quantised[1])
    assert layer.weight_scale.data_ptr() != quantised[1].data_ptr()


def test_a_sum_over_the_ranks_is_not_left_out(monkeypatch):
    calls = []
    for name in ("rmsnorm_quant_int8", "fused_add_rmsnorm_quant_int8", "per_token_quant_int8"):
        monkeypatch.setattr(layers.ops, name, lambda x, *a, name=name: (calls.append(name), (x, x))[1])
    norm = layers.RMSNorm(16)
    x = torch.zeros(2, 16)
    norm.forward_quant(x)
    norm.forward_quant(x, torch.zeros(2, 16))
    assert calls == ["rmsnorm_quant_int8", "fused_add_rmsnorm_quant_int8"]
    x._spd_pending_all_reduce = True
    with pytest.raises(AssertionError):
        norm.forward_quant(x)
    reduced = torch.ones(2, 16)
    monkeypatch.setattr(layers.RMSNorm, "forward", lambda self, x, residual: (reduced, residual + 1))
    tokens, residual = norm.forward_quant(x, torch.zeros(2, 16))
    assert tokens.q is reduced and residual.sum() == 32 and calls[2:] == ["per_token_quant_int8"]
