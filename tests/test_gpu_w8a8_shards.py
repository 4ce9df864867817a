"""A feed-forward of 8-bit weights in two shards: each rank's part against its definition, and the norm behind their sum.  The ranks run one
after another on one GPU; their sum is made here."""
import pytest
import torch

from oracle import llama_oracle as O
from semi_pd_b200 import distributed, ops
from semi_pd_b200.configs import ModelConfig
from semi_pd_b200.layers import QuantizedTokens
from semi_pd_b200.llama import LlamaForCausalLM
from tests.test_gpu_w8a8_model import TINY, is_linear, quantised

pytestmark = pytest.mark.gpu
DEV = "cuda"
CFG = dict(TINY, hidden_size=1024, intermediate_size=2816, num_attention_heads=8, num_key_value_heads=2, num_hidden_layers=1)
H, I = 1024, 2816


class Comm:
    """The other rank's part is at hand; fused: in the norm's own kernel, as the peer-memory communicator does it."""

    def __init__(self, other, fused):
        self.other, self.fused = other, fused

    def all_reduce(self, x):
        return x.add_(self.other)

    def all_reduce_add_rmsnorm(self, x, residual, weight, eps):
        if self.fused:
            ops.fused_add_rmsnorm(self.all_reduce(x), residual, weight, eps)
        return self.fused


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("int8", [False, True], ids=["16-bit checkpoint", "8-bit checkpoint"])
def test_feed_forward(monkeypatch, int8, fused):
    weights = O.make_weights(O.OracleLlamaConfig(**CFG), torch.bfloat16)
    checkpoint = {}
    for k, w in weights.items():
        if int8 and is_linear(k):
            checkpoint[k], checkpoint[k + "_scale"] = quantised(w)
        else:
            checkpoint[k] = w
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(37, H, generator=g, device=DEV).bfloat16()
    r = torch.randn(37, H, generator=g, device=DEV).bfloat16()

    def quant(v):
        top = v.abs().amax(1, keepdim=True)
        t = v * 127 / top
        return torch.sign(t) * torch.floor(t.abs() + 0.5) * top / 127

    def shard(name, cut):
        """The numbers that a rank's integers stand for: 16-bit weights are quantised by the rank, 8-bit ones cut as they are."""
        w = weights["model.layers.0.mlp." + name].to(DEV)
        q, s = quantised(w if int8 else cut(w))
        return cut(q.double() * s.double()) if int8 else q.double() * s.double()

    monkeypatch.setattr(distributed, "_TP_SIZE", 2)
    y = x.double() + r.double()
    h = quant(y / torch.sqrt((y * y).mean(1, keepdim=True) + 1e-5) * weights["model.layers.0.post_attention_layernorm.weight"].to(DEV).double())
    parts, layers = [], []
    for rank in range(2):
        monkeypatch.setattr(distributed, "_TP_RANK", rank)
        m = LlamaForCausalLM(ModelConfig(name="tiny-llama-test", **CFG), device=DEV, quantization="w8a8_int8")
        m.load_weights(checkpoint.items())
        layer = m.model.layers[0]
        assert layer.mlp.down_proj.weight.shape == (H, I // 2) and layer.mlp.gate_up_proj.weight_scale.shape == (I, 1)
        tokens, residual = layer.post_attention_layernorm.forward_quant(x.clone(), r.clone())
        part = layer.mlp(tokens)
        assert part._spd_pending_all_reduce
        half = slice(rank * I // 2, (rank + 1) * I // 2)
        gate_up = (h @ shard("gate_up_proj.weight", lambda w: torch.cat([w[:I][half], w[I:][half]])).t()).to(torch.bfloat16).double()
        mid = quant(gate_up[:, :I // 2] * torch.sigmoid(gate_up[:, :I // 2]) * gate_up[:, I // 2:])
        want = mid @ shard("down_proj.weight", lambda w: w[:, half]).t()
        # as for the whole layer: the output's rounding, and integers beside a half, one in 200 at most, a thirtieth of the rms each
        assert ((part.double() - want).norm() / want.norm()).item() < 2.0 ** -9 + (1 / 200) ** 0.5 / 30
        parts.append(part)
        layers.append(layer)
    # what the next layer's norm makes of the parts: their sum and the residual, normed to 16 bits, then quantised
    total, kept = parts[0] + parts[1], residual.clone()
    ops.fused_add_rmsnorm(total, kept, layers[0].input_layernorm.weight, 1e-5)
    q, s = ops.per_token_quant_int8(total)
    distributed.set_current_comm(Comm(parts[1], fused))
    try:
        tokens, out = layers[0].input_layernorm.forward_quant(parts[0], residual)
    finally:
        distributed.set_current_comm(None)
    assert isinstance(tokens, QuantizedTokens) and tokens.dtype == torch.bfloat16
    assert torch.equal(tokens.q, q) and torch.equal(tokens.scales, s) and torch.equal(out, kept)
    assert not parts[0]._spd_pending_all_reduce
