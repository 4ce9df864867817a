"""A Llama model of 8-bit integer weights (quantization="w8a8_int8") and return_logprob through the serving path."""
import pytest
import torch

from oracle import llama_oracle as O
from semi_pd_b200 import ops
from semi_pd_b200.configs import ModelConfig, ServerArgs
from semi_pd_b200.forward_batch_info import ForwardBatch
from semi_pd_b200.layers import QuantizedTokens
from semi_pd_b200.model_runner import ModelRunner
from tests.helpers import GpuSession

pytestmark = pytest.mark.gpu
DEV = "cuda"
TINY = dict(hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
            vocab_size=1000, max_position_embeddings=2048)
LAYER_8B = dict(TINY, hidden_size=4096, intermediate_size=14336, num_attention_heads=32, num_key_value_heads=8, vocab_size=4096)


def is_linear(name):
    return name.endswith("proj.weight")


def quantised(w):
    top = w.double().abs().amax(1, keepdim=True)
    t = w.double() * 127 / top
    return (torch.sign(t) * torch.floor(t.abs() + 0.5)).to(torch.int8), (top / 127).float()


def runner(cfg, dtype, weights, quantization="w8a8_int8", graph_bs=None):
    sa = ServerArgs(model_path="tiny-llama-test", dtype="bfloat16" if dtype == torch.bfloat16 else "float16", load_format="external",
                    max_total_tokens=4096, max_running_requests=16, context_length=1024, disable_cuda_graph=graph_bs is None,
                    cuda_graph_bs=graph_bs, enable_semi_pd=True, quantization=quantization)
    mr = ModelRunner(ModelConfig(name="tiny-llama-test", **cfg), 0.5, 0, 0, 1, 0, sa)
    mr.model.load_weights(weights.items())
    mr.init_attention_backend()
    mr.init_cuda_graphs()
    return mr


def prompts(lens, vocab):
    return [[(7 + 13 * i + 31 * j) % vocab for i in range(n)] for j, n in enumerate(lens)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cfg", [TINY, LAYER_8B], ids=["tiny", "8b-2layer"])
def test_extend_and_decode_near_the_dequantised_model(cfg, dtype):
    """Logits against the oracle in fp32 on the weights that the integers stand for.  What differs is the activations' rounding to 8
    bits: half a step is max / 254 of a token, so a product's output gets noise of max / rms / 127 / sqrt(12).  Normed tokens of 4096
    gaussian values have a max of 4 times their rms: 0.9 %.  SiLU(g) u of two gaussians has rms 0.6 and, of 14336, values up to 9: 15
    times the rms, 3.4 %.  A layer's feed-forward: sqrt(2 0.9^2 + 3.4^2) = 3.7 %; two layers 5.2 % of what they add, and the
    residual stream holds more than that."""
    weights = O.make_weights(O.OracleLlamaConfig(**cfg), dtype)
    deq = {}
    for k, w in weights.items():
        if is_linear(k):
            q, s = quantised(w)
            deq[k] = (q.double() * s.double()).float()
        else:
            deq[k] = w.float()
    mr = runner(cfg, dtype, weights)
    gs = GpuSession(mr)
    oracle = O.LlamaOracle(O.OracleLlamaConfig(**cfg), deq, kv_slots=4096, max_reqs=17, max_ctx=1028, compute="fp32")
    os_ = O.OracleSession(oracle, 4096, 17)
    p = prompts([5, 1, 130, 300], cfg["vocab_size"])
    reqs, lg, _ = gs.extend(p)
    rids, lc, _ = os_.extend(p)
    rel = lambda a, b: ((a.double() - b.double()).norm() / b.double().norm()).item()  # noqa: E731
    assert rel(lg, lc) < 0.052, rel(lg, lc)
    for _ in range(3):
        tok = lc.argmax(-1).tolist()
        lg, _ = gs.decode(reqs, tok)
        lc, _ = os_.decode(rids, tok)
        assert rel(lg, lc) < 0.052, rel(lg, lc)


def test_layer_against_its_definition():
    """One feed-forward on the same 16-bit tokens: norm, gate and up, SiLU * mul, down, each quantised as defined, in 64 bits."""
    weights = O.make_weights(O.OracleLlamaConfig(**LAYER_8B), torch.bfloat16)
    mr = runner(LAYER_8B, torch.bfloat16, weights)
    layer = mr.model.model.layers[1]
    x = torch.randn(37, 4096, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).bfloat16()
    r = torch.randn(37, 4096, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).bfloat16()
    y = x.double() + r.double()
    tokens, residual = layer.post_attention_layernorm.forward_quant(x.clone(), r.clone())
    assert isinstance(tokens, QuantizedTokens) and torch.equal(residual, y.to(torch.bfloat16))
    out = layer.mlp(tokens)

    def quant(v):
        top = v.abs().amax(1, keepdim=True)
        t = v * 127 / top
        return torch.sign(t) * torch.floor(t.abs() + 0.5) * top / 127

    g = lambda n: weights["model.layers.1." + n].to(DEV)  # noqa: E731
    deq = lambda w: (lambda q, s: q.double() * s.double())(*quantised(w))  # noqa: E731
    h = quant(y / torch.sqrt((y * y).mean(1, keepdim=True) + 1e-5) * g("post_attention_layernorm.weight").double())
    gate_up = (h @ deq(g("mlp.gate_up_proj.weight")).t()).to(torch.bfloat16).double()  # what SiLU * mul reads is rounded
    h = quant(gate_up[:, :14336] * torch.sigmoid(gate_up[:, :14336]) * gate_up[:, 14336:])
    want = h @ deq(g("mlp.down_proj.weight")).t()
    # the output's rounding, 2^-9 in the mean of its 2^-8; an integer next to a half may fall to the other side where 32-bit
    # arithmetic differs (2e-5 of 127 steps either way: one in 200 at most), each a step of about max / 127, a thirtieth of the rms
    assert ((out.double() - want).norm() / want.norm()).item() < 2.0 ** -9 + (1 / 200) ** 0.5 / 30


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tokens_do_not_depend_on_their_batch(dtype):
    """Sums of integers have no order and a token's scale is its own: a row of a product is the same bits whatever tiles it was in."""
    g = torch.Generator(device=DEV).manual_seed(1)
    w, ws = ops.per_token_quant_int8(torch.randn(6144, 4096, generator=g, device=DEV).to(dtype))
    x = torch.randn(1500, 4096, generator=g, device=DEV).to(dtype)
    q, s = ops.per_token_quant_int8(x)
    whole = ops.int8_scaled_mm(q, w.t(), s, ws, dtype)
    for m in (1, 3, 33, 64, 100, 200, 256, 300, 513, 777):
        assert torch.equal(whole[:m], ops.int8_scaled_mm(q[:m], w.t(), s[:m], ws, dtype)), m


def test_decode_graphs_give_what_eager_steps_give():
    weights = O.make_weights(O.OracleLlamaConfig(**TINY), torch.bfloat16)
    logits = []
    for graph_bs in (None, [1, 2, 4]):
        gs = GpuSession(runner(TINY, torch.bfloat16, weights, graph_bs=graph_bs))
        reqs, lg, ids = gs.extend(prompts([5, 40, 7], 1000))
        logits.append([lg])
        for _ in range(3):
            lg, ids = gs.decode(reqs, ids.tolist())
            logits[-1].append(lg)
    for a, b in zip(*logits):
        assert torch.equal(a, b)


def test_checkpoint_of_8_bit_weights():
    weights = O.make_weights(O.OracleLlamaConfig(**TINY), torch.bfloat16)
    ready = {}
    for k, w in weights.items():
        if is_linear(k):
            ready[k], ready[k + "_scale"] = quantised(w)
        else:
            ready[k] = w
    out = []
    for w in (weights, ready, dict(reversed(ready.items()))):
        gs = GpuSession(runner(TINY, torch.bfloat16, w))
        out.append(gs.extend(prompts([5, 40, 7], 1000))[1])
        sd = gs.mr.model.state_dict()
        assert sd["model.layers.0.mlp.down_proj.weight"].dtype == torch.int8
        assert sd["model.layers.0.mlp.down_proj.weight_scale"].shape == (512, 1)
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])


def scored(mr, p, targets=None, rows=None):
    gs = GpuSession(mr)
    reqs = [gs.Req(f"r{i}", x, gs.SP()) for i, x in enumerate(p)]
    for r in reqs:
        r.init_next_round_input()
    sb = gs.SB.init_new(reqs, mr.req_to_token_pool, mr.token_to_kv_pool_allocator, mr.device)
    sb.return_logprob = True
    if targets is not None:
        sb.extend_input_logprob_token_ids = targets
    if rows is not None:
        sb.extend_logit_rows = rows
    sb.prepare_for_extend()
    fb = ForwardBatch.init_new(sb.get_model_worker_batch(), mr)
    out = mr.forward(fb)
    for r in reqs:
        mr.token_to_kv_pool_allocator.free_req(r.req_pool_idx)
        mr.req_to_token_pool.free(r.req_pool_idx)
    return out


@pytest.mark.parametrize("quantization", [None, "w8a8_int8"])
@pytest.mark.parametrize("lens", [[1], [5, 1, 130, 64], [400, 1, 257]])
def test_input_token_logprobs(lens, quantization):
    """Against the log-softmax of the logits that the same batch gives for all rows (which are rounded to 16 bits: half a step of the
    largest, 2^-9 of 8 at most, twice)."""
    weights = O.make_weights(O.OracleLlamaConfig(**TINY), torch.bfloat16)
    mr = runner(TINY, torch.bfloat16, weights, quantization)
    p = prompts(lens, 1000)
    T = sum(lens)
    every = torch.arange(T, device=DEV)
    out = scored(mr, p, rows=every)
    assert out.next_token_logits.shape == (T, 1000) and out.next_token_logits.abs().max() < 8
    logp = torch.log_softmax(out.next_token_logits.double(), 1)
    want = torch.zeros(T, dtype=torch.float64, device=DEV)
    at = 0
    for x in p:
        for i in range(len(x) - 1):
            want[at + i] = logp[at + i, x[i + 1]]
        at += len(x)
    got = out.input_token_logprobs
    assert got.shape == (T,) and got.dtype == torch.float32
    assert ((got.double() - want).abs() <= 2 * 8 * 2.0 ** -9).all()
    ends = torch.tensor(lens, device=DEV).cumsum(0) - 1
    assert (got[ends] == 0).all()
    # tokens of the caller's own, the next chunk's first among them
    targets = torch.arange(T, device=DEV) * 7 % 1000
    targets[::3] = -1
    got = scored(mr, p, targets=targets).input_token_logprobs
    want = torch.where(targets >= 0, logp[every, targets.clamp(min=0)], torch.zeros_like(want))
    assert ((got.double() - want).abs() <= 2 * 8 * 2.0 ** -9).all()


def test_no_logprobs_unless_asked_for():
    weights = O.make_weights(O.OracleLlamaConfig(**TINY), torch.bfloat16)
    mr = runner(TINY, torch.bfloat16, weights, None)
    gs = GpuSession(mr)
    sb = gs.SB.init_new([r := gs.Req("r", [1, 2, 3], gs.SP())], mr.req_to_token_pool, mr.token_to_kv_pool_allocator, mr.device)
    r.init_next_round_input()
    sb.prepare_for_extend()
    assert mr.forward(ForwardBatch.init_new(sb.get_model_worker_batch(), mr)).input_token_logprobs is None
