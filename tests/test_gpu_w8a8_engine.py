"""A model of 8-bit weights in the semi-PD engine (two workers at once on their parts of the GPU, decode graphs, chunked prefill) against the
same model one request at a time, and the operators' first calls inside a stream capture."""
import subprocess
import sys

import pytest
import torch

from oracle import llama_oracle as O
from tests.helpers import GpuSession

pytestmark = pytest.mark.gpu
CFG = dict(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
           vocab_size=1024, max_position_embeddings=2048)
NEW = 10


def server_args(graph_bs):
    from semi_pd_b200.configs import ServerArgs
    return ServerArgs(model_path="tiny", dtype="float16", load_format="external", max_total_tokens=8192, max_running_requests=16,
                      context_length=1024, enable_semi_pd=True, cuda_graph_bs=graph_bs, disable_cuda_graph=graph_bs is None,
                      chunked_prefill_size=96, max_prefill_tokens=4096, quantization="w8a8_int8")


def test_engine(monkeypatch):
    import semi_pd_b200.model_runner as MR
    from semi_pd_b200.configs import ModelConfig
    from semi_pd_b200.semi_pd_scheduler import SemiPDEngine
    weights = O.make_weights(O.OracleLlamaConfig(**CFG), torch.float16, seed=77)
    lens = [5, 130, 17, 64, 257, 1, 33, 200, 9, 128]
    prompts = [[(11 + 7 * i + 29 * j) % 1024 for i in range(n)] for j, n in enumerate(lens)]
    mr = MR.ModelRunner(ModelConfig(name="tiny", **CFG), 0.3, 0, 0, 1, 0, server_args(None))
    mr.model.load_weights(weights.items())
    mr.init_attention_backend()
    mr.init_cuda_graphs()
    expected = []
    for p in prompts:
        gs = GpuSession(mr)
        reqs, logits, ids = gs.extend([p])
        toks, margins = [], []
        for _ in range(NEW):
            top = logits.topk(2, -1).values[0]
            margins.append(float(top[0] - top[1]))
            toks.append(int(ids[0]))
            logits, ids = gs.decode(reqs, [toks[-1]])
        expected.append((toks, margins))
        mr.token_to_kv_pool_allocator.free_req(reqs[0].req_pool_idx)
        mr.req_to_token_pool.free(reqs[0].req_pool_idx)
    load = MR.ModelRunner.load_model

    def load_with_weights(self):
        load(self)
        self.model.load_weights(weights.items())

    monkeypatch.setattr(MR.ModelRunner, "load_model", load_with_weights)
    eng = SemiPDEngine(server_args([1, 2, 4, 8, 16]), gpu_id=0, model_config=ModelConfig(name="tiny", **CFG), prefill_sm_percent=50,
                       decode_sm_percent=50, partition="green")
    try:
        eng.warmup(prompt_len=8, n=2, max_new_tokens=2)
        rids = [eng.submit(p, NEW) for p in prompts]
        done = {r.rid: r for r in eng.wait(len(prompts), timeout=120)}
    finally:
        eng.shutdown()
    # Products are the same bits in any batch; attention is not (it is cut otherwise), and an activation's 16-bit rounding may move an
    # integer by a step, 1 / 127 of the largest: ids are compared up to a margin of 0.1 of logits of 1.5
    checked = 0
    for rid, (toks, margins) in zip(rids, expected):
        got = done[rid].output_ids
        assert len(got) == NEW
        for k in range(NEW):
            if margins[k] <= 0.1:
                break
            assert got[k] == toks[k], (rid, k, got, toks)
            checked += 1
    assert checked > len(prompts)


FIRST = """
import torch
from semi_pd_b200 import ops
g = torch.Generator(device="cuda").manual_seed(1)
x = torch.randn(%d, 512, generator=g, device="cuda").bfloat16()
r = torch.randn(%d, 512, generator=g, device="cuda").bfloat16()
w = torch.randint(-127, 128, (1024, 512), generator=g, device="cuda", dtype=torch.int8)
v = torch.randn(3000, 512, generator=g, device="cuda").bfloat16()
norm, ws, t = torch.ones(512, device="cuda").bfloat16(), torch.rand(1024, device="cuda"), torch.arange(len(x), device="cuda")
def step(r):
    q, s = ops.fused_add_rmsnorm_quant_int8(x, r, norm)
    h = ops.int8_scaled_mm(q, w.t(), s, ws, torch.bfloat16)
    return (*ops.silu_and_mul_quant_int8(h), *ops.rmsnorm_quant_int8(x, norm), *ops.per_token_quant_int8(x), *ops.linear_logprobs(x, v, t))
torch.cuda.synchronize()
graph, keep = torch.cuda.CUDAGraph(), r.clone()
with torch.cuda.graph(graph):
    out = step(r)
graph.replay()
torch.cuda.synchronize()
want = step(keep)
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(r, keep)
ops.check_waits()
print("captured")
"""


@pytest.mark.parametrize("rows", [3, 2000])
def test_first_calls_inside_a_capture(rows):
    out = subprocess.run([sys.executable, "-c", FIRST % (rows, rows)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]
