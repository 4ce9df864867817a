"""What the operators of 8-bit integers and log-probabilities refuse, before anything runs: through the C interface without a
device, and through ops for tensors that are not on one."""
import pytest
import torch

from semi_pd_b200 import _lib, ops
from semi_pd_b200._lib import lib

A = 4096  # an aligned address that nothing reads


def mm(out=A, a=A, b=A, sa=A, sb=A, bias=None, M=4, N=64, K=64, lda=64, ldb=64, ldc=64, dtype=0):
    return lib.spd_int8_scaled_mm(out, a, b, sa, sb, bias, M, N, K, lda, ldb, ldc, dtype, 0, 0, None)


@pytest.mark.parametrize("code,kw", [
    (-1, dict(out=None)), (-1, dict(a=None)), (-1, dict(b=None)), (-1, dict(sa=None)), (-1, dict(sb=None)), (-1, dict(M=-1)),
    (-1, dict(N=0)), (-1, dict(K=0)), (-1, dict(dtype=2)), (-1, dict(dtype=7)), (-1, dict(lda=48)), (-1, dict(ldb=48)), (-1, dict(ldc=56)),
    (-2, dict(K=56)), (-2, dict(N=60)), (-2, dict(lda=72)), (-2, dict(ldb=72)), (-2, dict(ldc=68)), (-2, dict(a=A + 8)),
    (-2, dict(b=A + 1)), (-2, dict(out=A + 2)), (-3, dict(K=131072, lda=131072, ldb=131072)),
    (-3, dict(M=1 << 27, N=1 << 20, ldc=1 << 20)), (-1, dict(M=1 << 31))])
def test_product_refuses(code, kw):
    assert mm(**kw) == code and lib.spd_last_error_string()


def test_no_tokens_is_no_work():
    assert mm(M=0) == 0
    assert lib.spd_quant_int8(A, A, A, None, None, 0, 64, 64, 0.0, 0, 0, 0, None) == 0


def quant(q=A, s=A, x=A, residual=None, weight=None, rows=2, dim=64, stride=64, silu=0, dtype=0):
    return lib.spd_quant_int8(q, s, x, residual, weight, rows, dim, stride, 1e-5, silu, dtype, 0, None)


@pytest.mark.parametrize("code,kw", [
    (-1, dict(q=None)), (-1, dict(s=None)), (-1, dict(x=None)), (-1, dict(rows=-1)), (-1, dict(dim=0)), (-1, dict(dtype=2)),
    (-1, dict(residual=A)), (-1, dict(weight=A, silu=1, stride=128)), (-1, dict(silu=1)), (-1, dict(stride=48)), (-2, dict(dim=72, stride=72)),
    (-2, dict(stride=68)), (-2, dict(x=A + 2)), (-2, dict(q=A + 8)), (-2, dict(weight=A + 2)), (-3, dict(dim=32784, stride=32784))])
def test_quant_refuses(code, kw):
    assert quant(**kw) == code


def score(lp=A, lse=A, x=A, w=A, xs=None, ws=None, t=A, M=2, V=100, K=64, ldx=64, ldw=64, dtype=0, work=A, room=None):
    room = lib.spd_linear_logprobs_workspace_bytes(M, V) if room is None else room
    return lib.spd_linear_logprobs(lp, lse, x, w, xs, ws, t, M, V, K, ldx, ldw, dtype, 0, work, room, 0, None)


@pytest.mark.parametrize("code,kw", [
    (-1, dict(lp=None)), (-1, dict(lse=None)), (-1, dict(x=None)), (-1, dict(w=None)), (-1, dict(t=None)), (-1, dict(work=None)),
    (-1, dict(M=-1, room=0)), (-1, dict(V=0, room=0)), (-1, dict(K=0)), (-1, dict(dtype=2)), (-1, dict(ldx=56)), (-1, dict(ldw=56)),
    (-1, dict(xs=A)), (-1, dict(ws=A)), (-1, dict(dtype=3)), (-1, dict(dtype=3, xs=A)), (-2, dict(K=60)), (-2, dict(ldx=68)),
    (-2, dict(ldw=68)), (-2, dict(dtype=3, xs=A, ws=A, K=56, ldx=56, ldw=56)), (-2, dict(x=A + 2)), (-2, dict(w=A + 2)),
    (-2, dict(work=A + 4)), (-4, dict(room=39)), (-3, dict(dtype=3, xs=A, ws=A, K=131072, ldx=131072, ldw=131072)),
    (-3, dict(M=1 << 27, V=1 << 20))])
def test_logprobs_refuse(code, kw):
    assert score(**kw) == code


def test_workspace_bytes():
    # two parts of every 256 rows of the vocabulary, 8 bytes each, and the target's logit
    assert lib.spd_linear_logprobs_workspace_bytes(3, 257) == 3 * (2 * 2 * 8 + 4)
    assert lib.spd_linear_logprobs_workspace_bytes(0, 257) == 0
    assert lib.spd_linear_logprobs_workspace_bytes(-1, 257) < 0 and lib.spd_linear_logprobs_workspace_bytes(1, 0) < 0


def test_there_is_no_cpu_path():
    x = torch.ones(2, 64, dtype=torch.bfloat16)
    i = torch.ones(2, 64, dtype=torch.int8)
    for call in (lambda: ops.per_token_quant_int8(x), lambda: ops.rmsnorm_quant_int8(x, x[0]),
                 lambda: ops.fused_add_rmsnorm_quant_int8(x, x, x[0]), lambda: ops.silu_and_mul_quant_int8(x),
                 lambda: ops.int8_scaled_mm(i, i.t(), torch.ones(2), torch.ones(2), torch.bfloat16),
                 lambda: ops.linear_logprobs(x, x, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_dtype_codes():
    assert _lib.SPD_I8 == 3 and "SPD_I8 3" in open(_lib.HEADER_PATH).read()


def test_quantization_flag():
    from semi_pd_b200.launch_server import prepare_server_args
    assert prepare_server_args([]).quantization is None
    assert prepare_server_args(["--quantization", "w8a8_int8"]).quantization == "w8a8_int8"
    with pytest.raises(SystemExit):
        prepare_server_args(["--quantization", "fp4"])


def tiny(quantization="w8a8_int8"):
    from semi_pd_b200.configs import get_model_config
    from semi_pd_b200.llama import LlamaForCausalLM
    return LlamaForCausalLM(get_model_config("tiny-llama-test"), device="cpu", quantization=quantization)


def checkpoint(model, int8=True):
    for name, shape in model.full_shapes().items():
        if int8 and name.endswith("proj.weight"):
            yield name, torch.ones(shape, dtype=torch.int8)
            yield name + "_scale", torch.full((shape[0],), 0.5)
        else:
            yield name, torch.ones(shape, dtype=torch.bfloat16)


def test_checkpoints_of_8_bit_weights():
    m = tiny()
    m.load_weights(checkpoint(m))
    q = m.model.layers[1].self_attn.qkv_proj
    assert q.weight.dtype == torch.int8 and q.weight_scale.shape == (q.weight.shape[0], 1) and q.weight_scale.dtype == torch.float32
    assert m.lm_head.weight.dtype == torch.bfloat16
    names = {n for n, _ in checkpoint(m)}
    assert names == set(m.state_dict())
    with pytest.raises(KeyError, match="missing"):
        m.load_weights((n, w) for n, w in checkpoint(m) if n != "model.layers.0.mlp.down_proj.weight_scale")
    with pytest.raises(ValueError, match="one scale"):
        m.load_weights((n, w[:-1] if n == "model.layers.0.mlp.down_proj.weight_scale" else w) for n, w in checkpoint(m))
    with pytest.raises(ValueError, match="quantization"):
        plain = tiny(None)
        plain.load_weights((n, w) for n, w in checkpoint(plain) if not n.endswith("_scale"))
    with pytest.raises(KeyError, match="unexpected"):
        plain.load_weights((n, w) for n, w in checkpoint(plain) if n.endswith("_scale"))
    with pytest.raises(ValueError, match="quantization"):
        tiny("int3")


def test_shards_of_8_bit_weights():
    from semi_pd_b200.layers import MergedColumnParallelLinear, QKVParallelLinear, RowParallelLinear
    scale = torch.arange((4 + 2 * 2) * 8, dtype=torch.float32)[:, None]
    parts = [QKVParallelLinear.shard(scale, 8, 4, 2, r, 2) for r in range(2)]
    w = scale.expand(-1, 16).contiguous()
    for r in range(2):
        assert torch.equal(QKVParallelLinear.shard(w, 8, 4, 2, r, 2)[:, :1], parts[r])
        assert torch.equal(MergedColumnParallelLinear.shard(w, r, 2)[:, :1], MergedColumnParallelLinear.shard(scale, r, 2))
        assert RowParallelLinear.shard(w, r, 2).shape == (64, 8)
