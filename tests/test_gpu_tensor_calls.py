"""The operators that take tensors in one call (csrc/tensorcalls.cpp) give what their Python form gives, and leave it what they do not
know: the same refusals."""
import pytest
import torch

from semi_pd_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def outcome(fn):
    try:
        out = fn()
    except Exception as e:  # noqa: BLE001  (the kind of refusal is what is compared)
        return type(e), str(e)
    return [(t.dtype, t.shape, t.stride(), t.cpu()) for t in (out if isinstance(out, tuple) else (out,))]


def both(monkeypatch, fn):
    assert _lib.tensor_calls is not None
    fast = outcome(fn)
    with monkeypatch.context() as m:
        m.setattr(ops, "tensor_calls", None)
        slow = outcome(fn)
    if isinstance(fast, list) and isinstance(slow, list):
        assert len(fast) == len(slow)
        for a, b in zip(fast, slow):
            assert a[:3] == b[:3] and torch.equal(a[3], b[3])
        return True
    assert fast == slow
    return False


def operands(dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    i = lambda *s: torch.randint(-127, 128, s, generator=g, device=DEV, dtype=torch.int8)  # noqa: E731
    return dict(x=r(5, 128).to(dtype), r=r(5, 128).to(dtype), w=r(128).to(dtype), a=i(5, 128), b=i(24, 128), sa=r(5, 1), sb=r(24), bias=r(24).to(dtype),
                v=r(300, 128).to(dtype), vi=i(300, 128), sv=r(300, 1), t=torch.arange(5, device=DEV))


def test_the_calls_of_every_form(monkeypatch):
    for dtype in (torch.bfloat16, torch.float16):
        o = operands(dtype)
        for fn in (lambda: ops.per_token_quant_int8(o["x"]), lambda: ops.per_token_quant_int8(o["x"][:, 16:48]),
                   lambda: ops.per_token_quant_int8(o["x"][:1]), lambda: ops.per_token_quant_int8(o["x"][:0]),
                   lambda: ops.rmsnorm_quant_int8(o["x"], o["w"], 1e-5), lambda: ops.rmsnorm_quant_int8(o["x"], o["w"], 1),
                   lambda: ops.fused_add_rmsnorm_quant_int8(o["x"], o["r"].clone(), o["w"]), lambda: ops.silu_and_mul_quant_int8(o["x"]),
                   lambda: ops.int8_scaled_mm(o["a"], o["b"].t(), o["sa"], o["sb"], dtype),
                   lambda: ops.int8_scaled_mm(o["a"], o["b"].t(), o["sa"], o["sb"], dtype, o["bias"], older_weight=True),
                   lambda: ops.int8_scaled_mm(o["a"][:, 16:64], o["b"][:, :48].t(), o["sa"], o["sb"], dtype, older_weight=1),
                   lambda: ops.linear_logprobs(o["x"], o["v"], o["t"]), lambda: ops.linear_logprobs(o["x"][:0], o["v"], o["t"][:0]),
                   lambda: ops.linear_logprobs(o["a"], o["vi"], o["t"], o["sa"], o["sv"], older_weight=True)):
            assert both(monkeypatch, fn)


def test_what_is_refused_stays_refused(monkeypatch):
    o = operands()
    bad = torch.bfloat16
    for fn in (lambda: ops.per_token_quant_int8(o["x"].float()), lambda: ops.per_token_quant_int8(o["x"][:, :24]),
               lambda: ops.per_token_quant_int8(o["x"].cpu()), lambda: ops.per_token_quant_int8(None), lambda: ops.per_token_quant_int8(o["x"][0]),
               lambda: ops.rmsnorm_quant_int8(o["x"], o["w"].half()), lambda: ops.rmsnorm_quant_int8(o["x"], o["w"][:64]),
               lambda: ops.fused_add_rmsnorm_quant_int8(o["x"], o["r"][:, ::2], o["w"]),
               lambda: ops.fused_add_rmsnorm_quant_int8(o["x"].t(), o["r"].t(), o["w"]), lambda: ops.silu_and_mul_quant_int8(o["x"][:, :40]),
               lambda: ops.int8_scaled_mm(o["a"], o["b"], o["sa"], o["sb"], bad), lambda: ops.int8_scaled_mm(o["a"], o["b"].t(), o["sa"], o["sb"], torch.float32),
               lambda: ops.int8_scaled_mm(o["a"], o["b"].t(), o["sb"], o["sb"], bad), lambda: ops.int8_scaled_mm(o["a"], o["b"].t(), o["sa"], o["sb"], bad, o["sb"]),
               lambda: ops.int8_scaled_mm(o["a"], o["b"][:20].t(), o["sa"], o["sb"][:20], bad), lambda: ops.int8_scaled_mm(o["a"].cpu(), o["b"].t(), o["sa"], o["sb"], bad),
               lambda: ops.linear_logprobs(o["x"], o["v"], o["t"].int()), lambda: ops.linear_logprobs(o["x"], o["v"].half(), o["t"]),
               lambda: ops.linear_logprobs(o["x"], o["v"], o["t"], o["sa"], o["sv"]), lambda: ops.linear_logprobs(o["a"], o["vi"], o["t"], o["sa"]),
               lambda: ops.linear_logprobs(o["x"], o["v"], o["t"][:3]), lambda: ops.linear_logprobs(o["x"][:, :60], o["v"][:, :60], o["t"])):
        assert not both(monkeypatch, fn)


def test_the_stream_is_the_current_one(monkeypatch):
    """A call under another stream runs on that one: it waits behind what is there, and the default stream's next work does not."""
    x = torch.zeros(64, 4096, device=DEV, dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(int(2e7))
        x.fill_(1)
        q, s = ops.per_token_quant_int8(x)
        x.fill_(3)
    side.synchronize()
    assert (q == 127).all() and torch.allclose(s, torch.full_like(s, 1 / 127))


def test_launches_are_counted():
    o = operands()
    n = _lib._Counter.launches
    ops.per_token_quant_int8(o["x"])
    ops.int8_scaled_mm(o["a"], o["b"].t(), o["sa"], o["sb"], torch.bfloat16)
    ops.linear_logprobs(o["x"], o["v"], o["t"])
    assert _lib._Counter.launches == n + 4
