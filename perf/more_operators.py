"""What the operators of models served in 8-bit integers are measured on: the quantisation of activations by token, alone and in
one pass with the norm or the activation before it, the product with 8-bit weights, and the log-probabilities of given tokens
from the last product, 16-bit or 8-bit, without its logits.

A case is a dict of plain values; its "op" says what it runs:

  product      ops.int8_scaled_mm: tokens times a layer's weights
  quant        ops.per_token_quant_int8: what a product takes
  norm_linear  ops.fused_add_rmsnorm_quant_int8 (ops.rmsnorm_quant_int8 without a residual), then the product
  act_linear   ops.silu_and_mul_quant_int8, then the product
  score        ops.linear_logprobs: log-softmax over the vocabulary at one token per row

`own` False computes a case in plain torch operations, True through the framework.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5
PIECE = 16384  # vocabulary rows whose logits the plain form holds at a time


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one request decodes: the projections of its query, key and value
        dict(name="product_1", op="product", dtype="bfloat16", tokens=1, n=6144, k=4096, bias=False),
        # a decode batch through a down projection: long rows, few of them
        dict(name="product_40_long_k", op="product", dtype="float16", tokens=40, n=4096, k=14336, bias=True),
        # a large decode batch through gate and up projections
        dict(name="product_160", op="product", dtype="bfloat16", tokens=160, n=28672, k=4096, bias=False),
        # a short prefill batch through a layer whose sizes fill no tile
        dict(name="product_777_ragged", op="product", dtype="float16", tokens=777, n=5000, k=1360, bias=True),
        # a whole prefill batch through gate and up projections
        dict(name="product_8192", op="product", dtype="bfloat16", tokens=8192, n=28672, k=4096, bias=False),
        # the output of attention before its projection: a prefill batch on a wide model
        dict(name="quant_5001", op="quant", dtype="float16", tokens=5001, k=8192),
        # a decode batch enters a layer
        dict(name="norm_linear_24", op="norm_linear", dtype="bfloat16", tokens=24, n=6144, k=4096, residual=True),
        # a prefill batch enters a layer
        dict(name="norm_linear_4099", op="norm_linear", dtype="float16", tokens=4099, n=6144, k=4096, residual=True),
        # a prefill batch leaves a feed-forward
        dict(name="act_linear_1300", op="act_linear", dtype="bfloat16", tokens=1300, n=4096, k=14336),
        # the log-probability of the token that one request has just chosen
        dict(name="score_1", op="score", dtype="bfloat16", tokens=1, n=128256, k=4096, int8=False, ignored=0.0),
        # the log-probabilities of a prompt's own tokens
        dict(name="score_500", op="score", dtype="float16", tokens=500, n=102400, k=2048, int8=False, ignored=0.1),
        # the same of a long prompt through an 8-bit last product
        dict(name="score_2047_int8", op="score", dtype="bfloat16", tokens=2047, n=128256, k=4096, int8=True, ignored=0.1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["product", "product", "quant", "norm_linear", "act_linear", "score"])
    case = dict(op=op, dtype=rng.choice(["bfloat16", "float16"]))
    if op == "quant":
        return dict(case, tokens=_log(rng, 1, 8192), k=16 * _log(rng, 2, 1792))
    while True:
        tokens, n, k = _log(rng, 1, 8192), 8 * _log(rng, 8, 3584), 16 * _log(rng, 8, 896)
        if op == "score":
            case = dict(case, tokens=min(tokens, 2047), n=8 * _log(rng, 125, 16032), k=k, int8=rng.random() < 0.4,
                        ignored=rng.choice([0.0, 0.1, 0.5]))
        elif op == "product":
            case = dict(case, tokens=tokens, n=n, k=k, bias=rng.random() < 0.5)
        elif op == "norm_linear":
            case = dict(case, tokens=tokens, n=n, k=k, residual=rng.random() < 0.7)
        else:
            case = dict(case, tokens=tokens, n=n, k=k)
        if case["k"] * case["n"] <= 4096 * 128256 and case["tokens"] * case["n"] * case["k"] <= 8192 * 28672 * 4096:
            return case


def work(case):
    m, k, size = case["tokens"], case["k"], 2
    if case["op"] == "quant":
        return {"bytes": m * (k * (size + 1) + 4), "flops": 4 * m * k}
    n = case["n"]
    flops = 2 * m * n * k
    if case["op"] == "score":
        cell = 1 if case["int8"] else size
        return {"bytes": (m + n) * (k * cell + (4 if case["int8"] else 0)) + m * (8 + 8), "flops": flops + 4 * m * n}
    moved = n * (k + 4) + m * n * size
    if case["op"] == "product":
        return {"bytes": moved + m * (k + 4) + (n * size if case["bias"] else 0), "flops": flops}
    if case["op"] == "norm_linear":
        return {"bytes": moved + k * size + m * k * size * (3 if case["residual"] else 1), "flops": flops + 8 * m * k}
    return {"bytes": moved + 2 * m * k * size, "flops": flops + 12 * m * k}


# ---------------------------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------------------------
def _hidden(rows, k, g, dtype):
    """Activations: tokens of different size, and a few channels that are far larger than the others in every token."""
    x = torch.randn(rows, k, generator=g, device=DEV)
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=g, device=DEV))
    loud = torch.randint(0, k, (max(1, k // 256),), generator=g, device=DEV)
    x[:, loud] *= 8
    return x.to(dtype)


def _int8(rows, k, g):
    """What a token's or a channel's numbers look like in 8 bits, the largest of each row 127."""
    q = (torch.randn(rows, k, generator=g, device=DEV) * 32).round_().clamp_(-127, 127).to(torch.int8)
    q[torch.arange(rows, device=DEV), torch.randint(0, k, (rows,), generator=g, device=DEV)] = 127
    return q


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype, m, k, op = DTYPES[case["dtype"]], case["tokens"], case["k"], case["op"]
    st = dict(case=case)
    if op == "quant":
        return dict(st, x=_hidden(m, k, g, dtype))
    n = case["n"]
    if op == "score":
        if case["int8"]:
            # the sizes of logits: about 2
            st.update(x=_int8(m, k, g), w=_int8(n, k, g),
                      xs=torch.rand(m, 1, generator=g, device=DEV) * 0.04 + 0.02,
                      ws=(torch.rand(n, 1, generator=g, device=DEV) * 0.6 + 0.7) * (2.0 / (0.04 * 1024 * math.sqrt(k))))
        else:
            st.update(x=torch.randn(m, k, generator=g, device=DEV).to(dtype),
                      w=(torch.randn(n, k, generator=g, device=DEV) * (2.0 / math.sqrt(k))).to(dtype))
        targets = torch.randint(0, n, (m,), generator=g, device=DEV)
        targets[torch.rand(m, generator=g, device=DEV) < case["ignored"]] = -1  # tokens that nothing is asked of
        return dict(st, targets=targets)
    # a layer's weight in 8 bits, [n, k] with a scale for each of its rows
    st.update(w=_int8(n, k, g), ws=(torch.rand(n, 1, generator=g, device=DEV) + 0.5) / (32 * math.sqrt(k)))
    if op == "product":
        st.update(x=_int8(m, k, g), xs=torch.rand(m, 1, generator=g, device=DEV) * 0.04 + 0.01,
                  bias=torch.randn(n, generator=g, device=DEV).to(dtype) if case["bias"] else None)
    elif op == "norm_linear":
        st.update(x=_hidden(m, k, g, dtype), norm=(1 + 0.1 * torch.randn(k, generator=g, device=DEV)).to(dtype),
                  residual=_hidden(m, k, g, dtype) if case["residual"] else None)
    else:
        st.update(x=_hidden(m, 2 * k, g, dtype))
    return st


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _plain_quant(y):
    """8-bit integers and a scale for each row.  A value half way between two integers goes away from zero; the quotient is
    taken in 64 bits, for it stands next to that border."""
    top = y.abs().amax(-1, keepdim=True).float().clamp(min=1e-10)
    t = y.double() * 127 / top.double()
    return (t.abs() + 0.5).floor().mul(t.sign()).to(torch.int8), top / 127


def _plain_product(x, w, xs, ws, bias, dtype):
    out = x.float() @ w.float().t() * xs * ws.t()
    return (out if bias is None else out + bias.float()).to(dtype)


def _plain_score(st):
    x, w, n = st["x"].float(), st["w"], st["case"]["n"]
    rows = torch.arange(len(x), device=x.device)
    target = st["targets"]
    top = torch.full((len(x), 1), -math.inf, device=x.device)
    total = torch.zeros(len(x), 1, device=x.device)
    at_target = torch.zeros(len(x), device=x.device)
    for a in range(0, n, PIECE):
        b = min(n, a + PIECE)
        logits = x @ w[a:b].float().t()
        if st["case"]["int8"]:
            logits = logits * st["xs"] * st["ws"][a:b].t()
        new = torch.maximum(top, logits.amax(-1, keepdim=True))
        total = total * torch.exp(top - new) + torch.exp(logits - new).sum(-1, keepdim=True)
        top = new
        here = (target >= a) & (target < b)
        at_target = torch.where(here, logits[rows, (target - a).clamp(0, b - a - 1)], at_target)
    lse = (top + torch.log(total)).squeeze(1)
    return torch.where(target >= 0, at_target - lse, torch.zeros_like(lse)), lse


def _plain(st):
    case = st["case"]
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op == "product":
        return _plain_product(st["x"], st["w"], st["xs"], st["ws"], st["bias"], dtype)
    if op == "quant":
        return _plain_quant(st["x"])
    if op == "score":
        return _plain_score(st)
    y = st["x"].float()
    out = []
    if op == "norm_linear":
        if st["residual"] is not None:
            y = y + st["residual"].float()
            st["residual"].copy_(y)
            out.append(st["residual"])
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * st["norm"].float()
    else:
        gate, up = y.chunk(2, -1)
        y = gate / (1 + torch.exp(-gate)) * up
    q, s = _plain_quant(y)
    return [_plain_product(q, st["w"], s, st["ws"], None, dtype)] + out


def run(state):
    if not own:
        return _plain(state)
    from semi_pd_b200 import ops
    case = state["case"]
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op == "product":
        return ops.int8_scaled_mm(state["x"], state["w"].t(), state["xs"], state["ws"], dtype, state["bias"], older_weight=True)
    if op == "quant":
        return ops.per_token_quant_int8(state["x"])
    if op == "score":
        return ops.linear_logprobs(state["x"], state["w"], state["targets"], state.get("xs"), state.get("ws"), older_weight=True)
    if op == "act_linear":
        q, s = ops.silu_and_mul_quant_int8(state["x"])
        return [ops.int8_scaled_mm(q, state["w"].t(), s, state["ws"], dtype, older_weight=True)]
    if state["residual"] is None:
        q, s = ops.rmsnorm_quant_int8(state["x"], state["norm"], EPS)
        return [ops.int8_scaled_mm(q, state["w"].t(), s, state["ws"], dtype, older_weight=True)]
    q, s = ops.fused_add_rmsnorm_quant_int8(state["x"], state["residual"], state["norm"], EPS)
    return [ops.int8_scaled_mm(q, state["w"].t(), s, state["ws"], dtype, older_weight=True), state["residual"]]


# ---------------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------
def _rows(m, n):
    """Rows at a time whose outputs take a gigabyte."""
    return max(1, (1 << 27) // max(n, 1)) if m else 1


def exact(case, seed):
    st = prepare(case, seed)
    op, m = case["op"], case["tokens"]

    def quantised(y):
        scale = torch.clamp(y.abs().amax(1, keepdim=True), min=1e-10) / 127
        t = y / scale
        return torch.sign(t) * torch.floor(torch.abs(t) + 0.5), scale

    if op == "quant":
        return None, quantised(st["x"].double())[1]
    wide = st["w"].double()
    if op == "score":
        if case["int8"]:
            wide *= st["ws"].double()
        lse, score = [], []
        for a in range(0, m, _rows(m, case["n"])):
            x = st["x"][a:a + _rows(m, case["n"])].double()
            if case["int8"]:
                x = x * st["xs"][a:a + len(x)].double()
            logits = x @ wide.t()
            t = st["targets"][a:a + len(x)]
            z = torch.logsumexp(logits, 1)
            lse.append(z)
            score.append((logits.gather(1, t.clamp(min=0)[:, None])[:, 0] - z) * (t >= 0))
        return torch.cat(score), torch.cat(lse)
    wide *= st["ws"].double()
    if op == "product":
        y, scale = st["x"].double(), st["xs"].double()
    elif op == "act_linear":
        gate, up = st["x"][:, :case["k"]].double(), st["x"][:, case["k"]:].double()
        y, scale = quantised(gate * torch.sigmoid(gate) * up)
    else:
        y = st["x"].double()
        if case["residual"]:
            y = y + st["residual"].double()
        kept = y.to(DTYPES[case["dtype"]]).double()
        y, scale = quantised(y / torch.sqrt((y * y).mean(1, keepdim=True) + EPS) * st["norm"].double())
    step = _rows(m, case["n"])
    out = torch.cat([(y[a:a + step] * scale[a:a + step]) @ wide.t() for a in range(0, m, step)])
    if op == "product":
        return out if st["bias"] is None else out + st["bias"].double()
    return [out, kept] if op == "norm_linear" and case["residual"] else [out]
