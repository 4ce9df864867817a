"""linear_logprobs against log-softmax in 64 bits."""
import pytest
import torch

from semi_pd_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def operands(m, v, k, dtype, seed=1):
    g = gen(seed)
    if dtype == torch.int8:
        x = torch.randint(-128, 128, (m, k), generator=g, device=DEV, dtype=torch.int8)
        w = torch.randint(-128, 128, (v, k), generator=g, device=DEV, dtype=torch.int8)
        xs = torch.rand(m, 1, generator=g, device=DEV) + 0.5
        ws = (torch.rand(v, 1, generator=g, device=DEV) + 0.5) * 3e-4 / k ** 0.5
        return x, w, xs, ws
    x = torch.randn(m, k, generator=g, device=DEV).to(dtype)
    w = (torch.randn(v, k, generator=g, device=DEV) * 2 / k ** 0.5).to(dtype)
    return x, w, None, None


def check(x, w, xs, ws, targets, got, older=False):
    lp, lse = got
    xd, wd = x.double(), w.double()
    if xs is not None:
        xd, wd = xd * xs.double().view(-1, 1), wd * ws.double().view(-1, 1)
    logits = xd @ wd.t()
    want = torch.logsumexp(logits, 1)
    # A logit of 16-bit operands: exact products, added up in K / 16 steps that each may lose 2^-23 of what has come together; of
    # 8-bit ones: an exact sum, three roundings.
    if xs is None:
        dl = ((xd.abs() @ wd.abs().t()) * (x.shape[1] / 16 + 4) * 2.0 ** -23).amax(1)
    else:
        dl = logits.abs().amax(1) * 3 * 2.0 ** -24
    # An exponential 2^-22, its argument 2^-24 of up to 1.45 (max - min), the sums of a tile 2^-24 for each of 36 steps, the join's
    # 20 steps of the same and the exponentials in it; the logarithm's value 2 roundings.
    spread = logits.amax(1) - logits.amin(1)
    tol = dl + 2.0 ** -22 * 20 + spread * 2.0 ** -23 + 60 * 2.0 ** -24 + (want.abs() + logits.abs().amax(1)) * 3 * 2.0 ** -24
    assert lp.dtype == lse.dtype == torch.float32 and lp.shape == lse.shape == (x.shape[0],)
    assert ((lse.double() - want).abs() <= tol).all(), ((lse.double() - want).abs() - tol).max()
    asked = (targets >= 0) & (targets < w.shape[0])
    rows = torch.arange(len(x), device=DEV)
    ref = logits[rows, targets.clamp(0, w.shape[0] - 1)] - want
    assert ((lp.double() - ref).abs() <= tol + dl + ref.abs() * 2.0 ** -24)[asked].all()
    assert (lp[~asked] == 0).all()


SHAPES = [(1, 1, 16), (1, 8, 64), (1, 1000, 512), (1, 32000, 2048), (3, 255, 128), (2, 257, 144), (31, 1024, 256), (33, 5001, 256),
          (64, 8192, 1024), (130, 999, 400), (256, 12803, 128), (257, 300, 1024), (300, 32001, 256), (700, 1024, 2048), (513, 129, 16),
          (1025, 50272, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.int8])
@pytest.mark.parametrize("m,v,k", SHAPES)
def test_logprobs(m, v, k, dtype):
    x, w, xs, ws = operands(m, v, k, dtype)
    targets = torch.randint(0, v, (m,), generator=gen(2), device=DEV)
    targets[::5] = -1
    targets[3::7] = v
    targets[1::9] = 0
    targets[2::9] = v - 1
    got = ops.linear_logprobs(x, w, targets, xs, ws)
    check(x, w, xs, ws, targets, got)
    again = ops.linear_logprobs(x, w, targets, xs, ws, older_weight=True)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("m", [5, 300])
def test_large_logits(m):
    """Logits of some thousands: one token has all of the probability, its own logprob is next to 0."""
    x, w, _, _ = operands(m, 3000, 256, torch.bfloat16)
    x = (x.float() * 1000).bfloat16()
    targets = (x.double() @ w.double().t()).argmax(1)
    check(x, w, None, None, targets, ops.linear_logprobs(x, w, targets))


@pytest.mark.parametrize("m", [5, 300])
def test_infinite_logits(m):
    """-inf logits weigh nothing, rows of nothing else are -inf, +inf is inf, NaN shows."""
    v, k = 1000, 64
    x, w = torch.ones(m, k, device=DEV, dtype=torch.bfloat16), torch.zeros(v, k, device=DEV, dtype=torch.bfloat16)
    w[:, 0] = torch.randn(v, generator=gen(1), device=DEV).bfloat16()
    w[::3, 1] = float("-inf")
    targets = torch.arange(m, device=DEV) % v
    lp, lse = ops.linear_logprobs(x, w, targets)
    logits = x.double() @ w.double().t()
    assert torch.allclose(lse.double(), torch.logsumexp(logits, 1), atol=1e-5)
    assert (lp[::3] == float("-inf")).all() and lp[1::3].isfinite().all()
    w[:, 1] = float("-inf")
    assert (ops.linear_logprobs(x, w, targets)[1] == float("-inf")).all()
    w[:, 1] = 0
    w[700, 1] = float("inf")
    lp, lse = ops.linear_logprobs(x, w, targets)
    assert (lse == float("inf")).all()
    w[700, 1] = float("nan")
    lp, lse = ops.linear_logprobs(x, w, targets)
    assert lse.isnan().all() and lp.isnan().all()


@pytest.mark.parametrize("m", [2, 400])
def test_strided_rows(m):
    x, w, _, _ = operands(m, 700, 512, torch.float16)
    targets = torch.arange(m, device=DEV)
    a, b = x[:, 64:320], w[:, 128:384]
    check(a, b, None, None, targets, ops.linear_logprobs(a, b, targets))


def test_no_rows():
    lp, lse = ops.linear_logprobs(torch.empty(0, 64, device=DEV, dtype=torch.float16), torch.ones(10, 64, device=DEV, dtype=torch.float16),
                                  torch.empty(0, device=DEV, dtype=torch.int64))
    assert lp.shape == lse.shape == (0,)


@pytest.mark.parametrize("m", [4, 300])
def test_budget_of_sms_and_graphs(m):
    x, w, _, _ = operands(m, 20000, 512, torch.bfloat16)
    targets = torch.arange(m, device=DEV) * 31
    want = ops.linear_logprobs(x, w, targets)
    ops.set_sm_budget(40)
    try:
        part = ops.linear_logprobs(x, w, targets)
    finally:
        ops.set_sm_budget(0)
    # a partition may cut the vocabulary into other tiles, whose sums are rounded in another order: held to the definition, as the
    # whole device's are
    check(x, w, None, None, targets, want)
    check(x, w, None, None, targets, part)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.linear_logprobs(x, w, targets)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(want[0], out[0]) and torch.equal(want[1], out[1])


def test_refusals():
    x, w, _, _ = operands(4, 50, 64, torch.bfloat16)
    xi, wi, xs, ws = operands(4, 50, 64, torch.int8)
    t = torch.zeros(4, device=DEV, dtype=torch.int64)
    for args in [(x, w.half(), t), (x, w[:, :32], t), (x, w, t.int()), (x, w, t[:3]), (x, w, t[:, None]), (x.t(), w, t), (x, w, t.cpu()),
                 (x, w, t, xs, ws), (xi, wi, t), (xi, wi, t, xs), (xi, wi, t, xs, ws[:40]), (xi, wi, t, xs.half(), ws), (x.float(), w.float(), t),
                 (x[:, :60], w[:, :60], t), (x[:, 1:33], w[:, :32], t), (xi[:, :56], wi[:, :56], t, xs, ws)]:
        with pytest.raises(RuntimeError):
            ops.linear_logprobs(*args)


def test_two_streams_at_once():
    """Calls of both forms on two streams beside one another, each with a workspace of its own."""
    sets = []
    for m, v, k, dtype in ((16, 30000, 1024, torch.bfloat16), (400, 20000, 512, torch.float16), (64, 30000, 1024, torch.int8)):
        x, w, xs, ws = operands(m, v, k, dtype)
        t = torch.arange(m, device=DEV) * 7
        sets.append((x, w, t, xs, ws, ops.linear_logprobs(x, w, t, xs, ws)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(30):
        with torch.cuda.stream(streams[i % 2]):
            got.append([ops.linear_logprobs(*s[:5]) for s in sets[i % 2:] + sets[:i % 2]])
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for (lp, lse), s in zip(outs, sets[i % 2:] + sets[:i % 2]):
            assert torch.equal(lp, s[5][0]) and torch.equal(lse, s[5][1])


def test_beside_products_of_few_values():
    # (CTAs with one k-block in their ring and 32 columns of TMEM, on the SMs of CTAs that take all columns)
    g = gen(40)
    a = torch.randint(-127, 128, (8, 128), generator=g, device=DEV, dtype=torch.int8)
    b = torch.randint(-127, 128, (8192, 128), generator=g, device=DEV, dtype=torch.int8)
    sa, sb = torch.rand(8, 1, generator=g, device=DEV), torch.rand(8192, 1, generator=g, device=DEV)
    x, w, _, _ = operands(600, 32000, 2048, torch.bfloat16)
    targets = torch.randint(0, 32000, (600,), generator=g, device=DEV)
    want_product = ops.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16)
    want = ops.linear_logprobs(x, w, targets)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    products, scores = [], []
    for _ in range(20):
        with torch.cuda.stream(one):
            scores.append(ops.linear_logprobs(x, w, targets))
        with torch.cuda.stream(two):
            products += [ops.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(p, want_product) for p in products)
    assert all(torch.equal(s[0], want[0]) and torch.equal(s[1], want[1]) for s in scores)
