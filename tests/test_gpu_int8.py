"""Operators of models served in 8-bit integers against their definitions in 64 bits: quantisation by token (alone, behind norms,
behind SiLU * mul) and the product with scales for each token and channel."""
import pytest
import torch

from semi_pd_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def hidden(rows, k, dtype, seed):
    g = gen(seed)
    x = torch.randn(rows, k, generator=g, device=DEV) * torch.exp(torch.randn(rows, 1, generator=g, device=DEV))
    x[:, ::37] *= 8
    return x.to(dtype)


def quantised(y):
    """The definition: scales and integers of y in 64 bits, halves away from zero."""
    top = y.abs().amax(1, keepdim=True).clamp(min=1e-10)
    t = y * 127 / top  # (y / (top / 127) would be rounded twice: off a half that it stands on)
    return torch.sign(t) * torch.floor(t.abs() + 0.5), top / 127


def close_quant(q, s, y, rel):
    """q and s of values known to `rel`: the scale within rel and two roundings of 2^-24, the integers equal where y / s is further
    from a half than those errors move it (and at most one off elsewhere)."""
    want, scale = quantised(y)
    err = rel + 4 * 2.0 ** -24
    assert ((s.double() - scale).abs() <= err * scale).all()
    t = (y / scale).abs()
    near = (t - torch.floor(t) - 0.5).abs() <= 4 * err * (t + 1)
    assert torch.equal(q.double()[~near], want[~near])
    assert ((q.double() - want).abs() <= 1).all()
    assert near.float().mean() < 0.01


SIZES = [(1, 16), (1, 4096), (3, 1024), (5, 1040), (33, 2064), (7, 8192), (2, 14336), (2, 16400), (3, 32768), (700, 256), (1501, 4096), (901, 2064),
         (601, 14336)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", SIZES)
def test_per_token_quant_is_exact(rows, k, dtype):
    x = hidden(rows, k, dtype, rows + k)
    x[0, 1] = x[0, 0] = x[0].abs().max()
    x[0, 2:6] = torch.tensor([0.5, -0.5, 0.25, -0.25], device=DEV, dtype=dtype) * x[0, 0]  # on a half: 63.5
    q, s = ops.per_token_quant_int8(x)
    want, scale = quantised(x.double())
    assert q.shape == (rows, k) and s.shape == (rows, 1) and q.dtype == torch.int8 and s.dtype == torch.float32
    assert torch.equal(q.double(), want)
    assert ((s.double() - scale).abs() <= 2.0 ** -24 * scale).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_per_token_quant_every_ratio_of_two_values(dtype):
    """Every 16-bit value between 0 and 1 below maxima of many significands: halves go away from zero, nothing else moves."""
    bits = torch.arange(0, torch.tensor([1.0], dtype=dtype).view(torch.int16).item() + 1, device=DEV, dtype=torch.int32)
    v = bits.to(torch.int16).view(dtype)
    v = v[v >= 2.0 ** -12]
    v = torch.cat([v, torch.zeros(-v.numel() % 16, device=DEV, dtype=dtype)])
    tops = (1 + torch.arange(0, 2048, 3, device=DEV) / 2048).to(dtype)
    for t in tops.split(256):
        x = torch.cat([v.expand(len(t), -1), t[:, None].expand(-1, 16)], 1).contiguous()
        q, _ = ops.per_token_quant_int8(x)
        assert torch.equal(q.double(), quantised(x.double())[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_per_token_quant_of_strided_rows(dtype):
    x = hidden(9, 1024, dtype, 1)[:, 512:768]
    q, s = ops.per_token_quant_int8(x)
    q2, s2 = ops.per_token_quant_int8(x.contiguous())
    assert torch.equal(q, q2) and torch.equal(s, s2)


@pytest.mark.parametrize("dtype", TYPES)
def test_per_token_quant_of_zeros_infinities_and_nan(dtype):
    x = torch.ones(4, 64, device=DEV, dtype=dtype)
    x[0] = 0
    x[1, 5] = float("inf")
    x[2, 7] = float("nan")
    q, s = ops.per_token_quant_int8(x)
    assert (q[0] == 0).all() and s[0].item() == pytest.approx(1e-10 / 127, rel=1e-6)
    assert s[1].isinf() and s[2].isnan()
    assert (q[3] == 127).all()
    w = torch.ones(8, 64, device=DEV, dtype=torch.int8)
    out = ops.int8_scaled_mm(q, w.t(), s, torch.ones(8, device=DEV), dtype)
    assert out[0].eq(0).all() and not out[1].isfinite().any() and out[2].isnan().all() and out[3].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", SIZES)
def test_rmsnorm_quant(rows, k, dtype):
    x, w = hidden(rows, k, dtype, rows), (1 + 0.1 * torch.randn(k, generator=gen(3), device=DEV)).to(dtype)
    q, s = ops.rmsnorm_quant_int8(x, w, 1e-5)
    v = x.double()
    # the sum of squares in 32 bits: k / 256 additions in a row and 13 levels; its root halves that; five more roundings
    close_quant(q, s, v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5) * w.double(), (k / 512 + 20) * 2.0 ** -24)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", SIZES)
def test_fused_add_rmsnorm_quant(rows, k, dtype):
    x, r = hidden(rows, k, dtype, rows), hidden(rows, k, dtype, rows + 1)
    w = (1 + 0.1 * torch.randn(k, generator=gen(3), device=DEV)).to(dtype)
    kept, total = x.clone(), x.float() + r.float()
    v = x.double() + r.double()
    q, s = ops.fused_add_rmsnorm_quant_int8(x, r, w, 1e-5)
    assert torch.equal(r, total.to(dtype)) and torch.equal(x, kept)
    # as above, and the sum's own rounding relative to it
    close_quant(q, s, v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5) * w.double(), (k / 512 + 22) * 2.0 ** -24)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", SIZES)
def test_silu_and_mul_quant(rows, k, dtype):
    x = hidden(rows, 2 * k, dtype, rows)
    q, s = ops.silu_and_mul_quant_int8(x)
    g, u = x[:, :k].double(), x[:, k:].double()
    # the exponential is good to 2 + 1.2 |g| units of 2^-23 (its argument is rounded at g log2 e), with a largest |g| whose product
    # counts; the quotient and the product two more
    close_quant(q, s, g * torch.sigmoid(g) * u, 64 * 2.0 ** -23)


def int8_rows(rows, k, seed):
    return torch.randint(-128, 128, (rows, k), generator=gen(seed), device=DEV, dtype=torch.int8)


def product(a, b, sa, sb, bias, dtype):
    """The definition in 64 bits and how far fp32 scaling and one rounding may be from it."""
    raw = (a.double() @ b.double().t()) * sa.double().view(-1, 1) * sb.double().view(1, -1)
    want = raw if bias is None else raw + bias.double()
    half = torch.finfo(dtype).eps / 2
    # the sum to fp32, times s_a, times s_b, the addition: 4 roundings of 2^-24; then one of the type (fp16: not below 2^-25)
    tol = want.abs() * half * (1 + 2.0 ** -8) + raw.abs() * 5 * 2.0 ** -24 + 2.0 ** -25
    return want, tol


SHAPES = [(1, 8, 16), (1, 256, 128), (1, 4096, 4096), (2, 136, 144), (17, 264, 1360), (32, 6144, 512), (33, 520, 2064),
          (64, 4096, 1024), (100, 1000, 656), (128, 512, 4096), (129, 2048, 2048), (160, 28672, 256), (200, 4096, 4096),
          (256, 776, 2576), (257, 1000, 144), (300, 128, 1024), (513, 520, 400), (777, 5000, 1360), (1300, 4096, 2048),
          (2050, 264, 16), (1024, 19200, 128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k, dtype):
    a, b = int8_rows(m, k, 1), int8_rows(n, k, 2)
    sa = torch.rand(m, 1, generator=gen(3), device=DEV) * 0.02 / k ** 0.5
    sb = torch.rand(n, 1, generator=gen(4), device=DEV) + 0.1
    bias = torch.randn(n, generator=gen(5), device=DEV).to(dtype) if (m + n) % 16 else None
    out = ops.int8_scaled_mm(a, b.t(), sa, sb, dtype, bias)
    want, tol = product(a, b, sa, sb, bias, dtype)
    assert out.dtype == dtype and out.shape == (m, n)
    bad = (out.double() - want).abs() > tol
    assert not bad.any(), (bad.nonzero()[:4].tolist(), int(bad.sum()))
    assert torch.equal(out, ops.int8_scaled_mm(a, b.t(), sa, sb, dtype, bias, older_weight=True))


@pytest.mark.parametrize("m", [3, 40, 160, 600])
def test_sums_that_need_32_bits_are_exact(m):
    k, n = 131056, 264
    a, b = torch.full((m, k), -128, device=DEV, dtype=torch.int8), torch.full((n, k), -128, device=DEV, dtype=torch.int8)
    b[1] = 127
    a[:, 5] = torch.arange(m, device=DEV).remainder(100).to(torch.int8)
    ones = torch.ones(max(m, n), device=DEV)
    scale = 2.0 ** -20
    out = ops.int8_scaled_mm(a, b.t(), ones[:m] * scale, ones[:n], torch.float16)
    want, tol = product(a, b, ones[:m] * scale, ones[:n], None, torch.float16)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("m", [5, 300])
def test_product_of_strided_operands(m):
    a, b = int8_rows(m, 512, 1)[:, 128:400], int8_rows(264, 1024, 2)[:, 16:288]
    sa, sb = torch.rand(m, device=DEV) * 1e-3, torch.rand(300, device=DEV)[3:267]
    out = ops.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16)
    want, tol = product(a, b, sa, sb, None, torch.bfloat16)
    assert ((out.double() - want).abs() <= tol).all()


def test_product_of_no_tokens():
    out = ops.int8_scaled_mm(int8_rows(0, 64, 1), int8_rows(16, 64, 2).t(), torch.ones(0, device=DEV), torch.ones(16, device=DEV),
                             torch.bfloat16)
    assert out.shape == (0, 16)
    q, s = ops.per_token_quant_int8(torch.empty(0, 64, device=DEV, dtype=torch.bfloat16))
    assert q.shape == (0, 64) and s.shape == (0, 1)


@pytest.mark.parametrize("m", [4, 150, 700])
@pytest.mark.parametrize("sms", [16, 40, 72])
def test_product_within_a_budget_of_sms(m, sms):
    a, b = int8_rows(m, 1040, 1), int8_rows(3000, 1040, 2)
    sa, sb = torch.rand(m, device=DEV) * 1e-3, torch.rand(3000, device=DEV)
    whole = ops.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16)
    ops.set_sm_budget(sms)
    try:
        part = ops.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16)
    finally:
        ops.set_sm_budget(0)
    assert torch.equal(whole, part)


def test_weights_that_the_call_before_writes():
    """Rows quantised right before the product that takes them as its weight (older_weight stays False)."""
    a = int8_rows(8, 4096, 1)
    sa = torch.full((8, 1), 1e-3, device=DEV)
    for seed in range(5):
        w = hidden(6144, 4096, torch.bfloat16, seed)
        torch.cuda.synchronize()
        q, s = ops.per_token_quant_int8(w)
        out = ops.int8_scaled_mm(a, q.t(), sa, s, torch.bfloat16)
        torch.cuda.synchronize()
        want, tol = product(a, q, sa, s, None, torch.bfloat16)
        assert ((out.double() - want).abs() <= tol).all()


def test_run_of_them_captured_and_on_two_streams():
    """Norm, product, SiLU * mul, product as a feed-forward runs them: captured graphs replayed on two streams at once give what the
    calls give."""
    g = gen(1)
    d, i = 1024, 2816
    gate_up, gs = ops.per_token_quant_int8((torch.randn(2 * i, d, generator=g, device=DEV) / 32).bfloat16())
    down, ds = ops.per_token_quant_int8((torch.randn(d, i, generator=g, device=DEV) / 53).bfloat16())
    norm = torch.ones(d, device=DEV, dtype=torch.bfloat16)

    def forward(x, r):
        q, s = ops.fused_add_rmsnorm_quant_int8(x, r, norm, 1e-5)
        h = ops.int8_scaled_mm(q, gate_up.t(), s, gs, torch.bfloat16, older_weight=True)
        q, s = ops.silu_and_mul_quant_int8(h)
        return ops.int8_scaled_mm(q, down.t(), s, ds, torch.bfloat16, older_weight=True)

    runs = []
    for m in (24, 300):
        x, r = hidden(m, d, torch.bfloat16, m), hidden(m, d, torch.bfloat16, m + 1)
        keep = r.clone()
        want = forward(x, r)
        r.copy_(keep)
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            out = forward(x, r)
        runs.append((graph, stream, out, want, r, keep, x))
    for _ in range(20):
        for graph, stream, out, want, r, keep, _ in runs:
            with torch.cuda.stream(stream):
                r.copy_(keep)
                graph.replay()
        torch.cuda.synchronize()
        for _, _, out, want, *_ in runs:
            assert torch.equal(out, want)


def test_refusals():
    a, b, x = int8_rows(4, 64, 1), int8_rows(16, 64, 2), torch.ones(4, 64, device=DEV, dtype=torch.bfloat16)
    s4, s16 = torch.ones(4, device=DEV), torch.ones(16, device=DEV)
    for args, kw in [((a, b, s4, s16, torch.bfloat16), {}), ((a.t(), b.t(), s4, s16, torch.bfloat16), {}),
                     ((a, b.t(), s16, s16, torch.bfloat16), {}), ((a, b.t(), s4, s4, torch.bfloat16), {}),
                     ((a, b.t(), s4.double(), s16, torch.bfloat16), {}), ((a, b.t(), s4, s16, torch.float32), {}),
                     ((x, b.t(), s4, s16, torch.bfloat16), {}), ((a, b.t(), s4, s16, torch.bfloat16), dict(bias=s16)),
                     ((a, b.t(), s4, s16, torch.bfloat16), dict(bias=s16[:8].bfloat16())), ((a[0], b.t(), s4, s16, torch.bfloat16), {}),
                     ((a[:, :56], b[:, :56].t(), s4, s16, torch.bfloat16), {}), ((a, b[:12].t(), s4, s16[:12], torch.bfloat16), {}),
                     ((a[:, 1:33], b[:, :32].t(), s4, s16, torch.bfloat16), {}), ((a, b.t(), s4, s16.cpu(), torch.bfloat16), {})]:
        with pytest.raises(RuntimeError):
            ops.int8_scaled_mm(*args, **kw)
    w = x[0].contiguous()
    for fn, args in [(ops.per_token_quant_int8, (x.float(),)), (ops.per_token_quant_int8, (x[0],)), (ops.per_token_quant_int8, (x.t(),)),
                     (ops.per_token_quant_int8, (x[:, :24],)), (ops.per_token_quant_int8, (x[:, 1:33],)), (ops.rmsnorm_quant_int8, (x, w.half())),
                     (ops.rmsnorm_quant_int8, (x, w[:32])), (ops.fused_add_rmsnorm_quant_int8, (x, x[:2], w)),
                     (ops.fused_add_rmsnorm_quant_int8, (x, x.half(), w)), (ops.silu_and_mul_quant_int8, (x[:, :40],)),
                     (ops.silu_and_mul_quant_int8, (x[:, :33],))]:
        with pytest.raises(RuntimeError):
            fn(*args)


def test_dispatcher_op():
    import semi_pd_b200.torch_ops  # noqa: F401
    a, b = int8_rows(4, 64, 1), int8_rows(16, 64, 2)
    sa, sb, bias = torch.rand(4, 1, device=DEV), torch.rand(16, 1, device=DEV), torch.ones(16, device=DEV, dtype=torch.float16)
    for kw in (None, bias):
        assert torch.equal(torch.ops.spd.int8_scaled_mm(a, b.t(), sa, sb, torch.float16, kw), ops.int8_scaled_mm(a, b.t(), sa, sb, torch.float16, kw))


@pytest.mark.parametrize("k", [1024, 4096, 14336])
def test_rows_do_not_depend_on_their_number(k):
    """A CTA a row and CTAs that take one row after another give the same bits, on the whole device and on a part of it."""
    x, r = hidden(2000, 2 * k, torch.bfloat16, 1), hidden(2000, k, torch.bfloat16, 2)
    w = (1 + 0.1 * torch.randn(k, generator=gen(3), device=DEV)).bfloat16()
    n = x[:, :k].contiguous()
    forms = [lambda m: ops.silu_and_mul_quant_int8(x[:m]), lambda m: ops.rmsnorm_quant_int8(n[:m], w),
             lambda m: ops.fused_add_rmsnorm_quant_int8(n[:m], r[:m].clone(), w)]
    for form in forms:
        q, s = form(2000)
        for m, sms in ((1, 0), (100, 0), (777, 0), (1999, 0), (2000, 40), (300, 16)):
            ops.set_sm_budget(sms)
            try:
                q2, s2 = form(m)
            finally:
                ops.set_sm_budget(0)
            assert torch.equal(q[:m], q2) and torch.equal(s[:m], s2)


@pytest.mark.parametrize("m,n", [(70000, 32768), (200, 11000000)])
def test_offsets_beyond_32_bits(m, n):
    """Outputs of more than 2^31 elements: the last rows and columns are where they belong."""
    a, b = int8_rows(m, 16, 1), int8_rows(n, 16, 2)
    sa, sb = torch.rand(m, device=DEV), torch.rand(n, device=DEV)
    out = ops.int8_scaled_mm(a, b.t(), sa, sb, torch.float16)
    assert out.numel() > 2 ** 31
    for r in (slice(0, 3), slice(m // 2, m // 2 + 3), slice(m - 3, m)):
        for c in (slice(0, 300), slice(n // 2, n // 2 + 300), slice(n - 300, n)):
            want, tol = product(a[r], b[c], sa[r], sb[c], None, torch.float16)
            fits = want.abs() < 65000  # (fp16 overflows beyond)
            assert (((out[r, c].double() - want).abs() <= tol) | ~fits).all()
    del out
    torch.cuda.empty_cache()


def test_quant_of_more_than_32_bits_of_elements():
    x = torch.empty(70000, 32768, device=DEV, dtype=torch.bfloat16)
    for part in x.split(10000):
        part.normal_()
    q, s = ops.per_token_quant_int8(x)
    for r in (slice(0, 2), slice(65000, 65002), slice(69998, 70000)):
        want, scale = quantised(x[r].double())
        assert torch.equal(q[r].double(), want)
    w = torch.ones(32768, device=DEV, dtype=torch.bfloat16)
    q2, s2 = ops.rmsnorm_quant_int8(x, w, 1e-5)
    for r in (slice(0, 2), slice(69998, 70000)):
        v = x[r].double()
        close_quant(q2[r], s2[r], v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5), (32768 / 512 + 20) * 2.0 ** -24)
    del x, q, q2
    torch.cuda.empty_cache()


def test_behind_a_long_kernel():
    """Waits inside a product start when the kernel before it is done, whatever that takes."""
    a, b = int8_rows(8, 1024, 1), int8_rows(512, 1024, 2)
    sa, sb = torch.rand(8, device=DEV), torch.rand(512, device=DEV)
    want = ops.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16)
    torch.cuda.synchronize()
    torch.cuda._sleep(int(4e9))
    out = ops.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16, older_weight=True)
    q, s = ops.per_token_quant_int8(out)
    out2 = ops.int8_scaled_mm(q, int8_rows(64, 512, 3).t(), s, sb[:64], torch.bfloat16, older_weight=True)
    torch.cuda.synchronize()
    ops.check_waits()
    assert torch.equal(out, want) and out2.isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1700, 8200, 528), (5000, 4104, 16), (600, 24008, 4096), (4100, 10248, 1040)])
def test_product_of_many_tiles(m, n, k, dtype):
    # (more tiles than pairs of CTAs, ragged at both edges; 24008 x 4096: three panels of weights, the last one narrower)
    a, b = int8_rows(m, k, 21), int8_rows(n, k, 22)
    sa = torch.rand(m, 1, generator=gen(23), device=DEV) * 0.02 / k ** 0.5
    sb = torch.rand(n, 1, generator=gen(24), device=DEV) + 0.1
    bias = torch.randn(n, generator=gen(25), device=DEV).to(dtype)
    for b_ in (bias, None):
        out = ops.int8_scaled_mm(a, b.t(), sa, sb, dtype, b_)
        want, tol = product(a, b, sa, sb, b_, dtype)
        assert ((out.double() - want).abs() <= tol).all()
        for _ in range(3):
            assert torch.equal(out, ops.int8_scaled_mm(a, b.t(), sa, sb, dtype, b_))


@pytest.mark.parametrize("m,n,k", [(5, 264, 144), (150, 1000, 528), (700, 1000, 144), (2100, 4104, 528)])
def test_results_inside_a_wider_buffer(m, n, k):
    # (a caller of the library: what is beside and behind the results stays as it was)
    from semi_pd_b200 import _lib
    a, b = int8_rows(m, k, 31), int8_rows(n, k, 32)
    sa = torch.rand(m, 1, generator=gen(33), device=DEV) * 0.02 / k ** 0.5
    sb = torch.rand(n, 1, generator=gen(34), device=DEV) + 0.1
    buf = torch.full((m + 3, n + 24), 77.0, device=DEV, dtype=torch.bfloat16)
    _lib.check(_lib.lib.spd_int8_scaled_mm(buf[1:, 8:].data_ptr(), a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), None, m, n, k, k, k,
                                           n + 24, 0, 0, 0, torch.cuda.current_stream().cuda_stream), "spd_int8_scaled_mm")
    assert torch.equal(buf[1:m + 1, 8:n + 8], ops.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16))
    buf[1:m + 1, 8:n + 8] = 77.0
    assert (buf == 77.0).all()


@pytest.mark.parametrize("k", [48, 528])
def test_integer_results_are_exact(k):
    # (scales of 1 and sums below 2^11: every result is a number of both types; each of the forms)
    for m, n in ((3, 512), (180, 2056), (900, 8200), (2500, 4104)):
        g = gen(m)
        a = torch.randint(-1, 2, (m, k), generator=g, device=DEV, dtype=torch.int8)
        b = torch.randint(-1, 2, (n, k), generator=g, device=DEV, dtype=torch.int8)
        a[:, k // 2:] = 0
        b[:, 256:] = 0  # at most 256 products of 1: exact in bf16
        one_a, one_b = torch.ones(m, 1, device=DEV), torch.ones(n, 1, device=DEV)
        assert torch.equal(ops.int8_scaled_mm(a, b.t(), one_a, one_b, torch.bfloat16).double(), a.double() @ b.double().t())


@pytest.mark.parametrize("sms", [0, 8, 72])
@pytest.mark.parametrize("m,n,k", [(1, 40008, 528), (3, 60000, 144), (100, 80024, 272), (250, 39000, 1040)])
def test_more_weight_tiles_than_run_at_once(m, n, k, sms):
    a, b = int8_rows(m, k, 41), int8_rows(n, k, 42)
    sa = torch.rand(m, 1, generator=gen(43), device=DEV) * 0.02 / k ** 0.5
    sb = torch.rand(n, 1, generator=gen(44), device=DEV) + 0.1
    bias = torch.randn(n, generator=gen(45), device=DEV).bfloat16()
    ops.set_sm_budget(sms)
    try:
        outs = [ops.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16, bias, older_weight=older) for older in (False, True, True)]
    finally:
        ops.set_sm_budget(0)
    want, tol = product(a, b, sa, sb, bias, torch.bfloat16)
    for out in outs:
        assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("m,n,k", [(2, 8, 60000), (1, 136, 131056), (40, 264, 30000), (200, 520, 40016)])
def test_long_rows_of_few_columns(m, n, k):
    # (far more k-blocks than the rings hold, and CTAs whose weight rows are all behind the last)
    a, b = int8_rows(m, k, 51), int8_rows(n, k, 52)
    sa = torch.rand(m, 1, generator=gen(53), device=DEV) * 0.02 / k ** 0.5
    sb = torch.rand(n, 1, generator=gen(54), device=DEV) + 0.1
    for older in (True, False):
        out = ops.int8_scaled_mm(a, b.t(), sa, sb, torch.bfloat16, older_weight=older)
        want, tol = product(a, b, sa, sb, None, torch.bfloat16)
        assert ((out.double() - want).abs() <= tol).all()
