"""attn_decode_shared: groups of requests over the same leading slots, against softmax attention in 64 bits.

The bound: with u half a step of the type, the weights p are rounded to p (1 + d), |d| <= u, in the products and in their sum
alike, so out moves by at most u / (1 - u) * sum p |v - out| / sum p; in fp16 weights below 2^-14 of the largest are rounded by
2^-25 of it each; the result is rounded once more.  Scores and sums are held in 32 bits: 1e-4 of the same sum covers them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128


def make_case(groups, alone=(), hq=8, hk=2, dtype=torch.bfloat16, seed=0, scattered=False, aligned=True, run=128):
    """groups: (shared tokens, [tokens behind them of every member]); alone: lengths of requests in no group, behind the rest.
    aligned: a member's own tokens begin in a run of their own, the shared ones' last run left as it is."""
    g = torch.Generator().manual_seed(seed)
    rows, lens, shared, indptr = [], [], [], [0]
    need = sum(-(-s // run) + sum(-(-t // run) + 1 for t in own) for s, own in groups) + sum(-(-n // run) for n in alone) + 1
    order = torch.randperm(need, generator=g)
    size = need * run + 1
    perm = torch.cat([torch.zeros(1, dtype=torch.int64), 1 + torch.randperm(size - 1, generator=g)])
    at = 0

    def take(n):
        nonlocal at
        pos = torch.arange(n)
        runs = order[at:at + -(-n // run)]
        at += len(runs)
        s = runs[pos // run] * run + 1 + pos % run if n else pos
        return perm[s] if scattered else s

    for s, own in groups:
        front = take(s)
        for t in own:
            if not aligned and s % run:  # as a fork leaves it: the last, partial run goes on
                pos = torch.arange(s % run, s % run + t)
                runs = order[at:at + -(-(s % run + t) // run)]
                at += len(runs)
                own_slots = runs[pos // run] * run + 1 + pos % run
                rows.append(torch.cat([front, perm[own_slots] if scattered else own_slots]))
            else:
                rows.append(torch.cat([front, take(t)]))
            lens.append(s + t)
        shared.append(s)
        indptr.append(len(rows))
    for n in alone:
        rows.append(take(n))
        lens.append(n)
    B = len(rows)
    table = torch.zeros(B + 2, max(lens + [1]) + 6, dtype=torch.int32)
    where = torch.randperm(B + 2, generator=g)[:B]
    for r, s in zip(where.tolist(), rows):
        table[r, :len(s)] = s.int()
    k, v = (torch.randn(size, hk, D, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(B, hq * D, generator=g).to(dtype)
    return dict(q=q, k=k, v=v, table=table, rpi=where, lens=lens, shared=shared, indptr=indptr, hq=hq, hk=hk, scale=D ** -0.5)


def reference(c):
    """(out, bound) in 64 bits."""
    hq, hk, dtype = c["hq"], c["hk"], c["q"].dtype
    u = torch.finfo(dtype).eps / 2
    out = torch.zeros(len(c["lens"]), hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b, n in enumerate(c["lens"]):
        if n == 0:
            continue
        s = c["table"][c["rpi"][b], :n].long().to(c["k"].device)
        k, v = (c[x][s].double().transpose(0, 1).repeat_interleave(hq // hk, 0) for x in "kv")  # [hq, n, D]
        sc = torch.einsum("hd,hnd->hn", c["q"][b].double().view(hq, D).to(k.device), k) * c["scale"]
        p = torch.softmax(sc, -1)
        o = torch.einsum("hn,hnd->hd", p, v)
        spread = torch.zeros_like(o)
        far = torch.zeros_like(o)
        for i in range(0, n, 2048):
            off = (v[:, i:i + 2048] - o[:, None]).abs()
            spread += torch.einsum("hn,hnd->hd", p[:, i:i + 2048], off)
            far = torch.maximum(far, off.amax(1))
        small = n * 2.0 ** -25 * p.amax(-1, keepdim=True) * far if dtype == torch.float16 else 0
        out[b] = o.cpu()
        tol[b] = ((u / (1 - u) + 1e-4) * spread + small + 1.01 * u * (o.abs() + u * spread) + 1e-6).cpu()
    return out, tol


def device(c):
    d = {x: c[x].to(DEV) for x in ("q", "k", "v", "table", "rpi")}
    d["seq"] = torch.tensor(c["lens"], dtype=torch.int64, device=DEV)
    d["indptr"] = torch.tensor(c["indptr"], dtype=torch.int32, device=DEV)
    d["shared"] = torch.tensor(c["shared"], dtype=torch.int64, device=DEV)
    return d


def call(c, d, bound=1 << 20, **kw):
    """bound: of the shared tokens, as large as a context may be: small batches, too, then take the kernel that shares."""
    from semi_pd_b200 import ops
    return ops.attn_decode_shared(d["q"], d["k"], d["v"], d["table"], d["rpi"], d["seq"], d["indptr"], d["shared"], bound, c["hq"],
                                  c["hk"], D, c["scale"], **kw)


def check(c, out, rows=None):
    want, tol = reference(c)
    err = (out.cpu().double().view(want.shape) - want).abs()
    worst = (err / tol.clamp_min(1e-30)).nan_to_num(1e9)
    assert bool((err <= tol).all()), f"{worst.max().item():.2f} of the bound at {tuple(torch.nonzero(worst == worst.max())[0].tolist())}"


LAYOUTS = {
    "two": ([(300, [20, 21])], []),
    "one tile": ([(128, [1, 1])], []),
    "all shared": ([(256, [0, 0, 0])], []),                   # no tokens of their own
    "less than a tile": ([(100, [5, 200, 1])], []),
    "nothing shared": ([(0, [40, 300])], [17]),
    "one member": ([(900, [10])], [5]),
    "some alone": ([(513, [7, 130, 1, 60])], [1, 0, 700]),
    "several": ([(384, [3, 9]), (0, [5]), (1000, [1, 2, 3, 4, 5]), (129, [256, 128])], [33]),
    "many": ([(2000, [1 + (37 * i) % 260 for i in range(70)])], []),
    "long": ([(9000, [50, 1, 400])], []),
    "empty batch of groups": ([], [5, 400, 129]),
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk", [(8, 2), (8, 8), (16, 2), (10, 2)])
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_layouts(layout, hq, hk, dtype):
    groups, alone = LAYOUTS[layout]
    c = make_case(groups, alone, hq, hk, dtype, seed=len(layout))
    check(c, call(c, device(c)))
    check(c, call(c, device(c), bound=max(c["shared"] + [0])))  # the tightest bound: by request where that is faster


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("members", [2, 15, 16, 17, 31, 33, 65])
def test_groups_of_query_heads(group, members):
    """Rows that fill a tile of 128 queries, end inside one and begin another."""
    c = make_case([(384, [1 + i % 7 for i in range(members)])], [], 2 * group, 2, torch.float16, seed=members)
    check(c, call(c, device(c)))


@pytest.mark.parametrize("scattered", [False, True])
@pytest.mark.parametrize("aligned", [False, True])
@pytest.mark.parametrize("shared", [1, 127, 128, 129, 1000, 1023, 1024, 1025])
def test_page_tables(shared, aligned, scattered):
    c = make_case([(shared, [30, 1, 129, 100]), (shared + 77, [3, 300])], [50], 8, 2, torch.bfloat16, shared, scattered, aligned)
    check(c, call(c, device(c)))


@pytest.mark.parametrize("sms", [1, 2, 9, 60])
def test_partitions(sms):
    from semi_pd_b200 import ops
    c = make_case([(1500, [10 + i for i in range(20)]), (640, [5, 6, 7])], [300], 16, 4, torch.bfloat16, sms)
    ops.set_sm_budget(sms)
    try:
        out = call(c, device(c))
    finally:
        ops.set_sm_budget(0)
    check(c, out)


def test_some_members_are_empty():
    """Padding rows of length 0 or 1 inside a group: they take nothing from the others."""
    c = make_case([(640, [10, 20, 30, 40, 50])], [9], 8, 2, torch.bfloat16, 3)
    c["lens"][1] = 0
    c["lens"][3] = 0
    check(c, call(c, device(c)))
    c["lens"][1] = 1       # shorter than the shared part: the group shares what all of them have
    check(c, call(c, device(c)))
    c["lens"] = [0] * 6
    out = call(c, device(c))
    assert bool((out == 0).all())


def test_group_lists_with_gaps_and_past_the_end():
    """Groups of no rows, rows before the first group, offsets past the batch: every row is still right."""
    c = make_case([(512, [4, 5, 6]), (256, [7, 8])], [3], 8, 2, torch.bfloat16, 5)
    for indptr, shared in (([0, 3, 3, 5], [512, 99999, 256]), ([1, 3, 5], [512, 256]), ([0, 3, 90], [512, 0]), ([0, 0, 0], [512, 512])):
        d = device(c)
        d["indptr"] = torch.tensor(indptr, dtype=torch.int32, device=DEV)
        d["shared"] = torch.tensor(shared, dtype=torch.int64, device=DEV)
        check(c, call(c, d))


def test_more_rows_and_groups_than_a_plan_holds():
    c = make_case([(256, [1 + i % 3, 2]) for i in range(300)], [], 4, 2, torch.bfloat16, 1)
    check(c, call(c, device(c)))
    c = make_case([(384, [1 + i % 5 for i in range(1100)])], [], 4, 2, torch.bfloat16, 2)
    check(c, call(c, device(c)))


def test_peaked_and_flat_scores():
    """A key that takes nearly all weight, first, last and in the middle; scores far below and above 0; all equal."""
    for at in (0, 700, 1279, 1300):
        c = make_case([(1280, [30, 40, 50])], [], 8, 2, torch.bfloat16, at)
        slot = c["table"][c["rpi"], at].long()
        c["k"][slot] = (c["q"][0].view(2, 4, D)[:, 0] * 3).to(torch.bfloat16)
        check(c, call(c, device(c)))
    for shift in (-40.0, 40.0):
        c = make_case([(640, [30, 40])], [], 8, 2, torch.float16, 9)
        c["k"][:, :, 0] = shift
        c["q"].view(2, 8, D)[:, :, 0] = 12.0
        check(c, call(c, device(c)))
    c = make_case([(640, [30, 40])], [], 8, 2, torch.float16, 9)
    c["q"].zero_()
    check(c, call(c, device(c)))


def test_slots_that_nobody_sees_hold_anything():
    """Infinities and NaN in slots of no request, behind the last token and in the dummy slot."""
    c = make_case([(500, [30, 1, 77]), (128, [1, 2])], [0, 3], 8, 2, torch.bfloat16, 4)
    seen = torch.zeros(c["k"].shape[0], dtype=torch.bool)
    for r, n in zip(c["rpi"].tolist(), c["lens"]):
        seen[c["table"][r, :n].long()] = True
    c["k"][~seen] = float("nan")
    c["v"][~seen] = float("inf")
    check(c, call(c, device(c)))


def test_a_negative_and_a_zero_scale():
    for scale in (-0.05, 0.0):
        c = make_case([(640, [30, 40, 1])], [7], 8, 2, torch.bfloat16, 2)
        c["scale"] = scale
        check(c, call(c, device(c)))


def test_strided_rows_own_output_and_workspace():
    from semi_pd_b200 import ops
    c = make_case([(1000, [30, 40, 1] * 6)], [7], 16, 4, torch.bfloat16, 2)
    d = device(c)
    B = len(c["lens"])
    wide = torch.randn(B, 24 * D, device=DEV).to(torch.bfloat16)
    wide[:, :16 * D] = d["q"]
    d["q"] = wide[:, :16 * D]
    out = torch.full((B, 20 * D), 7.0, dtype=torch.bfloat16, device=DEV)
    ws = ops.new_attn_shared_workspace(torch.device(DEV, 0), B, 16, 4, D)
    first = call(c, d, out=out[:, :16 * D], workspace=ws).clone()
    check(c, first.contiguous())
    assert bool((out[:, 16 * D:] == 7).all())
    for _ in range(3):  # counters are re-armed, parts are joined in a fixed order
        assert torch.equal(call(c, d, out=out[:, :16 * D], workspace=ws), first)
    assert torch.equal(call(c, d), first)


def test_same_result_without_sharing():
    """Against attn_decode, which reads every request's pages: within both bounds."""
    from semi_pd_b200 import ops
    c = make_case([(3000, [60 + i for i in range(24)])], [100], 32, 8, torch.bfloat16, 2)
    d = device(c)
    plain = ops.attn_decode(d["q"], d["k"], d["v"], d["table"], d["rpi"], d["seq"], 32, 8, D, c["scale"])
    _, tol = reference(c)
    assert bool(((call(c, d).double().cpu() - plain.double().cpu()).abs().view(tol.shape) <= 2 * tol).all())


def test_graph_and_another_stream():
    """A captured call follows the lengths and groups in its tensors; two graphs with scratch of their own run at once."""
    from semi_pd_b200 import ops
    c = make_case([(1400, [60 + i for i in range(12)])], [100], 16, 4, torch.bfloat16, 2)
    other = make_case([(700, [6 + i for i in range(12)])], [30], 16, 4, torch.bfloat16, 3)
    graphs = []
    for case in (c, other):
        d = device(case)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            call(case, d, bound=200000)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = call(case, d, bound=200000)
        graphs.append((graph, d, out, stream, case))
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, d, out, stream, case in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for graph, d, out, stream, case in graphs:
        check(case, out)
    graph, d, out, stream, case = graphs[0]
    case["lens"] = [n - 17 for n in case["lens"]]
    d["seq"].copy_(torch.tensor(case["lens"], device=DEV))
    d["shared"].fill_(1300)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.replay()
    torch.cuda.synchronize()
    check(case, out)


def test_refusals():
    from semi_pd_b200 import ops
    c = make_case([(300, [20, 21])], [], 8, 2)
    d = device(c)

    def bad(match, **change):
        e = dict(d, **change)
        with pytest.raises((RuntimeError, ValueError), match=match):
            call(c, e)

    bad("CUDA tensors", q=d["q"].cpu())
    bad("share a dtype", q=d["q"].half())
    bad("one request slot", q=d["q"][:1])
    bad("int64", seq=d["seq"].int())
    bad("int64", shared=d["shared"].int())
    bad("group_indptr", indptr=d["indptr"].long())
    bad("group_indptr", indptr=d["indptr"][:1])
    bad("req_to_token", table=d["table"].long())
    bad("contiguous", k=d["k"].repeat(1, 2, 1)[:, ::2])
    with pytest.raises(RuntimeError, match="negative"):
        call(c, d, bound=-1)
    with pytest.raises(RuntimeError, match="workspace"):
        call(c, d, workspace=torch.zeros(64, dtype=torch.uint8, device=DEV))
    with pytest.raises(RuntimeError, match="group"):
        ops.attn_decode_shared(torch.zeros(2, 9 * D, dtype=torch.bfloat16, device=DEV), d["k"][:, :1].contiguous(), d["v"][:, :1].contiguous(),
                               d["table"], d["rpi"], d["seq"], d["indptr"], d["shared"], 300, 9, 1, D, 0.1)
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.attn_decode_shared(torch.zeros(2, 4 * 64, dtype=torch.bfloat16, device=DEV), torch.zeros(9, 2, 64, dtype=torch.bfloat16, device=DEV),
                               torch.zeros(9, 2, 64, dtype=torch.bfloat16, device=DEV), d["table"], d["rpi"], d["seq"], d["indptr"],
                               d["shared"], 300, 4, 2, 64, 0.1)


def test_long_offsets():
    """Slots whose rows lie beyond 4 GB of the pool."""
    hk, rows = 8, (5 << 30) // (8 * D * 2) + 200
    c = make_case([(512, [5, 6, 130])], [40], 16, hk, torch.bfloat16, 2)
    need = c["k"].shape[0]
    shift = rows - need
    big = {}
    for x in "kv":
        big[x] = torch.zeros(rows, hk, D, dtype=torch.bfloat16, device=DEV)
        big[x][shift:] = c[x].to(DEV)
    d = device(c)
    d.update(big)
    d["table"] = torch.where(d["table"] > 0, d["table"] + shift, d["table"])
    check(c, call(c, d))
