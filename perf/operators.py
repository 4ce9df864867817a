"""What the operators for many continuations of one prompt are measured on: decode attention over a shared prefix, and the
copying, forking and compacting of the cache's pages.

A case is a dict of plain values; its "op" says which operator it is:

  shared   ops.attn_decode_shared: one new token per request; the requests of a group continue the same tokens
  copy     ops.kv_copy: rows of every layer's pool from slots to other slots
  fork     ops.kv_fork: children of requests share their whole runs of slots and get a copy of the last, partial one
  compact  ops.kv_compact: a request goes on with a subset of its tokens, in new slots

`own` False computes a case in plain torch operations, True through the framework.
"""
import math

import torch

own = False

DEV = "cuda"
RUN = 128  # slots of a run of the allocator
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # two samples of one short prompt, the smallest call a server makes
        dict(name="shared_2", op="shared", dtype="bfloat16", groups=1, members=2, prefix=300, tail=20, hq=32, hk=8,
             copied=True, scattered=False),
        # a saturated decode batch behind one system prompt
        dict(name="shared_64", op="shared", dtype="bfloat16", groups=1, members=64, prefix=8192, tail=130, hq=32, hk=8,
             copied=True, scattered=False),
        # eight prompts with a few samples each, of unequal and odd lengths, on a model with five query heads per key head
        dict(name="shared_8x6", op="shared", dtype="float16", groups=8, members=6, prefix=3001, tail=77, hq=40, hk=8,
             copied=False, scattered=False),
        # many samples of one prompt, every query head with its own keys
        dict(name="shared_160_mha", op="shared", dtype="bfloat16", groups=1, members=160, prefix=1500, tail=40, hq=32, hk=32,
             copied=True, scattered=False),
        # a few questions about one long document, a page table that another allocator wrote
        dict(name="shared_12_long", op="shared", dtype="bfloat16", groups=1, members=12, prefix=65536, tail=200, hq=32, hk=8,
             copied=True, scattered=True),
        # 256 samples over the same long context, eight query heads per key head
        dict(name="shared_256_long", op="shared", dtype="float16", groups=1, members=256, prefix=32768, tail=300, hq=64, hk=8,
             copied=True, scattered=False),
        # the tokens that a draft got right, moved behind one another
        dict(name="copy_12", op="copy", dtype="bfloat16", kind="mha", layers=32, heads=8, dim=128, tokens=12, scattered=True),
        # latent rows of a long request, moved whole
        dict(name="copy_12000_latent", op="copy", dtype="bfloat16", kind="latent", layers=27, heads=1, dim=576, tokens=12001,
             scattered=False),
        # one more sample of a prompt
        dict(name="fork_1", op="fork", dtype="bfloat16", kind="mha", layers=32, heads=8, dim=128, parents=1, children=1,
             tokens=1000),
        # sixteen samples each of eight prompts
        dict(name="fork_8x16", op="fork", dtype="float16", kind="mha", layers=16, heads=8, dim=128, parents=8, children=16,
             tokens=2000),
        # a request that goes on without the middle of its context
        dict(name="compact_1", op="compact", dtype="bfloat16", kind="mha", layers=32, heads=8, dim=128, requests=1, tokens=700,
             keep=0.5),
        # the same for a batch, in a 32-bit pool
        dict(name="compact_16", op="compact", dtype="float32", kind="mha", layers=8, heads=4, dim=128, requests=16, tokens=3000,
             keep=0.6),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["shared", "shared", "shared", "copy", "fork", "compact"])
    dtype = rng.choice(["bfloat16", "float16"])
    if op == "shared":
        while True:
            hq, hk = rng.choice([(32, 8), (40, 8), (32, 32), (16, 8), (64, 8), (16, 2), (28, 4), (8, 8)])
            case = dict(op=op, dtype=dtype, groups=_log(rng, 1, 16), members=_log(rng, 1, 256), prefix=_log(rng, 1, 65536),
                        tail=_log(rng, 1, 1000), hq=hq, hk=hk, copied=rng.random() < 0.5, scattered=rng.random() < 0.3)
            rows, (_, total) = case["groups"] * case["members"], _tokens(case)
            slots = case["groups"] * case["prefix"] + rows * (case["tail"] + RUN)
            if rows <= 512 and total * hq <= 256 * 33000 * 64 and slots * hk <= 400000 * 8 and rows * case["prefix"] <= 1 << 23:
                return case
    kind = rng.choice(["mha", "mha", "latent"])
    if kind == "latent":
        shape = dict(kind=kind, dtype=dtype, layers=rng.randint(1, 27), heads=1, dim=rng.choice([576, 320]))
    else:
        shape = dict(kind=kind, dtype=rng.choice([dtype, dtype, "float32"]), layers=rng.randint(1, 32),
                     heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]))
    token = _token_bytes(shape)
    if op == "copy":
        return dict(op=op, **shape, tokens=min(_log(rng, 1, 16000), max(1, (400 << 20) // token)), scattered=rng.random() < 0.5)
    if op == "fork":
        parents, children = _log(rng, 1, 8), _log(rng, 1, 16)
        while parents * (2200 + 128 * children) * token > 2 << 30 and parents * children > 1:
            parents, children = max(1, parents // 2), max(1, children // 2)
        return dict(op=op, **shape, parents=parents, children=children, tokens=_log(rng, 1, 2000))
    requests = _log(rng, 1, 16)
    return dict(op=op, **shape, requests=requests, tokens=min(_log(rng, 1, 3000), max(1, (600 << 20) // (token * requests))),
                keep=round(rng.uniform(0.05, 1.0), 2))


def _token_bytes(case):
    planes = case["layers"] * (1 if case["kind"] == "latent" else 2)
    return planes * case["heads"] * case["dim"] * DTYPES[case["dtype"]].itemsize


# ---------------------------------------------------------------------------------------------
# lengths: the same for every seed
# ---------------------------------------------------------------------------------------------
def _spread(mean, i, n):
    """Unequal lengths around a mean: three quarters to five quarters of it, odd ones among them, at least one."""
    return mean if n == 1 else max(1, (mean * 3) // 4 + (mean * ((i * 5) % n)) // (2 * max(n - 1, 1)))


def _lengths(case):
    """(prefix of every group, tails of its members); a tail counts the tokens behind the prefix, this step's among them."""
    n = case["groups"]
    rows = n * case["members"]
    out = []
    for g in range(n):
        tails = [_spread(case["tail"], g * case["members"] + m, rows) for m in range(case["members"])]
        out.append((_spread(case["prefix"], g, n), tails))
    return out


def _shared(case, prefix):
    """Slots the members have in common: whole runs where a fork copied the last, partial one."""
    return prefix // RUN * RUN if case["copied"] else prefix


def _tokens(case):
    """(tokens whose keys have to be read, tokens that the queries see)."""
    once = seen = 0
    for prefix, tails in _lengths(case):
        common = _shared(case, prefix)
        once += common + sum(prefix - common + t for t in tails)
        seen += sum(prefix + t for t in tails)
    return once, seen


def _fork_lengths(case):
    return [_spread(case["tokens"], i, case["parents"]) for i in range(case["parents"])]


def _kept(case):
    """Tokens and kept tokens of every request."""
    lens = [_spread(case["tokens"], i, case["requests"]) for i in range(case["requests"])]
    return lens, [max(1, int(n * case["keep"])) for n in lens]


def work(case):
    if case["op"] == "shared":
        size = DTYPES[case["dtype"]].itemsize
        once, seen = _tokens(case)
        rows = case["groups"] * case["members"]
        return {"bytes": 2 * once * case["hk"] * 128 * size + 2 * rows * case["hq"] * 128 * size + 4 * once,
                "flops": 4 * seen * case["hq"] * 128}
    token = _token_bytes(case)
    if case["op"] == "copy":
        return {"bytes": case["tokens"] * (2 * token + 16), "flops": 0}
    if case["op"] == "fork":
        lens = _fork_lengths(case)
        part = sum(n % RUN for n in lens)
        return {"bytes": part * token * (1 + case["children"]) + sum(lens) * 4 * (1 + case["children"]), "flops": 0}
    _, kept = _kept(case)
    return {"bytes": sum(kept) * (2 * token + 4 + 8 + 4 + 4), "flops": 0}


# ---------------------------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _slots(runs, n):
    """Slots of n tokens placed in these runs (slot 0 is the dummy slot)."""
    pos = torch.arange(n)
    return runs[pos // RUN] * RUN + 1 + pos % RUN


def _prepare_shared(case, seed):
    g = _gen(seed)
    cpu = torch.Generator().manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    lengths = _lengths(case)
    need = 1
    for prefix, tails in lengths:
        common = _shared(case, prefix)
        need += -(-common // RUN) + sum(-(-(prefix - common + t) // RUN) for t in tails)
    order = torch.randperm(need, generator=cpu)
    size = need * RUN + 1
    perm = torch.cat([torch.zeros(1, dtype=torch.int64), 1 + torch.randperm(size - 1, generator=cpu)])
    at, rows, seq, common_lens, indptr = 0, [], [], [], [0]

    def take(n):
        nonlocal at
        runs = order[at:at + -(-n // RUN)]
        at += len(runs)
        s = _slots(runs, n)
        return perm[s] if case["scattered"] else s

    for prefix, tails in lengths:
        common = _shared(case, prefix)
        front = take(common)
        for t in tails:
            rows.append(torch.cat([front, take(prefix - common + t)]))
            seq.append(prefix + t)
        common_lens.append(common)
        indptr.append(len(rows))
    n = len(rows)
    table = torch.zeros(n + 3, max(seq) + 4, dtype=torch.int32)
    where = torch.randperm(n + 3, generator=cpu)[:n]
    for r, slots in zip(where.tolist(), rows):
        table[r, :len(slots)] = slots.int()
    # keys of unit size with the first tokens of a prompt larger: they draw more of the attention, as they do in trained models
    k = torch.randn(size, case["hk"], 128, generator=g, device=DEV, dtype=dtype)
    v = torch.randn(size, case["hk"], 128, generator=g, device=DEV, dtype=dtype)
    first = torch.stack([r[0] for r in rows]).to(DEV)
    k[first] = k[first] * 3
    st = dict(case=case, q=torch.randn(n, case["hq"] * 128, generator=g, device=DEV, dtype=dtype), k=k, v=v,
              table=table.to(DEV), rpi=where.to(DEV), seq=torch.tensor(seq, device=DEV), seq_host=seq,
              indptr=torch.tensor(indptr, dtype=torch.int32, device=DEV), common=torch.tensor(common_lens, device=DEV),
              max_common=max(common_lens), scale=128 ** -0.5)
    if own:
        from semi_pd_b200 import ops
        st["workspace"] = ops.new_attn_shared_workspace(torch.device(DEV, torch.cuda.current_device()), n, case["hq"], case["hk"], 128)
    return st


def _pool(case, size, g):
    """A pool's buffers: every layer's keys and values, or its latent rows, in one allocation."""
    planes = case["layers"] * (1 if case["kind"] == "latent" else 2)
    slab = torch.randn(planes, size, case["heads"], case["dim"], generator=g, device=DEV, dtype=DTYPES[case["dtype"]])
    st = dict(case=case, slab=slab)
    if own:
        from semi_pd_b200 import ops
        st["planes"] = ops.KVPlanes(list(slab))
    return st


def _prepare_copy(case, seed):
    cpu = torch.Generator().manual_seed(seed)
    n = case["tokens"]
    runs = -(-n // RUN)
    order = torch.randperm(2 * runs + 1, generator=cpu)
    src, dst = _slots(order[:runs], n), _slots(order[runs:], n)
    if case["scattered"]:
        both = 1 + torch.randperm((2 * runs + 1) * RUN, generator=cpu)
        src, dst = both[:n], both[n:2 * n]
    st = _pool(case, (2 * runs + 1) * RUN + 1, _gen(seed))
    st.update(src=src.to(DEV), dst=dst.to(DEV))
    return st


def _prepare_fork(case, seed):
    cpu = torch.Generator().manual_seed(seed)
    lens = _fork_lengths(case)
    kids = case["children"]
    need = sum(-(-n // RUN) for n in lens) + len(lens) * kids
    order = torch.randperm(need, generator=cpu)
    ids = torch.randperm(len(lens) * (1 + kids) + 2, generator=cpu)
    table = torch.zeros(len(ids), max(lens) + 4, dtype=torch.int32)
    at, parents, children, seq, tail = 0, [], [], [], []
    for i, n in enumerate(lens):
        runs = order[at:at + -(-n // RUN)]
        at += len(runs)
        table[ids[i], :n] = _slots(runs, n).int()
        for c in range(kids):
            parents.append(int(ids[i]))
            children.append(int(ids[len(lens) + i * kids + c]))
            seq.append(n)
            tail.append(int(order[at]) * RUN + 1)
            at += 1
    st = _pool(case, need * RUN + 1, _gen(seed))
    st.update(table=table.to(DEV), **{k: torch.tensor(x, device=DEV) for k, x in
                                      (("parents", parents), ("children", children), ("seq", seq), ("tail", tail))})
    st["host"] = (parents, children, seq, tail)
    return st


def _prepare_compact(case, seed):
    cpu = torch.Generator().manual_seed(seed)
    lens, kept = _kept(case)
    need = sum(-(-n // RUN) + -(-k // RUN) for n, k in zip(lens, kept))
    order = torch.randperm(need, generator=cpu)
    ids = torch.randperm(2 * len(lens) + 1, generator=cpu)
    table = torch.zeros(len(ids), max(lens) + 4, dtype=torch.int32)
    at, keep, loc, indptr = 0, [], [], [0]
    for i, (n, k) in enumerate(zip(lens, kept)):
        runs = order[at:at + -(-n // RUN)]
        at += len(runs)
        table[ids[i], :n] = _slots(runs, n).int()
        # the first tokens and the latest ones stay, and some between them
        head = min(4, k)
        last = min(k - head, k // 2)
        mid = head + torch.randperm(n - head - last, generator=cpu)[:k - head - last].sort().values
        keep.append(torch.cat([torch.arange(head), mid, torch.arange(n - last, n)]))
        runs = order[at:at + -(-k // RUN)]
        at += len(runs)
        loc.append(_slots(runs, k))
        indptr.append(indptr[-1] + k)
    st = _pool(case, need * RUN + 1, _gen(seed))
    n = len(lens)
    st.update(table=table.to(DEV), src=ids[:n].to(DEV), dst=ids[n:2 * n].to(DEV), keep=torch.cat(keep).to(DEV),
              indptr=torch.tensor(indptr, device=DEV), loc=torch.cat(loc).to(DEV), host=(ids[:n].tolist(), ids[n:2 * n].tolist(), indptr))
    return st


def prepare(case, seed):
    return {"shared": _prepare_shared, "copy": _prepare_copy, "fork": _prepare_fork, "compact": _prepare_compact}[case["op"]](
        case, seed)


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _plain_shared(st):
    case = st["case"]
    hk, group = case["hk"], case["hq"] // case["hk"]
    q = st["q"].float().view(-1, hk, group, 128)
    out = torch.empty(q.shape, device=q.device)
    for b, n in enumerate(st["seq_host"]):
        slots = st["table"][st["rpi"][b], :n].long()
        k, v = st["k"][slots].float(), st["v"][slots].float()  # [n, hk, 128]
        s = torch.matmul(q[b], k.permute(1, 2, 0)) * st["scale"]  # [hk, group, n]
        p = torch.exp(s - s.amax(-1, keepdim=True))
        out[b] = torch.matmul(p, v.transpose(0, 1)) / p.sum(-1, keepdim=True)
    return out.view(-1, case["hq"] * 128).to(st["q"].dtype)


def _plain_fork(st):
    slab, table = st["slab"], st["table"]
    for parent, child, n, base in zip(*st["host"]):
        full = n // RUN * RUN
        table[child, :full] = table[parent, :full]
        if n > full:
            slots = torch.arange(base, base + n - full, device=table.device)
            slab[:, slots] = slab[:, table[parent, full:n].long()]
            table[child, full:n] = slots.int()


def _plain_compact(st):
    slab, table = st["slab"], st["table"]
    src, dst, indptr = st["host"]
    for i, (s, d) in enumerate(zip(src, dst)):
        loc = st["loc"][indptr[i]:indptr[i + 1]]
        slab[:, loc] = slab[:, table[s, st["keep"][indptr[i]:indptr[i + 1]]].long()]
        table[d, :len(loc)] = loc.int()


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        if op == "shared":
            return _plain_shared(state)
        if op == "copy":
            state["slab"][:, state["dst"]] = state["slab"][:, state["src"]]
            return state["slab"]
        (_plain_fork if op == "fork" else _plain_compact)(state)
        return [state["slab"], state["table"]]
    from semi_pd_b200 import ops
    if op == "shared":
        return ops.attn_decode_shared(state["q"], state["k"], state["v"], state["table"], state["rpi"], state["seq"],
                                      state["indptr"], state["common"], state["max_common"], case["hq"], case["hk"], 128,
                                      state["scale"], workspace=state["workspace"])
    if op == "copy":
        ops.kv_copy(state["planes"], state["src"], state["dst"])
        return state["slab"]
    if op == "fork":
        ops.kv_fork(state["planes"], state["table"], state["parents"], state["children"], state["seq"], state["tail"], RUN)
    else:
        ops.kv_compact(state["planes"], state["table"], state["src"], state["dst"], state["keep"], state["indptr"], state["loc"])
    return [state["slab"], state["table"]]


# ---------------------------------------------------------------------------------------------
# the same in 64 bits, from the definition: softmax over all of a request's tokens, its pages one after another
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] != "shared":
        return None  # bits that move: no numbers are computed
    st = prepare(case, seed)
    heads = case["hq"] // case["hk"]
    out = torch.zeros(len(st["seq_host"]), case["hq"], 128, dtype=torch.float64, device=DEV)
    for b, n in enumerate(st["seq_host"]):
        row = st["table"][st["rpi"][b]].long()
        q = st["q"][b].double().view(case["hq"], 128)
        top = torch.full((case["hq"], 1), -math.inf, dtype=torch.float64, device=DEV)
        total = torch.zeros(case["hq"], 1, dtype=torch.float64, device=DEV)
        acc = torch.zeros(case["hq"], 128, dtype=torch.float64, device=DEV)
        for at in range(0, n, 8192):
            slots = row[at:min(n, at + 8192)]
            k = st["k"][slots].double().repeat_interleave(heads, 1)
            v = st["v"][slots].double().repeat_interleave(heads, 1)
            s = (k * q).sum(-1).t() * st["scale"]  # [hq, tokens]
            new = torch.maximum(top, s.max(-1, keepdim=True).values)
            e, old = torch.exp(s - new), torch.exp(top - new)
            total = total * old + e.sum(-1, keepdim=True)
            acc = acc * old + torch.einsum("ht,thd->hd", e, v)
            top = new
        out[b] = acc / total
    return out.view(-1, case["hq"] * 128)
