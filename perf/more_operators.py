"""Cases of the operators for sampled continuations over the paged 4-bit cache, for timing and comparison.

rope    rotary positions of query and key rows before they are cached and
        attended: y = f R(a) x on the first r channels of every head, with the
        angle a = position * frequency_i of pair i, channels (i, i + r / 2) or
        (2 i, 2 i + 1); the other channels pass
fork    pages shared between requests: children take over a parent's pages,
        all bring new rows (a shared page that is written into is copied
        first, in every layer), then the children finish and what nobody else
        holds goes back to the free list
prefix  grouped-query attention of requests whose first pages are the same,
        those read once for all requests of a group
verify  drafted tokens against the target's probabilities p = softmax(l / T):
        draft d is accepted where u q(d) < p(d) (q = 1 for greedy drafts), the
        token after the accepted ones comes from max(p - q, 0), or from p
        behind the last draft: the first one in vocabulary order whose running
        sum passes u times the whole sum.  T = 0: all of p on the first largest
"""
import math
import random

import torch

own = False

HEAD_DIM = 128
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one new row for each of 256 requests, the q|k part of a fused projection
        dict(name="rope_decode", kind="rope", rows=256, n=256, heads=40, wide=48, dim=128, rot=128, dtype="bf16",
             pairs="half", scaling="none", far=40960, step=True, shape=1),
        # prompts of a long-context target whose frequencies are stretched, far positions
        dict(name="rope_prompt", kind="rope", rows=4128, n=1, heads=48, wide=48, dim=128, rot=128, dtype="f16",
             pairs="half", scaling="yarn", far=1 << 20, step=False, shape=2),
        # a prefill round over many requests
        dict(name="rope_prefill", kind="rope", rows=65521, n=128, heads=40, wide=48, dim=128, rot=128, dtype="bf16",
             pairs="half", scaling="none", far=40960, step=True, shape=3),
        # one prompt sampled four times, few layers: the latency of the page tables
        dict(name="fork_one", kind="fork", parents=1, children=3, ctx=2049, rows=1, layers=4, nkv=8, page=64, shape=4),
        # 32 prompts sampled sixteen times each, ragged lengths
        dict(name="fork_samples", kind="fork", parents=32, children=15, ctx=1024, rows=16, layers=16, nkv=8, page=64,
             shape=5),
        # eight samples of one prompt, one token each
        dict(name="prefix_samples", kind="prefix", groups=1, members=8, prefix=2048, tail=130, rows=1, ragged=False,
             nq=32, nkv=8, page=64, causal=True, dtype="bf16", shape=6),
        # one token each of 256 requests behind one system prompt
        dict(name="prefix_system", kind="prefix", groups=1, members=256, prefix=4096, tail=1024, rows=1, ragged=False,
             nq=32, nkv=8, page=64, causal=True, dtype="bf16", shape=7),
        # sixteen prompts sampled sixteen times, small pages, odd lengths
        dict(name="prefix_groups", kind="prefix", groups=16, members=16, prefix=8176, tail=515, rows=1, ragged=False,
             nq=28, nkv=4, page=16, causal=True, dtype="f16", shape=8),
        # verification of ragged drafts of 64 requests behind two long documents
        dict(name="prefix_verify", kind="prefix", groups=2, members=32, prefix=16384, tail=1024, rows=16, ragged=True,
             nq=40, nkv=8, page=64, causal=True, dtype="bf16", shape=9),
        # one request's block of 16 (the latency of a step)
        dict(name="verify_one", kind="verify", n=1, block=16, vocab=151936, dtype="bf16", temps="one", keep=0.8,
             probs=False, ragged=False, shape=10),
        # 256 requests in flight, greedy ones among them, ragged drafts
        dict(name="verify_serving", kind="verify", n=256, block=16, vocab=151936, dtype="bf16", temps="mixed", keep=0.8,
             probs=False, ragged=True, shape=11),
        # sampled drafts with their distributions, fp32, a vocabulary that is odd
        dict(name="verify_probs", kind="verify", n=48, block=8, vocab=32003, dtype="f32", temps="mixed", keep=0.6,
             probs=True, ragged=False, shape=12),
    ]


def _log_int(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    kind = rng.choice(["rope", "fork", "prefix", "prefix", "verify"])
    shape = rng.randrange(1 << 30)
    if kind == "rope":
        dim = rng.choice([128, 128, 64, 80, 96, 192, 256])
        rot = rng.choice([dim, dim, dim // 2, dim // 4 * 2 - 6])
        heads = rng.randint(1, 64)
        dtype = rng.choice(["f16", "bf16", "f32"])
        rows = _log_int(rng, 1, 65521 * 40 * 128 // (heads * dim * (2 if dtype == "f32" else 1)) // 2)
        return dict(kind=kind, rows=rows, n=_log_int(rng, 1, min(rows, 1000)), heads=heads, wide=heads + rng.choice([0, 8, 3]),
                    dim=dim, rot=rot, dtype=dtype, pairs=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), far=_log_int(rng, 1, 1 << 22),
                    step=rng.random() < 0.5, shape=shape)
    if kind == "fork":
        children = _log_int(rng, 1, 32)
        parents = _log_int(rng, 1, 512 // (children + 1))
        layers = rng.choice([1, 5, 16])
        page = rng.choice([16, 32, 64, 128])
        return dict(kind=kind, parents=parents, children=children, ctx=_log_int(rng, 1, 1024), rows=_log_int(rng, 1, 48),
                    layers=layers, nkv=rng.choice([1, 2, 4, 8]), page=page, shape=shape)
    if kind == "prefix":
        nq, nkv = rng.choice([(32, 8), (40, 8), (4, 2), (12, 4), (8, 8), (16, 1), (32, 4), (28, 4)])
        members = _log_int(rng, 1, 256)
        groups = _log_int(rng, 1, max(1, 256 // members))
        prefix, tail = _log_int(rng, 1, 16384), _log_int(rng, 1, 1024)
        rows = rng.choice([1, 1, _log_int(rng, 1, 32)])
        # no more products than prefix_verify's, no more cached rows than 300,000
        while (groups * members * rows * nq * (prefix + tail) > 64 * 16 * 40 * 17408 * 0.5 or
               groups * (prefix + members * tail) > 300000):
            members, rows, groups = max(1, members // 2), max(1, rows - rows // 4), max(1, groups // 2)
            prefix = max(1, prefix * 3 // 4)
        return dict(kind=kind, groups=groups, members=members, prefix=prefix, tail=max(tail, rows), rows=rows,
                    ragged=rng.random() < 0.5, nq=nq, nkv=nkv, page=rng.choice([16, 32, 64, 128]),
                    causal=rng.random() < 0.8, dtype=rng.choice(["f16", "bf16"]), shape=shape)
    vocab = rng.choice([151936, 32003, 8192, _log_int(rng, 2, 200000)])
    dtype = rng.choice(["f16", "bf16", "f32"])
    probs = rng.random() < 0.3
    block = rng.randint(1, 32)
    most = int(256 * 16 * 151936 * 0.4 / (vocab * block * (2 if dtype == "f32" else 1) * (3 if probs else 1)))
    return dict(kind=kind, n=_log_int(rng, 1, max(1, min(512, most))), block=block, vocab=vocab, dtype=dtype,
                temps=rng.choice(["one", "mixed"]), keep=rng.choice([0.3, 0.8, 0.95]), probs=probs,
                ragged=rng.random() < 0.5, shape=shape)


def _cdiv(a, b):
    return -(-a // b)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# what each case's requests look like, from the case alone
def _rope_rows(case):
    """New rows of each request and their cached rows afterwards."""
    rng = random.Random(case["shape"])
    n, rows = case["n"], case["rows"]
    cuts = sorted(rng.randint(0, rows) for _ in range(n - 1)) if rows > n else list(range(1, n))
    new = [b - a for a, b in zip([0] + cuts, cuts + [rows])]
    return new, [m + rng.randint(0, case["far"]) for m in new]


def _fork_lens(case):
    rng = random.Random(case["shape"])
    return [rng.randint(max(1, case["ctx"] // 2), case["ctx"]) if case["parents"] > 1 else case["ctx"]
            for _ in range(case["parents"])]


def _prefix_lens(case):
    """Per group: rows that all members share, in whole pages.  Per request: cached rows and query rows."""
    rng = random.Random(case["shape"])
    shared = [case["prefix"] // case["page"] * case["page"] for _ in range(case["groups"])]
    lens, new = [], []
    for s in shared:
        for k in range(case["members"]):
            m = rng.randint(0, case["rows"]) if case["ragged"] and k else case["rows"]
            lens.append(s + rng.randint(max(m, 1), max(case["tail"], m, 1)))
            new.append(m)
    return shared, lens, new


def _verify_counts(case):
    rng = random.Random(case["shape"])
    most = case["block"] - 1
    return [rng.randint(most // 2, most) if case["ragged"] else most for _ in range(case["n"])]


def _temperatures(case):
    rng = random.Random(case["shape"] + 1)
    if case["temps"] == "one":
        return [1.0] * case["n"]
    return [rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]) for _ in range(case["n"])]


def work(case):
    size = 4 if case.get("dtype") == "f32" else 2
    if case["kind"] == "rope":
        pairs = case["rows"] * case["heads"] * case["rot"] // 2
        return {"bytes": 2 * size * case["rows"] * case["heads"] * case["dim"] + 4 * case["n"], "flops": 6 * pairs}
    if case["kind"] == "fork":
        page, lens, k = case["page"], _fork_lens(case), case["children"]
        n = case["parents"] * (k + 1)
        held = sum(_cdiv(a, page) for a in lens)
        blocks = sum(k * _cdiv(a % page, 16) for a in lens)        # all but one holder copy a page that is not full
        # table entries out and in, counts, slots, the pages' blocks in and out
        return {"bytes": 24 * n + 4 * n * case["rows"] + 12 * held * k + 2 * 2304 * blocks * case["nkv"] * case["layers"],
                "flops": 0}
    if case["kind"] == "prefix":
        shared, lens, new = _prefix_lens(case)
        m = case["members"]
        keys = sum(shared) + sum(a - shared[i // m] for i, a in enumerate(lens) if new[i])
        pairs = sum(sum(a - b + j + 1 for j in range(b)) if case["causal"] else a * b for a, b in zip(lens, new))
        return {"bytes": keys * case["nkv"] * 144 + 4 * sum(new) * case["nq"] * HEAD_DIM + 4 * keys // case["page"],
                "flops": 4 * HEAD_DIM * case["nq"] * pairs}
    # the rows up to the first refused draft, as many as expected
    p = 0.95 * case["keep"]
    rows = sum(sum(p ** j for j in range(c + 1)) for c in _verify_counts(case))
    bytes_ = rows * case["vocab"] * size + (4 * case["n"] * case["vocab"] if case["probs"] else 0)
    return {"bytes": int(bytes_), "flops": int(4 * rows * case["vocab"])}


# ---------------------------------------------------------------- inputs
ROPE_SCALING = {"none": None, "linear": {"type": "linear", "factor": 8.0}, "ntk": {"type": "ntk", "factor": 4.0},
                "yarn": {"type": "yarn", "factor": 8.0, "original_max_position_embeddings": 32768}}
THETA = 1e6


def _rope_inputs(case, gen):
    wide = torch.randn(case["rows"], case["wide"], case["dim"], generator=gen, device="cuda").to(DTYPES[case["dtype"]])
    new, lens = _rope_rows(case)
    starts = [0]
    for m in new:
        starts.append(starts[-1] + m)
    if case["step"]:
        return wide[:, :case["heads"]], _i32(starts), _i32(lens), None
    positions = torch.randint(0, case["far"] + 1, (case["rows"],), generator=gen, device="cuda", dtype=torch.int32)
    return wide[:, :case["heads"]], None, None, positions


def _fork_inputs(case, gen):
    """Tables of the parents (request p * (children + 1)), an empty row for each child, and the layers' pools."""
    page, lens, k = case["page"], _fork_lens(case), case["children"]
    n = case["parents"] * (k + 1)
    held = [_cdiv(a, page) for a in lens]
    max_pages = _cdiv(case["ctx"] + case["rows"], page) + 1
    num_pages = sum(held) + n * (_cdiv(case["rows"], page) + 1) + 3
    perm = torch.randperm(num_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((n, max_pages), -1, dtype=torch.int32, device="cuda")
    at = 0
    for p, h in enumerate(held):
        table[p * (k + 1), :h] = perm[at:at + h]
        at += h
    pools = torch.randint(0, 256, (case["layers"], num_pages, case["nkv"], page // 16, 2304), generator=gen, device="cuda",
                          dtype=torch.uint8)
    full = lambda values: [v if i % (k + 1) == 0 else 0 for i, v in enumerate(x for x in values for _ in range(k + 1))]
    return dict(table=table, free=perm, head=_i32([at]), lens=_i32(full(lens)), pages=_i32(full(held)), pools=pools,
                src=_i32([p * (k + 1) for p in range(case["parents"]) for _ in range(k)]),
                dst=_i32([p * (k + 1) + 1 + c for p in range(case["parents"]) for c in range(k)]),
                new=_i32([case["rows"]] * n), holders=torch.zeros(2, num_pages, dtype=torch.int32, device="cuda"),
                status=torch.zeros(1, dtype=torch.int32, device="cuda"))


def _prefix_table(case, gen):
    """Block table whose members of a group share their first pages, the page of each owner's run of rows."""
    page, m = case["page"], case["members"]
    shared, lens, _ = _prefix_lens(case)
    runs = [("group", g, 0, s // page) for g, s in enumerate(shared)]
    runs += [("own", i, shared[i // m] // page, _cdiv(a, page)) for i, a in enumerate(lens)]
    total = sum(c - b for _, _, b, c in runs)
    perm = torch.randperm(total + 3, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(1, max(_cdiv(a, page) for a in lens))), -1, dtype=torch.int32, device="cuda")
    at, rows = 0, []
    for what, i, b, c in runs:
        pages = perm[at:at + c - b]
        at += c - b
        if what == "group":
            table[i * m:(i + 1) * m, b:c] = pages
            rows.append((what, i, pages, (c - b) * page))
        else:
            table[i, b:c] = pages
            rows.append((what, i, pages, lens[i] - b * page))
    return table, rows, total + 3


def _kv_rows(case, rows, gen):
    """K and V rows as a layer makes them: normed keys with a few strong channels, smaller values."""
    k = torch.randn(rows, case["nkv"], HEAD_DIM, generator=gen, device="cuda")
    k[:, :, 5::37] *= 4.0
    v = torch.randn(rows, case["nkv"], HEAD_DIM, generator=gen, device="cuda") * 0.3
    return k.to(DTYPES[case["dtype"]]), v.to(DTYPES[case["dtype"]])


def _query(case, rows, gen):
    return (torch.randn(rows, case["nq"], HEAD_DIM, generator=gen, device="cuda") * 0.8).to(DTYPES[case["dtype"]])


def _verify_inputs(case, gen):
    """Logits of a model that agrees with the drafts mostly: noise, and a draft that is likely at `keep` of the places."""
    n, b, vocab = case["n"], case["block"], case["vocab"]
    logits = torch.empty(n, b, vocab, dtype=DTYPES[case["dtype"]], device="cuda")
    drafts = torch.randint(0, vocab, (n, b - 1), generator=gen, device="cuda", dtype=torch.int32)
    likely = torch.rand(n, b - 1, generator=gen, device="cuda") < case["keep"]
    probs = torch.empty(n, b - 1, vocab, device="cuda") if case["probs"] else None
    for i in range(n):
        x = torch.randn(b, vocab, generator=gen, device="cuda") * 2.0
        rest = torch.logsumexp(x, -1)
        at = (torch.arange(b - 1, device="cuda"), drafts[i].long())
        lift = rest[:-1] + math.log(0.95 / 0.05)
        x[at] = torch.where(likely[i], lift, x[at])
        logits[i] = x.to(logits.dtype)
        if probs is not None:
            x = x[:-1] + torch.randn(b - 1, vocab, generator=gen, device="cuda") * 0.5
            x[at] = lift
            probs[i] = torch.softmax(x, -1)
    uniforms = torch.rand(n, b, generator=gen, device="cuda")
    return logits, drafts, uniforms, probs


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if own:
        import importlib
        sd = state["sd"] = importlib.import_module("mirror-sd_b200")
    if case["kind"] == "rope":
        x, starts, lens, positions = _rope_inputs(case, gen)
        state.update(x=x, starts=starts, lens=lens, positions=positions)
        if own:
            state["rope"] = sd.Rope(case["dim"], THETA, rotary_dim=case["rot"], interleaved=case["pairs"] == "interleaved",
                                    scaling=ROPE_SCALING[case["scaling"]], device="cuda")
            if case["step"]:
                state["positions"] = sd.PagedStep(starts, None, lens, None, None)
        else:
            state["freqs"], state["factor"] = _plain_frequencies(case)
    elif case["kind"] == "fork":
        state.update(_fork_inputs(case, gen))
        state["layers"] = list(state["pools"].unbind(0))
        k = case["children"] + 1
        state["keep"] = torch.where(torch.arange(state["lens"].numel(), device="cuda") % k == 0, state["lens"], 0)
    elif case["kind"] == "prefix":
        page = case["page"]
        table, rows, num_pages = _prefix_table(case, gen)
        _, lens, new = _prefix_lens(case)
        if own:
            pool = sd.q4_pool(num_pages, case["nkv"], page, device="cuda")
        else:
            pool = torch.zeros(2, num_pages * page, case["nkv"], HEAD_DIM, dtype=torch.float16, device="cuda")
        for _, _, pages, count in rows:
            if count == 0:
                continue
            pos = torch.arange(count, device="cuda")
            slots = pages.long()[pos // page] * page + pos % page
            k, v = _kv_rows(case, count, gen)
            if own:
                sd.q4_append(k, v, slots.to(torch.int32), pool)
            else:
                pool[0][slots], pool[1][slots] = _plain_stored(k), _plain_stored(v)
        starts = [0]
        for b in new:
            starts.append(starts[-1] + b)
        state.update(q=_query(case, sum(new), gen), pool=pool, table=table, lens=_i32(lens), starts=_i32(starts),
                     host_lens=lens, host_new=new)
        if own:
            # one plan serves all layers of a step
            state["plan"] = sd.paged_prefix_plan(table, state["lens"], [case["members"]] * case["groups"], page,
                                                 starts=state["starts"], max_rows=case["rows"], causal=case["causal"])
            state["workspace"] = sd.q4_prefix_workspace(sum(new), case["rows"], state["plan"].max_group, case["nq"],
                                                        case["nkv"], device="cuda")
    else:
        logits, drafts, uniforms, probs = _verify_inputs(case, gen)
        temps = 1.0 if case["temps"] == "one" else torch.tensor(_temperatures(case), device="cuda")
        state.update(logits=logits, drafts=drafts, uniforms=uniforms, probs=probs, temps=temps,
                     counts=_i32(_verify_counts(case)) if case["ragged"] else None)
    return state


# ---------------------------------------------------------------- the plain form
def _plain_frequencies(case):
    r = case["rot"]
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    s = ROPE_SCALING[case["scaling"]]
    theta = THETA * s["factor"] ** (r / (r - 2)) if s and s["type"] == "ntk" and r > 2 else THETA
    f = theta ** (-2 * i / r)
    if not s or s["type"] == "ntk":
        return f, 1.0
    if s["type"] == "linear":
        return f / s["factor"], 1.0
    # the pairs that turn often keep their frequency, those that turn less than once are stretched
    where = lambda turns: r * math.log(s["original_max_position_embeddings"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
    low, high = max(math.floor(where(32.0)), 0), min(math.ceil(where(1.0)), r - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return f / s["factor"] * ramp + f * (1 - ramp), 0.1 * math.log(s["factor"]) + 1.0


def _plain_rope(state):
    case, x = state["case"], state["x"]
    pos = state["positions"]
    if case["step"]:
        r = torch.arange(x.shape[0], device="cuda")
        seq = torch.searchsorted(state["starts"][1:].long(), r, right=True)
        pos = state["lens"][seq].long() - state["starts"][seq + 1].long() + r
    rot, out = case["rot"], x.clone(memory_format=torch.contiguous_format)
    step = max(1, (1 << 27) // (x.shape[1] * x.shape[2]))
    for a in range(0, x.shape[0], step):
        angle = pos[a:a + step].double()[:, None] * state["freqs"]
        cos, sin = (angle.cos() * state["factor"]).float()[:, None], (angle.sin() * state["factor"]).float()[:, None]
        y = x[a:a + step, :, :rot].float()
        if case["pairs"] == "half":
            u, v = y[..., :rot // 2], y[..., rot // 2:]
            y = torch.cat([u * cos - v * sin, v * cos + u * sin], -1)
        else:
            u, v = y[..., 0::2], y[..., 1::2]
            y = torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2)
        out[a:a + step, :, :rot] = y.to(x.dtype)
    return out


def _plain_fork(state):
    """fork, reserve with copy on write, page copies, release, as tensors."""
    page = state["case"]["page"]
    table, free, holders, pools = state["table"], state["free"], state["holders"], state["pools"]
    n, width = table.shape
    col = torch.arange(width, device="cuda")[None, :]
    src, dst = state["src"].long(), state["dst"].long()
    lens, pages, head = state["lens"].long().clone(), state["pages"].long().clone(), state["head"].long()
    # fork
    take = torch.minimum(pages[src], (lens[src] + page - 1) // page)
    given = col < take[:, None]
    entries = table[src]
    table[dst] = torch.where(given, entries, table[dst])
    holders[0].index_add_(0, entries[given].long(), torch.ones_like(entries[given]))
    lens[dst], pages[dst] = lens[src], take
    # reserve: a request that writes into a page that others hold takes one more page
    new = state["new"].long()
    starts = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
    starts[1:] = torch.cumsum(new, 0)
    tail = table.gather(1, (lens // page).clamp(max=width - 1)[:, None])[:, 0].long()
    writes = (new > 0) & (lens % page > 0)
    extra = torch.where(writes, holders[0].long()[tail.clamp(min=0)], 0)
    shares = writes & (extra > 0)
    same = shares[:, None] & shares[None, :] & (tail[:, None] == tail[None, :])
    rank = torch.tril(same, -1).sum(1)
    moves = shares & (rank < extra)
    want = torch.maximum(pages, (lens + new + page - 1) // page)
    need = want - pages + moves
    first = head + torch.cumsum(need, 0) - need
    old = torch.where(moves, tail, -1)
    fresh = torch.where(moves, free[first.clamp(max=free.numel() - 1)].long(), -1)
    take = (col >= pages[:, None]) & (col < want[:, None])
    at = first[:, None] + moves[:, None] + col - pages[:, None]
    table.copy_(torch.where(take, free[at.clamp(0, free.numel() - 1)], table))
    moved = moves.nonzero()[:, 0]
    table[moved, lens[moved] // page] = fresh[moved].to(torch.int32)
    holders[0].index_add_(0, tail[moved], torch.full_like(tail[moved], -1, dtype=torch.int32))
    r = torch.arange(state["case"]["rows"] * n, device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), r, right=True).clamp(max=n - 1)
    pos = lens[seq] + r - starts[seq]
    slots = table[seq, pos // page].long() * page + pos % page
    copies = torch.stack([old, fresh, torch.where(moves, lens % page, 0)], 1)
    lens_after, head_after = lens + new, head + need.sum()
    # the pages' rows, whole blocks of 16
    for blocks in range(1, page // 16 + 1):
        these = moved[(lens[moved] % page + 15) // 16 == blocks]
        if these.numel():
            pools[:, fresh[these], :, :blocks] = pools[:, old[these], :, :blocks]
    # release: what nobody else holds goes back, in the order of the last that gave it up
    keep = state["keep"].long()
    left = torch.minimum(want, (keep + page - 1) // page)
    back = table[(col >= left[:, None]) & (col < want[:, None])].long()
    order = torch.arange(back.numel(), device="cuda")
    dropped = torch.zeros_like(holders[0]).index_add_(0, back, torch.ones_like(back, dtype=torch.int32))
    last = torch.full((holders.shape[1],), -1, dtype=torch.int64, device="cuda").scatter_reduce_(0, back, order, "amax")
    gone = back[(last[back] == order) & (dropped[back] > holders[0][back])].to(torch.int32)
    holders[0].copy_((holders[0] - dropped).clamp(min=0))
    head_end = head_after - gone.numel()
    free[head_end + torch.arange(gone.numel(), device="cuda")] = gone
    i32 = lambda t: t.to(torch.int32)
    return (i32(starts), i32(slots), i32(lens_after), i32(want), i32(head_after), i32(copies), i32(left), i32(head_end), free,
            holders, table, state["status"], pools)


def _plain_stored(x):
    """What the 4-bit cache stands for after x is appended, exact in f16."""
    x = x.float().unflatten(-1, (8, 16))
    t = x.abs().amax(-1)
    t = t / torch.full_like(t, 7.5)     # a true division: a product with 1 / 7.5 may land above a scale that it equals
    _, e = torch.frexp(t)
    step = torch.ldexp(torch.ones_like(t), (e - 4).clamp(min=-17))
    s = (torch.ceil(t / step) * step).clamp(min=2.0 ** -17, max=9216.0)[..., None]
    q = torch.floor(x.abs() / s + 0.5).clamp(max=7.0)
    return (torch.where(x < 0, -q, q) * s).flatten(-2).to(torch.float16)


def _plain_prefix(state):
    case, page = state["case"], state["case"]["page"]
    nq, nkv, rows = case["nq"], case["nkv"], case["rows"]
    q, out, table = state["q"], torch.zeros_like(state["q"]), state["table"].long()
    starts, lens = state["starts"].long(), state["lens"].long()
    j = torch.arange(rows, device="cuda")[None, :]
    most = max(1, min(16, (1 << 26) // (max(state["host_lens"]) * nkv * HEAD_DIM)))
    for a in range(0, len(state["host_lens"]), most):
        b = min(a + most, len(state["host_lens"]))
        if sum(state["host_new"][a:b]) == 0:
            continue
        width = max(state["host_lens"][a:b])
        new = (starts[a + 1:b + 1] - starts[a:b])[:, None]
        at = (starts[a:b, None] + j).clamp(max=q.shape[0] - 1)
        pos = torch.arange(width, device="cuda")
        slots = (table[a:b][:, pos // page] * page + pos % page).clamp(min=0)
        qq = q[at].float().unflatten(2, (nkv, nq // nkv))
        s = torch.einsum("mjhgd,mkhd->mhgjk", qq, state["pool"][0][slots].float()) * HEAD_DIM ** -0.5
        end = lens[a:b, None] - new + j + 1 if case["causal"] else lens[a:b, None].expand(-1, rows)
        seen = pos < end[:, :, None]
        s = s.masked_fill(~seen[:, None, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
        o = torch.einsum("mhgjk,mkhd->mjhgd", p, state["pool"][1][slots].float()).flatten(2, 3)
        real = j < new
        out[at[real]] = o[real].to(out.dtype)
    return out


def _plain_verify(state):
    logits, drafts, u, probs = state["logits"], state["drafts"].long(), state["uniforms"], state["probs"]
    n, block, vocab = logits.shape
    temps = state["temps"] if torch.is_tensor(state["temps"]) else torch.full((n,), state["temps"], device="cuda")
    counts = state["counts"].long() if state["counts"] is not None else torch.full((n,), block - 1, device="cuda")
    index = torch.arange(vocab, device="cuda")
    accepted, tokens = [], []
    for i in range(n):
        x = logits[i].float()
        top = x.amax(-1, keepdim=True)
        first = torch.where(x == top, index, vocab).amin(-1)
        greedy = temps[i] < 1e-5
        t = torch.where(greedy, torch.ones_like(temps[i]), temps[i])
        d = drafts[i][:, None]
        total = torch.exp((x - top) / t).sum(-1, dtype=torch.float64)[:-1]
        p = torch.exp((x[:-1].gather(1, d) - top[:-1]).double()[:, 0] / t.double()) / total
        p = torch.where(greedy, (first[:-1] == drafts[i]).double(), p)
        q = probs[i].gather(1, d)[:, 0].double() if probs is not None else torch.ones_like(p)
        good = (u[i, :-1].double() * q < p) & (torch.arange(block - 1, device="cuda") < counts[i])
        a = torch.cumprod(good.long(), 0).sum()
        # the row behind the accepted drafts, in 64 bits
        x = x.index_select(0, a[None])[0].double()
        x = torch.exp((x - x.amax()) / t.double())
        x = torch.where(greedy, (index == first.index_select(0, a[None])).double(), x)
        x = x / x.sum()
        r = x
        if block > 1:
            j = a.clamp(max=block - 2)[None]
            if probs is not None:
                q = probs[i].index_select(0, j)[0].double()
            else:
                q = (index == drafts[i].index_select(0, j)).double()
            r = torch.where(a < counts[i], (x - q).clamp(min=0), x)
            r = torch.where(r.sum() > 0, r, x)
        c = torch.cumsum(r, 0)
        tokens.append(torch.searchsorted(c, u[i, -1].double() * c[-1], right=True).clamp(max=vocab - 1))
        accepted.append(a)
    return torch.stack(accepted).to(torch.int32), torch.stack(tokens).to(torch.int32)


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        return {"rope": _plain_rope, "fork": _plain_fork, "prefix": _plain_prefix, "verify": _plain_verify}[kind](state)
    sd = state["sd"]
    if kind == "rope":
        return sd.apply_rope(state["x"], state["rope"], state["positions"])
    if kind == "fork":
        page, table, free, holders, status = (case["page"], state["table"], state["free"], state["holders"], state["status"])
        lens, pages = sd.paged_fork(state["src"], state["dst"], state["lens"], state["pages"], table, holders,
                                    page_size=page, status=status)
        step, copies = sd.paged_reserve_forked(lens, state["new"], pages, table, free, state["head"], holders, page_size=page,
                                               num_slots=state["new"].numel() * case["rows"], status=status)
        sd.q4_copy_pages(state["layers"], copies)
        left, head = sd.paged_release_forked(state["keep"], step.pages, table, free, step.head, holders, page_size=page,
                                             status=status)
        return (step.starts, step.slots, step.lens, step.pages, step.head, copies, left, head, free, holders, table, status,
                state["pools"])
    if kind == "prefix":
        return sd.q4_prefix_attention(state["q"], state["pool"], state["table"], state["plan"], scale=HEAD_DIM ** -0.5,
                                      workspace=state["workspace"])
    return sd.verify_drafts(state["logits"], state["drafts"], state["uniforms"], state["temps"], draft_probs=state["probs"],
                            num_drafts=state["counts"])


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"rope": _exact_rope, "fork": _exact_fork, "prefix": _exact_prefix, "verify": _exact_verify}[case["kind"]](case, gen)


def _exact_rope(case, gen):
    x, starts, lens, positions = _rope_inputs(case, gen)
    if case["step"]:
        positions = torch.cat([torch.arange(L - m, L, device="cuda") for m, L in zip(*_rope_rows(case))])
    r, s, out = case["rot"], ROPE_SCALING[case["scaling"]], x.double()
    kind = s["type"] if s else "none"
    turned = torch.empty_like(out[:, :, :r])
    for i in range(r // 2):
        base = THETA * s["factor"] ** (r / (r - 2)) if kind == "ntk" and r > 2 else THETA
        f, factor = base ** (-2.0 * i / r), 1.0
        if kind == "linear":
            f /= s["factor"]
        if kind == "yarn":
            edge = [r * math.log(s["original_max_position_embeddings"] / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (32, 1)]
            low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), r - 1)
            stretched = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            f, factor = f * (1 - stretched + stretched / s["factor"]), 1.0 + 0.1 * math.log(s["factor"])
        a, b = (i, i + r // 2) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
        turn = torch.polar(torch.full_like(positions, factor, dtype=torch.float64), positions.double() * f)[:, None]
        z = torch.complex(out[:, :, a], out[:, :, b]) * turn
        turned[:, :, a], turned[:, :, b] = z.real, z.imag
    out[:, :, :r] = turned
    return out


def _exact_fork(case, gen):
    """One request after another on the host."""
    s = _fork_inputs(case, gen)
    page, rows, k = case["page"], case["rows"], case["children"] + 1
    table, free, head = s["table"].cpu().numpy(), s["free"].cpu().numpy(), int(s["head"])
    lens, pages = s["lens"].tolist(), s["pages"].tolist()
    held = [list(table[i, :h]) for i, h in enumerate(pages)]
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        held[b], lens[b] = list(held[a]), lens[a]
        table[b, :len(held[b])] = held[b]
    owners = {}
    for row in held:
        for p in row:
            owners[p] = owners.get(p, 0) + 1
    starts, slots, copies = [0], [], []
    for i, row in enumerate(held):
        copy = [-1, -1, 0]
        c = lens[i] // page
        if lens[i] % page and owners[row[c]] > 1:
            copy = [row[c], free[head], lens[i] % page]
            owners[row[c]] -= 1
            row[c] = table[i, c] = free[head]
            owners[row[c]] = 1
            head += 1
        while len(row) * page < lens[i] + rows:
            table[i, len(row)] = free[head]
            row.append(free[head])
            owners[free[head]] = 1
            head += 1
        slots += [int(row[r // page]) * page + r % page for r in range(lens[i], lens[i] + rows)]
        lens[i] += rows
        starts.append(starts[-1] + rows)
        copies.append(copy)
    for a, b, m in copies:
        if a >= 0:
            blocks = _cdiv(m, 16)
            s["pools"][:, int(b), :, :blocks] = s["pools"][:, int(a), :, :blocks]
    pages, head_after, gone, left = [len(row) for row in held], head, [], []
    for i, row in enumerate(held):
        left.append(_cdiv(lens[i] - rows, page) if i % k == 0 else 0)
        for p in row[left[i]:]:
            owners[p] -= 1
            if owners[p] == 0:
                gone.append(p)
    free[head - len(gone):head] = gone
    holders = torch.zeros_like(s["holders"])
    for p, c in owners.items():
        holders[0, int(p)] = max(c - 1, 0)
    return (_i32(starts), _i32(slots), _i32(lens), _i32(pages), _i32([head_after]), _i32([[int(v) for v in c] for c in copies]),
            _i32(left), _i32([head - len(gone)]), torch.from_numpy(free).cuda(), holders, torch.from_numpy(table).cuda(),
            torch.zeros_like(s["status"]), s["pools"])


def _exact_stored(x):
    steps = [m * 2.0 ** -17 for m in range(1, 8)] + [m * 2.0 ** (e - 17) for e in range(0, 31) for m in range(8, 16)]
    scales = torch.tensor([s for s in steps if s <= 9216.0], dtype=torch.float64, device="cuda")
    x = x.double().reshape(*x.shape[:-1], 8, 16)
    s = scales[torch.searchsorted(scales * 7.5, x.abs().amax(-1)).clamp(max=scales.numel() - 1)].unsqueeze(-1)
    return (torch.sign(x) * torch.clamp(torch.floor(x.abs() / s + 0.5), max=7.0) * s).flatten(-2)


def _exact_prefix(case, gen):
    """One request after another, its shared rows and its own."""
    _, rows, _ = _prefix_table(case, gen)
    shared, lens, new = _prefix_lens(case)
    stored = {}
    for what, i, _, count in rows:
        if count:
            stored[what, i] = tuple(_exact_stored(x) for x in _kv_rows(case, count, gen))
    q = _query(case, sum(new), gen).double()
    out, at, g = torch.zeros_like(q), 0, case["nq"] // case["nkv"]
    for i, (a, b) in enumerate(zip(lens, new)):
        if b == 0:
            continue
        parts = [stored[key] for key in (("group", i // case["members"]), ("own", i)) if key in stored]
        k, v = (torch.cat(x).permute(1, 0, 2) for x in zip(*parts))                                  # [nkv, a, 128]
        x = q[at:at + b].reshape(b, case["nkv"], g, HEAD_DIM).permute(1, 2, 0, 3).flatten(1, 2)       # [nkv, g b, 128]
        s = x @ k.transpose(1, 2) / math.sqrt(HEAD_DIM)
        if case["causal"]:
            hidden = torch.arange(a, device="cuda")[None, :] > torch.arange(a - b, a, device="cuda")[:, None]
            s = s.masked_fill(hidden.repeat(g, 1), -math.inf)
        o = torch.softmax(s, -1) @ v
        out[at:at + b] = o.reshape(case["nkv"], g, b, HEAD_DIM).permute(2, 0, 1, 3).flatten(1, 2)
        at += b
    return out


def _exact_verify(case, gen):
    logits, drafts, uniforms, probs = _verify_inputs(case, gen)
    counts, temps, vocab = _verify_counts(case), _temperatures(case), case["vocab"]
    accepted, tokens = [], []
    for i in range(case["n"]):
        u = uniforms[i].tolist()
        for j in range(counts[i] + 1):
            x = logits[i, j].double()
            if temps[i] == 0.0:
                p = torch.zeros_like(x)
                p[int((x == x.max()).nonzero()[0])] = 1.0
            else:
                p = torch.softmax(x / torch.tensor(temps[i], dtype=torch.float32).double().item(), 0)
            q = torch.zeros_like(x)
            if j < counts[i]:
                d = int(drafts[i, j])
                if probs is None:
                    q[d] = 1.0
                else:
                    q = probs[i, j].double()
                if u[j] * float(q[d]) < float(p[d]):
                    continue
            r = torch.clamp(p - q, min=0.0)
            if float(r.sum()) == 0.0:
                r = p
            run_sum = torch.cumsum(r, 0)
            accepted.append(j)
            tokens.append(min(int((run_sum <= u[-1] * float(run_sum[-1])).sum()), vocab - 1))
            break
    return _i32(accepted), _i32(tokens)
