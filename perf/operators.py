"""Cases of the paged 4-bit K/V cache operators, for timing and comparison.

Four operators, in the order in which a serving step calls them:

reserve  block tables and slot maps on the GPU: from the requests' lengths and
         the rows that each brings, pages off a free list into the block table,
         and the cache slot of every new row
append   K and V rows into their slots, 16 channels at a time as 4-bit whole
         numbers and one 8-bit scale (then read back: the values that the
         cache now stands for)
attend   grouped-query attention of each request's query rows over its cached
         rows, through the block table
release  the pages beyond the rows that a request keeps go back to the list

A cached row's group of 16 channels is x ~ q * s.  With a = max |x| (NaN counts
as 0), s is the smallest value >= a / 7.5 that has 3 mantissa bits, an exponent
of float16's range and at most 9216 (at least 2^-17), and q = x / s rounded to
the nearest whole number, halves away from 0, at most 7 in magnitude.

Query row j (of n) of a request with L cached rows has its keys end at
e = L - n + j + 1 (causal) or e = L, and sees key k < e where k < sink or
k >= e - window (window = 0: all).  A row that sees no key gives zeros.
"""
import math
import random

import torch

own = False

HEAD_DIM = 128
GROUP = 16
SCALE_CAP = 9216.0
SCALE_MIN = 2.0 ** -17
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one request with a 4K context brings its 32 block rows
        dict(name="reserve_one", kind="reserve", n=1, ctx=4096, spread="equal", rows=32, page=64, short=False, shape=1),
        # 256 requests in flight, 16 rows each, contexts of the serving benchmark
        dict(name="reserve_serving", kind="reserve", n=256, ctx=8192, spread="ragged", rows=16, page=64, short=False,
             shape=2),
        # the same batch gives back what verification rejected
        dict(name="release_trim", kind="release", n=256, ctx=8192, spread="ragged", page=64, finish=0.0, shape=3),
        # many long requests, a quarter of them finished, small pages
        dict(name="release_finish", kind="release", n=1000, ctx=32768, spread="ragged", page=16, finish=0.25, shape=4),
        # one new row for each of 256 requests, out of a fused q|k|v projection
        dict(name="append_decode", kind="append", rows=256, nq=32, nkv=8, page=64, dtype="bf16", fused=True, holes=0.0),
        # a 4K prompt and its block rows
        dict(name="append_prompt", kind="append", rows=4128, nq=40, nkv=8, page=64, dtype="f16", fused=False, holes=0.0),
        # a prefill round over many requests, some rows turned away
        dict(name="append_prefill", kind="append", rows=65521, nq=32, nkv=8, page=32, dtype="bf16", fused=True,
             holes=0.01),
        # the latency of one token of one request
        dict(name="attend_token", kind="attend", n=1, ctx=2049, spread="equal", rows=1, ragged_rows=False, nq=32, nkv=8,
             page=64, causal=True, sink=0, window=0, dtype="bf16", shape=5),
        # one token each of 256 requests
        dict(name="attend_decode", kind="attend", n=256, ctx=8192, spread="ragged", rows=1, ragged_rows=False, nq=32,
             nkv=8, page=64, causal=True, sink=0, window=0, dtype="bf16", shape=6),
        # the drafter's block rows over its sink and window, all requests
        dict(name="attend_draft", kind="attend", n=256, ctx=8192, spread="ragged", rows=16, ragged_rows=False, nq=32,
             nkv=8, page=64, causal=False, sink=64, window=1040, dtype="f16", shape=7),
        # verification of ragged drafts over long contexts, odd lengths, small pages
        dict(name="attend_verify", kind="attend", n=16, ctx=32768, spread="ragged", rows=32, ragged_rows=True, nq=40,
             nkv=8, page=32, causal=True, sink=0, window=0, dtype="bf16", shape=8),
        # one request's 32 block rows over a 32K context
        dict(name="attend_long", kind="attend", n=1, ctx=32800, spread="equal", rows=32, ragged_rows=False, nq=40, nkv=8,
             page=64, causal=False, sink=0, window=0, dtype="f16", shape=9),
    ]


def _log_int(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    kind = rng.choice(["reserve", "release", "append", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    shape = rng.randrange(1 << 30)
    spread = rng.choice(["equal", "ragged"])
    if kind == "reserve":
        n = _log_int(rng, 1, 1000)
        return dict(kind=kind, n=n, ctx=_log_int(rng, 1, 32768), spread=spread,
                    rows=_log_int(rng, 1, min(4096, 65536 // n)), page=page, short=rng.random() < 0.25, shape=shape)
    if kind == "release":
        return dict(kind=kind, n=_log_int(rng, 1, 1000), ctx=_log_int(rng, 1, 32768), spread=spread, page=page,
                    finish=rng.choice([0.0, 0.1, 1.0]), shape=shape)
    nq, nkv = rng.choice([(32, 8), (40, 8), (4, 2), (12, 4), (8, 8), (16, 1), (32, 4), (28, 4)])
    dtype = rng.choice(["f16", "bf16"])
    if kind == "append":
        return dict(kind=kind, rows=_log_int(rng, 1, 65521 * 8 // max(nkv, 8)), nq=nq, nkv=nkv, page=page, dtype=dtype,
                    fused=rng.random() < 0.5, holes=rng.choice([0.0, 0.05]))
    ctx = _log_int(rng, 1, 32768)
    rows = rng.choice([1, _log_int(rng, 1, 64)])
    # no more cached rows than attend_decode reads, no more products than attend_verify's
    most = min(256, 256 * 4352 // ctx, int(1.5e11 / (512.0 * nq * rows * ctx)))
    n = _log_int(rng, 1, max(1, most))
    windowed = rng.random() < 0.3
    return dict(kind=kind, n=n, ctx=ctx, spread=spread, rows=rows, ragged_rows=rng.random() < 0.5, nq=nq, nkv=nkv,
                page=page, causal=rng.random() < 0.5, sink=rng.choice([0, 5, 64]) if windowed else 0,
                window=_log_int(rng, 1, 2048) if windowed else 0, dtype=dtype, shape=shape)


def _cdiv(a, b):
    return -(-a // b)


def _lens(case):
    """The requests' cached rows, from the case alone."""
    rng = random.Random(case["shape"])
    n, ctx = case["n"], case["ctx"]
    if case["spread"] == "equal":
        return [ctx] * n
    lens = [rng.randint(max(1, ctx // 16), ctx) for _ in range(n)]
    if n >= 4:
        lens[n // 2] = 0          # a slot without a request
    return lens


def _new_rows(case, lens):
    """Query rows (attend) or new rows (reserve) of each request."""
    rng = random.Random(case["shape"] + 1)
    most = case["rows"]
    if case["kind"] == "reserve":
        ragged = case["spread"] == "ragged"
        return [rng.randint(0, most) if ragged else most for _ in lens]
    if case["ragged_rows"]:
        return [rng.randint(0, most) for _ in lens[:-1]] + [most]
    return [most] * len(lens)


def _visible(case, length, rows, j):
    """Number of keys that query row j of `rows` sees."""
    end = length - rows + j + 1 if case["causal"] else length
    if end <= 0:
        return 0
    if case["window"] == 0:
        return end
    return end - max(0, end - case["window"] - min(end, case["sink"]))


def work(case):
    if case["kind"] == "reserve":
        lens = _lens(case)
        new = _new_rows(case, lens)
        taken = sum(_cdiv(a + b, case["page"]) - _cdiv(a, case["page"]) for a, b in zip(lens, new))
        touched = sum(_cdiv(a + b, case["page"]) - a // case["page"] for a, b in zip(lens, new))
        return {"bytes": 24 * case["n"] + 4 * sum(new) + 4 * taken + 4 * touched, "flops": 0}
    if case["kind"] == "release":
        lens = _lens(case)
        keep = _keep(case, lens)
        freed = sum(_cdiv(a, case["page"]) - _cdiv(b, case["page"]) for a, b in zip(lens, keep))
        return {"bytes": 12 * case["n"] + 8 * freed, "flops": 0}
    if case["kind"] == "append":
        # rows in, packed rows out and in again, values out; an absolute maximum and a rounding each
        elems = case["rows"] * case["nkv"] * HEAD_DIM * 2
        return {"bytes": elems * 2 + 2 * elems * 9 // 16 + elems * 2 + 4 * case["rows"], "flops": 4 * elems}
    lens = _lens(case)
    new = _new_rows(case, lens)
    pairs = keys = 0
    for a, b in zip(lens, new):
        pairs += sum(_visible(case, a, b, j) for j in range(b))
        if b and case["window"]:
            low = max(0, (a - b + 1 if case["causal"] else a) - case["window"])
            keys += a - max(0, low - case["sink"])
        elif b:
            keys += a
    return {"bytes": keys * case["nkv"] * 144 + 4 * sum(new) * case["nq"] * HEAD_DIM + 4 * keys // case["page"],
            "flops": 4 * HEAD_DIM * case["nq"] * pairs}


def _keep(case, lens):
    """Rows that each request keeps: all but what verification rejected, or none."""
    rng = random.Random(case["shape"] + 2)
    return [0 if rng.random() < case["finish"] else max(0, a - rng.randint(0, 40)) for a in lens]


# ---------------------------------------------------------------- inputs
def _kv_rows(case, rows, gen):
    """K and V rows as a layer makes them: normed keys with a few strong channels, smaller values."""
    nkv = case["nkv"]
    k = torch.randn(rows, nkv, HEAD_DIM, generator=gen, device="cuda")
    strong = torch.ones(nkv, HEAD_DIM, device="cuda")
    strong[:, 5::37] = 4.0
    v = torch.randn(rows, nkv, HEAD_DIM, generator=gen, device="cuda") * 0.3
    dt = DTYPES[case["dtype"]]
    return (k * strong).to(dt), v.to(dt)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _paging(case, lens, held, gen, max_pages, spare):
    """Block table and free list of requests that hold `held` pages each."""
    total = sum(held)
    perm = torch.randperm(total + spare, generator=gen, device="cuda").to(torch.int32)
    width = torch.arange(max_pages, device="cuda")[None, :]
    held_t = torch.tensor(held, device="cuda")[:, None]
    first = torch.cumsum(held_t, 0) - held_t
    at = (first + width).clamp(max=max(total + spare - 1, 0))
    table = torch.where(width < held_t, perm[at], torch.full_like(perm[at], -1))
    return table.contiguous(), perm


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if own:
        import importlib
        state["sd"] = importlib.import_module("mirror-sd_b200")
    if case["kind"] in ("reserve", "release"):
        lens = _lens(case)
        held = [_cdiv(a, case["page"]) for a in lens]
        if case["kind"] == "reserve":
            new = _new_rows(case, lens)
            need = sum(_cdiv(a + b, case["page"]) - h for a, b, h in zip(lens, new, held))
            max_pages = max(_cdiv(case["ctx"] + case["rows"], case["page"]), 1)
            spare = need // 2 if case["short"] else need + need // 8 + 1
            state["new"] = _i32(new)
            state["capacity"] = max(case["n"] * case["rows"], 1)
        else:
            keep = _keep(case, lens)
            max_pages = max(_cdiv(case["ctx"], case["page"]), 1)
            spare = 7
            state["keep"] = _i32(keep)
        table, free = _paging(case, lens, held, gen, max_pages, spare)
        state.update(lens=_i32(lens), pages=_i32(held), table=table, free=free, head=_i32([sum(held)]),
                     status=torch.zeros(1, dtype=torch.int32, device="cuda"))
        return state
    if case["kind"] == "append":
        rows, nq, nkv, page = case["rows"], case["nq"], case["nkv"], case["page"]
        k, v = _kv_rows(case, rows, gen)
        if case["fused"]:
            wide = torch.zeros(rows, (nq + 2 * nkv) * HEAD_DIM, dtype=k.dtype, device="cuda")
            kk = wide[:, nq * HEAD_DIM:(nq + nkv) * HEAD_DIM].view(rows, nkv, HEAD_DIM)
            vv = wide[:, (nq + nkv) * HEAD_DIM:].view(rows, nkv, HEAD_DIM)
            kk.copy_(k)
            vv.copy_(v)
            k, v = kk, vv
        # runs of consecutive rows on pages in no order
        num_pages = _cdiv(rows, page) + 3
        perm = torch.randperm(num_pages, generator=gen, device="cuda")
        r = torch.arange(rows, device="cuda")
        slots = (perm[r // page] * page + r % page).to(torch.int32)
        if case["holes"]:
            slots[torch.rand(rows, generator=gen, device="cuda") < case["holes"]] = -1
        state.update(k=k, v=v, slots=slots)
        if own:
            state["pool"] = state["sd"].q4_pool(num_pages, nkv, page, device="cuda")
        else:
            state["pool"] = _plain_pool(num_pages * page, nkv)
        return state
    # attend: a filled cache and query rows
    lens = _lens(case)
    new = _new_rows(case, lens)
    page, nq, nkv = case["page"], case["nq"], case["nkv"]
    held = [_cdiv(a, page) for a in lens]
    max_pages = max(_cdiv(case["ctx"], page), 1)
    table, free = _paging(case, lens, held, gen, max_pages, 2)
    num_pages = int(free.numel())
    if own:
        pool = state["sd"].q4_pool(num_pages, nkv, page, device="cuda")
    else:
        pool = _plain_pool(num_pages * page, nkv)
    for slots, k, v in _fill(case, lens, table, gen):
        if own:
            state["sd"].q4_append(k, v, slots.to(torch.int32), pool)
        else:
            _plain_append(k, v, slots, pool)
    state["q"] = _query(case, sum(new), gen)
    starts = [0]
    for b in new:
        starts.append(starts[-1] + b)
    state.update(pool=pool, table=table, lens=_i32(lens), starts=_i32(starts), host_lens=lens, host_new=new)
    if own:
        state["workspace"] = state["sd"].q4_attention_workspace(len(lens), case["rows"], nq, nkv, device="cuda")
    return state


def _query(case, rows, gen):
    q = torch.randn(rows, case["nq"], HEAD_DIM, generator=gen, device="cuda") * 0.8
    return q.to(DTYPES[case["dtype"]])


def _fill(case, lens, table, gen):
    """The cached rows, a few requests at a time: (slots, k, v)."""
    page = case["page"]
    for i, a in enumerate(lens):
        if a:
            pos = torch.arange(a, device="cuda")
            k, v = _kv_rows(case, a, gen)
            yield table[i].long()[pos // page] * page + pos % page, k, v


# ---------------------------------------------------------------- the plain form
def _plain_pool(slots, nkv):
    """Codes (two 4-bit numbers to a byte, each q + 8) and scales of K and V."""
    pool = {}
    for name in ("k", "v"):
        pool[name] = torch.full((slots, nkv, HEAD_DIM // 2), 0x88, dtype=torch.uint8, device="cuda")
        pool[name + "s"] = torch.zeros(slots, nkv, HEAD_DIM // GROUP, dtype=torch.float16, device="cuda")
    return pool


def _plain_quantize(x):
    """[..., 128] -> whole numbers -7..7 (fp32) and scales (fp32, [..., 8])."""
    x = x.float()
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x).unflatten(-1, (HEAD_DIM // GROUP, GROUP))
    a = x.abs().amax(-1)
    t = a / torch.full_like(a, 7.5)     # a true division: a times 1 / 7.5 may land above a scale that is a / 7.5
    _, e = torch.frexp(t)
    step = torch.ldexp(torch.ones_like(t), (e - 4).clamp(min=-17))
    s = (torch.ceil(t / step) * step).clamp(min=SCALE_MIN, max=SCALE_CAP)
    q = torch.floor(x.abs() / s[..., None] + 0.5).clamp(max=7.0)
    return torch.where(x < 0, -q, q).flatten(-2), s


def _plain_append(k, v, slots, pool):
    keep = slots >= 0
    at = slots.long()[keep]
    for name, x in (("k", k), ("v", v)):
        q, s = _plain_quantize(x[keep])
        u = (q + 8).to(torch.uint8)
        pool[name][at] = u[..., 0::2] | (u[..., 1::2] << 4)
        pool[name + "s"][at] = s.to(torch.float16)


def _plain_values(pool, name, at):
    """fp32 values of the rows at slots `at`."""
    b = pool[name][at]
    u = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    s = pool[name + "s"][at].float()
    x = (u.float() - 8.0).unflatten(-1, (HEAD_DIM // GROUP, GROUP)) * s[..., None]
    return x.flatten(-2)


def _plain_read(slots, pool):
    out = []
    for name in ("k", "v"):
        x = _plain_values(pool, name, slots.long().clamp(min=0))
        out.append(torch.where((slots >= 0)[:, None, None], x, torch.zeros_like(x)).to(torch.float16))
    return tuple(out)


def _plain_reserve(state):
    page = state["case"]["page"]
    lens, new, pages = state["lens"].long(), state["new"].long(), state["pages"].long()
    table, free, head, capacity = state["table"], state["free"], state["head"].long(), state["capacity"]
    n, max_pages = table.shape
    starts = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
    starts[1:] = torch.cumsum(new, 0)
    want = (lens + new + page - 1) // page
    long = want > max_pages
    over = starts[1:] > capacity
    need = torch.where(long | over, torch.zeros_like(want), (want - pages).clamp(min=0))
    upto = torch.cumsum(need, 0)
    dry = (need > 0) & (upto > free.numel() - head)
    served = ~(long | over | dry)
    lens_after = torch.where(served, lens + new, lens)
    pages_after = torch.where(served, torch.maximum(pages, want), pages)
    head_after = head + torch.where(served, need, torch.zeros_like(need)).sum()
    col = torch.arange(max_pages, device="cuda")[None, :]
    src = head + (upto - need)[:, None] + col - pages[:, None]
    take = (col >= pages[:, None]) & (col < pages_after[:, None])
    table.copy_(torch.where(take, free[src.clamp(0, free.numel() - 1)], table))
    r = torch.arange(capacity, device="cuda")
    i = torch.searchsorted(starts[1:].contiguous(), r, right=True).clamp(max=n - 1)
    pos = lens[i] + r - starts[i]
    entry = table[i, (pos // page).clamp(0, max_pages - 1)].long()
    slots = torch.where((r < starts[n]) & served[i], entry * page + pos % page, torch.full_like(r, -1))
    status = dry.any().int() + 2 * long.any().int() + 4 * over.any().int()
    i32 = torch.int32
    return (starts.to(i32), slots.to(i32), lens_after.to(i32), pages_after.to(i32), head_after.to(i32), table,
            status.to(i32).reshape(1))


def _plain_release(state):
    page = state["case"]["page"]
    keep, pages, head = state["keep"].long(), state["pages"].long(), state["head"].long()
    table, free = state["table"], state["free"]
    left = torch.minimum(pages, (keep + page - 1) // page)
    back = pages - left
    upto = torch.cumsum(back, 0)
    head_after = head - upto[-1]
    col = torch.arange(table.shape[1], device="cuda")[None, :]
    give = (col >= left[:, None]) & (col < pages[:, None])
    dst = (head_after + (upto - back)[:, None] + col - left[:, None])[give]
    free[dst] = table[give]
    return left.to(torch.int32), head_after.to(torch.int32), free


def _visible_mask(case, lens, new, rows, width):
    """[m, rows, width]: which keys each query row sees."""
    j = torch.arange(rows, device="cuda")[None, :]
    end = lens[:, None] - new[:, None] + j + 1 if case["causal"] else lens[:, None].expand(-1, rows)
    end = torch.where(j < new[:, None], end, torch.zeros_like(end))[..., None]
    key = torch.arange(width, device="cuda")[None, None, :]
    seen = key < end
    if case["window"]:
        seen = seen & ((key < case["sink"]) | (key >= end - case["window"]))
    return seen


def _chunks(lens, most):
    """Runs of requests whose padded rows stay under `most`."""
    a = 0
    while a < len(lens):
        b, width = a, 0
        while b < len(lens) and (b == a or (b - a + 1) * max(width, lens[b]) <= most):
            width = max(width, lens[b])
            b += 1
        yield a, b, width
        a = b


def _plain_attend(state):
    case, page = state["case"], state["case"]["page"]
    nq, nkv, rows = case["nq"], case["nkv"], case["rows"]
    q, out = state["q"], torch.zeros_like(state["q"])
    starts, lens, table = state["starts"].long(), state["lens"].long(), state["table"].long()
    j = torch.arange(rows, device="cuda")[None, :]
    for a, b, width in _chunks(state["host_lens"], 65536):
        if width == 0 or sum(state["host_new"][a:b]) == 0:
            continue
        new = starts[a + 1:b + 1] - starts[a:b]
        at = (starts[a:b, None] + j).clamp(max=q.shape[0] - 1)
        qq = q[at].float().unflatten(2, (nkv, nq // nkv))                       # [m, rows, nkv, G, 128]
        pos = torch.arange(width, device="cuda")
        slots = (table[a:b][:, pos // page] * page + pos % page).clamp(min=0)   # [m, width]
        s = torch.einsum("mjhgd,mkhd->mhgjk", qq, _plain_values(state["pool"], "k", slots)) * HEAD_DIM ** -0.5
        seen = _visible_mask(case, lens[a:b], new, rows, width)[:, None, None]
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, torch.ones_like(total))
        o = torch.einsum("mhgjk,mkhd->mjhgd", p, _plain_values(state["pool"], "v", slots)).flatten(2, 3)
        real = j < new[:, None]
        out[at[real]] = o[real].to(out.dtype)
    return out


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "reserve":
            return _plain_reserve(state)
        if kind == "release":
            return _plain_release(state)
        if kind == "append":
            _plain_append(state["k"], state["v"], state["slots"], state["pool"])
            return _plain_read(state["slots"], state["pool"])
        return _plain_attend(state)
    sd = state["sd"]
    if kind == "reserve":
        step = sd.paged_reserve(state["lens"], state["new"], state["pages"], state["table"], state["free"], state["head"],
                                page_size=case["page"], num_slots=state["capacity"], status=state["status"])
        return step.starts, step.slots, step.lens, step.pages, step.head, state["table"], state["status"]
    if kind == "release":
        pages, head = sd.paged_release(state["keep"], state["pages"], state["table"], state["free"], state["head"],
                                       page_size=case["page"], status=state["status"])
        return pages, head, state["free"]
    if kind == "append":
        sd.q4_append(state["k"], state["v"], state["slots"], state["pool"])
        return sd.q4_read(state["pool"], state["slots"])
    return sd.q4_attention(state["q"], state["pool"], state["table"], state["lens"], starts=state["starts"],
                           max_rows=case["rows"], causal=case["causal"], sink=case["sink"], window=case["window"],
                           workspace=state["workspace"])


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_scales():
    """Every scale the format has, ascending: whole multiples of 2^-17 up to 7, then 8..15 at each exponent."""
    steps = [m * 2.0 ** -17 for m in range(1, 8)]
    steps += [m * 2.0 ** (e - 17) for e in range(0, 31) for m in range(8, 16)]
    return torch.tensor([s for s in steps if s <= SCALE_CAP], dtype=torch.float64, device="cuda")


def _exact_values(x):
    """What the cache stands for after a row x is appended, in 64 bits."""
    x = x.double()
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x).reshape(*x.shape[:-1], HEAD_DIM // GROUP, GROUP)
    scales = _exact_scales()
    peak = x.abs().max(-1).values
    s = scales[torch.searchsorted(scales * 7.5, peak).clamp(max=scales.numel() - 1)].unsqueeze(-1)
    q = torch.clamp(torch.floor(x.abs() / s + 0.5), max=7.0)
    return (torch.sign(x) * q * s).reshape(*x.shape[:-2], HEAD_DIM)


def _exact_pages(case, state):
    """reserve and release, one request after another on the host."""
    page = case["page"]
    free, head = state["free"].cpu().numpy().copy(), int(state["head"][0])
    table, pages = state["table"].cpu().numpy().copy(), state["pages"].tolist()
    if case["kind"] == "release":
        keep = state["keep"].tolist()
        left = [min(h, _cdiv(a, page)) for h, a in zip(pages, keep)]
        at = head - (sum(pages) - sum(left))
        first = at
        for i, (a, b) in enumerate(zip(left, pages)):
            free[at:at + b - a] = table[i, a:b]
            at += b - a
        return _i32(left), _i32([first]), torch.from_numpy(free).cuda()
    lens, new, capacity = state["lens"].tolist(), state["new"].tolist(), state["capacity"]
    room, start, starts, slots, status = free.size - head, 0, [0], [-1] * capacity, 0
    lens_after, pages_after, asked, given = [], [], 0, 0
    for i, (a, b, h) in enumerate(zip(lens, new, pages)):
        want = _cdiv(a + b, page)
        start += b
        starts.append(start)
        turned = (2 if want > table.shape[1] else 0) | (4 if start > capacity else 0)
        need = 0 if turned else max(0, want - h)
        asked += need
        if need and asked > room:
            turned |= 1
        status |= turned
        if turned:
            lens_after.append(a)
            pages_after.append(h)
            continue
        table[i, h:h + need] = free[head + given:head + given + need]
        given += need
        lens_after.append(a + b)
        pages_after.append(max(h, want))
        for r in range(b):
            pos = a + r
            slots[start - b + r] = int(table[i, pos // page]) * page + pos % page
    return (_i32(starts), _i32(slots), _i32(lens_after), _i32(pages_after), _i32([head + given]),
            torch.from_numpy(table).cuda(), _i32([status]))


def exact(case, seed):
    global own
    was, own = own, False
    try:
        if case["kind"] == "attend":
            return _exact_attend(case, seed)
        state = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "append":
        there = (state["slots"] >= 0)[:, None, None]
        return tuple(torch.where(there, _exact_values(x), 0.0) for x in (state["k"], state["v"]))
    return _exact_pages(case, state)


def _exact_attend(case, seed):
    """One request and one head group at a time; the inputs come off the generator in prepare's order."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens = _lens(case)
    new = _new_rows(case, lens)
    nq, nkv = case["nq"], case["nkv"]
    table, _ = _paging(case, lens, [_cdiv(a, case["page"]) for a in lens], gen, max(_cdiv(case["ctx"], case["page"]), 1), 2)
    # the query rows come last off the generator: a first walk over the cached rows finds them
    for _ in _fill(case, lens, table, gen):
        pass
    q = _query(case, sum(new), gen).double()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    _paging(case, lens, [_cdiv(a, case["page"]) for a in lens], gen, max(_cdiv(case["ctx"], case["page"]), 1), 2)
    rows = _fill(case, lens, table, gen)
    out = torch.zeros_like(q)
    at = 0
    for a, b in zip(lens, new):
        if a == 0:
            at += b
            continue
        _, k, v = next(rows)
        if b:
            k, v = _exact_values(k), _exact_values(v)
            seen = torch.zeros(b, a, dtype=torch.bool, device="cuda")
            for j in range(b):
                end = a - b + j + 1 if case["causal"] else a
                if end > 0:
                    seen[j, max(0, end - case["window"]) if case["window"] else 0:end] = True
                    seen[j, :min(case["sink"], end)] = True
            for h in range(nq):
                s = q[at:at + b, h] @ k[:, h * nkv // nq].T / math.sqrt(HEAD_DIM)
                s = s.masked_fill(~seen, -math.inf)
                w = torch.exp(s - s.max(1, keepdim=True).values).nan_to_num(0.0)
                out[at:at + b, h] = w @ v[:, h * nkv // nq] / w.sum(1, keepdim=True).clamp(min=1e-300)
        at += b
    return out
