"""64-bit restatements of the paged 4-bit cache's operators for the tests,
written from their definitions on numpy and host loops."""
import math

import numpy as np
import torch

D = 128


def scale_values():
    """Every scale of the format, ascending: 1..7 times 2^-17, then 8..15 at each exponent, up to 9216."""
    s = [m * 2.0 ** -17 for m in range(1, 8)]
    s += [m * 2.0 ** (e - 17) for e in range(31) for m in range(8, 16)]
    return np.array([v for v in s if v <= 9216.0])


def q4_values(x):
    """What the cache stands for after rows x [..., 128] are appended (float64 numpy)."""
    x = x.double().cpu().numpy()
    x = np.where(np.isnan(x), 0.0, x).reshape(*x.shape[:-1], 8, 16)
    scales = scale_values()
    at = np.searchsorted(scales * 7.5, np.abs(x).max(-1))
    s = scales[np.minimum(at, len(scales) - 1)][..., None]
    with np.errstate(invalid="ignore"):
        q = np.minimum(np.floor(np.abs(x) / s + 0.5), 7.0)
    return torch.from_numpy((np.sign(x) * q * s).reshape(*x.shape[:-2], D))


def reserve(lens, new, pages, table, free, head, page, num_slots):
    """(starts, slots, lens, pages, head, status) and the table changed in place (lists and numpy)."""
    starts, slots, status, asked, taken = [0], [-1] * num_slots, 0, 0, 0
    lens_out, pages_out = [], []
    for i, (a, b, h) in enumerate(zip(lens, new, pages)):
        a, b = max(a, 0), max(b, 0)
        starts.append(starts[-1] + b)
        want = -(-(a + b) // page)
        bad = (2 if want > table.shape[1] else 0) | (4 if starts[-1] > num_slots else 0)
        need = 0 if bad else max(want - h, 0)
        asked += need
        if need and asked > len(free) - head:
            bad |= 1
        status |= bad
        if bad:
            lens_out.append(a)
            pages_out.append(h)
            continue
        table[i, h:h + need] = free[head + taken:head + taken + need]
        taken += need
        lens_out.append(a + b)
        pages_out.append(max(h, want))
        for r in range(b):
            slots[starts[i] + r] = int(table[i, (a + r) // page]) * page + (a + r) % page
    return starts, slots, lens_out, pages_out, head + taken, status


def release(keep, pages, table, free, head, page):
    """(pages, head) and the free list changed in place."""
    left = [min(h, -(-max(k, 0) // page)) for k, h in zip(keep, pages)]
    at = new_head = head - sum(pages) + sum(left)
    for i, (a, b) in enumerate(zip(left, pages)):
        for c in range(a, b):
            free[at] = table[i, c]
            at += 1
    return left, new_head


def seen_keys(L, rows, j, causal, sink, window):
    """Boolean [L]: the keys that query row j of `rows` sees."""
    end = L - rows + j + 1 if causal else L
    k = np.arange(L)
    seen = k < end
    if window:
        seen &= (k < sink) | (k >= end - window)
    return seen


def attention(q, ks, vs, rows, scale, causal=False, sink=0, window=0):
    """q [T, NQ, 128]; ks, vs: the requests' values [L, NKV, 128] (float64); rows: query rows of each.
    Returns (out, tol_weights): the output and, per element, what the error bound of the tests needs:
    W = sum p |v| / sum p, A = the largest sum |q k| scale of the row, n keys, max |v|."""
    q = q.double().cpu()
    out, W = torch.zeros_like(q), torch.zeros_like(q)
    A, n, vmax = (torch.zeros(q.shape[0], q.shape[1], 1, dtype=torch.float64) for _ in range(3))
    at = 0
    for K, V, m in zip(ks, vs, rows):
        L = K.shape[0]
        for j in range(m):
            seen = torch.from_numpy(seen_keys(L, m, j, causal, sink, window))
            if L and bool(seen.any()):
                for h in range(q.shape[1]):
                    hk = h * K.shape[1] // q.shape[1]
                    k, v = K[seen, hk], V[seen, hk]
                    s = (k @ q[at + j, h]) * scale
                    p = torch.softmax(s, 0)
                    out[at + j, h] = p @ v
                    W[at + j, h] = p @ v.abs()
                    A[at + j, h] = float((k.abs() @ q[at + j, h].abs()).max()) * abs(scale)
                    n[at + j, h] = k.shape[0]
                    vmax[at + j, h] = float(v.abs().max())
        at += m
    return out, (W, A, n, vmax)


def attention_tolerance(ref, bound, dtype):
    """Largest error that the operator's arithmetic allows, element by element.
    - the output's rounding: 2^-11 (f16), 2^-8 (bf16) of it, and f16's 2^-24 step;
    - P rounded to f16, 2^-11 of each weight (and 2^-25 absolute of weights whose sum is at least 1), and
      the exponential's 2^-20;
    - scores summed in fp32 by the tensor cores: at most 128 additions, each off by 2^-22 of sum |q k|,
      a relative error of the weights, which moves the quotient by at most twice as much;
    - the n weighted rows summed in fp32, 16 at a time, then once more when parts are merged."""
    W, A, n, vmax = bound
    u = 2.0 ** -11 if dtype is torch.float16 else 2.0 ** -8
    return (u * ref.abs() + 2.0 ** -24 + W * (2.0 ** -11 + 2.0 ** -20 + 2 * 2.0 ** -15 * A + (n / 16 + 64) * 2.0 ** -22)
            + n * 2.0 ** -25 * vmax)


class Paging:
    """Requests of given lengths on shuffled pages: device table, lengths and each row's slot."""

    def __init__(self, lens, page, seed=0, spare=3, max_pages=None, first_page=0):
        rng = np.random.default_rng(seed)
        held = [-(-a // page) for a in lens]
        self.num_pages = sum(held) + spare + first_page
        perm = first_page + rng.permutation(sum(held) + spare).astype(np.int32)
        self.max_pages = max_pages or max(max(held), 1)
        self.table = np.full((len(lens), self.max_pages), -1, np.int32)
        at = 0
        for i, h in enumerate(held):
            self.table[i, :h] = perm[at:at + h]
            at += h
        self.lens, self.pages, self.page, self.free, self.head = list(lens), held, page, perm, at
        self.slots = [torch.tensor([int(self.table[i, r // page]) * page + r % page for r in range(a)],
                                   dtype=torch.int32) for i, a in enumerate(lens)]

    def dev(self, name):
        return torch.tensor(np.array(getattr(self, name)), dtype=torch.int32).cuda()


def scale_of(x):
    return 1.0 / math.sqrt(x)
