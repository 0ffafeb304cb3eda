"""Sequential restatement of the operators on pages that several requests hold, on Python lists."""


class Shared:
    """Requests' pages, lengths and holders; every operation takes the requests one after another."""

    def __init__(self, n, num_pages, page, max_pages):
        self.n, self.page, self.max_pages = n, page, max_pages
        self.lens, self.held = [0] * n, [[] for _ in range(n)]
        self.free, self.head = list(range(num_pages)), 0
        self.status = 0

    def owners(self):
        count = {}
        for row in self.held:
            for p in row:
                count[p] = count.get(p, 0) + 1
        return count

    def fork(self, src, dst, rows=None):
        lens, held, seen = list(self.lens), [list(r) for r in self.held], set()
        for j, (s, d) in enumerate(zip(src, dst)):
            first = d not in seen
            seen.add(d)
            if not (0 <= s < self.n and 0 <= d < self.n) or not first or lens[d] > 0 or held[d]:
                self.status |= 128
                continue
            take = lens[s] if rows is None else min(lens[s], max(rows[j], 0))
            self.lens[d] = take
            self.held[d] = held[s][:-(-take // self.page)]

    def reserve(self, new, num_slots):
        owners, starts, slots, copies, asked, taken, dry = self.owners(), [0], [-1] * num_slots, [], 0, 0, False
        before = dict(owners)
        served = []
        ranks = {}
        room = len(self.free) - self.head
        for i in range(self.n):
            m, a = max(new[i], 0), self.lens[i]
            starts.append(starts[-1] + m)
            want, bad = -(-(a + m) // self.page), 0
            if want > self.max_pages:
                bad |= 2
            if starts[-1] > num_slots:
                bad |= 4
            if m and not bad and any(before[p] > 1 for p in self.held[i][-(-a // self.page):want]):
                bad |= 256
            self.status |= bad
            copies.append((-1, -1, 0))
            served.append(False)
            if bad:
                continue
            shares = copy = False
            if m and a % self.page and a // self.page < len(self.held[i]):
                p = self.held[i][a // self.page]
                shares = before[p] > 1
                copy = shares and ranks.get(p, 0) < before[p] - 1
                ranks[p] = ranks.get(p, 0) + 1
            need = max(want - len(self.held[i]), 0) + copy
            asked += need
            if (need or shares) and asked > room:
                self.status |= 1
                continue
            served[i] = True
            if copy:
                to = self.free[self.head + taken]
                copies[i] = (p, to, a % self.page)
                self.held[i][a // self.page] = to
                taken += 1
            while len(self.held[i]) < want:
                self.held[i].append(self.free[self.head + taken])
                taken += 1
            for r in range(m):
                slots[starts[i] + r] = self.held[i][(a + r) // self.page] * self.page + (a + r) % self.page
            self.lens[i] += m
        self.head += taken
        return starts, slots, copies, served

    def release(self, keep):
        owners, back = self.owners(), []
        for i in range(self.n):
            left = min(len(self.held[i]), -(-max(keep[i], 0) // self.page))
            for p in self.held[i][left:]:
                owners[p] -= 1
                if owners[p] == 0:
                    back.append(p)
            self.held[i] = self.held[i][:left]
        self.head -= len(back)
        self.free[self.head:self.head + len(back)] = back
