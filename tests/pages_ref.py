"""The page pool's rules on lists: what forks, growth, ends and compaction leave, and the copies that they make."""


class Pages:
    def __init__(self, n_pages, page, max_seqs, width):
        self.page, self.width = page, width
        self.rows, self.lengths = [[] for _ in range(max_seqs)], [0] * max_seqs
        self.holders, self.missing, self.copies = [0] * n_pages, 0, []             # copies: (src, dst, rows)

    def table(self):
        return [r + [-1] * (self.width - len(r)) for r in self.rows]

    def _take(self, n):
        free = [e for e, h in enumerate(self.holders) if h == 0][:n]
        for e in free:
            self.holders[e] = 1
        self.missing += n - len(free)
        return free + [-1] * (n - len(free))

    def fork(self, parents):
        rows, lengths, want, seen = [], [], [], set()
        for s, p in enumerate(parents):
            if not 0 <= p < len(self.rows):
                rows.append([])
                lengths.append(0)
                continue
            row = list(self.rows[p])
            rest = self.lengths[p] % self.page
            if rest and p in seen and row[-1] >= 0:
                want.append((s, row.pop(), rest))
            seen.add(p)
            rows.append(row)
            lengths.append(self.lengths[p])
        for delta, table in ((-1, self.rows), (1, rows)):
            for row in table:
                for e in row:
                    if e >= 0:
                        self.holders[e] += delta
        for (s, src, rest), e in zip(want, self._take(len(want))):
            rows[s].append(e)
            if e >= 0:
                self.copies.append((src, e, rest))
        self.rows, self.lengths = rows, lengths

    def grow(self, counts):
        need = []
        for s, c in enumerate(counts):
            n = self.lengths[s] + max(c, 0)
            self.missing += n > self.width * self.page
            n = min(n, self.width * self.page)
            need.append(-(-n // self.page) - len(self.rows[s]))
            self.lengths[s] = n
        new = self._take(sum(need))
        for s, n in enumerate(need):
            self.rows[s] += new[:n]
            new = new[n:]

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.rows):
                for e in self.rows[s]:
                    if e >= 0:
                        self.holders[e] -= 1
                self.rows[s], self.lengths[s] = [], 0

    def compact(self):
        held = [e for e, h in enumerate(self.holders) if h]
        high = [e for e in held if e >= len(held)]
        to = dict(zip(high, [e for e, h in enumerate(self.holders) if not h]))
        for a, b in to.items():
            self.holders[b], self.holders[a] = self.holders[a], 0
            self.copies.append((a, b, self.page))
        self.rows = [[to.get(e, e) for e in r] for r in self.rows]
        return [to.get(e, e) for e in range(len(self.holders))]
