"""The page pool of include/bpdq_serve.h, page by page."""


def used(rows, page):
    return -(-rows // page)


class Pool:
    def __init__(self, n_pages, page, n_rows, width, reserved=0):
        self.page, self.width, self.n_pages = page, width, n_pages
        self.free = list(range(n_pages - 1, reserved - 1, -1))
        self.table = [[-1] * width for _ in range(n_rows)]
        self.lens = [0] * n_rows
        self.gone = [[0, 0] for _ in range(n_rows)]

    def rows(self, rows, n):
        """Each sequence's row, None where it is none or was named before."""
        seen, out = set(), []
        for r in (range(n) if rows is None else rows):
            good = 0 <= r < len(self.lens) and r not in seen
            out.append(r if good else None)
            if good:
                seen.add(r)
        return out

    def extend(self, new, n_tokens, rows=None, prefix_len=0):
        lens, refused, start, slots, pos, tables = [], [], [0], [], [], []
        asked = wanted = 0
        have = len(self.free)
        for r, k in zip(self.rows(rows, len(new)), new):
            old = 0 if r is None else self.lens[r]
            code, need = 0, 0
            if r is None or k < 0:
                code = 1
            elif old + k > self.width * self.page:
                code = 2
            else:
                need = used(old + k, self.page) - used(old, self.page)
                asked += need
                if need and asked > have:
                    code = 3
                else:
                    wanted += k
                    if wanted > n_tokens:
                        code = 4
            if code == 0:
                for i in range(need):
                    self.table[r][used(old, self.page) + i] = self.free.pop()
                for i in range(old, old + k):
                    pg = self.table[r][i // self.page]
                    slots.append(pg * self.page + i % self.page if 0 <= pg < self.n_pages else -1)
                    pos.append(prefix_len + i)
                self.lens[r] = old = old + k
            lens.append(old)
            refused.append(code)
            start.append(len(slots))
            n = used(old, self.page)
            tables.append((self.table[r][:n] if r is not None else []) + [-1] * (self.width - (n if r is not None else 0)))
        rest = [-1] * (n_tokens - len(slots))
        return dict(table=tables, lens=lens, q_start=start, slots=slots + rest, pos=pos + rest, refused=refused)

    def release(self, keep=None, rows=None, window=None, sinks=0):
        n = len(keep) if keep is not None else len(rows) if rows is not None else len(self.lens)
        back = []
        for b, r in enumerate(self.rows(rows, n)):
            if r is None:
                continue
            old = self.lens[r]
            new = old if keep is None else min(max(keep[b], 0), old)
            g0, g1 = (min(g, used(new, self.page)) for g in self.gone[r])
            if g0 == g1:
                g0 = g1 = 0
            slide, tail = [], list(range(used(new, self.page), used(old, self.page)))
            if window:
                first = g1 if g1 else used(sinks, self.page)
                last = max(0, new - window + 1) // self.page
                slide = list(range(first, last))
                if slide:
                    g0, g1 = (g0 if g1 else first), last
            tail = [i for i in tail if not self.gone[r][0] <= i < self.gone[r][1]]
            for i in slide + tail:
                back.append(self.table[r][i])
                self.table[r][i] = -1
            self.lens[r], self.gone[r] = new, [g0, g1]
        self.free += back[::-1]
