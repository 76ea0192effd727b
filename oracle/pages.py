"""CPU restatement of keeping the pages of a cache as include/fused_attn.h defines it, with lists.  TEST INFRASTRUCTURE ONLY.

`Keeper.check` says whether the counts of uses are those of the table; tests/test_pages.py pins the operations by closed forms.
"""


class Keeper:
    """table [S][W], starts [S], uses [N], P tokens of a page; holds[page]: whose first contents the page holds now."""

    def __init__(self, table, starts, uses, P):
        self.table = [list(row) for row in table]
        self.starts, self.uses, self.P = list(starts), list(uses), P
        self.S, self.W, self.N = len(self.table), len(self.table[0]), len(self.uses)
        self.holds = list(range(self.N))

    def is_page(self, page):
        return 0 <= page < self.N

    def check(self):
        uses = [0] * self.N
        for row in self.table:
            for page in row:
                if self.is_page(page):
                    uses[page] += 1
        return uses == self.uses

    def copy(self, sources, targets):
        was = list(self.holds)
        for a, b in zip(sources, targets):
            if self.is_page(a) and self.is_page(b):
                self.holds[b] = was[a]

    def free(self, sequences):
        for row in sequences:
            if 0 <= row < self.S:
                for page in self.table[row]:
                    if self.is_page(page):
                        self.uses[page] -= 1
                self.table[row], self.starts[row] = [-1] * self.W, 0

    def _free_pages(self):
        return [page for page in range(self.N) if self.uses[page] <= 0]

    def take(self, lens, L):
        free, missing = self._free_pages(), [0] * self.S
        for b in range(self.S):
            n = max(0, min(lens[b], L))
            if n == 0:
                continue
            low, high = max(self.starts[b], 0), max(self.starts[b] + n, 0)
            for w in range(-(-low // self.P), -(-high // self.P)):
                if w >= self.W:
                    missing[b] += 1
                elif not self.is_page(self.table[b][w]):
                    self.table[b][w] = free.pop(0) if free else -1
                    if self.table[b][w] < 0:
                        missing[b] += 1
                    else:
                        self.uses[self.table[b][w]] = 1
        return missing

    def fork(self, parents, children):
        free, forked = self._free_pages(), []
        starts, table, named = list(self.starts), [list(row) for row in self.table], set()
        for parent, child in zip(parents, children):
            again = child in named
            named.add(child)
            ok = 0 <= parent < self.S and 0 <= child < self.S and parent != child and starts[child] == 0 and not again
            n = max(starts[parent], 0) if ok else 0
            full, last = n // self.P, -1
            if ok and n % self.P and full < self.W and self.is_page(table[parent][full]):
                if free:
                    last = free.pop(0)
                    self.uses[last], self.holds[last] = 1, self.holds[table[parent][full]]
                else:
                    ok = False
            forked.append(int(ok))
            if not ok:
                continue
            for page in self.table[child]:
                if self.is_page(page):
                    self.uses[page] -= 1
            row = [table[parent][w] if w < full else last if w == full else -1 for w in range(self.W)]
            for page in row[:full]:
                if self.is_page(page):
                    self.uses[page] += 1
            self.table[child], self.starts[child] = row, n
        return forked

    def compact(self):
        used = [page for page in range(self.N) if self.uses[page] > 0]
        moved = [page if self.uses[page] > 0 else -1 for page in range(self.N)]
        for hole, page in zip([p for p in range(len(used)) if self.uses[p] <= 0], [p for p in used if p >= len(used)]):
            moved[page], self.holds[hole] = hole, self.holds[page]
            self.uses[hole], self.uses[page] = self.uses[page], 0
        self.table = [[moved[page] if self.is_page(page) else -1 for page in row] for row in self.table]
        return moved
