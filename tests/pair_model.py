"""A pair of blocks of the products over experts on a dispatch's rows, as roles that wait for barriers, on the host.

The barriers are those of the kernel: a count of arrivals and bytes on their way make a phase, and a wait is for the parity of a phase alone, so one that comes
two phases late does not end. Which role takes its next step, and which copy or product ends next, is drawn; ``slow`` roles come up a hundred
times less often than the others.
"""


class Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.bytes = self.phase = 0

    def arrive(self, expect=0):
        self.pending -= 1
        assert self.pending >= 0, "more arrivals than the barrier counts"
        self.bytes += expect
        self._end()

    def come(self, n):
        self.bytes -= n
        self._end()

    def _end(self):
        if self.pending == 0 and self.bytes == 0:
            self.pending, self.phase = self.count, self.phase + 1

    def passes(self, parity):
        return self.phase & 1 != parity


class Pair:
    """tiles: the bytes of rows that the two blocks copy for a step of each tile; up: the first product, whose role of rows reads lists, too."""

    def __init__(self, tiles, stages, steps, up):
        self.tiles, self.stages, self.steps, self.up = tiles, stages, steps, up
        self.full = [Barrier(2) for _ in range(stages)]  # the first block's
        self.empty = [[Barrier(1) for _ in range(stages)] for _ in range(2)]
        self.sums_full, self.sums_empty = [[Barrier(1) for _ in range(2)] for _ in range(2)], [Barrier(2) for _ in range(2)]
        self.list_full, self.list_empty = ([[Barrier(n) for _ in range(2)] for _ in range(2)] for n in (1, 2 if up else 1))
        self.copies, self.products = [], []  # on their way: copies end in any order, products in theirs
        self.roles = {("products", 0): self.issue()}
        for side in (0, 1):
            self.roles.update({("weights", side): self.load(side, False), ("rows", side): self.load(side, True), ("lists", side): self.lists(side),
                               ("epilogue", side): self.epilogue(side)})

    def load(self, side, rows):
        stage, phase = 0, 1
        for n, own in enumerate(self.tiles):
            if rows and self.up:
                yield self.list_full[side][n & 1], n >> 1 & 1
            for _ in range(self.steps):
                yield self.empty[side][stage], phase
                if side == 0:
                    self.full[stage].arrive(sum(own) if rows else 2)
                size = own[side] if rows else 1
                if size:
                    self.copies.append((self.full[stage], size))
                stage += 1
                if stage == self.stages:
                    stage, phase = 0, phase ^ 1
            if rows and self.up:
                self.list_empty[side][n & 1].arrive()

    def issue(self):
        stage, phase = 0, 0
        for n in range(len(self.tiles)):
            yield self.sums_empty[n & 1], n >> 1 & 1 ^ 1
            for _ in range(self.steps):
                yield self.full[stage], phase
                self.products.append([self.empty[side][stage] for side in (0, 1)])
                stage += 1
                if stage == self.stages:
                    stage, phase = 0, phase ^ 1
            self.products.append([self.sums_full[side][n & 1] for side in (0, 1)])

    def lists(self, side):
        for n in range(len(self.tiles)):
            yield self.list_empty[side][n & 1], n >> 1 & 1 ^ 1
            self.list_full[side][n & 1].arrive()

    def epilogue(self, side):
        for n in range(len(self.tiles)):
            yield self.list_full[side][n & 1], n >> 1 & 1
            yield self.sums_full[side][n & 1], n >> 1 & 1
            self.sums_empty[n & 1].arrive()
            self.list_empty[side][n & 1].arrive()

    def run(self, rng, slow=()):
        """The roles that never end: none of them where the pair gets through."""
        waits = {name: next(role) for name, role in self.roles.items()}
        while waits or self.copies or self.products:
            choices = [(name, 1 if name in slow else 100) for name, (barrier, parity) in waits.items() if barrier.passes(parity)]
            choices += [("copy", 100)] * bool(self.copies) + [("product", 100)] * bool(self.products)
            if not choices:
                return sorted(waits)
            what = rng.choices(*zip(*choices))[0]
            if what == "copy":
                barrier, size = self.copies.pop(rng.randrange(len(self.copies)))
                barrier.come(size)
            elif what == "product":
                first = self.products[0]  # arrives at one block, then at the other
                first.pop(rng.randrange(len(first))).arrive()
                if not first:
                    self.products.pop(0)
            else:
                try:
                    waits[what] = next(self.roles[what])
                except StopIteration:
                    del waits[what]
        return []
