"""Barriers, copies and products of a kernel whose warps hand tiles to one another, run step by step on the host under any schedule.

A warp is a generator.  It yields a barrier and a parity to wait for (and is sent True, or False where the model lets the wait run
out; a third value True: it may not) or None to let others go first.  What runs beside the warps -- copies, which land in any order, and products, which run in the order in
which they were issued -- lies in `copies` and `products`."""
import random


class Fault(AssertionError):
    """What must never happen: a stale or torn tile, an arrival nobody counts on, a wait that cannot end."""


class Bar:
    """An mbarrier: a phase ends when all arrivals and all announced bytes are in."""

    def __init__(self, count):
        self.count = self.pending = count
        self.tx = self.phase = 0

    def arrive(self, n=1, tx=0):
        for _ in range(n):
            if self.pending == 0:
                raise Fault("an arrival with none pending")
            self.pending -= 1
            self.tx += tx
            tx = 0
            self._turn()

    def landed(self):
        self.tx -= 1
        self._turn()

    def _turn(self):
        if self.pending == 0 and self.tx == 0:
            self.phase += 1
            self.pending = self.count

    def passed(self, parity):
        return (self.phase & 1) != parity


class Meeting:
    """A barrier of the hardware between `count` warps: `yield (meeting, meeting.join())`."""

    def __init__(self, count):
        self.count, self.here, self.phase = count, 0, 0

    def join(self):
        mine = self.phase
        self.here += 1
        if self.here == self.count:
            self.here = 0
            self.phase += 1
        return mine

    def passed(self, mine):
        return self.phase > mine


class Run:
    """One run of the warps.  late: warps that move only when nothing else can; held: (warp, number of its turns) after which it does not
    move until nothing else can; give_up: the chance per turn that a wait on an mbarrier that has not passed runs out."""

    def __init__(self, seed, late=(), held=None, give_up=0.0):
        self.r = random.Random(seed)
        self.late, self.held, self.give_up = late, held, give_up
        self.warps = {}
        self.copies, self.products = [], []
        self.failed = False  # a wait has run out: values may be wrong, the rest still has to hold

    def check(self, sound, *what):
        if not sound and not self.failed:
            raise Fault(what)

    def _landed(self):
        bar, done = self.copies.pop(self.r.randrange(len(self.copies)))
        done()
        bar.landed()

    def go(self):
        waits = {w: next(g, "end") for w, g in self.warps.items()}  # what each warp waits for
        waits = {w: x for w, x in waits.items() if x != "end"}
        turns = dict.fromkeys(self.warps, 0)
        freed = self.held is None
        while waits:
            ready = [w for w, x in waits.items() if x is None or x[0].passed(x[1])]
            timed = [w for w, x in waits.items() if x is not None and isinstance(x[0], Bar) and len(x) == 2 and not x[0].passed(x[1])]
            most = [w for w in ready if w not in self.late and (freed or w != self.held[0] or turns[w] < self.held[1])]
            beside = [k for k in ("copies", "products") if getattr(self, k) and k not in self.late]
            if self.give_up and timed and self.r.random() < self.give_up:
                w, answer = self.r.choice(timed), False
                self.failed = True
            elif most or beside:
                w, answer = self.r.choice(most + beside * 3), True
            elif self.failed and timed and self.r.random() < 0.5:
                w, answer = self.r.choice(timed), False  # one warp gives up after the other while what is late still runs
            elif self.copies or self.products:
                w, answer = ("copies" if self.copies else "products"), True
            elif ready:
                w, answer, freed = self.r.choice(ready), True, True
            elif self.failed and timed:
                w, answer = self.r.choice(timed), False
            else:
                raise Fault(("nobody can move", sorted(waits)))
            if w == "copies":
                self._landed()
            elif w == "products":
                self.products.pop(0)()
            else:
                turns[w] += 1
                try:
                    waits[w] = self.warps[w].send(answer if waits[w] is not None else None)
                except StopIteration:
                    del waits[w]
        if self.copies or self.products:
            raise Fault(("the block ends with work in flight", len(self.copies), len(self.products)))
