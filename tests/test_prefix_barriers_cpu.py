"""The barrier protocol of the block kernel of ml2_prefix_attention, run as a model: every role of a block (loads, the two
warps that feed the tensor core, softmax warps, and the asynchronous TMA and tensor core) is a coroutine that stops at its
waits; a random scheduler goes on with whoever may. What is checked: nobody is stuck, no slot is written while it is read, no
weights or results are used before they are there, and after a wait that ran out everybody still comes to an end with no copy
or product under way."""
import random

import pytest

RING, WARPS = 4, 4  # slots of keys and of values; softmax warps of a stream (8 in the kernel: the number does not matter)


class Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.phase = 0

    def arrive(self):
        self.pending -= 1
        assert self.pending >= 0
        if not self.pending:
            self.phase += 1
            self.pending = self.count

    def passed(self, parity):
        return (self.phase & 1) != parity


class Block:
    """A block's run: segments of (tiles, whether the two streams take them in turns)."""

    def __init__(self, segments, rng, gives_up=0.0, eager=False, settles="copies and products"):
        """gives_up: chance that a wait runs out, at every step; the rest makes mistakes on purpose."""
        self.segments, self.rng, self.gives_up, self.eager, self.settles = segments, rng, gives_up, eager, settles
        self.abort = False
        self.k_full, self.v_full = ([Barrier(1) for _ in range(RING)] for _ in range(2))
        self.q, self.end = ([Barrier(WARPS), Barrier(WARPS)], [Barrier(1), Barrier(1)])
        self.s, self.o = ([[Barrier(1) for _ in range(RING)] for _ in range(2)] for _ in range(2))
        self.p = [[Barrier(WARPS), Barrier(WARPS)] for _ in range(2)]
        self.k_in, self.v_in = [None] * RING, [None] * RING    # tile that lies in a slot
        self.copies, self.products = [], [[], []]              # under way
        self.scored, self.added, self.weighed = [0, 0], [0, 0], [[0] * WARPS, [0] * WARPS]

    @staticmethod
    def share(turns, n, s):
        """Tiles of a stream in a segment."""
        return (n + 1 - s) >> 1 if turns else n

    def steps(self, n, turns):
        width = 2 if turns else 1
        return -(-n // width), lambda j: range(j * width, min(n, (j + 1) * width))

    def order(self, n, turns):
        count, tiles = self.steps(n, turns)
        yield from (("k", t) for t in tiles(0))
        for j in range(count):
            yield from (("k", t) for t in tiles(j + 1))
            yield from (("v", t) for t in tiles(j))

    def loads(self):
        asked = {"k": 0, "v": 0}
        done = yield from self.ask(asked)
        if not done or "copies" in self.settles:  # copies land before the block ends
            for which, full in (("k", self.k_full), ("v", self.v_full)):
                for x in range(max(0, asked[which] - RING), asked[which]):
                    yield "always", full[x % RING], x // RING & 1

    def ask(self, asked):
        base = 0
        for n, turns in self.segments:
            for kind, t in self.order(n, turns):
                g = base + t
                for s in range(2):
                    if not (yield (self.s if kind == "k" else self.o)[s][g % RING], g // RING & 1 ^ 1):
                        return False
                self.copies.append((kind, g))
                asked[kind] += 1
            base += n
        return True

    def tma(self):
        while True:
            yield "copy"
            kind, g = self.copies.pop(self.rng.randrange(len(self.copies)))
            (self.k_in if kind == "k" else self.v_in)[g % RING] = g
            (self.k_full if kind == "k" else self.v_full)[g % RING].arrive()

    def feeds(self, s):
        done = yield from self.queue(s)
        if not done or "products" in self.settles:  # products end before the TMEM is given back
            self.products[s].append(self.end[s].arrive)
            yield "always", self.end[s], 0

    def queue(self, s):
        base = asked = added = handed = 0
        for n, turns in self.segments:
            if self.eager or self.share(turns, n, s):
                if not (yield self.q[s], handed & 1):
                    return False
                handed += 1
            for kind, t in self.order(n, turns):
                g, mine = base + t, not turns or (t & 1) == s
                if not (yield (self.k_full if kind == "k" else self.v_full)[g % RING], g // RING & 1):
                    return False
                if kind == "k":
                    if not mine:
                        self.s[s][g % RING].arrive()
                        continue
                    asked += 1

                    def scores(g=g, asked=asked):
                        assert self.k_in[g % RING] == g
                        self.scored[s] = asked
                        self.s[s][g % RING].arrive()
                    self.products[s].append(scores)
                else:
                    if not mine:
                        self.o[s][g % RING].arrive()
                        continue
                    if not (yield self.p[s][added & 1], added >> 1 & 1):
                        return False
                    assert self.abort or min(self.weighed[s]) >= added + 1
                    added += 1

                    def values(g=g, added=added):
                        assert self.v_in[g % RING] == g
                        self.added[s] = added
                        self.o[s][g % RING].arrive()
                    self.products[s].append(values)
            base += n
        return True

    def tensor_core(self, s):
        while True:
            yield "product", s
            self.products[s].pop(0)()

    def softmax(self, s, warp):
        """Never leaves early: without waits once one ran out, and whatever it reads then is not used."""
        base = used = 0
        dead = False
        for n, turns in self.segments:
            mine = self.share(turns, n, s)
            if self.eager or mine:
                self.q[s].arrive()
            for j in range(mine):
                g = base + (2 * j + s if turns else j)
                dead = dead or not (yield self.s[s][g % RING], g // RING & 1)
                assert self.abort or self.scored[s] >= used + 1
                if j > 0 and self.rng.random() < 0.3:  # the reference moves: the product before has to be done
                    before = g - (2 if turns else 1)
                    dead = dead or not (yield self.o[s][before % RING], before // RING & 1)
                    assert self.abort or self.added[s] == used
                self.weighed[s][warp] = used + 1
                self.p[s][used & 1].arrive()
                used += 1
            if mine:
                g = base + (2 * (mine - 1) + s if turns else mine - 1)
                dead = dead or not (yield self.o[s][g % RING], g // RING & 1)
                assert self.abort or self.added[s] == used
            base += n

    def run(self):
        """True when every role came to its end."""
        roles = [self.loads(), self.feeds(0), self.feeds(1)] + [self.softmax(s, w) for s in range(2) for w in range(WARPS)]
        engines = [self.tma(), self.tensor_core(0), self.tensor_core(1)]
        alive, engine_at = {i: next(r, None) for i, r in enumerate(roles)}, [next(e) for e in engines]
        alive = {i: w for i, w in alive.items() if w is not None}

        def may(w):
            if w == "copy":
                return bool(self.copies)
            if w[0] == "product":
                return bool(self.products[w[1]])
            if w[0] == "always":
                return w[1].passed(w[2])
            return w[0].passed(w[1]) or self.abort

        while alive:
            if not self.abort and self.rng.random() < self.gives_up:
                self.abort = True
            ready = [("role", i) for i, w in alive.items() if may(w)] + [("engine", i) for i, w in enumerate(engine_at) if may(w)]
            if not ready:
                return False
            what, i = self.rng.choice(ready)
            for _ in range(self.rng.choice([1, 1, 5, 50])):
                try:
                    if what == "engine":
                        if not may(engine_at[i]):
                            break
                        engine_at[i] = next(engines[i])
                    else:
                        w = alive[i]
                        if not may(w):
                            break
                        alive[i] = roles[i].send(w[0] == "always" or w[0].passed(w[1]))
                except StopIteration:
                    del alive[i]
                    break
        return True


def run_of_segments(rng):
    """Whole blocks of more than eight key tiles, but for the first and the last segment of a run."""
    tiles = rng.choice([9, 10, 16, 17])
    segments = [[tiles, rng.random() < 0.6] for _ in range(rng.randint(1, 5))]
    segments[0][0], segments[-1][0] = rng.randint(1, tiles), rng.randint(1, tiles)
    return [tuple(x) for x in segments]


@pytest.mark.parametrize("seed", range(4))
def test_every_role_comes_to_its_end(seed):
    rng = random.Random(seed)
    for _ in range(250):
        segments = run_of_segments(rng)
        block = Block(segments, rng)
        assert block.run(), segments
        assert not block.copies and not any(block.products)


@pytest.mark.parametrize("seed", range(4))
def test_every_role_comes_to_its_end_after_a_wait_ran_out(seed):
    rng = random.Random(100 + seed)
    aborted = 0
    for _ in range(250):
        segments = run_of_segments(rng)
        block = Block(segments, rng, gives_up=10 ** rng.uniform(-3.5, -0.5))
        assert block.run(), segments
        aborted += block.abort
        # copies have landed and products are done when the block ends
        assert not block.copies and not any(block.products)
    assert aborted > 100


def test_the_model_finds_queries_handed_over_for_no_tiles():
    """A stream without tiles in a segment could be two phases of its barrier ahead of the warp that waits for them."""
    rng = random.Random(7)
    assert any(not Block(run_of_segments(rng), rng, eager=True).run() for _ in range(400))


@pytest.mark.parametrize("settles", ["copies", "products"])
def test_the_model_finds_a_block_that_ends_with_work_under_way(settles):
    """Whoever has queued all of its work waits for the end of it too: others may have given up, and nobody else would."""
    rng = random.Random(8)
    left = 0
    for _ in range(400):
        block = Block(run_of_segments(rng), rng, gives_up=0.003, settles=settles)
        assert block.run()
        left += bool(block.copies or any(block.products))
    assert left > 0
