"""The barriers of the prompt kernel over the 4-bit cache (csrc/kv4_prefill.cu), on the CPU.

A CTA's sixteen warps, its tensor core and its barriers as coroutines that a random scheduler steps.  Checked in
every schedule: it ends; each wait is for the phase after one known to be complete (a parity wait cannot tell
phases two apart); each buffer holds the tile that its reader is at, from the read's begin to its end; nothing
asked of the tensor core is left at the CTA's end.  With waits that run out: it still ends, a unit is read only
where it is published and stays, and the tensor core is left idle.

The roles are restated here by hand, barrier by barrier, in the kernel's names.
"""
import random

import pytest

SOFT = 4  # softmax warps of a half


class Bar:
    def __init__(self, count):
        self.count, self.pending, self.done = count, count, 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.pending, self.done = self.count, self.done + 1


class Cta:
    """units: (tiles, turns) of each; expire: chance that a poll is a wait's last."""

    def __init__(self, units, seed, expire=0.0):
        self.r, self.units, self.expire = random.Random(seed), units, expire
        self.dead, self.queue, self.busy = False, [], False
        self.unit, self.unit_readers = [None] * 4, [0] * 4
        self.q = [[None] * SOFT, [None] * SOFT]
        self.at, self.par, self.k, self.v = [None] * 8, [None] * 8, [None] * 2, [None] * 2
        two = ("q_ready", 4), ("k_full", 3), ("v_full", 3), ("k_free", 1), ("v_free", 1), ("pv_done", 1), ("o_free", 4), \
            ("given", 4)
        self.bars = {(name, i): Bar(n) for name, n in two for i in range(2)}
        self.bars.update({(name, i): Bar(1) for name in ("at_full", "par_full") for i in range(8)})
        self.bars.update({(name, h, i): Bar(n) for name, n in (("qk_done", 1), ("p_ready", 4))
                          for h in range(2) for i in range(2)})
        self.bars["u_full"], self.bars["drained"] = Bar(1), Bar(1)

    # a poll, a wait, and the check that what a reader is at stays while it reads
    def ready(self, name, phase):
        done = self.bars[name].done
        if not self.dead:
            assert done in (phase, phase + 1), f"{name}: waiting for phase {phase}, {done} are done"
        return (done & 1) != (phase & 1)

    def wait(self, name, phase):
        while not self.ready(name, phase):
            if self.dead:
                return False
            if self.r.random() < self.expire:
                self.dead = True
                return False
            yield
        return True

    def holds(self, buffer, i, value):
        assert self.dead or buffer[i] == value, (buffer, i, value)

    def begin(self, seg):
        """Reads the unit in hand: published, and not replaced while anyone is at it."""
        assert self.unit[seg & 3] == seg
        self.unit_readers[seg & 3] += 1
        return self.units[seg]

    def end(self, seg):
        assert self.unit[seg & 3] == seg
        self.unit_readers[seg & 3] -= 1

    def softmax(self, half, warp):
        j = jh = given = 0
        for seg in range(len(self.units)):
            if not (yield from self.wait("u_full", seg)):
                return
            n, turns = self.begin(seg)
            yield
            self.q[half][warp] = seg
            self.bars["q_ready", half].arrive()
            own, step = ((n + 1 - half) >> 1, 2) if turns else (n, 1)
            last = j + n
            j += half if turns else 0
            for k in range(own + 1):
                if k < own:
                    yield from self.wait(("par_full", j & 7), j >> 3)
                    yield from self.wait(("qk_done", half, jh & 1), jh >> 1)
                    self.holds(self.par, j & 7, j)
                    yield
                    self.holds(self.par, j & 7, j)
                    self.bars["p_ready", half, jh & 1].arrive()
                    j, jh = j + step, jh + 1
                if k > 0:
                    yield from self.wait(("pv_done", half), jh - (2 if k < own else 1))
                    yield
                    self.bars["o_free", half].arrive()
            j = last
            if turns:
                if half == 0:
                    yield from self.wait(("given", 0), given)
                    assert self.dead or self.q[1] == [("sums", seg)] * SOFT
                    yield
                    assert self.dead or self.q[1] == [("sums", seg)] * SOFT
                else:
                    self.q[1][warp] = ("sums", seg)
                self.bars["given", 1 - half].arrive()
                if half == 1:
                    yield from self.wait(("given", 1), given)
                given += 1
            self.end(seg)

    def look(self):
        j = 0
        for seg in range(len(self.units)):
            if not (yield from self.wait("u_full", seg)):
                return
            n, _ = self.begin(seg)
            for k in range(n):
                if j > 1:
                    yield from self.wait(("k_free", j & 1), (j - 2) >> 1)
                yield
                self.at[j & 7] = j
                self.bars["at_full", j & 7].arrive()
                if k == 0:
                    for h in range(2):
                        yield from self.wait(("q_ready", h), seg)
                yield
                self.par[j & 7] = j
                self.bars["par_full", j & 7].arrive()
                j += 1
            self.end(seg)

    def unpack(self, buffer, full, free):
        j = 0
        for seg in range(len(self.units)):
            if not (yield from self.wait("u_full", seg)):
                return
            n, _ = self.begin(seg)
            for _ in range(n):
                yield from self.wait(("at_full", j & 7), j >> 3)
                yield
                self.holds(self.at, j & 7, j)
                if j > 1:
                    yield from self.wait((free, j & 1), (j - 2) >> 1)
                yield
                buffer[j & 1] = j
                self.bars[full, j & 1].arrive()
                j += 1
            self.end(seg)

    def issue(self):
        j, jh = 0, [0, 0]
        for seg, (n, turns) in enumerate(self.units):
            assert self.unit_readers[seg & 3] == 0 or self.unit[seg & 3] is None
            self.unit[seg & 3] = seg
            self.bars["u_full"].arrive()
            yield
            alive = True
            for h in range(2):
                alive &= yield from self.wait(("q_ready", h), seg)
            turns, last = int(turns), j + n
            tq, tp, h = [j, j + turns], [j, j + turns], 0
            while alive and (tp[0] < last or tp[1] < last):
                nq, np = jh[h] + ((tq[h] - j) >> turns), jh[h] + ((tp[h] - j) >> turns)
                if tq[h] < last and nq <= np + 1 and self.ready(("k_full", tq[h] & 1), tq[h] >> 1):
                    self.queue.append(("qk_done", h, nq & 1, self.k, tq[h]))
                    if turns or tq[h] < tq[1 - h]:
                        self.queue.append(("k_free", tq[h] & 1))
                    tq[h] += 1 + turns
                elif tp[h] < tq[h] and self.ready(("p_ready", h, np & 1), np >> 1) \
                        and self.ready(("v_full", tp[h] & 1), tp[h] >> 1):
                    if np > 0:
                        yield from self.wait(("o_free", h), np - 1)
                    self.queue.append(("pv_done", h, None, self.v, tp[h]))
                    if turns or tp[h] < tp[1 - h]:
                        self.queue.append(("v_free", tp[h] & 1))
                    tp[h] += 1 + turns
                elif self.r.random() < self.expire:
                    self.dead = True
                alive = not self.dead
                h ^= 1
                yield
            if not alive:
                break
            jh = [jh[0] + ((n + turns) >> turns), jh[1] + (n >> turns)]
            j = last
        self.queue.append(("drained",))
        while not self.bars["drained"].done:
            yield

    def tensor(self):
        """Products and arrivals in the order that they were asked for."""
        while True:
            if self.queue:
                what = self.queue[0]
                if len(what) == 5:
                    name, h, i, buffer, tile = what
                    self.holds(buffer, tile & 1, tile)
                    yield
                    self.holds(buffer, tile & 1, tile)
                    self.bars[(name, h) if i is None else (name, h, i)].arrive()
                else:
                    self.bars[what if len(what) == 2 else what[0]].arrive()
                self.queue.pop(0)
            yield

    def run(self):
        warps = [self.softmax(h, w) for h in range(2) for w in range(SOFT)]
        warps += [self.unpack(self.k, "k_full", "k_free") for _ in range(3)]
        warps += [self.unpack(self.v, "v_full", "v_free") for _ in range(3)] + [self.look(), self.issue()]
        speed = {id(w): self.r.random() ** 2 + 0.05 for w in warps}
        tensor, tensor_speed = self.tensor(), self.r.random() ** 2 + 0.05
        for _ in range(1_000_000):
            if not warps:
                break
            i = self.r.choices(range(len(warps) + 1), [speed[id(w)] for w in warps] + [tensor_speed])[0]
            if i == len(warps):
                next(tensor)
            elif next(warps[i], "over") == "over":
                warps.pop(i)
        assert not warps, "some warps wait for good"
        assert not self.queue, "products or arrivals are left"


def _units(seed):
    r = random.Random(seed)
    return [(r.randint(1, 9), r.random() < 0.5) for _ in range(r.randint(1, 6))]


@pytest.mark.parametrize("first", range(0, 200, 50))
def test_barriers_in_random_schedules(first):
    for seed in range(first, first + 50):
        Cta(_units(seed), seed).run()


@pytest.mark.parametrize("expire", [1.0, 0.1, 0.003])
def test_waits_that_run_out(expire):
    dead = 0
    for seed in range(100):
        cta = Cta(_units(seed), seed, expire)
        cta.run()
        dead += cta.dead
    assert dead > 10


def test_the_checks_see_a_mistake():
    """A tile's parameters in a ring of two instead of eight: some schedule replaces them under a reader."""
    class Short(Cta):
        def look(self):
            for step in super().look():
                self.par = [p if p is None or p + 2 > max(x for x in self.par if x is not None) else None
                            for p in self.par]
                yield step

    with pytest.raises(AssertionError):
        for seed in range(200):
            Short(_units(seed), seed).run()
