"""The hand-overs of the tree attention kernel (it_tree_attention_tc.cu) as a model: roles, barriers that show a waiter one bit, copies and products that complete later.

Every wait is checked when it is tried: a barrier whose phases have run more than one ahead of the waiter (or lag two behind) shows the wrong bit.  Every place (ring slots, scores, P, O^T, the
rows' factors) is checked for being overwritten before its last reader is through, and for being read before it holds what the reader wants.  Schedules are random, with one role
at a time made to lag far behind, and every schedule has to end."""
import random

import pytest

KEYS, LIMIT, SMALL = 128, 227 * 1024, 3 * 1024


def shape(split, nb, nr):
    """TcTree's numbers."""
    nc, mt, box = nr * (2 if split else 1), nb // 2, KEYS * 128
    parts = 1 if not split or nr > 32 else 2 if nr == 32 else nb
    slot = nb * box
    slots = min((LIMIT - SMALL - nb * nc * 128 - (2 if nc > 64 else 1) * box) // slot, 6)
    ks = (slots + 1) // 2
    assert slots >= 2 and 2 * parts * nc + mt * nc <= 512
    return dict(nb=nb, mt=mt, ks=ks, vs=slots - ks)


class Barrier:
    def __init__(self, name, count):
        self.name, self.count, self.have, self.done = name, count, 0, 0

    def arrive(self):
        self.have += 1
        assert self.have <= self.count
        if self.have == self.count:
            self.have, self.done = 0, self.done + 1

    def passed(self, phase):
        """mbarrier test_wait with the parity of `phase`; phase -1: the one before the first, which has passed."""
        assert phase <= self.done <= phase + 1, f"{self.name}: waiting for phase {phase}, {self.done} are complete"
        return self.done % 2 != phase % 2


class Model:
    FACTORS = 2

    def __init__(self, s, n, first_masked, rng, groups=2, warps=2):
        self.__dict__.update(s)
        self.n, self.first_masked, self.rng, self.groups, self.warps = n, first_masked, rng, groups, warps
        soft = groups * warps
        B = lambda name, k, c: [Barrier(f"{name}{i}", c) for i in range(k)]  # noqa: E731
        self.kboxes, self.vpairs = self.ks * self.nb, self.vs * self.mt
        self.kfull, self.kempty, self.vfull, self.vempty = B("kfull", self.kboxes, 1), B("kempty", self.kboxes, 1), B("vfull", self.vpairs, 1), B("vempty", self.vpairs, 1)
        self.sfull, self.sfree, self.pfull, self.ofull = B("sfull", 2, 1), B("sfree", 2, soft), B("pfull", 1, soft)[0], B("ofull", self.mt, 1)
        self.met = [[0] * 100 for _ in range(groups + 1)]                # arrivals at the k-th barrier of a group, and of all groups
        self.pipe, self.copies = [], []                                  # products in order; copies in any order
        self.K, self.V, self.S, self.P, self.O, self.factors = {}, {}, {}, {}, {}, {}      # place -> [what it holds, readers still to come]
        self.clean = set()
        self.roles = {"load_k": self.load_k(), "load_v": self.load_v(), "issue": self.issue()}
        for g in range(groups):
            for w in range(warps):
                self.roles[f"soft{g}{w}"] = self.softmax(g, w)

    def put(self, where, place, what, readers):
        if place in where:
            assert where[place][1] == 0, f"{place} still holds {where[place]} when {what} comes"
        where[place] = [what, readers]

    def take(self, where, place, what):
        assert where[place][0] == what, f"{place} holds {where[place]}, not {what}"
        where[place][1] -= 1

    # ---- roles: generators that yield a condition to wait for
    def load_k(self):
        for k in range(self.n * self.nb):
            at = k % self.kboxes
            if k >= self.kboxes:
                yield lambda: self.kempty[at].passed(k // self.kboxes - 1)
            self.copies.append(lambda at=at, k=k: (self.put(self.K, at, k, 1), self.kfull[at].arrive()))
        yield None

    def load_v(self):
        for k in range(self.n * self.mt):
            at = k % self.vpairs
            if k >= self.vpairs:
                yield lambda: self.vempty[at].passed(k // self.vpairs - 1)
            look = self.groups * self.warps if k // self.mt >= self.first_masked else 0      # warps that look at a masked tile's V
            self.copies.append(lambda at=at, k=k, look=look: (self.put(self.V, at, k, 1 + look), self.vfull[at].arrive()))
        yield None

    def issue(self):
        si = kb = oi = om = 0
        while oi < self.n:
            pair, box = oi * self.mt + om, kb % self.kboxes
            if oi < si and (om > 0 or self.pfull.passed(oi)) and self.vfull[pair % self.vpairs].passed(pair // self.vpairs):
                def done(pair=pair, oi=oi, om=om):
                    self.take(self.V, pair % self.vpairs, pair)
                    assert self.V[pair % self.vpairs][1] == 0, "V is read before all have looked at it"
                    assert oi < self.first_masked or oi in self.clean, "V is read before it is clean"
                    self.take(self.P, 0, oi)
                    self.put(self.O, om, oi, self.groups * self.warps)
                    self.ofull[om].arrive()
                    self.vempty[pair % self.vpairs].arrive()
                self.pipe.append(done)
                om += 1
                if om == self.mt:
                    om, oi = 0, oi + 1
            elif si < self.n and (kb % self.nb or self.sfree[si & 1].passed((si >> 1) - 1)) and self.kfull[box].passed(kb // self.kboxes):
                def done(si=si, kb=kb):
                    self.take(self.K, kb % self.kboxes, kb)
                    self.kempty[kb % self.kboxes].arrive()
                    if kb % self.nb == 0:
                        self.put(self.S, si & 1, si, self.groups * self.warps)
                    if kb % self.nb == self.nb - 1:
                        self.sfull[si & 1].arrive()
                self.pipe.append(done)
                kb += 1
                si += kb % self.nb == 0
            yield lambda: True
        yield None

    def meet(self, who, k, count):
        """The k-th barrier of a group (or, who == groups, of all)."""
        self.met[who][k] += 1
        return lambda: self.met[who][k] == count

    def softmax(self, g, w):
        masked = 0
        for i in range(self.n + 1):
            if i < self.n:
                yield lambda: self.sfull[i & 1].passed(i >> 1)
                self.take(self.S, i & 1, i)
                self.sfree[i & 1].arrive()
                yield lambda: True
                yield self.meet(g, i, self.warps)                        # whether the references move, or their new values
                if w == 0:                                               # all write the same
                    self.put(self.factors, (g, i % self.FACTORS), i, self.warps)
                yield self.meet(g, 50 + i, self.warps) if w else lambda: True       # (each warp writes what it reads itself)
                if w == 0:
                    self.met[g][50 + i] += 1
            if i > 0:
                for m in range(self.mt):
                    yield lambda: self.ofull[m].passed(i - 1)
                    self.take(self.O, m, i - 1)
                self.take(self.factors, (g, (i - 1) % self.FACTORS), i - 1)
                yield lambda: True
            if i == self.n:
                break
            if g == 0 and w == 0:
                self.put(self.P, 0, i, self.mt)
            yield lambda: True
            if i >= self.first_masked:
                for m in range(self.mt):
                    pair = i * self.mt + m
                    yield lambda: self.vfull[pair % self.vpairs].passed(pair // self.vpairs)
                    self.take(self.V, pair % self.vpairs, pair)
                yield self.meet(self.groups, masked, self.groups * self.warps)
                masked += 1
                self.clean.add(i)
            self.pfull.arrive()
        assert all(v[1] == 0 for v in self.K.values()) and all(v[1] == 0 for v in self.P.values()), "K's and P's places are used again"
        yield None

    # ---- one schedule
    def run(self, lag):
        rng, waits = self.rng, {}
        for name, r in self.roles.items():
            waits[name] = next(r)
        idle = 0
        while any(w is not None for w in waits.values()):
            moved = False
            act = rng.random()
            if act < 0.25 and self.pipe and (lag != "pipe" or rng.random() < 0.03):
                self.pipe.pop(0)()
                moved = True
            elif act < 0.4 and self.copies and (lag != "copies" or rng.random() < 0.03):
                self.copies.pop(rng.randrange(len(self.copies)))()
                moved = True
            else:
                name = rng.choice(list(waits))
                if waits[name] is not None and (name != lag or rng.random() < 0.02) and waits[name]():
                    waits[name] = next(self.roles[name])
                    moved = name != "issue" or waits[name] is None
            idle = 0 if moved else idle + 1
            assert idle < 20000, "nothing moves: " + ", ".join(k for k, w in waits.items() if w is not None)


@pytest.mark.parametrize("split,nb,nr", [(s, nb, nr) for s in (True, False) for nb in (2, 4) for nr in (16, 32, 64)])
def test_every_schedule_ends_and_nothing_is_overwritten(split, nb, nr):
    s = shape(split, nb, nr)
    rng = random.Random(nb * 1000 + nr + split)
    for trial in range(8):
        n = rng.choice((0, 1, 2, 3, 5, 9, 14))
        for masked in {n, max(n - 1, 0), max(n - 3, 0)}:                    # tiles from here on are masked
            for lag in (None, "pipe", "copies", "soft00", "soft11", "issue", "load_k", "load_v"):
                if rng.random() < 0.5:
                    Model(s, n, masked, rng).run(lag)


def test_the_model_sees_places_that_are_taken_too_early():
    """One set of factors in place of two: a fast warp's next tile would overwrite what a slow one still needs.  And P handed on without waiting for the last product."""
    s = shape(False, 2, 16)

    class OneSet(Model):
        FACTORS = 1

    class NoWait(Model):
        def softmax(self, g, w):
            for i in range(self.n):
                yield lambda: self.sfull[i & 1].passed(i >> 1)
                self.take(self.S, i & 1, i)
                self.sfree[i & 1].arrive()
                if g == 0 and w == 0:
                    self.put(self.P, 0, i, self.mt)
                yield lambda: True
                self.pfull.arrive()
            yield None

    for wrong in (OneSet, NoWait):
        rng = random.Random(1)
        with pytest.raises(AssertionError):
            for _ in range(200):
                wrong(s, 9, 9, rng).run(rng.choice((None, "issue", "pipe", "soft01")))
