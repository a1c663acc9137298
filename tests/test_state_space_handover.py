"""Who arms which barrier in the tcgen05 output pass of the state space scan (ssm_out_umma_kernel), as a model on the CPU.

Two warps wait with a limit: the one that issues products (C and B there, z armed) and the one that copies (x, z and the completions;
C, B and x armed).  A barrier may only be armed again when its last phase is complete, also where one wait has run out: the phase may then
still be open, and the warp that ran out is not always the one that would arm it: that one looks for itself.  The model runs the warps' programs in random order and lets one
wait run out at a time, with the copy that it waited for finishing after everything else.
"""
import random

import pytest

CHUNKS = 4
MEMBERS = {"NEXT": {"mma", "ctl", "elem", "tab"}, "WX": {"elem", "mma"}, "P": {"elem", "mma"}, "YF": {"elem", "mma"}, "G": {"ctl", "elem"},
           "Y": {"ctl", "elem"}, "PX": {"ctl", "elem"}, "DS": {"ctl", "tab", "elem"}, "END": {"mma", "ctl", "elem", "tab"}}


class Fault(Exception):
    pass


class Cta:
    def __init__(self, late, looks, seed, early=0.0):
        self.late, self.looks, self.rng, self.early = late, looks, random.Random(seed), early
        self.expired = False                       # what nobody will complete runs out
        self.armed = dict.fromkeys(("c", "b", "x", "z", "g", "y", "ds", "px"), 0)
        self.done = dict(self.armed)
        self.arrived = {n: set() for n in MEMBERS}
        self.phase = dict.fromkeys(MEMBERS, 0)

    def arm(self, bar):
        if self.done[bar] < self.armed[bar]:
            raise Fault(f"{bar} armed in an open phase")
        self.armed[bar] += 1

    def commit(self, bar):                         # completes by itself, in order
        self.armed[bar] += 1
        self.done[bar] += 1

    def arrive(self, who, name):
        if who in self.arrived[name]:
            raise Fault(f"{who} twice at {name}")
        self.arrived[name].add(who)
        if self.arrived[name] == MEMBERS[name]:
            self.arrived[name] = set()
            self.phase[name] += 1

    def sync(self, who, name):
        target = self.phase[name] + 1
        self.arrive(who, name)
        while self.phase[name] < target:
            yield "barrier"

    def wait(self, me, bar, k):                    # bounded: gives up once
        if me["dead"]:
            return
        out = self.late == (me["name"], bar, k) or self.rng.random() < self.early
        while self.done[bar] <= k and not out:
            yield "copy"
            out = self.expired
        if out:                                    # (also where it was complete after all)
            me["dead"] = True

    def complete_or_dead(self, me, bar):
        me["dead"] = me["dead"] or (self.looks and self.done[bar] < self.armed[bar])

    def drain(self, bar):
        while self.done[bar] < self.armed[bar]:
            yield "drain"

    def mma(self):
        me = dict(name="mma", dead=False)

        def scores(c):
            yield from self.wait(me, "c", c)
            yield from self.wait(me, "b", c)
            self.commit("g")
            yield from self.sync("mma", "YF")
            self.commit("y")
        self.arm("z")
        yield from scores(0)
        for c in range(CHUNKS):
            yield from self.sync("mma", "NEXT")
            if c > 0:
                self.complete_or_dead(me, "z")
                if not me["dead"]:
                    self.arm("z")
            yield from self.sync("mma", "WX")
            if c + 1 < CHUNKS:
                self.commit("ds")
            yield from self.sync("mma", "P")
            self.commit("px")
            if c + 1 < CHUNKS:
                yield from scores(c + 1)
        yield from self.drain("z")
        yield from self.sync("mma", "END")

    def ctl(self):
        me = dict(name="ctl", dead=False)
        for bar in "xcb":
            self.arm(bar)
        self.arrive("ctl", "DS")
        for c in range(CHUNKS):
            more = c + 1 < CHUNKS
            yield from self.wait(me, "x", c)
            yield from self.sync("ctl", "NEXT")
            yield from self.wait(me, "g", c)
            self.arrive("ctl", "G")
            if more:
                self.complete_or_dead(me, "c")
                self.complete_or_dead(me, "b")
            yield from self.wait(me, "y", c)
            if more and not me["dead"]:
                self.arm("c")
            if more:
                yield from self.wait(me, "ds", c)
                if not me["dead"]:
                    self.arm("b")
                self.arrive("ctl", "DS")
            yield from self.wait(me, "z", c)
            self.arrive("ctl", "Y")
            yield from self.wait(me, "px", c)
            if more and not me["dead"]:
                self.arm("x")
            self.arrive("ctl", "PX")
        for bar in "cbx":
            yield from self.drain(bar)
        yield from self.sync("ctl", "END")

    def tab(self):
        for _ in range(CHUNKS):
            self.arrive("tab", "DS")
            yield from self.sync("tab", "NEXT")
        yield from self.sync("tab", "END")

    def elem(self):
        yield from self.sync("elem", "DS")
        self.arrive("elem", "YF")
        for c in range(CHUNKS):
            last = c + 1 == CHUNKS
            yield from self.sync("elem", "NEXT")
            self.arrive("elem", "WX")
            yield from self.sync("elem", "G")
            if not last:
                yield from self.sync("elem", "DS")
            yield from self.sync("elem", "Y")
            self.arrive("elem", "P")
            yield from self.sync("elem", "PX")
            if not last:
                self.arrive("elem", "YF")
        yield from self.sync("elem", "END")

    def run(self):
        warps = {n: getattr(self, n)() for n in ("mma", "ctl", "elem", "tab")}
        waits = dict.fromkeys(warps, None)
        idle = 0
        while warps:
            open_copies = [b for b in "cbxz" if self.done[b] < self.armed[b]]
            late = self.late[1:] if self.late else None
            ready = [b for b in open_copies if (b, self.done[b]) != late]
            if ready and self.rng.random() < 0.3:
                self.done[self.rng.choice(ready)] += 1
                idle = 0
                continue
            name = self.rng.choice(sorted(warps))
            before = (dict(self.phase), {k: set(v) for k, v in self.arrived.items()}, dict(self.armed))
            try:
                waits[name] = next(warps[name])
            except StopIteration:
                del warps[name]
                idle = 0
                continue
            idle = idle + 1 if before == (self.phase, self.arrived, self.armed) else 0
            if idle > 200:                         # nothing else can happen: the late copy arrives
                if open_copies:
                    self.done[open_copies[0]] += 1
                elif self.expired:
                    raise Fault("everybody waits")
                else:
                    self.expired = True
                idle = 0
        assert self.done == self.armed, "left with copies in flight"


LATE = [("mma", b, k) for b in "cb" for k in range(CHUNKS)] + [("ctl", b, k) for b in ("x", "z", "g", "y", "px") for k in range(CHUNKS)] + \
       [("ctl", "ds", k) for k in range(CHUNKS - 1)]


def test_no_wait_runs_out():
    for seed in range(20):
        Cta(None, True, seed).run()


@pytest.mark.parametrize("late", LATE, ids=lambda t: "-".join(map(str, t)))
def test_one_wait_runs_out(late):
    for seed in range(20):
        Cta(late, True, seed).run()


def test_any_waits_run_out():
    for seed in range(300):
        Cta(None, True, seed, early=0.04).run()


@pytest.mark.parametrize("late", [("mma", "c", 0), ("mma", "b", 1), ("ctl", "z", 0)], ids=lambda t: "-".join(map(str, t)))
def test_why_the_one_that_arms_looks(late):
    """Going by its own waits alone it arms a barrier again whose copy is late"""
    def faults(seed):
        try:
            Cta(late, False, seed).run()
        except Fault as e:
            return "armed in an open phase" in str(e)
        return False
    assert any(faults(s) for s in range(20))
