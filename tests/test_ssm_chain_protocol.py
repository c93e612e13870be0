"""CPU model of the mbarrier protocol of the chunked selective scan
(fastaf_kernel_b200/csrc/gdn_ssm_tc.cu), run under random schedules: no deadlock, no parity
wait more than one phase away, every read of the chunk it expects, no buffer written while an
asynchronous access of it is in flight, and, when waits run out, every role finishing with
nothing in flight.  The simulator is the one of the delta rule's chains."""
import os
import random
import re

import pytest

from test_tc_chain_protocol import Bar, ProtocolError, Sim

KERNEL = os.path.join(os.path.dirname(__file__), "..", "fastaf_kernel_b200", "csrc", "gdn_ssm_tc.cu")
Q4 = range(4)
M_WARPS, SPLIT_WARPS = 3, 4


def counts(heads):
    one = dict(g=1, mread=M_WARPS, mready=M_WARPS, mx=1, s=1, sready=4, split=SPLIT_WARPS, yread=4, yst=4, yfree=4)
    two = dict(full=1, empty=1, zfull=1, gates=heads, ydone=4, cs=1)
    return {**one, **{f"{k}{i}": v for k, v in two.items() for i in (0, 1)}}


class Scan(Sim):
    def __init__(self, nch, heads, gated, plant=None):
        super().__init__(nch, plant)
        self.heads, self.gated = heads, gated
        self.b = {k: Bar(k, v) for k, v in counts(heads).items()}


def issuer(sim):
    who, nch = "issuer", sim.nch
    ng = nmx = ncs = ns = nfree = 0

    def seen(bar, k):
        return sim.b[bar].test(k, who)

    while nfree < nch:
        sim.progress = False
        if ns < ng and seen("sready", ns) and seen("split", ns):
            sim.mma({("B", ns & 1): ns, **{("WX", w): ns for w in range(SPLIT_WARPS)}},
                    {("S", q): (("dec", ns), ("S", ns + 1)) for q in Q4}, f"S update({ns})")
            sim.commit("s")
            ns += 1
            sim.progress = True
        if (ncs < ng and (ncs < ns or seen("sready", ncs))
                and (ncs == 0 or sim.plant == "no_yread" or seen("yread", ncs - 1))):
            sim.mma({("C", ncs & 1): ncs, **{("SB", ncs & 1, q): ncs for q in Q4}},
                    {("YI", q): (None, ncs) for q in Q4}, f"Yi({ncs})")
            sim.commit(f"cs{ncs & 1}")
            ncs += 1
            sim.progress = True
        if (nmx < ng and seen("mready", nmx) and (nmx < ns or seen("split", nmx))
                and (nmx == 0 or seen("yread", nmx - 1))):
            sim.mma({("X", nmx & 1): nmx, **{("M", w): nmx for w in range(M_WARPS)}},
                    {("YA", q): (None, nmx) for q in Q4}, f"Ya({nmx})")
            sim.commit("mx")
            nmx += 1
            sim.progress = True
        if (ng < nch and ng <= nfree + 1 and seen(f"full{ng & 1}", ng >> 1)
                and (ng == 0 or sim.plant == "no_mread" or seen("mread", ng - 1))):
            sim.mma({("C", ng & 1): ng, ("B", ng & 1): ng}, {("G",): (None, ng)}, f"G({ng})")
            sim.commit("g")
            ng += 1
            sim.progress = True
        if nfree < min(ns, ncs, nmx):
            sim.commit(f"empty{nfree & 1}")
            nfree += 1
            sim.progress = True
        if not sim.progress and sim.abort:
            break
        yield None
    for bar, k in (("g", ng - 1), ("mx", nmx - 1), ("s", ns - 1)):
        if k >= 0:
            yield ("drain", bar, k)
    for c in range(max(0, ncs - 2), ncs):
        yield ("drain", f"cs{c & 1}", c >> 1)
    for c in range(max(0, nfree - 2), nfree):
        yield ("drain", f"empty{c & 1}", c >> 1)


def copier(sim):
    issued = z = 0
    for c in range(sim.nch):
        st = c & 1
        if c >= 2 and sim.plant != "no_empty" and not (yield ("wait", f"empty{st}", (c - 2) >> 1)):
            break
        sim.copy([("C", st), ("B", st), ("X", st)], c, f"full{st}", "copier")
        issued += 1
        if sim.gated:
            if c >= 2 and not (yield ("wait", f"ydone{st}", (c - 2) >> 1)):
                break
            sim.copy([("Z", st)], c, f"zfull{st}", "copier")
            z += 1
    for c in range(max(0, issued - 2), issued):
        yield ("drain", f"full{c & 1}", c >> 1)
    for c in range(max(0, z - 2), z):
        yield ("drain", f"zfull{c & 1}", c >> 1)


def gates(sim, head):
    for c in range(sim.nch):
        if c >= 2 and not (yield ("wait", f"ydone{c & 1}", (c - 2) >> 1)):
            return
        sim.write(("GT", c & 1, head), c, f"gates{head}")
        yield None
        sim.b[f"gates{c & 1}"].arrive()


def read_gates(sim, c, who):
    for h in range(sim.heads):
        sim.read(("GT", c & 1, h), c, who)


def state(sim, q):
    who, ok = f"state{q}", True
    sim.write(("S", q), ("S", 0), who)
    for c in range(sim.nch):
        if not (ok := (yield ("wait", f"gates{c & 1}", c >> 1))):
            break
        read_gates(sim, c, who)
        if c >= 2 and not (ok := (yield ("wait", f"cs{c & 1}", (c - 2) >> 1))):
            break
        if c >= 1 and not (ok := (yield ("wait", "s", c - 1))):
            break
        sim.read(("S", q), ("S", c), who)
        yield None
        sim.write(("SB", c & 1, q), c, who)
        sim.write(("S", q), ("dec", c), who)
        yield None
        sim.b["sready"].arrive()
    if ok and (yield ("wait", "s", sim.nch - 1)):
        sim.read(("S", q), ("S", sim.nch), who)


def outputs(sim, q):
    who = f"out{q}"
    for c in range(sim.nch):
        st = c & 1
        if sim.gated and not (yield ("wait", f"zfull{st}", c >> 1)):
            return
        if not (yield ("wait", f"cs{st}", c >> 1)) or not (yield ("wait", "mx", c)):
            return
        if c > 0 and sim.plant != "no_yfree" and not (yield ("wait", "yfree", c - 1)):
            return
        for half in (0, 1):
            sim.read(("YI", q), c, who)
            sim.read(("YA", q), c, who)
            read_gates(sim, c, who)
            yield None
            if half == 1:
                sim.b["yread"].arrive()
            if sim.gated:
                sim.read(("Z", st), c, who)
            sim.write(("STG", q), c, who)
        yield None
        sim.b[f"ydone{st}"].arrive()
        sim.b["yst"].arrive()
        if not (yield ("wait", "yst", c)):
            return
        for _ in range(2):
            for k in Q4:
                sim.read(("STG", k), c, who)
            yield None
        sim.b["yfree"].arrive()


def scores(sim, w):
    who = f"m{w}"
    for c in range(sim.nch):
        if not (yield ("wait", f"gates{c & 1}", c >> 1)) or not (yield ("wait", "g", c)):
            return
        sim.read(("G",), c, who)
        yield None
        sim.b["mread"].arrive()
        if c >= 1 and sim.plant != "no_mx" and not (yield ("wait", "mx", c - 1)):
            return
        read_gates(sim, c, who)
        sim.write(("M", w), c, who)
        yield None
        sim.b["mready"].arrive()


def split(sim, w):
    who = f"split{w}"
    for c in range(sim.nch):
        st = c & 1
        if not (yield ("wait", f"gates{st}", c >> 1)) or not (yield ("wait", f"full{st}", c >> 1)):
            return
        if c >= 1 and not (yield ("wait", "s", c - 1)):
            return
        read_gates(sim, c, who)
        sim.read(("X", st), c, who)
        yield None
        sim.write(("WX", w), c, who)
        yield None
        sim.b["split"].arrive()


def run(nch, seed, heads=2, gated=True, plant=None, timeouts=False, max_steps=300000):
    sim = Scan(nch, heads, gated, plant)
    rng = random.Random(seed)
    sim.progress, sim.timeouts = False, timeouts
    roles = {"issuer": issuer(sim), "copier": copier(sim)}
    roles.update({f"gates{h}": gates(sim, h) for h in range(heads)})
    roles.update({f"state{q}": state(sim, q) for q in Q4})
    roles.update({f"out{q}": outputs(sim, q) for q in Q4})
    roles.update({f"m{w}": scores(sim, w) for w in range(M_WARPS)})
    roles.update({f"split{w}": split(sim, w) for w in range(SPLIT_WARPS)})
    waiting, done = {}, set()

    def step(name, value=None):
        try:
            r = roles[name].send(value)
        except StopIteration:
            done.add(name)
            return
        if isinstance(r, tuple):
            waiting[name] = r

    for name in roles:
        step(name)
    idle = 0
    for _ in range(max_steps):
        live = [n for n in roles if n not in done]
        if not live:
            if sim.pipe or sim.copies:
                raise ProtocolError("the CTA exits with MMAs or copies in flight")
            return sim
        ready = []
        for n in live:
            if n in waiting:
                kind, bar, k = waiting[n]
                if sim.b[bar].test(k, n):
                    ready.append((n, True))
                elif kind == "wait" and (sim.abort or (timeouts and rng.random() < 0.002)):
                    ready.append((n, False))
            else:
                ready.append((n, None))
        if sim.pipe:
            ready.append(("pipe", None))
        ready += [("copy", i) for i in range(len(sim.copies))]
        # (the polling issuer is always ready; a schedule in which nothing else is and it
        # makes no progress is a deadlock)
        idle = idle + 1 if ready == [("issuer", None)] and not sim.progress else 0
        if not ready or (idle > 3 and not timeouts):
            raise ProtocolError(f"deadlock: waiting {waiting}")
        if idle > 50:
            sim.abort = True        # the issuing thread's own limit
        name, val = ready[rng.randrange(len(ready))]
        if name == "pipe":
            sim.retire_pipe()
        elif name == "copy":
            sim.retire_copy(val)
        else:
            if val is False:
                sim.abort = True
            waiting.pop(name, None)
            step(name, val)
    raise ProtocolError("schedule did not finish")


@pytest.mark.parametrize("heads,gated", [(1, False), (2, True)])
@pytest.mark.parametrize("nch", [1, 2, 3, 4, 5, 9])
def test_random_schedules(nch, heads, gated):
    for seed in range(40):
        sim = run(nch, 100 * nch + seed, heads, gated)
        assert all(sim.tags[("S", q)] == ("S", nch) for q in Q4)


@pytest.mark.parametrize("plant", ["no_yread", "no_mread", "no_empty", "no_yfree", "no_mx"])
def test_planted_mistakes_are_caught(plant):
    with pytest.raises(ProtocolError):
        for seed in range(300):
            run(5, seed, plant=plant)


@pytest.mark.parametrize("nch", [1, 2, 3, 6])
def test_give_up_path_ends_with_nothing_in_flight(nch):
    aborted = sum(run(nch, 900 * nch + seed, timeouts=True).abort for seed in range(80))
    assert aborted > 10


def test_barrier_counts_match_the_kernel():
    src = open(KERNEL).read()
    consts = {k: int(v) for k, v in re.findall(r"\b(k\w+Warps) = (\d+)", src)}
    found = {}
    for name, two, n in re.findall(r"mbar_init\(bar\(bars\.(\w+?)(\[i\])?\), (\w+)\)", src):
        v = {"kHeads": 2}.get(n) or (int(n) if n.isdigit() else consts[n])
        found.update({name + i: v for i in (("0", "1") if two else ("",))})
    assert found == counts(2)
