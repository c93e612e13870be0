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
M_WARPS, SPLIT_WARPS, Y_WARPS = 3, 8, 8


Z_BEHIND = 2
STAGES, GATE_STAGES = 3, 4


def counts(heads, local=False):
    c = dict(s=1, cs=1, yread=Y_WARPS)
    for k, n, v in (("full", STAGES, 1), ("empty", STAGES, 2), ("update", 2, SPLIT_WARPS if local else 4 + SPLIT_WARPS), ("last", 2, 1),
                    ("g", 2, 1), ("mread", 2, M_WARPS), ("gates", GATE_STAGES, heads if local else 1), ("ydone", GATE_STAGES, 4 + SPLIT_WARPS if local else Y_WARPS),
                    ("mx", 2, 1), ("mready", 2, M_WARPS), ("zfull", 2, 1), ("yst", 2, Y_WARPS), ("yfree", 2, 1)):
        c.update({f"{k}{i}": v for i in range(n)})
    return c


class Scan(Sim):
    def __init__(self, nch, heads, gated, plant=None, local=False):
        super().__init__(nch, plant)
        self.heads, self.gated, self.m_buffers, self.g_buffers = heads, gated, 2, 3 - heads
        self.b = {k: Bar(k, v) for k, v in counts(heads, local).items()}
        self.local = local     # the state path alone


# The tensor pipe is modelled in order over both issuing threads; a commit arrives when its own
# thread's products are done, which in order is no later.
def issue_state(sim):
    """S update(c), then G(c + 1)."""
    nch, ng, ns = sim.nch, 0, 0

    def scores(c):
        if not (yield ("wait", f"full{c % STAGES}", c // STAGES)):
            return False
        n = sim.g_buffers
        if c >= n and sim.plant != "no_mread" and not (yield ("wait", f"mread{c % n}", c // n - 1)):
            return False
        sim.mma({("C", c % STAGES): c, ("B", c % STAGES): c}, {("G", c % n): (None, c)}, f"G({c})")
        sim.commit(f"g{c % n}")
        return True

    ok = sim.local or (yield from scores(0))
    ng += ok and not sim.local
    for c in range(nch):
        if not ok or (sim.local and not (yield ("wait", f"full{c % STAGES}", c // STAGES))):
            break
        if not (yield ("wait", f"update{c & 1}", c >> 1)):
            break
        sim.mma({("B", c % STAGES): c, **{("W", c & 1 if sim.local else 0, w): c for w in range(SPLIT_WARPS)}},
                {("S", q): ((("S", c) if c else None) if sim.local else ("dec", c), ("S", c + 1)) for q in Q4}, f"S update({c})")
        sim.commit(f"g{c & 1}" if sim.local else "s")
        for _ in range(2 if sim.local else 1):
            sim.commit(f"empty{c % STAGES}")
        ns += 1
        yield None
        if c + 1 < nch and not sim.local:
            ok = yield from scores(c + 1)
            ng += ok
    sim.commit("last0")
    yield ("drain", "last0", 0)
    for c in range(max(0, ng - sim.g_buffers), ng):
        yield ("drain", f"g{c % sim.g_buffers}", c // sim.g_buffers)
    if sim.local:
        for c in range(max(0, ns - 2), ns):
            yield ("drain", f"g{c & 1}", c >> 1)
    elif ns:
        yield ("drain", "s", ns - 1)


def issue_outputs(sim):
    """Yi(c), Ya(c)."""
    nmx = 0
    for c in range(sim.nch):
        if not (yield ("wait", f"full{c % STAGES}", c // STAGES)) or not (yield ("wait", f"update{c & 1}", c >> 1)):
            break
        if c >= 1 and sim.plant != "no_yread" and not (yield ("wait", "yread", c - 1)):
            break
        sim.mma({("C", c % STAGES): c, **{("SB", q): c for q in Q4}},
                {("YI", q): (None, c) for q in Q4}, f"Yi({c})")
        sim.commit("cs")
        if not (yield ("wait", f"mready{c % sim.m_buffers}", c // sim.m_buffers)):
            break
        sim.mma({("X", c % STAGES): c, **{("M", c % sim.m_buffers, w): c for w in range(M_WARPS)}},
                {("YA", q): (None, c) for q in Q4}, f"Ya({c})")
        sim.commit(f"mx{c % sim.m_buffers}")
        sim.commit(f"empty{c % STAGES}")
        nmx += 1
        yield None
    sim.commit("last1")
    yield ("drain", "last1", 0)
    for c in range(max(0, nmx - sim.m_buffers), nmx):
        yield ("drain", f"mx{c % sim.m_buffers}", c // sim.m_buffers)


def copier(sim):
    issued = z = 0
    for c in range(sim.nch + (Z_BEHIND if sim.gated else 0)):
        if c < sim.nch:
            st = c % STAGES
            if c >= STAGES and sim.plant != "no_empty" and not (yield ("wait", f"empty{st}", c // STAGES - 1)):
                break
            sim.copy(([] if sim.local else [("C", st)]) + [("B", st), ("X", st)], c, f"full{st}", "copier")
            issued += 1
        k = c - Z_BEHIND
        if sim.gated and k >= 0:
            if k >= 2 and sim.plant != "no_yfree" and not (yield ("wait", f"yfree{k & 1}", (k >> 1) - 1)):
                break
            sim.copy([("ZY", k & 1, w) for w in range(Y_WARPS)], ("z", k), f"zfull{k & 1}", "copier")
            z += 1
    for c in range(max(0, issued - STAGES), issued):
        yield ("drain", f"full{c % STAGES}", c // STAGES)
    for c in range(max(0, z - 2), z):
        yield ("drain", f"zfull{c & 1}", c >> 1)


def gates(sim, heads):
    for c in range(sim.nch):
        gs = c % GATE_STAGES
        for head in heads:
            if head == heads[0] and c >= GATE_STAGES and not (yield ("wait", f"ydone{gs}", c // GATE_STAGES - 1)):
                return
            sim.write(("GT", gs, head), c, f"gates{heads[0]}")
            yield None
        sim.b[f"gates{gs}"].arrive()


def gates_full(c):
    return ("wait", f"gates{c % GATE_STAGES}", c // GATE_STAGES)


def read_gates(sim, c, who):
    for h in range(sim.heads):
        sim.read(("GT", c % GATE_STAGES, h), c, who)


def state(sim, q):
    who, ok = f"state{q}", True
    if sim.local:
        for c in range(sim.nch):
            if not (yield gates_full(c)):
                break
            if c + 1 < sim.nch:
                sim.b[f"ydone{c % GATE_STAGES}"].arrive()
        yield ("drain", "last0", 0)
        if not sim.abort:
            read_gates(sim, sim.nch - 1, who)
            sim.read(("S", q), ("S", sim.nch), who)
        return
    sim.write(("S", q), ("S", 0), who)
    for c in range(sim.nch):
        if not (ok := (yield gates_full(c))):
            break
        read_gates(sim, c, who)
        if c >= 1 and sim.plant != "late_copy" and not (ok := (yield ("wait", "cs", c - 1))):
            break
        if c >= 1 and not (ok := (yield ("wait", "s", c - 1))):
            break
        sim.read(("S", q), ("S", c), who)
        yield None
        sim.write(("SB", q), c, who)
        sim.write(("S", q), ("dec", c), who)
        yield None
        sim.b[f"update{c & 1}"].arrive()
    if ok and (yield ("wait", "s", sim.nch - 1)):
        sim.read(("S", q), ("S", sim.nch), who)


def outputs(sim, w):
    who, q = f"out{w}", w % 4
    for c in range(sim.nch):
        if not (yield ("wait", f"mx{c % sim.m_buffers}", c // sim.m_buffers)):
            return
        for _ in range(2):
            sim.read(("YI", q), c, who)
            sim.read(("YA", q), c, who)
            read_gates(sim, c, who)
            yield None
        sim.b["yread"].arrive()
        yield None
        sim.b[f"ydone{c % GATE_STAGES}"].arrive()
        if sim.gated and not (yield ("wait", f"zfull{c & 1}", c >> 1)):
            return
        if not sim.gated and c >= 2 and sim.plant != "no_yfree" and not (yield ("wait", f"yfree{c & 1}", (c >> 1) - 1)):
            return
        for part in range(2):
            if sim.gated and part == 0:
                sim.read(("ZY", c & 1, w), ("z", c), who)
                yield None
            sim.write(("ZY", c & 1, w), c, who)
            yield None
        yield None
        sim.b[f"yst{c & 1}"].arrive()


def rows(sim):
    """The output rows' stores (the bulk store's reads end before yfree)."""
    for c in range(sim.nch):
        if not (yield ("wait", f"yst{c & 1}", c >> 1)):
            return
        for _ in range(2):
            for k in range(Y_WARPS):
                sim.read(("ZY", c & 1, k), c, "rows")
            yield None
        sim.b[f"yfree{c & 1}"].arrive()


def scores(sim, w):
    who = f"m{w}"
    for c in range(sim.nch):
        if not (yield gates_full(c)) or not (yield ("wait", f"g{c % sim.g_buffers}", c // sim.g_buffers)):
            return
        m = c % sim.m_buffers
        if c >= sim.m_buffers and sim.plant != "no_mx" and not (yield ("wait", f"mx{m}", c // sim.m_buffers - 1)):
            return
        for _ in range(2):
            sim.read(("G", c % sim.g_buffers), c, who)
            read_gates(sim, c, who)
            sim.write(("M", m, w), c, who)
            yield None
        sim.b[f"mread{c % sim.g_buffers}"].arrive()
        sim.b[f"mready{m}"].arrive()


def split(sim, q):
    who = f"split{q}"
    for c in range(sim.nch):
        st = c % STAGES
        if not (yield gates_full(c)) or not (yield ("wait", f"full{st}", c // STAGES)):
            return
        read_gates(sim, c, who)
        if sim.local:
            sim.b[f"ydone{c % GATE_STAGES}"].arrive()
        sim.read(("X", st), c, who)
        yield None
        if sim.local:
            if c >= 2 and sim.plant != "no_s" and not (yield ("wait", f"g{c & 1}", (c >> 1) - 1)):
                return
        elif c >= 1 and sim.plant != "no_s" and not (yield ("wait", "s", c - 1)):
            return
        sim.write(("W", c & 1 if sim.local else 0, q), c, who)
        yield None
        sim.b[f"update{c & 1}"].arrive()


def run(nch, seed, heads=2, gated=True, plant=None, timeouts=False, local=False, max_steps=300000):
    sim = Scan(nch, heads, gated, plant, local)
    rng = random.Random(seed)
    roles = {"state issue": issue_state(sim), "output issue": issue_outputs(sim), "copier": copier(sim)}
    turns = [[h] for h in range(heads)] if local else [list(range(heads))]      # of the gates' warps
    roles.update({f"gates{t[0]}": gates(sim, t) for t in turns})
    roles.update({f"state{q}": state(sim, q) for q in Q4})
    roles.update({f"out{w}": outputs(sim, w) for w in range(Y_WARPS)})
    roles.update({f"m{w}": scores(sim, w) for w in range(M_WARPS)})
    roles.update({f"split{w}": split(sim, w) for w in range(SPLIT_WARPS)})
    roles["rows"] = rows(sim)
    if local:
        roles = {k: v for k, v in roles.items() if k in ("state issue", "copier") or k.startswith(("gates", "state", "split"))}
    waiting, done = {}, set()
    starved = rng.choice(sorted(roles)) if seed % 2 else None

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
        if not ready:
            raise ProtocolError(f"deadlock: waiting {waiting}")
        # (every other schedule holds one role back, so that the others run as far ahead as they may)
        if starved and len(ready) > 1 and rng.random() < 0.97:
            ready = [r for r in ready if r[0] != starved] or ready
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


@pytest.mark.parametrize("heads,gated", [(1, False), (1, True), (2, False), (2, True)])
@pytest.mark.parametrize("nch", [1, 2, 3, 4, 5, 9])
def test_random_schedules(nch, heads, gated):
    for seed in range(40):
        sim = run(nch, 100 * nch + seed, heads, gated)
        assert all(sim.tags[("S", q)] == ("S", nch) for q in Q4)


@pytest.mark.parametrize("heads", [1, 2])
@pytest.mark.parametrize("nch", [1, 2, 5, 9])
def test_random_schedules_of_the_local_pass(nch, heads):
    for seed in range(40):
        sim = run(nch, 100 * nch + seed, heads, False, local=True)
        assert all(sim.tags[("S", q)] == ("S", nch) for q in Q4)
        run(nch, 700 * nch + seed, heads, False, timeouts=True, local=True)


@pytest.mark.parametrize("plant", ["no_yread", "no_mread", "no_empty", "no_yfree", "no_mx", "no_s", "late_copy"])
def test_planted_mistakes_are_caught(plant):
    with pytest.raises(ProtocolError):
        for seed in range(300):
            run(5, seed, gated=plant != "no_empty", plant=plant)


@pytest.mark.parametrize("nch", [1, 2, 3, 6])
def test_give_up_path_ends_with_nothing_in_flight(nch):
    aborted = sum(run(nch, 900 * nch + seed, timeouts=True).abort for seed in range(80))
    assert aborted > 10


def test_barrier_counts_match_the_kernel():
    src = open(KERNEL).read()
    consts = {k: int(v) for k, v in re.findall(r"\b(k\w+Warps) = (\d+)", src)}
    found = {}
    sizes = {k: int(v) for k, v in re.findall(r"constexpr int (k\w*Stages) = (\d+)", src)}
    loop = None
    for bound, name, many, n in re.findall(r"for \(int i = 0; i < (kStages|kGateStages|2); \+\+i\) \{|mbar_init\(bar\(bars\.(\w+?)(\[i\])?\), (\w+)\)",
                                           src):
        if bound:
            loop = sizes.get(bound) or int(bound)
            continue
        v = {"kHeads": 2, "kGateReaders": Y_WARPS, "kUpdateArrivals": 4 + SPLIT_WARPS, "kGateWriters": 1}.get(n) or (int(n) if n.isdigit() else consts[n])
        found.update({name + i: v for i in (map(str, range(loop)) if many else ("",))})
    assert found == counts(2)


def test_planted_mistakes_of_the_local_pass_are_caught():
    for plant in ("no_s", "no_empty"):
        with pytest.raises(ProtocolError):
            for seed in range(300):
                run(6, seed, gated=False, plant=plant, local=True)
