"""The scan's protocol with the state update in three terms.  With one head, and in the local pass,
the third lies beside the others and shares their hand-overs (the model of
test_ssm_chain_protocol.py holds as it is); with two heads of the main pass it takes the place of
bf16(S) once Yi has read that, and its products follow the next chunk's scores, which is modelled
here on top of the outputs' reads of x."""
import pytest

import test_ssm_chain_protocol as model
import test_ssm_skip_protocol as skip
from test_ssm_chain_protocol import KERNEL, M_WARPS, SPLIT_WARPS, STAGES, ProtocolError, Q4, gates_full, read_gates

SB = [("SB", w) for w in range(SPLIT_WARPS)]      # the rows of one split warp each; quadrant w % 4


def counts(heads, local=False, _plain=model.counts):
    return dict(_plain(heads, local), third=SPLIT_WARPS)


def issue_state(sim):
    nch, ng, ns = sim.nch, 0, 0

    def scores(c):
        if not (yield ("wait", f"full{c % STAGES}", c // STAGES)):
            return False
        if c >= 1 and not (yield ("wait", "mread0", c - 1)):
            return False
        sim.mma({("C", c % STAGES): c, ("B", c % STAGES): c}, {("G", 0): (None, c)}, f"G({c})")
        sim.commit("g0")
        return True

    ok = yield from scores(0)
    ng += ok
    for c in range(nch):
        if not ok or not (yield ("wait", f"update{c & 1}", c >> 1)):
            break
        sim.mma({("B", c % STAGES): c, **{("W", 0, w): c for w in range(SPLIT_WARPS)}},
                {("S", q): (("dec", c), ("two", c)) for q in Q4}, f"two terms({c})")
        if sim.plant == "early_s":
            sim.commit("s")
        yield None
        if c + 1 < nch:
            ok = yield from scores(c + 1)
            ng += ok
            if not ok:
                break
        if not (yield ("wait", "third", c)):
            break
        sim.mma({("B", c % STAGES): c, **{p: ("third", c) for p in SB}},
                {("S", q): (("two", c), ("S", c + 1)) for q in Q4}, f"third term({c})")
        if sim.plant != "early_s":
            sim.commit("s")
        sim.commit(f"empty{c % STAGES}")
        ns += 1
        yield None
    sim.commit("last0")
    yield ("drain", "last0", 0)
    if ng:
        yield ("drain", "g0", ng - 1)
    if ns:
        yield ("drain", "s", ns - 1)


def issue_outputs(sim):
    nmx = 0
    for c in range(sim.nch):
        if not (yield ("wait", f"full{c % STAGES}", c // STAGES)) or not (yield ("wait", f"update{c & 1}", c >> 1)):
            break
        if c >= 1 and not (yield ("wait", "yread", c - 1)):
            break
        sim.mma({("C", c % STAGES): c, **{p: c for p in SB}}, {("YI", q): (None, c) for q in Q4}, f"Yi({c})")
        sim.commit("cs")
        if not (yield ("wait", f"mready{c % 2}", c // 2)):
            break
        sim.mma({("X", c % STAGES): c, **{("M", c % 2, w): c for w in range(M_WARPS)}},
                {("YA", q): (None, c) for q in Q4}, f"Ya({c})")
        sim.commit(f"mx{c % 2}")
        sim.commit(f"empty{c % STAGES}")
        nmx += 1
        yield None
    sim.commit("last1")
    yield ("drain", "last1", 0)
    for c in range(max(0, nmx - 2), nmx):
        yield ("drain", f"mx{c % 2}", c // 2)


def state(sim, q):
    who, ok = f"state{q}", True
    sim.write(("S", q), ("S", 0), who)
    for c in range(sim.nch):
        if not (ok := (yield gates_full(c))):
            break
        read_gates(sim, c, who)
        if c >= 1 and not (ok := (yield ("wait", "cs", c - 1))):
            break
        if c >= 1 and sim.plant != "no_s" and not (ok := (yield ("wait", "s", c - 1))):
            break
        sim.read(("S", q), ("S", c), who)
        yield None
        for w in (q, q + 4):
            sim.write(("SB", w), c, who)
        sim.write(("S", q), ("dec", c), who)
        yield None
        sim.b[f"update{c & 1}"].arrive()
    if ok and (yield ("wait", "s", sim.nch - 1)):
        sim.read(("S", q), ("S", sim.nch), who)


def split(sim, w):
    who = f"split{w}"
    for c in range(sim.nch):
        st = c % STAGES
        if not (yield gates_full(c)) or not (yield ("wait", f"full{st}", c // STAGES)):
            return
        read_gates(sim, c, who)
        sim.read(("X", st), c, who)
        yield None
        if c >= 1 and not (yield ("wait", "s", c - 1)):
            return
        sim.write(("W", 0, w), c, who)
        yield None
        sim.b[f"update{c & 1}"].arrive()
        if sim.plant != "no_cs" and not (yield ("wait", "cs", c)):
            return
        sim.write(("SB", w), ("third", c), who)
        yield None
        sim.b["third"].arrive()


@pytest.fixture(autouse=True)
def _roles(monkeypatch):
    for name, role in (("counts", counts), ("issue_state", issue_state), ("issue_outputs", issue_outputs), ("state", state),
                       ("split", split), ("copier", skip.copier), ("outputs", skip.outputs)):
        monkeypatch.setattr(model, name, role)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("nch", [1, 2, 3, 4, 5, 9, 14])
def test_random_schedules(nch, gated):
    for seed in range(60):
        sim = model.run(nch, 100 * nch + seed, 2, gated)
        assert all(sim.tags[("S", q)] == ("S", nch) for q in Q4)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("nch", [1, 2, 3, 6, 10])
def test_give_up_path_ends_with_nothing_in_flight(nch, gated):
    aborted = sum(model.run(nch, 900 * nch + seed, 2, gated, timeouts=True).abort for seed in range(80))
    assert aborted > 10


@pytest.mark.parametrize("plant", ["no_cs", "early_s", "no_s"])
def test_planted_mistakes_are_caught(plant):
    with pytest.raises(ProtocolError):
        for seed in range(400):
            model.run(6, seed, 2, False, plant=plant)


def test_the_kernel_has_the_models_order_and_count():
    src = " ".join(open(KERNEL).read().split())
    assert "mbar_init(smem_u32(&bars.third), kSplitWarps);" in src
    issue = src[src.index("-- state update and G"):src.index("-- Yi and Ya")]
    loop = issue[issue.index("for (int c = 0; ok && c < nch; ++c)"):]
    order = [loop.index(s) for s in ("bars.update[c & 1]", "tm + TM::S, w + 8 * k", "scores(c + 1)", "bars.third", "TM::W3 + 8 * k",
                                     "mma_commit(bar(bars.s))", "mma_commit(bar(bars.empty[c % kStages])); } __syncwarp(); ++ns")]
    assert order == sorted(order)
    w = src[src.index("-- w x in three terms"):]
    order = [w.index(s) for s in ("bars.update[c & 1]", "bar(bars.cs), c, kSsmCS", "TM::W3), w3", "tmem_wait_st", "&bars.third")
             if s != "tmem_wait_st"]
    assert order == sorted(order)
