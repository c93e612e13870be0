"""The scan's protocol with the outputs' reads of x (for D x): the model of
test_ssm_chain_protocol.py, whose output warps here read the stage's x tile before they hand
back a chunk's gates, and whose copies wait for that before they fill the stage again."""
import random

import pytest

import test_ssm_chain_protocol as model
from test_ssm_chain_protocol import GATE_STAGES, KERNEL, STAGES, Y_WARPS, Z_BEHIND, ProtocolError, Q4, read_gates


def copier(sim):
    issued = z = 0
    for c in range(sim.nch + (Z_BEHIND if sim.gated else 0)):
        if c < sim.nch:
            st = c % STAGES
            if c >= STAGES:
                if not (yield ("wait", f"empty{st}", c // STAGES - 1)):
                    break
                k = c - STAGES
                if sim.plant != "no_x" and not (yield ("wait", f"ydone{k % GATE_STAGES}", k // GATE_STAGES)):
                    break
            sim.copy([("C", st), ("B", st), ("X", st)], c, f"full{st}", "copier")
            issued += 1
        k = c - Z_BEHIND
        if sim.gated and k >= 0:
            if k >= 2 and not (yield ("wait", f"yfree{k & 1}", (k >> 1) - 1)):
                break
            sim.copy([("ZY", k & 1, w) for w in range(Y_WARPS)], ("z", k), f"zfull{k & 1}", "copier")
            z += 1
    for c in range(max(0, issued - STAGES), issued):
        yield ("drain", f"full{c % STAGES}", c // STAGES)
    for c in range(max(0, z - 2), z):
        yield ("drain", f"zfull{c & 1}", c >> 1)


def outputs(sim, w):
    who, q = f"out{w}", w % 4
    for c in range(sim.nch):
        if not (yield ("wait", f"mx{c % sim.m_buffers}", c // sim.m_buffers)):
            return
        if not (yield ("wait", f"full{c % STAGES}", c // STAGES)):
            return
        sim.read(("YI", q), c, who)
        sim.read(("YA", q), c, who)
        read_gates(sim, c, who)
        yield None
        sim.b["yread"].arrive()
        yield None
        for _ in range(2):
            if sim.plant == "late_x":
                break
            sim.read(("X", c % STAGES), c, who)
            yield None
        sim.b[f"ydone{c % GATE_STAGES}"].arrive()
        if sim.plant == "late_x":
            yield None
            sim.read(("X", c % STAGES), c, who)
        if sim.gated and not (yield ("wait", f"zfull{c & 1}", c >> 1)):
            return
        if not sim.gated and c >= 2 and not (yield ("wait", f"yfree{c & 1}", (c >> 1) - 1)):
            return
        if sim.gated:
            sim.read(("ZY", c & 1, w), ("z", c), who)
            yield None
        sim.write(("ZY", c & 1, w), c, who)
        yield None
        sim.b[f"yst{c & 1}"].arrive()


@pytest.fixture(autouse=True)
def _roles(monkeypatch):
    monkeypatch.setattr(model, "copier", copier)
    monkeypatch.setattr(model, "outputs", outputs)


@pytest.mark.parametrize("heads,gated", [(1, False), (1, True), (2, False), (2, True)])
@pytest.mark.parametrize("nch", [1, 2, 3, 4, 5, 9, 14])
def test_random_schedules(nch, heads, gated):
    for seed in range(40):
        sim = model.run(nch, 100 * nch + seed, heads, gated)
        assert all(sim.tags[("S", q)] == ("S", nch) for q in Q4)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("nch", [1, 2, 3, 6, 10])
def test_give_up_path_ends_with_nothing_in_flight(nch, gated):
    aborted = sum(model.run(nch, 900 * nch + seed, gated=gated, timeouts=True).abort for seed in range(80))
    assert aborted > 10


@pytest.mark.parametrize("plant", ["no_x", "late_x"])
def test_planted_mistakes_are_caught(plant):
    with pytest.raises(ProtocolError):
        for seed in range(400):
            model.run(7, seed, heads=1 + random.Random(seed).randrange(2), gated=False, plant=plant)


def test_the_kernel_waits_as_the_model_does():
    src = " ".join(open(KERNEL).read().split())
    assert ("if (!LOCAL && c >= kStages && !wait.warp(bar(bars.ydone[(c - kStages) & (kGateStages - 1)]), "
            "(c - kStages) / kGateStages, kSsmY)) break;") in src
    at = src.index("-- outputs")
    outs = src[at:src.index("-- output rows")]
    order = [outs.index(s) for s in ("kSsmMX", "bars.full[c % kStages]", "bars.yread", "ldsm_x4_t(xr", "bars.ydone",
                                     "bars.zfull", "bars.yst")]
    assert order == sorted(order)
