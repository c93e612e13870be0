"""The scan's local pass over the segments of cut prompts: its barrier counts and registers, and
segments long enough that its rings go round many times and its copies run ahead into L2.

The GPU cases are compared with the token-serial kernel, which is compared with 64 bits
elsewhere, and whose sums of magnitudes (the scan of |x|, |B|, |C| and |state|) the tolerances are
relative to.  Both results are off by half a step of y and 2^-16 of the magnitudes; the chunked one
by another (1 + 2^-8) 2^-8 of the magnitudes without |D x|.  States: 2^-15 of the magnitudes for the
chunked kernel; for the token-serial one a step's decay and sum are off by 1.3 x 2^-22 (two units in
the last place of the exponential, half a one of the sum), over a window of 1 / (1 - decay) < 16
steps with dt_bias above -3 (E softplus(N(-3, 1)) > 0.07, rates at least 1): 2^-17.
"""
import os
import re

import pytest
import torch

import test_ssm_chain_protocol as model
from test_register_budget import NVCC, _ptxas_report
from test_state_space import F64, HALF, TINY, _check, _scan, _scan_inputs

SOURCE = open(os.path.join(os.path.dirname(__file__), "..", "fastaf_kernel_b200", "csrc", "gdn_ssm_tc.cu")).read()


# ------------------------------------------------------------------- counts and registers

def _value(expr, names):
    """An integer expression of the kernel's: names, &&, ?: and numbers."""
    m = re.fullmatch(r"(.+?) \? (.+?) : (.+)", expr)
    if m:
        return _value(m[2], names) if all(names[c.strip()] for c in m[1].split("&&")) else _value(m[3], names)
    return int(expr) if expr.isdigit() else names[expr]


def _counts(pair, local):
    """What every barrier is initialised with in one of the kernel's four instances."""
    names = {"PAIR": pair, "LOCAL": local}
    for line in re.findall(r"constexpr int (k\w+ = [^;]+);", SOURCE):
        for k, v in re.findall(r"(k\w+) = ([^,]+)", line):
            try:
                names[k] = _value(v.strip(), names)
            except KeyError:
                pass                              # (of other things than barriers)
    found, loop = {}, None
    for bound, name, many, n in re.findall(
            r"for \(int i = 0; i < (\w+); \+\+i\) \{|mbar_init\(bar\(bars\.(\w+?)(\[i\])?\), (\w+)\)", SOURCE):
        if bound:
            loop = names.get(bound) or (int(bound) if bound.isdigit() else None)
            continue
        found.update({name + i: _value(n, names) for i in (map(str, range(loop)) if many else ("",))})
    return found


@pytest.mark.parametrize("local", [False, True])
@pytest.mark.parametrize("heads", [1, 2])
def test_barrier_counts_of_every_instance(heads, local):
    assert _counts(heads == 2, local) == model.counts(heads, local)


@pytest.mark.skipif(NVCC is None, reason="nvcc not available")
def test_no_instance_spills(tmp_path):
    rep = {k: v for k, v in _ptxas_report("gdn_ssm_tc.cu", tmp_path).items() if "ssm_tc_kernel" in k}
    assert len(rep) == 4, sorted(rep)                     # heads of 128 or pairs of 64 x main, local pass
    for name, (regs, st, ld) in rep.items():
        assert regs <= 72 and st == 0 and ld == 0, f"{name}: {regs} registers, spills {st}/{ld} bytes"


# --------------------------------------------------------------------------- long segments

def _segment_chunks(tokens, num_seqs, chains, sms):
    """The rule that cuts prompts, in chunks of 64 tokens (0: whole)."""
    body = SOURCE[SOURCE.index("int64_t segment_tokens("):]
    whole, extra, fixed = (float(v) for v in re.search(
        r"double least = ([\d.]+) \*.*?\(\1 \+ ([\d.]+)\) \* static_cast<double>\(part\) \+ ([\d.]+);", body, re.S).groups())
    assert "const int64_t most = sms / chains < chunks / 4 ? sms / chains : chunks / 4;" in body
    chunks = -(-tokens // (num_seqs * 64))
    best, least = 0, whole * chunks
    for k in range(2, min(sms // chains, chunks // 4) + 1):
        part = -(-chunks // k)
        if (whole + extra) * part + fixed < least:
            least, best = (whole + extra) * part + fixed, part
    return best


CASES = [
    # lengths, heads, groups, head size, chains a sequence, chunks of a segment on 148 SMs, state, z
    ([6000], 32, 16, 128, 32, 24, True, False),
    ([16384], 64, 1, 64, 32, 64, False, True),
    ([6001], 63, 1, 64, 32, 24, True, True),                  # a lone head in the last pair
    ([9000], 33, 3, 64, 18, 18, True, False),                 # one in every group
    ([5000, 1, 7300], 14, 7, 128, 14, 22, True, True),
    ([4097, 3000, 4800], 20, 4, 64, 12, 16, False, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0][0]}-H{c[1]}G{c[2]}P{c[3]}")
def test_the_cases_have_long_segments(case):
    lengths, H, G, P, chains, chunks, _, _ = case
    assert chains == (G * (-(-(H // G) // 2)) if P == 64 else H)
    assert _segment_chunks(sum(lengths), len(lengths), chains * len(lengths), 148) == chunks


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0][0]}-H{c[1]}G{c[2]}P{c[3]}")
def test_long_segments(case):
    lengths, H, G, P, _, _, state, z = case
    i = _scan_inputs(lengths, H, G, P, wide=True, state=state, z=z, seed=95)
    i["dt_bias"] = i["dt_bias"].clamp(min=-3.0)
    out, new = _scan(i, lengths, method="tcgen05")
    ref, ref_new = _scan(i, lengths, method="recurrent")
    mags = {k: (None if i[k] is None else i[k].abs()) for k in ("x", "B", "C", "state")}
    own, smag = _scan(dict(i, **mags, D=None, z=None), lengths, method="recurrent")
    own = own.to(F64) * (1 + 2 * HALF)                                   # (rounded to bf16)
    skip = (i["D"].to(F64)[:, None] * i["x"].to(F64)).abs()
    if z:
        gate = (i["z"].to(F64) * torch.sigmoid(i["z"].to(F64))).abs()
        own, skip = own * gate, skip * gate
    want = ref.to(F64)
    _check("y", out, want.cpu(), (2 * HALF * (1 + 2 * HALF) * want.abs() + HALF * (1 + HALF) * own
                                  + 2.0 ** -15 * (own + skip) + TINY).cpu())
    _check("state", new, ref_new.to(F64).cpu(), ((2.0 ** -15 + 2.0 ** -16) * smag.to(F64) + TINY).cpu())
    again = _scan(i, lengths, method="tcgen05")
    assert torch.equal(again[0], out) and torch.equal(again[1], new)
