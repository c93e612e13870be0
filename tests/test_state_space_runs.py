"""The convolution where a thread takes more than one batch of rows: large batches, whose threads
carry their window from batch to batch, go round the ring of rows ahead and meet sequence
boundaries in later batches, and single tokens of several sequences a thread.

Tolerances are those of test_state_space.py; the 64-bit reference runs on the GPU.
"""
import os
import re

import pytest
import torch

import fastaf_kernel_b200 as fk
from test_state_space import DEV, F64, HALF, TINY, _conv_inputs, _cu

SOURCE = os.path.join(os.path.dirname(__file__), "..", "fastaf_kernel_b200", "csrc", "gdn_conv.cu")
C = 8192


def _rule():
    """(longest, shortest) run of prompts and of single tokens, threads wanted on an SM, and channels
    of a thread: what pick_run is given, read from the source."""
    src = open(SOURCE).read()
    consts = {k: int(v) for k, v in re.findall(r"constexpr int (k\w+) = (\d+);", src)}
    num = lambda v: consts.get(v) or int(v)
    (p, d) = re.findall(r"pick_run\(p\.rows, p\.channels / kVec, (\w+), (\w+)\)", src)
    want, = re.findall(r"const int64_t want = static_cast<int64_t>\(sm_count\(\)\) \* (\d+);", src)
    assert "int run = longest;" in src and "while (run > shortest && ((rows + run - 1) / run) * groups < want) run /= 2;" in src
    return tuple(map(num, p)), tuple(map(num, d)), int(want), consts["kVec"], consts["kBatchRows"], consts["kBatches"]


def _run_of(rows, channels, decode, sms):
    prompts, tokens, want, vec, _, _ = _rule()
    longest, shortest = tokens if decode else prompts
    run = longest
    while run > shortest and -(-rows // run) * (channels // vec) < want * sms:
        run //= 2
    return run


def _sms():
    return torch.cuda.get_device_properties(DEV).multi_processor_count


def _lengths(rows):
    """Ragged lengths that sum to rows: tiny and empty ones in a row, so that several boundaries
    fall into one batch, and longer ones that end anywhere in a run."""
    lengths, k = [], 0
    while sum(lengths) < rows:
        lengths += [k % 6, 0, 1 + 13 * k % 40, 97 + 11 * k]
        k += 1
    over = sum(lengths) - rows
    while over:
        cut = min(over, lengths[-1])
        lengths[-1] -= cut
        over -= cut
        if over:
            lengths.pop()
    return lengths + [0]


def _check_conv(y, new, x, w, b, st, lengths, act):
    """Against 64 bits, some channels at a time."""
    n, K = len(lengths), w.shape[1]
    starts = [sum(lengths[:i]) for i in range(n)]
    # rows of [state; x] of all sequences, one behind the other
    at = torch.cat([torch.arange(K - 1 + L) + (s + i * (K - 1)) for i, (s, L) in enumerate(zip(starts, lengths))])
    assert at.numel() == sum(lengths) + n * (K - 1)
    place = torch.cat([torch.arange(L) + s + (i + 1) * (K - 1) for i, (s, L) in enumerate(zip(starts, lengths))]).to(DEV)
    front = torch.cat([torch.arange(K - 1) + s + i * (K - 1) for i, s in enumerate(starts)]).to(DEV)
    last = torch.cat([torch.arange(K - 1) + s + L + i * (K - 1) for i, (s, L) in enumerate(zip(starts, lengths))]).to(DEV)
    for c in range(0, x.shape[1], 2048):
        sl = slice(c, c + 2048)
        wide = min(2048, x.shape[1] - c)
        rows = torch.zeros((at.numel(), wide), dtype=F64, device=DEV)
        rows[place] = x[:, sl].to(F64)
        if st is not None:
            rows[front] = st[:, :, sl].reshape(-1, wide).to(F64)
        terms = [rows[place - (K - 1 - k)] * w[sl, k].to(F64) for k in range(K)]
        want, mag = sum(terms), sum(t.abs() for t in terms)
        if b is not None:
            want, mag = want + b[sl].to(F64), mag + b[sl].to(F64).abs()
        if act:
            want = want * torch.sigmoid(want)
        over = (y[:, sl].to(F64) - want).abs() - (HALF * want.abs() + 2.0 ** -16 * mag + TINY)
        assert bool((over <= 0).all()), f"channels {c}..: {int((over > 0).sum())} off, by up to {float(over.max()):.3e}"
        assert torch.equal(new[:, :, sl].reshape(-1, wide).to(F64), rows[last])


def test_the_rule_is_read_from_the_source():
    prompts, tokens, want, vec, batch, batches = _rule()
    assert prompts == (64, 4) and tokens == (4, 1) and want == 1024 and vec == 4 and (batch, batches) == (4, 4)


PROMPTS = [
    # rows, the run they get on 148 SMs, width, bias, state, wide rows, activation, type of the weights
    (613, 8, 4, True, True, False, "silu", torch.float32),
    (1201, 16, 3, False, True, True, None, torch.bfloat16),
    (2417, 32, 2, True, False, False, "silu", torch.bfloat16),
    (2417, 32, 4, False, True, True, "silu", torch.float32),
    (4801, 64, 4, True, True, False, "silu", torch.float32),
    (4863, 64, 3, False, False, True, None, torch.float32),
    (4801, 64, 2, True, True, True, "silu", torch.float32),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,run,K,bias,state,wide,act,dtype", PROMPTS)
def test_conv_prefill_of_long_runs(rows, run, K, bias, state, wide, act, dtype):
    if _sms() == 148:
        assert _run_of(rows, C, False, 148) == run
    lengths = _lengths(rows)
    x, w, b, st = _conv_inputs(lengths, C, K, bias, state, wide, dtype, seed=90)
    y, new = fk.conv_prefill(x, w, b, st, _cu(lengths), activation=act)
    fk.device_status()
    _check_conv(y, new, x, w, b, st, lengths, act)


@pytest.mark.gpu
def test_long_runs_split_and_rows_behind():
    """Run 64: packed parts, rows behind the last sequence, and a whole batch as one sequence."""
    rows, kept = 4801, 4750
    x, w, b, st = _conv_inputs([rows], C, 4, seed=91)
    y, new = fk.conv_prefill(x, w, b, st, _cu([rows]))
    fk.device_status()
    _check_conv(y, new, x, w, b, st, [rows], "silu")
    parts, new2 = fk.conv_prefill(x, w, b, st, _cu([rows]), split=(2048, 4088, 2056))
    assert torch.equal(torch.cat(parts, 1), y) and torch.equal(new, new2)
    out = torch.full((rows, C), 7.0, dtype=torch.bfloat16, device=DEV)
    fk.conv_prefill(x, w, b, st, _cu([kept]), output=out)
    with pytest.raises(ValueError, match="cu_seqlens"):
        fk.device_status()
    assert torch.equal(out[:kept], y[:kept]) and bool((out[kept:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("K", [2, 3, 4])
@pytest.mark.parametrize("batch,run", [(151, 2), (301, 4), (515, 4)])
def test_conv_decode_of_several_sequences_a_thread(batch, run, K):
    if _sms() == 148:
        assert _run_of(batch, C, True, 148) == run
    lengths = [1] * batch
    x, w, b, st = _conv_inputs(lengths, C, K, wide=batch == 301, seed=92)
    y, new = fk.conv_decode(x, w, b, st)
    _check_conv(y, new, x, w, b, st, lengths, "silu")
    kept = st.clone()
    y2, n2 = fk.conv_decode(x, w, b, kept, new_state=kept)
    assert n2 is kept and torch.equal(y2, y) and torch.equal(kept, new)
    (p, q), n3 = fk.conv_decode(x, w, b, st, split=(8, C - 8))
    assert torch.equal(torch.cat([p, q], 1), y) and torch.equal(n3, new)
    none, _ = fk.conv_decode(x, w, None, None, activation=None)
    want = (x.to(F64) * w[:, K - 1].to(F64))
    assert bool(((none.to(F64) - want).abs() <= (HALF + 2.0 ** -16) * want.abs() + TINY).all())
