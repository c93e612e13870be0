"""Decays at the ends of their range: rates exp(A_log) beyond fp32, which forget the state at
every step that has a length, and steps of length zero, which leave it alone all the same.

A chunk's log2 decays are sums of up to 64 terms of at most 160 here, below 2^14, so that one
fp32 rounding of them is off by up to 2^-11 and an exponential of a difference of two of them
by 2 ln 2 2^-11 < 2^-10 relative; all other tolerances are those of test_state_space.py.
"""
import pytest
import torch

from test_state_space import HALF, METHODS, TINY, _check, _ref, _scan, _scan_inputs, _step


def _check_y(out, ref, method):
    y, ymag, _, _ = ref
    rounded = HALF * (1 + HALF) + 2.0 ** -10 if method == "tcgen05" else 0.0
    _check("y", out.reshape(y.shape), y, HALF * y.abs() + (rounded + 2.0 ** -16) * ymag + TINY)


@pytest.mark.gpu
@pytest.mark.parametrize("rate", [88.0, 88.6, 100.0, 3e38])
@pytest.mark.parametrize("length", [64, 70, 127, 129])
@pytest.mark.parametrize("H,G,P", [(2, 1, 128), (3, 1, 64)])
@pytest.mark.parametrize("method", METHODS)
def test_rates_beyond_fp32(method, H, G, P, length, rate):
    """Whole and partial chunks, two sequences: the state is what the last token adds, and
    finite everywhere; heads beside them are as they are without."""
    lengths = [length, 65]
    i = _scan_inputs(lengths, H, G, P, seed=80)
    plain = _scan(i, lengths, method=method)
    j = dict(i, A_log=i["A_log"].clone())
    j["A_log"][1] = rate
    out, new = _scan(j, lengths, method=method)
    # (in 64 bits exp(200) is far beyond what the smallest step here needs to forget everything)
    ref = _ref(dict(j, A_log=j["A_log"].clamp(max=200.0)), lengths)
    _check_y(out, ref, method)
    _check("state", new, ref[2], 2.0 ** -15 * ref[3] + TINY)
    keep = [h for h in range(H) if h != 1]
    assert torch.equal(out[:, keep], plain[0][:, keep]) and torch.equal(new[:, keep], plain[1][:, keep])


@pytest.mark.gpu
@pytest.mark.parametrize("method", METHODS)
def test_steps_of_length_zero_at_rates_beyond_fp32(method):
    """dt = -inf: a step of exactly zero leaves the state alone at any rate."""
    lengths = [90, 40]
    i = _scan_inputs(lengths, 4, 2, 64, dt_dtype=torch.float32, seed=81)
    i["A_log"][1:3] = 100.0
    i["dt"][60:90] = float("-inf")                     # the first sequence's last tokens
    i["dt"][100, 2] = float("-inf")
    out, new = _scan(i, lengths, method=method)
    ref = _ref(i, lengths)
    _check_y(out, ref, method)
    _check("state", new, ref[2], 2.0 ** -15 * ref[3] + TINY)


@pytest.mark.gpu
def test_single_tokens_at_rates_beyond_fp32():
    i = _scan_inputs([1] * 5, 4, 2, 64, dt_dtype=torch.float32, seed=82)
    i["A_log"][1:3] = 100.0
    i["dt"][2:4] = float("-inf")
    out, new = _step(i)
    ref = _ref(i, [1] * 5)
    _check_y(out, ref, "decode")
    _check("state", new, ref[2], 2.0 ** -18 * ref[3] + TINY)
    assert torch.equal(new[2:4], i["state"][2:4])


@pytest.mark.gpu
@pytest.mark.parametrize("H,P", [(2, 128), (3, 64)])
def test_rates_beyond_fp32_in_cut_prompts(H, P):
    """Segments, whose local pass sums decays from their ends."""
    lengths = [2500, 2533]
    i = _scan_inputs(lengths, H, 1, P, seed=83)
    i["A_log"][1] = 100.0
    out, new = _scan(i, lengths, method="tcgen05")
    ref = _ref(i, lengths)
    _check_y(out, ref, "tcgen05")
    _check("state", new, ref[2], 2.0 ** -15 * ref[3] + TINY)
