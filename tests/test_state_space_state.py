"""The state that comes back is as good as fp32 sums, from either prompt kernel.

A term dt' x decay B of the state is off by at most 2^-20 of itself: half a step for the product in
fp32, two units in the last place for the exponential (2^-22), as much for softplus and its
division, and for the sum of log2 decays s behind a token, of at most 6 additions, 6 s 2^-24 ln 2
times a weight 2^-s, below 2^-22 of the largest weight.  A token's error is the same for all its
terms; tokens' terms have signs of their own, so that the error's norm is at most 2^-20 of the
state's.  The tensor core's sums measured 1e-7 of the state for 128 tokens without a decay, below
2^-21 for the windows here.  Together below 1.5 x 2^-20, where a term cut to 16 bits would be off by
2^-18 (3.8e-6).
"""
import pytest
import torch

from test_state_space import F64, METHODS, _ref, _scan, _scan_inputs

BOUND = 1.5 * 2.0 ** -20

SHAPES = [
    # lengths, heads, groups, head size
    ([64], 2, 1, 128),
    ([130, 1, 63, 400], 4, 2, 128),
    ([200, 7, 128], 3, 1, 64),              # a lone head in the last pair
    ([1000], 4, 4, 64),                     # one head a group: lone in every pair
    ([1300, 1640, 2000], 3, 1, 64),         # cut into segments
    ([3000, 2500], 2, 1, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dt_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("method", METHODS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{sum(s[0])}-H{s[1]}G{s[2]}P{s[3]}")
def test_state_is_as_good_as_fp32_sums(shape, method, state, dt_dtype):
    lengths, H, G, P = shape
    i = _scan_inputs(lengths, H, G, P, state=state, z=False, dt_dtype=dt_dtype, seed=100)
    i["dt_bias"] = i["dt_bias"].clamp(min=-3.0)              # (windows of 16 tokens and less, on average)
    _, new = _scan(i, lengths, method=method)
    want = _ref(i, lengths)[2]
    for n in range(len(lengths)):
        for h in range(H):
            err, size = (new[n, h].cpu().to(F64) - want[n, h]).norm(), want[n, h].norm()
            assert float(err) <= BOUND * float(size), f"sequence {n}, head {h}: {float(err / size):.2e}"
