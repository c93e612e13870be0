"""The scan's skip term D x, which every kernel computes in fp32: it takes no part in the
operand roundings of the chunked kernel's products.

Tolerances (notation of test_state_space.py): a bf16 result is off by half a step, 2^-8 of
it; fp32 sums and the gate by 2^-16 of the terms' magnitudes at most; the chunked kernel's
products by another (1 + 2^-8) 2^-8 of the magnitudes of the scan's own terms, without
|D x|.
"""
import pytest
import torch

import fastaf_kernel_b200 as fk
from test_state_space import F64, HALF, METHODS, TINY, _check, _ref, _scan, _scan_inputs, _step

SHAPES = [
    # lengths, heads, groups, head size
    ([130, 1, 63, 65], 4, 2, 128),
    ([200, 7, 128], 3, 1, 64),              # an odd number of heads in a group
    ([1300, 1640, 2000], 3, 1, 64),         # cut into segments
]


def _skip(i):
    """D x, with the gate where there is one, in 64 bits."""
    y = i["D"].cpu().to(F64)[:, None] * i["x"].cpu().to(F64)
    if i["z"] is not None:
        z = i["z"].cpu().to(F64)
        y = y * z * torch.sigmoid(z)
    return y


def _off_grid(heads, dev):
    """Values of D halfway between bf16 numbers, of both signs and several magnitudes."""
    k = torch.arange(heads, device=dev)
    return (1.0 + 2.0 ** -8 + k * 2.0 ** -6) * torch.where(k % 2 == 0, 1.0, -8.0)


@pytest.mark.gpu
@pytest.mark.parametrize("zero", ["B", "C"])
@pytest.mark.parametrize("z", [False, True])
@pytest.mark.parametrize("method", METHODS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"H{s[1]}G{s[2]}P{s[3]}")
def test_skip_alone_is_rounded_once(shape, method, z, zero):
    """With B or C zero, y is D x (gated), rounded once: 2^-8 of it, and 2^-16 for the fp32
    product and the gate."""
    lengths, H, G, P = shape
    i = _scan_inputs(lengths, H, G, P, z=z, state=zero == "C", seed=70)
    i[zero] = torch.zeros_like(i[zero])
    i["D"] = _off_grid(H, i["x"].device)
    out, _ = _scan(i, lengths, method=method)
    want = _skip(i)
    _check("y", out, want, (HALF + 2.0 ** -16) * want.abs() + TINY)


@pytest.mark.gpu
@pytest.mark.parametrize("z", [False, True])
@pytest.mark.parametrize("method", METHODS)
@pytest.mark.parametrize("scale", [0.01, 1.0, 100.0])
@pytest.mark.parametrize("shape", SHAPES[:2], ids=lambda s: f"H{s[1]}G{s[2]}P{s[3]}")
def test_scan_terms_beside_a_skip(shape, scale, method, z):
    """The scan's own terms keep their precision beside a D of any size: no allowance for
    operand roundings of |D x|."""
    lengths, H, G, P = shape
    i = _scan_inputs(lengths, H, G, P, z=z, seed=71)
    i["D"] = _off_grid(H, i["x"].device) * scale
    out, _ = _scan(i, lengths, method=method)
    y, ymag, _, _ = _ref(i, lengths)
    rounded = HALF * (1 + HALF) if method == "tcgen05" else 0.0
    own = (ymag - _skip(i).abs()).clamp(min=0)
    _check("y", out, y, HALF * y.abs() + rounded * own + 2.0 ** -16 * ymag + TINY)


@pytest.mark.gpu
@pytest.mark.parametrize("P", [64, 128])
def test_prompt_and_step_apply_the_same_skip(P):
    """x of the prompt's tokens and of the next one through the same D: equal bits where the
    scan adds nothing."""
    lengths, H = [70], 4
    i = _scan_inputs(lengths, H, 2, P, z=False, state=False, seed=72)
    i["C"] = torch.zeros_like(i["C"])
    i["D"] = _off_grid(H, i["x"].device)
    prompts = [_scan(i, lengths, method=m)[0] for m in METHODS]
    rows = {k: (None if i[k] is None else i[k]) for k in ("x", "dt", "B", "C")}
    steps, _ = _step(dict(i, **rows, state=None))
    fk.device_status()
    for got in prompts:
        assert torch.equal(got, steps[:, 0])
