"""Calls that the documentation allows and that are easy to get wrong: no rows, single rows, types
that are converted, offsets on the host or in 64 bits, broadcast and far-apart rows, the same
tensor twice, and the largest group."""
import pytest
import torch

import fastaf_kernel_b200 as fk
from test_state_space import (DEV, HALF, METHODS, TINY, _check, _check_scan, _conv_inputs, _conv_ref, _cu, _ref, _scan,
                              _scan_inputs, _step)


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("state", [False, True])
def test_no_rows(state):
    x, w, b, st = _conv_inputs([0, 0, 0], 64, 4, state=state)
    y, new = fk.conv_prefill(x, w, b, st, _cu([0, 0, 0]))
    assert y.shape == (0, 64) and torch.equal(new, st if state else torch.zeros_like(new))
    (p, q), _ = fk.conv_prefill(x, w, b, st, _cu([0, 0, 0]), split=(8, 56))
    assert p.shape == (0, 8) and q.shape == (0, 56)
    y, new = fk.conv_decode(x, w, b, st[:0] if state else None)
    assert y.shape == (0, 64) and new.shape == (0, 3, 64)
    i = _scan_inputs([0, 0], 3, 1, 64, state=state)
    for m in ("auto", "recurrent"):
        out, new = _scan(i, [0, 0], method=m)
        assert out.shape == (0, 3, 64) and torch.equal(new, i["state"] if state else torch.zeros_like(new))
    out, new = _step(dict(i, state=None))
    assert out.shape == (0, 1, 3, 64) and new.shape == (0, 3, 64, 128)
    y, new = fk.conv_prefill(x, w, b, None, torch.zeros(1, dtype=torch.int32, device=DEV))       # no sequence either
    assert y.shape == (0, 64) and new.shape == (0, 3, 64)


@pytest.mark.gpu
def test_one_row_of_a_wider_one():
    """A single row is contiguous whatever its stride says."""
    x, w, b, st = _conv_inputs([1], 64, 4, wide=True)
    y, new = fk.conv_prefill(x, w, b, st, _cu([1]))
    ry, mag, rs = _conv_ref(x, w, b, st, [1], "silu")
    _check("y", y, ry, HALF * ry.abs() + 2.0 ** -16 * mag + TINY)
    _check("state", new, rs, 0.0)
    i = _scan_inputs([1], 6, 2, 64, wide=True)
    out, new = _scan(i, [1])
    _check_scan(out, new, _ref(i, [1]), "recurrent")
    assert _same(_step(i), (out[:, None], new))


@pytest.mark.gpu
@pytest.mark.parametrize("method", METHODS)
def test_offsets_of_other_types_and_places(method):
    lengths = [70, 0, 61]
    x, w, b, st = _conv_inputs(lengths, 64, 4)
    i = _scan_inputs(lengths, 2, 1, 64)
    scan = lambda cu: fk.ssm_prefill(i["x"], i["dt"], i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], i["state"], cu,
                                     z=i["z"], method=method)
    conv = lambda cu: fk.conv_prefill(x, w, b, st, cu)
    cu = _cu(lengths)
    spread = torch.stack([cu, cu], 1)[:, 0]                      # not contiguous
    for other in (cu.long(), cu.cpu(), cu.cpu().long(), spread):
        assert _same(scan(other), scan(cu)) and _same(conv(other), conv(cu))
    for bad in (cu.cpu() + 1, cu.cpu().flip(0), cu[None], cu[:0]):
        with pytest.raises(ValueError):
            scan(bad)
        with pytest.raises(ValueError):
            conv(bad)
    fk.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("method", METHODS)
def test_types_that_are_converted(method):
    """Parameters and states of types the kernels do not read: the bits of converted ones."""
    lengths = [70, 61]
    x, w, b, st = _conv_inputs(lengths, 64, 4)
    half = lambda t: t.half()
    assert _same(fk.conv_prefill(x, half(w), half(b), st, _cu(lengths)),
                 fk.conv_prefill(x, half(w).float(), half(b).float(), st, _cu(lengths)))
    assert _same(fk.conv_prefill(x, w, b.to(torch.bfloat16), st, _cu(lengths)),
                 fk.conv_prefill(x, w, b.to(torch.bfloat16).float(), st, _cu(lengths)))
    assert _same(fk.conv_prefill(x, w, b, st.float(), _cu(lengths)), fk.conv_prefill(x, w, b, st, _cu(lengths)))
    i = _scan_inputs(lengths, 2, 1, 64)
    j = dict(i, dt=i["dt"].half(), A_log=i["A_log"].double(), D=i["D"].half(), dt_bias=i["dt_bias"].to(torch.bfloat16),
             state=i["state"].double())
    k = dict(i, dt=i["dt"].half().float(), D=i["D"].half().float(), dt_bias=i["dt_bias"].to(torch.bfloat16).float())
    assert _same(_scan(j, lengths, method=method), _scan(k, lengths, method=method))


@pytest.mark.gpu
@pytest.mark.parametrize("method", METHODS)
def test_broadcast_rows_and_the_same_tensor_twice(method):
    """Rows expanded from one (stride 0), B as C, and x as z."""
    lengths = [70, 61]
    T = sum(lengths)
    x, w, b, st = _conv_inputs(lengths, 64, 4)
    assert _same(fk.conv_prefill(x[:1].expand(T, 64), w, b, st[:1].expand(2, 3, 64), _cu(lengths)),
                 fk.conv_prefill(x[:1].repeat(T, 1), w, b, st[:1].repeat(2, 1, 1), _cu(lengths)))
    i = _scan_inputs(lengths, 4, 2, 64)
    j = dict(i, dt=i["dt"][:1].expand(T, 4), B=i["B"][:1].expand(T, 2, 128), state=i["state"][:1].expand(2, 4, 64, 128))
    k = {n: (t.contiguous() if t is not None else None) for n, t in j.items()}
    assert _same(_scan(j, lengths, method=method), _scan(k, lengths, method=method))
    j = dict(i, C=i["B"], z=i["x"])
    k = dict(i, C=i["B"].clone(), z=i["x"].clone())
    assert _same(_scan(j, lengths, method=method), _scan(k, lengths, method=method))
    out, new = _scan(j, lengths, method=method)
    _check_scan(out, new, _ref(j, lengths), method)


@pytest.mark.gpu
@pytest.mark.parametrize("H,G,P", [(128, 1, 64), (129, 1, 64), (130, 130, 64), (64, 1, 128)])
def test_wide_layers(H, G, P):
    """128 heads and more in one group, and a group for every head."""
    lengths = [66, 5]
    i = _scan_inputs(lengths, H, G, P, seed=110)
    for method in METHODS:
        out, new = _scan(i, lengths, method=method)
        _check_scan(out, new, _ref(i, lengths), method)


@pytest.mark.gpu
def test_two_host_threads():
    """Calls from two threads on streams of their own give the bits of calls from one."""
    import threading
    lengths = [[70, 200], [4133]]
    ins = [_scan_inputs(n, 2, 1, 128, seed=120 + k) for k, n in enumerate(lengths)]
    call = lambda k: fk.ssm_prefill(*(ins[k][n] for n in ("x", "dt", "A_log", "B", "C", "D", "dt_bias", "state")),
                                    _cu(lengths[k]), z=ins[k]["z"])
    want = [call(0), call(1)]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[k].append(call(k))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                                    # (reported by the assertion below)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and all(_same(r, want[k]) for k in (0, 1) for r in got[k])
    fk.device_status()
