"""Destinations of the state space calls overlap nothing that a call reads, nor each other: every
pair is refused on the host, before any launch, and an arena whose tensors touch is served."""
import ctypes

import pytest
import torch

import fastaf_kernel_b200 as fk
from fastaf_kernel_b200 import _lib
from test_state_space import DEV, _conv_inputs, _cu, _scan_inputs

BAD = _lib.GDN_ERR_INVALID_ARGUMENT
MB = 1 << 20

# (These pass addresses of nothing; where they were not refused, a GPU would be asked to use them.)
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: only where nothing can be launched")

N, T, C, W = 3, 200, 64, 4
H, G, P = 4, 2, 64


def _conv(decode, **at):
    """A call of the convolution on made-up addresses, 1 MB apart but for those given: x in rows
    of 2 C elements, two outputs of C / 2."""
    names = ("x", "weight", "bias", "state", "cu_seqlens", "out0", "out1", "new_state")
    a = {k: (k_ + 1) * MB for k_, k in enumerate(names)} | at
    outs, widths = (ctypes.c_void_p * 2)(a["out0"], a["out1"]), (ctypes.c_int64 * 2)(C // 2, C // 2)
    lib = _lib.load()
    if decode:
        return lib.gdn_conv_decode(a["x"], 2 * C, a["weight"], a["bias"], 0, a["state"], T, C, W, 1, outs, widths, 2,
                                   a["new_state"], None)
    return lib.gdn_conv_prefill(a["x"], 2 * C, a["weight"], a["bias"], 0, a["state"], a["cu_seqlens"], N, T, C, W, 1, outs,
                                widths, 2, a["new_state"], None)


def _conv_bytes(decode):
    rows = ((T - 1) * 2 * C + C) * 2
    state = (T if decode else N) * (W - 1) * C * 2
    return dict(x=rows, weight=C * W * 4, bias=C * 4, state=state, cu_seqlens=(N + 1) * 4, out0=T * C, out1=T * C,
                new_state=state)


def _scan(decode, dt_dtype=0, **at):
    names = ("x", "dt", "A_log", "B", "C", "D", "dt_bias", "z", "state", "cu_seqlens", "output", "new_state")
    a = {k: (k_ + 1) * (64 * MB) for k_, k in enumerate(names)} | at
    head = (a["x"], 0, a["dt"], 0, a["A_log"], a["B"], 2 * G * 128, a["C"], 2 * G * 128, a["D"], a["dt_bias"], a["z"], 0,
            a["state"])
    tail = (H, G, P, 128, dt_dtype, 0, a["output"], a["new_state"])
    lib = _lib.load()
    if decode:
        return lib.gdn_ssm_decode(*head, T, *tail, None)
    return lib.gdn_ssm_prefill(*head, a["cu_seqlens"], N, T, *tail, 0, None)


def _scan_bytes(decode):
    wide, bc = T * H * P * 2, ((T - 1) * 2 * G * 128 + G * 128) * 2
    state = (T if decode else N) * H * P * 128 * 4
    return dict(x=wide, dt=T * H * 4, A_log=H * 4, B=bc, C=bc, D=H * 4, dt_bias=H * 4, z=wide, state=state,
                cu_seqlens=(N + 1) * 4, output=wide, new_state=state)


def _pairs(call, sizes, outputs, decode):
    for out in outputs:
        for other in sizes:
            if other == out or (decode and other == "cu_seqlens"):
                continue
            if other == "state" and out == "new_state":
                continue                                       # (has rules and tests of its own)
            yield call, out, other, decode


CONV_OUT, SCAN_OUT = ("out0", "out1", "new_state"), ("output", "new_state")
PAIRS = [p for d in (False, True) for p in (*_pairs("conv", _conv_bytes(d), CONV_OUT, d),
                                            *_pairs("scan", _scan_bytes(d), SCAN_OUT, d))]


@no_gpu
@pytest.mark.parametrize("call,out,other,decode", PAIRS, ids=lambda v: str(v))
def test_every_pair_is_refused(call, out, other, decode):
    """The destination at the other tensor, inside it, at its last bytes, and ending in its first."""
    fn, sizes = (_conv, _conv_bytes(decode)) if call == "conv" else (_scan, _scan_bytes(decode))
    lib, base = _lib.load(), 4096 * MB
    n, m = sizes[out], sizes[other]
    up = lambda v: v // 16 * 16
    for at in (base, base - up(n - 1), base + up(m - 1)):
        assert fn(decode, **{other: base, out: at}) == BAD
        assert b"overlap" in lib.gdn_last_error()
    if n > m:
        assert fn(decode, **{other: base + 64, out: base}) == BAD     # all of it inside the destination


@no_gpu
def test_dt_is_measured_in_its_own_type():
    """fp32 dt reaches twice as far as bf16."""
    at = dict(dt=4096 * MB, output=4096 * MB + T * H * 2)
    assert _scan(True, 0, **at) == BAD
    assert _scan(True, 1, **at) != BAD                                # (no device to launch on)


@no_gpu
def test_a_destination_between_rows_is_none_of_them():
    """One sequence's packed output in the columns beside a row of x, with another row behind it."""
    lib = _lib.load()
    call = lambda x, out, rows=1: lib.gdn_conv_decode(
        x, 4 * C, MB, None, 0, None, rows, C, W, 1, (ctypes.c_void_p * 1)(out), (ctypes.c_int64 * 1)(C), 1, 8 * MB, None)
    assert call(4 * MB, 4 * MB + C * 2) != BAD
    assert call(4 * MB, 4 * MB + C * 2 - 16) == BAD
    assert call(4 * MB, 4 * MB + C * 2, 2) != BAD                     # two packed rows still end before the next of x
    assert call(4 * MB, 4 * MB + C * 2, 4) == BAD


def _arena(pieces):
    """Views of one allocation for (shape, dtype) pieces, each right behind the one before, up to
    the 16 bytes that all of them start on."""
    sizes = [-(-torch.empty(0, dtype=d).element_size() * torch.Size(s).numel() // 16) * 16 for s, d in pieces]
    buf = torch.zeros(sum(sizes), dtype=torch.uint8, device=DEV)
    views, at = [], 0
    for (s, d), n in zip(pieces, sizes):
        k = torch.empty(0, dtype=d).element_size() * torch.Size(s).numel()
        views.append(buf[at:at + k].view(d).view(s))
        at += n
    return views


@pytest.mark.gpu
def test_tensors_that_touch_are_served():
    bf16, f32, lengths = torch.bfloat16, torch.float32, [70, 33, 26]
    x, w, b, st = _conv_inputs(lengths, C, W)
    T_ = sum(lengths)
    want = fk.conv_prefill(x, w, b, st, _cu(lengths))
    y, xa, new, sta, wa = _arena([((T_, C), bf16), ((T_, C), bf16), ((3, W - 1, C), bf16), ((3, W - 1, C), bf16), ((C, W), f32)])
    xa.copy_(x), sta.copy_(st), wa.copy_(w)
    fk.conv_prefill(xa, wa, b, sta, _cu(lengths), output=y, new_state=new)
    assert torch.equal(y, want[0]) and torch.equal(new, want[1])
    i = _scan_inputs(lengths, H, G, P)
    call = lambda x, dt, state, **kw: fk.ssm_prefill(x, dt, i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], state,
                                                     _cu(lengths), z=i["z"], **kw)
    want = call(i["x"], i["dt"], i["state"])
    dt, y, xa, new, sta = _arena([((T_, H), bf16), ((T_, H, P), bf16), ((T_, H, P), bf16), ((3, H, P, 128), f32),
                                  ((3, H, P, 128), f32)])
    xa.copy_(i["x"]), dt.copy_(i["dt"]), sta.copy_(i["state"])
    call(xa, dt, sta, output=y, new_state=new)
    fk.device_status()
    assert torch.equal(y, want[0]) and torch.equal(new, want[1])


@pytest.mark.gpu
def test_python_names_what_overlaps():
    lengths = [70, 33]
    i = _scan_inputs(lengths, 4, 2, 64, state=False, dt_dtype=torch.float32)
    one = torch.zeros(103 * 4 * 64 * 4, dtype=torch.uint8, device=DEV)
    dt, out = one[:103 * 4 * 4].view(torch.float32).view(103, 4), one[:103 * 4 * 64 * 2].view(torch.bfloat16).view(103, 4, 64)
    with pytest.raises(ValueError, match="output must not overlap dt"):
        fk.ssm_prefill(i["x"], dt, i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], None, _cu(lengths), output=out)
    x, w, b, _ = _conv_inputs(lengths, 64, 4)
    with pytest.raises(ValueError, match="new_state must not overlap x"):
        fk.conv_prefill(x, w, b, None, _cu(lengths), new_state=x.view(-1)[:2 * 3 * 64].view(2, 3, 64))
