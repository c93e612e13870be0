"""The short causal convolution and the selective scan: refusals on the host, and parity of
every kernel with a plain 64-bit implementation.

Tolerances count roundings.  A bf16 result may be half a step (2^-8 relative) off.  The
CUDA-core kernels compute in fp32 otherwise: a sum of n terms is off by at most n 2^-24 of
the sum of the terms' magnitudes, which the reference computes beside the sum; 2^-16 of it
covers every length here together with the exponentials (a few 2^-22).  The tensor-core scan
also rounds one operand of each product of y to bf16 (the state, or the masked scores),
another 2^-8 of the magnitudes, and splits the state update's scaled operand into two bf16
numbers, off by 2^-16 relative, so its state is held to 2^-15 of the magnitudes.
"""
import math

import pytest
import torch

import fastaf_kernel_b200 as fk
from fastaf_kernel_b200 import _lib
from fastaf_kernel_b200 import workloads as W

DEV = torch.device("cuda", 0)
HALF = torch.finfo(torch.bfloat16).eps / 2      # 2^-8
F64 = torch.float64
TINY = 1e-30
METHODS = ["recurrent", "tcgen05"]


# --------------------------------------------------------------------------- references

def _conv_ref(x, weight, bias, state, lengths, act):
    """y, the sum of its terms' magnitudes, and the new state, in 64 bits on the CPU."""
    x, w = x.cpu().to(F64), weight.cpu().to(F64)
    C, K = w.shape
    ys, mags, news, at = [], [], [], 0
    for n, L in enumerate(lengths):
        front = state[n].cpu().to(F64) if state is not None else torch.zeros((K - 1, C), dtype=F64)
        rows = torch.cat([front, x[at:at + L]])
        y, mag = torch.zeros((L, C), dtype=F64), torch.zeros((L, C), dtype=F64)
        for k in range(K):
            y += rows[k:k + L] * w[:, k]
            mag += (rows[k:k + L] * w[:, k]).abs()
        if bias is not None:
            y, mag = y + bias.cpu().to(F64), mag + bias.cpu().to(F64).abs()
        ys.append(y * torch.sigmoid(y) if act else y)
        mags.append(mag)
        news.append(rows[L:])
        at += L
    return torch.cat(ys), torch.cat(mags), torch.stack(news)


def _scan_ref(x, dt, A_log, B, C, D, dt_bias, state, lengths, z):
    """y, its magnitudes, the new state and its magnitudes, in 64 bits on the CPU."""
    c = lambda t: None if t is None else t.cpu().to(F64)
    x, dt, A_log, B, C, D, dt_bias, state, z = (c(t) for t in (x, dt, A_log, B, C, D, dt_bias, state, z))
    T, H, P = x.shape
    R = H // B.shape[1]
    N = len(lengths)
    step = dt + (dt_bias if dt_bias is not None else 0)
    step = torch.where(step > 20, step, torch.log1p(torch.exp(step.clamp(max=20))))
    y, ymag = torch.zeros((T, H, P), dtype=F64), torch.zeros((T, H, P), dtype=F64)
    new = state.clone() if state is not None else torch.zeros((N, H, P, 128), dtype=F64)
    nmag = new.abs()
    at = 0
    for n, L in enumerate(lengths):
        for t in range(at, at + L):
            decay = torch.exp(-torch.exp(A_log) * step[t])[:, None, None]
            add = (step[t][:, None] * x[t])[:, :, None] * B[t].repeat_interleave(R, 0)[:, None, :]
            new[n] = new[n] * decay + add
            nmag[n] = nmag[n] * decay + add.abs()
            Ct = C[t].repeat_interleave(R, 0)[:, None, :]
            y[t] = (new[n] * Ct).sum(-1)
            ymag[t] = (nmag[n] * Ct.abs()).sum(-1)
            if D is not None:
                y[t] += D[:, None] * x[t]
                ymag[t] += (D[:, None] * x[t]).abs()
        at += L
    if z is not None:
        gate = z * torch.sigmoid(z)
        y, ymag = y * gate, ymag * gate.abs()
    return y, ymag, new, nmag


def _check(name, got, ref, tol):
    got = got.detach().cpu().to(F64)
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    over = (got - ref).abs() - tol
    assert bool((over <= 0).all()), f"{name}: {int((over > 0).sum())} of {over.numel()} off, by up to {float(over.max()):.3e}"


def _check_scan(out, new, ref, method):
    y, ymag, s, smag = ref
    rounded = HALF if method == "tcgen05" else 0.0
    _check("y", out.reshape(y.shape), y, HALF * y.abs() + (rounded * (1 + HALF) + 2.0 ** -16) * ymag + TINY)
    _check("state", new, s, (2.0 ** -15 if method == "tcgen05" else 2.0 ** -18) * smag + TINY)


# ------------------------------------------------------------------------------- inputs

def _wide_rows(total, widths, wide, g, dev):
    """bf16 rows of the widths: packed, or slices of one wider row with 24 more columns."""
    if wide:
        return list(torch.randn((total, sum(widths) + 24), generator=g, device=dev).to(torch.bfloat16)
                    [:, :sum(widths)].split(widths, 1))
    return [torch.randn((total, w), generator=g, device=dev).to(torch.bfloat16) for w in widths]


def _cu(lengths, dev=DEV):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device=dev)


def _conv_inputs(lengths, C, K, bias=True, state=True, wide=False, dtype=torch.float32, seed=1, dev=DEV):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = _wide_rows(sum(lengths), [C], wide, g, dev)[0]
    weight = torch.randn((C, K), generator=g, device=dev).to(dtype)
    b = torch.randn(C, generator=g, device=dev).to(dtype) if bias else None
    st = torch.randn((len(lengths), K - 1, C), generator=g, device=dev).to(torch.bfloat16) if state else None
    return x, weight, b, st


def _scan_inputs(lengths, H, G, P, wide=False, state=True, z=True, dt_dtype=torch.bfloat16, params=torch.float32,
                 seed=1, dev=DEV, strong=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    T = sum(lengths)
    x, B, C, zz = _wide_rows(T, [H * P, G * 128, G * 128, H * P], wide, g, dev)
    dt = torch.randn((T, H + (8 if wide else 0)), generator=g, device=dev).to(dt_dtype)[:, :H]
    A_log = torch.log(torch.rand(H, generator=g, device=dev) * 15 + 1).to(params)
    dt_bias = (torch.rand(H, generator=g, device=dev) * 4 - (1 if strong else 5)).to(params)
    D = torch.randn(H, generator=g, device=dev).to(params)
    st = torch.randn((len(lengths), H, P, 128), generator=g, device=dev) if state else None
    return dict(x=x.view(T, H, P), dt=dt, A_log=A_log, B=B.view(T, G, 128), C=C.view(T, G, 128), D=D, dt_bias=dt_bias,
                state=st, z=zz.view(T, H, P) if z else None)


def _scan(i, lengths, **kw):
    out = fk.ssm_prefill(i["x"], i["dt"], i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], i["state"], _cu(lengths),
                         z=i["z"], **kw)
    fk.device_status()
    return out


def _step(i, **kw):
    u = lambda t: None if t is None else t.unsqueeze(1)
    return fk.ssm_decode(u(i["x"]), u(i["dt"]), i["A_log"], u(i["B"]), u(i["C"]), i["D"], i["dt_bias"],
                         kw.pop("state", i["state"]), z=u(i["z"]), **kw)


def _ref(i, lengths):
    return _scan_ref(i["x"], i["dt"], i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], i["state"], lengths, i["z"])


def _part(i, sl, state):
    rows = {k: (None if i[k] is None else i[k][sl]) for k in ("x", "dt", "B", "C", "z")}
    return dict(i, **rows, state=state)


# -------------------------------------------------------------------- refusals, on the CPU

def _conv_c(lib, decode=False, **over):
    import ctypes
    a = dict(x=16, xs=0, weight=16, bias=None, wd=0, state=16, cu=16, N=1, T=4, C=64, W=4, act=1, outs=(16,), widths=(64,),
             new=1 << 20)
    a.update(over)
    n = len(a["outs"])
    outs, widths = (ctypes.c_void_p * max(n, 1))(*a["outs"]), (ctypes.c_int64 * max(n, 1))(*a["widths"])
    if decode:
        return lib.gdn_conv_decode(a["x"], a["xs"], a["weight"], a["bias"], a["wd"], a["state"], a["N"], a["C"], a["W"],
                                   a["act"], outs, widths, n, a["new"], None)
    return lib.gdn_conv_prefill(a["x"], a["xs"], a["weight"], a["bias"], a["wd"], a["state"], a["cu"], a["N"], a["T"],
                                a["C"], a["W"], a["act"], outs, widths, n, a["new"], None)


BAD, UNSUPPORTED = _lib.GDN_ERR_INVALID_ARGUMENT, _lib.GDN_ERR_UNSUPPORTED


@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("over,code", [
    (dict(W=1), UNSUPPORTED), (dict(W=5), UNSUPPORTED), (dict(C=60, widths=(60,)), BAD), (dict(C=0), BAD),
    (dict(wd=3), BAD), (dict(act=2), BAD), (dict(N=-1), BAD), (dict(xs=56), BAD), (dict(xs=68), BAD),
    (dict(outs=(), widths=()), BAD), (dict(outs=(16,) * 5, widths=(8,) * 5), BAD),
    (dict(outs=(16, 16), widths=(32, 24)), BAD), (dict(outs=(16, 16), widths=(36, 28)), BAD),
    (dict(x=None), BAD), (dict(x=8), BAD), (dict(weight=None), BAD), (dict(new=None), BAD), (dict(outs=(8,)), BAD),
    (dict(state=24), BAD), (dict(state=(1 << 20) + 16), BAD),           # misaligned, partial overlap
])
def test_conv_rejects_bad_arguments(decode, over, code):
    lib = _lib.load()
    assert _conv_c(lib, decode, **over) == code
    assert lib.gdn_last_error().decode()


def test_conv_prefill_rejects_an_in_place_state_and_no_cu_seqlens():
    lib = _lib.load()
    assert _conv_c(lib, state=1 << 20) == BAD
    assert _conv_c(lib, cu=None) == BAD
    assert _conv_c(lib, T=1 << 31) == BAD


def _ssm_c(lib, decode=False, **over):
    a = dict(x=16, xs=0, dt=16, ds=0, A=16, B=16, Bs=0, C=16, Cs=0, D=None, bias=None, z=None, zs=0, state=16, cu=16,
             N=1, T=64, H=4, G=2, P=64, S=128, dd=1, pd=0, out=16, new=1 << 24, method=0)
    a.update(over)
    head = [a[k] for k in ("x", "xs", "dt", "ds", "A", "B", "Bs", "C", "Cs", "D", "bias", "z", "zs", "state")]
    tail = [a[k] for k in ("H", "G", "P", "S", "dd", "pd", "out", "new")]
    if decode:
        return lib.gdn_ssm_decode(*head, a["N"], *tail, None)
    return lib.gdn_ssm_prefill(*head, a["cu"], a["N"], a["T"], *tail, a["method"], None)


@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("over,code", [
    (dict(P=32), UNSUPPORTED), (dict(P=96), UNSUPPORTED), (dict(S=64), UNSUPPORTED), (dict(H=3), BAD), (dict(G=0), BAD),
    (dict(H=0), BAD), (dict(dd=2), BAD), (dict(pd=-1), BAD), (dict(N=-1), BAD), (dict(xs=255), BAD), (dict(xs=260), BAD),
    (dict(zs=128), BAD), (dict(Bs=128), BAD), (dict(Cs=257), BAD), (dict(ds=3), BAD), (dict(ds=1 << 31), BAD),
    (dict(x=None), BAD), (dict(dt=None), BAD), (dict(A=None), BAD), (dict(out=None), BAD), (dict(new=None), BAD),
    (dict(x=8), BAD), (dict(B=2), BAD), (dict(z=8), BAD), (dict(out=24), BAD), (dict(state=(1 << 24) + 16), BAD),
])
def test_scan_rejects_bad_arguments(decode, over, code):
    lib = _lib.load()
    assert _ssm_c(lib, decode, **over) == code
    assert lib.gdn_last_error().decode()


def test_scan_prefill_rejects_methods_states_and_sizes():
    lib = _lib.load()
    assert _ssm_c(lib, method=1) == BAD and _ssm_c(lib, method=7) == BAD
    assert _ssm_c(lib, state=1 << 24) == BAD
    assert _ssm_c(lib, cu=None) == BAD
    assert _ssm_c(lib, T=1 << 31) == BAD


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    assert _conv_c(lib, N=0, T=0) == _lib.GDN_OK and _conv_c(lib, True, N=0) == _lib.GDN_OK
    assert _ssm_c(lib, N=0, T=0) == _lib.GDN_OK and _ssm_c(lib, True, N=0) == _lib.GDN_OK


def test_there_is_no_cpu_path():
    cpu = torch.device("cpu")
    x, w, b, st = _conv_inputs([4, 2], 16, 4, dev=cpu)
    with pytest.raises(ValueError, match="CUDA"):
        fk.conv_prefill(x, w, b, st, _cu([4, 2], cpu))
    with pytest.raises(ValueError, match="CUDA"):
        fk.conv_decode(x[:2], w, b, st)
    i = _scan_inputs([4, 2], 4, 2, 64, dev=cpu)
    with pytest.raises(ValueError, match="CUDA"):
        fk.ssm_prefill(i["x"], i["dt"], i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], i["state"], _cu([4, 2], cpu))
    with pytest.raises(ValueError):
        fk.ssm_method(4, "chunked")


# ------------------------------------------------------------------------ the convolution

@pytest.mark.gpu
@pytest.mark.parametrize("lengths,C,K,bias,state,wide,act,dtype", [
    ([1], 8, 4, False, False, False, "silu", torch.float32),
    ([5, 0, 1, 2, 3, 40, 0], 40, 4, True, True, True, "silu", torch.float32),
    ([0, 0, 3], 16, 3, True, False, False, None, torch.bfloat16),
    ([700, 1, 33], 1032, 2, True, True, True, "silu", torch.bfloat16),
    ([64, 129], 8192, 4, False, True, False, "silu", torch.float32),
    ([2500], 256, 4, True, True, False, None, torch.float32),
])
def test_conv_prefill_matches_64_bits(lengths, C, K, bias, state, wide, act, dtype):
    x, w, b, st = _conv_inputs(lengths, C, K, bias, state, wide, dtype)
    y, new = fk.conv_prefill(x, w, b, st, _cu(lengths), activation=act)
    fk.device_status()
    ry, mag, rs = _conv_ref(x, w, b, st, lengths, act)
    _check("y", y, ry, HALF * ry.abs() + 2.0 ** -16 * mag + TINY)
    _check("state", new, rs, 0.0)


@pytest.mark.gpu
def test_conv_split_writes_packed_parts():
    lengths = [30, 7]
    x, w, b, st = _conv_inputs(lengths, 96, 4)
    y, new = fk.conv_prefill(x, w, b, st, _cu(lengths))
    parts, new2 = fk.conv_prefill(x, w, b, st, _cu(lengths), split=(8, 64, 24))
    assert [tuple(p.shape) for p in parts] == [(37, 8), (37, 64), (37, 24)] and all(p.is_contiguous() for p in parts)
    assert torch.equal(torch.cat(parts, 1), y) and torch.equal(new, new2)
    d, _ = fk.conv_decode(x[:2], w, b, st)
    parts, _ = fk.conv_decode(x[:2], w, b, st, split=(8, 64, 24))
    assert torch.equal(torch.cat(parts, 1), d)


@pytest.mark.gpu
@pytest.mark.parametrize("B,C,K,state", [(1, 8, 2, True), (3, 1032, 3, False), (77, 40, 4, True), (300, 2048, 4, True)])
def test_conv_decode_continues_prefill(B, C, K, state):
    """Prefill of L tokens equals prefill of all but the last and one decode step, bit for bit."""
    lengths = [1 + (5 * i) % 7 for i in range(B)]
    x, w, b, st = _conv_inputs(lengths, C, K, state=state)
    cu = _cu(lengths)
    y, new = fk.conv_prefill(x, w, b, st, cu)
    last = (cu[1:] - 1).long()
    keep = torch.ones(x.shape[0], dtype=torch.bool, device=DEV)
    keep[last] = False
    _, mid = fk.conv_prefill(x[keep], w, b, st, _cu([n - 1 for n in lengths]))
    yd, nd = fk.conv_decode(x[last], w, b, mid)
    assert torch.equal(yd, y[last]) and torch.equal(nd, new)
    y2, n2 = fk.conv_decode(x[last], w, b, mid, new_state=mid)
    fk.device_status()
    assert n2 is mid and torch.equal(y2, yd) and torch.equal(mid, nd)
    ry, mag, rs = _conv_ref(x, w, b, st, lengths, "silu")
    _check("y", yd, ry[last.cpu()], HALF * ry[last.cpu()].abs() + 2.0 ** -16 * mag[last.cpu()] + TINY)


@pytest.mark.gpu
def test_conv_sequences_do_not_mix():
    """NaN and infinities of one sequence and its state stay in it."""
    lengths = [9, 20, 6]
    x, w, b, st = _conv_inputs(lengths, 64, 4)
    y, new = fk.conv_prefill(x, w, b, st, _cu(lengths))
    x2, st2 = x.clone(), st.clone()
    x2[9:29:2] = float("nan")
    x2[10:29:2] = float("inf")
    st2[1] = float("nan")
    y2, new2 = fk.conv_prefill(x2, w, b, st2, _cu(lengths))
    for s in (slice(0, 9), slice(29, 35)):
        assert torch.equal(y2[s], y[s])
    assert torch.equal(new2[0], new[0]) and torch.equal(new2[2], new[2])


# ------------------------------------------------------------------------------- the scan

CASES = [
    # lengths, heads, groups, head size, wide rows, state, z
    ([1], 1, 1, 64, False, False, False),
    ([64], 1, 1, 128, False, True, False),
    ([100], 2, 1, 64, False, True, True),
    ([64, 64], 3, 1, 64, False, False, True),                 # an odd number of heads in a group
    ([130, 1, 0, 63, 65], 4, 2, 128, True, True, True),
    ([200, 0, 7, 128], 6, 2, 64, True, True, False),
    ([0, 3, 70, 0], 4, 4, 64, False, True, True),             # one head a group
    ([517], 2, 2, 128, True, False, False),
    ([4000, 0, 65, 1500], 2, 1, 128, False, True, True),       # cut into segments, sequences of mean length
    ([1300, 1640, 2000], 3, 1, 64, True, True, False),
    ([1, 4900, 333], 1, 1, 64, False, False, True),
]


def _ids(c):
    return "-".join(map(str, c[0])) + f"-H{c[1]}G{c[2]}P{c[3]}"


@pytest.mark.gpu
@pytest.mark.parametrize("method", METHODS + ["auto"])
@pytest.mark.parametrize("case", CASES, ids=_ids)
def test_scan_matches_64_bits(method, case):
    lengths, H, G, P, wide, state, z = case
    if method == "tcgen05" and sum(lengths) < 64:
        pytest.skip("the tensor-core scan takes 64 tokens and more")
    i = _scan_inputs(lengths, H, G, P, wide, state, z)
    out, new = _scan(i, lengths, method=method)
    ran = fk.ssm_method(sum(lengths), method, len(lengths))
    _check_scan(out, new, _ref(i, lengths), ran)


@pytest.mark.gpu
@pytest.mark.parametrize("method", METHODS)
@pytest.mark.parametrize("over", [
    dict(dt_dtype=torch.float32), dict(params=torch.bfloat16), dict(strong=True), dict(strong=True, state=False, z=False),
])
def test_scan_types_and_strong_decays(method, over):
    lengths = [90, 64, 33]
    i = _scan_inputs(lengths, 4, 2, 64, seed=5, **over)
    out, new = _scan(i, lengths, method=method)
    _check_scan(out, new, _ref(i, lengths), method)


@pytest.mark.gpu
@pytest.mark.parametrize("method", METHODS)
def test_scan_without_skip_and_bias(method):
    lengths = [70, 31]
    i = dict(_scan_inputs(lengths, 4, 1, 128, seed=6, z=False), D=None, dt_bias=None)
    out, new = _scan(i, lengths, method=method)
    _check_scan(out, new, _ref(i, lengths), method)


@pytest.mark.gpu
@pytest.mark.parametrize("method", METHODS)
def test_scan_sequences_do_not_mix(method):
    """NaN and infinities of one sequence and its state stay in it, also where it shares a
    64-row tile with its neighbours; outputs behind the last token are not written."""
    lengths = [70, 40, 90]
    i = _scan_inputs(lengths, 4, 2, 64, seed=7)
    out, new = _scan(i, lengths, method=method)
    j = {k: (None if v is None else v.clone()) for k, v in i.items()}
    for k in ("x", "B", "C", "z", "dt"):
        j[k][70:110:2] = float("nan")
        j[k][71:110:2] = float("inf")
    j["state"][1] = float("nan")
    buf = torch.full((205, 4, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    out2, new2 = _scan(j, lengths, method=method, output=buf[:200])
    for s in (slice(0, 70), slice(110, 200)):
        assert torch.equal(out2[s], out[s])
    assert torch.equal(new2[0], new[0]) and torch.equal(new2[2], new[2])
    assert bool((buf[200:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("method", METHODS)
def test_scan_empty_sequences_keep_their_state(method):
    lengths = [0, 80, 0]
    i = _scan_inputs(lengths, 2, 1, 128, seed=8)
    _, new = _scan(i, lengths, method=method)
    assert torch.equal(new[0], i["state"][0]) and torch.equal(new[2], i["state"][2])
    _, new = _scan(dict(i, state=None), lengths, method=method)
    assert not new[0].any() and not new[2].any()


@pytest.mark.gpu
def test_scan_without_tokens():
    i = _scan_inputs([0, 0], 2, 1, 64, seed=9)
    out, new = _scan(i, [0, 0])
    assert out.shape == (0, 2, 64) and torch.equal(new, i["state"])


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,G,P,wide,state,z", [
    (1, 1, 1, 64, False, True, False), (3, 6, 2, 64, True, False, True), (5, 4, 4, 128, True, True, True),
    (130, 32, 16, 128, False, True, False),
])
def test_scan_decode_matches_64_bits(B, H, G, P, wide, state, z):
    i = _scan_inputs([1] * B, H, G, P, wide, state, z, seed=10)
    out, new = _step(i)
    ref = _ref(i, [1] * B)
    _check_scan(out, new, ref, "decode")
    if state:
        st = i["state"].clone()
        out2, new2 = _step(i, state=st, new_state=st)
        assert new2 is st and torch.equal(out2, out) and torch.equal(st, new)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [[0, 90, 60, 200], [5, 90, 120, 200], [0, 90, 120, 180], [0, -4, 400, 200]])
@pytest.mark.parametrize("op", ["conv"] + METHODS)
def test_malformed_cu_seqlens_on_the_device_is_reported(op, bad):
    """The kernels clamp the offsets (every access stays in bounds) and record the error."""
    cu = torch.tensor(bad, dtype=torch.int32, device=DEV)
    if op == "conv":
        x, w, b, st = _conv_inputs([90, 30, 80], 64, 4)
        fk.conv_prefill(x, w, b, st, cu)
    else:
        i = _scan_inputs([90, 30, 80], 2, 1, 64)
        fk.ssm_prefill(i["x"], i["dt"], i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], i["state"], cu, z=i["z"],
                       method=op)
    with pytest.raises(ValueError, match="cu_seqlens"):
        fk.device_status()
    fk.device_status()


# ------------------------------------------------------------- a run of them, as it is used

@pytest.mark.gpu
@pytest.mark.parametrize("method", METHODS)
def test_layer_prompt_then_tokens(method):
    """A state space layer: convolution of the projected rows, split into x, B and C, the
    gated scan; then token by token in place.  The steps' outputs are those of the whole
    prompt at once, to the tolerance of two results with one set of roundings each."""
    H, G, P, lengths, steps = 4, 2, 64, [70, 33], 5
    g = torch.Generator(device=DEV).manual_seed(20)
    widths = (H * P, G * 128, G * 128)
    total = [n + steps for n in lengths]
    proj = torch.randn((sum(total), sum(widths)), generator=g, device=DEV).to(torch.bfloat16)
    w = torch.randn((sum(widths), 4), generator=g, device=DEV) * 0.5
    i = _scan_inputs(total, H, G, P, state=False, seed=21)

    def run(rows, cu, conv_state, state, sl):
        (x, B, C), conv_state = fk.conv_prefill(rows, w, None, conv_state, cu, split=widths)
        T = x.shape[0]
        y, state = fk.ssm_prefill(x.view(T, H, P), i["dt"][sl], i["A_log"], B.view(T, G, 128), C.view(T, G, 128), i["D"],
                                  i["dt_bias"], state, cu, z=i["z"][sl], method=method)
        return y, conv_state, state, (x, B, C)

    whole, conv_end, end, (x, B, C) = run(proj, _cu(total), None, None, slice(None))
    first = torch.cat([torch.arange(0, 70), torch.arange(75, 108)]).to(DEV)
    y, conv_state, state, _ = run(proj[first], _cu(lengths), None, None, first)
    full = dict(i, x=x.view(-1, H, P), B=B.view(-1, G, 128), C=C.view(-1, G, 128), state=None)
    ry, ymag, rs, smag = _ref(full, total)
    tol = HALF * ry.abs() + ((HALF * (1 + HALF) if method == "tcgen05" else 0) + 2.0 ** -14) * ymag + TINY
    _check("prompt", y, ry[first.cpu()], tol[first.cpu()])
    for t in range(steps):
        at = torch.tensor([70 + t, 75 + 33 + t], device=DEV)
        (xs, Bs, Cs), conv_state = fk.conv_decode(proj[at], w, None, conv_state, split=widths, new_state=conv_state)
        one = dict(i, x=xs.view(2, H, P), B=Bs.view(2, G, 128), C=Cs.view(2, G, 128), dt=i["dt"][at], z=i["z"][at])
        yt, state = _step(one, state=state, new_state=state)
        _check("token", yt.reshape(2, H, P), ry[at.cpu()], tol[at.cpu()])
    fk.device_status()
    assert torch.equal(conv_state, conv_end)
    _check("state", state, rs, 2.0 ** -14 * smag + TINY)
    _check("whole state", end, rs, 2.0 ** -14 * smag + TINY)


@pytest.mark.gpu
def test_convolution_in_front_of_the_delta_rule():
    """q, k and v straight from the convolution's packed parts, prompt then one token."""
    Hq, Hv, lengths = 4, 8, [300, 41]
    x = W.prefill_inputs(lengths, seed=3, Hq=Hq, Hv=Hv, device=DEV)
    widths = (Hq * 128, Hq * 128, Hv * 128)
    proj, w, _, st = _conv_inputs(lengths, sum(widths), 4, wide=True, seed=4)
    heads = lambda t, h: t.view(-1, h, 128)

    def run(q, k, v):
        return fk.kernel(heads(q, Hq), heads(k, Hq), heads(v, Hv), x["state"], x["A_log"], x["a"], x["dt_bias"], x["b"],
                         _cu(lengths), x["scale"], use_qk_l2norm=True)

    parts, conv_state = fk.conv_prefill(proj, w, None, st, _cu(lengths), split=widths)
    one, _ = fk.conv_prefill(proj, w, None, st, _cu(lengths))
    o, s = run(*parts)
    o2, s2 = run(*(p.contiguous() for p in one.split(widths, 1)))
    fk.device_status()
    assert torch.equal(o, o2) and torch.equal(s, s2) and bool(torch.isfinite(o.float()).all())
    (q, k, v), conv_state = fk.conv_decode(proj[:2], w, None, conv_state, split=widths, new_state=conv_state)
    o, s = fk.kernel_decode(q.view(2, 1, Hq, 128), k.view(2, 1, Hq, 128), v.view(2, 1, Hv, 128), s, x["A_log"],
                            x["a"][:2, None], x["dt_bias"], x["b"][:2, None], x["scale"], new_state=s, use_qk_l2norm=True)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(o.float()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("method", METHODS)
def test_graphs_and_streams(method):
    """The four operators captured into two graphs and replayed, and run on a side stream,
    give the eager bits; a prompt behind another one on the same stream too."""
    lengths = [70, 129, 5]
    x, w, b, st = _conv_inputs(lengths, 512, 4, seed=30)
    i = _scan_inputs(lengths, 4, 2, 64, seed=31)
    one = _part(i, slice(0, 3), i["state"])
    cu = _cu(lengths)

    def run():
        y, cs = fk.conv_prefill(x, w, b, st, cu)
        yd, csd = fk.conv_decode(x[:3], w, b, cs)
        o, s = fk.ssm_prefill(i["x"], i["dt"], i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], i["state"], cu, z=i["z"],
                              method=method)
        od, sd = _step(one, state=s)
        return y, cs, yd, csd, o, s, od, sd

    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        graphs.append((graph, outs))
    for _ in range(2):
        for graph, outs in graphs:
            for o in outs:
                o.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(outs, want))
    fk.device_status()


@pytest.mark.gpu
def test_python_refusals():
    x, w, b, st = _conv_inputs([4, 2], 16, 4)
    cu = _cu([4, 2])
    with pytest.raises(TypeError):
        fk.conv_prefill(x.float(), w, b, st, cu)
    for kw in (dict(split=(8,)), dict(split=(4, 12)), dict(split=()), dict(activation="relu"), dict(new_state=st),
               dict(output=torch.empty_like(x)[:, :8])):
        with pytest.raises(ValueError):
            fk.conv_prefill(x, w, b, st, cu, **kw)
    with pytest.raises(NotImplementedError):
        fk.conv_prefill(x, torch.cat([w, w], 1), b, st, cu)
    with pytest.raises(ValueError):
        fk.conv_prefill(x, w, b, st[:1], cu)
    with pytest.raises(ValueError):
        fk.conv_prefill(x, w, b, st, cu.cpu() + 1)
    with pytest.raises(ValueError):
        fk.conv_decode(x[:2], w, b, st.float(), new_state=st.float())
    i = _scan_inputs([4, 2], 4, 2, 64)
    args = (i["x"], i["dt"], i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], i["state"], cu)
    with pytest.raises(NotImplementedError):
        fk.ssm_prefill(*args, method="tcgen05")             # fewer than 64 tokens
    for at, bad in ((1, i["dt"][:, :2]), (2, i["A_log"][:2]), (3, i["B"][:4]), (4, i["C"][:, :1]), (7, i["state"][:1])):
        with pytest.raises(ValueError):
            fk.ssm_prefill(*args[:at], bad, *args[at + 1:])
    with pytest.raises(NotImplementedError):
        fk.ssm_prefill(i["x"][:, :, :32], *args[1:])
    with pytest.raises(ValueError):
        fk.ssm_prefill(*args, z=i["z"][:3])
    with pytest.raises(ValueError):
        fk.ssm_prefill(*args, new_state=i["state"])
    with pytest.raises(ValueError):
        fk.ssm_decode(*args[:8])


def test_required_tensors_are_named():
    x = torch.zeros(4, 16, dtype=torch.bfloat16)
    with pytest.raises((TypeError, ValueError)):
        fk.conv_prefill(None, x, None, None, x)
    with pytest.raises((TypeError, ValueError)):
        fk.ssm_decode(None, x, x, x, x, None, None, None)


@pytest.mark.parametrize("decode", [False, True])
def test_conv_outputs_overlap_nothing(decode):
    """x itself, its last bytes, or another output as an output: refused before any launch."""
    lib = _lib.load()
    base = dict(N=4, T=4, C=16, widths=(8, 8), state=None, new=1 << 20)
    for over in (dict(x=1 << 16, outs=(1 << 16, 1 << 17)), dict(x=1 << 16, outs=(1 << 17, (1 << 16) + 112)),
                 dict(x=1 << 16, outs=(1 << 17, (1 << 17) + 48)), dict(x=1 << 16, xs=64, outs=(1 << 17, (1 << 16) + 400))):
        assert _conv_c(lib, decode=decode, **base, **over) == BAD
        assert b"overlap" in lib.gdn_last_error()


def test_scan_outputs_overlap_nothing():
    lib = _lib.load()
    at = lambda x=1 << 20, B=1 << 21, C=1 << 22, z=1 << 23, out=1 << 24: lib.gdn_ssm_decode(
        x, 0, 1 << 16, 0, 1 << 17, B, 0, C, 0, None, None, z, 0, None, 3, 2, 1, 64, 128, 0, 0, out, 1 << 25, None)
    for over in (dict(out=1 << 20), dict(out=(1 << 21) + 752), dict(out=(1 << 22) - 752), dict(out=(1 << 23) + 16)):
        assert at(**over) == BAD
        assert b"overlap" in lib.gdn_last_error()


@pytest.mark.gpu
def test_python_refuses_missing_and_overlapping_tensors():
    x, w, b, st = _conv_inputs([4, 2], 16, 4)
    cu = _cu([4, 2])
    with pytest.raises(TypeError):
        fk.conv_prefill(x, None, b, st, cu)
    with pytest.raises(ValueError):
        fk.conv_prefill(x, w, b, st, cu, output=x)
    part = torch.empty((6, 8), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        fk.conv_prefill(x, w, b, st, cu, split=(8, 8), output=(part, part))
    i = _scan_inputs([4, 2], 4, 2, 64)
    for at in range(1, 5):
        args = [i["x"], i["dt"], i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], i["state"], cu]
        args[at] = None
        with pytest.raises(TypeError):
            fk.ssm_prefill(*args)
    with pytest.raises(ValueError):
        fk.ssm_prefill(i["x"], i["dt"], i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], i["state"], cu, z=i["z"],
                       output=i["z"])


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["conv"] + METHODS)
def test_rows_behind_the_last_sequence_stay(op):
    """Offsets that end in front of the last row (reported, as any that are not offsets over
    all rows): the rows behind are left as they were, the sequences' own are right."""
    lengths, T = [90, 0, 43], 200
    if op == "conv":
        x, w, b, st = _conv_inputs([90, 0, 110], 64, 4)
        out = torch.full((T, 64), 7.0, dtype=torch.bfloat16, device=DEV)
        y, new = fk.conv_prefill(x, w, b, st, _cu(lengths), output=out)
        want = fk.conv_prefill(x[:133], w, b, st, _cu(lengths))
    else:
        i = _scan_inputs([90, 0, 110], 2, 1, 64)
        out = torch.full((T, 2, 64), 7.0, dtype=torch.bfloat16, device=DEV)
        y, new = fk.ssm_prefill(i["x"], i["dt"], i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], i["state"],
                                _cu(lengths), z=i["z"], method=op, output=out)
        s = _part(i, slice(0, 133), i["state"])
        want = fk.ssm_prefill(s["x"], s["dt"], s["A_log"], s["B"], s["C"], s["D"], s["dt_bias"], s["state"],
                              _cu(lengths), z=s["z"], method=op)
    with pytest.raises(ValueError, match="cu_seqlens"):
        fk.device_status()
    assert y is out and bool((out[133:] == 7.0).all())
    assert torch.equal(out[:133], want[0]) and torch.equal(new, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [2, 3, 4])
def test_views_off_their_alignment(dtype, K):
    """Weights that start off a 16-byte boundary, and rows that the kernels cannot read in
    place: the bits of packed, aligned copies."""
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)
    lengths = [30, 7, 60]
    x, w, b, st = _conv_inputs(lengths, 72, K, dtype=dtype)
    want = fk.conv_prefill(x, w, b, st, _cu(lengths))
    for args in ((x, off(w), off(b), st), (off(x), w, b, off(st)), (x.t().contiguous().t(), w.t().contiguous().t(), b, st),
                 (torch.cat([x, x[:, :1]], 1)[:, :72], w, off(b), st)):
        got = fk.conv_prefill(*args, _cu(lengths))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        got = fk.conv_decode(args[0][:3], *args[1:])
        one = fk.conv_decode(x[:3], w, b, st)
        assert torch.equal(got[0], one[0]) and torch.equal(got[1], one[1])
    i = _scan_inputs(lengths, 2, 1, 64, dt_dtype=dtype, params=dtype, seed=2)
    for method in METHODS:
        want = _scan(i, lengths, method=method)
        for other in ({k: (off(v) if v is not None else None) for k, v in i.items()},
                      dict(i, x=i["x"].transpose(0, 1).contiguous().transpose(0, 1), z=i["z"].transpose(1, 2).contiguous().transpose(1, 2),
                           dt=i["dt"].t().contiguous().t(), state=i["state"].transpose(2, 3).contiguous().transpose(2, 3))):
            got = _scan(other, lengths, method=method)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["conv"] + METHODS)
def test_hundreds_of_short_sequences(op):
    lengths = [(7 * n) % 6 for n in range(600)]
    if op == "conv":
        x, w, b, st = _conv_inputs(lengths, 40, 4)
        y, new = fk.conv_prefill(x, w, b, st, _cu(lengths))
        ry, mag, rs = _conv_ref(x, w, b, st, lengths, "silu")
        _check("y", y, ry, HALF * ry.abs() + 2.0 ** -16 * mag + TINY)
        assert torch.equal(new.cpu().to(F64), rs)
    else:
        i = _scan_inputs(lengths, 2, 1, 64)
        out, new = _scan(i, lengths, method=op)
        _check_scan(out, new, _ref(i, lengths), op)


@pytest.mark.gpu
@pytest.mark.parametrize("method", METHODS)
def test_steps_of_nothing_and_of_a_great_deal(method):
    """A dt of -inf leaves the state alone, a very large one forgets it; NaN parameters of a
    head stay in that head and do not vanish.  The log2 decays of a chunk sum to less than
    1024 here (160 a step at most), so each of up to 8 fp32 additions behind an exponent is
    off by 2^-15 at most, and the exponential by 8 ln 2 2^-15 < 2^-12 relative."""
    lengths = [150]
    i = _scan_inputs(lengths, 4, 1, 64, dt_dtype=torch.float32)
    i["dt"][5:9] = float("-inf")
    i["dt"][40, 1] = 1000.0
    i["dt"][70:75, 2] = 300.0
    out, new = _scan(i, lengths, method=method)
    y, ymag, st, smag = _ref(i, lengths)
    rounded = HALF if method == "tcgen05" else 0.0
    _check("y", out, y, HALF * y.abs() + (rounded * (1 + HALF) + 2.0 ** -16 + 2.0 ** -12) * ymag + TINY)
    _check("state", new, st, (2.0 ** -15 + 2.0 ** -12) * smag + TINY)
    for name in ("A_log", "dt_bias"):
        j = dict(i)
        j[name] = i[name].clone()
        j[name][1] = float("nan")
        o2, n2 = _scan(j, lengths, method=method)
        keep = [0, 2, 3]
        assert torch.equal(o2[:, keep], out[:, keep]) and torch.equal(n2[:, keep], new[:, keep])
        assert bool(torch.isnan(n2[:, 1]).all()) and bool(torch.isnan(o2[:, 1].float()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("P", [64, 128])
def test_cut_prompts_in_graphs_and_on_two_streams(P):
    """A prompt that is cut into segments takes a workspace from the pool: two captured calls
    replayed at once, and two eager ones on two streams, give the bits of single calls."""
    lengths = [4133]
    a, b = (_scan_inputs(lengths, 2, 1, P, seed=s) for s in (41, 42))
    call = lambda i: fk.ssm_prefill(i["x"], i["dt"], i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], i["state"], cu,
                                    z=i["z"], method="tcgen05")
    cu = _cu(lengths)
    want = [call(a), call(b)]
    _check_scan(*want[0], _ref(a, lengths), "tcgen05")
    graphs = []
    for i in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = call(i)
        graphs.append((graph, outs))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for graph, outs in graphs:
            for o in outs:
                o.zero_()
        torch.cuda.synchronize()
        for s, (graph, _outs) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_g, outs), w in zip(graphs, want):
            assert torch.equal(outs[0], w[0]) and torch.equal(outs[1], w[1])
        got = []
        for s, i in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(call(i))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
    fk.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,H,P,z", [([700, 300, 513], 32, 128, True), ([700, 300, 513], 5, 64, False),
                                           ([4000], 2, 128, True)])
def test_scan_waits_run_out_then_next_call_is_correct(lengths, H, P, z):
    """With a 1 ns limit the scan's waits run out: the call returns and the status says so; the
    next call, which allocates the same tensor memory, gives the usual bits."""
    lib = _lib.load()
    i = _scan_inputs(lengths, H, 1, P, z=z, seed=43)
    want = _scan(i, lengths, method="tcgen05")
    prev = lib.gdn_set_wait_limit_ns(1)
    try:
        with pytest.raises(_lib.GdnError) as ei:
            _scan(i, lengths, method="tcgen05")
        assert ei.value.status == _lib.GDN_ERR_DEVICE_TIMEOUT
    finally:
        lib.gdn_set_wait_limit_ns(prev)
    fk.device_status()
    got = _scan(i, lengths, method="tcgen05")
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows so far apart, and a state so large, that element offsets pass 2^31."""
    T, H, G, P, C = 2304, 2, 1, 64, 512
    wide = torch.randn((T, 1 << 10), device=DEV).to(torch.bfloat16).repeat(1, 1 << 10)      # 4.8 GB
    cols = lambda at, n: wide[:, at:at + n]
    i = _scan_inputs([T], H, G, P, seed=50)
    far = dict(i, x=cols(0, 128).view(T, H, P), B=cols(128, 128).view(T, G, 128), C=cols(256, 128).view(T, G, 128),
               z=cols(384, 128).view(T, H, P), dt=cols(512, H))
    near = {k: (v.contiguous() if v is not None else None) for k, v in far.items()}
    for method in METHODS:
        a, b = _scan(far, [T], method=method), _scan(near, [T], method=method)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x, w, bias, st = _conv_inputs([T], C, 4)
    a, b = fk.conv_prefill(cols(0, C), w, bias, st, _cu([T])), fk.conv_prefill(cols(0, C).contiguous(), w, bias, st, _cu([T]))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    st = st.expand(T, -1, -1).contiguous()
    a, b = fk.conv_decode(cols(0, C), w, bias, st), fk.conv_decode(cols(0, C).contiguous(), w, bias, st)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    del wide, far, near
    batch, H, P = 4200, 32, 128                                                             # 8.8 GB of state
    i = _scan_inputs([batch], H, 8, P, state=False, seed=51)
    state = torch.randn((1, H, P, 128), device=DEV).repeat(batch, 1, 1, 1)
    tail = slice(batch - 3, batch)
    want = _step(_part(i, tail, state[tail].clone()))
    got, _ = _step(i, state=state, new_state=state)
    assert torch.equal(got[tail], want[0]) and torch.equal(state[tail], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [[0, 3000, 1000, 4133], [0, 4133, 0, 4133], [2000, 1, 4000, 4133], [0, 9000, -5, 4133]])
def test_malformed_cu_seqlens_of_a_cut_prompt_is_reported(bad):
    """Segments of offsets that overlap or run backwards stay inside the workspace; the next
    good call gives the usual bits."""
    lengths = [1300, 1333, 1500]
    i = _scan_inputs(lengths, 2, 1, 128, seed=60)
    want = _scan(i, lengths, method="tcgen05")
    fk.ssm_prefill(i["x"], i["dt"], i["A_log"], i["B"], i["C"], i["D"], i["dt_bias"], i["state"],
                   torch.tensor(bad, dtype=torch.int32, device=DEV), z=i["z"], method="tcgen05")
    with pytest.raises(ValueError, match="cu_seqlens"):
        fk.device_status()
    got = _scan(i, lengths, method="tcgen05")
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
