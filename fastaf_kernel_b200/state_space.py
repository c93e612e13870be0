"""State space layers beside Gated DeltaNet ones: the short causal convolution in front of
either layer's recurrence, and the selective scan with one decay per head, for prompts and
for single tokens.

The manner is that of ``kernel`` and ``kernel_decode``: packed varlen prompts with
``cu_seqlens``, bf16 rows, gate inputs and parameters in fp32 or bf16, an fp32 k-last state,
value-returning calls with keyword-only ``output=`` / ``new_state=`` destinations, on the
current torch CUDA stream of the inputs' device, with no CPU path.  Rows may be slices of a
wider projection output: they are read through their row stride, without a copy.

The reference has neither operator; its entry points start at q, k and v.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .api import _GATE_DTYPES, _check_cu_seqlens_host, _gate

__all__ = ["conv_prefill", "conv_decode", "ssm_prefill", "ssm_decode", "ssm_method"]

_ACTIVATIONS = {None: _lib.GDN_ACTIVATION_NONE, "silu": _lib.GDN_ACTIVATION_SILU}
_METHODS = {"auto": _lib.GDN_PREFILL_AUTO, "recurrent": _lib.GDN_PREFILL_RECURRENT,
            "tcgen05": _lib.GDN_PREFILL_TCGEN05}
_MAX_OUTPUTS = 4
_BF16, _F32 = torch.bfloat16, torch.float32

Outputs = Union[torch.Tensor, Tuple[torch.Tensor, ...]]

# (single-token calls take a few microseconds of GPU time: the checks below look at each
# tensor once and build no torch objects on the way)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _device_of(names, required, optional) -> int:
    """The CUDA device index of the first tensor, which all the given ones are on."""
    tensors = required + optional
    try:
        index = tensors[0].get_device()
        if index >= 0:
            for t in required:
                if t.get_device() != index:
                    break
            else:
                for t in optional:
                    if t is not None and t.get_device() != index:
                        break
                else:
                    return index
    except AttributeError:
        pass
    for i, (name, t) in enumerate(zip(names.split(), tensors)):
        if t is None and i >= len(required):
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path), got {t.device}")
        if t.get_device() != tensors[0].get_device():
            raise ValueError(f"{name} is on {t.device}, expected {tensors[0].device}")
    raise TypeError("x must be a torch.Tensor")


def _call(fn, index: int, args) -> None:
    """One C call on the current stream of device ``index``."""
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc)


def _rows(name: str, t: torch.Tensor, width: int) -> Tuple[torch.Tensor, int, int]:
    """bf16 rows of ``width`` elements (the last dimensions of ``t``, packed among
    themselves) as the kernels read them: the tensor, its address and its row stride in
    elements.  Rows that do not start on a 16-byte boundary or are not packed become a
    packed copy."""
    if t.dtype != _BF16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    at = t.data_ptr()
    if t.is_contiguous():
        if at % 16:      # (a contiguous slice may still start off a 16-byte boundary)
            t = t.clone()
            at = t.data_ptr()
        return t, at, width
    strides, step, packed = t.stride(), 1, True
    for n, st in zip(reversed(t.shape[1:]), reversed(strides[1:])):
        packed = packed and (n == 1 or st == step)
        step *= n
    stride = strides[0] if t.shape[0] > 1 else width
    if packed and stride >= width and stride % 8 == 0 and stride < 1 << 31 and at % 16 == 0:
        return t, at, stride
    t = t.contiguous()
    return t, t.data_ptr(), width


def _dt_rows(t: torch.Tensor, heads: int) -> Tuple[torch.Tensor, int]:
    """dt as the kernels read it: fp32 or bf16 rows of ``heads`` elements and their stride."""
    if t.dtype not in _GATE_DTYPES:
        t = t.float()
    if t.is_contiguous():
        return t, heads
    if t.stride(-1) == 1 or heads == 1:
        stride = t.stride(0) if t.shape[0] > 1 else heads
        if heads <= stride < 1 << 31:
            return t, stride
    return t.contiguous(), heads


def _destination(name: str, t: Optional[torch.Tensor], shape, dtype, like: torch.Tensor) -> torch.Tensor:
    if t is None:
        return like.new_empty(shape) if like.dtype == dtype else like.new_empty(shape, dtype=dtype)
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous() or t.device != like.device:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {like.device}")
    return t


def _state(state: Optional[torch.Tensor], new_state: Optional[torch.Tensor], shape, dtype):
    """The state as the kernels read it.  A state that is also the destination has to be
    readable as it is: a converted copy would leave it half old."""
    if state is None:
        return None
    if state.shape != shape:
        raise ValueError(f"state must have shape {tuple(shape)}, got {tuple(state.shape)}")
    if state.dtype == dtype and state.is_contiguous() and state.data_ptr() % 16 == 0:
        return state
    if new_state is not None and new_state.data_ptr() == state.data_ptr():
        raise ValueError(f"an in-place state must be a contiguous, 16-byte aligned {dtype} tensor")
    return state.to(dtype).contiguous().clone()


def _cu(cu_seqlens: torch.Tensor, T: int, x: torch.Tensor, validate: bool) -> Tuple[torch.Tensor, int]:
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be a 1-D tensor of at least one entry")
    if cu_seqlens.is_cuda:
        if cu_seqlens.get_device() != x.get_device():
            raise ValueError(f"cu_seqlens is on {cu_seqlens.device}, expected {x.device}")
    elif validate:
        _check_cu_seqlens_host(cu_seqlens.detach().to(torch.int64), T)
    if cu_seqlens.shape[0] == 1 and T:
        raise ValueError("cu_seqlens names no sequence but there are tokens")
    if cu_seqlens.dtype != torch.int32 or not cu_seqlens.is_cuda or not cu_seqlens.is_contiguous():
        cu_seqlens = cu_seqlens.to(device=x.device, dtype=torch.int32).contiguous()
    return cu_seqlens, cu_seqlens.shape[0] - 1


# ------------------------------------------------------------------------ the convolution

def _conv(x, weight, bias, state, num_seqs, activation, split, output, new_state):
    """The checks and conversions of both convolution calls: the C call's arguments (without
    cu_seqlens and sizes that only prefill has), the outputs and the new state."""
    if x.dim() != 2:
        raise ValueError("x must be [rows, channels]")
    T, C = x.shape
    if weight.dim() != 2 or weight.shape[0] != C:
        raise ValueError(f"weight must be [channels, width] = [{C}, width], got {tuple(weight.shape)}")
    W = weight.shape[1]
    if W < 2 or W > 4:
        raise NotImplementedError(f"width={W} is not supported (2, 3 or 4)")
    if C == 0 or C % 8:
        raise ValueError(f"channels={C} must be a positive multiple of 8")
    if activation not in _ACTIVATIONS:
        raise ValueError("activation must be None or 'silu'")
    if bias is not None and bias.shape != (C,):
        raise ValueError(f"bias must be [{C}]")
    weight = _gate(weight)
    if bias is not None:
        bias = _gate(bias)
        if bias.dtype != weight.dtype:
            weight, bias = weight.float(), bias.float()
    x, at, stride = _rows("x", x, C)
    if split is None:
        y = _destination("output", output, (T, C), _BF16, x)
        outs: Sequence[torch.Tensor] = (y,)
        widths: Sequence[int] = (C,)
    else:
        widths = split
        if not 1 <= len(widths) <= _MAX_OUTPUTS or any([n <= 0 or n % 8 for n in widths]) or sum(widths) != C:
            raise ValueError(f"split must be 1 to {_MAX_OUTPUTS} positive multiples of 8 that add up to {C} channels")
        if output is not None and len(output) != len(widths):
            raise ValueError("output must hold one tensor per split")
        y = outs = (tuple([x.new_empty((T, n)) for n in widths]) if output is None else
                    tuple([_destination("output", t, (T, n), _BF16, x) for t, n in zip(output, widths)]))
    shape = (num_seqs, W - 1, C)
    new_state = _destination("new_state", new_state, shape, _BF16, x if state is None else state)
    state = _state(state, new_state, shape, _BF16)
    n = len(widths)
    head = (at, stride, weight.data_ptr(), None if bias is None else bias.data_ptr(), _GATE_DTYPES[weight.dtype],
            None if state is None else state.data_ptr())
    tail = (_ACTIVATIONS[activation], (ctypes.c_void_p * n)(*[t.data_ptr() for t in outs]),
            (ctypes.c_int64 * n)(*widths), n, new_state.data_ptr())
    # (the converted copies live until the call has been enqueued)
    return head, tail, (T, C, W), y, new_state, (x, weight, bias, state)


def conv_prefill(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                 state: Optional[torch.Tensor], cu_seqlens: torch.Tensor, *,
                 activation: Optional[str] = "silu", split: Optional[Sequence[int]] = None,
                 output=None, new_state: Optional[torch.Tensor] = None,
                 validate: bool = True) -> Tuple[Outputs, torch.Tensor]:
    """Short depthwise causal convolution over packed sequences:
    y[t, c] = act(bias[c] + sum_w weight[c, w] * x[t - (W-1) + w, c]).

    x [T, C] bf16 (C a multiple of 8; a slice of wider rows is read in place); weight [C, W]
    with W = 2, 3 or 4, and bias [C] or None, fp32 or bf16; state [N, W-1, C] bf16 (the rows
    in front of each sequence, oldest first) or None for zeros; cu_seqlens [N+1] as for
    ``kernel``.  ``activation`` is "silu" or None.  Returns (y [T, C] bf16, new_state
    [N, W-1, C] bf16), the new state being the last W-1 rows of [state; x].

    ``split`` gives the widths of up to four packed tensors that take the channels side by
    side, such as q, k and v for ``kernel`` or x, B and C for ``ssm_prefill``; y (and
    ``output``) is then a tuple of [T, width] tensors.  Outputs and new_state must overlap
    neither each other nor an input.
    """
    index = _device_of("x weight bias state", (x, weight), (bias, state))
    if x.dim() != 2:
        raise ValueError("x must be [T, channels]")
    cu, N = _cu(cu_seqlens, x.shape[0], x, validate)
    head, tail, sizes, y, new_state, held = _conv(x, weight, bias, state, N, activation, split, output, new_state)
    _call(_lib.load().gdn_conv_prefill, index, (*head, cu.data_ptr(), N, *sizes, *tail))
    return y, new_state


def conv_decode(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                state: Optional[torch.Tensor], *, activation: Optional[str] = "silu",
                split: Optional[Sequence[int]] = None, output=None,
                new_state: Optional[torch.Tensor] = None) -> Tuple[Outputs, torch.Tensor]:
    """``conv_prefill`` for one token of each sequence: x [B, C], state [B, W-1, C] bf16 or
    None.  Returns (y [B, C], new_state); pass ``new_state=state`` to update it in place."""
    index = _device_of("x weight bias state", (x, weight), (bias, state))
    if x.dim() != 2:
        raise ValueError("x must be [B, channels]")
    head, tail, sizes, y, new_state, held = _conv(x, weight, bias, state, x.shape[0], activation, split, output,
                                                  new_state)
    _call(_lib.load().gdn_conv_decode, index, (*head, *sizes, *tail))
    return y, new_state


# ------------------------------------------------------------------------------- the scan

def ssm_method(total_tokens: int, method: str = "auto", num_seqs: int = 1) -> str:
    """Name of the scan kernel an ``ssm_prefill`` call with ``method`` runs for
    ``total_tokens`` packed tokens in ``num_seqs`` sequences on the current CUDA device."""
    if method not in _METHODS:
        raise ValueError(f"method must be one of {sorted(_METHODS)}")
    code = _lib.load().gdn_ssm_resolve(int(total_tokens), int(num_seqs), _METHODS[method])
    return {v: k for k, v in _METHODS.items()}[code]


def _ssm(x, dt, A_log, B, C, D, dt_bias, state, z, num_seqs, output, new_state):
    """The checks and conversions of both scan calls."""
    shape, Bs, ds = x.shape, B.shape, dt.shape
    rank, H, P = len(shape), shape[-2], shape[-1]
    if P != 64 and P != 128:
        raise NotImplementedError(f"head_size={P} is not supported (64 or 128)")
    if len(Bs) != rank or Bs[:-2] != shape[:-2]:
        raise ValueError(f"B must be [..., groups, state_size] with the leading sizes of x {list(shape)}, got {list(Bs)}")
    G, S = Bs[-2], Bs[-1]
    if S != 128:
        raise NotImplementedError(f"state_size={S} is not supported (only 128)")
    if C.shape != Bs:
        raise ValueError(f"C shape {list(C.shape)} must equal B shape {list(Bs)}")
    if H == 0 or G == 0 or H % G:
        raise ValueError(f"{H} heads must be a positive multiple of {G} groups")
    if ds != shape[:-1]:
        raise ValueError(f"dt must be {list(shape[:-1])}, got {list(ds)}")
    per_head = (H,)
    if A_log.shape != per_head or (D is not None and D.shape != per_head) or (
            dt_bias is not None and dt_bias.shape != per_head):
        raise ValueError(f"A_log, D and dt_bias must be [heads] = [{H}]")
    if z is not None and z.shape != shape:
        raise ValueError(f"z shape {list(z.shape)} must equal x shape {list(shape)}")
    x, xp, sx = _rows("x", x, H * P)
    B, Bp, sB = _rows("B", B, G * S)
    C, Cp, sC = _rows("C", C, G * S)
    zp, sz = None, 0
    if z is not None:
        z, zp, sz = _rows("z", z, H * P)
    dt, sdt = _dt_rows(dt, H)
    A_log = _gate(A_log)
    D = None if D is None else _gate(D)
    dt_bias = None if dt_bias is None else _gate(dt_bias)
    if (D is not None and D.dtype != A_log.dtype) or (dt_bias is not None and dt_bias.dtype != A_log.dtype):
        A_log = A_log.float()
        D = None if D is None else D.float()
        dt_bias = None if dt_bias is None else dt_bias.float()
    output = _destination("output", output, shape, _BF16, x)
    state_shape = (num_seqs, H, P, S)
    new_state = _destination("new_state", new_state, state_shape, _F32, x if state is None else state)
    state = _state(state, new_state, state_shape, _F32)
    head = (xp, sx, dt.data_ptr(), sdt, A_log.data_ptr(), Bp, sB, Cp, sC, None if D is None else D.data_ptr(),
            None if dt_bias is None else dt_bias.data_ptr(), zp, sz, None if state is None else state.data_ptr())
    tail = (H, G, P, S, _GATE_DTYPES[dt.dtype], _GATE_DTYPES[A_log.dtype], output.data_ptr(), new_state.data_ptr())
    # (the converted copies live until the call has been enqueued)
    return head, tail, output, new_state, (x, dt, A_log, B, C, D, dt_bias, z, state)


def ssm_prefill(x: torch.Tensor, dt: torch.Tensor, A_log: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                D: Optional[torch.Tensor], dt_bias: Optional[torch.Tensor], state: Optional[torch.Tensor],
                cu_seqlens: torch.Tensor, *, z: Optional[torch.Tensor] = None,
                output: Optional[torch.Tensor] = None, new_state: Optional[torch.Tensor] = None,
                method: str = "auto", validate: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """Selective scan with one decay per head over packed sequences:

        dt' = softplus(dt + dt_bias),  S <- exp(-exp(A_log) dt') S + dt' x B^T,
        y = S C + D x,  and with ``z``  y <- y * silu(z).

    x, z [T, H, P] bf16 (P = 64 or 128); dt [T, H]; B, C [T, G, 128] bf16, shared by the
    H / G consecutive heads of a group; A_log, D, dt_bias [H] (D and dt_bias may be None);
    state [N, H, P, 128] fp32 or None for zeros; cu_seqlens [N+1] as for ``kernel``.  Returns
    (y [T, H, P] bf16, new_state [N, H, P, 128] fp32); a sequence of length 0 keeps its
    state.  ``output`` and new_state must overlap neither each other nor an input.

    ``method`` chooses the kernel: "tcgen05" (64-token chunks on the tensor cores, from 64
    tokens), "recurrent" (CUDA cores, one token after the other) or "auto" (what
    ``ssm_method`` reports).  State and D x are as good as fp32 sums from either; "tcgen05"
    rounds one operand of each of y's products to bf16 (the state in S C, the scores of a
    chunk's own tokens).  "auto" and the cutting of few long prompts go by the whole batch, so
    a prompt may come out with other last bits in another batch.
    """
    index = _device_of("x dt A_log B C D dt_bias state z", (x, dt, A_log, B, C), (D, dt_bias, state, z))
    if x.dim() != 3:
        raise ValueError("x must be [T, heads, head_size]")
    if method not in _METHODS:
        raise ValueError(f"method must be one of {sorted(_METHODS)}")
    T = x.shape[0]
    cu, N = _cu(cu_seqlens, T, x, validate)
    head, tail, output, new_state, held = _ssm(x, dt, A_log, B, C, D, dt_bias, state, z, N, output, new_state)
    _call(_lib.load().gdn_ssm_prefill, index, (*head, cu.data_ptr(), N, T, *tail, _METHODS[method]))
    return output, new_state


def ssm_decode(x: torch.Tensor, dt: torch.Tensor, A_log: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
               D: Optional[torch.Tensor], dt_bias: Optional[torch.Tensor], state: Optional[torch.Tensor], *,
               z: Optional[torch.Tensor] = None, output: Optional[torch.Tensor] = None,
               new_state: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One step of ``ssm_prefill``'s scan for each sequence: x, z [B, 1, H, P]; dt [B, 1, H];
    B, C [B, 1, G, 128]; state [B, H, P, 128] fp32 or None.  Returns (y [B, 1, H, P] bf16,
    new_state); pass ``new_state=state`` to update the state in place."""
    index = _device_of("x dt A_log B C D dt_bias state z", (x, dt, A_log, B, C), (D, dt_bias, state, z))
    if x.dim() != 4 or x.shape[1] != 1:
        raise ValueError("x must be [B, 1, heads, head_size]")
    batch = x.shape[0]
    head, tail, output, new_state, held = _ssm(x, dt, A_log, B, C, D, dt_bias, state, z, batch, output, new_state)
    _call(_lib.load().gdn_ssm_decode, index, (*head, batch, *tail))
    return output, new_state
