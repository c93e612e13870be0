"""The state space layer's operators as they are measured: the short causal convolution and
the selective scan with one decay per head, for prompts and for single tokens.

``run`` makes one pass: with ``own`` the calls a user makes of the package, otherwise the
same operators in elementary torch operations.  ``exact`` computes the same outputs in 64
bits, from the recurrences as they are defined.
"""

import math

import torch

own = False

CHUNK = 64   # the plain scan's block length


# ------------------------------------------------------------------------------ the cases

def listed():
    return [
        # The convolution in front of a Gated DeltaNet layer's q, k, v (2 * 16 * 128 + 32 * 128
        # channels): a few short prompts, half of them continued from a cached state.
        {"name": "conv prefill 4 prompts", "op": "conv_prefill", "lengths": "413,64,512,291", "channels": 8192,
         "width": 4, "act": True, "bias": False, "split": "2048,2048,4096", "state": True, "pad": 0},
        # A batch of long prompts, the projection's output holding other columns beside them.
        {"name": "conv prefill 16 x 4096", "op": "conv_prefill",
         "lengths": ",".join(["4096"] * 16), "channels": 8192, "width": 4, "act": True, "bias": False,
         "split": "2048,2048,4096", "state": False, "pad": 4160},
        # One token each of a small and of a large serving batch.
        {"name": "conv decode 4", "op": "conv_decode", "batch": 4, "channels": 8192, "width": 4, "act": True,
         "bias": False, "split": "2048,2048,4096", "pad": 0},
        {"name": "conv decode 512", "op": "conv_decode", "batch": 512, "channels": 8192, "width": 4, "act": True,
         "bias": True, "split": "", "pad": 4160},
        # Four short prompts, half with a state: latency.
        {"name": "ssm prefill 4 prompts", "op": "ssm_prefill", "lengths": "413,64,512,291", "heads": 32, "groups": 16,
         "head": 128, "state": True, "z": False, "wide": False},
        # The long batch.
        {"name": "ssm prefill 16 x 8192", "op": "ssm_prefill", "lengths": ",".join(["8192"] * 16), "heads": 32,
         "groups": 16, "head": 128, "state": True, "z": False, "wide": False},
        # One long prompt: few (sequence, head) pairs.  Heads of 64, one B and C for all of them,
        # x, B and C slices of the convolution's output, with the output gate.
        {"name": "ssm prefill 1 x 16384", "op": "ssm_prefill", "lengths": "16384", "heads": 64, "groups": 1, "head": 64,
         "state": False, "z": True, "wide": True},
        # Prompts of odd lengths, one of a single token.
        {"name": "ssm prefill ragged", "op": "ssm_prefill",
         "lengths": "1,733,2049,129,1500,64,1027,977", "heads": 24, "groups": 8, "head": 64, "state": True, "z": True,
         "wide": True},
        # One token each.
        {"name": "ssm decode 4", "op": "ssm_decode", "batch": 4, "heads": 32, "groups": 16, "head": 128, "z": False,
         "wide": False},
        {"name": "ssm decode 77", "op": "ssm_decode", "batch": 77, "heads": 64, "groups": 1, "head": 64, "z": True,
         "wide": True},
        {"name": "ssm decode 512", "op": "ssm_decode", "batch": 512, "heads": 32, "groups": 16, "head": 128, "z": False,
         "wide": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv_prefill", "conv_decode", "ssm_prefill", "ssm_prefill", "ssm_decode"])
    if op.startswith("conv"):
        parts = [8 * _log(rng, 4, 340) for _ in range(3)]
        case = {"op": op, "channels": sum(parts), "width": rng.choice([2, 3, 4, 4]), "act": rng.random() < 0.8,
                "bias": rng.random() < 0.5, "split": ",".join(map(str, parts)) if rng.random() < 0.6 else "",
                "pad": rng.choice([0, 8 * rng.randrange(1, 300)])}
    else:
        head = rng.choice([64, 128])
        groups = rng.choice([1, 2, 4, 8])
        heads = groups * rng.randrange(1, 4096 // (head * groups) + 1)
        case = {"op": op, "heads": heads, "groups": groups, "head": head, "z": rng.random() < 0.5,
                "wide": rng.random() < 0.5}
    if op.endswith("decode"):
        case["batch"] = _log(rng, 1, 512)
    else:
        n = _log(rng, 1, 16)
        top = _log(rng, 16, 4096)
        case["lengths"] = ",".join(str(rng.randrange(max(1, top // 3), top + 1)) for _ in range(n))
        case["state"] = rng.random() < 0.6
    return case


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def _parts(case):
    return [int(n) for n in case["split"].split(",")] if case["split"] else None


STATE = 128   # elements of B and C, columns of the state


# ------------------------------------------------------------------------- their inputs

def _rows(total, widths, wide, g, dev, silu=True):
    """bf16 rows of the given widths: slices of one wider row, as a projection or the
    convolution emits them, or packed tensors."""
    def fill(*shape):
        x = torch.randn(shape, generator=g, device=dev)
        return (x * torch.sigmoid(x) if silu else x).to(torch.bfloat16)
    if wide:
        return list(fill(total, sum(widths)).split(widths, dim=1))
    return [fill(total, w) for w in widths]


def _starts(lengths, dev):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=dev)


def _plan(lengths, extra, dev):
    """Row numbers that the plain forms index by: for every token its row among the rows of
    all sequences when `extra` rows stand in front of each; and the last `extra` rows."""
    place, last, at = [], [], 0
    for n in lengths:
        place.append(torch.arange(at + extra, at + extra + n))
        at += extra + n
        last.append(torch.arange(at - extra, at))
    return torch.cat(place).to(dev), torch.stack(last).to(dev)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(int(seed))
    s = {"case": dict(case), "op": case["op"]}
    if case["op"].startswith("conv"):
        C, W = case["channels"], case["width"]
        lengths = _lengths(case) if case["op"] == "conv_prefill" else [1] * case["batch"]
        total, n = sum(lengths), len(lengths)
        s["x"] = torch.randn((total, C + case["pad"]), generator=g, device=dev).to(torch.bfloat16)[:, :C]
        s["weight"] = (torch.rand((C, W), generator=g, device=dev) * 2 - 1) / math.sqrt(W)
        s["bias"] = (torch.rand(C, generator=g, device=dev) - 0.5) if case["bias"] else None
        s["state"] = torch.randn((n, W - 1, C), generator=g, device=dev).to(torch.bfloat16)
        s["split"] = _parts(case)
        s["lengths"] = lengths
        if case["op"] == "conv_prefill":
            s["cu"] = _starts(lengths, dev)
            s["place"], s["last"] = _plan(lengths, W - 1, dev)
            if case["state"]:
                s["state"][::2] = 0       # every other prompt starts anew
            else:
                s["state"] = None
        return s
    H, G, P = case["heads"], case["groups"], case["head"]
    lengths = _lengths(case) if case["op"] == "ssm_prefill" else [1] * case["batch"]
    total, n = sum(lengths), len(lengths)
    x, B, C = _rows(total, [H * P, G * STATE, G * STATE], case["wide"], g, dev)
    z, dt = _rows(total, [H * P, H], case["wide"], g, dev, silu=False)
    lead = (total,) if case["op"] == "ssm_prefill" else (total, 1)
    s["x"], s["z"] = x.view(*lead, H, P), z.view(*lead, H, P) if case["z"] else None
    s["B"], s["C"], s["dt"] = B.view(*lead, G, STATE), C.view(*lead, G, STATE), dt.view(*lead, H)
    s["A_log"] = torch.log(torch.rand(H, generator=g, device=dev) * 15.0 + 1.0)
    step = torch.exp(torch.rand(H, generator=g, device=dev) * math.log(100.0) + math.log(1e-3))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))     # softplus(dt_bias) in [0.001, 0.1]
    s["D"] = 1.0 + 0.1 * torch.randn(H, generator=g, device=dev)
    s["state"] = 0.2 * torch.randn((n, H, P, STATE), generator=g, device=dev)
    if case["op"] == "ssm_prefill":
        s["cu"] = _starts(lengths, dev)
        most = -(-max(lengths) // CHUNK) * CHUNK
        at = torch.arange(most, device=dev)
        long = torch.tensor(lengths, device=dev)
        s["there"] = at[None, :] < long[:, None]                                   # [n, most]
        s["row"] = (s["cu"][:-1, None] + at[None, :]).clamp(max=total - 1).long()  # [n, most]
        if case["state"]:
            s["state"][1::2] = 0
        else:
            s["state"] = None
    return s


# ------------------------------------------------------------------------ the plain forms

def _silu(x):
    return x / (1 + torch.exp(-x))


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(x.clamp(max=20))))


def _split(y, parts):
    return list(t.contiguous() for t in y.split(parts, dim=1)) if parts else y


def _conv(s):
    W = s["weight"].shape[1]
    x, n = s["x"].float(), len(s["lengths"])
    state = s["state"].float() if s["state"] is not None else x.new_zeros((n, W - 1, x.shape[1]))
    if s["op"] == "conv_decode":
        rows = torch.cat([state, x[:, None]], dim=1)
        y = (rows * s["weight"].float().t()).sum(dim=1)
        new = rows[:, 1:]
    else:
        rows = x.new_empty((x.shape[0] + n * (W - 1), x.shape[1]))
        rows[s["place"]] = x
        # (the rows in front of each sequence: its last rows, moved up by its length)
        front = s["last"] - torch.tensor(s["lengths"], device=x.device)[:, None]
        rows[front] = state
        y = sum(rows[s["place"] - (W - 1 - w)] * s["weight"][:, w].float() for w in range(W))
        new = rows[s["last"]]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["act"]:
        y = _silu(y)
    return _split(y.to(torch.bfloat16), s["split"]), new.to(torch.bfloat16)


def _ssm_decode(s):
    x, B, C = s["x"][:, 0].float(), s["B"][:, 0].float(), s["C"][:, 0].float()
    H, G = x.shape[1], B.shape[1]
    dt = _softplus(s["dt"][:, 0].float() + s["dt_bias"])
    decay = torch.exp(-torch.exp(s["A_log"]) * dt)
    B, C = (t[:, :, None].expand(-1, -1, H // G, -1).reshape(-1, H, 1, STATE) for t in (B, C))
    new = s["state"] * decay[..., None, None] + (dt[..., None] * x)[..., None] * B
    y = (new * C).sum(dim=-1) + s["D"][:, None] * x
    if s["z"] is not None:
        y = y * _silu(s["z"][:, 0].float())
    return y.to(torch.bfloat16)[:, None], new


def _ssm_prefill(s):
    T, H, P = s["x"].shape
    G = s["B"].shape[1]
    R, L = H // G, CHUNK
    n, most = s["row"].shape
    K = most // L
    dev = s["x"].device
    dt = _softplus(s["dt"].float() + s["dt_bias"])[s["row"]] * s["there"][..., None]        # [n, most, H]
    a = (dt.double() * -torch.exp(s["A_log"].double())).view(n, K, L, G, R).cumsum(dim=2)   # sums of log decays
    dt = dt.view(n, K, L, G, R)
    x = (s["x"].float()[s["row"]] * s["there"][..., None, None]).view(n, K, L, G, R, P)
    B, C = ((t.float()[s["row"]] * s["there"][..., None, None]).view(n, K, L, G, STATE) for t in (s["B"], s["C"]))
    # within a block
    i = torch.arange(L, device=dev)
    back = (i[:, None] >= i[None, :]).view(1, 1, 1, 1, L, L)
    al = a.permute(0, 1, 3, 4, 2)                                                          # [n, K, G, R, L]
    M = torch.where(back, torch.exp((al[..., :, None] - al[..., None, :]).clamp(max=0)).float(), torch.zeros((), device=dev))
    M = M * torch.einsum("nkigs,nkjgs->nkgij", C, B)[:, :, :, None] * dt.permute(0, 1, 3, 4, 2)[..., None, :]
    y = torch.einsum("nkgrij,nkjgrp->nkigrp", M, x)
    # what each block adds to the state, and the state in front of each block
    xw = x * (torch.exp(a[:, :, -1:] - a).float() * dt)[..., None]
    added = torch.einsum("nkjgrp,nkjgs->nkgrps", xw, B).reshape(n, K, H, P * STATE)
    first = s["state"].reshape(n, 1, H, P * STATE) if s["state"] is not None else added.new_zeros((n, 1, H, P * STATE))
    added = torch.cat([first, added], dim=1).permute(0, 2, 1, 3)                           # [n, H, K + 1, P * S]
    e = a[:, :, -1].reshape(n, K, H).cumsum(dim=1).permute(0, 2, 1)
    e = torch.cat([e.new_zeros((n, H, 1)), e], dim=2)                                      # [n, H, K + 1]
    k = torch.arange(K + 1, device=dev)
    carry = torch.where(k[:, None] >= k[None, :], torch.exp((e[..., :, None] - e[..., None, :]).clamp(max=0)).float(),
                        torch.zeros((), device=dev))
    states = torch.matmul(carry, added)                                                    # [n, H, K + 1, P * S]
    S = states[:, :, :K].reshape(n, G, R, K, P, STATE)
    y = y + torch.einsum("nkigs,ngrkps->nkigrp", C, S) * torch.exp(a).float()[..., None]
    y = y.reshape(n * most, H, P)[s["there"].reshape(-1)] + s["D"][:, None] * s["x"].float()
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    return y.to(torch.bfloat16), states[:, :, K].reshape(n, H, P, STATE)


def run(state):
    s = state
    if own:
        import fastaf_kernel_b200 as fk
        if s["op"] == "conv_prefill":
            y, new = fk.conv_prefill(s["x"], s["weight"], s["bias"], s["state"], s["cu"],
                                     activation="silu" if s["case"]["act"] else None, split=s["split"])
        elif s["op"] == "conv_decode":
            y, new = fk.conv_decode(s["x"], s["weight"], s["bias"], s["state"],
                                    activation="silu" if s["case"]["act"] else None, split=s["split"])
        elif s["op"] == "ssm_prefill":
            y, new = fk.ssm_prefill(s["x"], s["dt"], s["A_log"], s["B"], s["C"], s["D"], s["dt_bias"], s["state"],
                                    s["cu"], z=s["z"])
        else:
            y, new = fk.ssm_decode(s["x"], s["dt"], s["A_log"], s["B"], s["C"], s["D"], s["dt_bias"], s["state"],
                                   z=s["z"])
        y = list(y) if isinstance(y, tuple) else y
    elif s["op"].startswith("conv"):
        y, new = _conv(s)
    elif s["op"] == "ssm_prefill":
        y, new = _ssm_prefill(s)
    else:
        y, new = _ssm_decode(s)
    return {"y": y, "state": new}


# ---------------------------------------------------------------------------- their work

def work(case):
    if case["op"].startswith("conv"):
        n, total = (len(_lengths(case)), sum(_lengths(case))) if "lengths" in case else (case["batch"], case["batch"])
        C, W = case["channels"], case["width"]
        kept = n * (W - 1) * C * 2
        held = 1 if case.get("state", True) else 0
        return {"bytes": 2 * total * C * 2 + (1 + held) * kept + C * W * 4 + (C * 4 if case["bias"] else 0),
                "flops": 2.0 * total * C * W}
    H, G, P = case["heads"], case["groups"], case["head"]
    n, total = (len(_lengths(case)), sum(_lengths(case))) if "lengths" in case else (case["batch"], case["batch"])
    kept = n * H * P * STATE * 4
    held = 1 if case.get("state", True) else 0
    tokens = total * (2 * H * P * 2 + (H * P * 2 if case["z"] else 0) + 2 * G * STATE * 2 + H * 2)
    # the recurrence itself: decay, outer product and read-out of a [P, STATE] state per token
    # and head, or in blocks of 64 tokens, whichever is less
    token = 5 * P * STATE
    block = 2 * (CHUNK * STATE * G / H / 2 + CHUNK * P / 2 + 2 * P * STATE)
    return {"bytes": tokens + (1 + held) * kept, "flops": float(total * H * min(token, block))}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"].startswith("conv"):
        W, C = s["weight"].shape[1], s["x"].shape[1]
        w = s["weight"].to(f64)
        y, new, at = [], [], 0
        for k, length in enumerate(s["lengths"]):
            seq = s["x"][at:at + length].to(f64)
            before = s["state"][k].to(f64) if s["state"] is not None else torch.zeros((W - 1, C), dtype=f64, device=seq.device)
            padded = torch.cat([before, seq])
            out = torch.zeros_like(seq)
            for j in range(W):
                out += padded[j:j + length] * w[:, j]
            if s["bias"] is not None:
                out += s["bias"].to(f64)
            y.append(out * torch.sigmoid(out) if case["act"] else out)
            new.append(padded[length:])
            at += length
        y = torch.cat(y)
        parts = _parts(case)
        return {"y": list(y.split(parts, dim=1)) if parts else y, "state": torch.stack(new)}
    H, G, P = case["heads"], case["groups"], case["head"]
    shape = s["x"].shape
    x, dt = s["x"].reshape(-1, H, P), s["dt"].reshape(-1, H)
    B, C = s["B"].reshape(-1, G, STATE), s["C"].reshape(-1, G, STATE)
    dev = x.device
    lengths = _lengths(case) if case["op"] == "ssm_prefill" else [1] * case["batch"]
    start = torch.tensor([sum(lengths[:k]) for k in range(len(lengths))] if len(lengths) < 64 else list(range(len(lengths))), device=dev)
    order = sorted(range(len(lengths)), key=lambda k: -lengths[k])
    start = start[torch.tensor(order, device=dev)]
    S = torch.zeros((len(lengths), H, P, STATE), dtype=f64, device=dev)
    if s["state"] is not None:
        S += s["state"][torch.tensor(order, device=dev)]
    A, bias, D = -torch.exp(s["A_log"].to(f64)), s["dt_bias"].to(f64), s["D"].to(f64)
    y = torch.empty(x.shape, dtype=f64, device=dev)
    for t in range(max(lengths)):
        live = sum(n > t for n in lengths)            # the longest come first
        r = start[:live] + t
        step = torch.nn.functional.softplus(dt[r].to(f64) + bias)
        xt = x[r].to(f64)
        Bt, Ct = (v[r].to(f64).repeat_interleave(H // G, dim=1) for v in (B, C))
        S[:live] *= torch.exp(A * step)[..., None, None]
        S[:live] += (step[..., None] * xt)[..., None] * Bt[:, :, None, :]
        y[r] = torch.einsum("nhps,nhs->nhp", S[:live], Ct) + D[:, None] * xt
    if s["z"] is not None:
        z = s["z"].reshape(-1, H, P).to(f64)
        y = y * z * torch.sigmoid(z)
    back = torch.empty_like(S)
    back[torch.tensor(order, device=dev)] = S
    return {"y": y.reshape(shape), "state": back}
