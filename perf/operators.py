"""Cases for the operators of a state-space layer that stand around the chunked scan: the residual's
addition with the root-mean-square norm that opens a layer, the short causal convolution, and the
token-by-token selective scan (prompts, gradients, single tokens).

Each case is a dict of plain values; `prepare` makes what a program holds before the call, `run` makes
one pass (the plain torch form, or with `own` set the package's kernels), `exact` computes the same
outputs in 64 bits from the definition, `work` says what a pass cannot do without.

Layouts are the package's: positions before channels, x (batch, seqlen, channels), B and C (batch,
seqlen, ngroups, dstate).  Random values follow its benchmark data: x, B, C, D ~ N(0, 1),
A = -exp(U[0, ln 16]), dt_bias the inverse softplus of U[1e-3, 1e-1]."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


# ---------------------------------------------------------------------------------------------------
# cases

def listed():
    return [
        # a generated token's way through one layer for four sequences: 8-bit input of the projection
        dict(name="norm_token_e4m3", op="norm", batch=4, seqlen=1, dim=2560, dtype="bf16", residual="bf16", out="e4m3"),
        # a batch of prompts before an 8-bit projection
        dict(name="norm_prompt_e4m3", op="norm", batch=8, seqlen=4096, dim=2560, dtype="bf16", residual="bf16", out="e4m3"),
        # training with the residual stream in 32 bits, forward and gradients
        dict(name="norm_train", op="norm_train", batch=4, seqlen=2047, dim=4096, dtype="bf16", residual="fp32"),
        # a batch of prompts: x, B and C of 80 heads of 64 and one group of 128, read out of the projection's buffer
        dict(name="conv_prompt", op="conv", batch=8, seqlen=4096, channels=5376, width=4, dtype="bf16", extra=5200, packed=False),
        # training on packed sequences: 24 heads of 64 and one group of 128, an odd length
        dict(name="conv_train_packed", op="conv_train", batch=3, seqlen=2049, channels=1792, width=4, dtype="bf16", extra=0, packed=True),
        # one token for each of 64 running sequences
        dict(name="conv_step", op="conv_step", batch=64, channels=5376, width=4, dtype="bf16", slots=96),
        # prompts through the gated scan
        dict(name="scan_prompt", op="scan", batch=2, seqlen=4096, channels=5120, dstate=16, ngroups=1, dtype="bf16",
             gate=True, packed=False, initial=False),
        # one long document on few channels (a shard of a layer): odd length, continued from a state
        dict(name="scan_prompt_long", op="scan", batch=1, seqlen=65537, channels=320, dstate=16, ngroups=1, dtype="bf16",
             gate=True, packed=False, initial=True),
        # packed sequences in 32 bits with groups and a larger state
        dict(name="scan_prompt_groups", op="scan", batch=3, seqlen=777, channels=1536, dstate=64, ngroups=4, dtype="fp32",
             gate=False, packed=True, initial=False),
        # training, forward and all gradients
        dict(name="scan_train", op="scan_train", batch=2, seqlen=2048, channels=5120, dstate=16, ngroups=1, dtype="bf16",
             gate=True, packed=False),
        # one token of a single sequence: latency
        dict(name="scan_step_channels", op="scan_step", form="channels", batch=1, heads=1536, headdim=1, dstate=16, ngroups=1,
             dtype="bf16", state="fp32", slots=4),
        # one token for each of 128 running sequences that the chunked scan began
        dict(name="scan_step_heads", op="scan_step", form="heads", batch=128, heads=80, headdim=64, dstate=128, ngroups=1,
             dtype="bf16", state="fp32", slots=160),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_train", "conv", "conv_train", "conv_step", "scan", "scan", "scan_train", "scan_step"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("norm", "norm_train"):
        dim = _spread(rng, 64, 10240) if rng.random() < 0.4 else 8 * _spread(rng, 16, 1280)
        rows = _spread(rng, 1, max(1, min(40000, 60_000_000 // dim)))
        batch = rng.choice([b for b in (1, 2, 3, 4, 8) if b <= rows])
        c = dict(op=op, batch=batch, seqlen=rows // batch, dim=dim, dtype=dtype, residual=rng.choice([dtype, "fp32", "none"]))
        if op == "norm":
            c["out"] = rng.choice([dtype, "e4m3", "int8"])
        elif c["residual"] == "none":
            c["residual"] = dtype
        return c
    if op in ("conv", "conv_train"):
        channels = _spread(rng, 64, 8192) if rng.random() < 0.4 else 8 * _spread(rng, 16, 1024)
        tokens = _spread(rng, 2, max(2, (90_000_000 if op == "conv" else 20_000_000) // channels))
        batch = rng.choice([b for b in (1, 2, 3, 4, 8) if b <= tokens])
        return dict(op=op, batch=batch, seqlen=tokens // batch, channels=channels, width=rng.choice([2, 3, 4, 4]), dtype=dtype,
                    extra=rng.choice([0, 24, 2048]), packed=rng.random() < 0.4)
    if op == "conv_step":
        batch = _spread(rng, 1, 512)
        return dict(op=op, batch=batch, channels=_spread(rng, 64, 10240), width=rng.choice([2, 3, 4, 4]), dtype=dtype,
                    slots=batch + rng.randrange(64))
    if op in ("scan", "scan_train"):
        ngroups = rng.choice([1, 1, 2, 4])
        dstate = rng.choice([8, 16, 16, 16, 24, 32, 64, 128])
        channels = ngroups * _spread(rng, 32, 5120 // ngroups)
        most = (600_000_000 if op == "scan" else 300_000_000) // (channels * dstate)
        tokens = _spread(rng, 1, max(1, min(60000 if op == "scan" else 20000, most)))
        batch = rng.choice([b for b in (1, 2, 3, 4) if b <= tokens])
        c = dict(op=op, batch=batch, seqlen=tokens // batch, channels=channels, dstate=dstate, ngroups=ngroups, dtype=dtype,
                 gate=rng.random() < 0.6, packed=rng.random() < 0.3)
        if op == "scan":
            c["initial"] = rng.random() < 0.5
        return c
    if rng.random() < 0.5:
        batch = _spread(rng, 1, 256)
        return dict(op=op, form="channels", batch=batch, heads=_spread(rng, 64, 8192), headdim=1, dstate=rng.choice([8, 16, 16, 32]),
                    ngroups=1, dtype=dtype, state=rng.choice(["fp32", "fp32", dtype]), slots=batch + rng.randrange(32))
    batch = _spread(rng, 1, 96)
    ngroups = rng.choice([1, 1, 2, 8])
    return dict(op=op, form="heads", batch=batch, heads=ngroups * _spread(rng, 1, 96 // ngroups), headdim=rng.choice([32, 64, 64, 128]),
                dstate=rng.choice([16, 64, 128, 128]), ngroups=ngroups, dtype=dtype, state=rng.choice(["fp32", "fp32", dtype]),
                slots=batch + rng.randrange(32))


# ---------------------------------------------------------------------------------------------------
# inputs

def _maker(seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    return gen, normal, uniform


def _packed_index(batch, seqlen, gen):
    """Sequence numbers of packed sequences: a new one begins about every 200 positions; rows start at 0."""
    cut = torch.rand((batch, seqlen), generator=gen, device="cuda") < 1.0 / 200
    cut[:, 0] = False
    return cut.cumsum(1).to(torch.int32)


def prepare(case, seed):
    c = case
    gen, normal, uniform = _maker(seed)
    dtype = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] in ("norm", "norm_train"):
        shape = (c["batch"], c["seqlen"], c["dim"])
        s["x"] = normal(*shape, dtype=dtype)
        s["residual"] = None if c["residual"] == "none" else normal(*shape, dtype=DTYPES[c["residual"]]).mul_(2)
        s["weight"] = 1 + 0.1 * normal(c["dim"])
        if c["op"] == "norm_train":
            s["dout"] = normal(*shape, dtype=dtype)
            s["dresidual"] = normal(*shape, dtype=DTYPES[c["residual"]])
        return s
    if c["op"] in ("conv", "conv_train"):
        # x is a column range of the projection's output
        s["x"] = normal(c["batch"], c["seqlen"], c["channels"] + c["extra"], dtype=dtype)[..., c["extra"]:]
        s["weight"] = (uniform(c["channels"], c["width"]) * 2 - 1) / math.sqrt(c["width"])
        s["bias"] = (uniform(c["channels"]) * 2 - 1) / math.sqrt(c["width"])
        s["seq_idx"] = _packed_index(c["batch"], c["seqlen"], gen) if c["packed"] else None
        s["initial"] = None
        if c["op"] == "conv_train":
            s["dout"] = normal(c["batch"], c["seqlen"], c["channels"], dtype=dtype)
        return s
    if c["op"] == "conv_step":
        s["x"] = normal(c["batch"], c["channels"], dtype=dtype)
        s["state"] = normal(c["slots"], c["width"] - 1, c["channels"], dtype=dtype)
        s["weight"] = (uniform(c["channels"], c["width"]) * 2 - 1) / math.sqrt(c["width"])
        s["bias"] = (uniform(c["channels"]) * 2 - 1) / math.sqrt(c["width"])
        s["index"] = torch.randperm(c["slots"], generator=gen, device="cuda")[:c["batch"]].to(torch.int32)
        return s
    d0 = uniform(c["heads"] if c["op"] == "scan_step" else c["channels"]) * (1e-1 - 1e-3) + 1e-3
    s["dt_bias"] = d0 + torch.log(-torch.expm1(-d0))
    if c["op"] in ("scan", "scan_train"):
        b, l, d, n, g = c["batch"], c["seqlen"], c["channels"], c["dstate"], c["ngroups"]
        s["x"], s["dt"] = normal(b, l, d, dtype=dtype), normal(b, l, d, dtype=dtype)
        s["A"] = -torch.exp(uniform(d, n) * math.log(16.0))
        s["B"], s["C"] = normal(b, l, g, n, dtype=dtype), normal(b, l, g, n, dtype=dtype)
        s["D"] = normal(d)
        s["z"] = normal(b, l, d, dtype=dtype) if c["gate"] else None
        s["seq_idx"] = _packed_index(b, l, gen) if c["packed"] else None
        s["initial"] = normal(b, d, n) if c.get("initial") else None
        if c["op"] == "scan_train":
            s["dout"] = normal(b, l, d, dtype=dtype)
        return s
    b, h, p, n, g = c["batch"], c["heads"], c["headdim"], c["dstate"], c["ngroups"]
    wide = (h, p) if c["form"] == "heads" else (h,)
    s["x"], s["z"] = normal(b, *wide, dtype=dtype), normal(b, *wide, dtype=dtype)
    s["dt"] = normal(b, h, dtype=dtype)
    s["A"] = -torch.exp(uniform(*((h,) if c["form"] == "heads" else (h, n))) * math.log(16.0))
    s["B"], s["C"] = normal(b, g, n, dtype=dtype), normal(b, g, n, dtype=dtype)
    s["D"] = normal(h)
    s["state"] = normal(c["slots"], *wide, n, dtype=DTYPES[c["state"]])
    s["index"] = torch.randperm(c["slots"], generator=gen, device="cuda")[:b].to(torch.int32)
    return s


# ---------------------------------------------------------------------------------------------------
# one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "norm_train": _own_norm_train, "conv": _own_conv, "conv_train": _own_conv_train,
                "conv_step": _own_conv_step, "scan": _own_scan, "scan_train": _own_scan_train, "scan_step": _own_scan_step}[op](state)
    return {"norm": _norm, "norm_train": _norm_train, "conv": _conv, "conv_train": _conv_train, "conv_step": _conv_step,
            "scan": _scan, "scan_train": _scan_train, "scan_step": _scan_step}[op](state)


# --- the package's calls

def _codes(q):
    """8-bit whole numbers as the values they stand for (times the row's scale)."""
    return q.to(torch.bfloat16) if q.dtype == torch.int8 else q


def _own_norm(s):
    from mamba_fused_minimal_b200.kernels.add_rms_norm import _add_rms_norm_fwd
    kind = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}.get(s["case"]["out"])
    out, total, rstd, scales = _add_rms_norm_fwd(s["x"], s["weight"], residual=s["residual"], eps=EPS, out_dtype=kind)
    return {"out": _codes(out), "residual": total, "scales": scales}


def _own_norm_train(s):
    from mamba_fused_minimal_b200.kernels.add_rms_norm import _add_rms_norm_bwd, _add_rms_norm_fwd
    out, total, rstd, _ = _add_rms_norm_fwd(s["x"], s["weight"], residual=s["residual"], eps=EPS)
    dx, dres, dweight = _add_rms_norm_bwd(s["dout"], total, s["weight"], rstd, dresidual=s["dresidual"], x_dtype=s["x"].dtype)
    return {"out": out, "residual": total, "dx": dx, "dresidual": dres, "dweight": dweight}


def _own_conv(s):
    from mamba_fused_minimal_b200.kernels.short_conv import _short_conv_fwd
    out, final = _short_conv_fwd(s["x"], s["weight"], bias=s["bias"], apply_silu=True, initial_states=s["initial"],
                                 seq_idx=s["seq_idx"], return_final_states=True)
    return {"out": out, "final": final}


def _own_conv_train(s):
    from mamba_fused_minimal_b200.kernels.short_conv import _short_conv_bwd, _short_conv_fwd
    out, _ = _short_conv_fwd(s["x"], s["weight"], bias=s["bias"], apply_silu=True, seq_idx=s["seq_idx"])
    dx, dweight, dbias, _ = _short_conv_bwd(s["dout"], s["x"], s["weight"], bias=s["bias"], apply_silu=True, seq_idx=s["seq_idx"])
    return {"out": out, "dx": dx, "dweight": dweight, "dbias": dbias}


def _own_conv_step(s):
    from mamba_fused_minimal_b200.kernels.short_conv import _short_conv_step
    out = _short_conv_step(s["x"], s["state"], s["weight"], bias=s["bias"], apply_silu=True, state_indices=s["index"])
    return {"out": out, "state": s["state"]}


def _own_scan(s):
    from mamba_fused_minimal_b200.kernels.token_scan import _token_scan_fwd
    out, final, _ = _token_scan_fwd(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                    dt_softplus=True, initial_states=s["initial"], seq_idx=s["seq_idx"])
    return {"out": out, "final": final}


def _own_scan_train(s):
    from mamba_fused_minimal_b200.kernels.token_scan import _token_scan_bwd, _token_scan_fwd
    out, final, saved = _token_scan_fwd(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                        dt_softplus=True, seq_idx=s["seq_idx"], for_backward=True)
    dx, ddt, dA, dB, dC, dD, dz, dbias, _ = _token_scan_bwd(s["dout"], s["x"], s["dt"], s["A"], s["B"], s["C"], saved, D=s["D"],
                                                            z=s["z"], dt_bias=s["dt_bias"], dt_softplus=True, seq_idx=s["seq_idx"])
    return {"out": out, "final": final, "dx": dx, "ddt": ddt, "dA": dA, "dB": dB, "dC": dC, "dD": dD, "dz": dz, "dbias": dbias}


def _own_scan_step(s):
    from mamba_fused_minimal_b200.kernels.token_scan import _token_scan_step
    out = _token_scan_step(s["state"], s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                           dt_softplus=True, state_indices=s["index"])
    return {"out": out, "state": s["state"]}


# --- the plain forms, in 32 bits

def _norm_parts(s):
    total = s["x"].float()
    if s["residual"] is not None:
        total = total + s["residual"].float()
    rstd = torch.rsqrt((total * total).mean(-1, keepdim=True) + EPS)
    return total, rstd, total * rstd * s["weight"]


def _norm(s):
    total, _, y = _norm_parts(s)
    kind = s["case"]["out"]
    kept = None if s["residual"] is None else total.to(s["residual"].dtype)
    if kind in DTYPES:
        return {"out": y.to(DTYPES[kind]), "residual": kept, "scales": None}
    most = 448.0 if kind == "e4m3" else 127.0
    scales = y.abs().amax(-1, keepdim=True) / most
    q = y / scales
    q = q.to(torch.float8_e4m3fn) if kind == "e4m3" else torch.round(q).to(torch.bfloat16)
    return {"out": q, "residual": kept, "scales": scales.squeeze(-1)}


def _norm_train(s):
    total, _, y = _norm_parts(s)
    kept = total.to(s["residual"].dtype)
    # the gradient at what was kept: y_i = w_i t_i r, r = (mean t^2 + eps)^(-1/2)
    t = kept.float()
    r = torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)
    dout = s["dout"].float()
    hat = t * r
    wd = dout * s["weight"]
    grad = (wd - hat * (wd * hat).mean(-1, keepdim=True)) * r + s["dresidual"].float()
    dweight = (dout * hat).sum((0, 1), dtype=torch.float64).float()
    return {"out": y.to(s["x"].dtype), "residual": kept, "dx": grad.to(s["x"].dtype), "dresidual": grad.to(kept.dtype), "dweight": dweight}


def _silu(v):
    return v / (1 + torch.exp(-v))


def _dsilu(v):
    g = 1 / (1 + torch.exp(-v))
    return g * (1 + v * (1 - g))


def _conv_taps(s):
    """(batch, seqlen, channels, width) of what each position's taps see, and the pre-activation."""
    x, w = s["x"].float(), s["weight"]
    width = w.shape[1]
    lead = x.new_zeros(x.shape[0], width - 1, x.shape[2])
    taps = torch.cat([lead, x], 1).unfold(1, width, 1)
    if s["seq_idx"] is not None:
        at = torch.cat([s["seq_idx"].new_full((x.shape[0], width - 1), -1), s["seq_idx"]], 1).unfold(1, width, 1)
        taps = taps * (at == s["seq_idx"][..., None])[:, :, None, :]
    return taps, (taps * w).sum(-1) + s["bias"]


def _conv(s):
    _, pre = _conv_taps(s)
    x, w = s["x"], s["weight"].shape[1]
    final = torch.cat([x.new_zeros(x.shape[0], w - 1, x.shape[2]), x], 1)[:, -(w - 1):]
    if s["seq_idx"] is not None:
        at = torch.cat([s["seq_idx"].new_full((x.shape[0], w - 1), -1), s["seq_idx"]], 1)[:, -(w - 1):]
        final = final * (at == s["seq_idx"][:, -1:])[..., None]
    return {"out": _silu(pre).to(x.dtype), "final": final.contiguous()}


def _conv_train(s):
    taps, pre = _conv_taps(s)
    dpre = s["dout"].float() * _dsilu(pre)
    width = s["weight"].shape[1]
    dweight = (taps * dpre[..., None]).sum((0, 1), dtype=torch.float64).float()
    dbias = dpre.sum((0, 1), dtype=torch.float64).float()
    # x at position t is seen through tap k by position t + width - 1 - k
    after = torch.cat([dpre, dpre.new_zeros(dpre.shape[0], width - 1, dpre.shape[2])], 1).unfold(1, width, 1).flip(-1)
    if s["seq_idx"] is not None:
        at = torch.cat([s["seq_idx"], s["seq_idx"].new_full((dpre.shape[0], width - 1), -1)], 1).unfold(1, width, 1).flip(-1)
        after = after * (at == s["seq_idx"][..., None])[:, :, None, :]
    dx = (after * s["weight"]).sum(-1)
    return {"out": _silu(pre).to(s["x"].dtype), "dx": dx.to(s["x"].dtype), "dweight": dweight, "dbias": dbias}


def _conv_step(s):
    at = s["index"].long()
    seen = torch.cat([s["state"][at], s["x"][:, None]], 1)
    pre = (seen.float() * s["weight"].t()).sum(1) + s["bias"]
    s["state"][at] = seen[:, 1:]
    return {"out": _silu(pre).to(s["x"].dtype), "state": s["state"]}


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _running(a, u):
    """h[:, t] = a[:, t] h[:, t - 1] + u[:, t], by doubling the reach; a and u are used up."""
    reach = 1
    while reach < a.shape[1]:
        u[:, reach:] = u[:, reach:] + a[:, reach:] * u[:, :-reach]
        a[:, reach:] = a[:, reach:] * a[:, :-reach]
        reach *= 2
    return u


def _scan_parts(s):
    """delta, the decays a and the states h (batch, seqlen, channels, dstate), and y before the gate."""
    x, A = s["x"].float(), s["A"]
    rep = A.shape[0] // s["B"].shape[2]
    delta = _softplus(s["dt"].float() + s["dt_bias"])
    a = torch.exp(delta[..., None] * A)
    if s["seq_idx"] is not None:
        a[:, 1:] *= (s["seq_idx"][:, 1:] == s["seq_idx"][:, :-1])[..., None, None]
    u = (delta * x)[..., None] * s["B"].float().repeat_interleave(rep, 2)
    if s["initial"] is not None:
        u[:, 0] += a[:, 0] * s["initial"]
    h = _running(a.clone(), u)
    y = torch.einsum("bldn,bldn->bld", h, s["C"].float().repeat_interleave(rep, 2)) + s["D"] * x
    return delta, a, h, y


def _scan(s):
    _, _, h, y = _scan_parts(s)
    final = h[:, -1].clone()
    out = y if s["z"] is None else y * _silu(s["z"].float())
    return {"out": out.to(s["x"].dtype), "final": final}


def _scan_train(s):
    x, A, B, C = s["x"].float(), s["A"], s["B"].float(), s["C"].float()
    b, l, d = x.shape
    g, n = B.shape[2:]
    rep = d // g
    delta, a, h, y = _scan_parts(s)
    out, final, dy, dz = y, h[:, -1].clone(), s["dout"].float(), None
    if s["z"] is not None:
        z = s["z"].float()
        out, dz = y * _silu(z), (dy * y * _dsilu(z)).to(s["z"].dtype)
        dy = dy * _silu(z)
    dC = (dy[..., None] * h).view(b, l, g, rep, n).sum(3)
    h[:, 1:] = h[:, :-1].clone()
    h[:, 0] = 0
    carried = a * h                                  # what of the state before reaches position t
    del h
    # gradient of the states, from the last position to the first
    back = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1).flip(1)
    grad = _running(back, (dy[..., None] * C.repeat_interleave(rep, 2)).flip(1)).flip(1)
    gB = (grad * B.repeat_interleave(rep, 2)).sum(-1)
    dB = (grad * (delta * x)[..., None]).view(b, l, g, rep, n).sum(3)
    moved = grad * carried
    ddelta = gB * x + (moved * A).sum(-1)
    dA = (moved * delta[..., None]).sum((0, 1), dtype=torch.float64).float()
    raw = s["dt"].float() + s["dt_bias"]
    ddt = ddelta / (1 + torch.exp(-raw))
    return {"out": out.to(s["x"].dtype), "final": final, "dx": (gB * delta + s["D"] * dy).to(s["x"].dtype), "ddt": ddt.to(s["dt"].dtype),
            "dA": dA, "dB": dB.to(s["B"].dtype), "dC": dC.to(s["C"].dtype), "dD": (dy * x).sum((0, 1), dtype=torch.float64).float(),
            "dz": dz, "dbias": ddt.sum((0, 1), dtype=torch.float64).float()}


def _scan_step(s):
    c = s["case"]
    b, h, p, n = c["batch"], c["heads"], c["headdim"], c["dstate"]
    at = s["index"].long()
    rep = h // c["ngroups"]
    x, z = s["x"].float().view(b, h, p), s["z"].float().view(b, h, p)
    delta = _softplus(s["dt"].float() + s["dt_bias"])[..., None, None]
    A = s["A"].view(h, 1, -1)
    B, C = (s[k].float().repeat_interleave(rep, 1)[:, :, None, :] for k in "BC")
    new = s["state"][at].view(b, h, p, n).float() * torch.exp(delta * A) + delta * x[..., None] * B
    y = (new * C).sum(-1) + s["D"][:, None] * x
    s["state"][at] = new.view(b, *s["state"].shape[1:]).to(s["state"].dtype)
    return {"out": (y * _silu(z)).view(s["x"].shape).to(s["x"].dtype), "state": s["state"]}


# ---------------------------------------------------------------------------------------------------
# the definitions in 64 bits: positions one after another

def exact(case, seed):
    c = case
    s = prepare(c, seed)
    f = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    return {"norm": _exact_norm, "norm_train": _exact_norm_train, "conv": _exact_conv, "conv_train": _exact_conv_train,
            "conv_step": _exact_conv_step, "scan": _exact_scan, "scan_train": _exact_scan_train, "scan_step": _exact_scan_step}[c["op"]](s, f)


def _exact_rows(f):
    t = f["x"] if f["residual"] is None else f["x"] + f["residual"]
    root = torch.sqrt(torch.linalg.vector_norm(t, dim=-1, keepdim=True) ** 2 / t.shape[-1] + EPS)
    return t, root, f["weight"] * (t / root)


def _exact_norm(s, f):
    t, _, y = _exact_rows(f)
    kind = s["case"]["out"]
    kept = None if s["residual"] is None else t
    if kind in DTYPES:
        return {"out": y, "residual": kept, "scales": None}
    scales = torch.maximum(y.amax(-1), -y.amin(-1)) / {"e4m3": 448, "int8": 127}[kind]
    q = y / scales[..., None]
    if kind == "int8":
        return {"out": q.round(), "residual": kept, "scales": scales}
    # four significant bits, none below 2^-9
    unit = torch.exp2(torch.clamp(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -60))), min=-6) - 3)
    return {"out": torch.round(q / unit) * unit, "residual": kept, "scales": scales}


def _exact_norm_train(s, f):
    t, root, y = _exact_rows(f)
    kept = t.to(s["residual"].dtype).double()
    root_k = torch.sqrt((kept ** 2).sum(-1, keepdim=True) / kept.shape[-1] + EPS)
    wd = f["weight"] * f["dout"]
    along = (wd * kept).sum(-1, keepdim=True)
    grad = wd / root_k - kept * along / (kept.shape[-1] * root_k ** 3) + f["dresidual"]
    return {"out": y, "residual": t, "dx": grad, "dresidual": grad, "dweight": torch.einsum("bld,bld->d", f["dout"], kept / root_k)}


def _exact_conv_pre(s, f):
    x, w = f["x"], f["weight"]
    width, l = w.shape[1], x.shape[1]
    pre = f["bias"].expand_as(x).clone()
    for back in range(min(width, l)):
        seen = x[:, :l - back] * w[:, width - 1 - back]
        if s["seq_idx"] is not None:
            seen = torch.where((s["seq_idx"][:, back:] == s["seq_idx"][:, :l - back])[..., None], seen, 0.0)
        pre[:, back:] += seen
    return pre


def _exact_conv(s, f):
    pre = _exact_conv_pre(s, f)
    x, width = f["x"], f["weight"].shape[1]
    b, l, ch = x.shape
    final = x.new_zeros(b, width - 1, ch)
    for back in range(1, min(width, l + 1)):
        last = x[:, l - back]
        if s["seq_idx"] is not None:
            last = torch.where((s["seq_idx"][:, l - back] == s["seq_idx"][:, l - 1])[:, None], last, 0.0)
        final[:, width - 1 - back] = last
    return {"out": pre * torch.sigmoid(pre), "final": final}


def _exact_conv_train(s, f):
    pre = _exact_conv_pre(s, f)
    x, w = f["x"], f["weight"]
    width, l = w.shape[1], x.shape[1]
    g = torch.sigmoid(pre)
    dpre = f["dout"] * (g + pre * g * (1 - g))
    dx, dweight = torch.zeros_like(x), torch.zeros_like(w)
    for back in range(min(width, l)):
        here, there = dpre[:, back:], x[:, :l - back]
        if s["seq_idx"] is not None:
            here = torch.where((s["seq_idx"][:, back:] == s["seq_idx"][:, :l - back])[..., None], here, 0.0)
        dx[:, :l - back] += here * w[:, width - 1 - back]
        dweight[:, width - 1 - back] = torch.einsum("blc,blc->c", here, there)
    return {"out": pre * g, "dx": dx, "dweight": dweight, "dbias": dpre.sum((0, 1))}


def _exact_conv_step(s, f):
    at = s["index"].long()
    old, w = f["state"][at], f["weight"]
    pre = f["bias"] + f["x"] * w[:, -1] + torch.einsum("bkc,ck->bc", old, w[:, :-1])
    state = f["state"].clone()
    state[at, :-1] = old[:, 1:]
    state[at, -1] = f["x"]
    return {"out": pre * torch.sigmoid(pre), "state": state}


def _exact_forward(s, f, keep):
    b, l, d = f["x"].shape
    group = torch.arange(d, device="cuda") // (d // f["B"].shape[2])
    delta = torch.nn.functional.softplus(f["dt"] + f["dt_bias"], threshold=60)
    h = f["initial"] if s["initial"] is not None else f["x"].new_zeros(b, d, f["A"].shape[1])
    y, kept = torch.empty_like(f["x"]), []
    for t in range(l):
        if s["seq_idx"] is not None and t > 0:
            h = h * (s["seq_idx"][:, t] == s["seq_idx"][:, t - 1])[:, None, None]
        if keep:
            kept.append(h)
        h = torch.exp(delta[:, t, :, None] * f["A"]) * h + (delta[:, t] * f["x"][:, t])[..., None] * f["B"][:, t, group]
        y[:, t] = (h * f["C"][:, t, group]).sum(-1)
    return delta, group, kept, h, y + f["D"] * f["x"]


def _exact_scan(s, f):
    if s["case"]["seqlen"] * max(1.0, s["x"].shape[0] * s["A"].numel() / 4e6) > 100_000:
        return None
    _, _, _, h, y = _exact_forward(s, f, False)
    return {"out": y if s["z"] is None else y * f["z"] * torch.sigmoid(f["z"]), "final": h}


def _exact_scan_train(s, f):
    c = s["case"]
    if c["seqlen"] > 25_000 or c["batch"] * c["seqlen"] * c["channels"] * c["dstate"] > 1_000_000_000:
        return None
    delta, group, before, last, y = _exact_forward(s, f, True)
    x, A, B, C = f["x"], f["A"], f["B"], f["C"]
    b, l, d = x.shape
    ng, n = B.shape[2:]
    out, dy, dz = y, f["dout"], None
    if s["z"] is not None:
        gate = torch.sigmoid(f["z"])
        out, dz, dy = y * f["z"] * gate, dy * y * (gate + f["z"] * gate * (1 - gate)), dy * f["z"] * gate
    dx, ddelta = f["D"] * dy, torch.zeros_like(x)
    dA, dB, dC = torch.zeros_like(A), torch.zeros_like(B), torch.zeros_like(C)
    g = x.new_zeros(b, d, n)
    for t in reversed(range(l)):
        a = torch.exp(delta[:, t, :, None] * A)
        u = (delta[:, t] * x[:, t])[..., None]
        Bt, h0 = B[:, t, group], before[t]
        dC[:, t] = (dy[:, t, :, None] * (a * h0 + u * Bt)).view(b, ng, d // ng, n).sum(2)
        g = g + dy[:, t, :, None] * C[:, t, group]
        dB[:, t] = (g * u).view(b, ng, d // ng, n).sum(2)
        through = (g * Bt).sum(-1)
        dx[:, t] += through * delta[:, t]
        moved = g * a * h0
        ddelta[:, t] = through * x[:, t] + (moved * A).sum(-1)
        dA += (moved * delta[:, t, :, None]).sum(0)
        g = g * a
        if s["seq_idx"] is not None and t > 0:
            g = g * (s["seq_idx"][:, t] == s["seq_idx"][:, t - 1])[:, None, None]
    ddt = ddelta * torch.sigmoid(f["dt"] + f["dt_bias"])
    return {"out": out, "final": last, "dx": dx, "ddt": ddt, "dA": dA, "dB": dB, "dC": dC, "dD": torch.einsum("bld,bld->d", dy, x),
            "dz": dz, "dbias": ddt.sum((0, 1))}


def _exact_scan_step(s, f):
    c = s["case"]
    b, h, p, n = c["batch"], c["heads"], c["headdim"], c["dstate"]
    group = torch.arange(h, device="cuda") // (h // c["ngroups"])
    delta = torch.nn.functional.softplus(f["dt"] + f["dt_bias"], threshold=60)
    at = s["index"].long()
    decay = torch.exp(torch.einsum("bh,hn->bhn", delta, f["A"].view(h, -1)))
    x = f["x"].view(b, h, p)
    new = f["state"][at].view(b, h, p, n) * decay[:, :, None, :] + torch.einsum("bhp,bhn->bhpn", x * delta[..., None], f["B"][:, group])
    y = torch.einsum("bhpn,bhn->bhp", new, f["C"][:, group]) + f["D"][None, :, None] * x
    state = f["state"].clone()
    state[at] = new.view(b, *state.shape[1:])
    return {"out": y.view_as(f["x"]) * f["z"] * torch.sigmoid(f["z"]), "state": state}


# ---------------------------------------------------------------------------------------------------
# what a pass cannot do without: every input read once, every output written once

def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] in ("norm", "norm_train"):
        rows = c["batch"] * c["seqlen"]
        n = rows * c["dim"]
        wide = 0 if c["residual"] == "none" else 4 if c["residual"] == "fp32" else size
        if c["op"] == "norm":
            out = size if c["out"] in DTYPES else 1
            return {"bytes": n * (size + 2 * wide + out) + c["dim"] * 4 + (0 if c["out"] in DTYPES else rows * 4), "flops": 6 * n}
        # forward: x, residual in; sum, out out.  gradients: dout, dresidual and the sum in; dx and the residual's out
        return {"bytes": n * (size + 2 * wide + size) + n * (size + 2 * wide + size + wide) + c["dim"] * 8, "flops": 18 * n}
    if c["op"] in ("conv", "conv_train"):
        n = c["batch"] * c["seqlen"] * c["channels"]
        both = c["channels"] * (c["width"] + 1) * 4
        if c["op"] == "conv":
            return {"bytes": 2 * n * size + both + c["batch"] * (c["width"] - 1) * c["channels"] * size, "flops": n * (2 * c["width"] + 4)}
        return {"bytes": 5 * n * size + 3 * both, "flops": n * (8 * c["width"] + 12)}
    if c["op"] == "conv_step":
        n = c["batch"] * c["channels"]
        return {"bytes": n * size * 2 * c["width"] + c["channels"] * (c["width"] + 1) * 4, "flops": n * (2 * c["width"] + 4)}
    if c["op"] in ("scan", "scan_train"):
        n = c["batch"] * c["seqlen"] * c["channels"]
        bc = 2 * c["batch"] * c["seqlen"] * c["ngroups"] * c["dstate"] * size
        ends = c["batch"] * c["channels"] * c["dstate"] * 4 * (2 if c.get("initial") else 1)
        each = n * c["dstate"]
        if c["op"] == "scan":
            return {"bytes": n * size * (4 if c["gate"] else 3) + bc + ends, "flops": 7 * each}
        # forward, then x, dt, dout (z) read again and dx, ddt (dz) written, B and C read and their gradients written
        return {"bytes": n * size * ((4 + 6) if c["gate"] else (3 + 5)) + 3 * bc + ends + 3 * c["channels"] * c["dstate"] * 4, "flops": 25 * each}
    n = c["batch"] * c["heads"] * c["headdim"]
    wide = 4 if c["state"] == "fp32" else size
    return {"bytes": 2 * n * c["dstate"] * wide + n * size * 3 + 2 * c["batch"] * c["ngroups"] * c["dstate"] * size, "flops": 6 * n * c["dstate"]}
