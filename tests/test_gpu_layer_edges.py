"""The operators around the scan where their arithmetic has an edge: what a rounding is made of, infinities behind
a border, values near the smallest number, parameters in 16 bits, scratch that is used again and again.

Tolerances as in test_gpu_layer_ops.py, fixed before the first run; what differs is derived at the test."""
import math

import pytest
import torch

from oracle import layer_oracle as L
from test_gpu_layer_ops import TYPES, U, cuda, half_step, maker, norm_err, ops, packed, scan_inputs, within

pytestmark = pytest.mark.gpu

KEYS = ("x", "dt", "A", "B", "C")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,l,d,n,g", [(2, 20, 48, 16, 1), (1, 17, 7, 5, 1), (1, 20, 24, 64, 2), (1, 20, 33, 8, 1), (1, 12, 9, 256, 1)])
def test_gate_gradient_is_rounded_once(cuda_device, dtype, b, l, d, n, g):
    """dz = dout y silu'(z) element by element: y may be off by what 66 u a position allows, the gate's derivative
    by 80 u of its terms' absolute values, and one rounding of the result stands on top."""
    scan = ops()[2]
    inp = scan_inputs(b, l, d, n, g, dtype, 70 + l)
    pos = [inp[k] for k in KEYS]
    _, _, y, size = L.token_scan(*pos, D=inp["D"], z=inp["z"], dt_bias=inp["dt_bias"], dt_softplus=True)
    dout = maker(71)(b, l, d, dtype=dtype)
    z = inp["z"].double()
    s = torch.sigmoid(z)
    ref = dout.double() * y * s * (1 + z * (1 - s))
    terms = (dout.double() * s * (1 + z.abs() * (1 - s))).abs()
    dpos = cuda(*pos)
    kw = {k: inp[k].to("cuda") for k in ("D", "z", "dt_bias")}
    _, _, saved = scan._token_scan_fwd(*dpos, dt_softplus=True, for_backward=True, **kw)
    dz = scan._token_scan_bwd(dout.to("cuda"), *dpos, saved, dt_softplus=True, **kw)[6]
    within(dz, ref, size * terms, (66 * l + 80) * U, dtype)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("where", ["dout", "C", "z", "dt", "dfinal"])
@pytest.mark.parametrize("b,l,d,n,cuts", [(2, 61, 20, 16, (22, 45)), (1, 61, 9, 64, (33, 34)), (1, 1700, 24, 16, (301, 1600)), (1, 1700, 24, 8, (512, 1111))])
def test_gradients_of_a_sequence_see_no_later_one(cuda_device, bad, where, b, l, d, n, cuts):
    """Packed sequences: an infinity or a NaN of the last one leaves the bits of the others' gradients, for rows
    that one block walks and rows that are cut into segments, with borders at even and odd positions."""
    scan = ops()[2]
    inp = {k: v.to("cuda") for k, v in scan_inputs(b, l, d, n, 1, torch.float32, 72).items()}
    seq = torch.zeros(b, l, dtype=torch.int32, device="cuda")
    for c in cuts:
        seq[:, c:] += 1
    r = maker(73)
    inp |= dict(dout=r(b, l, d).to("cuda"), dfinal=r(b, d, n).to("cuda"), init=r(b, d, n).to("cuda"))

    def grads(v):
        kw = dict(D=v["D"], z=v["z"], dt_bias=v["dt_bias"], dt_softplus=True, initial_states=v["init"], seq_idx=seq)
        pos = [v[k] for k in KEYS]
        _, _, saved = scan._token_scan_fwd(*pos, for_backward=True, **kw)
        return scan._token_scan_bwd(v["dout"], *pos, saved, dfinal_states=v["dfinal"], **kw)

    poisoned = dict(inp)
    poisoned[where] = inp[where].clone()
    if where == "dfinal":
        poisoned[where][:, :, n // 2] = bad
    else:
        poisoned[where][:, cuts[-1]:cuts[-1] + 3] = bad
        poisoned[where][:, -1] = bad
    good, got = grads(inp), grads(poisoned)
    names = ("dx", "ddt", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dinitial")
    for i in (0, 1, 3, 4, 6):
        assert torch.isfinite(good[i]).all() and torch.equal(got[i][:, :cuts[-1]], good[i][:, :cuts[-1]]), names[i]
    assert torch.equal(got[8], good[8]) and torch.isfinite(good[8]).all()


@pytest.mark.parametrize("dim", [96, 97, 2560, 33024])
@pytest.mark.parametrize("kind,most", [(torch.int8, 127.0), (torch.float8_e4m3fn, 448.0)])
@pytest.mark.parametrize("dtype", TYPES[:2])
def test_norm_in_8_bits_of_tiny_rows(cuda_device, dim, kind, most, dtype):
    """Rows whose largest |y| lies between 1 and the smallest numbers, through small weights and through small rows
    under eps: what the codes stand for.  On top of test_norm_forward's bound half a unit of the smallest numbers,
    2^-150, for y itself and, |code| times, for the scale that is kept."""
    fwd = ops()[0]._add_rms_norm_fwd
    x = maker(74)(12, dim)
    x[1], x[2], x[11] = 0, x[2] * 1e15, x[11] * 1e-15
    for i, p in enumerate((8, 20, 30, 33, 35, 36, 37)):
        x[3 + i] *= 10.0 ** -p
    x = x.to(dtype)
    tol = (dim / 64 + 16) * U
    for power in (0, 12, 20, 30, 34, 35, 36, 37):
        w = (1 + 0.1 * maker(75)(dim)) * 10.0 ** -power
        y, _ = L.add_rms_norm(x, w)
        q, _, _, sc = fwd(*cuda(x, w), out_dtype=kind)
        q, sc = q.cpu().float().double(), sc.cpu().double()
        assert torch.isfinite(q).all() and torch.isfinite(sc).all()
        assert (q[1] == 0).all() and sc[1] == 0
        ref_sc = y.abs().amax(-1) / most
        assert ((sc - ref_sc).abs() <= (tol + 2 * U) * ref_sc + 2.0 ** -149).all()
        rows = ref_sc >= 2.0 ** -135                   # below it the scale itself has lost its digits
        step = ref_sc[:, None] * 0.5 if kind is torch.int8 else torch.maximum(y.abs() * 2.0 ** -4, ref_sc[:, None] * 2.0 ** -10)
        bound = step * (1 + 1e-5) + (tol + 4 * U) * y.abs() * 17 + (q.abs() + 1) * 2.0 ** -149
        # a scale of so few digits may round down: the largest codes end at `most`
        bound = bound + (2.0 ** -149 / ref_sc.clamp_min(2.0 ** -149))[:, None] * y.abs()
        bad = ((q * sc[:, None] - y).abs() > bound)[rows]
        assert not bad.any(), (power, bad.any(-1).nonzero().flatten().tolist())
        top = q.abs().amax(-1)
        assert (top[rows & (ref_sc > 0)] == most).all(), (power, top.tolist())


def test_conv_gradients_refuse_wide_filters(cuda_device):
    _, conv, _ = ops()
    for width in (1, 5, 9, 17):
        x, w = torch.zeros(2, 40, 64, device="cuda"), torch.zeros(64, width, device="cuda")
        with pytest.raises(RuntimeError, match="not 2, 3 or 4"):
            conv._short_conv_bwd(x, x, w)


def in_pieces(scan, dout, dfinal, pos, kw, size):
    """Forward and gradients of a sequence piece by piece, each from the state the one before it left."""
    pieces, state = [], kw["initial_states"]
    l = dout.shape[1]
    cut = lambda t, lo, hi: t if t is None or t.dim() < 3 else t[:, lo:hi]  # noqa: E731
    for lo in range(0, l, size):
        hi = min(l, lo + size)
        p = [cut(t, lo, hi) for t in pos]
        k = dict(kw, z=cut(kw["z"], lo, hi), initial_states=state)
        out, state, saved = scan._token_scan_fwd(*p, for_backward=True, **k)
        pieces.append((lo, hi, p, k, saved, out))
    grads, g = [], dfinal
    for lo, hi, p, k, saved, _ in reversed(pieces):
        grads.insert(0, scan._token_scan_bwd(dout[:, lo:hi], *p, saved, dfinal_states=g, **k))
        g = grads[0][8]
    join = lambda i: None if grads[0][i] is None else torch.cat([t[i] for t in grads], 1)  # noqa: E731
    total = lambda i: sum(t[i].double() for t in grads)  # noqa: E731
    return [join(0), join(1), total(2), join(3), join(4), total(5), join(6), total(7), g]


@pytest.mark.parametrize("dtype,b,l,d,n,g,piece", [
    (torch.float32, 1, 300, 1024, 256, 1, 96),           # many channel blocks: a few positions at a time
    (torch.bfloat16, 3, 437, 600, 200, 2, 112),          # the batch, too, in parts
    (torch.bfloat16, 1, 17001, 32, 256, 1, 4096),        # few channels, long: segments within each range
])
def test_scan_gradients_of_long_states_in_ranges(cuda_device, dtype, b, l, d, n, g, piece):
    """Problems whose channel blocks' shares of dB and dC do not fit the scratch at once, against the same sequence
    in pieces that do: the same sums, cut elsewhere.  Per tensor 64 u sqrt(l), and half a step where it is kept
    in 16 bits (once for each side)."""
    scan = ops()[2]
    inp = {k: v.to("cuda") for k, v in scan_inputs(b, l, d, n, g, dtype, 76).items()}
    r = maker(77)
    dout, dfinal, init = r(b, l, d, dtype=dtype).to("cuda"), r(b, d, n).to("cuda"), r(b, d, n).to("cuda")
    pos = [inp[k] for k in KEYS]
    kw = dict(D=inp["D"], z=inp["z"], dt_bias=inp["dt_bias"], dt_softplus=True, initial_states=init)
    _, _, saved = scan._token_scan_fwd(*pos, for_backward=True, **kw)
    got = scan._token_scan_bwd(dout, *pos, saved, dfinal_states=dfinal, **kw)
    again = scan._token_scan_bwd(dout, *pos, saved, dfinal_states=dfinal, **kw)
    ref = in_pieces(scan, dout, dfinal, pos, kw, piece)
    names = ("dx", "ddt", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dinitial")
    for name, a, a2, e in zip(names, got, again, ref):
        step = 2 * half_step(dtype) if name in ("dx", "ddt", "dB", "dC", "dz") else 0
        assert torch.equal(a, a2) and norm_err(a, e.double().cpu()) <= 4 * 64 * U * math.sqrt(l) + step, name


def test_scan_gradients_in_ranges_against_the_oracle(cuda_device):
    """The same against autograd through the 64-bit definition, with packed sequences, a gradient of the last
    state and none."""
    scan = ops()[2]
    b, l, d, n = 1, 300, 1024, 256
    inp = {k: v.to("cuda") for k, v in scan_inputs(b, l, d, n, 1, torch.float32, 78).items()}
    r = maker(79)
    dout, dfinal, init = r(b, l, d).to("cuda"), r(b, d, n).to("cuda"), r(b, d, n).to("cuda")
    seq = packed(b, l, 5).to("cuda")
    kw = dict(D=inp["D"], dt_bias=inp["dt_bias"], initial_states=init)
    leaves = [inp[k].double().requires_grad_() for k in KEYS]
    lkw = {k: v.double().requires_grad_() for k, v in kw.items()}
    for s, df in ((None, dfinal), (seq, None)):
        for t in (*leaves, *lkw.values()):
            t.grad = None
        out, last, _, _ = L.token_scan(*leaves, dt_softplus=True, seq_idx=s, **lkw)
        ((out * dout.double()).sum() + (0 if df is None else (last * df.double()).sum())).backward()
        pos = [inp[k] for k in KEYS]
        _, _, saved = scan._token_scan_fwd(*pos, dt_softplus=True, seq_idx=s, for_backward=True, **kw)
        g = scan._token_scan_bwd(dout, *pos, saved, dt_softplus=True, seq_idx=s, dfinal_states=df, **kw)
        for a, t in zip((*g[:6], g[7], g[8]), (*leaves, lkw["D"], lkw["dt_bias"], lkw["initial_states"])):
            assert norm_err(a, t.grad.cpu()) <= 4 * 64 * U * math.sqrt(l)


def test_chunk_kernels_outputs_pass_the_dispatcher(cuda_device):
    """Dispatch modes see the outputs that the chunk kernels' calls allocate."""
    from torch.utils._python_dispatch import TorchDispatchMode
    from mamba_fused_minimal_b200.kernels.ssd_chunk_state import _chunk_cumsum_fwd

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.shapes = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            if func.overloadpacket in (torch.ops.aten.empty, torch.ops.aten.empty_strided):
                self.shapes.append(tuple(out.shape))
            return out

    dt, A = torch.rand(2, 64, 4, device="cuda"), -torch.rand(4, device="cuda")
    with Seen() as seen:
        outs = _chunk_cumsum_fwd(dt, A, 32)
    for t in outs:
        assert tuple(t.shape) in seen.shapes


def test_growing_states_across_segments(cuda_device):
    """Positive A: over a segment the decay passes the largest number, where the state it multiplies is zero.  Few
    channels and a long row are cut into segments; the result is the one of the definition."""
    scan = ops()[2]
    b, l, d, n = 1, 1700, 8, 16
    r = maker(80)
    x, dout = r(b, l, d), r(b, l, d)
    x[:, :l - 20] = 0
    dout[:, 20:] = 0
    dt, A = torch.ones(b, l, d), torch.full((d, n), 0.5)
    B, C = r(b, l, 1, n), r(b, l, 1, n)
    leaves = [t.double().requires_grad_() for t in (x, dt, A, B, C)]
    out, last, _, size = L.token_scan(*leaves)
    pos = cuda(x, dt, A, B, C)
    got, fin, saved = scan._token_scan_fwd(*pos, for_backward=True)
    # 20 positions count, each with the sum of 16 terms
    within(got, out.detach(), size, 66 * 20 * U, torch.float32)
    assert norm_err(fin, last) <= 66 * 20 * U
    g = scan._token_scan_bwd(dout.to("cuda"), *pos, saved)
    # x is zero wherever the gradient reaches: only dx is not zero
    (out * dout.double()).sum().backward()
    assert all(torch.isfinite(t).all() for t in g if t is not None)
    assert norm_err(g[0], leaves[0].grad) <= 66 * 20 * U
    assert all((t == 0).all() for t in (g[1], g[2], g[3], g[4]))


P16 = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("ptype", P16)
@pytest.mark.parametrize("dim", [96, 97, 33024])
def test_norm_weight_in_16_bits(cuda_device, ptype, dim):
    norm = ops()[0]
    r = maker(81)
    x, w, dout = r(5, dim, dtype=torch.bfloat16), (1 + 0.1 * r(dim)).to(ptype), r(5, dim, dtype=torch.bfloat16)
    y, _ = L.add_rms_norm(x, w)
    tol = (dim / 64 + 32) * U
    out, _, rstd, _ = norm._add_rms_norm_fwd(*cuda(x, w))
    within(out, y, y.abs(), tol, torch.bfloat16)
    xd, wd = x.double().requires_grad_(), w.double().requires_grad_()
    (L.add_rms_norm(xd, wd)[0] * dout.double()).sum().backward()
    dx, _, dw = norm._add_rms_norm_bwd(*cuda(dout, x, w), rstd)
    size = xd.grad.abs() + (dout.double() * wd).abs().detach() * rstd.double().cpu()[:, None]
    within(dx, xd.grad, size, tol, torch.bfloat16)
    assert dw.dtype == torch.float32
    within(dw, wd.grad, (dout.double() * x.double() * rstd.double().cpu()[:, None]).abs().sum(0), tol, torch.float32)
    # the weight is widened exactly: the bits of the same weight in fp32
    for kind in (None, torch.int8, torch.float8_e4m3fn):
        a, b = (norm._add_rms_norm_fwd(x.to("cuda"), v.to("cuda"), out_dtype=kind)[0] for v in (w, w.float()))
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("ptype", P16)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels,width", [(72, 4), (13, 3), (70, 2)])
def test_conv_parameters_in_16_bits(cuda_device, ptype, dtype, channels, width):
    """16-bit filters and biases are widened exactly: the bits of the same ones in fp32, which the other tests
    hold against the oracle."""
    conv = ops()[1]
    r = maker(82)
    x, w, bias = r(2, 37, channels, dtype=dtype).to("cuda"), r(channels, width).to(ptype).to("cuda"), r(channels).to(ptype).to("cuda")
    state = r(2, width - 1, channels, dtype=dtype).to("cuda")

    def work(w, bias):
        out, fin = conv._short_conv_fwd(x, w, bias=bias, initial_states=state, return_final_states=True)
        st = state.clone()
        step = conv._short_conv_step(x[:, 0], st, w, bias=bias)
        return [out, fin, step, st, *conv._short_conv_bwd(x, x, w, bias=bias, initial_states=state)]

    for a, b in zip(work(w, bias), work(w.float(), bias.float())):
        assert a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("ptype", P16)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,l,d,n,g", [(2, 40, 48, 16, 1), (1, 1500, 10, 5, 2), (1, 33, 24, 64, 1)])
def test_scan_parameters_in_16_bits(cuda_device, ptype, dtype, b, l, d, n, g):
    """A, D, dt_bias and the initial states in 16 bits: the bits of the same ones in fp32."""
    scan = ops()[2]
    inp = {k: v.to("cuda") for k, v in scan_inputs(b, l, d, n, g, dtype, 83).items()}
    for k in ("A", "D", "dt_bias"):
        inp[k] = inp[k].to(ptype)
    init = maker(84)(b, d, n).to(ptype).to("cuda")
    dout = maker(85)(b, l, d, dtype=dtype).to("cuda")

    def work(wide):
        f = (lambda t: t.float()) if wide else (lambda t: t)
        pos = [inp["x"], inp["dt"], f(inp["A"]), inp["B"], inp["C"]]
        kw = dict(D=f(inp["D"]), z=inp["z"], dt_bias=f(inp["dt_bias"]), dt_softplus=True)
        out, fin, saved = scan._token_scan_fwd(*pos, for_backward=True, initial_states=f(init), **kw)
        gr = scan._token_scan_bwd(dout, *pos, saved, initial_states=f(init), **kw)
        st = init.float()
        tok = scan._token_scan_step(st, inp["x"][:, 0], inp["dt"][:, 0], pos[2], inp["B"][:, 0], inp["C"][:, 0], D=kw["D"], z=inp["z"][:, 0],
                                    dt_bias=kw["dt_bias"], dt_softplus=True)
        return [out, fin, *gr, tok, st]

    for a, c in zip(work(False), work(True)):
        assert a.dtype == c.dtype and torch.equal(a, c)


@pytest.mark.parametrize("ptype", P16)
@pytest.mark.parametrize("headdim,n", [(64, 128), (8, 16), (33, 20)])
def test_step_parameters_in_16_bits_per_head(cuda_device, ptype, headdim, n):
    scan = ops()[2]
    r = maker(86)
    b, h = 3, 4
    x, dt, B, C = (r(b, *s, dtype=torch.bfloat16).to("cuda") for s in ((h, headdim), (h,), (1, n), (1, n)))
    A, D, bias = (-torch.rand(h, generator=torch.Generator().manual_seed(1))).to(ptype).to("cuda"), r(h).to(ptype).to("cuda"), r(h).to(ptype).to("cuda")
    state = r(b, h, headdim, n).to("cuda")
    outs = []
    for f in (lambda t: t, lambda t: t.float()):
        st = state.clone()
        outs.append((scan._token_scan_step(st, x, dt, f(A), B, C, D=f(D), dt_bias=f(bias), dt_softplus=True), st))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_gradients_of_a_sequence_see_no_earlier_one(cuda_device):
    """Packed sequences, the other way: an infinity or a NaN of an earlier sequence, and initial states that no position
    sees, leave the bits of the later ones' gradients; scan and convolution, short rows and segments."""
    _, conv, scan = ops()
    r = maker(90)
    for b, l, d, n, cut in ((2, 61, 20, 16, 33), (1, 1700, 24, 8, 801)):
        inp = {k: v.to("cuda") for k, v in scan_inputs(b, l, d, n, 1, torch.float32, 91).items()}
        seq = torch.zeros(b, l, dtype=torch.int32, device="cuda")
        seq[:, cut:] = 1
        inp |= dict(dout=r(b, l, d).to("cuda"), init=r(b, d, n).to("cuda"), cinit=r(b, 3, d).to("cuda"), w=r(d, 4).to("cuda"))

        def work(v, seq):
            kw = dict(D=v["D"], z=v["z"], dt_bias=v["dt_bias"], dt_softplus=True, initial_states=v["init"], seq_idx=seq)
            pos = [v[k] for k in KEYS]
            out, fin, saved = scan._token_scan_fwd(*pos, for_backward=True, **kw)
            g = scan._token_scan_bwd(v["dout"], *pos, saved, **kw)
            ckw = dict(bias=v["D"], initial_states=v["cinit"], seq_idx=seq)
            c, cf = conv._short_conv_fwd(v["x"], v["w"], return_final_states=True, **ckw)
            cg = conv._short_conv_bwd(v["dout"], v["x"], v["w"], dfinal_states=inp["cinit"], **ckw)
            return [t[:, cut:] for t in (out, g[0], g[1], g[3], g[4], g[6], c, cg[0])] + [fin, cf], [g[2], g[5], g[7], g[8], cg[1], cg[2], cg[3]]

        good, _ = work(inp, seq)
        for bad in (float("nan"), float("inf")):
            for key in ("x", "dt", "B", "C", "z", "dout", "init", "cinit"):
                v = dict(inp)
                v[key] = inp[key].clone()
                v[key][:, :3] = bad
                if key not in ("init", "cinit"):
                    v[key][:, cut - 2:cut] = bad
                for a, c in zip(work(v, seq)[0], good):
                    assert torch.equal(a, c), (key, bad)
        # rows that do not begin with sequence 0 see nothing of the initial states, and hand nothing back to them
        v = dict(inp, init=torch.full_like(inp["init"], float("nan")), cinit=torch.full_like(inp["cinit"], float("nan")))
        a, b_ = work(inp, seq + 1), work(v, seq + 1)
        for p, q in zip((*a[0], *a[1]), (*b_[0], *b_[1])):
            assert torch.equal(p, q)
        assert (a[1][3] == 0).all() and (a[1][6] == 0).all()


def test_scan_gradients_in_ranges_captured_and_on_another_stream(cuda_device):
    """The launches of a problem that is walked in ranges as one graph, replayed with other inputs, beside an eager call
    on another stream."""
    scan = ops()[2]
    b, l, d, n = 1, 300, 1024, 256

    def inputs(seed):
        v = {k: t.to("cuda") for k, t in scan_inputs(b, l, d, n, 1, torch.bfloat16, seed).items()}
        v["dout"] = maker(seed + 1)(b, l, d, dtype=torch.bfloat16).to("cuda")
        return v

    def work(v):
        pos = [v[k] for k in KEYS]
        kw = dict(D=v["D"], z=v["z"], dt_bias=v["dt_bias"], dt_softplus=True)
        _, _, saved = scan._token_scan_fwd(*pos, for_backward=True, **kw)
        return [t for t in scan._token_scan_bwd(v["dout"], *pos, saved, **kw) if t is not None]

    first, second = inputs(92), inputs(94)
    want = [[t.clone() for t in work(v)] for v in (first, second)]
    static, stream = {k: t.clone() for k, t in first.items()}, torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work(static)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(static)
    for k, t in second.items():
        static[k].copy_(t)
    stream.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        graph.replay()
        with torch.cuda.stream(stream):
            eager = work(first)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(outs, want[1]))
    assert all(torch.equal(a, c) for a, c in zip(eager, want[0]))
