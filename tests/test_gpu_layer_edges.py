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
