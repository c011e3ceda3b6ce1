"""The operators around the scan on the GPU against the 64-bit oracle.

Tolerances, fixed before the first run.  u = 2^-24.  A result stored in type t carries at most half a step,
h(t) = eps(t) / 2 relative to the value.  On top of it stands what the fp32 computation may be off:

* norm: a sum of dim squares, a reciprocal root and three products: at most (dim / 64 + 16) u relative to y
  (a block adds at most dim / 64 terms one after another on top of its tree);
* convolution: at most 5 products and sums, and the gate's exponential, whose relative error is at most
  (2 + |pre|) * 4u: with |pre| <= 16 that is 80 u relative to the sum of the terms' absolute values;
* scan: a decay exp(dt' A) is off by at most 64 u relative (exponential 4 u, dt' 4 u times an exponent of at
  most 8, beyond which the term has vanished below e^-8; products), a step adds at most 2 u: after l
  positions (64 + 2) l u relative to the sum of the terms' absolute values, `size` of the oracle.
* gradients: the same sums once more, over channels or positions: the bound is applied to the 2-norm, for
  which independent roundings add up like a root: 64 u sqrt(l) + h(t), times 2 for the gate's saved output
  (itself rounded to its type).
"""
import math

import pytest
import torch

from oracle import layer_oracle as L

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype != torch.float32 else U


def ops():
    from mamba_fused_minimal_b200.kernels import add_rms_norm, short_conv, token_scan
    return add_rms_norm, short_conv, token_scan


def within(got, ref, size, tol, dtype):
    """|got - ref| <= tol * size + half a step of the stored value (and of the smallest number of its type)."""
    got = got.double().cpu()
    tiny = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[dtype]
    bound = tol * size + half_step(dtype) * (ref.abs() + tol * size) + tiny
    bad = ~((got - ref).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {((got - ref).abs() / bound).max().item():.3g} of the bound"


def norm_err(got, ref):
    got, ref = got.detach().double().cpu(), ref.detach()
    return ((got - ref).norm() / ref.norm().clamp_min(1e-300)).item()


def cuda(*ts):
    return [None if t is None else t.to("cuda") for t in ts]


def maker(seed):
    gen = torch.Generator().manual_seed(seed)
    return lambda *s, dtype=torch.float32: torch.randn(*s, generator=gen).to(dtype)


# ---------------------------------------------------------------------------------------------- norm
NORM_DIMS = [1, 7, 64, 257, 2560, 8200, 20001, 33024]


@pytest.mark.parametrize("dim", NORM_DIMS)
@pytest.mark.parametrize("dtype,rtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                         (torch.float16, torch.float16), (torch.float16, torch.float32), (torch.bfloat16, None)])
def test_norm_forward(cuda_device, dim, dtype, rtype):
    fwd = ops()[0]._add_rms_norm_fwd
    r = maker(dim)
    x, w = r(2, 3, dim, dtype=dtype), 1 + 0.1 * r(dim)
    res = None if rtype is None else 2 * r(2, 3, dim, dtype=rtype)
    y, t = L.add_rms_norm(x, w, res)
    xc, wc, rc = cuda(x, w, res)
    out, total, rstd, scales = fwd(xc, wc, residual=rc)
    tol = (dim / 64 + 16) * U
    assert scales is None and out.dtype == dtype and rstd.shape == (2, 3)
    within(out, y, y.abs(), tol, dtype)
    if res is None:
        assert total is None
        kept = x.double()
    else:
        assert total.dtype == rtype
        within(total, t, t.abs(), U, rtype)
        kept = total.double().cpu()
    ref_r = 1 / torch.sqrt((kept ** 2).mean(-1) + 1e-5)
    within(rstd, ref_r, ref_r.abs(), tol, torch.float32)
    # 8 bits: the value a code stands for is off by half a step of the code and by its scale
    for kind, most in ((torch.int8, 127.0), (torch.float8_e4m3fn, 448.0)):
        q, total8, _, sc = fwd(xc, wc, residual=rc, out_dtype=kind)
        assert q.dtype == kind and q.shape == x.shape and sc.shape == (2, 3)
        ref_sc = y.abs().amax(-1) / most
        within(sc, ref_sc, ref_sc, tol + 2 * U, torch.float32)
        val = q.to(torch.float32).double().cpu() * sc.double().cpu()[..., None]
        step = ref_sc[..., None] * 0.5 if kind is torch.int8 else torch.maximum(y.abs() * 2.0 ** -4, ref_sc[..., None] * 2.0 ** -10)
        assert ((val - y).abs() <= step * (1 + 1e-5) + (tol + 4 * U) * y.abs() * 17).all()
        if total is not None:
            assert torch.equal(total8, total)


def test_norm_first_layer_keeps_x_in_32_bits(cuda_device):
    x, w = maker(5)(3, 65, dtype=torch.bfloat16), torch.ones(65)
    out, total, _, _ = ops()[0]._add_rms_norm_fwd(*cuda(x, w), residual_dtype=torch.float32)
    assert total.dtype == torch.float32 and torch.equal(total.cpu(), x.float())
    assert out.shape == (3, 65)


@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
def test_norm_odd_rows_in_8_bits(cuda_device, kind):
    """A row of zeros has scale 0 and codes 0; infinities and NaN make the scale NaN and leave their
    neighbours alone; the smallest and the largest values keep finite scales."""
    x = maker(6)(6, 96)
    x[0] = 0
    x[1, 5] = float("inf")
    x[2, 95] = float("nan")
    x[3] *= 1e-22
    x[4] *= 1e15
    q, _, rstd, sc = ops()[0]._add_rms_norm_fwd(*cuda(x, torch.ones(96)), out_dtype=kind, eps=0.0)
    q2, _, _, sc2 = ops()[0]._add_rms_norm_fwd(*cuda(x[5:], torch.ones(96)), out_dtype=kind, eps=0.0)
    sc, q = sc.cpu(), q.cpu()
    assert sc[1].isnan() and sc[2].isnan()
    assert torch.equal(q[5:].view(torch.uint8), q2.cpu().view(torch.uint8)) and torch.equal(sc[5:], sc2.cpu())
    q0, _, _, sc0 = ops()[0]._add_rms_norm_fwd(*cuda(torch.zeros(1, 96), torch.ones(96)), out_dtype=kind)
    assert sc0.item() == 0 and (q0.float() == 0).all()
    # tiny weights: y far below the smallest scale's reciprocal
    q1, _, _, sc1 = ops()[0]._add_rms_norm_fwd(*cuda(x[5:], torch.full((96,), 1e-37)), out_dtype=kind)
    assert torch.isfinite(sc1).all() and torch.isfinite(q1.float()).all()


def test_norm_strided_rows(cuda_device):
    """Rows that are column ranges of a wider buffer, an odd offset among them (the scalar route), and a
    batch stride that is not seqlen rows."""
    fwd = ops()[0]._add_rms_norm_fwd
    buf = maker(7)(4, 9, 200, dtype=torch.bfloat16).to("cuda")
    w = torch.ones(64, device="cuda")
    for view in (buf[:, 2:7, 8:72], buf[1:3, :, 3:67], buf.transpose(0, 1)[:, :, 16:80], buf[0, :, 5:69]):
        a = fwd(view, w, residual=view)
        b = fwd(view.contiguous(), w, residual=view.contiguous())
        assert all(torch.equal(p, q) for p, q in zip(a[:2], b[:2]))


@pytest.mark.parametrize("rows,dim", [(400, 64), (1300, 743), (700, 744), (310, 4097), (900, 2560)])
def test_norm_gradients_of_many_rows(cuda_device, rows, dim):
    """More rows than blocks: rows one after another in a block, and its share of the weight's gradient."""
    bwd = ops()[0]._add_rms_norm_bwd
    r = maker(rows)
    total, w, dout = 2 * r(rows, dim, dtype=torch.bfloat16), 1 + 0.1 * r(dim), r(rows, dim, dtype=torch.bfloat16)
    td, wd = total.double().requires_grad_(), w.double().requires_grad_()
    (L.add_rms_norm(td, wd)[0] * dout.double()).sum().backward()
    rstd = (1 / torch.sqrt((total.double() ** 2).mean(-1) + 1e-5)).float()
    dx, _, dw = bwd(*cuda(dout, total, w, rstd))
    size = td.grad.abs() + (dout.double() * wd).abs().detach() * rstd.double()[:, None]
    within(dx, td.grad, size, (dim / 64 + 32) * U, torch.bfloat16)
    terms = (dout.double() * td.detach() * rstd.double()[:, None]).abs().sum(0)
    # at most rows / blocks terms one after another, the blocks' shares in strides of 32
    within(dw, wd.grad, terms, (rows / 148 + 64) * U, torch.float32)


@pytest.mark.parametrize("dim", [1, 33, 256, 4097, 9000, 16384, 20001])
@pytest.mark.parametrize("dtype,stype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
def test_norm_gradients(cuda_device, dim, dtype, stype):
    bwd = ops()[0]._add_rms_norm_bwd
    r = maker(dim + 1)
    total, w = 2 * r(3, 5, dim, dtype=stype), 1 + 0.1 * r(dim)
    dout, dres = r(3, 5, dim, dtype=dtype), r(3, 5, dim, dtype=stype)
    td, wd = total.double().requires_grad_(), w.double().requires_grad_()
    y, _ = L.add_rms_norm(td, wd)
    (y * dout.double()).sum().backward()
    rstd = (1 / torch.sqrt((total.double() ** 2).mean(-1) + 1e-5)).float()
    args = cuda(dout, total, w, rstd, dres)
    dx, din, dw = bwd(*args)
    ref = td.grad + dres.double()
    size = ref.abs() + (td.grad.abs() + (dout.double() * wd).abs().detach() / torch.sqrt((td.detach() ** 2).mean(-1, keepdim=True) + 1e-5))
    tol = (dim / 64 + 32) * U
    within(dx, ref, size, tol, dtype)
    within(din, ref, size, tol, stype)
    assert din.dtype == stype and dx.dtype == dtype and ((din is dx) or stype != dtype)
    terms = (dout.double() * td.detach() * rstd.double()[..., None]).abs().sum((0, 1))
    within(dw, wd.grad, terms, 32 * U, torch.float32)
    again = bwd(*args)
    assert all(torch.equal(a, b) for a, b in zip((dx, din, dw), again))
    dx0, _, _ = bwd(*args[:4])
    within(dx0, td.grad, size, tol, dtype)


# ---------------------------------------------------------------------------------------------- conv
def packed(b, l, seed, first=0):
    gen = torch.Generator().manual_seed(seed)
    cut = torch.rand(b, l, generator=gen) < 0.15
    cut[:, 0] = False
    return (cut.cumsum(1) + first).to(torch.int32)


CONV_CASES = [
    # batch, seqlen, channels, width, silu, bias, init, seq
    (2, 70, 64, 4, True, True, True, False),
    (1, 1, 8, 4, True, True, True, False),
    (3, 2, 24, 4, True, False, False, False),
    (2, 3, 16, 2, False, True, True, True),
    (2, 131, 40, 3, True, True, True, True),
    (1, 65, 7, 4, True, True, False, True),
    (2, 33, 1033, 4, False, False, True, False),
    (1, 129, 1544, 4, True, True, True, True),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CONV_CASES)
def test_conv_forward_and_gradients(cuda_device, dtype, case):
    b, l, c, width, silu, has_bias, has_init, has_seq = case
    _, conv, _ = ops()
    r = maker(l * c)
    x, w = r(b, l, c, dtype=dtype), 0.5 * r(c, width)
    bias = 0.5 * r(c) if has_bias else None
    init = r(b, width - 1, c, dtype=dtype) if has_init else None
    seq = packed(b, l, l) if has_seq else None
    dout, dfin = r(b, l, c, dtype=dtype), r(b, width - 1, c, dtype=dtype)
    leaves = [None if t is None else t.double().requires_grad_() for t in (x, w, bias, init)]
    out, fin = L.short_conv(leaves[0], leaves[1], leaves[2], silu, leaves[3], seq)
    size, _ = L.short_conv(x.abs(), w.abs(), None if bias is None else bias.abs(), False, None if init is None else init.abs(), seq)
    assert size.max() <= 16
    xc, wc, bc, ic, sc, dc, fc = cuda(x, w, bias, init, seq, dout, dfin)
    got, gfin = conv._short_conv_fwd(xc, wc, bias=bc, apply_silu=silu, initial_states=ic, seq_idx=sc, return_final_states=True)
    within(got, out.detach(), size, 80 * U, dtype)
    assert torch.equal(gfin.double().cpu(), fin.detach())
    none, nofin = conv._short_conv_fwd(xc, wc, bias=bc, apply_silu=silu, initial_states=ic, seq_idx=sc)
    assert nofin is None and torch.equal(none, got)

    ((out * dout.double()).sum() + (fin * dfin.double()).sum()).backward()
    grads = conv._short_conv_bwd(dc, xc, wc, bias=bc, apply_silu=silu, initial_states=ic, seq_idx=sc, dfinal_states=fc)
    again = conv._short_conv_bwd(dc, xc, wc, bias=bc, apply_silu=silu, initial_states=ic, seq_idx=sc, dfinal_states=fc)
    for name, g, g2, leaf, t in zip(("dx", "dweight", "dbias", "dinitial"), grads, again, leaves, (dtype, torch.float32, torch.float32, dtype)):
        if leaf is None:
            assert g is None
            continue
        assert g.dtype == t and torch.equal(g, g2), name
        assert norm_err(g, leaf.grad) <= 256 * U + half_step(t), name


@pytest.mark.parametrize("dtype,channels,has_seq", [(torch.bfloat16, 2056, True), (torch.float32, 2056, False), (torch.float16, 2049, True)])
def test_conv_long_strips_are_the_short_ones(cuda_device, dtype, channels, has_seq):
    """A batch large enough for the longest strips gives each row the bits that the row gives alone, where it is
    cut into short ones; the filters' gradients are the rows' sum (64 terms more or less one after another)."""
    _, conv, _ = ops()
    r = maker(90)
    b, l = 16, 260
    x, dout = r(b, l, channels, dtype=dtype).to("cuda"), r(b, l, channels, dtype=dtype).to("cuda")
    w, bias, init = (0.5 * r(channels, 4)).to("cuda"), r(channels).to("cuda"), r(b, 3, channels, dtype=dtype).to("cuda")
    seq = packed(b, l, 7).to("cuda") if has_seq else None
    kw = lambda i: dict(bias=bias, initial_states=init[i], seq_idx=None if seq is None else seq[i])  # noqa: E731
    every = slice(0, b)
    out, fin = conv._short_conv_fwd(x, w, return_final_states=True, **kw(every))
    dx, dw, db, di = conv._short_conv_bwd(dout, x, w, dfinal_states=init, **kw(every))
    dws, dbs = 0, 0
    for i in range(b):
        one = slice(i, i + 1)
        o1, f1 = conv._short_conv_fwd(x[one], w, return_final_states=True, **kw(one))
        g = conv._short_conv_bwd(dout[one], x[one], w, dfinal_states=init[one], **kw(one))
        assert torch.equal(out[one], o1) and torch.equal(fin[one], f1) and torch.equal(dx[one], g[0]) and torch.equal(di[one], g[3])
        dws, dbs = dws + g[1].double(), dbs + g[2].double()
    assert norm_err(dw, dws.cpu()) <= 64 * U and norm_err(db, dbs.cpu()) <= 64 * U


def test_conv_in_pieces_is_the_whole(cuda_device):
    """A sequence in pieces, each continued from the last one's state, then single tokens from a pool of
    slots: the bits of the whole sequence at once."""
    _, conv, _ = ops()
    r = maker(11)
    x, w, bias = cuda(r(3, 50, 72, dtype=torch.bfloat16), r(72, 4), r(72))
    whole, _ = conv._short_conv_fwd(x, w, bias=bias)
    state, outs = None, []
    for t0, t1 in ((0, 1), (1, 3), (3, 35), (35, 40)):
        o, state = conv._short_conv_fwd(x[:, t0:t1], w, bias=bias, initial_states=state, return_final_states=True)
        outs.append(o)
    pool = torch.randn(7, 3, 72, device="cuda").to(torch.bfloat16)
    idx = torch.tensor([5, 0, 3], dtype=torch.int32, device="cuda")
    pool[idx.long()] = state
    kept = pool.clone()
    for t in range(40, 50):
        outs.append(conv._short_conv_step(x[:, t], pool, w, bias=bias, state_indices=idx)[:, None])
    assert torch.equal(torch.cat(outs, 1), whole)
    others = [1, 2, 4, 6]
    assert torch.equal(pool[others], kept[others])
    assert torch.equal(pool[idx.long()], x[:, 47:50])


def test_offsets_past_32_bits(cuda_device):
    """Batch and position strides whose products pass 2^31 elements: rows of one huge buffer."""
    norm, conv, scan = ops()
    l, d, n = 5, 64, 16
    pitch = 2 ** 31 // 4 + 64                          # elements between positions: the fifth lies past 2^31
    buf = torch.zeros(4 * pitch + 4096, dtype=torch.bfloat16, device="cuda")
    r = maker(60)
    small = r(1, l, 3 * d + 2 * n, dtype=torch.bfloat16).to("cuda")
    big = torch.as_strided(buf, (1, l, 3 * d + 2 * n), (4 * pitch, pitch, 1))
    big.copy_(small)
    w, cw, A = torch.ones(d, device="cuda"), r(d, 4).to("cuda"), -torch.rand(d, n, device="cuda")

    def work(t):
        x, dt, z, B, C = t.split([d, d, d, n, n], dim=-1)
        B, C = B.unsqueeze(2), C.unsqueeze(2)
        y, total, rstd, _ = norm._add_rms_norm_fwd(x, w, residual=z)
        c, _ = conv._short_conv_fwd(x, cw)
        out, fin, saved = scan._token_scan_fwd(x, dt, A, B, C, z=z, dt_softplus=True, for_backward=True)
        g = scan._token_scan_bwd(dt, x, dt, A, B, C, saved, z=z, dt_softplus=True)
        return [y, total, rstd, c, *conv._short_conv_bwd(dt, x, cw)[:2], *norm._add_rms_norm_bwd(dt, x, w, rstd, dresidual=z), out, fin, *g]

    for a, b in zip(work(big), work(small)):
        assert (a is None and b is None) or torch.equal(a, b)


def test_conv_masked_positions_may_hold_anything(cuda_device):
    """What another sequence holds does not reach a position, infinities and NaN included; forward and dx."""
    _, conv, _ = ops()
    r = maker(12)
    x, w = r(1, 40, 16), r(16, 4)
    seq = torch.zeros(1, 40, dtype=torch.int32)
    seq[:, 20:] = 1
    bad = x.clone()
    bad[:, 17:20] = float("nan")
    bad[:, 18] = float("inf")
    xc, bc, wc, sc = cuda(x, bad, w, seq)
    good, _ = conv._short_conv_fwd(xc, wc, seq_idx=sc)
    got, _ = conv._short_conv_fwd(bc, wc, seq_idx=sc)
    assert torch.equal(got[:, 20:], good[:, 20:]) and torch.equal(got[:, :17], good[:, :17])
    dout = torch.randn(1, 40, 16, device="cuda")
    ok = conv._short_conv_bwd(dout, xc, wc, seq_idx=sc)[0]
    dx = conv._short_conv_bwd(dout, bc, wc, seq_idx=sc)[0]
    assert torch.equal(dx[:, 20:], ok[:, 20:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,channels", [(4, 64), (3, 1100), (2, 13)])
def test_conv_step(cuda_device, dtype, width, channels):
    _, conv, _ = ops()
    r = maker(channels)
    x, state, w, bias = r(5, channels, dtype=dtype), r(9, width - 1, channels, dtype=dtype), r(channels, width), r(channels)
    idx = torch.tensor([8, -1, 2, 9, 0], dtype=torch.int32)       # the second and fourth rows are padding
    xc, st, wc, bc, ic = cuda(x, state.clone(), w, bias, idx)
    out = conv._short_conv_step(xc, st, wc, bias=bc, state_indices=ic)
    live = [0, 2, 4]
    slots = idx[live].long()
    ref, fin = L.short_conv(x[live][:, None], w, bias, True, state[slots])
    size, _ = L.short_conv(x[live][:, None].abs(), w.abs(), bias.abs(), False, state[slots].abs())
    within(out[live].cpu(), ref[:, 0], size[:, 0], 80 * U, dtype)
    assert (out[[1, 3]] == 0).all()
    expect = state.clone()
    expect[slots] = fin.to(dtype)
    assert torch.equal(st.cpu(), expect)


def test_conv_step_slots_named_twice(cuda_device):
    """The first row of a slot is served, later ones are padding; more rows than slots too."""
    _, conv, _ = ops()
    r = maker(14)
    x, state, w = r(300, 24).to("cuda"), r(4, 3, 24).to("cuda"), r(24, 4).to("cuda")
    idx = torch.tensor([1, 1, 3] + [-1] * 280 + [3, 0] + [1] * 14 + [2], dtype=torch.int32, device="cuda")
    first = [0, 2, 284, 299]
    alone = state.clone()
    ref = conv._short_conv_step(x[first], alone, w, state_indices=idx[first])
    out = conv._short_conv_step(x, state, w, state_indices=idx)
    assert torch.equal(out[first], ref) and torch.equal(state, alone)
    rest = [i for i in range(300) if i not in first]
    assert (out[rest] == 0).all()
    # without indices: rows past the slots are padding
    out = conv._short_conv_step(x, state, w)
    assert (out[4:] == 0).all() and (out[:4] != 0).any()


# ---------------------------------------------------------------------------------------------- scan
def scan_inputs(b, l, d, n, g, dtype, seed, dt_dtype=None):
    r = maker(seed)
    gen = torch.Generator().manual_seed(seed)
    A = -torch.exp(torch.rand(d, n, generator=gen) * math.log(16.0))
    d0 = torch.rand(d, generator=gen) * (1e-1 - 1e-3) + 1e-3
    return dict(x=r(b, l, d, dtype=dtype), dt=r(b, l, d, dtype=dt_dtype or dtype), A=A, B=r(b, l, g, n, dtype=dtype), C=r(b, l, g, n, dtype=dtype),
                D=r(d), z=r(b, l, d, dtype=dtype), dt_bias=d0 + torch.log(-torch.expm1(-d0)))


SCAN_CASES = [
    # batch, seqlen, channels, dstate, groups, gate, D, init, seq
    (2, 100, 48, 16, 1, True, True, True, False),
    (1, 1, 16, 16, 1, True, True, True, False),
    (2, 1, 5, 3, 1, False, False, False, False),
    (1, 33, 66, 8, 2, True, True, False, True),
    (2, 47, 36, 24, 3, False, True, True, True),
    (1, 64, 16, 64, 1, True, True, True, True),
    (1, 40, 24, 128, 1, True, True, True, False),
    (1, 21, 9, 256, 1, False, True, True, True),
    (1, 18, 6, 1, 2, True, False, True, False),
    (1, 3000, 24, 16, 1, True, True, True, False),       # few channels, long: segments
    (1, 2100, 20, 8, 2, True, True, True, True),
    (1, 1700, 8, 48, 1, False, True, False, False),
]


def scan_call(inp, case):
    b, l, d, n, g, gate, has_D, has_init, has_seq = case
    init = maker(l + d)(b, d, n) if has_init else None
    # packed rows that begin with sequence 0 (the initial states') or, in every third case, not
    seq = packed(b, l, l + d, first=1 if has_seq and n % 3 == 0 else 0) if has_seq else None
    kw = dict(D=inp["D"] if has_D else None, z=inp["z"] if gate else None, dt_bias=inp["dt_bias"], initial_states=init, seq_idx=seq)
    return [inp[k] for k in ("x", "dt", "A", "B", "C")], kw


@pytest.mark.parametrize("dtype,dt_dtype", [(torch.float32, None), (torch.bfloat16, None), (torch.float16, torch.float32)])
@pytest.mark.parametrize("case", SCAN_CASES)
def test_scan_forward(cuda_device, dtype, dt_dtype, case):
    b, l, d, n, g = case[:5]
    scan = ops()[2]
    pos, kw = scan_call(scan_inputs(b, l, d, n, g, dtype, l + n, dt_dtype), case)
    out, last, _, size = L.token_scan(*pos, dt_softplus=True, **kw)
    dpos, dkw = cuda(*pos), dict(zip(kw, cuda(*kw.values())))
    got, fin, saved = scan._token_scan_fwd(*dpos, dt_softplus=True, **dkw)
    assert saved is None and got.dtype == dtype and fin.dtype == torch.float32
    tol = 66 * U * l
    gate = 1.0 if kw["z"] is None else (kw["z"].double() * torch.sigmoid(kw["z"].double())).abs()
    within(got, out, size * gate, tol + 80 * U, dtype)
    assert norm_err(got, out) <= 64 * U * math.sqrt(l) + half_step(dtype)
    assert norm_err(fin, last) <= 64 * U * math.sqrt(l)
    # the form that keeps what the gradients need gives the same bits
    got2, fin2, saved = scan._token_scan_fwd(*dpos, dt_softplus=True, for_backward=True, **dkw)
    assert torch.equal(got, got2) and torch.equal(fin, fin2) and saved is not None


@pytest.mark.parametrize("dtype,dt_dtype", [(torch.float32, None), (torch.bfloat16, None), (torch.float16, torch.float32)])
@pytest.mark.parametrize("case", SCAN_CASES)
def test_scan_gradients(cuda_device, dtype, dt_dtype, case):
    b, l, d, n, g = case[:5]
    scan = ops()[2]
    pos, kw = scan_call(scan_inputs(b, l, d, n, g, dtype, l + n, dt_dtype), case)
    leaf = lambda t: t.double().requires_grad_() if t is not None and t.is_floating_point() else t  # noqa: E731
    lpos, lkw = [leaf(t) for t in pos], {k: leaf(t) for k, t in kw.items()}
    out, last, _, _ = L.token_scan(*lpos, dt_softplus=True, **lkw)
    r = maker(l * d + 5)
    dout, dfin = r(b, l, d, dtype=dtype), r(b, d, n)
    ((out * dout.double()).sum() + (last * dfin.double()).sum()).backward()
    dpos, dkw = cuda(*pos), dict(zip(kw, cuda(*kw.values())))
    _, _, saved = scan._token_scan_fwd(*dpos, dt_softplus=True, for_backward=True, **dkw)
    args = (dout.to("cuda"), *dpos, saved)
    grads = scan._token_scan_bwd(*args, dt_softplus=True, dfinal_states=dfin.to("cuda"), **dkw)
    again = scan._token_scan_bwd(*args, dt_softplus=True, dfinal_states=dfin.to("cuda"), **dkw)
    names = ("dx", "ddt", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dinitial")
    leaves = (*lpos, lkw["D"], lkw["z"], lkw["dt_bias"], lkw["initial_states"])
    kinds = (dtype, dt_dtype or dtype, torch.float32, dtype, dtype, torch.float32, dtype, torch.float32, torch.float32)
    for name, g1, g2, lf, t in zip(names, grads, again, leaves, kinds):
        if lf is None:
            assert g1 is None, name
            continue
        assert g1.dtype == t and g1.shape == lf.shape and torch.equal(g1, g2), name
        ref = lf.grad
        if ref.norm() == 0:                                # no position sees it
            assert (g1 == 0).all(), name
            continue
        # per tensor, and the tensor may be small against its terms where few positions add up: 4x
        assert norm_err(g1, ref) <= 4 * 64 * U * math.sqrt(l) + 2 * half_step(t) + (half_step(dtype) if name == "dz" else 0), name


def test_scan_gradients_against_differences(cuda_device):
    """The kernels' own forward pass along a direction: (f(v + e w) - f(v - e w)) / 2e against the gradient.
    e = 2^-7: the third-order term is about e^2 / 6 = 1e-5 relative, the roundings of f about
    u sqrt(count) / e = 2^-24 * 64 * 2^7 = 5e-4 of a value's size: 1 percent holds both."""
    scan = ops()[2]
    inp = {k: v.to("cuda") for k, v in scan_inputs(2, 70, 32, 16, 1, torch.float32, 9).items()}
    keys = ("x", "dt", "A", "B", "C")
    kw = lambda v: dict(D=v["D"], z=v["z"], dt_bias=v["dt_bias"], dt_softplus=True)  # noqa: E731
    dout = torch.randn(2, 70, 32, device="cuda")
    _, _, saved = scan._token_scan_fwd(*[inp[k] for k in keys], for_backward=True, **kw(inp))
    g = scan._token_scan_bwd(dout, *[inp[k] for k in keys], saved, **kw(inp))
    grads = dict(zip(("x", "dt", "A", "B", "C", "D", "z", "dt_bias"), g))
    f = lambda v: (scan._token_scan_fwd(*[v[k] for k in keys], **kw(v))[0].double() * dout.double()).sum().item()  # noqa: E731
    e = 2.0 ** -7
    for k, gk in grads.items():
        w = gk / gk.norm() * math.sqrt(gk.numel()) * 0.1          # along the gradient: the difference is large
        up, dn = dict(inp), dict(inp)
        up[k], dn[k] = inp[k] + e * w, inp[k] - e * w
        assert (f(up) - f(dn)) / (2 * e) == pytest.approx((gk.double() * w.double()).sum().item(), rel=1e-2), k


@pytest.mark.parametrize("dt_limit", [(0.02, 0.1), (0.0, 0.05)])
def test_scan_dt_limits(cuda_device, dt_limit):
    """Clamped steps, with and without softplus; nothing passes back through a clamped one."""
    scan = ops()[2]
    inp = scan_inputs(1, 60, 16, 16, 1, torch.float32, 21)
    for softplus in (True, False):
        leaves = {k: v.double().requires_grad_() for k, v in inp.items()}
        out, _, _, size = L.token_scan(*[leaves[k] for k in ("x", "dt", "A", "B", "C")], D=leaves["D"], dt_bias=leaves["dt_bias"],
                                       dt_softplus=softplus, dt_limit=dt_limit)
        pos = cuda(*[inp[k] for k in ("x", "dt", "A", "B", "C")])
        kw = dict(D=inp["D"].to("cuda"), dt_bias=inp["dt_bias"].to("cuda"), dt_softplus=softplus, dt_limit=dt_limit)
        got, _, saved = scan._token_scan_fwd(*pos, for_backward=True, **kw)
        within(got, out.detach(), size, 66 * U * 60, torch.float32)
        dout = maker(3)(1, 60, 16)
        (out * dout.double()).sum().backward()
        g = scan._token_scan_bwd(dout.to("cuda"), *pos, saved, **kw)
        assert norm_err(g[1], leaves["dt"].grad) <= 256 * U * math.sqrt(60)
        assert torch.equal(g[1].cpu() == 0, leaves["dt"].grad == 0)


@pytest.mark.parametrize("dt_limit", [(0.0, float("inf")), (0.01, 0.2)])
def test_scan_infinities_and_nan_stay_in_their_channel(cuda_device, dt_limit):
    """A NaN or an infinity in one channel's x or dt reaches that channel from there on and no other, forward,
    gradients of the other channels and steps alike; a clamp does not swallow it."""
    scan = ops()[2]
    inp = {k: v.to("cuda") for k, v in scan_inputs(1, 50, 40, 16, 1, torch.float32, 33).items()}
    keys = ("x", "dt", "A", "B", "C")
    kw = dict(dt_softplus=True, dt_limit=dt_limit)
    good, gfin, gsaved = scan._token_scan_fwd(*[inp[k] for k in keys], for_backward=True, **kw)
    others = [c for c in range(40) if c not in (3, 17)]
    for key in ("x", "dt"):
        bad = dict(inp)
        bad[key] = inp[key].clone()
        bad[key][:, 20, 3] = float("nan")
        bad[key][:, 25, 17] = float("inf")
        got, fin, saved = scan._token_scan_fwd(*[bad[k] for k in keys], for_backward=True, **kw)
        assert torch.equal(got[..., others], good[..., others]) and torch.equal(fin[:, others], gfin[:, others])
        assert torch.equal(got[:, :20, 3], good[:, :20, 3]) and torch.equal(got[:, :25, 17], good[:, :25, 17])
        assert got[:, 20:, 3].isnan().all() and fin[:, 3].isnan().all()
        dout = torch.ones_like(good)
        a = scan._token_scan_bwd(dout, *[inp[k] for k in keys], gsaved, **kw)
        b = scan._token_scan_bwd(dout, *[bad[k] for k in keys], saved, **kw)
        for i in (0, 1):                                # dx, ddt
            assert torch.equal(a[i][..., others], b[i][..., others])
        assert torch.equal(a[2][others], b[2][others])  # dA
        st = torch.zeros(1, 40, 16, device="cuda")
        out = scan._token_scan_step(st, bad["x"][:, 20], bad["dt"][:, 20], inp["A"], inp["B"][:, 20], inp["C"][:, 20], **kw)
        assert out[:, 3].isnan().all() and torch.isfinite(out[:, others]).all() and torch.isfinite(st[:, others]).all()


def test_scan_packed_sequences_are_the_sequences(cuda_device):
    """Packed sequences give what the sequences give one by one, also where another sequence holds NaN."""
    scan = ops()[2]
    inp = scan_inputs(1, 90, 32, 16, 1, torch.float32, 4)
    seq = torch.zeros(1, 90, dtype=torch.int32)
    seq[:, 41:] = 1
    pos = cuda(*[inp[k] for k in ("x", "dt", "A", "B", "C")])
    kw = dict(dt_bias=inp["dt_bias"].to("cuda"), dt_softplus=True)
    whole, fin, _ = scan._token_scan_fwd(*pos, seq_idx=seq.to("cuda"), **kw)
    cut = lambda lo, hi: [p if p.dim() == 2 else p[:, lo:hi] for p in pos]  # noqa: E731
    a, _, _ = scan._token_scan_fwd(*cut(0, 41), **kw)
    b, fb, _ = scan._token_scan_fwd(*cut(41, 90), **kw)
    ref = torch.cat([a, b], 1)
    # other tiles, so other orders of the sums over the state: l u of the values
    torch.testing.assert_close(whole, ref, atol=66 * U * 90 * ref.abs().max().item(), rtol=0)
    torch.testing.assert_close(fin, fb, atol=66 * U * 90 * fb.abs().max().item(), rtol=0)
    bad = [p.clone() for p in pos]
    bad[0][:, 30:41] = float("nan")
    got, gfin, _ = scan._token_scan_fwd(*bad, seq_idx=seq.to("cuda"), **kw)
    assert torch.equal(got[:, 41:], whole[:, 41:]) and torch.equal(got[:, :30], whole[:, :30]) and torch.equal(gfin, fin)


def test_scan_strides_and_other_streams(cuda_device):
    """Inputs that are column ranges of one projection buffer (odd offsets too), a transposed batch, and a
    call on another stream."""
    scan = ops()[2]
    r = maker(31)
    b, l, d, n = 2, 50, 40, 16
    buf = r(b, l, 3 * d + 2 * n + 3, dtype=torch.bfloat16).to("cuda")
    A, bias = (-torch.rand(d, n) - 0.1).to("cuda"), r(d).to("cuda")
    for off in (0, 1, 3):
        x, z, dt = buf[..., off:off + d], buf[..., off + d:off + 2 * d], buf[..., off + 2 * d:off + 3 * d]
        B, C = (buf[..., 3 * d - 40 + k * n:3 * d - 40 + k * n + n].unsqueeze(2) for k in range(2))
        args = (x, dt, A, B, C)
        kw = dict(z=z, dt_bias=bias, dt_softplus=True, for_backward=True)
        plain = [t.contiguous() for t in args]
        ref, rfin, rsaved = scan._token_scan_fwd(*plain, **{**kw, "z": z.contiguous()})
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got, fin, saved = scan._token_scan_fwd(*args, **kw)
            g = scan._token_scan_bwd(x, *args, saved, z=z, dt_bias=bias, dt_softplus=True)
        torch.cuda.current_stream().wait_stream(stream)
        assert torch.equal(got, ref) and torch.equal(fin, rfin)
        gr = scan._token_scan_bwd(x.contiguous(), *plain, rsaved, z=z.contiguous(), dt_bias=bias, dt_softplus=True)
        assert all(p is q or torch.equal(p, q) for p, q in zip(g, gr))
        torch.cuda.synchronize()
    xt, dtt = buf.transpose(0, 1)[..., :d], buf.transpose(0, 1)[..., d:2 * d]
    Bt = buf.transpose(0, 1)[..., 2 * d:2 * d + n].unsqueeze(2)
    got, _, _ = scan._token_scan_fwd(xt, dtt, A, Bt, Bt, dt_softplus=True)
    ref, _, _ = scan._token_scan_fwd(xt.contiguous(), dtt.contiguous(), A, Bt.contiguous(), Bt.contiguous(), dt_softplus=True)
    assert torch.equal(got, ref)


# ---------------------------------------------------------------------------------------------- step
STEP_CASES = [
    # batch, heads, headdim (0: per channel), dstate, groups
    (3, 4, 64, 128, 1), (2, 6, 48, 128, 2), (1, 3, 16, 64, 1), (2, 4, 8, 16, 2), (2, 2, 33, 20, 1), (1, 2, 64, 256, 1), (2, 3, 20, 13, 3),
    (3, 130, 0, 16, 1), (1, 1536, 0, 16, 1), (2, 37, 0, 8, 1), (2, 24, 0, 5, 2), (1, 10, 0, 64, 2), (1, 6, 0, 300, 1),
]


@pytest.mark.parametrize("dtype,state_dtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                               (torch.float16, torch.float16)])
@pytest.mark.parametrize("case", STEP_CASES)
def test_step(cuda_device, dtype, state_dtype, case):
    b, h, p, n, g = case
    scan = ops()[2]
    r = maker(h * n + p)
    wide = (h, p) if p else (h,)
    x, z, state = r(b, *wide, dtype=dtype), r(b, *wide, dtype=dtype), r(b + 4, *wide, n, dtype=state_dtype)
    dt, bias = r(b, h, dtype=dtype), r(h) - 2
    A = -torch.exp(r(h) if p else r(h, n))
    B, C = r(b, g, n, dtype=dtype), r(b, g, n, dtype=dtype)
    D = r(*wide) if p == 64 else r(h)
    idx = torch.randperm(b + 4, generator=torch.Generator().manual_seed(1))[:b].to(torch.int32)
    out, new = L.token_scan_step(state[idx.long()], x, dt, A, B, C, D, z, bias, True)
    size, _ = L.token_scan_step(state[idx.long()].abs(), x.abs(), dt, A, B.abs(), C.abs(), D.abs(), None, bias, True)
    xc, zc, st, dc, bc, Ac, Bc, Cc, Dc, ic = cuda(x, z, state.clone(), dt, bias, A, B, C, D, idx)
    got = scan._token_scan_step(st, xc, dc, Ac, Bc, Cc, D=Dc, z=zc, dt_bias=bc, dt_softplus=True, state_indices=ic)
    # one position: 66 u of the state's terms, the sum over n, the gate
    gate = (z.double() * torch.sigmoid(z.double())).abs()
    within(got, out, size * gate, (66 + n + 80) * U, dtype)
    habs, _ = L.token_scan_step(state[idx.long()].abs(), x.abs(), dt, A, B.abs(), C, None, None, bias, True)
    _, sabs = L.token_scan_step(state[idx.long()].abs(), x.abs(), dt, A, B.abs(), C, None, None, bias, True)
    within(st[ic.long()], new, sabs, 66 * U, state_dtype)
    rest = [i for i in range(b + 4) if i not in idx.tolist()]
    assert torch.equal(st[rest].cpu(), state[rest])
    # without indices row i uses slot i
    st2 = state[:b].clone().to("cuda")
    got2 = scan._token_scan_step(st2, xc, dc, Ac, Bc, Cc, D=Dc, z=zc, dt_bias=bc, dt_softplus=True)
    ref2, _ = L.token_scan_step(state[:b], x, dt, A, B, C, D, z, bias, True)
    size2, _ = L.token_scan_step(state[:b].abs(), x.abs(), dt, A, B.abs(), C.abs(), D.abs(), None, bias, True)
    within(got2, ref2, size2 * gate, (66 + n + 80) * U, dtype)


@pytest.mark.parametrize("per_head", [True, False])
def test_step_padding_and_slots_named_twice(cuda_device, per_head):
    """Rows outside the slots and later rows of a slot named twice: zeros, and no state touched."""
    scan = ops()[2]
    r = maker(8)
    wide = (3, 32) if per_head else (70,)
    h, n = wide[0], 16
    x, state = r(6, *wide).to("cuda"), r(5, *wide, n).to("cuda")
    dt, A = r(6, h).to("cuda"), -torch.rand(*((h,) if per_head else (h, n)), device="cuda")
    B, C = r(6, 1, n).to("cuda"), r(6, 1, n).to("cuda")
    idx = torch.tensor([2, -1, 2, 5, 4, 4], dtype=torch.int32, device="cuda")
    before = state.clone()
    out = scan._token_scan_step(state, x, dt, A, B, C, dt_softplus=True, state_indices=idx)
    alone = before.clone()
    keep = [0, 4]
    ref = scan._token_scan_step(alone, x[keep], dt[keep], A, B[keep], C[keep], dt_softplus=True, state_indices=idx[keep])
    assert torch.equal(out[keep], ref) and torch.equal(state, alone)
    assert (out[[1, 2, 3, 5]] == 0).all()
    assert torch.equal(state[[0, 1, 3]], before[[0, 1, 3]])


def test_step_offsets_past_32_bits(cuda_device):
    """A pool of states with more than 2^31 elements: its last slot, and one past the 32-bit mark."""
    scan = ops()[2]
    h, p, n = 80, 64, 128
    slots = 2 ** 31 // (h * p * n) + 3
    state = torch.zeros(slots, h, p, n, device="cuda", dtype=torch.bfloat16)
    r = maker(2)
    x, dt, A = r(2, h, p, dtype=torch.bfloat16).to("cuda"), r(2, h, dtype=torch.bfloat16).to("cuda"), -torch.rand(h, device="cuda")
    B, C = r(2, 1, n, dtype=torch.bfloat16).to("cuda"), r(2, 1, n, dtype=torch.bfloat16).to("cuda")
    idx = torch.tensor([slots - 1, slots - 2], dtype=torch.int32, device="cuda")
    out = scan._token_scan_step(state, x, dt, A, B, C, dt_softplus=True, state_indices=idx)
    small = torch.zeros(2, h, p, n, device="cuda", dtype=torch.bfloat16)
    ref = scan._token_scan_step(small, x, dt, A, B, C, dt_softplus=True)
    assert torch.equal(out, ref) and torch.equal(state[idx.long()], small)
    assert not state[:slots - 2].any()


# ------------------------------------------------------------------------------------------ together
def test_prompt_then_tokens_per_channel(cuda_device):
    """A layer's operators in a row as they are used: norm, convolution, scan for a prompt, then token by
    token from the states the prompt left: against the same sequence in one piece."""
    norm, conv, scan = ops()
    r = maker(17)
    b, l, extra, d, n = 2, 37, 6, 48, 16
    u, res = r(b, l + extra, d).to("cuda"), r(b, l + extra, d).to("cuda")
    w, cw, cb = (1 + 0.1 * r(d)).to("cuda"), r(d, 4).to("cuda"), r(d).to("cuda")
    A, D, bias = -torch.rand(d, n, device="cuda") - 0.1, r(d).to("cuda"), (r(d) - 2).to("cuda")
    dt, B, C, z = (r(b, l + extra, *s).to("cuda") for s in ((d,), (1, n), (1, n), (d,)))

    def prompt(t0, t1):
        y = norm._add_rms_norm_fwd(u[:, t0:t1], w, residual=res[:, t0:t1])[0]
        c, cstate = conv._short_conv_fwd(y, cw, bias=cb, return_final_states=True)
        out, state, _ = scan._token_scan_fwd(c, dt[:, t0:t1], A, B[:, t0:t1], C[:, t0:t1], D=D, z=z[:, t0:t1], dt_bias=bias, dt_softplus=True)
        return out, cstate, state

    whole, wc, ws = prompt(0, l + extra)
    out, cstate, state = prompt(0, l)
    outs = [out]
    for t in range(l, l + extra):
        y = norm._add_rms_norm_fwd(u[:, t], w, residual=res[:, t])[0]
        c = conv._short_conv_step(y, cstate, cw, bias=cb)
        outs.append(scan._token_scan_step(state, c, dt[:, t], A, B[:, t], C[:, t], D=D, z=z[:, t], dt_bias=bias, dt_softplus=True)[:, None])
    got = torch.cat(outs, 1)
    tol = 66 * U * (l + extra)
    assert norm_err(got, whole.double().cpu()) <= tol and norm_err(state, ws.double().cpu()) <= tol
    assert norm_err(cstate, wc.double().cpu()) <= 16 * U


def test_chunk_kernels_then_tokens_per_head(cuda_device):
    """A prompt through the chunk kernels, continued token by token from their final_states, against the
    chunk kernels on the longer sequence.  Their 16-bit operands round B's scaled rows to bf16, so the
    states agree to 1e-2 as everywhere else in the suite."""
    from mamba_fused_minimal_b200.main import _mamba_chunk_scan_combined_fwd_concurrent as combined
    from oracle import ssd_oracle as O
    scan = ops()[2]
    b, l, extra, h, p, g, n = 2, 512, 8, 4, 64, 1, 128
    inp = {k: v.to("cuda") for k, v in O.make_inputs(b, l + extra, h, p, g, n, dtype=torch.bfloat16, seed=12).items()}
    cut = lambda k, lo, hi: inp[k][:, lo:hi]  # noqa: E731
    call = lambda hi: combined(cut("x", 0, hi), cut("dt", 0, hi), inp["A"], cut("B", 0, hi), cut("C", 0, hi), 256, D=inp["D"],  # noqa: E731
                               dt_bias=inp["dt_bias"], dt_softplus=True)
    whole = call(l + extra)
    head = call(l)
    state = head[5]
    assert state.shape == (b, h, p, n) and state.dtype == torch.float32
    outs = [scan._token_scan_step(state, inp["x"][:, t], inp["dt"][:, t], inp["A"], inp["B"][:, t], inp["C"][:, t], D=inp["D"],
                                  dt_bias=inp["dt_bias"], dt_softplus=True) for t in range(l, l + extra)]
    got, ref = torch.stack(outs, 1).float(), whole[0][:, l:].float()
    assert ((got - ref).abs().max() / ref.abs().max()).item() <= 1e-2
    assert ((state - whole[5]).abs().max() / whole[5].abs().max()).item() <= 1e-2


@pytest.mark.parametrize("seqlen,nheads,ngroups", [(512, 8, 1), (300, 4, 2), (1, 8, 1)])
def test_layer_pipeline_of_main(cuda_device, seqlen, nheads, ngroups):
    """The layer's operators as the package's command runs them, also with slots of a pool."""
    from mamba_fused_minimal_b200.main import _layer_prompt_fwd, _layer_token_step, check_prompt_then_tokens
    assert check_prompt_then_tokens(seqlen=seqlen, tokens=3, nheads=nheads, ngroups=ngroups, verbose=False)
    r = maker(seqlen)
    h, p, n, dtype = nheads, 64, 128, torch.bfloat16
    width = h * p + 2 * ngroups * n
    u, res = r(2, seqlen + 1, width, dtype=dtype).to("cuda"), r(2, seqlen + 1, width, dtype=dtype).to("cuda")
    dt = r(2, seqlen + 1, h, dtype=dtype).to("cuda")
    kw = dict(norm_weight=torch.ones(width, device="cuda"), conv_weight=r(width, 4).to("cuda"), conv_bias=r(width).to("cuda"),
              A=-torch.rand(h, device="cuda"), ngroups=ngroups, dstate=n, dt_softplus=True)
    _, _, cs, st = _layer_prompt_fwd(u[:, :-1], res[:, :-1], dt[:, :-1], chunk_size=128, **kw)
    cpool, spool = torch.zeros(5, 3, width, dtype=dtype, device="cuda"), torch.zeros(5, h, p, n, device="cuda")
    idx = torch.tensor([4, 1], dtype=torch.int32, device="cuda")
    cpool[idx.long()], spool[idx.long()] = cs, st
    a, ra = _layer_token_step(u[:, -1], res[:, -1], dt[:, -1], conv_state=cs, state=st, **kw)
    b, rb = _layer_token_step(u[:, -1], res[:, -1], dt[:, -1], conv_state=cpool, state=spool, state_indices=idx, **kw)
    assert torch.equal(a, b) and torch.equal(ra, rb)
    assert torch.equal(cpool[idx.long()], cs) and torch.equal(spool[idx.long()], st) and not spool[[0, 2, 3]].any()


def test_captured_and_replayed(cuda_device):
    """Forward, gradients and steps captured into graphs; two graphs replayed side by side on two streams with
    other inputs each give what the eager calls give."""
    norm, conv, scan = ops()
    r = maker(40)
    b, l, d, n = 1, 1200, 32, 16                     # long and narrow: the scan uses its workspace
    A, w, cw = -torch.rand(d, n, device="cuda"), torch.ones(d, device="cuda"), r(d, 4).to("cuda")

    def work(v):
        y, total, rstd, _ = norm._add_rms_norm_fwd(v["x"], w, residual=v["x"])
        dn = norm._add_rms_norm_bwd(v["dout"], total, w, rstd)
        c, _ = conv._short_conv_fwd(y, cw)
        dc = conv._short_conv_bwd(v["dout"], y, cw)
        out, fin, saved = scan._token_scan_fwd(c, v["dt"], A, v["B"], v["C"], dt_softplus=True, for_backward=True)
        g = scan._token_scan_bwd(v["dout"], c, v["dt"], A, v["B"], v["C"], saved, dt_softplus=True)
        tok = scan._token_scan_step(v["state"].copy_(fin), c[:, 0], v["dt"][:, 0], A, v["B"][:, 0], v["C"][:, 0], dt_softplus=True)
        return [t for t in (y, total, *dn, c, *dc, out, fin, *g, tok, v["state"]) if t is not None]

    def inputs(seed):
        q = maker(seed)
        return {k: q(b, l, *s).to("cuda") for k, s in dict(x=(d,), dt=(d,), dout=(d,), B=(1, n), C=(1, n)).items()} | {
            "state": torch.empty(b, d, n, device="cuda")}

    ref = [[t.clone() for t in work(inputs(s))] for s in (1, 2)]
    statics, graphs, outs = [inputs(3), inputs(4)], [], []
    stream = torch.cuda.Stream()
    for v in statics:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            work(v)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(work(v))
        graphs.append(graph)
    for v, s in zip(statics, (1, 2)):
        for k, t in inputs(s).items():
            v[k].copy_(t)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(outs, ref):
        assert all(torch.equal(a, c) for a, c in zip(got, want))


BANDED = [(torch.bfloat16, 5, 37, 40, 16, 1), (torch.float32, 1, 1100, 21, 8, 3), (torch.float16, 2, 19, 24, 128, 1)]


@pytest.mark.parametrize("dtype,b,l,d,n,g", BANDED)
def test_inputs_between_nan_bands_and_outputs_between_canaries(cuda_device, dtype, b, l, d, n, g):
    """Reads and writes outside the tensors, looked for as in test_gpu_guard_bands.py: inputs between NaNs,
    outputs between canaries, the bits of ordinary tensors."""
    from mamba_fused_minimal_b200._ext import C as ext
    from test_gpu_guard_bands import BAND, banded
    norm, conv, scan = ops()
    v = {k: t.to("cuda") for k, t in scan_inputs(b, l, d, n, g, dtype, 50).items()}
    r = maker(51)
    v |= dict(cw=r(d, 4).to("cuda"), w=r(d).to("cuda"), dout=r(b, l, d, dtype=dtype).to("cuda"), seq=packed(b, l, 3).to("cuda"),
              ci=r(b, 3, d, dtype=dtype).to("cuda"), si=r(b, d, n).to("cuda"))

    def work(v):
        y, total, rstd, _ = norm._add_rms_norm_fwd(v["x"], v["w"], residual=v["dout"])
        q, _, _, sc = norm._add_rms_norm_fwd(v["x"], v["w"], out_dtype=torch.int8)
        dn = norm._add_rms_norm_bwd(v["dout"], total, v["w"], rstd, dresidual=v["z"])
        c, cf = conv._short_conv_fwd(v["x"], v["cw"], bias=v["D"], initial_states=v["ci"], seq_idx=v["seq"], return_final_states=True)
        dc = conv._short_conv_bwd(v["dout"], v["x"], v["cw"], bias=v["D"], initial_states=v["ci"], seq_idx=v["seq"], dfinal_states=v["ci"])
        kw = dict(D=v["D"], z=v["z"], dt_bias=v["dt_bias"], dt_softplus=True, initial_states=v["si"], seq_idx=v["seq"])
        pos = [v[k] for k in ("x", "dt", "A", "B", "C")]
        out, fin, saved = scan._token_scan_fwd(*pos, for_backward=True, **kw)
        g = scan._token_scan_bwd(v["dout"], *pos, saved, dfinal_states=v["si"], **kw)
        st = v["si"].clone()
        tok = scan._token_scan_step(st, v["x"][:, 0], v["dt"][:, 0], v["A"], v["B"][:, 0], v["C"][:, 0], D=v["D"], dt_bias=v["dt_bias"],
                                    dt_softplus=True)
        cs = v["ci"].clone()
        ct = conv._short_conv_step(v["x"][:, 0], cs, v["cw"], bias=v["D"])
        torch.cuda.synchronize()
        return [y, total, rstd, q, sc, *dn, c, cf, *dc, out, fin, *saved, *g, st, tok, cs, ct]

    ref = work(v)
    guarded = {k: banded(t) for k, t in v.items()}
    try:
        ext.debug_set_guard_bytes(BAND)
        got = work(guarded)
        damaged = ext.debug_check_guards()
    finally:
        ext.debug_set_guard_bytes(0)
        ext.debug_check_guards()
    assert damaged == 0
    for i, (a, c) in enumerate(zip(got, ref)):
        assert torch.isfinite(c.float()).all() and torch.equal(a, c), i


def test_refusals(cuda_device):
    """What the kernels do not take is refused before anything is enqueued."""
    norm, conv, scan = ops()
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    bf = torch.bfloat16
    one = [z(1, 4, 8), z(1, 4, 8), z(8, 4), z(1, 4, 1, 4), z(1, 4, 1, 4)]
    for match, call in [
        ("contiguous in its last", lambda: norm._add_rms_norm_fwd(z(2, 8, 16).transpose(1, 2), z(8))),
        ("residual must have", lambda: norm._add_rms_norm_fwd(z(2, 8), z(8), residual=z(2, 8, dtype=bf))),
        ("positive|NULL", lambda: norm._add_rms_norm_fwd(z(0, 8), z(8))),
        ("not fp32 / bf16 / fp16", lambda: norm._add_rms_norm_fwd(z(2, 8, dtype=torch.float64), z(8))),
        ("must be a CUDA tensor", lambda: norm._add_rms_norm_fwd(z(2, 8), torch.zeros(8))),
        ("dout must have", lambda: norm._add_rms_norm_bwd(z(2, 8), z(2, 8), z(8), z(2), x_dtype=bf)),
        ("not 2, 3 or 4", lambda: conv._short_conv_fwd(z(1, 4, 8), z(8, 5))),
        ("not 2, 3 or 4", lambda: conv._short_conv_step(z(1, 8), z(1, 4, 8), z(8, 5))),
        ("positive|NULL", lambda: conv._short_conv_fwd(z(1, 0, 8), z(8, 4))),
        ("whole numbers", lambda: conv._short_conv_fwd(z(1, 4, 8), z(8, 4), seq_idx=z(1, 4))),
        ("must have x's dtype", lambda: conv._short_conv_step(z(1, 8), z(1, 3, 8, dtype=bf), z(8, 4))),
        ("int32", lambda: conv._short_conv_step(z(1, 8), z(1, 3, 8), z(8, 4), state_indices=z(1, dtype=torch.int64))),
        ("single memory location", lambda: conv._short_conv_step(z(1, 8), z(1, 3, 8).expand(4, 3, 8), z(8, 4))),
        ("dstate 257", lambda: scan._token_scan_fwd(z(1, 4, 8), z(1, 4, 8), z(8, 257), z(1, 4, 1, 257), z(1, 4, 1, 257))),
        ("dt must have", lambda: scan._token_scan_fwd(one[0], one[1].to(bf), *one[2:])),
        ("same dtype", lambda: scan._token_scan_fwd(*one[:3], one[3].to(bf), one[4])),
        ("positive|NULL", lambda: scan._token_scan_fwd(z(1, 0, 8), z(1, 0, 8), z(8, 4), z(1, 0, 1, 4), z(1, 0, 1, 4))),
        ("checkpoints must be", lambda: scan._token_scan_bwd(one[0], *one, (z(1, 1, 8, 4, dtype=bf), None))),
        ("int32", lambda: scan._token_scan_step(z(2, 8, 4), z(1, 8), z(1, 8), z(8, 4), z(1, 1, 4), z(1, 1, 4), state_indices=z(1))),
    ]:
        with pytest.raises(RuntimeError, match=match):
            call()
