"""The operators around the scan in 64 bits, from their definitions, one position after another.  TEST
INFRASTRUCTURE ONLY, like ssd_oracle.py; plain torch on the CPU (or any device), differentiable, so that
autograd gives the gradients' formulas.  Inputs of any float type; outputs are fp64 and unrounded."""
import torch


def _d(t):
    return None if t is None else t.double()


def add_rms_norm(x, weight, residual=None, eps=1e-5):
    """(y, t)"""
    t = _d(x) if residual is None else _d(x) + _d(residual)
    return t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * _d(weight), t


def _same(seq_idx, t, s):
    """(batch, 1): whether positions t and s < t belong to one sequence; before the first lies sequence 0."""
    if seq_idx is None:
        return True
    return (seq_idx[:, t] == (seq_idx[:, s] if s >= 0 else 0))[:, None]


def short_conv(x, weight, bias=None, apply_silu=True, initial_states=None, seq_idx=None):
    """(out, final_states)"""
    x, w = _d(x), _d(weight)
    b, l, c = x.shape
    width = w.shape[1]
    before = x.new_zeros(b, width - 1, c) if initial_states is None else _d(initial_states)
    zero = torch.zeros((), dtype=torch.float64, device=x.device)

    def at(s):
        return x[:, s] if s >= 0 else before[:, s + width - 1]

    out = []
    for t in range(l):
        acc = x.new_zeros(b, c) if bias is None else _d(bias).expand(b, c)
        for k in range(width):
            s = t - (width - 1) + k
            same = _same(seq_idx, t, s)
            acc = acc + w[:, k] * (at(s) if same is True else torch.where(same, at(s), zero))
        out.append(acc * torch.sigmoid(acc) if apply_silu else acc)
    final = []
    for k in range(width - 1):
        s = l - (width - 1) + k
        same = _same(seq_idx, l - 1, s)
        final.append(at(s) if same is True else torch.where(same, at(s), zero))
    return torch.stack(out, 1), torch.stack(final, 1)


def _dt(dt, dt_bias, dt_softplus, dt_limit):
    d = _d(dt) if dt_bias is None else _d(dt) + _d(dt_bias)
    if dt_softplus:
        d = torch.clamp(d, min=0) + torch.log1p(torch.exp(-d.abs()))
    return torch.clamp(d, min=dt_limit[0], max=dt_limit[1])


def token_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, dt_limit=(0.0, float("inf")), initial_states=None,
               seq_idx=None):
    """(out, final_states, out_x, size): `size` is out_x with every term taken at its absolute value, what an
    error bound of a sum is relative to."""
    x, A, B, C = _d(x), _d(A), _d(B), _d(C)
    b, l, d = x.shape
    g, n = B.shape[2:]
    group = torch.arange(d, device=x.device) // (d // g)
    delta = _dt(dt, dt_bias, dt_softplus, dt_limit)
    h = x.new_zeros(b, d, n) if initial_states is None else _d(initial_states)
    habs = h.abs().detach()
    ys, sizes = [], []
    for t in range(l):
        same = _same(seq_idx, t, t - 1)
        if same is not True:
            h, habs = h * same[..., None], habs * same[..., None]
        a = torch.exp(delta[:, t, :, None] * A)
        u = (delta[:, t] * x[:, t])[..., None] * B[:, t, group]
        h = a * h + u
        habs = (a * habs + u.abs()).detach()
        y = (h * C[:, t, group]).sum(-1)
        size = (habs * C[:, t, group].abs()).sum(-1)
        if D is not None:
            y = y + _d(D) * x[:, t]
            size = size + (_d(D) * x[:, t]).abs()
        ys.append(y)
        sizes.append(size.detach())
    y = torch.stack(ys, 1)
    out = y if z is None else y * _d(z) * torch.sigmoid(_d(z))
    return out, h, y, torch.stack(sizes, 1)


def token_scan_step(state, x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, dt_limit=(0.0, float("inf"))):
    """(out, new state) of rows whose state is given row by row: state (b, h, p, n) with A (h,), or (b, d, n)
    with A (d, n)."""
    per_head = state.dim() == 4
    h = x.shape[1]
    group = torch.arange(h, device=x.device) // (h // B.shape[1])
    delta = _dt(dt, dt_bias, dt_softplus, dt_limit)
    Bh, Ch = _d(B)[:, group], _d(C)[:, group]
    if per_head:
        a = torch.exp(delta * _d(A))[..., None, None]
        new = _d(state) * a + (delta[..., None] * _d(x))[..., None] * Bh[:, :, None]
        y = (new * Ch[:, :, None]).sum(-1)
        if D is not None:
            y = y + (_d(D)[:, None] if D.dim() == 1 else _d(D)) * _d(x)
    else:
        new = _d(state) * torch.exp(delta[..., None] * _d(A)) + (delta * _d(x))[..., None] * Bh
        y = (new * Ch).sum(-1)
        if D is not None:
            y = y + _d(D) * _d(x)
    return (y if z is None else y * _d(z) * torch.sigmoid(_d(z))), new
