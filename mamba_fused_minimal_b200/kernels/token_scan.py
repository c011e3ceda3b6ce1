"""Selective scan, position by position, with a decay for each channel and state component; the chunk kernels
of this package have one decay for each head.  Prompts, gradients, and single tokens; the single-token
step takes both forms, so it also continues what the chunk kernels began (their final_states are its
state).  Plain calls: their results carry no autograd history.  The reference has no counterpart."""
from .._ext import C as _C


def _token_scan_fwd(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, dt_limit=(0.0, float("inf")),
                    initial_states=None, seq_idx=None, for_backward=False):
    """x, dt, z (batch, seqlen, channels), A (channels, dstate), B, C (batch, seqlen, ngroups, dstate), D and
    dt_bias (channels,).  Per channel, with its group's B and C:

        dt' = clamp(softplus?(dt + dt_bias), *dt_limit)
        h = exp(dt' * A) * h + dt' * x * B;   y = sum(C * h) + D * x;   out = y, or y * silu(z)

    h (fp32) starts from initial_states (batch, channels, dstate) or zero; with seq_idx (batch, seqlen) it is
    dropped where the sequence changes, and initial_states belong to sequence 0.  dt has x's dtype or fp32.

    Returns (out, final_states, saved): final_states (batch, channels, dstate) fp32, and with for_backward
    what `_token_scan_bwd` needs, else None: the states before every 16th position and, with z, y before the
    gate, in fp32 (dstate / 4 and 4 bytes for each position and channel)."""
    # the front end asserts the shapes
    out, final, checkpoints, out_x = _C.token_scan_fwd(x, dt, A, B, C, D, z, dt_bias, dt_softplus, dt_limit[0], dt_limit[1],
                                                       initial_states, seq_idx, for_backward)
    return out, final, (checkpoints, out_x) if for_backward else None


def _token_scan_bwd(dout, x, dt, A, B, C, saved, D=None, z=None, dt_bias=None, dt_softplus=False, dt_limit=(0.0, float("inf")),
                    initial_states=None, seq_idx=None, dfinal_states=None):
    """Gradients of `_token_scan_fwd`, called with the same inputs and with what it saved.  Returns (dx, ddt, dA,
    dB, dC, dD, dz, ddt_bias, dinitial_states): dA, dD, ddt_bias and dinitial_states in fp32, the others in
    their input's dtype; None for what was not given.  The same inputs give the same bits.  Scratch: up to 512 MB
    and a few times the states (or 16 positions' shares of dB and dC, where those are more)."""
    checkpoints, out_x = saved
    return _C.token_scan_bwd(dout, x, dt, A, B, C, checkpoints, out_x, D, z, dt_bias, dt_softplus, dt_limit[0], dt_limit[1],
                             initial_states, seq_idx, dfinal_states)


def _token_scan_step(state, x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, dt_limit=(0.0, float("inf")),
                     state_indices=None):
    """One position of each running sequence; `state` is updated IN PLACE.  Two forms:

      per head:    state (slots, nheads, headdim, dstate), x, z (batch, nheads, headdim), A (nheads,),
                   D (nheads,) or (nheads, headdim) -- the chunk kernels' form and layouts
      per channel: state (slots, channels, dstate), x, z (batch, channels), A (channels, dstate), D (channels,)

    dt (batch, nheads or channels), dt_bias (nheads or channels,), B, C (batch, ngroups, dstate).  The state
    may be fp32, bf16 or fp16; the update is computed in fp32 and y sees it before it is rounded.

    state_indices (batch,) int32 gives each row's slot (without it row i uses slot i).  A row whose index
    lies outside the slots, or whose slot an earlier row names too, is padding: its output is zero and no
    state is touched.  Returns out, x's shape and dtype."""
    # the front end asserts the shapes: a token's call is short
    return _C.token_scan_step(state, x, dt, A, B, C, D, z, dt_bias, dt_softplus, dt_limit[0], dt_limit[1], state_indices)
