"""Short causal convolution over the sequence, one filter of 2 to 4 taps for each channel: what stands
between a layer's input projection and the scan (its channels are x, B and C side by side).  Prompts,
gradients and single tokens, as plain calls (their results carry no autograd history).  The reference has no
counterpart.

The state of a sequence is its last width - 1 inputs, (width - 1, channels), oldest first."""
from .._ext import C as _C


def _short_conv_fwd(x, weight, bias=None, apply_silu=True, initial_states=None, seq_idx=None, return_final_states=False):
    """x (batch, seqlen, channels) with contiguous channels (a column range of a wider buffer will do),
    weight (channels, width):

        out[t] = act(bias + sum_k weight[:, k] * x[t - (width - 1) + k]),  act = silu or nothing

    Before the first position stand initial_states (batch, width - 1, channels) or zeros.  With seq_idx
    (batch, seqlen) a position sees only its own sequence; initial_states belong to sequence 0.
    Returns (out, final_states); final_states is None unless asked for."""
    # the front end asserts the shapes
    return _C.short_conv_fwd(x, weight, bias, apply_silu, initial_states, seq_idx, return_final_states)


def _short_conv_bwd(dout, x, weight, bias=None, apply_silu=True, initial_states=None, seq_idx=None, dfinal_states=None):
    """Gradients of `_short_conv_fwd` from its inputs (nothing has to be kept).  Returns (dx, dweight, dbias,
    dinitial_states): x's dtype, except dweight and dbias in fp32; dbias and dinitial_states are None where
    bias and initial_states are.  The same inputs give the same bits."""
    return _C.short_conv_bwd(dout, x, weight, bias, apply_silu, initial_states, seq_idx, dfinal_states)


def _short_conv_step(x, conv_state, weight, bias=None, apply_silu=True, state_indices=None):
    """One position of each running sequence: x (batch, channels), conv_state (slots, width - 1, channels),
    which is shifted by one position IN PLACE.  state_indices (batch,) int32 gives each row's slot (without
    it row i uses slot i).  A row whose index lies outside the slots, or whose slot an earlier row names
    too, is padding: its output is zero and no state is touched.  Returns out (batch, channels)."""
    # the front end asserts the shapes: a token's call is short
    return _C.short_conv_step(x, conv_state, weight, bias, apply_silu, state_indices)
