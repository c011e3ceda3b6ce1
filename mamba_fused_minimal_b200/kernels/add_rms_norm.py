"""Residual addition + root-mean-square norm, the step that opens every layer around the scan: forward with
an output in x's type or in 8 bits with one scale a row, and the gradients.  Plain calls: their results carry no
autograd history.  The reference has no counterpart (its path begins behind a layer's input projection)."""
from .._ext import C as _C


def _add_rms_norm_fwd(x, weight, residual=None, eps=1e-5, out_dtype=None, residual_dtype=None):
    """x (batch, seqlen, dim) or (rows, dim), weight (dim,).  With t = x + residual in fp32:

        out = t / sqrt(mean(t^2) + eps) * weight

    in x's dtype, or for out_dtype torch.int8 / torch.float8_e4m3fn as codes with out = codes * scales,
    scales = max|out| of the row / 127 or / 448 (0 for a row of zeros, NaN for a row that holds an infinity
    or a NaN).

    Returns (out, residual_out, rstd, scales).  residual_out is t in the residual's dtype (x's dtype or
    fp32), or in `residual_dtype` where there is no residual yet; None if neither is given.  rstd
    (rows..., fp32), of residual_out as it was kept, is for the gradients; scales (rows..., fp32) takes its
    place where out is in 8 bits (the other of the two is None).

    The squares are summed in fp32: |t| has to stay below about 1e19 / sqrt(dim)."""
    # the front end asserts the shapes: a token's call is short
    return _C.add_rms_norm_fwd(x, weight, residual, eps, out_dtype, residual_dtype)


def _add_rms_norm_bwd(dout, total, weight, rstd, dresidual=None, x_dtype=None):
    """Gradients of `_add_rms_norm_fwd` in x's type.  `total` is what was normalised as it was kept:
    residual_out, or x itself where there is none.  dresidual: the gradient that reaches residual_out from
    the layers behind (total's dtype).  x_dtype: x's dtype, by default dout's.

    Returns (dx, dresidual_in, dweight): one gradient in x's dtype and in total's (one tensor where they
    agree), and the weight's in fp32."""
    assert total.dim() in (2, 3)
    assert dout.shape == total.shape
    assert weight.shape == total.shape[-1:]
    assert rstd.shape == total.shape[:-1]
    if dresidual is not None:
        assert dresidual.shape == total.shape
    return _C.add_rms_norm_bwd(dout, total, weight, rstd, dresidual, x_dtype)
