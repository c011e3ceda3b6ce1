"""Refusals and sizes of the operators around the scan that need no GPU: what a workspace query answers for any
parameters, and calls with tensors of too few dimensions."""
import ctypes

import pytest
import torch

from mamba_fused_minimal_b200._ext import load_abi

I32, I64, PTR = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p


def struct(name, fields):
    return type(name, (ctypes.Structure,), {"_fields_": fields})


def query(name, params):
    fn = getattr(load_abi(), name + "_workspace_bytes")
    fn.restype = ctypes.c_size_t
    return fn(ctypes.byref(params))


Conv = struct("Conv", [(k, PTR) for k in "x weight bias init seq out fin".split()] +
              [(k, I32) for k in "xd wd bd batch seqlen channels width silu".split()] + [("xs", I64 * 2), ("ss", I64 * 2)])
ConvBwd = struct("ConvBwd", [("conv", Conv)] + [(k, PTR) for k in "dout dfinal dx dweight dbias dinit".split()] +
                 [("ds", I64 * 2), ("workspace", PTR), ("bytes", ctypes.c_size_t)])
NormBwd = struct("NormBwd", [(k, PTR) for k in "dout total weight rstd dres dx dresin dweight".split()] +
                 [(k, I32) for k in "xd td wd batch seqlen dim".split()] + [("s", I64 * 6), ("workspace", PTR), ("bytes", ctypes.c_size_t)])


@pytest.mark.parametrize("width", [-1, 0, 1, 5, 9, 17, 64])
def test_conv_workspace_of_a_filter_that_is_not_taken(width):
    p = ConvBwd()
    p.conv.batch, p.conv.seqlen, p.conv.channels, p.conv.width = 2, 40, 64, width
    assert query("ssd_short_conv_bwd", p) == 0


@pytest.mark.parametrize("field", ["batch", "seqlen", "channels"])
@pytest.mark.parametrize("value", [0, -1, -2 ** 31])
def test_conv_workspace_of_no_size(field, value):
    p = ConvBwd()
    p.conv.batch, p.conv.seqlen, p.conv.channels, p.conv.width = 2, 40, 64, 4
    assert query("ssd_short_conv_bwd", p) > 0
    setattr(p.conv, field, value)
    assert query("ssd_short_conv_bwd", p) == 0


@pytest.mark.parametrize("field", ["batch", "seqlen", "dim"])
@pytest.mark.parametrize("value", [0, -1, -2 ** 31])
def test_norm_workspace_of_no_size(field, value):
    p = NormBwd()
    p.batch, p.seqlen, p.dim = 2, 40, 64
    assert query("ssd_add_rms_norm_bwd", p) == 80 * 64 * 4
    setattr(p, field, value)
    assert query("ssd_add_rms_norm_bwd", p) == 0


Scan = struct("Scan", [(k, PTR) for k in "x dt A B C D z bias init seq out out_x fin ckpt".split()] +
              [(k, I32) for k in "xd dtd Ad Dd bd id batch seqlen channels ngroups dstate softplus".split()] +
              [("dt_min", ctypes.c_float), ("dt_max", ctypes.c_float), ("s", I64 * 14), ("workspace", PTR), ("bytes", ctypes.c_size_t)])
ScanBwd = struct("ScanBwd", [("scan", Scan)] + [(k, PTR) for k in "dout dfinal dx ddt dA dB dC dD dz dbias dinit".split()] +
                 [("ds", I64 * 2), ("workspace", PTR), ("bytes", ctypes.c_size_t)])


@pytest.mark.parametrize("batch,seqlen,channels,ngroups,dstate", [
    (1, 4096, 2048, 1, 128), (8, 4096, 5120, 1, 128), (2, 2048, 5120, 1, 256), (1, 65537, 296, 1, 256), (1, 1 << 20, 5120, 8, 64),
    (64, 4096, 5120, 1, 16), (3, 1000, 64, 64, 256), (1, 40000, 8192, 1, 200), (2, 2048, 5120, 1, 16), (1, 1, 1, 1, 1)])
def test_scan_gradients_scratch_is_bounded(batch, seqlen, channels, ngroups, dstate):
    """Whatever the problem's size: 512 MB for the channel blocks' shares of dB and dC, or 16 positions' of one batch
    element where those are more, and a few times the states (as many as there are batch elements, or blocks
    on the GPU, whichever is more)."""
    p = ScanBwd()
    s = p.scan
    for k in "x dt A B C".split():
        setattr(s, k, 16)                  # never followed: a query looks at sizes only
    s.batch, s.seqlen, s.channels, s.ngroups, s.dstate = batch, seqlen, channels, ngroups, dstate
    s.xd = s.dtd = 1
    padded = max(8, 1 << (dstate - 1).bit_length())
    tiles = -(-(channels // ngroups) // (256 // padded))
    shares = 16 * ngroups * tiles * 2 * dstate * 4
    states = channels * dstate * 4
    got = query("ssd_token_scan_bwd", p)
    assert 0 < got <= max(2 ** 29, shares) + 6 * batch * states + 8 * 2 ** 20


def test_tensors_of_no_dimension_are_refused():
    from mamba_fused_minimal_b200.kernels.add_rms_norm import _add_rms_norm_bwd, _add_rms_norm_fwd
    from mamba_fused_minimal_b200.kernels.short_conv import _short_conv_bwd, _short_conv_fwd, _short_conv_step
    from mamba_fused_minimal_b200.kernels.token_scan import _token_scan_bwd, _token_scan_fwd, _token_scan_step
    z = torch.zeros
    calls = [(_add_rms_norm_fwd, [z(2, 8), z(8)]),
             (_add_rms_norm_bwd, [z(2, 8), z(2, 8), z(8), z(2)]),
             (_short_conv_fwd, [z(1, 4, 8), z(8, 4)]),
             (_short_conv_bwd, [z(1, 4, 8), z(1, 4, 8), z(8, 4)]),
             (_short_conv_step, [z(1, 8), z(1, 3, 8), z(8, 4)]),
             (_token_scan_fwd, [z(1, 4, 8), z(1, 4, 8), z(8, 4), z(1, 4, 1, 4), z(1, 4, 1, 4)]),
             (lambda *a: _token_scan_bwd(*a, (z(1, 1, 8, 4), None)),
              [z(1, 4, 8), z(1, 4, 8), z(1, 4, 8), z(8, 4), z(1, 4, 1, 4), z(1, 4, 1, 4)]),
             (_token_scan_step, [z(1, 8, 4), z(1, 8), z(1, 8), z(8, 4), z(1, 1, 4), z(1, 1, 4)]),
             (_token_scan_step, [z(1, 2, 4, 4), z(1, 2, 4), z(1, 2), z(2), z(1, 1, 4), z(1, 1, 4)])]
    for call, args in calls:
        for i in range(len(args)):
            with pytest.raises(AssertionError):
                call(*[z(()) if k == i else a for k, a in enumerate(args)])
