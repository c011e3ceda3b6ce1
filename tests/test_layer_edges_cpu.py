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
