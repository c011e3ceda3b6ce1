"""The operators around the scan without a GPU: refusals of the Python layer and of the C ABI, and the 64-bit
oracle against plain formulas, autograd's gradients against differences, and the chunked oracle."""
import ctypes

import pytest
import torch

from mamba_fused_minimal_b200._ext import load_abi
from mamba_fused_minimal_b200.kernels.add_rms_norm import _add_rms_norm_bwd, _add_rms_norm_fwd
from mamba_fused_minimal_b200.kernels.short_conv import _short_conv_bwd, _short_conv_fwd, _short_conv_step
from mamba_fused_minimal_b200.kernels.token_scan import _token_scan_bwd, _token_scan_fwd, _token_scan_step
from oracle import layer_oracle as L
from oracle import ssd_oracle as O

ENTRY_POINTS = ["ssd_add_rms_norm_fwd", "ssd_add_rms_norm_bwd", "ssd_short_conv_fwd", "ssd_short_conv_bwd", "ssd_short_conv_step",
                "ssd_token_scan_fwd", "ssd_token_scan_bwd", "ssd_token_scan_step"]


@pytest.mark.parametrize("name", ENTRY_POINTS)
def test_null_and_empty_parameters_are_rejected_with_a_message(name):
    lib = load_abi()
    lib.ssd_last_error.restype = ctypes.c_char_p
    assert getattr(lib, name)(None, None) == 1
    assert b"NULL" in lib.ssd_last_error()
    # a struct of zeros: no pointers, no sizes; nothing is enqueued
    zeros = ctypes.create_string_buffer(1024)
    assert getattr(lib, name)(zeros, None) == 1
    assert len(lib.ssd_last_error()) > 0


@pytest.mark.parametrize("name", ["ssd_add_rms_norm_bwd", "ssd_short_conv_bwd", "ssd_token_scan", "ssd_token_scan_bwd"])
def test_workspace_sizes_of_null_are_zero(name):
    fn = getattr(load_abi(), name + "_workspace_bytes")
    fn.restype = ctypes.c_size_t
    assert fn(None) == 0


def _scan_inputs(b=2, l=5, d=4, n=3, g=2):
    return [torch.zeros(b, l, d), torch.zeros(b, l, d), torch.zeros(d, n), torch.zeros(b, l, g, n), torch.zeros(b, l, g, n)]


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 8)
    for call in [lambda: _add_rms_norm_fwd(x, torch.zeros(8)),
                 lambda: _add_rms_norm_bwd(x, x, torch.zeros(8), torch.zeros(2, 3)),
                 lambda: _short_conv_fwd(x, torch.zeros(8, 4)),
                 lambda: _short_conv_bwd(x, x, torch.zeros(8, 4)),
                 lambda: _short_conv_step(x[:, 0], torch.zeros(2, 3, 8), torch.zeros(8, 4)),
                 lambda: _token_scan_fwd(*_scan_inputs()),
                 lambda: _token_scan_bwd(torch.zeros(2, 5, 4), *_scan_inputs(), (torch.zeros(2, 1, 4, 3), None)),
                 lambda: _token_scan_step(torch.zeros(2, 4, 3), torch.zeros(2, 4), torch.zeros(2, 4), torch.zeros(4, 3),
                                          torch.zeros(2, 2, 3), torch.zeros(2, 2, 3))]:
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_shapes_are_asserted():
    x = torch.zeros(2, 3, 8)
    sx, sdt, sA, sB, sC = _scan_inputs()
    for call in [lambda: _add_rms_norm_fwd(x, torch.zeros(7)),
                 lambda: _add_rms_norm_fwd(x, torch.zeros(8), residual=torch.zeros(2, 3, 7)),
                 lambda: _add_rms_norm_fwd(x, torch.zeros(8), out_dtype=torch.int16),
                 lambda: _add_rms_norm_bwd(x, x, torch.zeros(8), torch.zeros(2, 4)),
                 lambda: _short_conv_fwd(x, torch.zeros(7, 4)),
                 lambda: _short_conv_fwd(x, torch.zeros(8, 4), initial_states=torch.zeros(2, 4, 8)),
                 lambda: _short_conv_fwd(x, torch.zeros(8, 4), seq_idx=torch.zeros(2, 4, dtype=torch.int32)),
                 lambda: _short_conv_bwd(x[:, :2], x, torch.zeros(8, 4)),
                 lambda: _short_conv_step(x[:, 0], torch.zeros(2, 2, 8), torch.zeros(8, 4)),
                 lambda: _short_conv_step(x[:, 0], torch.zeros(2, 3, 8), torch.zeros(8, 4), state_indices=torch.zeros(3, dtype=torch.int32)),
                 lambda: _token_scan_fwd(sx, sdt, sA[:, :2], sB, sC),
                 lambda: _token_scan_fwd(sx[..., :3], sdt[..., :3], sA[:3], sB, sC),
                 lambda: _token_scan_fwd(sx, sdt, sA, sB, sC, D=torch.zeros(3)),
                 lambda: _token_scan_bwd(sx, sx, sdt, sA, sB, sC, (torch.zeros(2, 2, 4, 3), None)),
                 lambda: _token_scan_bwd(sx, sx, sdt, sA, sB, sC, (torch.zeros(2, 1, 4, 3), None), z=sx),
                 lambda: _token_scan_step(torch.zeros(2, 4, 1, 3), sx[:, 0], sdt[:, 0], sA, sB[:, 0], sC[:, 0]),
                 lambda: _token_scan_step(torch.zeros(2, 4, 3), sx[:, 0], sdt[:, 0], torch.zeros(4), sB[:, 0], sC[:, 0])]:
        with pytest.raises(AssertionError):
            call()


def test_oracle_conv_is_a_convolution():
    gen = torch.Generator().manual_seed(1)
    x, w, bias = torch.randn(2, 9, 5, generator=gen), torch.randn(5, 4, generator=gen), torch.randn(5, generator=gen)
    out, final = L.short_conv(x, w, bias, apply_silu=False)
    ref = torch.nn.functional.conv1d(x.double().transpose(1, 2), w.double()[:, None], bias.double(), padding=3, groups=5)[..., :9]
    torch.testing.assert_close(out, ref.transpose(1, 2), atol=1e-13, rtol=1e-13)
    assert torch.equal(final, x.double()[:, -3:])
    # packed sequences are the sequences one by one
    seq = torch.tensor([[0, 0, 0, 0, 1, 1, 1, 1, 1]]).expand(2, 9)
    packed, _ = L.short_conv(x, w, bias, seq_idx=seq)
    parts = [L.short_conv(x[:, :4], w, bias)[0], L.short_conv(x[:, 4:], w, bias)[0]]
    torch.testing.assert_close(packed, torch.cat(parts, 1), atol=1e-13, rtol=1e-13)


def test_oracle_scan_against_the_chunked_oracle():
    """With one decay a head the scan by channels is what the chunk kernels' oracle computes."""
    b, l, h, p, g, n = 2, 37, 4, 3, 2, 5
    inp = O.make_inputs(b, l, h, p, g, n, dtype=torch.float32, seed=3)
    dA, dt = O.chunk_cumsum_fwd(inp["dt"], inp["A"], 16, dt_bias=inp["dt_bias"], dt_softplus=True)
    states, fin = O.fused_state_fwd(inp["B"], inp["x"], dt, dA, torch.float32)
    cb = O.bmm_chunk_fwd(inp["C"], inp["B"], 16, output_dtype=torch.float32)
    ref, _ = O.chunk_scan_fwd(cb, inp["x"], dt, dA, inp["C"], states, D=inp["D"])
    wide = lambda t: t.repeat_interleave(p, -1)  # noqa: E731
    out, last, _, _ = L.token_scan(inp["x"].reshape(b, l, h * p), wide(inp["dt"]), wide(inp["A"])[:, None].expand(-1, n), inp["B"], inp["C"],
                                   D=wide(inp["D"]), dt_bias=wide(inp["dt_bias"]), dt_softplus=True)
    torch.testing.assert_close(out.view(b, l, h, p), ref.double(), atol=2e-4, rtol=2e-4)
    torch.testing.assert_close(last.view(b, h, p, n), fin.double(), atol=2e-4, rtol=2e-4)
    # and the step continues it
    state, outs = torch.zeros(b, h, p, n, dtype=torch.float64), []
    for t in range(l):
        o, state = L.token_scan_step(state, inp["x"][:, t], inp["dt"][:, t], inp["A"], inp["B"][:, t], inp["C"][:, t], D=inp["D"],
                                     dt_bias=inp["dt_bias"], dt_softplus=True)
        outs.append(o)
    torch.testing.assert_close(torch.stack(outs, 1), out.view(b, l, h, p), atol=1e-12, rtol=1e-12)


def test_oracle_gradients_against_differences():
    gen = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).requires_grad_()  # noqa: E731
    seq = torch.tensor([[0, 0, 0, 1, 1, 2, 2]])
    assert torch.autograd.gradcheck(lambda x, w, res: L.add_rms_norm(x, w, res)[0], (r(2, 3, 5), r(5), r(2, 3, 5)))
    assert torch.autograd.gradcheck(lambda x, w, bb, i: L.short_conv(x, w, bb, initial_states=i, seq_idx=seq), (r(1, 7, 3), r(3, 4), r(3), r(1, 3, 3)))
    A = (-torch.rand(4, 3, generator=gen, dtype=torch.float64) - 0.2).requires_grad_()
    assert torch.autograd.gradcheck(
        lambda x, dt, a, B, C, D, z, bias, i: L.token_scan(x, dt, a, B, C, D, z, bias, True, initial_states=i, seq_idx=seq)[:2],
        (r(1, 7, 4), r(1, 7, 4), A, r(1, 7, 2, 3), r(1, 7, 2, 3), r(4), r(1, 7, 4), r(4), r(1, 4, 3)))
