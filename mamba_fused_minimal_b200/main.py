"""The reference's end-to-end check (main.py there): three forward pipelines built from the
same seven functions -- all five unfused kernels, and the two pipelines whose middle step
is a fused entry point -- and a comparison of their six outputs with
isclose(rtol=1e-2, atol=1e-3).

Then the same scan as a layer uses it: residual addition and norm, short convolution, chunk pipeline for a
prompt, and the prompt's continuation token by token from the states that it left, against the longer
prompt.

    python -m mamba_fused_minimal_b200.main
"""
import torch
from einops import rearrange

from .kernels.add_rms_norm import _add_rms_norm_fwd
from .kernels.fused_concurrent import _fused_chunk_state_state_passing_fwd_concurrent
from .kernels.fused_globalbar import _fused_chunk_state_state_passing_fwd_globalbar
from .kernels.rand_data import generate_dummy_data
from .kernels.short_conv import _short_conv_fwd, _short_conv_step
from .kernels.ssd_bmm import _bmm_chunk_fwd
from .kernels.ssd_chunk_scan import _bmm_chunk_scan_fwd, _chunk_scan_fwd
from .kernels.ssd_chunk_state import _chunk_cumsum_fwd, _chunk_state_fwd
from .kernels.ssd_state_passing import _state_passing_fwd
from .kernels.state_path import _state_path_fwd
from .kernels.token_scan import _token_scan_step

TENSOR_NAMES = ["out", "out_x", "dt", "dA_cumsum", "states", "final_states"]


def dim_checks_common(x, dt, A, B, C, D=None, z=None):
    """Shape assertions and contiguity fixes of the reference's main.py:32-56."""
    batch, seqlen, nheads, headdim = x.shape
    _, _, ngroups, dstate = B.shape
    assert nheads % ngroups == 0
    assert B.shape == (batch, seqlen, ngroups, dstate)
    assert x.shape == (batch, seqlen, nheads, headdim)
    assert dt.shape == (batch, seqlen, nheads)
    assert A.shape == (nheads,)
    assert C.shape == B.shape
    if z is not None:
        assert z.shape == x.shape
    if D is not None:
        assert D.shape == (nheads, headdim) or D.shape == (nheads,)
    if B.stride(-1) != 1:
        B = B.contiguous()
    if C.stride(-1) != 1:
        C = C.contiguous()
    if x.stride(-1) != 1 and x.stride(1) != 1:
        x = x.contiguous()
    if z is not None and z.stride(-1) != 1 and z.stride(1) != 1:
        z = z.contiguous()
    if D is not None and D.stride(-1) != 1:
        D = D.contiguous()
    return x, dt, A, B, C, D, z, dstate


def _mamba_chunk_scan_combined_fwd_original(x, dt, A, B, C, chunk_size, D=None, z=None, dt_bias=None,
                                            dt_softplus=False, dt_limit=(0.0, float("inf"))):
    """Five separate kernels (main.py:60-74)."""
    x, dt, A, B, C, D, z, dstate = dim_checks_common(x, dt, A, B, C, D, z)
    dA_cumsum, dt = _chunk_cumsum_fwd(dt, A, chunk_size, dt_bias=dt_bias, dt_softplus=dt_softplus,
                                      dt_limit=dt_limit)
    states = _chunk_state_fwd(B, x, dt, dA_cumsum, seq_idx=None, states_in_fp32=True)
    states, final_states = _state_passing_fwd(rearrange(states, "... p n -> ... (p n)"), dA_cumsum[:, :, :, -1],
                                              initial_states=None, seq_idx=None, chunk_size=chunk_size,
                                              out_dtype=C.dtype)
    states, final_states = [rearrange(t, "... (p n) -> ... p n", n=dstate) for t in [states, final_states]]
    CB = _bmm_chunk_fwd(C, B, chunk_size, seq_idx=None, output_dtype=torch.float32)
    out, out_x = _chunk_scan_fwd(CB, x, dt, dA_cumsum, C, states, D=D, z=z, seq_idx=None)
    return out, out_x, dt, dA_cumsum, states, final_states


def _combined_fused(fused_fn, x, dt, A, B, C, chunk_size, D, z, dt_bias, initial_states, seq_idx, dt_softplus,
                    dt_limit):
    x, dt, A, B, C, D, z, dstate = dim_checks_common(x, dt, A, B, C, D, z)
    if fused_fn is None:
        # Two calls, two launches where the tcgen05 kernels take the problem: the cumsum and the fused
        # state step behind `_state_path_fwd` (same four tensors, bit for bit, as the two calls of the
        # other branch), and the chunk bmm inside the chunk scan (`_bmm_chunk_scan_fwd`; cb never
        # exists in memory).
        dA_cumsum, dt, states, final_states = _state_path_fwd(dt, A, B, x, chunk_size, C.dtype, dt_bias=dt_bias,
                                                              dt_softplus=dt_softplus, dt_limit=dt_limit,
                                                              initial_states=initial_states, seq_idx=seq_idx)
        out, out_x = _bmm_chunk_scan_fwd(C, B, x, dt, dA_cumsum, states, D=D, z=z, seq_idx=seq_idx)
        return out, out_x, dt, dA_cumsum, states, final_states
    CB = _bmm_chunk_fwd(C, B, chunk_size, seq_idx=seq_idx, output_dtype=torch.float32)
    dA_cumsum, dt = _chunk_cumsum_fwd(dt, A, chunk_size, dt_bias=dt_bias, dt_softplus=dt_softplus, dt_limit=dt_limit)
    states, final_states = fused_fn(B, x, dt, dA_cumsum, C.dtype, initial_states=initial_states, seq_idx=seq_idx,
                                    states_in_fp32=True)
    out, out_x = _chunk_scan_fwd(CB, x, dt, dA_cumsum, C, states, D=D, z=z, seq_idx=seq_idx)
    return out, out_x, dt, dA_cumsum, states, final_states


def _mamba_chunk_scan_combined_fwd_globalbar(x, dt, A, B, C, chunk_size, D=None, z=None, dt_bias=None,
                                             initial_states=None, seq_idx=None, cu_seqlens=None, dt_softplus=False,
                                             dt_limit=(0.0, float("inf"))):
    """main.py:78-88."""
    return _combined_fused(_fused_chunk_state_state_passing_fwd_globalbar, x, dt, A, B, C, chunk_size, D, z,
                           dt_bias, initial_states, seq_idx, dt_softplus, dt_limit)


def _mamba_chunk_scan_combined_fwd_concurrent(x, dt, A, B, C, chunk_size, D=None, z=None, dt_bias=None,
                                              initial_states=None, seq_idx=None, cu_seqlens=None,
                                              dt_softplus=False, dt_limit=(0.0, float("inf"))):
    """main.py:93-103.  The four calls there are two here: `_state_path_fwd` (cumsum + fused state step) and
    `_bmm_chunk_scan_fwd` (chunk bmm + chunk scan); the global-barrier pipeline above keeps the four."""
    return _combined_fused(None, x, dt, A, B, C, chunk_size, D, z, dt_bias, initial_states, seq_idx, dt_softplus,
                           dt_limit)


def _layer_prompt_fwd(u, residual, dt, norm_weight, conv_weight, conv_bias, A, ngroups, dstate, chunk_size, D=None, dt_bias=None,
                      dt_softplus=False):
    """A layer's operators on a prompt: u and residual (batch, seqlen, d + 2 * ngroups * dstate), the channels of
    x, B and C side by side, are added and normalised, pass the short convolution, and the scan runs through
    the chunk kernels.  Returns (out (batch, seqlen, nheads, headdim), residual, conv_state, state)."""
    batch, seqlen, width = u.shape
    nheads = A.shape[0]
    d = width - 2 * ngroups * dstate
    y, residual, _, _ = _add_rms_norm_fwd(u, norm_weight, residual=residual)
    xbc, conv_state = _short_conv_fwd(y, conv_weight, bias=conv_bias, return_final_states=True)
    x, B, C = xbc.split([d, ngroups * dstate, ngroups * dstate], dim=-1)
    out, _, _, _, _, state = _mamba_chunk_scan_combined_fwd_concurrent(
        x.unflatten(-1, (nheads, d // nheads)), dt, A, B.unflatten(-1, (ngroups, dstate)), C.unflatten(-1, (ngroups, dstate)), chunk_size, D,
        dt_bias=dt_bias, dt_softplus=dt_softplus)
    return out, residual, conv_state, state


def _layer_token_step(u, residual, dt, norm_weight, conv_weight, conv_bias, A, ngroups, dstate, conv_state, state, D=None, dt_bias=None,
                      dt_softplus=False, state_indices=None):
    """The same operators on one more position of each sequence: u and residual (batch, d + 2 * ngroups * dstate),
    dt (batch, nheads); conv_state and state, as `_layer_prompt_fwd` returns them or pools of slots, are
    updated in place.  Returns (out (batch, nheads, headdim), residual)."""
    nheads = A.shape[0]
    d = u.shape[-1] - 2 * ngroups * dstate
    y, residual, _, _ = _add_rms_norm_fwd(u, norm_weight, residual=residual)
    xbc = _short_conv_step(y, conv_state, conv_weight, bias=conv_bias, state_indices=state_indices)
    x, B, C = xbc.split([d, ngroups * dstate, ngroups * dstate], dim=-1)
    out = _token_scan_step(state, x.unflatten(-1, (nheads, d // nheads)), dt, A, B.unflatten(-1, (ngroups, dstate)),
                           C.unflatten(-1, (ngroups, dstate)), D=D, dt_bias=dt_bias, dt_softplus=dt_softplus, state_indices=state_indices)
    return out, residual


def check_prompt_then_tokens(seqlen=512, tokens=8, nheads=80, headdim=64, ngroups=1, dstate=128, chunk_size=256, dtype=torch.bfloat16, verbose=True):
    """A prompt and `tokens` single steps behind it against the prompt that holds them all: within 1e-2 of the
    largest value (the chunk kernels round their scaled operands to `dtype`, the step does not)."""
    torch.manual_seed(42)
    width = nheads * headdim + 2 * ngroups * dstate
    u, residual = (torch.randn(2, seqlen + tokens, width, dtype=dtype, device="cuda") for _ in range(2))
    dt = torch.rand(2, seqlen + tokens, nheads, dtype=dtype, device="cuda") * 0.5 + 0.5
    params = dict(norm_weight=torch.ones(width, device="cuda"), conv_weight=torch.randn(width, 4, device="cuda") * 0.5,
                  conv_bias=torch.randn(width, device="cuda") * 0.1, A=-torch.rand(nheads, device="cuda"), ngroups=ngroups, dstate=dstate)
    more = dict(D=torch.randn(nheads, device="cuda"), dt_bias=torch.rand(nheads, device="cuda") * 0.5 - 0.25, dt_softplus=True)
    whole = _layer_prompt_fwd(u, residual, dt, chunk_size=chunk_size, **params, **more)
    _, _, conv_state, state = _layer_prompt_fwd(u[:, :seqlen], residual[:, :seqlen], dt[:, :seqlen], chunk_size=chunk_size, **params, **more)
    outs = [_layer_token_step(u[:, t], residual[:, t], dt[:, t], conv_state=conv_state, state=state, **params, **more)[0]
            for t in range(seqlen, seqlen + tokens)]
    ok = True
    for name, a, b in (("out", torch.stack(outs, 1), whole[0][:, seqlen:]), ("conv_state", conv_state, whole[2]), ("state", state, whole[3])):
        err = ((a.float() - b.float()).abs().max() / b.float().abs().max()).item()
        ok = ok and err <= 1e-2
        if verbose:
            print(f"    {name}: largest difference {err:.2e} of the largest value")
    return ok


def check_same_tensors(t1, t2, tensor_name, verbose=True):
    """Elementwise isclose(rtol=0.01, atol=0.001, equal_nan=True) as in main.py:109-143."""
    if t1 is None and t2 is None:
        return True
    if t1 is None or t2 is None:
        if verbose:
            print(f"    {tensor_name}: one of the two results is None")
        return False
    close = torch.isclose(t1, t2, rtol=0.01, atol=0.001, equal_nan=True)
    num_mismatch = int((~close).sum().item())
    if verbose:
        if num_mismatch > 0:
            idx = torch.nonzero(~close)[:5].tolist()
            print(f"    {tensor_name}: {num_mismatch} mismatches, first at {idx}")
        else:
            mid = t1.numel() // 2
            a = ["{:.4f}".format(v) for v in t1.reshape(-1)[mid:mid + 4].tolist()]
            b = ["{:.4f}".format(v) for v in t2.reshape(-1)[mid:mid + 4].tolist()]
            print(f"    {tensor_name} tensors match, example elems: {a} vs {b}")
    return num_mismatch == 0


def check_same_results(res1, res2, verbose=True):
    all_match = True
    for i in range(len(res1)):
        all_match = check_same_tensors(res1[i], res2[i], TENSOR_NAMES[i], verbose) and all_match
    if verbose:
        print("results match" if all_match else "RESULTS DO NOT MATCH")
    return all_match


def main():
    x, A, B, C, D, dt, dt_bias = generate_dummy_data()
    chunk_size = 256
    original = _mamba_chunk_scan_combined_fwd_original(x, dt, A, B, C, chunk_size, D, dt_bias=dt_bias)
    print("-------------------- original vs itself")
    ok0 = check_same_results(original, original)
    globalbar = _mamba_chunk_scan_combined_fwd_globalbar(x, dt, A, B, C, chunk_size, D, dt_bias=dt_bias)
    print("-------------------- global-barrier entry point vs original")
    ok1 = check_same_results(globalbar, original)
    concurrent = _mamba_chunk_scan_combined_fwd_concurrent(x, dt, A, B, C, chunk_size, D, dt_bias=dt_bias)
    print("-------------------- concurrent entry point vs original")
    ok2 = check_same_results(concurrent, original)
    print("-------------------- a prompt and its next tokens vs the longer prompt")
    ok3 = check_prompt_then_tokens()
    print("results:", "all good" if ok0 and ok1 and ok2 and ok3 else "bad")
    return ok0 and ok1 and ok2 and ok3


if __name__ == "__main__":
    raise SystemExit(0 if main() else 1)
