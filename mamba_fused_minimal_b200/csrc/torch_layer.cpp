// PyTorch front end of the operators around the scan (sections 8 to 10 of include/ssd_b200.h): the residual
// addition + root-mean-square norm, the short causal convolution and the token-by-token selective scan.
// Scratch memory is
// allocated for each call, so two captured graphs never share any.  Shapes are asserted here, with the
// AssertionError that the other shims raise in Python: for small calls that took as long as the rest of it.
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/EmptyTensor.h>

#include <limits>
#include <tuple>

#include "torch_common.h"

using namespace ssd_torch;

namespace {

int32_t i32(int64_t v) {
  TORCH_CHECK(v <= std::numeric_limits<int32_t>::max(), "a size of ", v, " is too large");
  return static_cast<int32_t>(v);
}

void assert_shapes(bool ok, const char* what) {
  if (ok) return;
  PyErr_SetString(PyExc_AssertionError, what);
  throw pybind11::error_already_set();
}
bool is_1d(const OptTensor& t, int64_t n) { return !t.has_value() || (t->dim() == 1 && t->size(0) == n); }
bool is_3d(const OptTensor& t, int64_t a, int64_t b, int64_t c) {
  return !t.has_value() || (t->dim() == 3 && t->size(0) == a && t->size(1) == b && t->size(2) == c);
}
bool is_2d(const OptTensor& t, int64_t a, int64_t b) { return !t.has_value() || (t->dim() == 2 && t->size(0) == a && t->size(1) == b); }
bool is_like(const OptTensor& t, const Tensor& x) { return !t.has_value() || t->sizes() == x.sizes(); }

void check_input(const Tensor& t) { TORCH_CHECK(t.is_cuda(), "x must be a CUDA tensor (libssd_b200 has no CPU path)"); }

void check_inner(const Tensor& t, const char* name) {
  TORCH_CHECK(t.size(-1) == 1 || t.stride(-1) == 1, name, " must be contiguous in its last dimension");
}

// strides of the dimensions before the last, as (b, l); a 2-D tensor is one batch element
void row_strides(int64_t (&dst)[2], const Tensor& t) {
  dst[0] = t.dim() == 3 ? t.stride(0) : 0;
  dst[1] = t.stride(t.dim() - 2);
}

Tensor int_index(const Tensor& t, const Tensor& like, const char* name) {
  check_cuda(t, like, name);
  TORCH_CHECK(at::isIntegralType(t.scalar_type(), false), name, " must hold whole numbers");
  return as_int32(t);
}

int out_code(at::ScalarType st) {
  if (st == at::kChar) return SSD_I8;
  if (st == at::kFloat8_e4m3fn) return SSD_E4M3;
  return dtype_code(st);
}

Tensor scratch(size_t bytes, const Tensor& like) {
  return at::detail::empty_cuda({(int64_t)bytes}, at::kByte, like.device(), c10::nullopt);
}

// a parameter: any of the three types, made contiguous
void param(const OptTensor& t, const Tensor& like, const char* name, Tensor& hold, const void*& ptr, int32_t& dtype) {
  if (!t.has_value()) return;
  check_cuda(*t, like, name);
  hold = t->contiguous();
  ptr = hold.data_ptr();
  dtype = dtype_code(hold, name);
}

// ---- residual addition + root-mean-square norm --------------------------------------------------------
std::tuple<Tensor, OptTensor, OptTensor, OptTensor> add_rms_norm_fwd(const Tensor& x, const Tensor& weight, const OptTensor& residual,
                                                                  double eps, std::optional<at::ScalarType> out_dtype,
                                                                  std::optional<at::ScalarType> residual_dtype) {
  assert_shapes((x.dim() == 2 || x.dim() == 3) && weight.dim() == 1 && weight.size(0) == x.size(-1) && is_like(residual, x),
                "x (batch, seqlen, dim) or (rows, dim), weight (dim,), residual as x");
  assert_shapes(!out_dtype.has_value() || *out_dtype == x.scalar_type() || *out_dtype == at::kChar || *out_dtype == at::kFloat8_e4m3fn,
                "out_dtype: x's dtype, int8 or float8_e4m3fn");
  check_input(x);
  c10::cuda::CUDAGuard guard(x.device());
  check_inner(x, "x");
  ssd_add_rms_norm_params_t p{};
  p.x = x.data_ptr();
  p.x_dtype = dtype_code(x, "x");
  p.batch = x.dim() == 3 ? i32(x.size(0)) : 1;
  p.seqlen = i32(x.size(-2));
  p.dim = i32(x.size(-1));
  row_strides(p.x_stride, x);
  Tensor wh;
  param(weight, x, "weight", wh, p.weight, p.weight_dtype);
  auto rdt = residual_dtype;
  if (residual.has_value()) {
    check_cuda(*residual, x, "residual");
    check_inner(*residual, "residual");
    TORCH_CHECK(!rdt.has_value() || *rdt == residual->scalar_type(), "residual_dtype is ", *rdt, " but the residual's is ",
                residual->scalar_type());
    rdt = residual->scalar_type();
    p.residual = residual->data_ptr();
    row_strides(p.residual_stride, *residual);
  }
  OptTensor total, rstd, scales;
  p.residual_dtype = p.x_dtype;
  if (rdt.has_value()) {
    p.residual_dtype = dtype_code(*rdt);
    total = alloc_direct(x.sizes(), x.options().dtype(*rdt));
    p.residual_out = total->data_ptr();
  }
  const at::ScalarType odt = out_dtype.value_or(x.scalar_type());
  p.out_dtype = out_code(odt);
  Tensor out = alloc_direct(x.sizes(), x.options().dtype(odt));
  const auto f32 = x.options().dtype(at::kFloat);
  const auto rows = x.sizes().slice(0, x.dim() - 1);
  if (p.out_dtype == SSD_I8 || p.out_dtype == SSD_E4M3) {
    scales = alloc_direct(rows, f32);
    p.scales = scales->data_ptr<float>();
  } else {
    rstd = alloc_direct(rows, f32);
    p.rstd = rstd->data_ptr<float>();
  }
  p.out = out.data_ptr();
  p.eps = static_cast<float>(eps);
  check_rc(ssd_add_rms_norm_fwd(&p, current_stream(x)), "ssd_add_rms_norm_fwd");
  return {out, total, rstd, scales};
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_bwd(const Tensor& dout, const Tensor& total, const Tensor& weight, const Tensor& rstd,
                                                    const OptTensor& dresidual, std::optional<at::ScalarType> x_dtype) {
  check_input(total);
  c10::cuda::CUDAGuard guard(total.device());
  check_cuda(dout, total, "dout");
  check_cuda(rstd, total, "rstd");
  check_inner(dout, "dout");
  check_inner(total, "total");
  const at::ScalarType xdt = x_dtype.value_or(dout.scalar_type());
  TORCH_CHECK(dout.scalar_type() == xdt, "dout must have x's dtype, ", xdt);
  TORCH_CHECK(rstd.scalar_type() == at::kFloat, "rstd must be fp32");
  ssd_add_rms_norm_bwd_params_t p{};
  p.dout = dout.data_ptr();
  p.total = total.data_ptr();
  Tensor wh, rh = rstd.contiguous();
  param(weight, total, "weight", wh, p.weight, p.weight_dtype);
  p.rstd = rh.data_ptr<float>();
  p.x_dtype = dtype_code(xdt);
  p.total_dtype = dtype_code(total, "total");
  p.batch = total.dim() == 3 ? i32(total.size(0)) : 1;
  p.seqlen = i32(total.size(-2));
  p.dim = i32(total.size(-1));
  row_strides(p.dout_stride, dout);
  row_strides(p.total_stride, total);
  if (dresidual.has_value()) {
    check_cuda(*dresidual, total, "dresidual");
    check_inner(*dresidual, "dresidual");
    TORCH_CHECK(dresidual->scalar_type() == total.scalar_type(), "dresidual must have the residual's dtype, ", total.scalar_type());
    p.dresidual = dresidual->data_ptr();
    row_strides(p.dresidual_stride, *dresidual);
  }
  Tensor dx = alloc_direct(total.sizes(), total.options().dtype(xdt));
  Tensor dres = dx;
  if (xdt != total.scalar_type()) {
    dres = alloc_direct(total.sizes(), total.options());
    p.dresidual_in = dres.data_ptr();
  }
  Tensor dweight = alloc_direct({total.size(-1)}, total.options().dtype(at::kFloat));
  p.dx = dx.data_ptr();
  p.dweight = dweight.data_ptr<float>();
  p.workspace_bytes = ssd_add_rms_norm_bwd_workspace_bytes(&p);
  Tensor ws = scratch(p.workspace_bytes, total);
  p.workspace = ws.data_ptr();
  check_rc(ssd_add_rms_norm_bwd(&p, current_stream(total)), "ssd_add_rms_norm_bwd");
  return {dx, dres, dweight};
}

// ---- short causal convolution ------------------------------------------------------------------------
struct ConvHold {
  Tensor weight, bias, init, seq;
};

void fill_conv(ssd_short_conv_params_t& p, ConvHold& h, const Tensor& x, const Tensor& weight, const OptTensor& bias, bool silu,
               const OptTensor& initial_states, const OptTensor& seq_idx) {
  assert_shapes(x.dim() == 3 && weight.dim() == 2 && weight.size(0) == x.size(2) && is_1d(bias, x.size(2)) &&
                    is_3d(initial_states, x.size(0), weight.size(1) - 1, x.size(2)) && is_2d(seq_idx, x.size(0), x.size(1)),
                "x (batch, seqlen, channels), weight (channels, width), bias (channels,), initial_states (batch, width - 1, channels), "
                "seq_idx (batch, seqlen)");
  check_input(x);
  check_inner(x, "x");
  p.x = x.data_ptr();
  p.x_dtype = dtype_code(x, "x");
  p.batch = i32(x.size(0));
  p.seqlen = i32(x.size(1));
  p.channels = i32(x.size(2));
  p.width = i32(weight.size(1));
  p.silu = silu;
  copy_strides(p.x_stride, x, {0, 1});
  param(weight, x, "weight", h.weight, p.weight, p.weight_dtype);
  param(bias, x, "bias", h.bias, p.bias, p.bias_dtype);
  if (initial_states.has_value()) {
    check_cuda(*initial_states, x, "initial_states");
    TORCH_CHECK(initial_states->scalar_type() == x.scalar_type(), "initial_states must have x's dtype");
    h.init = initial_states->contiguous();
    p.initial_states = h.init.data_ptr();
  }
  if (seq_idx.has_value()) {
    h.seq = int_index(*seq_idx, x, "seq_idx");
    p.seq_idx = h.seq.data_ptr<int32_t>();
    copy_strides(p.seq_idx_stride, h.seq, {0, 1});
  }
}

std::tuple<Tensor, OptTensor> short_conv_fwd(const Tensor& x, const Tensor& weight, const OptTensor& bias, bool silu,
                                             const OptTensor& initial_states, const OptTensor& seq_idx, bool return_final) {
  c10::cuda::OptionalCUDAGuard guard(x.is_cuda() ? c10::optional<c10::Device>(x.device()) : c10::nullopt);
  ssd_short_conv_params_t p{};
  ConvHold h;
  fill_conv(p, h, x, weight, bias, silu, initial_states, seq_idx);
  Tensor out = alloc_direct(x.sizes(), x.options());
  OptTensor fin;
  p.out = out.data_ptr();
  if (return_final) {
    fin = alloc_direct({x.size(0), weight.size(1) - 1, x.size(2)}, x.options());
    p.final_states = fin->data_ptr();
  }
  check_rc(ssd_short_conv_fwd(&p, current_stream(x)), "ssd_short_conv_fwd");
  return {out, fin};
}

std::tuple<Tensor, Tensor, OptTensor, OptTensor> short_conv_bwd(const Tensor& dout, const Tensor& x, const Tensor& weight,
                                                                const OptTensor& bias, bool silu, const OptTensor& initial_states,
                                                                const OptTensor& seq_idx, const OptTensor& dfinal) {
  c10::cuda::OptionalCUDAGuard guard(x.is_cuda() ? c10::optional<c10::Device>(x.device()) : c10::nullopt);
  assert_shapes(x.dim() == 3 && weight.dim() == 2 && dout.sizes() == x.sizes(), "x (batch, seqlen, channels), weight (channels, width), dout as x");
  assert_shapes(is_3d(dfinal, x.size(0), weight.size(1) - 1, x.size(2)), "dfinal_states (batch, width - 1, channels)");
  ssd_short_conv_bwd_params_t p{};
  ConvHold h;
  fill_conv(p.conv, h, x, weight, bias, silu, initial_states, seq_idx);
  check_cuda(dout, x, "dout");
  check_inner(dout, "dout");
  TORCH_CHECK(dout.scalar_type() == x.scalar_type(), "dout must have x's dtype");
  p.dout = dout.data_ptr();
  copy_strides(p.dout_stride, dout, {0, 1});
  Tensor fh;
  if (dfinal.has_value()) {
    check_cuda(*dfinal, x, "dfinal_states");
    TORCH_CHECK(dfinal->scalar_type() == x.scalar_type(), "dfinal_states must have x's dtype");
    fh = dfinal->contiguous();
    p.dfinal_states = fh.data_ptr();
  }
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor dx = alloc_direct(x.sizes(), x.options());
  Tensor dweight = alloc_direct(weight.sizes(), f32);
  OptTensor dbias, dinit;
  p.dx = dx.data_ptr();
  p.dweight = dweight.data_ptr<float>();
  if (bias.has_value()) {
    dbias = alloc_direct(bias->sizes(), f32);
    p.dbias = dbias->data_ptr<float>();
  }
  if (initial_states.has_value()) {
    dinit = alloc_direct(initial_states->sizes(), x.options());
    p.dinitial_states = dinit->data_ptr();
  }
  p.workspace_bytes = ssd_short_conv_bwd_workspace_bytes(&p);
  Tensor ws = scratch(p.workspace_bytes, x);
  p.workspace = ws.data_ptr();
  check_rc(ssd_short_conv_bwd(&p, current_stream(x)), "ssd_short_conv_bwd");
  return {dx, dweight, dbias, dinit};
}

const int32_t* slots_of(const OptTensor& indices, const Tensor& like, Tensor& hold) {
  if (!indices.has_value()) return nullptr;
  check_cuda(*indices, like, "state_indices");
  TORCH_CHECK(indices->scalar_type() == at::kInt, "state_indices must be int32");
  hold = indices->contiguous();
  return hold.data_ptr<int32_t>();
}

Tensor short_conv_step(const Tensor& x, Tensor conv_state, const Tensor& weight, const OptTensor& bias, bool silu,
                       const OptTensor& state_indices) {
  assert_shapes(x.dim() == 2 && conv_state.dim() == 3 && weight.dim() == 2 && conv_state.size(2) == x.size(1) && weight.size(0) == x.size(1) &&
                    weight.size(1) == conv_state.size(1) + 1 && is_1d(bias, x.size(1)) && is_1d(state_indices, x.size(0)),
                "x (batch, channels), conv_state (slots, width - 1, channels), weight (channels, width), bias (channels,), state_indices (batch,)");
  check_input(x);
  c10::cuda::CUDAGuard guard(x.device());
  check_inner(x, "x");
  check_cuda(conv_state, x, "conv_state");
  check_inner(conv_state, "conv_state");
  TORCH_CHECK(conv_state.scalar_type() == x.scalar_type(), "conv_state must have x's dtype");
  at::assert_no_internal_overlap(conv_state);
  ssd_short_conv_step_params_t p{};
  Tensor wh, bh, ih;
  p.x = x.data_ptr();
  p.conv_state = conv_state.data_ptr();
  param(weight, x, "weight", wh, p.weight, p.weight_dtype);
  param(bias, x, "bias", bh, p.bias, p.bias_dtype);
  p.state_indices = slots_of(state_indices, x, ih);
  Tensor out = alloc_direct(x.sizes(), x.options());
  p.out = out.data_ptr();
  p.x_dtype = dtype_code(x, "x");
  p.batch = i32(x.size(0));
  p.slots = i32(conv_state.size(0));
  p.channels = i32(x.size(1));
  p.width = i32(weight.size(1));
  p.silu = silu;
  p.x_stride = x.stride(0);
  copy_strides(p.state_stride, conv_state, {0, 1});
  check_rc(ssd_short_conv_step(&p, current_stream(x)), "ssd_short_conv_step");
  return out;
}

// ---- token-by-token selective scan ---------------------------------------------------------------------
struct ScanHold {
  Tensor A, D, bias, init, seq;
};

void fill_scan(ssd_token_scan_params_t& p, ScanHold& h, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
               const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias, bool dt_softplus, double dt_min, double dt_max,
               const OptTensor& initial_states, const OptTensor& seq_idx) {
  assert_shapes(x.dim() == 3 && B.dim() == 4 && dt.sizes() == x.sizes() && B.size(0) == x.size(0) && B.size(1) == x.size(1) && B.size(2) > 0 &&
                    x.size(2) % B.size(2) == 0 && C.sizes() == B.sizes(),
                "x and dt (batch, seqlen, channels), B and C (batch, seqlen, ngroups, dstate), ngroups dividing channels");
  const int64_t d = x.size(2), n = B.size(3);
  assert_shapes(A.dim() == 2 && A.size(0) == d && A.size(1) == n && is_1d(D, d) && is_like(z, x) && is_1d(dt_bias, d) &&
                    is_3d(initial_states, x.size(0), d, n) && is_2d(seq_idx, x.size(0), x.size(1)),
                "A (channels, dstate), D and dt_bias (channels,), z as x, initial_states (batch, channels, dstate), seq_idx (batch, seqlen)");
  check_input(x);
  check_inner(x, "x");
  check_cuda(dt, x, "dt");
  check_inner(dt, "dt");
  for (const Tensor* t : {&B, &C}) {
    check_cuda(*t, x, "B and C");
    check_inner(*t, "B and C");
    TORCH_CHECK(t->scalar_type() == x.scalar_type(), "B, C and x must have the same dtype");
  }
  p.x = x.data_ptr();
  p.dt = dt.data_ptr();
  p.B = B.data_ptr();
  p.C = C.data_ptr();
  p.x_dtype = dtype_code(x, "x");
  p.dt_dtype = dtype_code(dt, "dt");
  param(A, x, "A", h.A, p.A, p.A_dtype);
  param(D, x, "D", h.D, p.D, p.D_dtype);
  param(dt_bias, x, "dt_bias", h.bias, p.dt_bias, p.bias_dtype);
  param(initial_states, x, "initial_states", h.init, p.initial_states, p.init_dtype);
  if (z.has_value()) {
    check_cuda(*z, x, "z");
    check_inner(*z, "z");
    TORCH_CHECK(z->scalar_type() == x.scalar_type(), "z and x must have the same dtype");
    p.z = z->data_ptr();
    copy_strides(p.z_stride, *z, {0, 1});
  }
  if (seq_idx.has_value()) {
    h.seq = int_index(*seq_idx, x, "seq_idx");
    p.seq_idx = h.seq.data_ptr<int32_t>();
    copy_strides(p.seq_idx_stride, h.seq, {0, 1});
  }
  p.batch = i32(x.size(0));
  p.seqlen = i32(x.size(1));
  p.channels = i32(x.size(2));
  p.ngroups = i32(B.size(2));
  p.dstate = i32(B.size(3));
  p.dt_softplus = dt_softplus;
  p.dt_min = static_cast<float>(dt_min);
  p.dt_max = static_cast<float>(dt_max);
  copy_strides(p.x_stride, x, {0, 1});
  copy_strides(p.dt_stride, dt, {0, 1});
  copy_strides(p.B_stride, B, {0, 1, 2});
  copy_strides(p.C_stride, C, {0, 1, 2});
}

std::tuple<Tensor, Tensor, OptTensor, OptTensor> token_scan_fwd(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                                                                const Tensor& C, const OptTensor& D, const OptTensor& z,
                                                                const OptTensor& dt_bias, bool dt_softplus, double dt_min, double dt_max,
                                                                const OptTensor& initial_states, const OptTensor& seq_idx,
                                                                bool for_backward) {
  c10::cuda::OptionalCUDAGuard guard(x.is_cuda() ? c10::optional<c10::Device>(x.device()) : c10::nullopt);
  ssd_token_scan_params_t p{};
  ScanHold h;
  fill_scan(p, h, x, dt, A, B, C, D, z, dt_bias, dt_softplus, dt_min, dt_max, initial_states, seq_idx);
  const int64_t b = x.size(0), l = x.size(1), d = x.size(2), n = B.size(3);
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor out = alloc_direct(x.sizes(), x.options());
  Tensor fin = alloc_direct({b, d, n}, f32);
  OptTensor out_x, ckpt;
  p.out = out.data_ptr();
  p.final_states = fin.data_ptr<float>();
  if (for_backward) {
    ckpt = alloc_direct({b, (l + SSD_TOKEN_SCAN_CHECKPOINT - 1) / SSD_TOKEN_SCAN_CHECKPOINT, d, n}, f32);
    p.checkpoints = ckpt->data_ptr<float>();
    if (z.has_value()) {
      out_x = alloc_direct(x.sizes(), f32);
      p.out_x = out_x->data_ptr<float>();
    }
  }
  p.workspace_bytes = ssd_token_scan_workspace_bytes(&p);
  Tensor ws;
  if (p.workspace_bytes > 0) {
    ws = scratch(p.workspace_bytes, x);
    p.workspace = ws.data_ptr();
  }
  check_rc(ssd_token_scan_fwd(&p, current_stream(x)), "ssd_token_scan_fwd");
  return {out, fin, ckpt, out_x};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, OptTensor, OptTensor, OptTensor, OptTensor> token_scan_bwd(
    const Tensor& dout, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& ckpt,
    const OptTensor& out_x, const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias, bool dt_softplus, double dt_min,
    double dt_max, const OptTensor& initial_states, const OptTensor& seq_idx, const OptTensor& dfinal) {
  c10::cuda::OptionalCUDAGuard guard(x.is_cuda() ? c10::optional<c10::Device>(x.device()) : c10::nullopt);
  assert_shapes(dout.sizes() == x.sizes() && out_x.has_value() == z.has_value() && is_like(out_x, x), "dout as x, out_x with z and as x");
  assert_shapes(x.dim() == 3 && B.dim() == 4, "x (batch, seqlen, channels), B (batch, seqlen, ngroups, dstate)");
  const int64_t blocks = (x.size(1) + SSD_TOKEN_SCAN_CHECKPOINT - 1) / SSD_TOKEN_SCAN_CHECKPOINT;
  assert_shapes(ckpt.dim() == 4 && ckpt.size(0) == x.size(0) && ckpt.size(1) == blocks && ckpt.size(2) == x.size(2) && ckpt.size(3) == B.size(3) &&
                    is_3d(dfinal, x.size(0), x.size(2), B.size(3)),
                "checkpoints of the same forward call, dfinal_states (batch, channels, dstate)");
  ssd_token_scan_bwd_params_t p{};
  ScanHold h;
  fill_scan(p.scan, h, x, dt, A, B, C, D, z, dt_bias, dt_softplus, dt_min, dt_max, initial_states, seq_idx);
  check_cuda(dout, x, "dout");
  check_inner(dout, "dout");
  TORCH_CHECK(dout.scalar_type() == x.scalar_type(), "dout must have x's dtype");
  check_cuda(ckpt, x, "checkpoints");
  TORCH_CHECK(ckpt.scalar_type() == at::kFloat && ckpt.is_contiguous(), "the forward call's checkpoints must be fp32 and contiguous");
  p.scan.checkpoints = ckpt.data_ptr<float>();
  if (z.has_value()) {
    TORCH_CHECK(out_x.has_value() && out_x->scalar_type() == at::kFloat && out_x->is_contiguous(),
                "with z the forward call's output before the gate is needed, fp32 and contiguous");
    check_cuda(*out_x, x, "out_x");
    p.scan.out_x = out_x->data_ptr<float>();
  }
  p.dout = dout.data_ptr();
  copy_strides(p.dout_stride, dout, {0, 1});
  Tensor fh;
  if (dfinal.has_value()) {
    check_cuda(*dfinal, x, "dfinal_states");
    fh = dfinal->to(at::kFloat).contiguous();
    p.dfinal_states = fh.data_ptr<float>();
  }
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor dx = alloc_direct(x.sizes(), x.options()), ddt = alloc_direct(dt.sizes(), dt.options()), dA = alloc_direct(A.sizes(), f32);
  Tensor dB = alloc_direct(B.sizes(), B.options()), dC = alloc_direct(C.sizes(), C.options());
  OptTensor dD, dz, dbias, dinit;
  p.dx = dx.data_ptr();
  p.ddt = ddt.data_ptr();
  p.dA = dA.data_ptr<float>();
  p.dB = dB.data_ptr();
  p.dC = dC.data_ptr();
  if (D.has_value()) {
    dD = alloc_direct(D->sizes(), f32);
    p.dD = dD->data_ptr<float>();
  }
  if (z.has_value()) {
    dz = alloc_direct(x.sizes(), x.options());
    p.dz = dz->data_ptr();
  }
  if (dt_bias.has_value()) {
    dbias = alloc_direct(dt_bias->sizes(), f32);
    p.ddt_bias = dbias->data_ptr<float>();
  }
  if (initial_states.has_value()) {
    dinit = alloc_direct(initial_states->sizes(), f32);
    p.dinitial_states = dinit->data_ptr<float>();
  }
  p.workspace_bytes = ssd_token_scan_bwd_workspace_bytes(&p);
  Tensor ws = scratch(p.workspace_bytes, x);
  p.workspace = ws.data_ptr();
  check_rc(ssd_token_scan_bwd(&p, current_stream(x)), "ssd_token_scan_bwd");
  return {dx, ddt, dA, dB, dC, dD, dz, dbias, dinit};
}

// per_head: state (slots, h, p, n), x (b, h, p), A (h,); else state (slots, d, n), x (b, d), A (d, n)
Tensor token_scan_step(Tensor state, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                       const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias, bool dt_softplus, double dt_min, double dt_max,
                       const OptTensor& state_indices) {
  const int64_t rank = x.dim(), batch = rank > 1 ? x.size(0) : 0, heads = rank > 1 ? x.size(1) : 0;
  assert_shapes((rank == 2 || rank == 3) && state.dim() == rank + 1 && B.dim() == 3 && C.sizes() == B.sizes() && B.size(0) == batch && B.size(1) > 0 &&
                    heads % B.size(1) == 0 && state.sizes().slice(1, rank - 1) == x.sizes().slice(1) && state.size(-1) == B.size(2),
                "state (slots, nheads, headdim, dstate) with x (batch, nheads, headdim), or (slots, channels, dstate) with (batch, channels); "
                "B and C (batch, ngroups, dstate)");
  assert_shapes(dt.dim() == 2 && dt.size(0) == batch && dt.size(1) == heads &&
                    (rank == 3 ? A.dim() == 1 : A.dim() == 2 && A.size(1) == B.size(2)) && A.size(0) == heads && is_like(z, x) && is_1d(dt_bias, heads) &&
                    is_1d(state_indices, batch) &&
                    (!D.has_value() || (D->dim() == 1 && D->size(0) == heads) || (rank == 3 && D->sizes() == x.sizes().slice(1))),
                "dt (batch, nheads), A (nheads,) or (channels, dstate), D (nheads,) or (nheads, headdim), z as x, dt_bias (nheads,), "
                "state_indices (batch,)");
  check_input(x);
  c10::cuda::CUDAGuard guard(x.device());
  check_cuda(state, x, "state");
  check_inner(state, "state");
  at::assert_no_internal_overlap(state);
  check_cuda(dt, x, "dt");
  check_cuda(A, x, "A");
  for (const Tensor* t : {&B, &C}) {
    check_cuda(*t, x, "B and C");
    check_inner(*t, "B and C");
    TORCH_CHECK(t->scalar_type() == x.scalar_type(), "B, C and x must have the same dtype");
  }
  const bool per_head = state.dim() == 4;
  ssd_token_scan_step_params_t p{};
  p.state = state.data_ptr();
  p.x = x.data_ptr();
  p.dt = dt.data_ptr();
  p.A = A.data_ptr();
  p.B = B.data_ptr();
  p.C = C.data_ptr();
  p.state_dtype = dtype_code(state, "state");
  p.x_dtype = dtype_code(x, "x");
  p.dt_dtype = dtype_code(dt, "dt");
  p.A_dtype = dtype_code(A, "A");
  p.batch = i32(x.size(0));
  p.slots = i32(state.size(0));
  p.nheads = i32(x.size(1));
  p.headdim = per_head ? i32(x.size(2)) : 1;
  p.ngroups = i32(B.size(1));
  p.dstate = i32(B.size(2));
  p.dt_softplus = dt_softplus;
  p.dt_min = static_cast<float>(dt_min);
  p.dt_max = static_cast<float>(dt_max);
  copy_strides(p.state_stride, state, {0, 1});
  p.state_stride[2] = per_head ? state.stride(2) : 0;
  copy_strides(p.x_stride, x, {0, 1});
  p.x_stride[2] = per_head ? x.stride(2) : 0;
  copy_strides(p.dt_stride, dt, {0, 1});
  p.A_stride[0] = A.stride(0);
  p.A_stride[1] = per_head ? 0 : A.stride(1);
  copy_strides(p.B_stride, B, {0, 1});
  copy_strides(p.C_stride, C, {0, 1});
  if (D.has_value()) {
    check_cuda(*D, x, "D");
    p.D = D->data_ptr();
    p.D_dtype = dtype_code(*D, "D");
    p.D_stride[0] = D->stride(0);
    p.D_stride[1] = D->dim() == 2 ? D->stride(1) : 0;
  }
  if (z.has_value()) {
    check_cuda(*z, x, "z");
    TORCH_CHECK(z->scalar_type() == x.scalar_type(), "z and x must have the same dtype");
    p.z = z->data_ptr();
    copy_strides(p.z_stride, *z, {0, 1});
    p.z_stride[2] = per_head ? z->stride(2) : 0;
  }
  if (dt_bias.has_value()) {
    check_cuda(*dt_bias, x, "dt_bias");
    p.dt_bias = dt_bias->data_ptr();
    p.bias_dtype = dtype_code(*dt_bias, "dt_bias");
    p.bias_stride = dt_bias->stride(0);
  }
  Tensor ih;
  p.state_indices = slots_of(state_indices, x, ih);
  Tensor out = alloc_direct(x.sizes(), x.options());
  p.out = out.data_ptr();
  check_rc(ssd_token_scan_step(&p, current_stream(x)), "ssd_token_scan_step");
  return out;
}

}  // namespace

void ssd_torch::bind_layer(pybind11::module& m) {
  m.def("add_rms_norm_fwd", &add_rms_norm_fwd);
  m.def("add_rms_norm_bwd", &add_rms_norm_bwd);
  m.def("short_conv_fwd", &short_conv_fwd);
  m.def("short_conv_bwd", &short_conv_bwd);
  m.def("short_conv_step", &short_conv_step);
  m.def("token_scan_fwd", &token_scan_fwd);
  m.def("token_scan_bwd", &token_scan_bwd);
  m.def("token_scan_step", &token_scan_step);
}
