// Host side of the operators in native code: allocate the outputs and the workspace, launch through
// the C ABI. What bounds a small call is the host (a 16-token FP8 linear: two kernels of 2.6 and 4.3
// us behind 21 us of Python), and in Python every allocation, stream look-up and ctypes call costs
// 1.5 to 3 us; here an allocate-and-launch body is one call. The checks of an operator's arguments,
// its autograd node and its module stay in Python, and every function takes the stream it launches on
// (torch's current stream of the tensors' device, as a handle). The rotary positions and the paged
// cache's operators are here as a whole, their checks and the one's autograd node too: their kernels
// take 3 to 6 us in a decode step, less than the same checks take in Python.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <sstream>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "../../../include/flower_amd.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// A status other than the caller's error (FLW_E_INVALID / FLW_E_UNSUPPORTED, a ValueError).
struct FlowerError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check(int rc, const char* what) {
  if (rc == FLW_OK) return;
  const std::string msg = flw_last_error();
  if (rc == FLW_E_INVALID || rc == FLW_E_UNSUPPORTED) throw py::value_error(std::string(what) + ": " + msg);
  throw FlowerError(std::string(what) + " failed (" + std::to_string(rc) + "): " + msg);
}

void* str(int64_t stream) { return reinterpret_cast<void*>(stream); }
int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kFloat) return FLW_F32;
  if (t.scalar_type() == at::kBFloat16) return FLW_BF16;
  throw py::value_error("unsupported dtype (float32 or bfloat16)");
}
Tensor empty(const Tensor& like, at::IntArrayRef sizes, at::ScalarType dt) {
  return at::empty(sizes, like.options().dtype(dt).requires_grad(false));
}
Tensor workspace(const Tensor& like, size_t bytes) {
  return empty(like, {(int64_t)(bytes < 256 ? 256 : bytes)}, at::kByte);
}
uint8_t* u8(const Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }
float* f32(const Tensor& t) { return static_cast<float*>(t.data_ptr()); }
uint32_t* u32(const Tensor& t) { return static_cast<uint32_t*>(t.data_ptr()); }
void* opt(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

// x as rows the kernels read in place; a copy when its columns are not contiguous or its rows not
// 16-byte aligned.
Tensor rows16(const Tensor& x) {
  return x.stride(-1) != 1 || x.stride(0) % 8 != 0 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0
             ? x.contiguous()
             : x;
}

// ---------------------------------------------------------------- quantisers of matrices

// One e4m3 scale for the matrix: codes [R, C], scale [1]. A contiguous matrix goes to the quantiser
// as a flat grid of rows of 64 to 1024 values (one chunk of 128 such rows per workgroup): the widest
// rows that still leave two chunks per compute unit, so the passes spread over the GPU whatever the
// matrix's shape while every quantising workgroup folds as few amax partials as possible.
std::tuple<Tensor, Tensor> quant_tensorwise(const Tensor& x, int64_t compute_units, int64_t stream) {
  const int64_t R = x.size(0), C = x.size(1), n = R * C;
  int64_t rows = R, cols = C, ld = x.stride(0);
  if (x.is_contiguous() && n % 64 == 0) {
    cols = 64;
    while (cols < 1024 && n % (2 * cols) == 0 && (n / (2 * cols) + 127) / 128 >= 2 * compute_units) cols *= 2;
    rows = n / cols;
    ld = cols;
  }
  Tensor codes = empty(x, {R, C}, at::kByte), scale = empty(x, {1}, at::kFloat);
  Tensor ws = workspace(x, flw_quant_workspace_bytes(1, 1, rows, cols));
  check(flw_quant_e4m3(x.data_ptr(), dtype_code(x), 1, 1, rows, cols, rows * ld, rows * ld, ld, FLW_SCALE_TENSOR,
                       FLW_LAYOUT_BHTD, u8(codes), f32(scale), ws.data_ptr(), (size_t)ws.numel(), str(stream)),
        "tensorwise e4m3");
  return {codes, scale};
}

std::tuple<Tensor, Tensor, Tensor> quant_tensor_t(const Tensor& x, int64_t ld, const OptTensor& amax, int64_t stream) {
  const int64_t R = x.size(0), C = x.size(1);
  Tensor x8 = empty(x, {R, C}, at::kByte), x8t = empty(x, {C, ld}, at::kByte), sx = empty(x, {1}, at::kFloat);
  int rc;
  if (amax) {
    rc = flw_quant_tensor_t_e4m3_amax(x.data_ptr(), R, C, x.stride(0), u32(*amax), u8(x8), C, u8(x8t), ld, f32(sx),
                                      str(stream));
  } else {
    Tensor ws = workspace(x, flw_quant_tensor_t_workspace_bytes(R, C));
    rc = flw_quant_tensor_t_e4m3(x.data_ptr(), R, C, x.stride(0), u8(x8), C, u8(x8t), ld, f32(sx), ws.data_ptr(),
                                 (size_t)ws.numel(), str(stream));
  }
  check(rc, "tensorwise e4m3 (rows and columns)");
  return {x8, x8t, sx};
}

std::tuple<Tensor, Tensor> quant_rows(const Tensor& x, const char* what, int64_t stream) {
  const int64_t R = x.size(0), C = x.size(1);
  Tensor codes = empty(x, {R, C}, at::kByte), scale = empty(x, {R}, at::kFloat);
  check(flw_quant_rows_e4m3(x.data_ptr(), dtype_code(x), R, C, x.stride(0), u8(codes), f32(scale), str(stream)), what);
  return {codes, scale};
}

std::tuple<Tensor, Tensor> quant_cols(const Tensor& x, bool per_column, int64_t ld, int64_t stream) {
  const int64_t R = x.size(0), C = x.size(1);
  Tensor codes = empty(x, {C, ld}, at::kByte), scale = empty(x, {per_column ? C : 1}, at::kFloat);
  Tensor ws = workspace(x, flw_quant_cols_workspace_bytes(R, C));
  check(flw_quant_cols_e4m3(x.data_ptr(), dtype_code(x), R, C, x.stride(0),
                            per_column ? FLW_SCALE_COLUMN : FLW_SCALE_TENSOR, u8(codes), ld, f32(scale), ws.data_ptr(),
                            (size_t)ws.numel(), str(stream)),
        "quantize_cols");
  return {codes, scale};
}

Tensor transpose_codes(const Tensor& c8, int64_t ld, int64_t stream) {
  const int64_t R = c8.size(0), C = c8.size(1);
  Tensor out = empty(c8, {C, ld}, at::kByte);
  check(flw_transpose_e4m3(u8(c8), R, C, c8.stride(0), u8(out), ld, str(stream)), "transpose codes");
  return out;
}

// ---------------------------------------------------------------- GEMMs

Tensor scaled_mm(const Tensor& a8, const Tensor& sa, const Tensor& b8, const Tensor& sb, const OptTensor& res,
                 bool may_split, int64_t stream) {
  const int64_t M = a8.size(0), K = a8.size(1), N = b8.size(0);
  Tensor y = empty(a8, {M, N}, at::kBFloat16);
  if (res) {
    check(flw_fp8_scaled_mm_residual(u8(a8), M, K, u8(b8), N, f32(sa), sa.numel(), f32(sb), sb.numel(), y.data_ptr(),
                                     N, res->data_ptr(), res->stride(0), str(stream)),
          "fp8_scaled_mm_residual");
    return y;
  }
  const size_t need = may_split ? flw_fp8_scaled_mm_workspace_bytes(M, N, K) : 0;
  if (need > 0) {
    Tensor ws = workspace(a8, need);
    check(flw_fp8_scaled_mm_ws(u8(a8), M, K, u8(b8), N, f32(sa), sa.numel(), f32(sb), sb.numel(), y.data_ptr(), N,
                               ws.data_ptr(), (size_t)ws.numel(), str(stream)),
          "fp8_scaled_mm");
  } else {
    check(flw_fp8_scaled_mm(u8(a8), M, K, u8(b8), N, f32(sa), sa.numel(), f32(sb), sb.numel(), y.data_ptr(), N,
                            str(stream)),
          "fp8_scaled_mm");
  }
  return y;
}

// The rowwise (A8W8) and weight-only (W8A16) linears on bf16 rows x [M, K].
Tensor linear(const Tensor& x, const Tensor& w8, const Tensor& w_scale, bool weight_only, int64_t stream) {
  const int64_t M = x.size(0), K = x.size(1), N = w8.size(0);
  Tensor y = empty(x, {M, N}, at::kBFloat16);
  if (weight_only) {
    check(flw_fp8_linear(x.data_ptr(), M, K, x.stride(0), u8(w8), N, f32(w_scale), w_scale.numel(), FLW_GEMM_W8A16,
                         y.data_ptr(), N, nullptr, 0, str(stream)),
          "fp8_linear(weight_only)");
  } else {
    Tensor ws = workspace(x, flw_fp8_linear_workspace_bytes(M, K, FLW_GEMM_A8W8));
    check(flw_fp8_linear(x.data_ptr(), M, K, x.stride(0), u8(w8), N, f32(w_scale), w_scale.numel(), FLW_GEMM_A8W8,
                         y.data_ptr(), N, ws.data_ptr(), (size_t)ws.numel(), str(stream)),
          "fp8_linear");
  }
  return y;
}

// ---------------------------------------------------------------- bf16 attention

std::tuple<Tensor, Tensor> swa_bf16_fwd(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window,
                                        bool token_major, const char* what, int64_t stream) {
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3);
  Tensor out = token_major ? empty(q, {B, T, H, D}, at::kBFloat16) : empty(q, {B, H, T, D}, at::kBFloat16);
  Tensor lse = empty(q, {B, H, T}, at::kFloat);
  check(flw_swa_bf16_fwd_layout(q.data_ptr(), k.data_ptr(), v.data_ptr(), B, H, T, D, window, out.data_ptr(),
                                token_major ? FLW_LAYOUT_BTHD : FLW_LAYOUT_BHTD, f32(lse), str(stream)),
        what);
  return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> swa_bf16_bwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out,
                                                const Tensor& dout, bool token_major, const Tensor& lse,
                                                int64_t window, const char* what, int64_t stream) {
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3);
  Tensor dq = empty(q, {B, H, T, D}, at::kBFloat16), dk = empty(q, {B, H, T, D}, at::kBFloat16),
         dv = empty(q, {B, H, T, D}, at::kBFloat16);
  Tensor ws = workspace(q, flw_swa_bf16_bwd_workspace_bytes(B, H, T, D));
  check(flw_swa_bf16_bwd_layout(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(),
                                token_major ? FLW_LAYOUT_BTHD : FLW_LAYOUT_BHTD, f32(lse), B, H, T, D, window,
                                dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), (size_t)ws.numel(),
                                str(stream)),
        what);
  return {dq, dk, dv};
}

// ---------------------------------------------------------------- FP8 attention

// (x, its {b, h, t} strides) readable in place: D contiguous, 16-byte rows.
Tensor in_place(const Tensor& x, int64_t* st) {
  const int64_t vec = x.scalar_type() == at::kFloat ? 4 : 8;
  auto ok = [vec](const Tensor& t) {
    return t.stride(3) == 1 && t.stride(0) % vec == 0 && t.stride(1) % vec == 0 && t.stride(2) % vec == 0 &&
           reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  };
  Tensor y = ok(x) ? x : x.contiguous();
  if (!ok(y)) throw py::value_error("cannot read the tensor in place");
  for (int i = 0; i < 3; ++i) st[i] = y.stride(i);
  return y;
}
int64_t groups(int gran, int64_t B, int64_t H) {
  return gran == FLW_SCALE_TENSOR ? 1 : gran == FLW_SCALE_HEAD ? H : B * H;
}

Tensor fp8_swa_forward(const Tensor& q0, const Tensor& k0, const Tensor& v0, int64_t window, int gran,
                       const OptTensor& out0, const OptTensor& amax, int64_t stream) {
  const int64_t B = q0.size(0), H = q0.size(1), T = q0.size(2), D = q0.size(3);
  int64_t st[12];
  Tensor q = in_place(q0, st), k = in_place(k0, st + 3), v = in_place(v0, st + 6);
  Tensor out = out0 ? *out0 : empty(q, {B, H, T, D}, q.scalar_type());
  for (int i = 0; i < 3; ++i) st[9 + i] = out.stride(i);
  Tensor ws = workspace(q, flw_fp8_swa_workspace_bytes(B, H, T, D));
  const int rc =
      amax ? flw_fp8_swa_attention_forward_amax(q.data_ptr(), k.data_ptr(), v.data_ptr(), dtype_code(q), st, B, H, T, D,
                                                window, gran, u32(*amax), out.data_ptr(), nullptr, ws.data_ptr(),
                                                (size_t)ws.numel(), str(stream))
           : flw_fp8_swa_attention_forward(q.data_ptr(), k.data_ptr(), v.data_ptr(), dtype_code(q), st, B, H, T, D,
                                           window, gran, out.data_ptr(), nullptr, ws.data_ptr(), (size_t)ws.numel(),
                                           str(stream));
  check(rc, "fp8_swa_attention_forward");
  return out;
}

// The trainable FP8 attention's forward: (out, q8, k8, V tiles, scales).
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> fp8_swa_train_fwd(const Tensor& q0, const Tensor& k0,
                                                                     const Tensor& v0, int64_t window, int gran,
                                                                     int64_t stream) {
  const int64_t B = q0.size(0), H = q0.size(1), T = q0.size(2), D = q0.size(3);
  int64_t st[9];
  Tensor q = in_place(q0, st), k = in_place(k0, st + 3), v = in_place(v0, st + 6);
  const int dt = dtype_code(q);
  const int64_t G = groups(gran, B, H);
  Tensor q8 = empty(q, {B, H, T, D}, at::kByte), k8 = empty(q, {B, H, T, D}, at::kByte);
  Tensor vt = empty(q, {(int64_t)flw_vtile_bytes(B, H, T, D)}, at::kByte), scales = empty(q, {3 * G}, at::kFloat);
  Tensor ws = workspace(q, 3 * flw_quant_workspace_bytes(B, H, T, D));
  check(flw_quant_qkv_e4m3(q.data_ptr(), k.data_ptr(), v.data_ptr(), dt, B, H, T, D, st, gran, u8(q8), u8(k8), u8(vt),
                           f32(scales), ws.data_ptr(), (size_t)ws.numel(), str(stream)),
        "fp8_swa_attention (quantise)");
  Tensor out = empty(q, {B, H, T, D}, q.scalar_type());
  const int64_t s8[3] = {H * T * D, T * D, D};
  const float* s = f32(scales);
  check(flw_fp8_swa_fwd(u8(q8), s8, u8(k8), s8, u8(vt), s, s + G, s + 2 * G, gran, out.data_ptr(), dt, s8, B, H, T, D,
                        window, str(stream)),
        "fp8_swa_attention (forward)");
  return {out, q8, k8, vt, scales};
}

// Its backward: bf16 attention, forward statistics recomputed, at the dequantised Q, K, V.
std::tuple<Tensor, Tensor, Tensor> fp8_swa_train_bwd(const Tensor& q8, const Tensor& k8, const Tensor& vt,
                                                     const Tensor& scales, const Tensor& dout, int64_t window,
                                                     int gran, int64_t stream) {
  const int64_t B = q8.size(0), H = q8.size(1), T = q8.size(2), D = q8.size(3), G = groups(gran, B, H);
  const float* s = f32(scales);
  Tensor x[3];
  const Tensor* codes[3] = {&q8, &k8, &vt};
  for (int i = 0; i < 3; ++i) {
    x[i] = empty(q8, {B, H, T, D}, at::kBFloat16);
    check(flw_dequant_e4m3(u8(*codes[i]), i == 2 ? FLW_LAYOUT_VTILE : FLW_LAYOUT_BHTD, B, H, T, D, s + i * G, gran,
                           x[i].data_ptr(), FLW_BF16, str(stream)),
          "dequantize_e4m3");
  }
  auto [o, lse] = swa_bf16_fwd(x[0], x[1], x[2], window, false, "fp8_swa_attention (recompute)", stream);
  return swa_bf16_bwd(x[0], x[1], x[2], o, dout, false, lse, window, "fp8_swa_attention (backward)", stream);
}

// ---------------------------------------------------------------- heads, norms, SwiGLU

std::tuple<Tensor, Tensor, Tensor> qkv_heads_fwd(const Tensor& y, int64_t B, int64_t T, int64_t H, bool norm, double eps,
                                                 const Tensor& cos, const Tensor& sin, int64_t ld, int64_t stream) {
  const int64_t D = y.size(-1) / (3 * H);
  Tensor q = empty(y, {B, H, T, D}, at::kBFloat16), k = empty(y, {B, H, T, D}, at::kBFloat16),
         v = empty(y, {B, H, T, D}, at::kBFloat16);
  check(flw_qkv_heads_fwd(y.data_ptr(), B, T, H, D, ld, norm, (float)eps, cos.data_ptr(), sin.data_ptr(), q.data_ptr(),
                          k.data_ptr(), v.data_ptr(), str(stream)),
        "qkv_heads");
  return {q, k, v};
}

Tensor qkv_heads_bwd(const Tensor& y, int64_t B, int64_t T, int64_t H, bool norm, double eps, const Tensor& cos,
                     const Tensor& sin, int64_t ld, const Tensor& dq, const Tensor& dk, const Tensor& dv,
                     int64_t stream) {
  const int64_t C = y.size(-1), D = C / (3 * H);
  Tensor dy = empty(y, {B, T, C}, at::kBFloat16);
  check(flw_qkv_heads_bwd(y.data_ptr(), B, T, H, D, ld, norm, (float)eps, cos.data_ptr(), sin.data_ptr(), dq.data_ptr(),
                          dk.data_ptr(), dv.data_ptr(), dy.data_ptr(), C, nullptr, nullptr, 0, str(stream)),
        "qkv_heads backward");
  return dy;
}

// RMSNorm of rows x [rows, cols], returned in `shape`; with a, of s = x + a, which is returned too
// (as rows).
std::tuple<Tensor, OptTensor> rmsnorm_fwd(const Tensor& x, const OptTensor& a, const Tensor& weight, double eps,
                                          const std::vector<int64_t>& shape, int64_t stream) {
  const int64_t R = x.size(0), C = x.size(1);
  Tensor h = empty(x, shape, at::kBFloat16);
  if (!a) {
    check(flw_rmsnorm_fwd(x.data_ptr(), R, C, x.stride(0), weight.data_ptr(), (float)eps, h.data_ptr(), C, str(stream)),
          "RMSNorm");
    return {h, std::nullopt};
  }
  Tensor s = empty(x, {R, C}, at::kBFloat16);
  check(flw_add_rmsnorm_fwd(x.data_ptr(), a->data_ptr(), R, C, x.stride(0), a->stride(0), weight.data_ptr(), (float)eps,
                            s.data_ptr(), C, h.data_ptr(), C, str(stream)),
        "residual add + RMSNorm");
  return {h, s};
}

std::tuple<Tensor, Tensor> rmsnorm_bwd(const Tensor& x, const Tensor& weight, double eps, const Tensor& dh,
                                       const OptTensor& dres, int64_t stream) {
  const int64_t R = x.size(0), C = x.size(1);
  Tensor dx = empty(x, {R, C}, at::kBFloat16), dw = empty(x, {C}, at::kBFloat16);
  Tensor ws = workspace(x, flw_rmsnorm_bwd_workspace_bytes(R, C));
  check(flw_rmsnorm_bwd(x.data_ptr(), R, C, x.stride(0), weight.data_ptr(), (float)eps, dh.data_ptr(), dh.stride(0),
                        opt(dres), dres ? dres->stride(0) : 0, dx.data_ptr(), C, dw.data_ptr(), ws.data_ptr(),
                        (size_t)ws.numel(), str(stream)),
        "RMSNorm backward");
  return {dx, dw};
}

// silu(g) * u of rows, returned in `shape`, with its maximum |h| when with_amax.
std::tuple<Tensor, OptTensor> swiglu_fwd(const Tensor& g, const Tensor& u, bool with_amax,
                                         const std::vector<int64_t>& shape, int64_t stream) {
  const int64_t R = g.size(0), C = g.size(1);
  Tensor h = empty(g, shape, at::kBFloat16);
  OptTensor amax, ws;
  if (with_amax) {
    amax = empty(g, {1}, at::kInt);
    ws = workspace(g, flw_swiglu_amax_workspace_bytes(R, C));
  }
  check(flw_swiglu_fwd(g.data_ptr(), u.data_ptr(), R, C, g.stride(0), u.stride(0), h.data_ptr(), C,
                       static_cast<uint32_t*>(opt(amax)), opt(ws), ws ? (size_t)ws->numel() : 0, str(stream)),
        "SwiGLU");
  return {h, amax};
}

std::tuple<Tensor, Tensor, OptTensor> swiglu_bwd(const Tensor& g, const Tensor& u, const Tensor& dh, bool with_amax,
                                                 int64_t stream) {
  const int64_t R = g.size(0), C = g.size(1);
  Tensor dg = empty(g, {R, C}, at::kBFloat16), du = empty(g, {R, C}, at::kBFloat16);
  OptTensor amax, ws;
  if (with_amax) {
    amax = empty(g, {2}, at::kInt);
    ws = workspace(g, flw_swiglu_amax_workspace_bytes(R, C));
  }
  check(flw_swiglu_bwd(g.data_ptr(), u.data_ptr(), R, C, g.stride(0), u.stride(0), dh.data_ptr(), dh.stride(0),
                       dg.data_ptr(), du.data_ptr(), C, static_cast<uint32_t*>(opt(amax)), opt(ws),
                       ws ? (size_t)ws->numel() : 0, str(stream)),
        "SwiGLU backward");
  return {dg, du, amax};
}

// ---------------------------------------------------------------- the fused decoder block's passes

// RMSNorm (weight given) or GELU of bf16 rows, then their per-row codes; h, when given, receives the
// normed / activated rows.
std::tuple<Tensor, Tensor> act_quant_rows(const Tensor& x, const OptTensor& weight, double eps, const OptTensor& h,
                                          int64_t stream) {
  const int64_t R = x.size(0), C = x.size(1);
  Tensor codes = empty(x, {R, C}, at::kByte), scale = empty(x, {R}, at::kFloat);
  if (weight)
    check(flw_rmsnorm_quant_rows_e4m3(x.data_ptr(), R, C, C, weight->data_ptr(), (float)eps, u8(codes), f32(scale),
                                      opt(h), str(stream)),
          "rmsnorm");
  else
    check(flw_gelu_quant_rows_e4m3(x.data_ptr(), R, C, C, u8(codes), f32(scale), opt(h), str(stream)), "gelu");
  return {codes, scale};
}

// The QKV projection with QK-norm, RoPE and the per-head maxima in its epilogue: (qkv, maxima).
std::tuple<Tensor, Tensor> qkv_norm_rope_amax(const Tensor& a8, const Tensor& sa, const Tensor& b8, const Tensor& sb,
                                              int64_t head_dim, bool norm, double eps, const Tensor& cos,
                                              const Tensor& sin, int64_t T, int64_t stream) {
  const int64_t M = a8.size(0), K = a8.size(1), N = b8.size(0);
  Tensor y = empty(a8, {M, N}, at::kBFloat16), amax = empty(a8, {N / head_dim}, at::kInt);
  check(flw_fp8_scaled_mm_qk_norm_rope_amax(u8(a8), M, K, u8(b8), N, f32(sa), sa.numel(), f32(sb), sb.numel(),
                                            y.data_ptr(), N, head_dim, N / 3 * 2, norm, (float)eps, cos.data_ptr(),
                                            sin.data_ptr(), T, u32(amax), str(stream)),
        "qkv + qk-norm + rope + amax");
  return {y, amax};
}

// ---------------------------------------------------------------- rotary positions, paged cache
// These check their arguments here and run on the device of their tensors, whichever is current.

template <typename... A>
std::string text(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  return s.str();
}
#define REFUSE_UNLESS(cond, ...) \
  do {                           \
    if (!(cond)) throw py::value_error(text(__VA_ARGS__)); \
  } while (0)

void require_gpu(const Tensor& t) {
  if (!t.is_cuda())
    throw std::runtime_error(text("flower_amd operators run only on a ROCm GPU (gfx950); got a tensor on ", t.device(),
                                  ". There is no CPU fallback."));
}
void check_ints(const char* name, const Tensor& t, at::IntArrayRef sizes, const Tensor& with) {
  REFUSE_UNLESS(t.scalar_type() == at::kInt && t.sizes() == sizes && t.is_contiguous() && t.device() == with.device(), name,
                " must be a contiguous int32 tensor ", sizes, " on ", with.device(), ", got ", t.sizes(), " ", t.scalar_type(),
                " on ", t.device());
}

// A derivative of t is asked for in reverse mode (backward); in forward mode, which no operator here has: none is dropped.
// (A tensor that autograd never touched, most of them, has no record to ask.)
bool plain(const Tensor& t) { return t.unsafeGetTensorImpl()->autograd_meta() == nullptr; }
bool wants_backward(const Tensor& t) { return !plain(t) && t.requires_grad() && c10::GradMode::is_enabled(); }
void refuse_tangent(const char* what, const Tensor& t) {
  if (!plain(t) && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
    throw std::runtime_error(text(what, " has no forward-mode derivative: call it on tensors without a tangent"));
}

int32_t* i32(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }
int32_t* i32(const OptTensor& t) { return t ? i32(*t) : nullptr; }
float* f32(const OptTensor& t) { return t ? f32(*t) : nullptr; }
int cache_code(const Tensor& pages) { return pages.scalar_type() == at::kBFloat16 ? FLW_BF16 : FLW_E4M3; }

// (B, heads, T, D) as the kernels read it, and its strides: x itself where its rows are contiguous and 16-byte aligned (a
// dimension of one may have whatever stride), else a copy.
Tensor heads(const Tensor& x, int64_t* st) {
  const int64_t vec = x.scalar_type() == at::kFloat ? 4 : 8;
  bool ok = x.stride(3) == 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (x.size(i) == 1 || x.stride(i) % vec == 0);
  Tensor y = ok ? x : x.clone(at::MemoryFormat::Contiguous);
  for (int i = 0; i < 3; ++i) st[i] = y.size(i) == 1 ? 0 : y.stride(i);
  return y;
}

void check_head_dim(int64_t D) { REFUSE_UNLESS(D == 32 || D == 64 || D == 128, "head_dim must be 32/64/128, got ", D); }

void check_rotary_tables(const Tensor& cos, const Tensor& sin, const Tensor& q) {
  REFUSE_UNLESS(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat,
                "cos and sin must be float32 [positions, rotary_dim / 2] tables of one shape, got ", cos.sizes(), " ",
                cos.scalar_type(), " and ", sin.sizes(), " ", sin.scalar_type());
  REFUSE_UNLESS(cos.size(0) > 0 && cos.is_contiguous() && sin.is_contiguous() && cos.data_ptr() != nullptr &&
                    reinterpret_cast<uintptr_t>(cos.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(sin.data_ptr()) % 16 == 0,
                "cos and sin must be contiguous, 16-byte aligned and not empty");
  const int64_t R = 2 * cos.size(1);
  REFUSE_UNLESS(R > 0 && R <= q.size(3) && R % 8 == 0, "rotary_dim must be a multiple of 8 up to the head_dim ", q.size(3),
                ", got ", R);
  REFUSE_UNLESS(cos.device() == q.device() && sin.device() == q.device(), "cos and sin must be on ", q.device());
  REFUSE_UNLESS(!wants_backward(cos) && !wants_backward(sin), "the rotary tables take no gradient");
  refuse_tangent("a rotary table", cos);
  refuse_tangent("a rotary table", sin);
}

// q, k (undefined: none) turned, contiguous: (q') or (q', k').
std::vector<Tensor> rope(const Tensor& q0, const Tensor& k0, const Tensor& cos, const Tensor& sin, const Tensor& positions,
                         bool half, bool inverse, int64_t stream) {
  c10::DeviceGuard guard(q0.device());
  int64_t st[6] = {};
  Tensor q = heads(q0, st), k;
  std::vector<Tensor> out{empty(q0, q0.sizes(), q0.scalar_type())};
  if (k0.defined()) {
    k = heads(k0, st + 3);
    out.push_back(empty(k0, k0.sizes(), k0.scalar_type()));
  }
  const bool pos = positions.defined();
  check(flw_rope(q.data_ptr(), st, q.size(1), k.defined() ? k.data_ptr() : nullptr, st + 3, k.defined() ? k.size(1) : 0,
                 dtype_code(q), q.size(0), q.size(2), q.size(3), f32(cos), f32(sin), cos.size(0), 2 * cos.size(1),
                 half ? FLW_ROPE_HALF : FLW_ROPE_INTERLEAVED, inverse, pos ? positions.data_ptr() : nullptr,
                 pos && positions.scalar_type() == at::kLong ? 64 : 32, pos && positions.dim() == 2 ? positions.stride(0) : 0,
                 out[0].data_ptr(), k.defined() ? out[1].data_ptr() : nullptr, str(stream)),
        "apply_rotary");
  return out;
}

// The rotation is linear, its gradient the opposite rotation of the gradient: the node is its own backward. The backward runs
// on the stream that the forward ran on, as torch's engine runs it.
struct RopeNode : torch::autograd::Function<RopeNode> {
  static std::vector<Tensor> forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const OptTensor& k,
                                     const Tensor& cos, const Tensor& sin, const OptTensor& positions, bool half, bool inverse,
                                     int64_t stream) {
    const Tensor pos = positions.value_or(Tensor());
    ctx->save_for_backward({cos, sin, pos});
    ctx->set_materialize_grads(false);
    ctx->saved_data["how"] = (int64_t)(half | inverse << 1 | k.has_value() << 2);
    ctx->saved_data["stream"] = stream;
    return rope(q, k.value_or(Tensor()), cos, sin, pos, half, inverse, stream);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    torch::autograd::variable_list out(8);
    const auto saved = ctx->get_saved_variables();
    const int64_t how = ctx->saved_data["how"].toInt(), stream = ctx->saved_data["stream"].toInt();
    const bool two = how & 4, q = g[0].defined(), k = two && g[1].defined();
    if (!q && !k) return out;
    for (const Tensor& t : g)
      if (t.defined()) refuse_tangent("apply_rotary's gradient", t);
    const Tensor& first = q ? g[0] : g[1];
    const bool half = (how & 1) != 0, inverse = (how & 2) == 0;
    const auto x = c10::GradMode::is_enabled()            // a gradient of the gradient may be asked for
                       ? apply(first, q && k ? OptTensor(g[1]) : OptTensor(), saved[0], saved[1],
                               saved[2].defined() ? OptTensor(saved[2]) : OptTensor(), half, inverse, stream)
                       : rope(first, q && k ? g[1] : Tensor(), saved[0], saved[1], saved[2], half, inverse, stream);
    if (q) out[0] = x[0];
    if (k) out[1] = x[q ? 1 : 0];
    return out;
  }
};

std::tuple<Tensor, OptTensor> apply_rotary(const Tensor& q, const OptTensor& k, const Tensor& cos, const Tensor& sin,
                                           const OptTensor& positions, bool half, int64_t stream) {
  REFUSE_UNLESS(q.dim() == 4 && (!k || k->dim() == 4), "expected (B, H, T, D), got ", q.sizes(), k ? text(", ", k->sizes()) : "");
  const int64_t B = q.size(0), T = q.size(2);
  REFUSE_UNLESS(!k || (k->size(0) == B && k->size(2) == T && k->size(3) == q.size(3) && k->scalar_type() == q.scalar_type() &&
                       k->device() == q.device()),
                "q and k differ: ", q.sizes(), " ", q.scalar_type(), ", ", k ? text(k->sizes(), " ", k->scalar_type()) : "");
  check_head_dim(q.size(3));
  if (q.scalar_type() != at::kBFloat16 && q.scalar_type() != at::kFloat)
    throw py::type_error(text("apply_rotary takes bfloat16 or float32 inputs; got ", q.scalar_type()));
  REFUSE_UNLESS(q.numel() > 0 && (!k || k->numel() > 0), "q and k must not be empty");
  check_rotary_tables(cos, sin, q);
  OptTensor at = positions;
  if (positions) {
    const Tensor& pos = *positions;
    const bool one = pos.dim() == 1 && pos.size(0) == T, each = pos.dim() == 2 && pos.size(0) == B && pos.size(1) == T;
    REFUSE_UNLESS((one || each) && (pos.scalar_type() == at::kInt || pos.scalar_type() == at::kLong), "positions must be int32 or "
                  "int64 (", T, ",) or (", B, ", ", T, "), got ", pos.sizes(), " ", pos.scalar_type());
    REFUSE_UNLESS(pos.device() == q.device(), "positions must be on ", q.device());
    if (T > 1 && pos.stride(-1) != 1) at = pos.contiguous();
  }
  refuse_tangent("apply_rotary", q);
  if (k) refuse_tangent("apply_rotary", *k);
  require_gpu(q);
  const bool grad = wants_backward(q) || (k && wants_backward(*k));
  const auto x = grad ? RopeNode::apply(q, k, cos, sin, at, half, false, stream)
                      : rope(q, k.value_or(Tensor()), cos, sin, at.value_or(Tensor()), half, false, stream);
  return {x[0], k ? OptTensor(x[1]) : OptTensor()};
}

// A pool of one layer (dims 4) or of all layers (dims 5).
void check_pool(const Tensor& k, const Tensor& v, int64_t dims) {
  REFUSE_UNLESS(k.dim() == dims && v.dim() == dims, "k_pages and v_pages must have ", dims, " dimensions, got ", k.sizes(), ", ",
                v.sizes());
  bool match = k.size(dims - 1) == v.size(dims - 2) && k.size(dims - 2) == v.size(dims - 1);
  for (int i = 0; i < dims - 2; ++i) match = match && k.size(i) == v.size(i);
  REFUSE_UNLESS(match, "k_pages (.., pages, kv heads, page size, D) and v_pages (.., pages, kv heads, D, page size) do not match: ",
                k.sizes(), ", ", v.sizes());
  if (k.scalar_type() != v.scalar_type() || (k.scalar_type() != at::kBFloat16 && k.scalar_type() != at::kFloat8_e4m3fn))
    throw py::type_error(text("the cache holds bfloat16 or float8_e4m3fn, got ", k.scalar_type(), " and ", v.scalar_type()));
  REFUSE_UNLESS(k.is_contiguous() && v.is_contiguous(), "k_pages and v_pages must be contiguous");
  REFUSE_UNLESS(k.device() == v.device(), "k_pages and v_pages must be on one device");
  REFUSE_UNLESS(k.numel() > 0, "the pool must not be empty");
}
void check_scales(const Tensor& k_pages, const OptTensor& k_scale, const OptTensor& v_scale) {
  if (k_pages.scalar_type() == at::kBFloat16) {
    REFUSE_UNLESS(!k_scale && !v_scale, "a bfloat16 cache takes no scales");
    return;
  }
  for (const OptTensor* t : {&k_scale, &v_scale})
    REFUSE_UNLESS(*t && (*t)->scalar_type() == at::kFloat && (*t)->dim() == 1 && (*t)->size(0) == k_pages.size(1) &&
                      (*t)->is_contiguous() && (*t)->device() == k_pages.device(),
                  "an e4m3 cache needs ", t == &k_scale ? "k_scale" : "v_scale", ", contiguous float32 (", k_pages.size(1), ",) on ",
                  k_pages.device());
}
void refuse_gradients(const char* what, const Tensor& t) {
  if (wants_backward(t))
    throw std::runtime_error(text(what, " is forward-only: call it under torch.no_grad() or on detached tensors"));
  refuse_tangent(what, t);
}
void check_tokens(const char* what, const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& tables,
                  const Tensor& lens, const OptTensor& counts, const OptTensor& k_scale, const OptTensor& v_scale) {
  check_pool(k_pages, v_pages, 4);
  REFUSE_UNLESS(q.dim() == 4, "expected (B, H, T, D), got ", q.sizes());
  if (q.scalar_type() != at::kBFloat16) throw py::type_error(text(what, " takes bfloat16 heads; got ", q.scalar_type()));
  check_head_dim(q.size(3));
  REFUSE_UNLESS(q.numel() > 0, "q must not be empty");
  REFUSE_UNLESS(q.size(3) == k_pages.size(3) && q.size(1) % k_pages.size(1) == 0, "q ", q.sizes(), " does not match the pool's ",
                k_pages.size(1), " kv heads of ", k_pages.size(3), " values");
  REFUSE_UNLESS(q.device() == k_pages.device(), "q is on ", q.device(), ", the pages on ", k_pages.device());
  REFUSE_UNLESS(tables.dim() == 2 && tables.size(0) == q.size(0) && tables.size(1) > 0, "tables must be (", q.size(0),
                ", entries), got ", tables.sizes());
  check_ints("tables", tables, tables.sizes(), q);
  check_ints("lens", lens, {q.size(0)}, q);
  if (counts) check_ints("counts", *counts, {q.size(0)}, q);
  check_scales(k_pages, k_scale, v_scale);
  for (const Tensor* t : {&q, &k_pages, &v_pages}) refuse_gradients(what, *t);
  for (const OptTensor* t : {&k_scale, &v_scale})
    if (*t) refuse_gradients(what, **t);
}

std::tuple<Tensor, OptTensor> paged_append(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& k_pages,
                                           const Tensor& v_pages, const Tensor& tables, const Tensor& lens,
                                           const OptTensor& counts, const OptTensor& cos, const OptTensor& sin, bool half,
                                           const std::optional<double>& eps, const OptTensor& k_scale,
                                           const OptTensor& v_scale, bool return_k, int64_t stream) {
  check_tokens("paged_append", q0, k_pages, v_pages, tables, lens, counts, k_scale, v_scale);
  for (const Tensor* t : {&k0, &v0}) {
    REFUSE_UNLESS(t->dim() == 4 && t->size(0) == q0.size(0) && t->size(1) == k_pages.size(1) && t->size(2) == q0.size(2) &&
                      t->size(3) == q0.size(3) && t->scalar_type() == q0.scalar_type() && t->device() == q0.device(),
                  "k and v must be (", q0.size(0), ", ", k_pages.size(1), ", ", q0.size(2), ", ", q0.size(3), ") as q, got ",
                  t->sizes(), " ", t->scalar_type());
    refuse_gradients("paged_append", *t);
  }
  REFUSE_UNLESS(cos.has_value() == sin.has_value(), "give both cos and sin, or neither");
  if (cos) check_rotary_tables(*cos, *sin, q0);
  REFUSE_UNLESS(!eps || *eps >= 0.0, "norm_eps must be non-negative");
  require_gpu(q0);
  c10::DeviceGuard guard(q0.device());
  int64_t st[9];
  Tensor q = heads(q0, st), k = heads(k0, st + 3), v = heads(v0, st + 6);
  Tensor qo = empty(q, q.sizes(), at::kBFloat16);
  OptTensor ko;
  if (return_k) ko = empty(k, k.sizes(), at::kBFloat16);
  check(flw_paged_append(q.data_ptr(), st, k.data_ptr(), st + 3, v.data_ptr(), st + 6, q.size(0), q.size(1), k.size(1), q.size(2),
                         q.size(3), k_pages.data_ptr(), v_pages.data_ptr(), cache_code(k_pages), k_pages.size(0),
                         k_pages.size(2), i32(tables), tables.size(1), i32(lens), i32(counts), eps.has_value(),
                         (float)eps.value_or(0.0), f32(cos), f32(sin), cos ? cos->size(0) : 0, cos ? 2 * cos->size(1) : 0,
                         half ? FLW_ROPE_HALF : FLW_ROPE_INTERLEAVED, f32(k_scale), f32(v_scale), qo.data_ptr(), opt(ko),
                         str(stream)),
        "paged_append");
  return {qo, ko};
}

// out (B, H, T, D), a view of token-major storage, and the log-sum-exp when asked for.
std::tuple<Tensor, OptTensor> paged_attention(const Tensor& q0, const Tensor& k_pages, const Tensor& v_pages,
                                              const Tensor& tables, const Tensor& lens, const OptTensor& counts,
                                              int64_t window, const std::optional<double>& scale, const OptTensor& k_scale,
                                              const OptTensor& v_scale, bool with_lse, int64_t stream) {
  check_tokens("paged_attention", q0, k_pages, v_pages, tables, lens, counts, k_scale, v_scale);
  require_gpu(q0);
  c10::DeviceGuard guard(q0.device());
  int64_t st[6];
  Tensor q = heads(q0, st);
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3), KV = k_pages.size(1), page = k_pages.size(2);
  Tensor out = empty(q, {B, T, H, D}, at::kBFloat16);
  st[3] = T * H * D; st[4] = D; st[5] = H * D;
  OptTensor lse, ws;
  if (with_lse) lse = empty(q, {B, H, T}, at::kFloat);
  const size_t need = flw_paged_attention_workspace_bytes(B, H, KV, T, D, cache_code(k_pages), page, tables.size(1), window);
  if (need > 0) ws = workspace(q, need);
  check(flw_paged_attention(q.data_ptr(), st, k_pages.data_ptr(), v_pages.data_ptr(), cache_code(k_pages), k_pages.size(0), page,
                            i32(tables), tables.size(1), i32(lens), i32(counts), f32(k_scale), f32(v_scale), B, H, KV, T, D,
                            window, (float)(scale ? *scale : 1.0 / std::sqrt((double)D)), out.data_ptr(), st + 3, f32(lse),
                            opt(ws), need, str(stream)),
        "paged_attention");
  return {out.transpose(1, 2), lse};
}

void check_state(const Tensor& tables, const Tensor& refs) {
  REFUSE_UNLESS(tables.dim() == 2 && refs.dim() == 1 && tables.numel() > 0 && refs.numel() > 0,
                "tables must be (S, entries) and refs (pages,), not empty, got ", tables.sizes(), ", ", refs.sizes());
  check_ints("tables", tables, tables.sizes(), tables);
  check_ints("refs", refs, refs.sizes(), tables);
}
// k_pages, v_pages of all layers (L, P, ..), or of one.
std::pair<Tensor, Tensor> all_layers(const Tensor& k, const Tensor& v, const Tensor& refs) {
  const bool one = k.dim() == 4 && v.dim() == 4;
  std::pair<Tensor, Tensor> kv = one ? std::make_pair(k.unsqueeze(0), v.unsqueeze(0)) : std::make_pair(k, v);
  check_pool(kv.first, kv.second, 5);
  REFUSE_UNLESS(kv.first.size(1) == refs.size(0) && k.device() == refs.device(), "the pool ", k.sizes(), " on ", k.device(),
                " is not of refs' ", refs.size(0), " pages");
  return kv;
}
// The tensors to write: `out`, one for each input (each may be that input, but overlap no other), or new ones.
std::vector<Tensor> outputs(const std::optional<std::vector<Tensor>>& out, const std::vector<Tensor>& in, const Tensor& arg) {
  std::vector<Tensor> to;
  if (!out) {
    for (const Tensor& t : in) to.push_back(empty(t, t.sizes(), at::kInt));
    return to;
  }
  REFUSE_UNLESS(out->size() == in.size(), "out takes ", in.size(), " tensors, got ", out->size());
  auto overlap = [](const Tensor& a, const Tensor& b) {
    return i32(a) < i32(b) + b.numel() && i32(b) < i32(a) + a.numel();
  };
  for (size_t i = 0; i < in.size(); ++i) {
    const Tensor& o = (*out)[i];
    check_ints("out", o, in[i].sizes(), in[i]);
    bool bad = arg.defined() && overlap(o, arg);
    for (size_t j = 0; j < in.size(); ++j)
      bad = bad || (overlap(o, in[j]) && !(i == j && i32(o) == i32(in[j]))) || (j < i && overlap(o, (*out)[j]));
    REFUSE_UNLESS(!bad, "an output may be its own input, and overlap nothing else");
  }
  return *out;
}

using OutTensors = std::optional<std::vector<Tensor>>;

std::tuple<Tensor, Tensor, Tensor, Tensor> reserve_pages(const Tensor& tables, const Tensor& lens, const Tensor& refs,
                                                         const Tensor& counts, int64_t page, const std::optional<int64_t>& window,
                                                         const OutTensors& out, int64_t stream) {
  check_state(tables, refs);
  const int64_t S = tables.size(0), P = refs.size(0);
  check_ints("lens", lens, {S}, tables);
  check_ints("counts", counts, {S}, tables);
  REFUSE_UNLESS(!window || *window > 0, "window must be positive");
  require_gpu(tables);
  const std::vector<Tensor> to = outputs(out, {tables, lens, refs}, counts);
  c10::DeviceGuard guard(tables.device());
  Tensor granted = empty(lens, {S}, at::kInt), ws = workspace(lens, flw_reserve_pages_workspace_bytes(S, P));
  check(flw_reserve_pages(i32(tables), i32(lens), i32(refs), i32(counts), S, tables.size(1), P, page, window.value_or(0), i32(to[0]),
                          i32(to[1]), i32(to[2]), i32(granted), ws.data_ptr(), (size_t)ws.numel(), str(stream)),
        "reserve_pages");
  return {to[0], to[1], to[2], granted};
}

std::tuple<Tensor, Tensor, Tensor, OptTensor> reorder_pages(const Tensor& k_pages, const Tensor& v_pages, const Tensor& tables,
                                                            const Tensor& lens, const Tensor& refs, const Tensor& parents,
                                                            const OutTensors& out, bool with_kept, int64_t stream) {
  check_state(tables, refs);
  const int64_t S = tables.size(0), M = tables.size(1), P = refs.size(0);
  check_ints("lens", lens, {S}, tables);
  check_ints("parents", parents, {S}, tables);
  const auto [k, v] = all_layers(k_pages, v_pages, refs);
  require_gpu(tables);
  const std::vector<Tensor> to = outputs(out, {tables, lens, refs}, parents);
  c10::DeviceGuard guard(tables.device());
  Tensor ws = workspace(lens, flw_reorder_pages_workspace_bytes(S, M, P));
  OptTensor kept;
  if (with_kept) kept = empty(lens, {S}, at::kInt);
  check(flw_reorder_pages_kept(k.data_ptr(), v.data_ptr(), cache_code(k), k.size(0), P, k.size(2), k.size(3), k.size(4),
                               i32(tables), i32(lens), i32(refs), i32(parents), S, M, i32(to[0]), i32(to[1]), i32(to[2]),
                               i32(kept), ws.data_ptr(), (size_t)ws.numel(), str(stream)),
        "reorder_pages");
  return {to[0], to[1], to[2], kept};
}

std::tuple<Tensor, Tensor, Tensor> compact_pages(const Tensor& k_pages, const Tensor& v_pages, const Tensor& tables,
                                                 const Tensor& refs, const OutTensors& out, int64_t stream) {
  check_state(tables, refs);
  const auto [k, v] = all_layers(k_pages, v_pages, refs);
  require_gpu(tables);
  const int64_t P = refs.size(0);
  const std::vector<Tensor> to = outputs(out, {tables, refs}, Tensor());
  c10::DeviceGuard guard(tables.device());
  Tensor live = empty(refs, {1}, at::kInt), ws = workspace(refs, flw_compact_pages_workspace_bytes(P));
  check(flw_compact_pages(k.data_ptr(), v.data_ptr(), cache_code(k), k.size(0), P, k.size(2), k.size(3), k.size(4), i32(tables),
                          i32(refs), tables.size(0), tables.size(1), i32(to[0]), i32(to[1]), i32(live), ws.data_ptr(),
                          (size_t)ws.numel(), str(stream)),
        "compact_pages");
  return {to[0], to[1], live};
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.attr("torch_version") = FLW_TORCH_VERSION;   // compared at load: tensors cross here in that build's layout
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const FlowerError& e) {
      py::object type = py::module_::import("flower_amd._lib").attr("FlowerError");
      PyErr_SetString(type.ptr(), e.what());
    }
  });
  // The GIL is let go while a body allocates and launches, as torch's own operators do.
  using nogil = py::call_guard<py::gil_scoped_release>;
  m.def("rows16", &rows16, nogil());
  m.def("quant_tensorwise", &quant_tensorwise, nogil());
  m.def("quant_tensor_t", &quant_tensor_t, nogil());
  m.def("quant_rows", &quant_rows, nogil());
  m.def("quant_cols", &quant_cols, nogil());
  m.def("transpose_codes", &transpose_codes, nogil());
  m.def("scaled_mm", &scaled_mm, nogil());
  m.def("linear", &linear, nogil());
  m.def("swa_bf16_fwd", &swa_bf16_fwd, nogil());
  m.def("swa_bf16_bwd", &swa_bf16_bwd, nogil());
  m.def("fp8_swa_forward", &fp8_swa_forward, nogil());
  m.def("fp8_swa_train_fwd", &fp8_swa_train_fwd, nogil());
  m.def("fp8_swa_train_bwd", &fp8_swa_train_bwd, nogil());
  m.def("qkv_heads_fwd", &qkv_heads_fwd, nogil());
  m.def("qkv_heads_bwd", &qkv_heads_bwd, nogil());
  m.def("rmsnorm_fwd", &rmsnorm_fwd, nogil());
  m.def("rmsnorm_bwd", &rmsnorm_bwd, nogil());
  m.def("swiglu_fwd", &swiglu_fwd, nogil());
  m.def("swiglu_bwd", &swiglu_bwd, nogil());
  m.def("act_quant_rows", &act_quant_rows, nogil());
  m.def("qkv_norm_rope_amax", &qkv_norm_rope_amax, nogil());
  m.def("apply_rotary", &apply_rotary, nogil());
  m.def("paged_append", &paged_append, nogil());
  m.def("paged_attention", &paged_attention, nogil());
  m.def("reserve_pages", &reserve_pages, nogil());
  m.def("reorder_pages", &reorder_pages, nogil());
  m.def("compact_pages", &compact_pages, nogil());
}
