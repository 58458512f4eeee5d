// Rows of activations or weights in 8 bits with one fp32 scale a row, straight from what produces them:
//   h = x | rmsnorm(x) w | rmsnorm(x + a) w | gelu(x) | silu(x) b
//   s = max(max|h| / Q, 1e-12), Q = 127 (int8) or 448 (e4m3);  code = rne(h / s), the quotient in fp32.
// The sum x + a is the residual stream: it is rounded to x's type, written, and the norm is of the rounded sum, which is what
// the next layer and a backward pass read. h itself stays in fp32 up to its code: rounded to bf16 first, as the separate norm
// and cast would, values near the row's maximum were off by half an int8 step more. e4m3 codes of h can therefore differ in
// the last place from flw_rmsnorm_quant_rows_e4m3's, which keeps that rounding.
// int8 holds no NaN: a row whose maximum is not finite gets the scale NaN and codes 0, so its products are NaN. e4m3 rows
// do as flw_quant_rows_e4m3's.
//
// One pass over memory. A row is held by LPR lanes (64, 256 or 1024 threads), each up to four chunks of 8 values in
// registers, between the loads, the sum of squares, the maximum and the codes; wider rows are refused. Bound by HBM for many rows
// ([65536, 4096] into int8: as they are 134 us, 6.0 TB/s, addition and norm 314, 6.0, SwiGLU 228, 5.9), norm alone (168, 4.8) and GELU
// (209, 3.9) by what the vector unit issues; by the latency of load, reduction, reduction, store for few.
#include "flw_common.h"

namespace flw {

constexpr int kRows8None = 0, kRows8Norm = 1, kRows8AddNorm = 2, kRows8Gelu = 3, kRows8Swiglu = 4;
constexpr int64_t kRows8MaxCols = 32768;

struct Rows8Params {
  const void* x;
  const void* b;           // the residual's addend (AddNorm), or up (Swiglu)
  const void* w;           // norm weight
  void* sum;               // x + b (AddNorm)
  uint8_t* codes;          // [rows, cols], row stride cs
  float* scale;
  int64_t rows, xs, bs, ss, cs;
  int cols;
  float eps;
  int w32;                 // the weight is fp32 beside bf16 rows
  int e4m3;
};

// 8 values from column c (c < cols) of a row, zeros past the row's end. ALIGNED: cols % 8 == 0 and 16-byte rows; else the
// loads are by element-aligned vectors (which gfx950 takes at any address), the row's last values one by one.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void rows8_load(const T* row, int c, int cols, float* f) {
  struct __attribute__((packed, aligned(sizeof(T)))) V { uint32_t w[4]; };
  constexpr int N = Vec16<T>::N;
  if (ALIGNED || c + 8 <= cols) {
#pragma unroll
    for (int j = 0; j < 8; j += N) {
      uint4 q;
      if constexpr (ALIGNED) {
        q = *reinterpret_cast<const uint4*>(row + c + j);
      } else {
        const V v = *reinterpret_cast<const V*>(row + c + j);
        q = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
      }
      Vec16<T>::unpack(q, f + j);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v = 0.0f;
      if (c + j < cols) {
        if constexpr (sizeof(T) == 2) v = bf16_to_f32(row[c + j]);
        else v = row[c + j];
      }
      f[j] = v;
    }
  }
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void rows8_store(T* row, int c, int cols, const float* f) {
  if constexpr (ALIGNED && sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(row + c) = make_uint4(bf16x2_rne(f[0], f[1]), bf16x2_rne(f[2], f[3]), bf16x2_rne(f[4], f[5]),
                                                    bf16x2_rne(f[6], f[7]));
  } else if constexpr (ALIGNED) {
    *reinterpret_cast<float4*>(row + c) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(row + c + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else if (c + 8 <= cols) {
    struct __attribute__((packed, aligned(sizeof(T)))) V { uint32_t w[2 * sizeof(T)]; } v;
#pragma unroll
    for (int j = 0; j < 8; j += 4 / sizeof(T)) {
      if constexpr (sizeof(T) == 2) v.w[j / 2] = bf16x2_rne(f[j], f[j + 1]);
      else v.w[j] = __float_as_uint(f[j]);
    }
    *reinterpret_cast<V*>(row + c) = v;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < cols) {
        if constexpr (sizeof(T) == 2) row[c + j] = (uint16_t)f32_to_bf16_bits(f[j]);
        else row[c + j] = f[j];
      }
  }
}

// x / (1 + exp(-x)): the exponent -x / ln 2 as a rounded product and what the rounding and the constant leave, which the power
// takes as a factor 1 + ln 2 * rest; the quotient by a reciprocal and one correction. x from 87 on, and 0 (|silu| < 2e-36) below
// -87, infinities included: between, fp32 holds the power and its inverse. [65536, 4096]: 228 us into int8 (5.9 TB/s), 256 with expf.
__device__ __forceinline__ float silu(float x) {
  constexpr float L = 1.44269502162933350f, REST = 1.92596298e-8f, LN2 = 0.69314718f;            // 1 / ln 2 = L + REST
  const float hi = -x * L, lo = fmaf(-x, REST, fmaf(-x, L, -hi)), e = __builtin_amdgcn_exp2f(hi);
  const float d = 1.0f + fmaf(e, lo * LN2, e), r = __builtin_amdgcn_rcpf(d), q = x * r, v = fmaf(fmaf(-q, d, x), r, q);
  return x > 87.0f ? x : x < -87.0f ? 0.0f : v;
}

// x Phi(x) = max(x, 0) - |x| Q(|x|), where Q(z) = 1 - Phi(z) = exp(-z^2 / 2) R(z). R is smooth and slow, as 1 / z is: a polynomial of
// degree 9 in t = 1 / (1 + z / 4), fitted to z <= 14 (relative error 2.8e-8 with its coefficients in fp32; Q(14) is below fp32). One
// exponential, one reciprocal with its correction and 9 products, where erff takes a wave of mixed values through both of its
// ranges. Of normal bf16 values a result is off by 6e-8 of itself on average, 7e-7 at most (0.5 x (1 + erf): 2.9e-7, and a third of
// itself at x = -5, where the sum cancels). -inf gives the limit, 0. [32768, 4096] into e4m3: 119 us, 129 with erff.
__device__ __forceinline__ float gelu(float x) {
  const float z = fminf(fabsf(x), 16.0f), d = fmaf(0.25f, z, 1.0f);
  float t = __builtin_amdgcn_rcpf(d), r = 0.033946678042411804f;
  t = fmaf(fmaf(-d, t, 1.0f), t, t);
  r = fmaf(r, t, -0.19617709517478943f);
  r = fmaf(r, t, 0.3950009346008301f);
  r = fmaf(r, t, -0.33346861600875854f);
  r = fmaf(r, t, 0.30448636412620544f);
  r = fmaf(r, t, -0.020383795723319054f);
  r = fmaf(r, t, 0.12156785279512405f);
  r = fmaf(r, t, 0.09482026845216751f);
  r = fmaf(r, t, 0.10022899508476257f);
  r = fmaf(r, t, -2.1599986212095246e-05f);
  return fmaf(-z * __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f), r, x < 0.0f ? 0.0f : x);
}

// One value of every lane of a row, combined over the row's LPR lanes (the same bits in all of them).
template <int LPR, typename F>
__device__ __forceinline__ uint32_t rows8_reduce(uint32_t v, uint32_t* red, F f) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = f(v, (uint32_t)__shfl_xor((int)v, o, 64));
  if constexpr (LPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < LPR / 64; ++i) v = f(v, red[i]);
  }
  return v;
}

template <typename T, int OP, int LPR, int NC, bool ALIGNED>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void rows8_kernel(Rows8Params p) {
  __shared__ uint32_t red[2][LPR > 64 ? LPR / 64 : 1];
  constexpr int RPB = LPR > 64 ? 1 : 4;            // rows a workgroup
  const int64_t row = (int64_t)blockIdx.x * RPB + (RPB > 1 ? threadIdx.x / LPR : 0);
  if (row >= p.rows) return;                       // uniform over a row's lanes
  const int lane = threadIdx.x % LPR, cols = p.cols;
  const T* x = static_cast<const T*>(p.x) + row * p.xs;
  float f[NC][8];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = 8 * (lane + LPR * i);
    if (c < cols) {
      rows8_load<T, ALIGNED>(x, c, cols, f[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[i][e] = 0.0f;
    }
  }
  if constexpr (OP == kRows8AddNorm || OP == kRows8Swiglu) {
    const T* b = static_cast<const T*>(p.b) + row * p.bs;
    float g[NC][8];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = 8 * (lane + LPR * i);
      if (c < cols) rows8_load<T, ALIGNED>(b, c, cols, g[i]);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = 8 * (lane + LPR * i);
      if (c >= cols) continue;
      if constexpr (OP == kRows8AddNorm) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i][e] = round_to<T>(f[i][e] + g[i][e]);
        rows8_store<T, ALIGNED>(static_cast<T*>(p.sum) + row * p.ss, c, cols, f[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i][e] = silu(f[i][e]) * g[i][e];
      }
    }
  }
  if constexpr (OP == kRows8Norm || OP == kRows8AddNorm) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(f[i][e], f[i][e], ss);
    ss = __uint_as_float(rows8_reduce<LPR>(__float_as_uint(ss), red[0], [](uint32_t a, uint32_t b) {
      return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
    const float r = 1.0f / __builtin_sqrtf(ss / (float)cols + p.eps);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = 8 * (lane + LPR * i);
      if (c >= cols) continue;
      float g[8];
      if (sizeof(T) == 2 && p.w32) rows8_load<float, ALIGNED>(static_cast<const float*>(p.w), c, cols, g);
      else rows8_load<T, ALIGNED>(static_cast<const T*>(p.w), c, cols, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[i][e] = f[i][e] * r * g[e];
    }
  }
  if constexpr (OP == kRows8Gelu) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) f[i][e] = gelu(f[i][e]);
  }
  uint32_t m = 0;                                  // |h| as bit patterns: NaN above infinity above the rest
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) { const uint32_t a = abs_bits(f[i][e]); m = m > a ? m : a; }
  m = rows8_reduce<LPR>(m, red[1], [](uint32_t a, uint32_t b) { return a > b ? a : b; });
  uint8_t* dst = p.codes + row * p.cs;
  const Int8Scale s8(m);
  float s = s8.scale;
  if (p.e4m3) {
    s = __uint_as_float(m) / kE4m3Max;
    s = s < kEps ? kEps : s;                       // NaN stays
  }
  if (lane == 0) p.scale[row] = s;
  const float rcp = 1.0f / s;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = 8 * (lane + LPR * i);
    if (c >= cols) continue;
    uint32_t w[2] = {0, 0};
    if (!p.e4m3) {
      const uint2 t = s8.codes(f[i]);
      w[0] = t.x; w[1] = t.y;
    } else if (s8.finite) {
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        int t = __builtin_amdgcn_cvt_pk_fp8_f32(div_by_scale(f[i][e], s, rcp), div_by_scale(f[i][e + 1], s, rcp), 0, false);
        w[e >> 2] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(div_by_scale(f[i][e + 2], s, rcp), div_by_scale(f[i][e + 3], s, rcp),
                                                             t, true);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e >> 2] |= (f32_to_e4m3(f[i][e] / s) & 0xFFu) << (8 * (e & 3));
    }
    if constexpr (ALIGNED) {
      *reinterpret_cast<uint2*>(dst + c) = make_uint2(w[0], w[1]);
    } else if (c + 8 <= cols) {
      struct __attribute__((packed, aligned(1))) V { uint32_t w[2]; };
      *reinterpret_cast<V*>(dst + c) = V{w[0], w[1]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < cols) dst[c + e] = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
    }
  }
}

// Column sums of bf16 rows (a bias's gradient), in two passes of a fixed order: each workgroup sums 512 columns (8 a lane) of
// a chunk of rows, its four waves every fourth row, into part [chunks][cols]; then the chunks of each column are summed. Chunks of
// 128 rows, of 32 for few rows, which 128 would leave to a few workgroups (both launches, us, at 32 / 128: [64, 1280] 4.5 / 4.9,
// [517, 1280] 4.8 / 5.9, [2048, 3840] 6.3 / 6.6, [4096, 5120] 12.6 / 10.2; [16384, 5120] 28.8, 5.8 TB/s).
constexpr int64_t sum_rows(int64_t rows) { return rows <= 2048 ? 32 : 128; }

template <bool ALIGNED>
__global__ __launch_bounds__(256) void col_sum_kernel(const uint16_t* __restrict__ x, int64_t rows, int cols, int64_t xs,
                                                      int chunk, float* __restrict__ part) {
  __shared__ float fold[3][512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 512 + 8 * lane;
  const int64_t r1 = min(rows, (int64_t)(blockIdx.y + 1) * chunk);
  float acc[8] = {};
  if (c < cols) {
#pragma unroll 4
    for (int64_t r = (int64_t)blockIdx.y * chunk + wave; r < r1; r += 4) {
      float f[8];
      rows8_load<uint16_t, ALIGNED>(x + r * xs, c, cols, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += f[e];
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) fold[wave - 1][64 * e + lane] = acc[e];
  }
  __syncthreads();
  if (wave > 0 || c >= cols) return;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (c + e < cols)
      part[(int64_t)blockIdx.y * cols + c + e] = ((acc[e] + fold[0][64 * e + lane]) + fold[1][64 * e + lane]) + fold[2][64 * e + lane];
}

// 16 columns a workgroup, 16 slices of the chunks each.
__global__ __launch_bounds__(256) void col_sum_fold_kernel(const float* __restrict__ part, int chunks, int cols, void* __restrict__ out,
                                                           int out32) {
  __shared__ float red[16][17];
  const int cl = threadIdx.x & 15, s = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  float a = 0.0f;
  if (c < cols)
    for (int k = s; k < chunks; k += 16) a += part[(int64_t)k * cols + c];
  red[s][cl] = a;
  __syncthreads();
  if (s > 0 || c >= cols) return;
#pragma unroll
  for (int j = 1; j < 16; ++j) a += red[j][cl];
  if (out32) static_cast<float*>(out)[c] = a;
  else static_cast<uint16_t*>(out)[c] = (uint16_t)f32_to_bf16_bits(a);
}

template <typename T, int OP, bool ALIGNED>
static const void* rows8_of(int lpr, int nc) {
#define FLW_ROWS8(L, N) reinterpret_cast<const void*>(&rows8_kernel<T, OP, L, N, ALIGNED>)
  static const void* const table[3][4] = {{FLW_ROWS8(64, 1), FLW_ROWS8(64, 2), FLW_ROWS8(64, 3), FLW_ROWS8(64, 4)},
                                          {FLW_ROWS8(256, 1), FLW_ROWS8(256, 2), FLW_ROWS8(256, 3), FLW_ROWS8(256, 4)},
                                          {FLW_ROWS8(1024, 1), FLW_ROWS8(1024, 2), FLW_ROWS8(1024, 3), FLW_ROWS8(1024, 4)}};
#undef FLW_ROWS8
  return table[lpr == 64 ? 0 : lpr == 256 ? 1 : 2][nc - 1];
}

static bool rows_ok(const void* p, int64_t stride, int64_t cols, size_t size) {
  return p != nullptr && stride >= cols && (uintptr_t)p % size == 0;
}
static bool rows16(const void* p, int64_t stride, size_t size) {
  return p == nullptr || ((uintptr_t)p % 16 == 0 && stride * (int64_t)size % 16 == 0);
}

template <int OP>
static int rows8(Rows8Params p, int dtype, int64_t cols, int weight_dtype, int code_type, void* stream, const char* name) {
  FLW_REQUIRE(dtype == FLW_F32 || dtype == FLW_BF16, FLW_E_UNSUPPORTED, "dtype %d not supported (f32=0, bf16=1)", dtype);
  FLW_REQUIRE(code_type == FLW_I8 || code_type == FLW_E4M3, FLW_E_UNSUPPORTED, "codes must be int8 or e4m3, got %d", code_type);
  FLW_REQUIRE(p.rows >= 0 && cols > 0, FLW_E_INVALID, "empty or negative shape (%lld, %lld)", (long long)p.rows, (long long)cols);
  FLW_REQUIRE(cols <= kRows8MaxCols, FLW_E_UNSUPPORTED, "rows of at most %lld values, got %lld", (long long)kRows8MaxCols,
              (long long)cols);
  FLW_REQUIRE(p.rows <= 0x7FFFFFFFll, FLW_E_UNSUPPORTED, "too many rows");
  const size_t size = dtype == FLW_F32 ? 4 : 2;
  if (p.rows == 0) return FLW_OK;
  FLW_REQUIRE(rows_ok(p.x, p.xs, cols, size) && rows_ok(p.codes, p.cs, cols, 1) && rows_ok(p.scale, cols, cols, 4), FLW_E_INVALID,
              "null or misaligned pointer, or a row stride below the row");
  if (OP == kRows8AddNorm || OP == kRows8Swiglu)
    FLW_REQUIRE(rows_ok(p.b, p.bs, cols, size), FLW_E_INVALID, "the second input: null, misaligned, or a row stride below the row");
  if (OP == kRows8AddNorm)
    FLW_REQUIRE(rows_ok(p.sum, p.ss, cols, size), FLW_E_INVALID, "the sum: null, misaligned, or a row stride below the row");
  if (OP == kRows8Norm || OP == kRows8AddNorm) {
    FLW_REQUIRE(weight_dtype == dtype || weight_dtype == FLW_F32, FLW_E_UNSUPPORTED, "the weight must be fp32 or of the rows' type");
    p.w32 = weight_dtype == FLW_F32;
    FLW_REQUIRE(rows_ok(p.w, cols, cols, p.w32 ? 4 : 2), FLW_E_INVALID, "the weight is null or misaligned");
    FLW_REQUIRE(p.eps >= 0.0f, FLW_E_INVALID, "eps must be non-negative");
  }
  p.cols = (int)cols;
  p.e4m3 = code_type == FLW_E4M3;
  const bool aligned = cols % 8 == 0 && rows16(p.x, p.xs, size) && rows16(p.b, p.bs, size) && rows16(p.sum, p.ss, size) &&
                       rows16(p.w, 0, 4) && (uintptr_t)p.codes % 8 == 0 && p.cs % 8 == 0;
  // The fewest lanes whose four chunks hold the row, and more for few rows, where a row's latency counts and no lane is missed
  // elsewhere (us, on 64 / 256 lanes: addnorm [1, 1280] 4.4 / 3.1, [1024, 1280] 5.6 / 4.4, [8192, 1280] 17.6 / 17.9, norm there
  // 10.2 / 12.6; on 256 / 1024: addnorm [24, 3392] 4.3 / 3.7, [1024, 4096] 9.3 / 10.2).
  const int lpr = cols <= 512 || (cols <= 2048 && p.rows > 2048) ? 64 : cols <= 2048 || (cols <= 8192 && p.rows > 128) ? 256 : 1024;
  const int nc = (int)((cols + 8 * lpr - 1) / (8 * lpr));
  const void* kernel = dtype == FLW_F32 ? (aligned ? rows8_of<float, OP, true>(lpr, nc) : rows8_of<float, OP, false>(lpr, nc))
                                        : (aligned ? rows8_of<uint16_t, OP, true>(lpr, nc) : rows8_of<uint16_t, OP, false>(lpr, nc));
  const int64_t rpb = lpr == 64 ? 4 : 1, groups = (p.rows + rpb - 1) / rpb, threads = lpr == 64 ? 256 : lpr;
  FLW_REQUIRE(groups * threads <= 0xFFFFFFFFll, FLW_E_UNSUPPORTED, "too many rows");       // a launch holds fewer than 2^32 threads
  (void)launch_timed(kernel, dim3((unsigned)groups), dim3((unsigned)threads), static_cast<hipStream_t>(stream), p);
  return check_launch(name);
}

}  // namespace flw

using namespace flw;

extern "C" int flw_rows8(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_row_stride, int code_type, void* codes,
                         int64_t codes_row_stride, float* scale, void* stream) {
  Rows8Params p{};
  p.x = x; p.rows = rows; p.xs = x_row_stride; p.codes = static_cast<uint8_t*>(codes); p.cs = codes_row_stride; p.scale = scale;
  return rows8<kRows8None>(p, dtype, cols, dtype, code_type, stream, "flw_rows8");
}

extern "C" int flw_rows8_rmsnorm(const void* x, const void* residual, int dtype, int64_t rows, int64_t cols, int64_t x_row_stride,
                                 int64_t residual_row_stride, const void* weight, int weight_dtype, float eps, void* sum,
                                 int64_t sum_row_stride, int code_type, void* codes, int64_t codes_row_stride, float* scale,
                                 void* stream) {
  Rows8Params p{};
  p.x = x; p.rows = rows; p.xs = x_row_stride; p.codes = static_cast<uint8_t*>(codes); p.cs = codes_row_stride; p.scale = scale;
  p.w = weight; p.eps = eps;
  if (residual == nullptr) return rows8<kRows8Norm>(p, dtype, cols, weight_dtype, code_type, stream, "flw_rows8_rmsnorm");
  p.b = residual; p.bs = residual_row_stride; p.sum = sum; p.ss = sum_row_stride;
  return rows8<kRows8AddNorm>(p, dtype, cols, weight_dtype, code_type, stream, "flw_rows8_rmsnorm");
}

extern "C" int flw_rows8_gelu(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_row_stride, int code_type,
                              void* codes, int64_t codes_row_stride, float* scale, void* stream) {
  Rows8Params p{};
  p.x = x; p.rows = rows; p.xs = x_row_stride; p.codes = static_cast<uint8_t*>(codes); p.cs = codes_row_stride; p.scale = scale;
  return rows8<kRows8Gelu>(p, dtype, cols, dtype, code_type, stream, "flw_rows8_gelu");
}

extern "C" int flw_rows8_swiglu(const void* gate, const void* up, int dtype, int64_t rows, int64_t cols, int64_t gate_row_stride,
                                int64_t up_row_stride, int code_type, void* codes, int64_t codes_row_stride, float* scale,
                                void* stream) {
  Rows8Params p{};
  p.x = gate; p.rows = rows; p.xs = gate_row_stride; p.codes = static_cast<uint8_t*>(codes); p.cs = codes_row_stride; p.scale = scale;
  p.b = up; p.bs = up_row_stride;
  return rows8<kRows8Swiglu>(p, dtype, cols, dtype, code_type, stream, "flw_rows8_swiglu");
}

static int64_t sum_chunks(int64_t rows) { return (rows + sum_rows(rows) - 1) / sum_rows(rows); }

extern "C" size_t flw_col_sum_workspace_bytes(int64_t rows, int64_t cols) {
  return rows <= 0 || cols <= 0 ? 0 : (size_t)(sum_chunks(rows) * cols * 4);
}

extern "C" int flw_col_sum(const void* x, int64_t rows, int64_t cols, int64_t x_row_stride, void* out, int out_dtype, void* workspace,
                           size_t workspace_bytes, void* stream) {
  FLW_REQUIRE(rows > 0 && cols > 0, FLW_E_INVALID, "empty or negative shape (%lld, %lld)", (long long)rows, (long long)cols);
  FLW_REQUIRE(cols <= 0x7FFFFE00ll && sum_chunks(rows) <= 65535, FLW_E_UNSUPPORTED, "too many rows or columns");
  FLW_REQUIRE(out_dtype == FLW_F32 || out_dtype == FLW_BF16, FLW_E_UNSUPPORTED, "dtype %d not supported (f32=0, bf16=1)", out_dtype);
  FLW_REQUIRE(rows_ok(x, x_row_stride, cols, 2) && rows_ok(out, cols, cols, out_dtype == FLW_F32 ? 4 : 2), FLW_E_INVALID,
              "null or misaligned pointer, or a row stride below the row");
  const size_t need = flw_col_sum_workspace_bytes(rows, cols);
  FLW_REQUIRE(workspace_bytes >= need && workspace != nullptr && (uintptr_t)workspace % 16 == 0, FLW_E_WORKSPACE,
              "workspace needs %zu bytes (16-byte aligned), got %zu", need, workspace_bytes);
  const int chunks = (int)sum_chunks(rows);
  const bool aligned = cols % 8 == 0 && rows16(x, x_row_stride, 2);
  const Timer tm = take_timer();
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* part = static_cast<float*>(workspace);
  (void)launch_args(aligned ? reinterpret_cast<const void*>(&col_sum_kernel<true>) : reinterpret_cast<const void*>(&col_sum_kernel<false>),
                    dim3((unsigned)((cols + 511) / 512), (unsigned)chunks), dim3(256), 0, s, tm.start, nullptr,
                    static_cast<const uint16_t*>(x), rows, (int)cols, x_row_stride, (int)sum_rows(rows), part);
  (void)launch_args(reinterpret_cast<const void*>(&col_sum_fold_kernel), dim3((unsigned)((cols + 15) / 16)), dim3(256), 0, s, nullptr,
                    tm.stop, static_cast<const float*>(part), chunks, (int)cols, out, (int)(out_dtype == FLW_F32));
  return check_launch("flw_col_sum");
}
