// The 8-bit integer linear for gfx950: y[M, N] (bf16) = (a[M, K] . b[N, K]^T) sa[m] sb[n] + bias[n], then residual + y.
//
// The products are summed in int32 by the integer MFMA, exactly (|a b| <= 2^14, K <= 131071), so that every tile and every
// split of K gives the same bits; one conversion to fp32 and two products follow. y is rounded to bf16 before the
// residual is added, and the sum again, as the block's separate linear and add round.
//
// Both operands lie along K. An MFMA only needs a and b to agree on which k a lane's byte is, so the 32 consecutive bytes of a
// row that a lane holds (half h = lane / 32 of a 64-deep chunk) feed two v_mfma_i32_32x32x32_i8, 16 bytes each. The product is
// taken transposed, C^T = b a^T: a lane of the 32 x 32 accumulator owns one output row m and n = 8 g + 4 h + 0..3.
#include "flw_common.h"

namespace flw {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

struct Int8Params {
  const int8_t* a;         // [M, K], row stride as
  const int8_t* b;         // [N, K], row stride bs
  int64_t as, bs;
  const float* sa;         // M or 1
  const float* sb;         // N or 1
  int sa_step, sb_step;
  const void* bias;        // N, fp32 or bf16, or null
  int bias32;
  const uint16_t* res;     // [M, N], row stride rs, or null
  int64_t rs;
  uint16_t* y;             // [M, N], row stride ys
  int64_t ys;
  int M, N, K;
  int tiles_n, tiles_m;
};

// 16 bytes of row p from k on, zeros past K. Any alignment.
__device__ __forceinline__ uint4 load_k16(const int8_t* p, int k, int K) {
  struct __attribute__((packed, aligned(1))) V { uint32_t w[4]; };
  if (k + 16 <= K) {
    const V v = *reinterpret_cast<const V*>(p + k);
    return make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
  }
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (k + j < K) w[j >> 2] |= (uint32_t)(uint8_t)p[k + j] << (8 * (j & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float int8_bias(const Int8Params& p, int n) {
  if (p.bias == nullptr) return 0.0f;
  return p.bias32 ? static_cast<const float*>(p.bias)[n] : bf16_to_f32(static_cast<const uint16_t*>(p.bias)[n]);
}

// Any sizes and alignments: tiles of 64 (n) x 64 (m), 2 x 2 waves, 128 K bytes a stage through registers into two LDS
// buffers; the next stage's loads are in flight during the products.
constexpr int kIK = 128;

__device__ __forceinline__ int i8_off(int r, int c) { return r * kIK + 16 * (c ^ ((r >> 1) & 7)); }

__global__ __launch_bounds__(256) void int8_any_kernel(Int8Params p) {
  __shared__ __align__(16) uint8_t lds[2][2][64 * kIK];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wn = wave & 1, wm = wave >> 1;
  const int n0 = (int)(blockIdx.x % p.tiles_n) * 64, m0 = (int)(blockIdx.x / p.tiles_n) * 64;
  uint4 rb[2], ra[2];
  auto load = [&](int k0) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = (tid + 256 * j) >> 3, k = k0 + 16 * (tid & 7), n = n0 + r, m = m0 + r;
      rb[j] = n < p.N ? load_k16(p.b + n * p.bs, k, p.K) : make_uint4(0, 0, 0, 0);
      ra[j] = m < p.M ? load_k16(p.a + m * p.as, k, p.K) : make_uint4(0, 0, 0, 0);
    }
  };
  auto store = [&](int buf) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int off = i8_off((tid + 256 * j) >> 3, tid & 7);
      *reinterpret_cast<uint4*>(&lds[buf][0][off]) = rb[j];
      *reinterpret_cast<uint4*>(&lds[buf][1][off]) = ra[j];
    }
  };
  v16i acc = {};
  load(0);
  store(0);
  __syncthreads();
  const int stages = (p.K + kIK - 1) / kIK;
  for (int s = 0; s < stages; ++s) {
    const bool more = s + 1 < stages;
    if (more) load((s + 1) * kIK);
#pragma unroll
    for (int q = 0; q < 4; ++q) {                  // 16-byte chunks 4 (q / 2) + 2 (lane / 32) + q % 2 of the row
      const int c = 4 * (q >> 1) + 2 * (lane >> 5) + (q & 1);
      const v4i fb = *reinterpret_cast<const v4i*>(&lds[s & 1][0][i8_off(32 * wn + (lane & 31), c)]);
      const v4i fa = *reinterpret_cast<const v4i*>(&lds[s & 1][1][i8_off(32 * wm + (lane & 31), c)]);
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb, fa, acc, 0, 0, 0);
    }
    if (more) store((s + 1) & 1);
    __syncthreads();
  }
  const int m = m0 + 32 * wm + (lane & 31);
  if (m >= p.M) return;
  const float sa = p.sa[(int64_t)m * p.sa_step];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int n = n0 + 32 * wn + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
    if (n >= p.N) continue;
    float v = (float)acc[e] * sa * p.sb[(int64_t)n * p.sb_step] + int8_bias(p, n);
    if (p.res) v = round_bf16(v) + bf16_to_f32(p.res[m * p.rs + n]);
    p.y[m * p.ys + n] = (uint16_t)f32_to_bf16_bits(v);
  }
}

// Codes of int8 within [-128, 127]: K products of at most 2^14 fit an int32.
constexpr int64_t kInt8MaxK = 131071;

static int int8_mm(Int8Params p, int64_t M, int64_t N, int64_t K, int64_t sa_count, int64_t sb_count, int bias_dtype, hipStream_t s,
                   const char* name) {
  FLW_REQUIRE(M >= 0 && N > 0 && K > 0, FLW_E_INVALID, "empty or negative shape (%lld, %lld, %lld)", (long long)M, (long long)N,
              (long long)K);
  FLW_REQUIRE(K <= kInt8MaxK, FLW_E_UNSUPPORTED, "K must be <= %lld for an exact int32 sum, got %lld", (long long)kInt8MaxK,
              (long long)K);
  FLW_REQUIRE(M <= 0x7FFFFF00ll && N <= 0x7FFFFF00ll, FLW_E_UNSUPPORTED, "too many rows or columns");
  FLW_REQUIRE((sa_count == M || sa_count == 1) && (sb_count == N || sb_count == 1), FLW_E_INVALID,
              "scales must be one a row and column, or one (got %lld for %lld rows, %lld for %lld columns)", (long long)sa_count,
              (long long)M, (long long)sb_count, (long long)N);
  if (M == 0) return FLW_OK;
  FLW_REQUIRE(p.a != nullptr && p.b != nullptr && p.sa != nullptr && p.sb != nullptr && p.y != nullptr, FLW_E_INVALID, "null pointer");
  FLW_REQUIRE(p.as >= K && p.bs >= K && p.ys >= N && (p.res == nullptr || p.rs >= N), FLW_E_INVALID, "a row stride below the row");
  FLW_REQUIRE((uintptr_t)p.y % 2 == 0 && (uintptr_t)p.res % 2 == 0 && (uintptr_t)p.sa % 4 == 0 && (uintptr_t)p.sb % 4 == 0,
              FLW_E_INVALID, "misaligned pointer");
  FLW_REQUIRE(p.bias == nullptr || ((bias_dtype == FLW_F32 || bias_dtype == FLW_BF16) &&
                                    (uintptr_t)p.bias % (bias_dtype == FLW_F32 ? 4 : 2) == 0),
              FLW_E_INVALID, "the bias must be aligned bf16 or fp32");
  p.M = (int)M; p.N = (int)N; p.K = (int)K;
  p.sa_step = sa_count > 1; p.sb_step = sb_count > 1;
  p.bias32 = bias_dtype == FLW_F32;
  p.tiles_n = (int)((N + 63) / 64);
  p.tiles_m = (int)((M + 63) / 64);
  FLW_REQUIRE((int64_t)p.tiles_n * p.tiles_m <= 0x7FFFFFFFll, FLW_E_UNSUPPORTED, "too many output tiles");
  (void)launch_timed(reinterpret_cast<const void*>(&int8_any_kernel), dim3((unsigned)(p.tiles_n * p.tiles_m)), dim3(256), s, p);
  return check_launch(name);
}

}  // namespace flw

using namespace flw;

extern "C" int flw_int8_scaled_mm(const int8_t* a, int64_t M, int64_t K, int64_t a_row_stride, const int8_t* b, int64_t N,
                                  int64_t b_row_stride, const float* a_scale, int64_t a_scale_count, const float* b_scale,
                                  int64_t b_scale_count, const void* bias, int bias_dtype, const void* residual,
                                  int64_t residual_row_stride, void* y, int64_t y_row_stride, void* stream) {
  Int8Params p{};
  p.a = a; p.as = a_row_stride; p.b = b; p.bs = b_row_stride;
  p.sa = a_scale; p.sb = b_scale; p.bias = bias;
  p.res = static_cast<const uint16_t*>(residual); p.rs = residual_row_stride;
  p.y = static_cast<uint16_t*>(y); p.ys = y_row_stride;
  return int8_mm(p, M, N, K, a_scale_count, b_scale_count, bias_dtype, static_cast<hipStream_t>(stream), "flw_int8_scaled_mm");
}

// The codes' rows start on 16 bytes whatever K, the scales behind them.
static int64_t linear_ld(int64_t K) { return (K + 15) / 16 * 16; }

extern "C" size_t flw_int8_linear_workspace_bytes(int64_t M, int64_t K) {
  return M <= 0 || K <= 0 ? 0 : (size_t)(M * linear_ld(K) + 4 * M);
}

extern "C" int flw_int8_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t x_row_stride, const int8_t* b, int64_t N,
                               int64_t b_row_stride, const float* b_scale, int64_t b_scale_count, const void* bias, int bias_dtype,
                               const void* residual, int64_t residual_row_stride, void* y, int64_t y_row_stride, void* workspace,
                               size_t workspace_bytes, void* stream) {
  FLW_REQUIRE(M >= 0 && K > 0, FLW_E_INVALID, "empty or negative shape (%lld, %lld)", (long long)M, (long long)K);
  const size_t need = flw_int8_linear_workspace_bytes(M, K);
  FLW_REQUIRE(workspace_bytes >= need && (need == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0)), FLW_E_WORKSPACE,
              "workspace needs %zu bytes (16-byte aligned), got %zu", need, workspace_bytes);
  const int64_t ld = linear_ld(K);
  int8_t* codes = static_cast<int8_t*>(workspace);
  float* scale = M > 0 ? reinterpret_cast<float*>(codes + M * ld) : nullptr;
  const Timer tm = take_timer();
  arm_timer({tm.start, nullptr});
  int rc = flw_rows8(x, dtype, M, K, x_row_stride, FLW_I8, codes, ld, scale, stream);
  arm_timer({nullptr, rc ? nullptr : tm.stop});
  if (rc == FLW_OK)
    rc = flw_int8_scaled_mm(codes, M, K, ld, b, N, b_row_stride, scale, M, b_scale, b_scale_count, bias, bias_dtype, residual,
                            residual_row_stride, y, y_row_stride, stream);
  arm_timer({});                                   // of a call that launched nothing
  return rc;
}
