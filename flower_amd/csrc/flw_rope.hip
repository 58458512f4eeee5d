// Rotary positions of q and k (apply_rotary, forward and gradient), and the new tokens' way into a paged key-value
// cache (paged_append): QK-norm, rotary positions, and the write of k and v to their pages.
//
// A pair (a, b) of a head's first R values becomes (a c - b s, b c + a s) with c, s = the tables' entry of the token's
// position and the pair: pairs next to each other (interleaved) or R / 2 apart (half). The gradient is the same with
// -s. Tables are fp32, [rows, R / 2]; the arithmetic is fp32 and rounds once, at the store.
//
// Both are one read and one write of the heads, bound by HBM (a decode step's by its launch). A thread holds one unit
// of 8 values (4 pairs) of a token's head rows and goes from head to head, so that it loads the token's angles once:
// a table row of R floats for each head row of D 2-byte values would otherwise be twice the heads' own bytes.
//
// Measured: rotary of 2 x 8192 tokens, 20 + 20 heads of 64 (168 MB): 31 us, 5.4 TB/s; with q and k read through the caches 36. In
// fp32 (336 MB), which reads through the caches, 77 us, 4.4 TB/s.
// Appending 8192 tokens of 16 + 4 + 4 heads of 128 to an e4m3 cache (92 MB): 25 us, 3.6 TB/s (to a bf16 one 19 us, 5.3);
// with q's, k's and v's heads in one loop 27, read past the caches 30 and more (half layout: a line is read in two parts). A decode
// step's append: 5 us, its launch.

#include "flw_common.h"

namespace flw {

struct RopeTables {
  const float* cos;
  const float* sin;
  int64_t rows;
  int R, half;
};

// A unit's angles: c[i], s[i] of pairs 4 u + i. A position outside the tables gives NaN.
struct RopeUnit {
  float4 c, s;
  bool turns;
  __device__ __forceinline__ void load(const RopeTables& t, int64_t pos, int u, bool inverse) {
    turns = 8 * u < t.R;
    c = s = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
    if (!turns) return;
    if (pos < 0 || pos >= t.rows) {
      const float nan = __builtin_nanf("");
      c = s = make_float4(nan, nan, nan, nan);
      return;
    }
    c = *reinterpret_cast<const float4*>(t.cos + pos * (t.R / 2) + 4 * u);
    s = *reinterpret_cast<const float4*>(t.sin + pos * (t.R / 2) + 4 * u);
    if (inverse) s = make_float4(-s.x, -s.y, -s.z, -s.w);
  }
  // f: the unit's pairs as a0 b0 a1 b1 ...
  __device__ __forceinline__ void turn(float* f) const {
    if (!turns) return;
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = f[2 * i], b = f[2 * i + 1];
      f[2 * i] = fmaf(a, cc[i], -(b * ss[i]));
      f[2 * i + 1] = fmaf(b, cc[i], a * ss[i]);
    }
  }
};

// Where a unit's values lie in a head row: eight in a run (split == 0), or four at `first` and four `split` later.
struct RopePlace {
  int first, split;
  __device__ __forceinline__ RopePlace(const RopeTables& t, int u) {
    const bool two = t.half && 8 * u < t.R;
    first = two ? 4 * u : 8 * u;
    split = two ? t.R / 2 : 0;
  }
};

typedef uint32_t RopeRun __attribute__((ext_vector_type(4)));
// PAST: past the caches, where eight bf16 values lie in a run.
template <bool PAST>
__device__ __forceinline__ void unit_load(const uint16_t* row, RopePlace at, float* f) {
  if (at.split == 0) {
    const RopeRun* from = reinterpret_cast<const RopeRun*>(row + at.first);
    const RopeRun x = PAST ? __builtin_nontemporal_load(from) : *from;
    Vec16<uint16_t>::unpack(make_uint4(x[0], x[1], x[2], x[3]), f);
  } else {
    const uint2 a = *reinterpret_cast<const uint2*>(row + at.first);
    const uint2 b = *reinterpret_cast<const uint2*>(row + at.first + at.split);
    const uint32_t x[2] = {a.x, a.y}, y[2] = {b.x, b.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[4 * i] = __uint_as_float(x[i] << 16);
      f[4 * i + 1] = __uint_as_float(y[i] << 16);
      f[4 * i + 2] = __uint_as_float(x[i] & 0xFFFF0000u);
      f[4 * i + 3] = __uint_as_float(y[i] & 0xFFFF0000u);
    }
  }
}
template <bool PAST>
__device__ __forceinline__ void unit_load(const float* row, RopePlace at, float* f) {
  const float4 a = *reinterpret_cast<const float4*>(row + at.first);
  const float4 b = *reinterpret_cast<const float4*>(row + at.first + (at.split == 0 ? 4 : at.split));
  const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = at.split == 0 ? x[i] : x[(i >> 1) + 4 * (i & 1)];
}
__device__ __forceinline__ void unit_store(uint16_t* row, RopePlace at, const float* f) {
  if (at.split == 0) {
    *reinterpret_cast<uint4*>(row + at.first) =
        make_uint4(bf16x2_rne(f[0], f[1]), bf16x2_rne(f[2], f[3]), bf16x2_rne(f[4], f[5]), bf16x2_rne(f[6], f[7]));
  } else {
    *reinterpret_cast<uint2*>(row + at.first) = make_uint2(bf16x2_rne(f[0], f[2]), bf16x2_rne(f[4], f[6]));
    *reinterpret_cast<uint2*>(row + at.first + at.split) = make_uint2(bf16x2_rne(f[1], f[3]), bf16x2_rne(f[5], f[7]));
  }
}
__device__ __forceinline__ void unit_store(float* row, RopePlace at, const float* f) {
  if (at.split == 0) {
    *reinterpret_cast<float4*>(row + at.first) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(row + at.first + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<float4*>(row + at.first) = make_float4(f[0], f[2], f[4], f[6]);
    *reinterpret_cast<float4*>(row + at.first + at.split) = make_float4(f[1], f[3], f[5], f[7]);
  }
}

struct RopeParams {
  const void* x[2];               // q, k
  int64_t sb[2], sh[2], st[2];
  void* out[2];                   // contiguous (B, heads, T, D)
  int heads[2];
  const void* positions;          // NULL: t
  int64_t pos_sb;
  int pos64, inverse;
  RopeTables tab;
  int B, T, ushift, per;          // D = 8 << ushift; heads a thread
};

template <typename E>
__global__ __launch_bounds__(256) void rope_kernel(RopeParams p) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  const uint32_t token = i >> p.ushift;
  if (token >= (uint32_t)p.B * (uint32_t)p.T) return;
  const int u = (int)(i & ((1u << p.ushift) - 1)), b = (int)(token / (uint32_t)p.T), t = (int)token - b * p.T;
  int64_t pos = t;
  if (p.positions != nullptr) {
    const int64_t at = b * p.pos_sb + t;
    pos = p.pos64 ? static_cast<const int64_t*>(p.positions)[at] : (int64_t)static_cast<const int32_t*>(p.positions)[at];
  }
  RopeUnit unit;
  unit.load(p.tab, pos, u, p.inverse != 0);
  const RopePlace at(p.tab, u);
  const int64_t D = 8ll << p.ushift;
  const int n = p.heads[0] + p.heads[1], h0 = (int)blockIdx.y * p.per, h1 = h0 + p.per < n ? h0 + p.per : n;
#pragma unroll 4
  for (int hh = h0; hh < h1; ++hh) {
    const int w = hh >= p.heads[0], h = w ? hh - p.heads[0] : hh;
    float f[8];
    unit_load<true>(static_cast<const E*>(p.x[w]) + b * p.sb[w] + h * p.sh[w] + t * p.st[w], at, f);
    unit.turn(f);
    unit_store(static_cast<E*>(p.out[w]) + (((int64_t)b * p.heads[w] + h) * p.T + t) * D, at, f);
  }
}

// ---------------------------------------------------------------- into the cache

struct AppendParams {
  const uint16_t* x[3];           // q, k, v (B, heads, T, D)
  int64_t sb[3], sh[3], st[3];
  uint16_t* q_out;                // contiguous (B, H, T, D)
  uint16_t* k_out;                // contiguous (B, KV, T, D), or NULL
  uint8_t* k;                     // (P, KV, page, D)
  uint8_t* v;                     // (P, KV, D, page)
  const int32_t* tables;
  const int32_t* lens;
  const int32_t* counts;
  const float* k_scale;           // e4m3 cache
  const float* v_scale;
  RopeTables tab;
  int64_t P;
  float eps;
  int norm, B, T, H, KV, M, shift, ushift, per, v_tiles, head_blocks, token_blocks;
};

__device__ __forceinline__ float clamp_e4m3(float x) {      // NaN stays NaN
  x = x > kE4m3Max ? kE4m3Max : x;
  return x < -kE4m3Max ? -kE4m3Max : x;
}
__device__ __forceinline__ uint32_t e4m3x2(float a, float b, float s) {      // IEEE divisions
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(a / s), clamp_e4m3(b / s), 0, false) & 0xFFFFu;
}

// The page of a position of sequence b, or -1 where its table holds none.
__device__ __forceinline__ int64_t append_page(const AppendParams& p, int b, int64_t pos) {
  const int64_t e = pos >> p.shift;
  if (pos < 0 || e >= p.M) return -1;
  const int32_t id = p.tables[(int64_t)b * p.M + e];
  return (uint32_t)id < (uint32_t)p.P ? id : -1;
}

// Base position (of token 0) and count of sequence b's new tokens.
__device__ __forceinline__ void append_span(const AppendParams& p, int b, int64_t* base, int* cnt) {
  int n = p.counts != nullptr ? p.counts[b] : p.T;
  n = n < 0 ? 0 : n;
  const int len = p.lens[b];
  *base = (int64_t)(len < 0 ? 0 : len) - n;
  *cnt = n < p.T ? n : p.T;
}

template <bool F8>
__global__ __launch_bounds__(256) void append_kernel(AppendParams p) {
  __shared__ __align__(16) uint16_t tile[64 * (128 + 8)];
  const int64_t D = 8ll << p.ushift;
  if ((int)blockIdx.x < p.head_blocks) {
    const int by = (int)blockIdx.x / p.token_blocks, bx = (int)blockIdx.x - by * p.token_blocks;
    const uint32_t i = bx * 256u + threadIdx.x;
    const uint32_t token = i >> p.ushift;
    if (token >= (uint32_t)p.B * (uint32_t)p.T) return;     // whole groups of 1 << ushift lanes
    const int U = 1 << p.ushift, u = (int)i & (U - 1), b = (int)(token / (uint32_t)p.T), t = (int)token - b * p.T;
    int64_t base;
    int cnt;
    append_span(p, b, &base, &cnt);
    const int64_t pos = base + t;
    const bool live = t < cnt && pos >= 0;
    RopeUnit unit;
    unit.load(p.tab, pos, u, false);
    const RopePlace at(p.tab, u);
    const int64_t page = live ? append_page(p, b, pos) : -1;
    const int off = (int)(pos & ((1 << p.shift) - 1)), psz = 1 << p.shift;
    // heads of q, of k, and of v where its tokens are few (v_tiles == 0): each value to its own place
    const int n = p.H + p.KV + (p.v_tiles == 0 ? p.KV : 0), h0 = by * p.per, h1 = h0 + p.per < n ? h0 + p.per : n;
    auto turned = [&](const uint16_t* row, float* f) __attribute__((always_inline)) {      // normed and turned; padding: zero
      unit_load<false>(row, at, f);
      if (p.norm) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(f[j], f[j], ss);
        const float r = __builtin_amdgcn_rsqf(group_sum(ss, U) / (float)D + p.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= r;
      }
      unit.turn(f);
      if (!live)
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = 0.0f;
    };
    const int hq = h1 < p.H ? h1 : p.H;
#pragma unroll 1
    for (int h = h0; h < hq; ++h) {
      float f[8];
      turned(p.x[0] + b * p.sb[0] + h * p.sh[0] + t * p.st[0], f);
      unit_store(p.q_out + (((int64_t)b * p.H + h) * p.T + t) * D, at, f);
    }
#pragma unroll 1
    for (int hh = h0 > hq ? h0 : hq; hh < h1; ++hh) {
      const int w = hh < p.H + p.KV ? 1 : 2, h = hh - (w == 1 ? p.H : p.H + p.KV);
      const uint16_t* row = p.x[w] + b * p.sb[w] + h * p.sh[w] + t * p.st[w];
      const int64_t head = (page * p.KV + h) * psz * D;
      float f[8];
      if (w == 2) {
        if (page < 0) continue;
        Vec16<uint16_t>::load(row + 8 * u, f);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const int64_t o = head + (int64_t)(8 * u + j) * psz + off;
          if constexpr (F8) {
            const uint32_t x = e4m3x2(f[j], f[j + 1], p.v_scale[h]);
            p.v[o] = (uint8_t)x;
            p.v[o + psz] = (uint8_t)(x >> 8);
          } else {
            reinterpret_cast<uint16_t*>(p.v)[o] = (uint16_t)(__float_as_uint(f[j]) >> 16);
            reinterpret_cast<uint16_t*>(p.v)[o + psz] = (uint16_t)(__float_as_uint(f[j + 1]) >> 16);
          }
        }
        continue;
      }
      turned(row, f);
      if (p.k_out != nullptr) unit_store(p.k_out + (((int64_t)b * p.KV + h) * p.T + t) * D, at, f);
      if (page < 0) continue;
      const int64_t o = head + (int64_t)off * D;
      if constexpr (F8) {
        const float s = p.k_scale[h];
        uint8_t* dst = p.k + o + at.first;
        if (at.split == 0) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(e4m3x2(f[0], f[1], s) | e4m3x2(f[2], f[3], s) << 16,
                                                      e4m3x2(f[4], f[5], s) | e4m3x2(f[6], f[7], s) << 16);
        } else {
          *reinterpret_cast<uint32_t*>(dst) = e4m3x2(f[0], f[2], s) | e4m3x2(f[4], f[6], s) << 16;
          *reinterpret_cast<uint32_t*>(dst + at.split) = e4m3x2(f[1], f[3], s) | e4m3x2(f[5], f[7], s) << 16;
        }
      } else {
        unit_store(reinterpret_cast<uint16_t*>(p.k) + o, at, f);
      }
    }
    return;
  }
  // v of many tokens: 64 positions (from a multiple of 64 on) of one head through LDS, written as runs along the page.
  int j = (int)blockIdx.x - p.head_blocks;
  const int b = j / (p.KV * p.v_tiles);
  j -= b * p.KV * p.v_tiles;
  const int h = j / p.v_tiles;
  int64_t base;
  int cnt;
  append_span(p, b, &base, &cnt);
  const int64_t first = base > 0 ? base : 0, end = base + cnt;
  const int64_t p0 = (first & ~63ll) + 64ll * (j - h * p.v_tiles);
  if (p0 >= end) return;                                     // the workgroup as one
  const int U = 1 << p.ushift, pitch = (int)D + 8;
  for (int e = threadIdx.x; e < 64 * U; e += 256) {
    const int r = e >> p.ushift, u = e & (U - 1);
    const int64_t pos = p0 + r;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (pos >= first && pos < end)
      x = *reinterpret_cast<const uint4*>(p.x[2] + b * p.sb[2] + h * p.sh[2] + (pos - base) * p.st[2] + 8 * u);
    *reinterpret_cast<uint4*>(tile + r * pitch + 8 * u) = x;
  }
  __syncthreads();
  const int psz = 1 << p.shift;
  for (int e = threadIdx.x; e < 8 * (int)D; e += 256) {
    const int c = e & 7, d = e >> 3;                         // positions p0 + 8 c .., all on one page
    const int64_t pos = p0 + 8 * c;
    if (pos >= end || pos + 8 <= first) continue;
    const int64_t page = append_page(p, b, pos);
    if (page < 0) continue;
    uint32_t x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = tile[(8 * c + i) * pitch + d];
    const int64_t o = ((page * p.KV + h) * D + d) * psz + (pos & (psz - 1));
    const bool whole = pos >= first && pos + 8 <= end;
    if constexpr (F8) {
      const float s = p.v_scale[h];
      uint32_t y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = e4m3x2(bf16_to_f32(x[2 * i]), bf16_to_f32(x[2 * i + 1]), s);
      if (whole) {
        *reinterpret_cast<uint2*>(p.v + o) = make_uint2(y[0] | y[1] << 16, y[2] | y[3] << 16);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (pos + i >= first && pos + i < end) p.v[o + i] = (uint8_t)(y[i >> 1] >> (8 * (i & 1)));
      }
    } else {
      uint16_t* v = reinterpret_cast<uint16_t*>(p.v);
      if (whole) {
        *reinterpret_cast<uint4*>(v + o) = make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (pos + i >= first && pos + i < end) v[o + i] = (uint16_t)x[i];
      }
    }
  }
}

static int rope_tables_check(const float* cos, const float* sin, int64_t rows, int64_t R, int64_t D, int layout) {
  FLW_REQUIRE(D == 32 || D == 64 || D == 128, FLW_E_UNSUPPORTED, "head_dim must be 32/64/128, got %lld", (long long)D);
  FLW_REQUIRE(layout == FLW_ROPE_INTERLEAVED || layout == FLW_ROPE_HALF, FLW_E_INVALID, "unknown rotary layout %d", layout);
  FLW_REQUIRE(cos && sin && rows > 0 && (((uintptr_t)cos | (uintptr_t)sin) & 15) == 0, FLW_E_INVALID,
              "rotary tables must be non-empty and 16-byte aligned");
  FLW_REQUIRE(R > 0 && R <= D && R % 8 == 0, FLW_E_UNSUPPORTED, "rotary_dim must be a multiple of 8 up to head_dim, got %lld",
              (long long)R);
  return FLW_OK;
}

static int head_rows_check(const void* x, const int64_t* s, int64_t vec, const char* what) {
  FLW_REQUIRE(x != nullptr && s != nullptr, FLW_E_INVALID, "null %s", what);
  FLW_REQUIRE(((uintptr_t)x & 15) == 0 && s[0] % vec == 0 && s[1] % vec == 0 && s[2] % vec == 0, FLW_E_INVALID,
              "%s rows must be 16-byte aligned", what);
  return FLW_OK;
}

}  // namespace flw

using namespace flw;

extern "C" int flw_rope(const void* q, const int64_t* q_strides, int64_t H, const void* k, const int64_t* k_strides,
                        int64_t KV, int dtype, int64_t B, int64_t T, int64_t D, const float* cos, const float* sin,
                        int64_t table_rows, int64_t rotary_dim, int layout, int inverse, const void* positions,
                        int positions_bits, int64_t positions_stride_b, void* q_out, void* k_out, void* stream) {
  int rc = rope_tables_check(cos, sin, table_rows, rotary_dim, D, layout);
  if (rc) return rc;
  FLW_REQUIRE(dtype == FLW_F32 || dtype == FLW_BF16, FLW_E_INVALID, "q and k must be fp32 or bf16");
  FLW_REQUIRE(B > 0 && T > 0 && H > 0 && KV >= 0, FLW_E_INVALID, "empty shape");
  const int64_t vec = dtype == FLW_F32 ? 4 : 8;
  if ((rc = head_rows_check(q, q_strides, vec, "q")) != 0) return rc;
  if (KV > 0 && (rc = head_rows_check(k, k_strides, vec, "k")) != 0) return rc;
  FLW_REQUIRE(q_out && ((uintptr_t)q_out & 15) == 0 && (KV == 0 || (k_out && ((uintptr_t)k_out & 15) == 0)), FLW_E_INVALID,
              "outputs must be non-null and 16-byte aligned");
  FLW_REQUIRE(positions == nullptr || positions_bits == 32 || positions_bits == 64, FLW_E_INVALID, "positions are int32 or int64");
  FLW_REQUIRE(B * T * (D / 8) <= 0x7FFFFFFFll - 255 && H <= 65536 && KV <= 65536, FLW_E_UNSUPPORTED, "shape too large");
  RopeParams p{};
  p.x[0] = q; p.x[1] = k; p.out[0] = q_out; p.out[1] = k_out;
  p.heads[0] = (int)H; p.heads[1] = (int)KV;
  p.sb[0] = q_strides[0]; p.sh[0] = q_strides[1]; p.st[0] = q_strides[2];
  if (KV > 0) { p.sb[1] = k_strides[0]; p.sh[1] = k_strides[1]; p.st[1] = k_strides[2]; }
  p.positions = positions; p.pos_sb = positions_stride_b; p.pos64 = positions_bits == 64; p.inverse = inverse;
  p.tab = RopeTables{cos, sin, table_rows, (int)rotary_dim, layout == FLW_ROPE_HALF};
  p.B = (int)B; p.T = (int)T; p.ushift = __builtin_ctzll(D / 8);
  const int64_t n = H + KV, bx = (B * T * (D / 8) + 255) / 256;
  int64_t by = 2048 / bx;                         // eight workgroups a compute unit, then heads in turn
  by = by < 1 ? 1 : by > n ? n : by;
  p.per = (int)((n + by - 1) / by);
  by = (n + p.per - 1) / p.per;
  const void* kern = dtype == FLW_F32 ? (const void*)&rope_kernel<float> : (const void*)&rope_kernel<uint16_t>;
  (void)launch_timed(kern, dim3((unsigned)bx, (unsigned)by), dim3(256), static_cast<hipStream_t>(stream), p);
  return check_launch("flw_rope");
}

extern "C" int flw_paged_append(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                const void* v, const int64_t* v_strides, int64_t B, int64_t H, int64_t KV, int64_t T,
                                int64_t D, void* k_pages, void* v_pages, int cache_dtype, int64_t num_pages,
                                int64_t page_size, const int32_t* tables, int64_t table_cols, const int32_t* lens,
                                const int32_t* counts, int qk_norm, float eps, const float* cos, const float* sin,
                                int64_t table_rows, int64_t rotary_dim, int layout, const float* k_scale,
                                const float* v_scale, void* q_out, void* k_out, void* stream) {
  int rc;
  if (cos != nullptr || sin != nullptr) {
    if ((rc = rope_tables_check(cos, sin, table_rows, rotary_dim, D, layout)) != 0) return rc;
  } else {
    FLW_REQUIRE(D == 32 || D == 64 || D == 128, FLW_E_UNSUPPORTED, "head_dim must be 32/64/128, got %lld", (long long)D);
  }
  FLW_REQUIRE(B > 0 && T > 0 && H > 0 && KV > 0 && num_pages > 0 && table_cols > 0, FLW_E_INVALID, "empty shape");
  if ((rc = head_rows_check(q, q_strides, 8, "q")) != 0) return rc;
  if ((rc = head_rows_check(k, k_strides, 8, "k")) != 0) return rc;
  if ((rc = head_rows_check(v, v_strides, 8, "v")) != 0) return rc;
  FLW_REQUIRE(k_pages && v_pages && tables && lens && q_out, FLW_E_INVALID, "null pointer");
  FLW_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)q_out | (uintptr_t)k_out) & 15) == 0, FLW_E_INVALID,
              "pages and outputs must be 16-byte aligned");
  FLW_REQUIRE(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0, FLW_E_UNSUPPORTED,
              "page size must be a power of two from 16 to 1024, got %lld", (long long)page_size);
  FLW_REQUIRE(cache_dtype == FLW_BF16 || cache_dtype == FLW_E4M3, FLW_E_INVALID, "the cache holds bf16 or e4m3");
  FLW_REQUIRE((cache_dtype == FLW_E4M3) == (k_scale != nullptr) && (k_scale != nullptr) == (v_scale != nullptr),
              FLW_E_INVALID, "an e4m3 cache takes k and v scales, a bf16 one none");
  FLW_REQUIRE(qk_norm == 0 || eps >= 0.0f, FLW_E_INVALID, "eps must be non-negative");
  FLW_REQUIRE(num_pages <= 0x7FFFFFFFll && table_cols <= 0x7FFFFFFFll && H <= 65536 && KV <= 65536 &&
              B * T * (D / 8) <= 0x7FFFFFFFll - 255, FLW_E_UNSUPPORTED, "shape too large");
  AppendParams p{};
  const void* xs[3] = {q, k, v};
  const int64_t* ss[3] = {q_strides, k_strides, v_strides};
  for (int i = 0; i < 3; ++i) {
    p.x[i] = static_cast<const uint16_t*>(xs[i]);
    p.sb[i] = ss[i][0]; p.sh[i] = ss[i][1]; p.st[i] = ss[i][2];
  }
  p.q_out = static_cast<uint16_t*>(q_out); p.k_out = static_cast<uint16_t*>(k_out);
  p.k = static_cast<uint8_t*>(k_pages); p.v = static_cast<uint8_t*>(v_pages);
  p.tables = tables; p.lens = lens; p.counts = counts; p.k_scale = k_scale; p.v_scale = v_scale;
  p.tab = RopeTables{cos, sin, table_rows, cos != nullptr ? (int)rotary_dim : 0, layout == FLW_ROPE_HALF};
  p.P = num_pages; p.eps = eps; p.norm = qk_norm;
  p.B = (int)B; p.T = (int)T; p.H = (int)H; p.KV = (int)KV; p.M = (int)table_cols;
  p.shift = __builtin_ctzll(page_size); p.ushift = __builtin_ctzll(D / 8);
  // v through LDS from 16 tokens on, where the runs along a page begin to fill
  p.v_tiles = T >= 16 ? (int)((T + 62) / 64 + 1) : 0;
  const int64_t n = H + KV + (p.v_tiles == 0 ? KV : 0), bx = (B * T * (D / 8) + 255) / 256;
  int64_t by = 2048 / bx;
  by = by < 1 ? 1 : by > n ? n : by;
  p.per = (int)((n + by - 1) / by);
  by = (n + p.per - 1) / p.per;
  const int64_t blocks = bx * by + B * KV * p.v_tiles;
  FLW_REQUIRE(blocks <= 0x7FFFFFFFll, FLW_E_UNSUPPORTED, "shape too large");
  p.token_blocks = (int)bx; p.head_blocks = (int)(bx * by);
  const void* kern = cache_dtype == FLW_E4M3 ? (const void*)&append_kernel<true> : (const void*)&append_kernel<false>;
  (void)launch_timed(kern, dim3((unsigned)blocks), dim3(256), static_cast<hipStream_t>(stream), p);
  return check_launch("flw_paged_append");
}
