// The 8-bit integer linear for gfx950: y[M, N] (bf16) = (a[M, K] . b[N, K]^T) sa[m] sb[n] + bias[n], then residual + y.
//
// The products are summed in int32 by the integer MFMA, exactly (|a b| <= 2^14, K <= 131071), so that every tile and every
// split of K gives the same bits; one conversion to fp32 and two products follow. y is rounded to bf16 before the
// residual is added, and the sum again, as the block's separate linear and add round and flw_fp8_scaled_mm_residual does: the fused and
// the separate addition give the same bits. It costs a result's error against 64 bits 2.2e-3 of its size where one rounding has 1.7e-3.
//
// Both operands lie along K. An MFMA only needs a and b to agree on which k a lane's byte is, so the 32 consecutive bytes of a
// row that a lane holds (half h = lane / 32 of a 64-deep chunk) feed two v_mfma_i32_32x32x32_i8, 16 bytes each. The product is
// taken transposed, C^T = b a^T: a lane of the 32 x 32 accumulator owns one output row m and n = 8 g + 4 h + 0..3.
#include <algorithm>
#include <type_traits>

#include "flw_common.h"

// m0 is clobbered by the direct-to-LDS loads below; nothing else here uses it. Between its write and the load stands the wait
// state that the hardware asks for, which the compiler does not put inside an assembly statement.
#pragma clang diagnostic ignored "-Winline-asm"

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
  const void* x;           // instead of a and sa: rows to quantise, bf16 or fp32 (x32), row stride xs
  int64_t xs;
  int x32;
  int M, N, K;
  int tiles_n, tiles_m;
  int wide;                // N % 8 == 0, rows of y and of the residual start on 16 bytes, fewer than 2^26 apart, sb too, one a column
};

// 16 bytes at any address.
__device__ __forceinline__ uint4 load_any16(const int8_t* p) {
  struct __attribute__((packed, aligned(1))) V { uint32_t w[4]; };
  const V v = *reinterpret_cast<const V*>(p);
  return make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
}
// v without its first s bytes, zeros behind (s >= 0).
__device__ __forceinline__ uint4 drop_bytes(uint4 v, int s) {
  uint64_t lo = v.x | (uint64_t)v.y << 32, hi = v.z | (uint64_t)v.w << 32;
  if (s >= 8) { lo = hi; hi = 0; }
  const int r = 8 * (s & 7);
  lo = s >= 16 ? 0 : r ? lo >> r | hi << (64 - r) : lo;
  hi >>= r;
  return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}

__device__ __forceinline__ float int8_bias(const Int8Params& p, int n) {
  if (p.bias == nullptr) return 0.0f;
  return p.bias32 ? static_cast<const float*>(p.bias)[n] : bf16_to_f32(static_cast<const uint16_t*>(p.bias)[n]);
}

// Where the 16-byte chunk c of row r of a tile lies in LDS, rows of 128 bytes: reads of a chunk of consecutive rows meet no bank twice.
__device__ __forceinline__ int swz(int r, int c) { return r * 128 + 16 * (c ^ ((r >> 1) & 7)); }

template <int N, int I = 0, typename F>
__device__ __forceinline__ void each_up(F f) {            // f(0), ..., f(N - 1), compile-time arguments
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each_up<N, I + 1>(f);
  }
}

// One output before the residual. The same operations in every kernel, so that all give the same bits.
__device__ __forceinline__ float int8_value(int acc, float sa, float sb, float bias) { return fmaf((float)acc * sa, sb, bias); }

// ---------------------------------------------------------------- tiles through LDS
//
// Operands with 16-byte rows and K % 16 == 0. A stage is the tile's b rows, then its a rows, 128 bytes of K each, moved global ->
// LDS without registers (global_load_lds_dwordx4: 64 lanes x 16 bytes, 8 whole 128-byte lines). A lane's place in LDS is fixed by
// the instruction, so the swizzle is made by the chunk that the lane fetches.
// The loads are written in assembly: the compiler then does not know of their writes to LDS and does not drain them before
// every read; each wave waits for its own loads and then for the others at a barrier.
// TAIL (K % 128 != 0): the last stage's chunks past K are loaded from the row's start instead (in bounds) and b's fragments of
// them are made zero.
// The first tile of a workgroup. The workgroups of an XCD (blockIdx % 8) take consecutive tiles, which are numbered in groups of
// 4 rows of tiles, m fastest: those that run together share their operands in the XCD's L2.
__device__ __forceinline__ int int8_first() {
  const int per = gridDim.x >> 3, more = gridDim.x & 7, xcd = blockIdx.x & 7;
  return xcd * per + min(xcd, more) + (blockIdx.x >> 3);
}
template <int BN, int BM>
__device__ __forceinline__ void int8_place(const Int8Params& p, int t, int& m0, int& n0) {
  const int first = t / (4 * p.tiles_n) * 4, in = t % (4 * p.tiles_n), gm = min(p.tiles_m - first, 4);
  m0 = (first + in % gm) * BM;
  n0 = in / gm * BN;
}

// The scales and biases of the columns n + 8 g + e, g, e = 0..3 (past N: of some column). All loads of a kind behind one branch: a
// branch a load, and each waited for the one before.
__device__ __forceinline__ void int8_columns(const Int8Params& p, int n, float (&sb)[16], float (&bias)[16]) {
  auto col = [&](int k) __attribute__((always_inline)) { return min(n + 2 * (k & 12) + (k & 3), p.N - 1); };
  if (p.wide) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 v = *reinterpret_cast<const float4*>(p.sb + min(n + 8 * g, p.N - 4));
      sb[4 * g] = v.x; sb[4 * g + 1] = v.y; sb[4 * g + 2] = v.z; sb[4 * g + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) sb[k] = p.sb[(int64_t)col(k) * p.sb_step];
  }
#pragma unroll
  for (int k = 0; k < 16; ++k) bias[k] = 0.0f;
  if (p.bias != nullptr) {
    if (p.bias32) {
#pragma unroll
      for (int k = 0; k < 16; ++k) bias[k] = static_cast<const float*>(p.bias)[col(k)];
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) bias[k] = bf16_to_f32(static_cast<const uint16_t*>(p.bias)[col(k)]);
    }
  }
}

// Eight bf16 sums.
__device__ __forceinline__ uint4 int8_plus(uint4 x, uint4 y) {
  float a[8], b[8];
  Vec16<uint16_t>::unpack(x, a);
  Vec16<uint16_t>::unpack(y, b);
#pragma unroll
  for (int e = 0; e < 8; ++e) a[e] += b[e];
  return make_uint4(bf16x2_rne(a[0], a[1]), bf16x2_rne(a[2], a[3]), bf16x2_rne(a[4], a[5]), bf16x2_rne(a[6], a[7]));
}

// 8 bf16 values to an aligned place; STREAM: past the caches.
template <bool STREAM>
__device__ __forceinline__ void int8_put(uint16_t* y, uint4 o) {
  if (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(v4i, o), reinterpret_cast<v4i*>(y));
  else *reinterpret_cast<uint4*>(y) = o;
}

// The 8 bf16 values o of row m from column n on (n % 8 == 0, m < M, n < N) into y, the residual added.
__device__ __forceinline__ void int8_store8(const Int8Params& p, int m, int n, uint4 o) {
  uint16_t* y = p.y + (int64_t)m * p.ys + n;
  const uint16_t* res = p.res ? p.res + (int64_t)m * p.rs + n : nullptr;
  if (p.wide) {
    if (res) o = int8_plus(o, *reinterpret_cast<const uint4*>(res));
    int8_put<false>(y, o);
    return;
  }
  if (n + 8 <= p.N) {                             // at any address
    struct __attribute__((packed, aligned(2))) V { uint32_t w[4]; };
    if (res) {
      const V r = *reinterpret_cast<const V*>(res);
      o = int8_plus(o, make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]));
    }
    *reinterpret_cast<V*>(y) = V{{o.x, o.y, o.z, o.w}};
    return;
  }
  float a[8];
  Vec16<uint16_t>::unpack(o, a);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (n + e < p.N) y[e] = (uint16_t)f32_to_bf16_bits(res ? a[e] + bf16_to_f32(res[e]) : a[e]);
}

// The scaled bf16 tile through LDS (row r: 2 BN bytes, 16-byte chunk c at c ^ (r % (BN / 8))), so that whole row segments are
// stored and the residual is read by whole segments.
template <int WN, int WM, int TN, int TM>
__device__ __forceinline__ void int8_epilogue(const Int8Params& p, const v16i (&acc)[TN][TM], uint8_t* lds, int m0, int n0, int wave,
                                              int lane) {
  constexpr int BN = 32 * WN * TN, BM = 32 * WM * TM, NT = 64 * WN * WM, CPR = BN / 8, ROWB = 2 * BN;
  static_assert(NT % CPR == 0, "a thread keeps its chunk column");
  constexpr int RPQ = NT / CPR, NQ = BM / RPQ;    // rows a pass of the stores
  const int wn = wave % WN, wm = wave / WN, hh = lane >> 5, tid = wave * 64 + lane, ch = tid % CPR, n = n0 + 8 * ch, r0 = tid / CPR;
  uint4 res[NQ];                                  // of wide rows, under way while the tile goes through LDS ([2048, 1280]: 11.4 -> 10.8 us)
  const bool early = p.wide && p.res != nullptr;
  if (early) {
#pragma unroll
    for (int q = 0; q < NQ; ++q)
      res[q] = *reinterpret_cast<const uint4*>(p.res + (int64_t)min(m0 + RPQ * q + r0, p.M - 1) * p.rs + min(n, p.N - 8));
  }
  float sa[TM];
#pragma unroll
  for (int j = 0; j < TM; ++j) sa[j] = p.sa[(int64_t)min(m0 + 32 * (TM * wm + j) + (lane & 31), p.M - 1) * p.sa_step];
#pragma unroll
  for (int i = 0; i < TN; ++i) {
    float sb[16], bias[16];
    int8_columns(p, n0 + 32 * (TN * wn + i) + 4 * hh, sb, bias);
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int r = 32 * (TM * wm + j) + (lane & 31);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = int8_value(acc[i][j][4 * g + e], sa[j], sb[4 * g + e], bias[4 * g + e]);
        const int ch = 4 * (TN * wn + i) + g;
        *reinterpret_cast<uint2*>(lds + r * ROWB + 16 * (ch ^ (r & (CPR - 1))) + 8 * hh) =
            make_uint2(bf16x2_rne(v[0], v[1]), bf16x2_rne(v[2], v[3]));
      }
    }
  }
  __builtin_amdgcn_s_waitcnt(0xC07F);             // lgkmcnt(0)
  lds_barrier();
  if (n >= p.N) return;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int r = RPQ * q + r0, m = m0 + r;
    if (m >= p.M) break;
    const uint4 o = *reinterpret_cast<const uint4*>(lds + r * ROWB + 16 * (ch ^ (r & (CPR - 1))));
    if (early) int8_put<false>(p.y + (int64_t)m * p.ys + n, int8_plus(o, res[q]));
    else int8_store8(p, m, n, o);
  }
}

// Any sizes and alignments: tiles of 64 T (n) x 64 T (m), 2 x 2 waves, 128 K bytes a stage through registers, stages of them under
// way, into two LDS buffers ([517, 1283] at K = 1291, T = 1: 9.5 us; 22 with one stage under way). Behind K a load takes the row's
// last 16 bytes, and what it should not have is dropped on the way to LDS: no load stands in a branch. SHORT: K < 16.
template <int T, bool SHORT>
__global__ __launch_bounds__(256) void int8_any_kernel(Int8Params p) {
  constexpr int kAhead = T == 1 ? 3 : 2, BT = 64 * T, J = 2 * T;
  __shared__ __align__(16) uint8_t lds[2][2][BT * 128];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wn = wave & 1, wm = wave >> 1;
  int m0, n0;
  int8_place<BT, BT>(p, int8_first(), m0, n0);
  const int c16 = 16 * (tid & 7), stages = (p.K + 127) >> 7;
  const int8_t* g[2][J];                          // b's and a's rows 32 j + tid / 8 (past the last: that one again)
#pragma unroll
  for (int j = 0; j < J; ++j) {
    g[0][j] = p.b + (int64_t)min(n0 + 32 * j + (tid >> 3), p.N - 1) * p.bs;
    g[1][j] = p.a + (int64_t)min(m0 + 32 * j + (tid >> 3), p.M - 1) * p.as;
  }
  uint4 v[kAhead][2][J];
  auto load = [&](int s, auto uc) __attribute__((always_inline)) {
    constexpr int u = decltype(uc)::value;
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if constexpr (SHORT) {
          uint8_t byte[16] = {};
          for (int k = 0; k < p.K; ++k)
            if (c16 == 0) byte[k] = (uint8_t)g[o][j][k];
          v[u][o][j] = __builtin_bit_cast(uint4, byte);
        } else {
          v[u][o][j] = load_any16(g[o][j] + min(128 * s + c16, p.K - 16));
        }
      }
  };
  v16i acc[T == 1 ? 2 : 1][T][T] = {};            // one block a wave: two sums, so that a product does not wait for the one before
  auto step = [&](int s, auto uc, bool last) __attribute__((always_inline)) {
    constexpr int u = decltype(uc)::value;
    const int buf = s & 1;
    if (!SHORT && last) {
#pragma unroll
      for (int j = 0; j < 2 * J; ++j) v[u][j / J][j % J] = drop_bytes(v[u][j / J][j % J], max(128 * s + c16 - (p.K - 16), 0));
    }
#pragma unroll
    for (int j = 0; j < 2 * J; ++j)
      *reinterpret_cast<uint4*>(&lds[buf][j / J][swz(32 * (j % J) + (tid >> 3), tid & 7)]) = v[u][j / J][j % J];
    __syncthreads();                              // stage s is there, and every wave is done with stage s - 1
    load(s + kAhead, uc);
#pragma unroll
    for (int q = 0; q < 4; ++q) {                 // 16-byte chunks 4 (q / 2) + 2 (lane / 32) + q % 2 of the row
      const int c = 4 * (q >> 1) + 2 * (lane >> 5) + (q & 1);
      v4i fb[T], fa[T];
#pragma unroll
      for (int i = 0; i < T; ++i) {
        fb[i] = *reinterpret_cast<const v4i*>(&lds[buf][0][swz(32 * (T * wn + i) + (lane & 31), c)]);
        fa[i] = *reinterpret_cast<const v4i*>(&lds[buf][1][swz(32 * (T * wm + i) + (lane & 31), c)]);
      }
#pragma unroll
      for (int i = 0; i < T; ++i)
#pragma unroll
        for (int j = 0; j < T; ++j) {
          v16i& sum = acc[T == 1 ? q & 1 : 0][i][j];
          sum = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[i], fa[j], sum, 0, 0, 0);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // Whole rounds of kAhead stages without a branch between their loads, which would make the compiler wait for loads of the later
  // stages too; then the last ones.
  each_up<kAhead>([&](auto u) __attribute__((always_inline)) { load(decltype(u)::value, u); });
  int s = 0;
  for (; s + kAhead < stages; s += kAhead)
    each_up<kAhead>([&](auto uc) __attribute__((always_inline)) { step(s + decltype(uc)::value, uc, false); });
  each_up<kAhead>([&](auto uc) __attribute__((always_inline)) {
    constexpr int u = decltype(uc)::value;
    if (s + u < stages) step(s + u, uc, s + u == stages - 1);
  });
  __syncthreads();                                // the epilogue overwrites the stages
  if constexpr (T == 1) acc[0][0][0] += acc[1][0][0];
  int8_epilogue<2, 2, T, T>(p, acc[0], &lds[0][0][0], m0, n0, wave, lane);
}

template <int WN, int WM, int TN, int TM, int NST, bool TAIL>
__global__ __launch_bounds__(64 * WN * WM) void int8_tile_kernel(Int8Params p) {
  constexpr int BK = 128, BN = 32 * WN * TN, BM = 32 * WM * TM, NW = WN * WM, kStage = (BN + BM) * BK;
  constexpr int RPI = 8, IPW = (BN + BM) / RPI / NW;      // rows a load, loads a wave and stage
  static_assert((BN + BM) % (RPI * NW) == 0 && BN % RPI == 0 && IPW * (NST - 1) < 64, "whole loads, countable by vmcnt");
  static_assert(NST * kStage >= BM * BN * 2, "the staged epilogue reuses the ring");
  __shared__ __align__(16) uint8_t lds[NST * kStage];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % WN, wm = wave / WN;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8_t*)lds;
  const int nst = (p.K + BK - 1) / BK;
  int m0, n0;
  int8_place<BN, BM>(p, int8_first(), m0, n0);

  const int8_t* const gb = p.b + (int64_t)n0 * p.bs;
  const int8_t* const ga = p.a + (int64_t)m0 * p.as;
  uint32_t goff[IPW];                             // within the tile's rows, below 2^32 (checked on the host)
  uint32_t past = 0;                              // bit q: load q's chunk of the last stage lies past K
  const int chunks = (p.K - (nst - 1) * BK) >> 4; // of the last stage
  // Lane i of load q fetches row 8 q + i / 8 of the wave's rows for place i % 8 in LDS.
  auto chunk_of = [&](int r) __attribute__((always_inline)) { return (lane & 7) ^ ((r >> 1) & 7); };
#pragma unroll
  for (int q = 0; q < IPW; ++q) {
    const int row0 = RPI * (wave * IPW + q), r = row0 + (lane >> 3), c = chunk_of(r);
    const int row = row0 >= BN ? min(r - BN, p.M - 1 - m0) : min(r, p.N - 1 - n0);
    goff[q] = (uint32_t)row * (uint32_t)(row0 >= BN ? p.as : p.bs) + 16u * (uint32_t)c;
    if (TAIL && c >= chunks) past |= 1u << q;
  }
  auto issue = [&](int s) __attribute__((always_inline)) {
    const uint32_t dst = lds0 + (uint32_t)(s % NST) * kStage;
#pragma unroll
    for (int q = 0; q < IPW; ++q) {
      const int row0 = RPI * (wave * IPW + q);
      const int8_t* src = row0 >= BN ? ga : gb;
      uint32_t off = goff[q] + (uint32_t)s * BK;
      if (TAIL && s == nst - 1 && ((past >> q) & 1u)) off = goff[q] - 16u * (uint32_t)chunk_of(row0 + (lane >> 3));
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst + row0 * BK), "v"(off), "s"(src)
                   : "memory", "m0");
    }
  };
  v16i acc[TN][TM];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = v16i{};
  v4i b[2][TN][2], a[2][TM][2];                   // [set][block][half]: set kc holds chunk kc (64 of K) of a stage
  auto read = [&](int s, auto kcc, bool last) __attribute__((always_inline)) {
    constexpr int kc = decltype(kcc)::value;
    const uint8_t* cur = lds + (s % NST) * kStage;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = 4 * kc + 2 * (lane >> 5) + h;
#pragma unroll
      for (int i = 0; i < TN; ++i) {
        b[kc][i][h] = *reinterpret_cast<const v4i*>(cur + swz(32 * (TN * wn + i) + (lane & 31), c));
        if (TAIL && last && c >= chunks) b[kc][i][h] = v4i{0, 0, 0, 0};
      }
#pragma unroll
      for (int j = 0; j < TM; ++j) a[kc][j][h] = *reinterpret_cast<const v4i*>(cur + swz(BN + 32 * (TM * wm + j) + (lane & 31), c));
    }
  };
  auto prod = [&](auto kcc) __attribute__((always_inline)) {
    constexpr int kc = decltype(kcc)::value;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[kc][i][h], a[kc][j][h], acc[i][j], 0, 0, 0);
  };
  using C0 = std::integral_constant<int, 0>;
  using C1 = std::integral_constant<int, 1>;
#pragma unroll
  for (int s = 0; s < NST; ++s)
    if (s < nst) issue(s);
  if (nst >= NST) __builtin_amdgcn_s_waitcnt(vmcnt_imm((NST - 1) * IPW));
  else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  lds_barrier();
  read(0, C0{}, nst == 1);
  int s = 0;
#pragma unroll 1
  for (; s + NST < nst; ++s) {
    read(s, C1{}, false);
    prod(C0{});
    __builtin_amdgcn_s_waitcnt(0xC07F);           // lgkmcnt(0): this wave's reads of stage s are done
    __builtin_amdgcn_s_waitcnt(vmcnt_imm((NST - 2) * IPW));     // this wave's loads of stage s + 1 landed
    lds_barrier();                                // ... and every wave's; stage s is retired
    issue(s + NST);
    read(s + 1, C0{}, false);
    prod(C1{});
  }
  // The last NST stages: nothing left to issue.
#pragma unroll 1
  for (; s < nst; ++s) {
    const bool last = s == nst - 1;
    read(s, C1{}, last);
    prod(C0{});
    if (!last) {
      __builtin_amdgcn_s_waitcnt(0xC07F);
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      lds_barrier();
      read(s + 1, C0{}, s + 1 == nst - 1);
    }
    prod(C1{});
  }
  __builtin_amdgcn_s_waitcnt(0xC07F);
  lds_barrier();                                  // the epilogue overwrites the ring
  int8_epilogue<WN, WM, TN, TM>(p, acc, lds, m0, n0, wave, lane);
}

// ---------------------------------------------------------------- large products
//
// Persistent 256 x 256 tiles, for K % 16 == 0, K > 128: a workgroup of WN x WM waves takes tiles L, L + G, ... and runs their stages (128 bytes
// of K each) as one stream through a ring of two LDS buffers: the loads of the next tile's first stages are under way while this
// one ends, and its output is written through 4 KB of LDS of each wave's own, so that a tile's end waits for no other
// wave and for no load.
// Two sets of fragments, a quarter of a stage (32 of K) each: while a quarter's products run, the next one's fragments are read,
// across the stage's barrier and the tile's end too. The order of a quarter is kept as it is written: a product, then part of the
// reads and loads, so that the wave issues none of them in a burst.
template <int WN, int WM, int TN, int TM, bool TAIL, bool STREAM, bool RES>
__global__ __launch_bounds__(64 * WN * WM) void int8_stream_kernel(Int8Params p) {
  constexpr int BK = 128, BN = 32 * WN * TN, BM = 32 * WM * TM, NW = WN * WM, kStage = (BN + BM) * BK;
  constexpr int RPI = 8, IPW = (BN + BM) / RPI / NW;                             // rows a load, loads a wave and stage
  static_assert((BN + BM) % (RPI * NW) == 0 && BN % (RPI * IPW) == 0 && TN % 2 == 0, "a wave's loads are of one operand");
  __shared__ __align__(16) uint8_t lds[2 * kStage + NW * 4096];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % WN, wm = wave / WN, hh = lane >> 5;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8_t*)lds + wave * (IPW * 1024);
  const int nst = (p.K + BK - 1) / BK, ntiles = p.tiles_n * p.tiles_m;
  // This wave's loads: rows row_w .. row_w + 8 IPW - 1 of b's tile (the first waves) or a's. Lane i of load q fetches row 8 q + i / 8
  // for place i % 8 in LDS.
  const int row_w = RPI * IPW * wave;
  const bool aop = row_w >= BN;
  const int8_t* src = nullptr;
  uint32_t goff[IPW];                             // within the tile's rows, below 2^32 (checked on the host)
  uint32_t past = 0;                              // bit q: load q's chunk of the last stage lies past K
  const int chunks = (p.K - (nst - 1) * BK) >> 4; // of the last stage
  auto chunk_of = [&](int r) __attribute__((always_inline)) { return (lane & 7) ^ ((r >> 1) & 7); };
  auto aim = [&](int t) __attribute__((always_inline)) {    // the loads at tile t
    int m0, n0;
    int8_place<BN, BM>(p, t, m0, n0);
    src = aop ? p.a + (int64_t)m0 * p.as : p.b + (int64_t)n0 * p.bs;
    const int rows = aop ? p.M - m0 : p.N - n0, base = aop ? row_w - BN : row_w;
    const uint32_t stride = (uint32_t)(aop ? p.as : p.bs);
#pragma unroll
    for (int q = 0; q < IPW; ++q) {
      const int r = base + RPI * q + (lane >> 3);
      goff[q] = (uint32_t)min(r, rows - 1) * stride + 16u * (uint32_t)chunk_of(r);
    }
  };
  if (TAIL) {
#pragma unroll
    for (int q = 0; q < IPW; ++q)
      if (chunk_of(row_w + RPI * q + (lane >> 3)) >= chunks) past |= 1u << q;
  }
  // Load q of stage s (of the tile that the loads aim at) into buffer buf.
  auto load_one = [&](int s, int buf, auto qc) __attribute__((always_inline)) {
    constexpr int q = decltype(qc)::value;
    uint32_t off = goff[q] + (uint32_t)s * BK;
    if (TAIL && s == nst - 1 && ((past >> q) & 1u)) off = goff[q] - 16u * (uint32_t)chunk_of(row_w + RPI * q + (lane >> 3));
    const uint32_t dst = lds0 + (uint32_t)buf * kStage + q * 1024;
    const int8_t* const from = src;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off), "s"(from) : "memory", "m0");
  };

  v16i acc[TN][TM];
  v4i b[2][TN], a[2][TM];                         // [set][block]: set x % 2 holds the quarter x of a stage
  constexpr int kReads = TN + TM, kProds = TN * TM;
  // Fragment f of quarter x of a stage in buffer buf: the a blocks, then the b blocks.
  auto read_one = [&](int buf, auto xc, auto fc, bool last) __attribute__((always_inline)) {
    constexpr int x = decltype(xc)::value, f = decltype(fc)::value;
    const uint8_t* cur = lds + buf * kStage;
    const int c = 4 * (x >> 1) + 2 * hh + (x & 1);
    if constexpr (f < TM) {
      a[x & 1][f] = *reinterpret_cast<const v4i*>(cur + swz(BN + 32 * (TM * wm + f) + (lane & 31), c));
    } else {
      constexpr int i = f - TM;
      b[x & 1][i] = *reinterpret_cast<const v4i*>(cur + swz(32 * (TN * wn + i) + (lane & 31), c));
      if (TAIL && last && c >= chunks) b[x & 1][i] = v4i{0, 0, 0, 0};
    }
  };
  // The products of quarter x; after each its share of the reads of the next quarter, of buffer rbuf,
  // and behind the last quarter's, of the loads.
  auto quarter = [&](auto xc, int rbuf, bool rlast, int ls, int lbuf) __attribute__((always_inline)) {
    constexpr int x = decltype(xc)::value;
    each_up<kProds>([&](auto uc) __attribute__((always_inline)) {
      constexpr int u = decltype(uc)::value, i = u / TM, j = u % TM;
      acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[x & 1][i], a[x & 1][j], acc[i][j], 0, 0, 0);
      constexpr int span = kProds * 3 / 4, lo = u * kReads / span, hi = (u + 1) * kReads / span;
      if constexpr (u < span)
        each_up<hi - lo>([&](auto fc) __attribute__((always_inline)) {
          read_one(rbuf, std::integral_constant<int, (x + 1) & 3>{}, std::integral_constant<int, lo + decltype(fc)::value>{}, rlast);
        });
      if constexpr (x == 3) {
        constexpr int l0 = u * IPW / kProds, l1 = (u + 1) * IPW / kProds;
        each_up<l1 - l0>([&](auto qc) __attribute__((always_inline)) { load_one(ls, lbuf, std::integral_constant<int, l0 + decltype(qc)::value>{}); });
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  using X0 = std::integral_constant<int, 0>;
  using X1 = std::integral_constant<int, 1>;
  using X2 = std::integral_constant<int, 2>;
  using X3 = std::integral_constant<int, 3>;

  // The tile at m0, n0: each wave 32 columns of its rows at a time through its own LDS (2 KB for 32 x 32 of them; row r: 64 bytes,
  // 16-byte chunk c at c ^ (r / 4 % 4)). A lane holds the scales and biases of columns 64 k + lane and hands them to the others; the
  // residual's next columns are under way while these are written ([16384, 5120] at K = 1280 with a residual 162 us, 180 with each
  // load where it is used; with a bias 117 and 133). Rows are reached by 32-bit offsets (checked on the host).
  static_assert(TM * 2048 <= 4096 && TN % 2 == 0, "the wave's own LDS");
  uint8_t* const own = lds + 2 * kStage + wave * 4096;
  auto write_out = [&](int m0, int n0) __attribute__((always_inline)) {
    int ln = lane;                                // the places below are worked out here, not held in registers through the stages
    asm volatile("" : "+v"(ln));
    const int h = ln >> 5, mw = min(m0 + 32 * TM * wm, p.M - 1), nw = min(n0 + 32 * TN * wn, p.N - 8);      // a wave without rows or columns: the last ones
    const bool some = m0 + 32 * TM * wm < p.M && n0 + 32 * TN * wn < p.N;
    const uint16_t* const res_w = RES ? p.res + (int64_t)mw * p.rs + nw : nullptr;
    uint16_t* const y_w = p.y + (int64_t)mw * p.ys + nw;
    const uint32_t rs = RES ? (uint32_t)p.rs : 0, ys = (uint32_t)p.ys;
    uint4 res[2][TM][2];
    auto fetch = [&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value;
      const uint32_t n = min(32 * i + 8 * (ln & 3), p.N - 8 - nw);
#pragma unroll
      for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t m = min(32 * j + 16 * q + (ln >> 2), p.M - 1 - mw);
          res[i & 1][j][q] = *reinterpret_cast<const uint4*>(res_w + (m * rs + n));
        }
    };
    float sa[TM], sbl[TN / 2], bl[TN / 2];
#pragma unroll
    for (int j = 0; j < TM; ++j) sa[j] = p.sa[(int64_t)min(mw + 32 * j + (ln & 31), p.M - 1) * p.sa_step];
#pragma unroll
    for (int k = 0; k < TN / 2; ++k) {
      const int n = min(nw + 64 * k + ln, p.N - 1);
      sbl[k] = p.sb[n];
      bl[k] = int8_bias(p, n);
    }
    if (RES) fetch(std::integral_constant<int, 0>{});
    asm volatile("" ::: "memory");
    each_up<TN>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value;
      if constexpr (RES && i + 1 < TN) fetch(std::integral_constant<int, i + 1>{});
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float sb[4], bias[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int from = 16 * h + 4 * (32 * (i & 1) + 8 * g + e);               // bytes
          sb[e] = __int_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_int(sbl[i / 2])));
          bias[e] = __int_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_int(bl[i / 2])));
        }
#pragma unroll
        for (int j = 0; j < TM; ++j) {
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = int8_value(acc[i][j][4 * g + e], sa[j], sb[e], bias[e]);
          *reinterpret_cast<uint2*>(own + j * 2048 + (ln & 31) * 64 + 16 * (g ^ ((ln >> 2) & 3)) + 8 * h) =
              make_uint2(bf16x2_rne(v[0], v[1]), bf16x2_rne(v[2], v[3]));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int j = 0; j < TM; ++j) acc[i][j] = v16i{};
      __builtin_amdgcn_s_waitcnt(0xC07F);         // lgkmcnt(0): the wave's own writes
      asm volatile("" ::: "memory");
      const int n = 32 * i + 8 * (ln & 3);
#pragma unroll
      for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int r = 16 * q + (ln >> 2), m = 32 * j + r;
          uint4 o = *reinterpret_cast<const uint4*>(own + j * 2048 + r * 64 + 16 * ((ln & 3) ^ ((r >> 2) & 3)));
          if (RES) o = int8_plus(o, res[i & 1][j][q]);
          if (some && m < p.M - mw && n < p.N - nw) int8_put<STREAM>(y_w + ((uint32_t)m * ys + (uint32_t)n), o);
        }
      asm volatile("" ::: "memory");
    });
  };

#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j) acc[i][j] = v16i{};
  int t = int8_first(), buf = 0;
  aim(t);
  each_up<IPW>([&](auto q) __attribute__((always_inline)) { load_one(0, 0, q); });
  each_up<IPW>([&](auto q) __attribute__((always_inline)) { load_one(1, 1, q); });
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(IPW));
  lds_barrier();
  each_up<kReads>([&](auto f) __attribute__((always_inline)) { read_one(0, X0{}, f, false); });
#pragma unroll 1
  for (; t < ntiles; t += gridDim.x) {
    // Behind the last tile the loads and reads run on over it again, and nothing uses them.
    const int next = t + (int)gridDim.x < ntiles ? t + (int)gridDim.x : t;
#pragma unroll 1
    for (int s = 0; s < nst; ++s) {
      const bool last = s == nst - 1;
      quarter(X0{}, buf, last, 0, 0);
      quarter(X1{}, buf, last, 0, 0);
      quarter(X2{}, buf, last, 0, 0);
      // The last quarter's fragments are read: the wave's reads of the stage are over, and its loads of the next one have landed.
      __builtin_amdgcn_s_waitcnt(0xC07F);
      __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      lds_barrier();                              // ... and every wave's: the stage's buffer is free
      int ls = s + 2;
      if (ls >= nst) {
        if (ls == nst) aim(next);
        ls -= nst;
      }
      quarter(X3{}, buf ^ 1, s + 1 == nst - 1, ls, buf);
      buf ^= 1;
    }
    int m0, n0;
    int8_place<BN, BM>(p, t, m0, n0);
    write_out(m0, n0);
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));       // no load is under way to LDS that is another workgroup's by then
}

// ---------------------------------------------------------------- few rows
//
// Decode steps: up to 16 rows and few enough channels for one workgroup a compute unit (int8_few), bound by the weight's bytes and
// by latency. A workgroup takes 16 output channels and all of K, cut among its 8 waves in blocks of 128; the weight goes from
// memory to registers, every 128-byte line read by one wave, the a rows through LDS; the waves' sums are joined in LDS.
// x given (not a): the rows are quantised here first, as flw_rows8 does it, by every workgroup for itself, while its first weight
// loads are under way: one launch instead of two for the price of reading x again from the L2.
// v_mfma_i32_16x16x64_i8: lane (row r = lane % 16, q = lane / 16) holds bytes 32 q + 16 j .. + 15 of a block's row for product j.
constexpr int kFewWaves = 8, kFewAhead = 4, kFewRows = 16;

__host__ __device__ __forceinline__ int few_ld(int K) { return (K + 127) / 128 * 128 + 16; }     // LDS bytes a row: rows on banks of their own
static int few_lds_bytes(int64_t M, int64_t K) { return (int)M * few_ld((int)K) + kFewWaves * 1024 + 4 * (kFewRows + kFewWaves); }

// The waves' shares of the rows: eight waves for one row, four for each of two, two for each of three or four, one for each of more;
// this wave is the sub-th of its row's, its rows are first, first + step, ...
__host__ __device__ __forceinline__ int few_waves(int M) { return M == 1 ? 8 : M == 2 ? 4 : M <= 4 ? 2 : 1; }
struct FewShare {
  int waves, sub, first, step;
  __device__ __forceinline__ explicit FewShare(int M) {
    const int wave = threadIdx.x >> 6;
    waves = few_waves(M);
    sub = wave & (waves - 1);
    first = wave / waves;
    step = kFewWaves / waves;
  }
};

template <typename T>
__device__ __forceinline__ void few_quantise(const Int8Params& p, uint8_t* rows, float* scale, uint32_t* red, int ld) {
  constexpr int U = 4;                            // loads under way
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const FewShare s(p.M);
  const int c0 = 8 * (64 * s.sub + lane), dc = 512 * s.waves;
  for (int r = s.first; r < p.M; r += s.step) {   // once where several waves share a row
    const T* x = static_cast<const T*>(p.x) + r * p.xs;
    float f[U][8];
    auto get = [&](int c) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 8; j += Vec16<T>::N)
          if (c + u * dc < p.K) Vec16<T>::load(x + c + u * dc + j, f[u] + j);
    };
    uint32_t m = 0;
    for (int c = c0; c < p.K; c += U * dc) {
      get(c);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t v = c + u * dc < p.K ? abs_bits(f[u][e]) : 0u;
          m = m > v ? m : v;
        }
    }
    m = wave_max_u32(m);
    if (s.waves > 1) {
      if (lane == 0) red[wave] = m;
      __syncthreads();
      for (int k = 0; k < s.waves; ++k) m = max(m, red[(wave & ~(s.waves - 1)) + k]);
    }
    const Int8Scale q(m);
    if (lane == 0 && s.sub == 0) scale[r] = q.scale;
    for (int c = c0; c < ld - 16; c += U * dc) {
      if (dc * U < p.K) get(c);                   // else the values are there still
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * dc < ld - 16) *reinterpret_cast<uint2*>(rows + r * ld + c + u * dc) = c + u * dc < p.K ? q.codes(f[u]) : make_uint2(0, 0);
    }
  }
  if (s.waves > 1 && s.first >= p.M) __syncthreads();       // the waves without a row (M = 3) meet the others
}

__global__ __launch_bounds__(64 * kFewWaves) void int8_few_kernel(Int8Params p) {
  extern __shared__ __align__(16) uint8_t few_lds[];
  const int ld = few_ld(p.K), lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, q = lane >> 4;
  uint8_t* const rows = few_lds;                                                // [M][ld]
  int* const sums = reinterpret_cast<int*>(rows + p.M * ld);                    // [8][64][4]
  float* const scale = reinterpret_cast<float*>(sums + kFewWaves * 256);
  uint32_t* const red = reinterpret_cast<uint32_t*>(scale + kFewRows);
  const int n0 = blockIdx.x * 16, blocks = (p.K + 127) >> 7;

  const int8_t* const w = p.b + (int64_t)min(n0 + row, p.N - 1) * p.bs;
  v4i bw[kFewAhead][2];
  auto load = [&](int k, v4i (&to)[2]) __attribute__((always_inline)) {         // block k; what lies past K meets zeros of a
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int c = 128 * k + 32 * q + 16 * j;
      to[j] = *reinterpret_cast<const v4i*>(w + (c < p.K ? c : 0));
    }
  };
#pragma unroll
  for (int u = 0; u < kFewAhead; ++u)
    if (wave + kFewWaves * u < blocks) load(wave + kFewWaves * u, bw[u]);

  if (p.x != nullptr) {
    if (p.x32) few_quantise<float>(p, rows, scale, red, ld);
    else few_quantise<uint16_t>(p, rows, scale, red, ld);
  } else {
    const FewShare s(p.M);
    const int end = ld - 16, dc = 1024 * s.waves;
    for (int r = s.first; r < p.M; r += s.step)
      for (int c = 16 * (64 * s.sub + lane); c < end; c += 4 * dc) {
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (c + u * dc < p.K) v[u] = *reinterpret_cast<const uint4*>(p.a + r * p.as + c + u * dc);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (c + u * dc < end) *reinterpret_cast<uint4*>(rows + r * ld + c + u * dc) = c + u * dc < p.K ? v[u] : make_uint4(0, 0, 0, 0);
      }
  }
  __syncthreads();
  // The scales, biases and residual of this thread's outputs (below), under way during the products.
  const int l = threadIdx.x, m = l & 15, n = n0 + 4 * (l >> 4);
  float sb[4], bias[4] = {}, res[4];
  if (l < 64) {
#pragma unroll
    for (int e = 0; e < 4; ++e) sb[e] = p.sb[(int64_t)min(n + e, p.N - 1) * p.sb_step];
    if (p.bias != nullptr) {
      if (p.bias32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) bias[e] = static_cast<const float*>(p.bias)[min(n + e, p.N - 1)];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) bias[e] = bf16_to_f32(static_cast<const uint16_t*>(p.bias)[min(n + e, p.N - 1)]);
      }
    }
    if (p.res != nullptr) {
#pragma unroll
      for (int e = 0; e < 4; ++e) res[e] = bf16_to_f32(p.res[min(m, p.M - 1) * p.rs + min(n + e, p.N - 1)]);
    }
  }
  const uint8_t* const a = rows + min(row, p.M - 1) * ld + 32 * q;
  v4i acc[2] = {};
  for (int k0 = wave; k0 < blocks; k0 += kFewWaves * kFewAhead) {
#pragma unroll
    for (int u = 0; u < kFewAhead; ++u) {
      const int k = k0 + kFewWaves * u;
      if (k >= blocks) break;                     // wave-uniform
#pragma unroll
      for (int j = 0; j < 2; ++j)
        acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bw[u][j], *reinterpret_cast<const v4i*>(a + 128 * k + 16 * j), acc[j], 0, 0, 0);
      const int ahead = k + kFewWaves * kFewAhead;
      if (ahead < blocks) load(ahead, bw[u]);
    }
  }
  *reinterpret_cast<v4i*>(sums + (wave * 64 + lane) * 4) = acc[0] + acc[1];
  __syncthreads();
  // Four outputs a thread: columns 4 (l / 16) + 0..3 of row l % 16 lie at l.
  if (l >= 64 || m >= p.M) return;
  v4i s = *reinterpret_cast<const v4i*>(sums + l * 4);
#pragma unroll
  for (int k = 1; k < kFewWaves; ++k) s += *reinterpret_cast<const v4i*>(sums + (k * 64 + l) * 4);
  const float sa = p.x != nullptr ? scale[m] : p.sa[(int64_t)m * p.sa_step];
  uint16_t* y = p.y + m * p.ys + n;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n + e >= p.N) break;
    float v = int8_value(s[e], sa, sb[e], bias[e]);
    if (p.res) v = round_bf16(v) + res[e];
    y[e] = (uint16_t)f32_to_bf16_bits(v);
  }
}

// Codes of int8 within [-128, 127]: K products of at most 2^14 fit an int32.
constexpr int64_t kInt8MaxK = 131071;

static bool on16(const void* p, int64_t stride_bytes, int64_t rows) {
  return (uintptr_t)p % 16 == 0 && (stride_bytes % 16 == 0 || rows == 1);
}

// The few-row kernel's shapes: one workgroup of 16 channels a compute unit at most ([16, 4096] at K = 4096 8.5 us against 8.9 on
// 64 x 32 tiles, [16, 1280] at K = 3392 5.3 against 8.8, [1, 3840] at K = 1280 3.5 against 4.5; beyond, [16, 8192] at K = 2048 7.2
// against 6.3), and rows that fit the LDS.
static bool few(int64_t M, int64_t N, int64_t K) {
  return M <= kFewRows && (N + 15) / 16 <= compute_units() && few_lds_bytes(M, K) <= 150 * 1024;
}

// Whether its workgroups quantise the rows themselves: up to 3584 values a wave (one launch against two, us: [1, 3840] at K = 1280 4.5
// and 6.4, [16, 3840] 6.9 and 7.9, [4, 4096] at K = 4096 8.4 and 9.7; equal at [8, 1280], K = 3392, and at [4, 2048], K = 8192; [16,
// 4096] at K = 4096 16.7 and 12.1).
static bool few_quantises(int64_t M, int64_t K) {
  const int waves = few_waves((int)M), rows = kFewWaves / waves;
  return (M + rows - 1) / rows * K <= 3584 * waves;
}

struct Int8Kernel {
  const void* fn;
  int bn, bm, threads;
  bool persistent;
};

template <int WN, int WM, int TN, int TM, int NST>
static Int8Kernel tile_of(bool tail) {
  return {tail ? reinterpret_cast<const void*>(&int8_tile_kernel<WN, WM, TN, TM, NST, true>)
               : reinterpret_cast<const void*>(&int8_tile_kernel<WN, WM, TN, TM, NST, false>),
          32 * WN * TN, 32 * WM * TM, 64 * WN * WM, false};
}
template <bool TAIL, bool RES>
static Int8Kernel stream_of(bool non_temporal) {
  return {non_temporal ? reinterpret_cast<const void*>(&int8_stream_kernel<2, 4, 4, 2, TAIL, true, RES>)
                       : reinterpret_cast<const void*>(&int8_stream_kernel<2, 4, 4, 2, TAIL, false, RES>),
          256, 256, 512, true};
}

// The tile for an [M, N] output. While one of the smaller tiles gives at most one tile a compute unit, the smallest such: a tile's
// time hardly depends on how many others run, and grows with its size (K = 1280, us: [64, 3840] 4.7 on 64 x 32, 5.0 on 64 x 64,
// 7.8 on 128 x 128; [512, 1280] 5.2 on 64 x 64, 8.1 on 128 x 128; [2048, 1280] 10.0 on 128 x 128, 11.7 on 64 x 64). Beyond, two
// workgroups of 128 x 128 share a unit, or the stream of 256 x 256 tiles, by their rounds: one of the pairs takes 0.52 to 0.66 of
// one of the stream ([8192, 3392] at K = 1280 51 us on pairs, 49 streamed; [32768, 1024] at K = 4096 176 and 154; [4096, 1280] at
// K = 3392, one round of either, 32 and 50).
// An output from 64 MiB on is stored past the caches, which it would sweep clean of the operands and not find room in ([8192, 5120]
// at K = 1280 72 -> 67 us, [16384, 5120] 151 -> 115; [8192, 3392] 50 either way, and a smaller one is still there for its reader).
static Int8Kernel kernel_of(const Int8Params& p) {
  const int64_t M = p.M, N = p.N, cus = compute_units();
  auto rounds = [M, N](int64_t bn, int64_t bm, int64_t at_once) { return ((N + bn - 1) / bn * ((M + bm - 1) / bm) + at_once - 1) / at_once; };
  const bool tail = p.K % 128 != 0;
  if (rounds(64, 32, cus) == 1) return tile_of<2, 1, 1, 1, 4>(tail);
  if (rounds(64, 64, cus) == 1) return tile_of<2, 2, 1, 1, 4>(tail);
  if (rounds(128, 128, cus) == 1) return tile_of<4, 2, 1, 2, 3>(tail);
  if (p.K > 128 && p.wide && (double)rounds(256, 256, cus) <= 0.6 * (double)rounds(128, 128, 2 * cus)) {
    const bool past = M * N * 2 >= 64ll << 20;
    if (p.res != nullptr) return tail ? stream_of<true, true>(past) : stream_of<false, true>(past);
    return tail ? stream_of<true, false>(past) : stream_of<false, false>(past);
  }
  return tile_of<4, 2, 1, 2, 2>(tail);
}

// Any alignment: tiles of 128 x 128 where there are three of 64 x 64 a compute unit and a tile is not mostly empty (us, on 64 / 128:
// [1000, 2000] at K = 1291 14.8 / 17.3, [1500, 2000] 19.6 / 17.9, [2000, 2000] at K = 2001 32.6 / 22.8, [8191, 3391] at K = 1279
// 131 / 84, [30, 50257] there 23.6 / 24.7).
static Int8Kernel any_of(const Int8Params& p) {
  const int64_t tiles = (((int64_t)p.N + 63) / 64) * (((int64_t)p.M + 63) / 64);
  if (p.K < 16) return {reinterpret_cast<const void*>(&int8_any_kernel<1, true>), 64, 64, 256, false};
  if (tiles < 3 * compute_units() || std::min(p.M, p.N) <= 64) return {reinterpret_cast<const void*>(&int8_any_kernel<1, false>), 64, 64, 256, false};
  return {reinterpret_cast<const void*>(&int8_any_kernel<2, false>), 128, 128, 256, false};
}

// p.x set: the rows are quantised by the few-row kernel (few() holds, 16-byte rows of x, K % 16 == 0).
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
  FLW_REQUIRE(p.x != nullptr || (p.a != nullptr && p.sa != nullptr), FLW_E_INVALID, "null pointer");
  FLW_REQUIRE(p.b != nullptr && p.sb != nullptr && p.y != nullptr, FLW_E_INVALID, "null pointer");
  FLW_REQUIRE((p.x != nullptr || p.as >= K) && p.bs >= K && p.ys >= N && (p.res == nullptr || p.rs >= N), FLW_E_INVALID,
              "a row stride below the row");
  FLW_REQUIRE((uintptr_t)p.y % 2 == 0 && (uintptr_t)p.res % 2 == 0 && (uintptr_t)p.sa % 4 == 0 && (uintptr_t)p.sb % 4 == 0,
              FLW_E_INVALID, "misaligned pointer");
  FLW_REQUIRE(p.bias == nullptr || ((bias_dtype == FLW_F32 || bias_dtype == FLW_BF16) &&
                                    (uintptr_t)p.bias % (bias_dtype == FLW_F32 ? 4 : 2) == 0),
              FLW_E_INVALID, "the bias must be aligned bf16 or fp32");
  p.M = (int)M; p.N = (int)N; p.K = (int)K;
  p.sa_step = sa_count > 1; p.sb_step = sb_count > 1;
  p.bias32 = bias_dtype == FLW_F32;
  // Rows that the vector kernels take, and tiles whose rows are reached by 32-bit offsets.
  const bool vector = K % 16 == 0 && on16(p.b, p.bs, N) && (p.x != nullptr || on16(p.a, p.as, M)) &&
                      std::max(M > 1 ? p.as : 0, N > 1 ? p.bs : 0) <= (0xFFFFFFFFll - K) / 256;
  if (vector && few(M, N, K)) {
    p.tiles_n = (int)((N + 15) / 16);
    const Timer tm = take_timer();
    (void)launch_ext(reinterpret_cast<const void*>(&int8_few_kernel), dim3((unsigned)p.tiles_n), dim3(64 * kFewWaves),
                     (size_t)few_lds_bytes(M, K), s, p, tm.start, tm.stop);
    return check_launch(name);
  }
  p.wide = N % 8 == 0 && p.sb_step == 1 && std::max(p.ys, p.rs) < 1 << 25 && (uintptr_t)p.sb % 16 == 0 && on16(p.y, 2 * p.ys, M) &&
           (p.res == nullptr || on16(p.res, 2 * p.rs, M));
  const Int8Kernel k = vector ? kernel_of(p) : any_of(p);
  const int64_t tiles_n = (N + k.bn - 1) / k.bn, tiles_m = (M + k.bm - 1) / k.bm;
  FLW_REQUIRE(k.persistent ? tiles_n * tiles_m <= 0x3FFFFFFFll : tiles_n * tiles_m * k.threads <= 0xFFFFFFFFll, FLW_E_UNSUPPORTED,
              "too many output tiles");         // a launch holds fewer than 2^32 threads
  p.tiles_n = (int)tiles_n;
  p.tiles_m = (int)tiles_m;
  const int64_t grid = k.persistent ? std::min<int64_t>(tiles_n * tiles_m, compute_units()) : tiles_n * tiles_m;
  (void)launch_timed(k.fn, dim3((unsigned)grid), dim3((unsigned)k.threads), s, p);
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
  if (M > 0 && K % 16 == 0 && few(M, N, K) && few_quantises(M, K) && (dtype == FLW_F32 || dtype == FLW_BF16) && on16(b, b_row_stride, N) &&
      on16(x, x_row_stride * (dtype == FLW_F32 ? 4 : 2), M) && x != nullptr && x_row_stride >= K && b_row_stride <= (0xFFFFFFFFll - K) / 256) {
    Int8Params p{};
    p.x = x; p.xs = x_row_stride; p.x32 = dtype == FLW_F32;
    p.b = b; p.bs = b_row_stride; p.sb = b_scale; p.bias = bias;
    p.res = static_cast<const uint16_t*>(residual); p.rs = residual_row_stride;
    p.y = static_cast<uint16_t*>(y); p.ys = y_row_stride;
    return int8_mm(p, M, N, K, M, b_scale_count, bias_dtype, static_cast<hipStream_t>(stream), "flw_int8_linear");
  }
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
