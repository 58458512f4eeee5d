// Attention of the newest tokens of each sequence over a paged key-value cache (the decode step).
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(q_i . k_j * scale - m_i),
//   over the keys j of i's sequence with max(0, i - window + 1) <= j <= i.
//
// The keys are read from their pages, so every byte of K and V in the window is read once and nothing else
// matters: the bound is HBM. A K / V head is shared by G query heads and by the T new tokens: their T G rows are
// the 16 columns of an MFMA tile (one tile for T G <= 16).
//
// One wave takes blocks of 64 keys on its own, from global memory to the accumulators without LDS or barriers:
//   S^T (keys x rows) = K Q^T on v_mfma_f32_16x16x32_bf16: a lane holds 16 scores of ONE row, so the running
//     maximum and sum are per lane, joined over the four lane groups by two lane swaps a block;
//   O^T (D x rows) += V^T P^T: a lane's scores are the operand P^T as they stand, because the K rows are taken in
//     the order that puts a lane's scores next to each other along the keys; V^T is read as it is, since a page
//     holds V as (D, page size).
// P goes to the product as two bf16 terms (p rounded, and what that lost), so that it carries 16 bits instead of 8:
// the matrix cores idle here, and one term would cost as much accuracy as the output's own rounding. Scores, the
// maximum, the sum and O are fp32.
// e4m3 pages: codes widened to bf16 in registers (exact); the K scale multiplies the score, the V scale the output.
//
// Work is cut over (sequence, kv head, row tile) and, where those are few, over the key range (`splits` parts a
// sequence, each of at least one block a wave); a second launch joins the parts.

#include "flw_common.h"

namespace flw {

typedef __bf16 pa_bf8 __attribute__((ext_vector_type(8)));
typedef float pa_f4 __attribute__((ext_vector_type(4)));

struct PagedAttn {
  const uint16_t* q;
  int64_t qsb, qsh, qst;
  const uint8_t* k;               // (P, KV, page, D)
  const uint8_t* v;               // (P, KV, D, page)
  const int32_t* tables;          // (B, M)
  const int32_t* lens;
  const int32_t* counts;          // NULL: T new tokens everywhere
  const float* k_scale;           // e4m3: one a kv head
  const float* v_scale;
  uint16_t* out;
  int64_t osb, osh, ost;
  float* lse;                     // (B, H, T) or NULL
  float* part;                    // splits > 1: (B, KV, tiles, splits) x [16 D + 32]
  int64_t P;
  int B, H, KV, G, T, rows, tiles, M, shift, window, splits, bshift;
  float scale;                    // softmax scale x log2 e
};

constexpr int kPaWaves = 4;       // waves a workgroup: each takes every 4th block of the part
constexpr float kPaLn2 = 0.69314718055994531f;

// Keys a block: 64, or 32 where 64 would not fit the registers (D = 128 in bf16: K and V are 64 words each a lane then).
template <int D, bool F8> constexpr int pa_block() { return D == 128 && !F8 ? 32 : 64; }

// One row tile's keys: rows r0 .. of `here` rows (tokens t_lo .. t_hi), keys [lo, hi), and its blocks of 2^bshift keys.
struct PaRange {
  int base, cnt, here, t_lo, t_hi, lo, hi, kb_lo, kb_hi, chunk, used;
  __device__ __forceinline__ PaRange(const PagedAttn& p, int b, int tile) {
    cnt = p.counts != nullptr ? p.counts[b] : p.T;
    cnt = cnt < 0 ? 0 : cnt;
    int len = p.lens[b];
    base = (len < 0 ? 0 : len) - cnt;                     // the first new token's position
    const int r0 = 16 * tile;
    here = p.rows - r0 < 16 ? p.rows - r0 : 16;
    t_lo = r0 / p.G;
    t_hi = (r0 + here - 1) / p.G;
    t_hi = t_hi < cnt ? t_hi : cnt - 1;
    lo = hi = 0;
    if (t_lo <= t_hi && p.window > 0) {
      const int64_t first = (int64_t)base + t_lo - p.window + 1, cap = (int64_t)p.M << p.shift;
      const int64_t last = (int64_t)base + t_hi + 1;      // positions past the table are answered with NaN: never read
      hi = (int)(last < cap ? last : cap);
      lo = (int)(first > 0 ? (first < cap ? first : cap) : 0);
    }
    kb_lo = lo >> p.bshift;
    kb_hi = hi > lo ? (hi + (1 << p.bshift) - 1) >> p.bshift : kb_lo;
    const int n = kb_hi - kb_lo;
    chunk = (n + p.splits - 1) / p.splits;
    chunk = chunk < kPaWaves ? kPaWaves : chunk;
    used = (n + chunk - 1) / chunk;
  }
};

// Writes output row r of (b, kvh) from its unnormalised O (4 values from dim d on), sum l and maximum m. A row without
// keys is zero, one past its table NaN.
__device__ __forceinline__ void pa_write(const PagedAttn& p, const PaRange& rg, int b, int kvh, int r, int d, float4 o,
                                         float l, float m) {
  const int t = r / p.G, h = kvh * p.G + (r - t * p.G);
  const bool real = t < rg.cnt && rg.base + t >= 0 && p.window > 0;
  const bool past = real && (int64_t)rg.base + t >= ((int64_t)p.M << p.shift);
  const float vs = p.v_scale != nullptr ? p.v_scale[kvh] : 1.0f;
  const float inv = real ? (past ? __builtin_nanf("") : vs / l) : 0.0f;
  if (!real) o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  *reinterpret_cast<uint2*>(p.out + (int64_t)b * p.osb + (int64_t)h * p.osh + (int64_t)t * p.ost + d) =
      make_uint2(bf16x2_rne(o.x * inv, o.y * inv), bf16x2_rne(o.z * inv, o.w * inv));
  if (p.lse != nullptr && d == 0)
    p.lse[((int64_t)b * p.H + h) * p.T + t] =
        !real ? -INFINITY : past ? __builtin_nanf("") : (m + __builtin_amdgcn_logf(l)) * kPaLn2;
}

// Eight e4m3 codes widened to bf16 (exact).
__device__ __forceinline__ pa_bf8 pa_widen(uint32_t lo, uint32_t hi) {
  const flw_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, false);
  const flw_bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, true);
  const flw_bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, false);
  const flw_bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, true);
  return pa_bf8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Whether a word of V (two bf16 or four e4m3) holds a NaN or an infinity.
template <bool F8>
__device__ __forceinline__ bool pa_not_finite(uint32_t w) {
  if constexpr (!F8) return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
  const uint32_t x = w & 0x7F7F7F7Fu;                       // a byte of 0x7F is NaN
  return ((x + 0x01010101u) & 0x80808080u) != 0;
}

// The 64 keys of a block as the lanes read them (n = lane & 15, g = lane >> 4). K: four tiles of 16 rows, tile i's
// row m being key koff(i, m); the scores of tile i then are keys koff(i, 4 g + j), j = 0 .. 3, and the 8 keys of a
// lane in V's step s are tiles 2 s and 2 s + 1: consecutive, one 16-byte read (bf16: 8 keys; e4m3: both steps' 16).
template <bool F8>
__device__ __forceinline__ int pa_koff(int i, int m) {
  return F8 ? 16 * (m >> 2) + 4 * i + (m & 3) : 32 * (i >> 1) + 8 * (m >> 2) + 4 * (i & 1) + (m & 3);
}

// The pages of a block's runs of 16 keys (a page holds at least 16): page numbers, 0 for a run outside the range and
// for one whose entry is no page; `bad` has the latter's bits.
struct PaPages {
  int id0, id1, id2, id3, bad;
};
template <int NK>
__device__ __forceinline__ PaPages pa_pages(const PagedAttn& p, const int32_t* row, int kb, int lo, int hi) {
  // scalar loads: the address is the wave's
  const __attribute__((address_space(4))) int32_t* crow = (const __attribute__((address_space(4))) int32_t*)row;
  int id[NK / 16], bad = 0;
#pragma unroll
  for (int c = 0; c < NK / 16; ++c) {
    const int pos = NK * kb + 16 * c;
    const bool in = pos < hi && pos + 16 > lo;
    const int e = in ? crow[pos >> p.shift] : 0;          // hi is at most the table's positions: the entry exists
    const bool ok = (uint32_t)e < (uint32_t)p.P;
    bad |= ok ? 0 : 1 << c;
    id[c] = ok ? e : 0;
  }
  if constexpr (NK == 64) return PaPages{id[0], id[1], id[2], id[3], bad};
  else return PaPages{id[0], id[1], 0, 0, bad};
}
template <int NK>
__device__ __forceinline__ int pa_page_of(PaPages pg, int c) {       // c differs between lanes
  const int a = c & 1 ? pg.id1 : pg.id0;
  if (NK == 32) return a;
  const int b = c & 1 ? pg.id3 : pg.id2;
  return c & 2 ? b : a;
}

template <int D, bool F8>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(PagedAttn p) {
  constexpr int KS = D / 32, DT = D / 16;
  constexpr int NK = pa_block<D, F8>(), KT = NK / 16, VS = NK / 32;   // keys a block, tiles of K, steps of V
  constexpr int KW = F8 ? D / 4 / 4 : D / 4 / 2;          // 32-bit words of K a lane holds per tile
  constexpr int VW = F8 ? 4 : 4 * VS;                          // and of V per tile of 16 dims
  constexpr int KPW = F8 ? 4 : 2;                         // keys a word of V
  constexpr uint32_t KMASK = F8 ? 0xFFu : 0xFFFFu;
  __shared__ float so[kPaWaves][16][D + 4];
  __shared__ float sm[kPaWaves][16], sl[kPaWaves][16];
  const int b = blockIdx.z, kvh = blockIdx.y;
  const int tile = (int)blockIdx.x / p.splits, split = (int)blockIdx.x - tile * p.splits;
  const PaRange rg(p, b, tile);
  if (split >= rg.used && split > 0) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int kb0 = rg.kb_lo + split * rg.chunk;
  const int kb1 = kb0 + rg.chunk < rg.kb_hi ? kb0 + rg.chunk : rg.kb_hi;
  const int32_t* trow = p.tables + (int64_t)b * p.M;

  // This lane's row (column n of the tiles) and the keys it sees: row_lo <= key <= row_hi.
  const int r = 16 * tile + n, rt = r / p.G;
  const bool real = n < rg.here && rt < rg.cnt;
  const int row_hi = real ? rg.base + rt : -1;
  const int64_t row_first = (int64_t)rg.base + rt - p.window + 1;
  const int row_lo = row_first > 0 ? (int)(row_first < 0x7FFFFFFF ? row_first : 0x7FFFFFFF) : 0;
  pa_bf8 qf[KS];
  {
    const uint16_t* qr = p.q + (int64_t)b * p.qsb + (int64_t)(kvh * p.G + (r - rt * p.G)) * p.qsh + (int64_t)rt * p.qst;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = F8 && KS > 1 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (real) w = *reinterpret_cast<const uint4*>(qr + d);
      qf[s] = __builtin_bit_cast(pa_bf8, w);
    }
  }
  const float c = p.k_scale != nullptr ? p.scale * p.k_scale[kvh] : p.scale;

  uint32_t kf[KT][KW], vf[DT][VW];
  const int psz = 1 << p.shift, pmask = psz - 1;
  const int64_t page_bytes = (int64_t)p.KV * psz * D * (F8 ? 1 : 2);   // of K, and of V
  const int64_t head_bytes = (int64_t)kvh * psz * D * (F8 ? 1 : 2);

  auto load_k = [&](PaPages pg, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      const int off = pa_koff<F8>(i, n);
      const int at = (NK * kb + off) & pmask;
      const uint8_t* base = p.k + (int64_t)pa_page_of<NK>(pg, off >> 4) * page_bytes + head_bytes;
      if constexpr (!F8) {
        const uint8_t* a = base + (uint32_t)(at * (2 * D) + 16 * g);
#pragma unroll
        for (int s = 0; s < KS; ++s) *reinterpret_cast<uint4*>(&kf[i][4 * s]) = *reinterpret_cast<const uint4*>(a + 64 * s);
      } else if constexpr (KS > 1) {
        const uint8_t* a = base + (uint32_t)(at * D + 16 * g);
#pragma unroll
        for (int s = 0; s < KS / 2; ++s) *reinterpret_cast<uint4*>(&kf[i][4 * s]) = *reinterpret_cast<const uint4*>(a + 64 * s);
      } else {
        *reinterpret_cast<uint2*>(&kf[i][0]) = *reinterpret_cast<const uint2*>(base + (uint32_t)(at * D + 8 * g));
      }
    }
  };
  auto load_v = [&](PaPages pg, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < (F8 ? 1 : VS); ++s) {
      const int off = F8 ? 16 * g : 32 * s + 8 * g;
      const int at = (NK * kb + off) & pmask;
      const uint8_t* base = p.v + (int64_t)pa_page_of<NK>(pg, off >> 4) * page_bytes + head_bytes;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<uint4*>(&vf[dt][4 * s]) =
            *reinterpret_cast<const uint4*>(base + (uint32_t)(((16 * dt + n) * psz + at) * (F8 ? 1 : 2)));
    }
  };

  pa_f4 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = pa_f4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;

  int kb = kb0 + wave;
  PaPages pg{};
  if (kb < kb1) {
    pg = pa_pages<NK>(p, trow, kb, rg.lo, rg.hi);
    load_k(pg, kb);
    load_v(pg, kb);
  }
  for (; kb < kb1; kb += kPaWaves) {
    const bool more = kb + kPaWaves < kb1;
    const int bad = pg.bad;
    if (more) pg = pa_pages<NK>(p, trow, kb + kPaWaves, rg.lo, rg.hi);
    // scores, in log2 units
    pa_f4 st[KT];
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      st[i] = pa_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        pa_bf8 a;
        if constexpr (F8) a = pa_widen(kf[i][2 * s], kf[i][2 * s + 1]);
        else a = __builtin_bit_cast(pa_bf8, make_uint4(kf[i][4 * s], kf[i][4 * s + 1], kf[i][4 * s + 2], kf[i][4 * s + 3]));
        st[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[s], st[i], 0, 0, 0);
      }
    }
    if (more) load_k(pg, kb + kPaWaves);
#pragma unroll
    for (int i = 0; i < KT; ++i) st[i] *= c;
    // Every row sees all of its keys, or the block is masked key by key.
    const bool edge = NK * kb < rg.base + rg.t_hi - p.window + 1 || NK * kb + NK - 1 > rg.base + rg.t_lo;
    if (edge || bad != 0) {
#pragma unroll
      for (int i = 0; i < KT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int off = pa_koff<F8>(i, 4 * g + j), key = NK * kb + off;
          float x = st[i][j];
          x = (bad >> (off >> 4)) & 1 ? __builtin_nanf("") : x;      // a seen key on no page: the row becomes NaN
          st[i][j] = key >= row_lo && key <= row_hi ? x : -INFINITY;
        }
    }
    float mx = st[0][0];
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) mx = fmaxf(mx, st[i][j]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mn = fmaxf(m, mx);
    const float ms = mn == -INFINITY ? 0.0f : mn;          // no key yet: every weight below is exp2(-inf) = 0
    if (__builtin_amdgcn_ballot_w64(mn > m) != 0) {
      const float alpha = __builtin_amdgcn_exp2f(m - ms);
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
      m = mn;
    }
    uint4 ph[VS], pl[VS];
#pragma unroll
    for (int s = 0; s < VS; ++s) {
      uint32_t hw[4], lw[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 2 * s + (e >> 1), j = 2 * (e & 1);
        const float a = __builtin_amdgcn_exp2f(st[i][j] - ms), bb = __builtin_amdgcn_exp2f(st[i][j + 1] - ms);
        l += a + bb;
        hw[e] = bf16x2_rne_raw(a, bb);
        lw[e] = bf16x2_rne_raw(a - __uint_as_float(hw[e] << 16), bb - __uint_as_float(hw[e] & 0xFFFF0000u));
      }
      ph[s] = make_uint4(hw[0], hw[1], hw[2], hw[3]);
      pl[s] = make_uint4(lw[0], lw[1], lw[2], lw[3]);
    }
    // V's operand of tile dt, step s.
    auto operand = [&](int dt, int s) __attribute__((always_inline)) -> pa_bf8 {
      if constexpr (F8) return pa_widen(vf[dt][2 * s], vf[dt][2 * s + 1]);
      else return __builtin_bit_cast(pa_bf8, make_uint4(vf[dt][4 * s], vf[dt][4 * s + 1], vf[dt][4 * s + 2], vf[dt][4 * s + 3]));
    };
    auto add = [&](int dt) __attribute__((always_inline)) {
#pragma unroll
      for (int s = 0; s < VS; ++s) {
        const pa_bf8 a = operand(dt, s);
        acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(pa_bf8, ph[s]), acc[dt], 0, 0, 0);
        acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(pa_bf8, pl[s]), acc[dt], 0, 0, 0);
      }
    };
    bool odd = false;
    if (edge) {
      // What the places outside [lo, hi) hold (another sequence's tokens, NaN) may not reach the product: their weight
      // is 0, but 0 x NaN is not. Where rows see different keys, the same holds for a key that one row sees and another
      // does not: a V that is not finite there sends the block the slow way below.
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        uint32_t keep = 0;
#pragma unroll
        for (int j = 0; j < KPW; ++j) {
          const int key = NK * kb + (F8 ? 16 * g + 4 * e + j : 32 * (e >> 2) + 8 * g + 2 * (e & 3) + j);
          keep |= key >= rg.lo && key < rg.hi ? KMASK << (32 / KPW * j) : 0u;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          vf[dt][e] &= keep;
          odd |= pa_not_finite<F8>(vf[dt][e]);
        }
      }
      odd = rg.t_lo != rg.t_hi && __builtin_amdgcn_ballot_w64(odd) != 0;
    }
    if (!odd) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) add(dt);
    } else {
      // Token by token: the V of the keys that token t does not see is zeroed for its product, and only t's columns take
      // the result.
      for (int t = rg.t_lo; t <= rg.t_hi; ++t) {
        const int64_t first = (int64_t)rg.base + t - p.window + 1;
        const int lo = first > rg.lo ? (int)(first < 0x7FFFFFFF ? first : 0x7FFFFFFF) : rg.lo;
        const int hi = rg.base + t + 1 < rg.hi ? rg.base + t + 1 : rg.hi;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const pa_f4 old = acc[dt];
          uint32_t was[VW];
#pragma unroll
          for (int e = 0; e < VW; ++e) {
            uint32_t keep = 0;
#pragma unroll
            for (int j = 0; j < KPW; ++j) {
              const int key = NK * kb + (F8 ? 16 * g + 4 * e + j : 32 * (e >> 2) + 8 * g + 2 * (e & 3) + j);
              keep |= key >= lo && key < hi ? KMASK << (32 / KPW * j) : 0u;
            }
            was[e] = vf[dt][e];
            vf[dt][e] &= keep;
          }
          add(dt);
          if (rt != t) acc[dt] = old;
#pragma unroll
          for (int e = 0; e < VW; ++e) vf[dt][e] = was[e];
        }
      }
    }
    if (more) load_v(pg, kb + kPaWaves);
  }

  // The four waves' parts joined.
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (g == 0) {
    sm[wave][n] = m;
    sl[wave][n] = l;
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
    *reinterpret_cast<float4*>(&so[wave][n][16 * dt + 4 * g]) = make_float4(acc[dt][0], acc[dt][1], acc[dt][2], acc[dt][3]);
  __syncthreads();
  for (int e = threadIdx.x; e < rg.here * (D / 4); e += 64 * kPaWaves) {
    const int row = e / (D / 4), d = 4 * (e - row * (D / 4));
    float mm = sm[0][row];
#pragma unroll
    for (int w = 1; w < kPaWaves; ++w) mm = fmaxf(mm, sm[w][row]);
    const float ms = mm == -INFINITY ? 0.0f : mm;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float ll = 0.0f;
#pragma unroll
    for (int w = 0; w < kPaWaves; ++w) {
      const float a = __builtin_amdgcn_exp2f(sm[w][row] - ms);
      const float4 x = *reinterpret_cast<const float4*>(&so[w][row][d]);
      o.x = fmaf(a, x.x, o.x); o.y = fmaf(a, x.y, o.y); o.z = fmaf(a, x.z, o.z); o.w = fmaf(a, x.w, o.w);
      ll = fmaf(a, sl[w][row], ll);
    }
    if (rg.used <= 1) {
      pa_write(p, rg, b, kvh, 16 * tile + row, d, o, ll, mm);
    } else {
      float* part = p.part + ((((int64_t)b * p.KV + kvh) * p.tiles + tile) * p.splits + split) * (16 * D + 32);
      *reinterpret_cast<float4*>(part + row * D + d) = o;
      if (d == 0) {
        part[16 * D + row] = mm;
        part[16 * D + 16 + row] = ll;
      }
    }
  }
}

// Joins the parts of one row: D / 4 threads across the row, 1024 / D groups of them over the parts.
template <int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttn p) {
  constexpr int C = D / 4, NG = 256 / C;
  __shared__ float4 so[NG][C];
  __shared__ float sl[NG], sm[NG];
  const int b = blockIdx.z, kvh = blockIdx.y;
  const int tile = (int)blockIdx.x >> 4, row = (int)blockIdx.x & 15;
  const PaRange rg(p, b, tile);
  if (rg.used <= 1 || row >= rg.here) return;
  const int col = threadIdx.x % C, grp = threadIdx.x / C;
  const float* part = p.part + (((int64_t)b * p.KV + kvh) * p.tiles + tile) * p.splits * (16 * D + 32);
  float mm = -INFINITY;
  for (int s = grp; s < rg.used; s += NG) mm = fmaxf(mm, part[(int64_t)s * (16 * D + 32) + 16 * D + row]);
  const float ms = mm == -INFINITY ? 0.0f : mm;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float ll = 0.0f;
  for (int s = grp; s < rg.used; s += NG) {
    const float* q = part + (int64_t)s * (16 * D + 32);
    const float a = __builtin_amdgcn_exp2f(q[16 * D + row] - ms);
    const float4 x = *reinterpret_cast<const float4*>(q + row * D + 4 * col);
    o.x = fmaf(a, x.x, o.x); o.y = fmaf(a, x.y, o.y); o.z = fmaf(a, x.z, o.z); o.w = fmaf(a, x.w, o.w);
    ll = fmaf(a, q[16 * D + 16 + row], ll);
  }
  so[grp][col] = o;
  if (col == 0) {
    sl[grp] = ll;
    sm[grp] = mm;
  }
  __syncthreads();
  if (grp != 0) return;
  float m = sm[0];
#pragma unroll
  for (int i = 1; i < NG; ++i) m = fmaxf(m, sm[i]);
  const float mz = m == -INFINITY ? 0.0f : m;
  o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  ll = 0.0f;
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const float a = __builtin_amdgcn_exp2f(sm[i] - mz);
    const float4 x = so[i][col];
    o.x = fmaf(a, x.x, o.x); o.y = fmaf(a, x.y, o.y); o.z = fmaf(a, x.z, o.z); o.w = fmaf(a, x.w, o.w);
    ll = fmaf(a, sl[i], ll);
  }
  pa_write(p, rg, b, kvh, 16 * tile + row, 4 * col, o, ll, m);
}

// Parts a key range may be cut into: four workgroups a compute unit over all rows, at least one block of keys a
// wave in each part, for the longest range that the table and the window allow.
static int64_t pa_splits(int64_t B, int64_t KV, int64_t tiles, int64_t page, int64_t M, int64_t T, int64_t window) {
  int64_t keys = M * page;               // blocks of 64 keys, the larger of the two: fewer parts
  if (window < keys) keys = window + T - 1 < keys ? window + T - 1 : keys;
  const int64_t most = (keys / 64 + 2 + kPaWaves - 1) / kPaWaves;
  const int64_t base = B * KV * tiles, want = (4ll * compute_units() + base - 1) / base;
  int64_t s = want < most ? want : most;
  return s < 1 ? 1 : s > 4096 ? 4096 : s;
}

}  // namespace flw

using namespace flw;

static int64_t pa_tiles(int64_t H, int64_t KV, int64_t T) { return (T * (H / KV) + 15) / 16; }

extern "C" size_t flw_paged_attention_workspace_bytes(int64_t B, int64_t H, int64_t KV, int64_t T, int64_t D,
                                                      int64_t page_size, int64_t table_cols, int64_t window) {
  if (B <= 0 || H <= 0 || KV <= 0 || H % KV != 0 || T <= 0 || D <= 0 || page_size <= 0 || table_cols <= 0 || window <= 0)
    return 0;
  const int64_t tiles = pa_tiles(H, KV, T), s = pa_splits(B, KV, tiles, page_size, table_cols, T, window);
  return s == 1 ? 0 : (size_t)(B * KV * tiles * s * (16 * D + 32) * 4);
}

extern "C" int flw_paged_attention(const void* q, const int64_t* q_strides, const void* k_pages, const void* v_pages,
                                   int cache_dtype, int64_t num_pages, int64_t page_size, const int32_t* tables,
                                   int64_t table_cols, const int32_t* lens, const int32_t* counts, const float* k_scale,
                                   const float* v_scale, int64_t B, int64_t H, int64_t KV, int64_t T, int64_t D,
                                   int64_t window, float scale, void* out, const int64_t* out_strides, float* lse,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  FLW_REQUIRE(q && q_strides && k_pages && v_pages && tables && lens && out && out_strides, FLW_E_INVALID, "null pointer");
  FLW_REQUIRE(B > 0 && H > 0 && KV > 0 && T > 0 && num_pages > 0 && table_cols > 0, FLW_E_INVALID, "empty shape");
  FLW_REQUIRE(D == 32 || D == 64 || D == 128, FLW_E_UNSUPPORTED, "head_dim must be 32/64/128, got %lld", (long long)D);
  FLW_REQUIRE(H % KV == 0, FLW_E_INVALID, "%lld query heads do not share %lld kv heads evenly", (long long)H, (long long)KV);
  FLW_REQUIRE(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0, FLW_E_UNSUPPORTED,
              "page size must be a power of two from 16 to 1024, got %lld", (long long)page_size);
  FLW_REQUIRE(cache_dtype == FLW_BF16 || cache_dtype == FLW_E4M3, FLW_E_INVALID, "the cache holds bf16 or e4m3");
  FLW_REQUIRE((cache_dtype == FLW_E4M3) == (k_scale != nullptr) && (k_scale != nullptr) == (v_scale != nullptr),
              FLW_E_INVALID, "an e4m3 cache takes k and v scales, a bf16 one none");
  FLW_REQUIRE(B <= 65535 && KV <= 65535 && H <= 65536 && T <= 65536 && num_pages <= 0x7FFFFFFFll &&
              table_cols * page_size <= 0x7FFFFFFFll - 64, FLW_E_UNSUPPORTED, "shape too large");
  FLW_REQUIRE((((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)out) & 15) == 0, FLW_E_INVALID,
              "q, pages and out must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    FLW_REQUIRE(q_strides[i] % 8 == 0 && out_strides[i] % 4 == 0, FLW_E_INVALID, "rows must be 16-byte aligned (out: 8)");
  const int64_t tiles = pa_tiles(H, KV, T);
  const int64_t w = window < 0 ? 0 : window > 0x7FFFFFFFll ? 0x7FFFFFFFll : window;
  const int64_t splits = w > 0 ? pa_splits(B, KV, tiles, page_size, table_cols, T, w) : 1;
  FLW_REQUIRE(tiles * (splits > 16 ? splits : 16) <= 0x7FFFFFFFll, FLW_E_UNSUPPORTED, "shape too large");
  const size_t need = splits == 1 ? 0 : (size_t)(B * KV * tiles * splits * (16 * D + 32) * 4);
  FLW_REQUIRE(need == 0 || (workspace != nullptr && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need),
              FLW_E_WORKSPACE, "workspace needs %zu bytes (16-byte aligned)", need);
  PagedAttn p{};
  p.q = static_cast<const uint16_t*>(q);
  p.qsb = q_strides[0]; p.qsh = q_strides[1]; p.qst = q_strides[2];
  p.k = static_cast<const uint8_t*>(k_pages); p.v = static_cast<const uint8_t*>(v_pages);
  p.tables = tables; p.lens = lens; p.counts = counts; p.k_scale = k_scale; p.v_scale = v_scale;
  p.out = static_cast<uint16_t*>(out);
  p.osb = out_strides[0]; p.osh = out_strides[1]; p.ost = out_strides[2];
  p.lse = lse; p.part = static_cast<float*>(workspace);
  p.P = num_pages; p.B = (int)B; p.H = (int)H; p.KV = (int)KV; p.G = (int)(H / KV); p.T = (int)T;
  p.rows = (int)(T * (H / KV)); p.tiles = (int)tiles; p.M = (int)table_cols; p.shift = __builtin_ctzll(page_size);
  p.bshift = D == 128 && cache_dtype == FLW_BF16 ? 5 : 6;
  p.window = (int)w; p.splits = (int)splits; p.scale = scale * 1.44269504088896341f;
  const bool f8 = cache_dtype == FLW_E4M3;
  const void* kern =
      D == 32 ? (f8 ? (const void*)&paged_attn_kernel<32, true> : (const void*)&paged_attn_kernel<32, false>)
    : D == 64 ? (f8 ? (const void*)&paged_attn_kernel<64, true> : (const void*)&paged_attn_kernel<64, false>)
              : (f8 ? (const void*)&paged_attn_kernel<128, true> : (const void*)&paged_attn_kernel<128, false>);
  const void* join = D == 32 ? (const void*)&paged_join_kernel<32>
                   : D == 64 ? (const void*)&paged_join_kernel<64> : (const void*)&paged_join_kernel<128>;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Timer tm = take_timer();
  (void)launch_ext(kern, dim3((unsigned)(tiles * splits), (unsigned)KV, (unsigned)B), dim3(64 * kPaWaves), 0, s, p,
                   tm.start, splits == 1 ? tm.stop : nullptr);
  if (splits > 1)
    (void)launch_ext(join, dim3((unsigned)(16 * tiles), (unsigned)KV, (unsigned)B), dim3(256), 0, s, p, nullptr, tm.stop);
  return check_launch("flw_paged_attention");
}
