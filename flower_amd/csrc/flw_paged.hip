// Attention of the newest tokens of each sequence over a paged key-value cache (the decode step).
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(q_i . k_j * scale - m_i),
//   over the keys j of i's sequence with max(0, i - window + 1) <= j <= i.
//
// Each K and V byte in the window is read once, from its page, and nothing else is of that size: the bound is HBM. A K / V head
// is shared by G query heads and by the T new tokens: their T G rows are the columns of MFMA tiles, 16 a wave.
//
// A workgroup of one to four waves (by its rows) takes blocks of 64 keys on its own. K and V of a block go from the pool
// straight to LDS (whole 128-byte lines, non-temporal: a plain reader gets 6.2 TB/s on this card and a non-temporal one 6.9, but
// half lines, which operands loaded to registers would be, lose by it), the next block's on their way while this one's are
// multiplied. A single wave needs no barrier, only its own count of loads; several meet once a block.
//   S^T (keys x rows) = K Q^T on v_mfma_f32_16x16x32_bf16: a lane holds 16 scores of ONE row, so the running maximum and
//     sum are per lane, joined over the four lane groups by two lane exchanges a block;
//   O^T (D x rows) += V^T P^T: a lane's scores are the operand P^T as they stand, because the K rows are taken in the
//     order that puts a lane's scores next to each other along the keys; V^T is read as it is, since a page holds V as
//     (D, page size).
// P goes to the product as two bf16 terms (p rounded, and what that lost), so that it carries 16 bits instead of 8: the
// matrix cores idle here, and one term would cost as much accuracy as the output's own rounding. Scores, the maximum, the
// sum and O are fp32.
// e4m3 pages: codes widened to bf16 in registers (exact); the K scale multiplies the score, the V scale the output.
//
// Work: an item is a (sequence, row group, kv head), its length the blocks of its key range. Either a workgroup an item (of one
// row tile: a wave, or four that take a quarter of its blocks each and join in LDS), or the blocks of all items laid end to end
// and cut into equal parts, one for each workgroup that the GPU holds; an item cut by a border leaves fp32 partial results, which
// a second launch joins. A workgroup begins an item's loads while it ends the one before.
//
// Measured: 64 sequences of up to 2048 keys, 20 heads of 64: 99 us, 6.1 TB/s of K and V. 4 sequences of 70 001 to 131 072 keys, 32
// heads on 4 of 128: 133 us with the join, 6.2 TB/s. Short calls are latency: 100 keys of 16 heads take 5.8 us, most of it the
// first fetch of the code and of the page numbers, the lengths and the keys that depend on each other.
//
// Keys and values that are not finite reach only the rows that see them; an infinite V may come out as NaN there, since the second
// term of its weight is often zero or of the other sign.

#include <utility>

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
  float* part;                    // balanced: two slots a wave of group_rows x (D + 2) floats
  int4* open;                     // balanced, an item: {the wave that began it, or -1 if that ended it, too; slot; last wave}
  int64_t P;
  int B, H, KV, G, T, rows, groups, M, shift, window, balanced;
  uint32_t by_g, by_groups, by_kv;   // x / G = x by_g >> 32 (0: the divisor is 1); groups and KV alike
  float scale;                    // softmax scale x log2 e
};

constexpr float kPaLn2 = 0.69314718055994531f;
constexpr int kPaKeys = 64;       // keys a block

// x / n by n's reciprocal rounded up (exact while x n < 2^32, which the host checks): a division is 30 instructions else, and
// what a short call costs is the code that it has to fetch.
__device__ __forceinline__ int pa_div(int x, uint32_t by) { return by == 0 ? x : (int)__umulhi((uint32_t)x, by); }

// The keys of one row group: rows r0 .. r0 + here (tokens t_lo .. t_hi), keys [lo, hi), blocks [kb_lo, kb_hi).
struct PaRange {
  int base, cnt, here, t_lo, t_hi, lo, hi, kb_lo, kb_hi;
  __device__ __forceinline__ PaRange(const PagedAttn& p, int b, int group, int group_rows) {
    cnt = p.counts != nullptr ? p.counts[b] : p.T;
    cnt = cnt < 0 ? 0 : cnt;
    const int len = p.lens[b];
    base = (len < 0 ? 0 : len) - cnt;                     // the first new token's position
    const int r0 = group_rows * group;
    here = p.rows - r0 < group_rows ? p.rows - r0 : group_rows;
    t_lo = pa_div(r0, p.by_g);
    t_hi = pa_div(r0 + here - 1, p.by_g);
    t_hi = t_hi < cnt ? t_hi : cnt - 1;
    lo = hi = 0;
    if (t_lo <= t_hi && p.window > 0) {
      const int64_t first = (int64_t)base + t_lo - p.window + 1, cap = (int64_t)p.M << p.shift;
      const int64_t last = (int64_t)base + t_hi + 1;      // positions past the table are answered with NaN: never read
      hi = (int)(last < cap ? last : cap);
      lo = (int)(first > 0 ? (first < cap ? first : cap) : 0);
    }
    kb_lo = lo / kPaKeys;
    kb_hi = hi > lo ? (hi + kPaKeys - 1) / kPaKeys : kb_lo;
  }
  __device__ __forceinline__ int blocks() const { return kb_hi > kb_lo ? kb_hi - kb_lo : 1; }   // an empty item counts one
};

// Output row r of (b, kvh), from its unnormalised O, sum l and maximum m. A row without keys is zero, one past its table NaN.
struct PaRow {
  uint16_t* out;
  int64_t lse;
  float inv;
  bool real, past;
  __device__ __forceinline__ PaRow(const PagedAttn& p, const PaRange& rg, int b, int kvh, int r, float l) {
    const int t = pa_div(r, p.by_g), h = kvh * p.G + (r - t * p.G);
    real = t < rg.cnt && rg.base + t >= 0 && p.window > 0;
    past = real && (int64_t)rg.base + t >= ((int64_t)p.M << p.shift);
    inv = past ? __builtin_nanf("") : (p.v_scale != nullptr ? p.v_scale[kvh] : 1.0f) / l;
    out = p.out + (int64_t)b * p.osb + (int64_t)h * p.osh + (int64_t)t * p.ost;
    lse = ((int64_t)b * p.H + h) * p.T + t;
  }
  __device__ __forceinline__ void write(int d, float x, float y, float z, float w) const {       // four values from d on
    const uint2 v = make_uint2(bf16x2_rne(x * inv, y * inv), bf16x2_rne(z * inv, w * inv));
    *reinterpret_cast<uint2*>(out + d) = make_uint2(real ? v.x : 0u, real ? v.y : 0u);
  }
  __device__ __forceinline__ void write_lse(const PagedAttn& p, float m, float l) const {
    if (p.lse != nullptr) p.lse[lse] = !real ? -INFINITY : past ? __builtin_nanf("") : (m + __builtin_amdgcn_logf(l)) * kPaLn2;
  }
};

// Eight e4m3 codes widened to bf16 (exact).
__device__ __forceinline__ uint4 pa_widen(uint32_t lo, uint32_t hi) {
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, true)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, true)));
}

// Workgroups that a compute unit holds, by the registers (at most 128 to 180 a lane) and by LDS (32 KB rings: four). One too many
// makes two rounds of the line: a fifth 32 KB ring, which was to fit the 160 KB and did not, 168 us instead of 148; a fourth
// workgroup of three waves of e4m3, D = 128, 152 instead of 133.
constexpr int pa_held(int D, bool f8, int waves) {
  return waves == 1 ? (D == 128 && !f8 ? 4 : 8) : D == 128 && !f8 ? 2 : waves == 4 || (waves == 3 && D == 128) ? 3 : 4;
}

// The geometry of a block of 64 keys, K and V alike 64 D values: how its 16-byte chunks lie in LDS, and which lane of which
// 1 KB load brings them. A load takes 64 chunks to consecutive places; a chunk's place within its row is its number xor a
// function of the row (kswz, vswz), so that the 16 lanes that read one operand together meet 16 different bank groups.
//
// K rows are taken in the order koff(i, m) (tile i's row m): the scores of tile i are then keys koff(i, 4 g + j), j = 0 .. 3,
// of lane group g, and the 8 keys of a lane in V's step s are tiles 2 s and 2 s + 1: consecutive, one 16-byte chunk of V
// (bf16: 8 keys; e4m3: both steps' 16).
//
// V: rows of 64 keys (WIDE: a page holds at least 64), or, for pages of 16 and 32, the block's four runs of 16 keys one after
// the other, so that one load stays within one page.
template <int D_, bool F8_, bool WIDE_, int WAVES>
struct PaBlock {
  static constexpr int D = D_;
  static constexpr bool F8 = F8_, WIDE = WIDE_;
  static constexpr int ES = F8 ? 1 : 2;                   // bytes a value
  static constexpr int KS = D / 32, DT = D / 16;          // MFMA steps over D of a score, tiles of 16 dims of O
  static constexpr int TILE = kPaKeys * D * ES;           // bytes of K, and of V
  static constexpr int NI = TILE / 1024;                  // loads of each
  // Blocks in LDS. One wave: what keeps 12 KB and more on their way (a second buffer at 8 KB a tile gained nothing).
  static constexpr int BUFS = WAVES > 1 || TILE <= 4096 ? 2 : 1;
  static constexpr int RING = 2 * BUFS * TILE;
  static constexpr int RB = D * ES, KC = RB / 16, KR = 64 / KC;       // a K row's bytes and chunks, rows a load
  static constexpr int VC = WIDE ? kPaKeys * ES / 16 : 16 * ES / 16;   // chunks of a V row (WIDE) or of a row's run
  static constexpr int VR = 64 / VC;                      // V rows a load
  static __device__ __forceinline__ int koff(int i, int m) {
    return F8 ? 16 * (m >> 2) + 4 * i + (m & 3) : 32 * (i >> 1) + 8 * (m >> 2) + 4 * (i & 1) + (m & 3);
  }
  // Bits of the row only (so that kswz(a ^ b) = kswz(a) ^ kswz(b)): those in which the rows read together differ.
  static __device__ __forceinline__ int kswz(int key) {
    const int hi = (key >> (F8 ? 4 : 3)) & 3;
    return KC == 16 ? (key & 3) | hi << 2 : KC == 8 ? ((key >> 1) & 1) | hi << 1 : KC == 4 ? hi : hi & 1;
  }
  static __device__ __forceinline__ int vswz(int d) {
    return VC == 8 ? (d >> 1) & 7 : VC == 4 ? (d >> 2) & 3 : VC == 2 ? (d >> 3) & 1 : 0;
  }
};

// 64 lanes' 16 bytes from sbase + voff to LDS at lds + OFF, in lane order, non-temporal (5 to 15 % faster where keys are read once,
// 7 % slower where eight row groups read them). Issued from inline assembly: the
// compiler then does not drain the loads before every read of LDS; the kernel waits for them itself, by count. A load to LDS that
// follows the write of M0 at once may go by M0's old value: one wait state, which the compiler does not put inside the statement.
template <int OFF>
__device__ __forceinline__ void pa_dma(uint32_t lds, uint32_t voff, const uint8_t* sbase) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds), "v"(voff), "s"(sbase), "n"(OFF)
                 : "memory", "m0", "scc");
}
template <int OFF>
__device__ __forceinline__ void pa_dma_lanes(uint32_t lds, const uint8_t* a) {       // each lane its own address
  asm volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(a), "n"(OFF)
                 : "memory", "m0", "scc");
}
// The results of a run of MFMAs, safe to read from here on whichever way the code goes. In a form of this kernel with branches
// inside its runs, results were seen stale, and the compiler's code was: two MFMAs into v[82:85]; s_cbranch_vccnz L; two MFMAs into
// other registers and their readers; L: v_cndmask of v85. The taken way had no wait states before that reader, where eight are
// due; along the other they had passed. A branch that passes over no MFMAs got its wait states on both ways. So no branch stands
// inside a run here, and its results are held back in one place before any that follows.
template <int N>
__device__ __forceinline__ void pa_settle(pa_f4 (&x)[N]) {
  static_assert(N == 2 || N == 4 || N == 8);
  if constexpr (N == 2) asm volatile("s_nop 15" : "+v"(x[0]), "+v"(x[1]));
  if constexpr (N == 4) asm volatile("s_nop 15" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
  if constexpr (N == 8)
    asm volatile("s_nop 15" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7]));
}
template <int N>
__device__ __forceinline__ void pa_wait() {               // until at most N loads are on their way
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Pages of a block's four runs of 16 keys (a page holds at least 16): page numbers, 0 for a run outside the range and for one
// whose entry is no page; `bad` has the latter's bits.
struct PaPages {
  int id0, id1, id2, id3, bad;
};
template <bool WIDE>
__device__ __forceinline__ PaPages pa_pages(const PagedAttn& p, const int32_t* row, int kb, int lo, int hi) {
  // scalar loads: the address is the wave's
  const __attribute__((address_space(4))) int32_t* crow = (const __attribute__((address_space(4))) int32_t*)row;
  int id[4], bad = 0;
#pragma unroll
  for (int c = 0; c < (WIDE ? 1 : 4); ++c) {
    const int pos = kPaKeys * kb + 16 * c;
    const bool in = pos < hi && pos + (WIDE ? kPaKeys : 16) > lo;
    const int e = in ? crow[pos >> p.shift] : 0;          // hi is at most the table's positions: the entry exists
    const bool ok = (uint32_t)e < (uint32_t)p.P;
    bad |= ok ? 0 : WIDE ? 15 : 1 << c;
    id[c] = ok ? e : 0;
  }
  if constexpr (WIDE) return PaPages{id[0], id[0], id[0], id[0], bad};
  else return PaPages{id[0], id[1], id[2], id[3], bad};
}

template <int D, bool F8, bool WIDE, int WAVES>
struct PaWave {
  using Blk = PaBlock<D, F8, WIDE, WAVES>;
  const PagedAttn& p;
  uint8_t* ring;                                          // this wave's LDS
  int lane, wave, n, g;
  uint32_t kvoff, vvoff;                                  // this lane's offset in a load of K, of V (swizzle: xor 16 x)
  int64_t page_bytes;

  __device__ __forceinline__ PaWave(const PagedAttn& p_, uint8_t* ring_) : p(p_), ring(ring_) {
    lane = threadIdx.x & 63;
    wave = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    n = lane & 15;
    g = lane >> 4;
    const int psz = 1 << p.shift;
    page_bytes = (int64_t)p.KV * psz * Blk::RB;
    const int kr = lane / Blk::KC, kc = lane % Blk::KC, vr = lane / Blk::VC, vc = lane % Blk::VC;
    kvoff = kr * Blk::RB + 16 * (kc ^ Blk::kswz(kr));
    vvoff = vr * psz * Blk::ES + 16 * (vc ^ Blk::vswz(vr));
  }
  __device__ __forceinline__ uint32_t lds(int off) const { return (uint32_t)(uintptr_t)(lds_u8_t*)(ring + off); }

  // K (V) of block kb, `head` bytes into its pages, to LDS at `to`: this wave's share of the loads.
  template <int J>
  __device__ __forceinline__ bool mine() const {          // load J of a tile is this wave's
    return WAVES == 1 || wave == J / ((Blk::NI + WAVES - 1) / WAVES);
  }
  static __device__ __forceinline__ int page_of(PaPages pg, int c) {
    return c == 0 ? pg.id0 : c == 1 ? pg.id1 : c == 2 ? pg.id2 : pg.id3;
  }
  template <int J>
  __device__ __forceinline__ void load_k1(PaPages pg, int kb, int64_t head, uint32_t to) const {
    const int pmask = (1 << p.shift) - 1;
    constexpr int row = J * Blk::KR, c = row >> 4;
    if constexpr (WIDE) {
      pa_dma<1024 * J>(to, (kvoff ^ (16u * Blk::kswz(row))) + row * Blk::RB,
                            p.k + pg.id0 * page_bytes + head + ((kPaKeys * kb) & pmask) * Blk::RB);
    } else if constexpr (Blk::KR <= 16) {
      pa_dma<1024 * J>(to, (kvoff ^ (16u * Blk::kswz(row))) + (row & 15) * Blk::RB,
                            p.k + page_of(pg, c) * page_bytes + head + ((kPaKeys * kb + 16 * c) & pmask) * Blk::RB);
    } else {                                              // 32 rows a load (e4m3, D = 32): two runs, perhaps two pages
      const int kr = lane / Blk::KC, at = (kPaKeys * kb + row + kr) & pmask;
      pa_dma_lanes<1024 * J>(to, p.k + (kr < 16 ? page_of(pg, c) : page_of(pg, c + 1)) * page_bytes + head + at * Blk::RB +
                                     16 * ((lane % Blk::KC) ^ Blk::kswz(row + kr)));
    }
  }
  template <int J>
  __device__ __forceinline__ void load_v1(PaPages pg, int kb, int64_t head, uint32_t to) const {
    const int psz = 1 << p.shift, pmask = psz - 1;
    if constexpr (WIDE) {
      constexpr int d = J * Blk::VR;
      pa_dma<1024 * J>(to, (vvoff ^ (16u * Blk::vswz(d))) + (uint32_t)(d * psz) * Blk::ES,
                            p.v + pg.id0 * page_bytes + head + ((kPaKeys * kb) & pmask) * Blk::ES);
    } else if constexpr (Blk::VR <= D) {
      constexpr int PER = D / Blk::VR, c = J / PER, d = (J % PER) * Blk::VR;      // loads a run
      pa_dma<1024 * J>(to, (vvoff ^ (16u * Blk::vswz(d))) + (uint32_t)(d * psz) * Blk::ES,
                            p.v + page_of(pg, c) * page_bytes + head + ((kPaKeys * kb + 16 * c) & pmask) * Blk::ES);
    } else {                                              // 64 rows a load (e4m3, D = 32): two runs, perhaps two pages
      const int c = 2 * J + (lane >> 5), d = lane & 31, id = lane < 32 ? page_of(pg, 2 * J) : page_of(pg, 2 * J + 1);
      pa_dma_lanes<1024 * J>(to, p.v + id * page_bytes + head + d * psz + ((kPaKeys * kb + 16 * c) & pmask));
    }
  }
  template <int... J>
  __device__ __forceinline__ void load_ks(std::integer_sequence<int, J...>, PaPages pg, int kb, int64_t head, uint32_t to) const {
    ((mine<J>() ? load_k1<J>(pg, kb, head, to) : void()), ...);
  }
  template <int... J>
  __device__ __forceinline__ void load_vs(std::integer_sequence<int, J...>, PaPages pg, int kb, int64_t head, uint32_t to) const {
    ((mine<J>() ? load_v1<J>(pg, kb, head, to) : void()), ...);
  }
  __device__ __forceinline__ void load_k(PaPages pg, int kb, int64_t head, int to) const {
    load_ks(std::make_integer_sequence<int, Blk::NI>{}, pg, kb, head, lds(to));
  }
  __device__ __forceinline__ void load_v(PaPages pg, int kb, int64_t head, int to) const {
    load_vs(std::make_integer_sequence<int, Blk::NI>{}, pg, kb, head, lds(to));
  }
  // K's operand of tile i, step s.
  __device__ __forceinline__ uint4 k_words(int from, int i, int s) const {      // 16 bytes: bf16 one step, e4m3 steps s, s + 1
    const int key = Blk::koff(i, n), chunk = F8 ? 4 * (s >> 1) + g : 4 * s + g;
    return *reinterpret_cast<const uint4*>(ring + from + key * Blk::RB + 16 * (chunk ^ Blk::kswz(key)));
  }
  __device__ __forceinline__ pa_bf8 k_operand(int from, int i, int s) const {
    if constexpr (!F8) {
      return __builtin_bit_cast(pa_bf8, k_words(from, i, s));
    } else if constexpr (D == 32) {
      const int key = Blk::koff(i, n);
      const uint2 w = *reinterpret_cast<const uint2*>(ring + from + key * 32 + 16 * ((g >> 1) ^ Blk::kswz(key)) + 8 * (g & 1));
      return __builtin_bit_cast(pa_bf8, pa_widen(w.x, w.y));
    } else {
      const uint4 w = k_words(from, i, s);
      return __builtin_bit_cast(pa_bf8, s & 1 ? pa_widen(w.z, w.w) : pa_widen(w.x, w.y));
    }
  }
  // The 16 bytes of V of dims' tile dt that step s reads (e4m3: both steps').
  __device__ __forceinline__ uint4 v_words(int from, int dt, int s) const {
    const int d = 16 * dt + n;
    if constexpr (WIDE) {
      const int chunk = F8 ? g : 4 * s + g;
      return *reinterpret_cast<const uint4*>(ring + from + 16 * (d * Blk::VC + (chunk ^ Blk::vswz(d))));
    } else {
      const int c = F8 ? g : 2 * s + (g >> 1), chunk = F8 ? 0 : g & 1;
      return *reinterpret_cast<const uint4*>(ring + from + 16 * ((c * D + d) * Blk::VC + (chunk ^ Blk::vswz(d))));
    }
  }
};

// The bits of the keys [lo, hi) in the 16 bytes of V that begin at key `key`: 8 bf16 or 16 e4m3 values.
template <bool F8>
__device__ __forceinline__ uint4 pa_keep(int key, int lo, int hi) {
  constexpr int N = F8 ? 16 : 8;
  const int a = lo - key < 0 ? 0 : lo - key > N ? N : lo - key, b = hi - key < 0 ? 0 : hi - key > N ? N : hi - key;
  const int bits = ((1 << b) - 1) & ~((1 << a) - 1);
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[e] = 0;
#pragma unroll
    for (int j = 0; j < N / 4; ++j)
      w[e] |= (uint32_t)((bits << (31 - (N / 4 * e + j))) >> 31) & (F8 ? 0xFFu << (8 * j) : 0xFFFFu << (16 * j));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pa_and(uint4 a, uint4 b) { return make_uint4(a.x & b.x, a.y & b.y, a.z & b.z, a.w & b.w); }
// Whether 16 bytes of V hold a NaN or an infinity.
template <bool F8>
__device__ __forceinline__ bool pa_not_finite(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t bad = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {       // the top bit of each value: e4m3 0x7F, bf16 an exponent of ones
    if constexpr (F8) bad |= ((w[e] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
    else bad |= ((w[e] & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
  }
  return bad != 0;
}

// One part of an item, blocks [kb, kb + blocks) of (b, row group, kvh), as its loads need it.
struct PaPart {
  const int32_t* trow;
  int64_t head;
  int lo, hi, kb, blocks;
};

// SPLIT > 1: that many waves a workgroup, each on its own as with WAVES = 1, share the blocks of one item and join in LDS.
template <int D, bool F8, bool WIDE, int WAVES, int SPLIT = 1>
__global__ __launch_bounds__(64 * WAVES * SPLIT, WAVES >= 3 ? (D == 128 && !F8 ? 2 : 3) : 2) void paged_attn_kernel(PagedAttn p) {
  using Blk = PaBlock<D, F8, WIDE, WAVES>;
  constexpr int DT = Blk::DT, KS = Blk::KS, NI = Blk::NI, TILE = Blk::TILE, ROWS = 16 * WAVES;
  constexpr int BUFS = Blk::BUFS, AHEAD = WAVES > 1 ? 1 : BUFS;
  static_assert(WAVES == 1 || SPLIT == 1);
  __shared__ __align__(1024) uint8_t rings[SPLIT * Blk::RING];
  const int sw = SPLIT == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  uint8_t* ring = rings + sw * Blk::RING;
  const PaWave<D, F8, WIDE, WAVES> wv(p, ring);
  const int n = wv.n, g = wv.g;
  const int me = (int)blockIdx.x, pairs = p.B * p.groups;
  auto range = [&](int pair) __attribute__((always_inline)) {
    const int b = pa_div(pair, p.by_groups);
    return PaRange(p, b, pair - b * p.groups, ROWS);
  };
  // The item at hand (pair: sequence and row group), its place [s, s + its blocks) on the line, and the block to go on at; the
  // line's length, a part's, and this wave's end.
  int pair, kvh, s = 0, cur = 0, total = 0, per = 0, to = 0;
  if (!p.balanced) {                                      // an item a wave: a line of its own
    pair = pa_div(me, p.by_kv);
    kvh = me - pair * p.KV;
    to = total = per = range(pair).blocks();
    if constexpr (SPLIT > 1) {
      cur = to * sw / SPLIT;
      to = to * (sw + 1) / SPLIT;
    }
  } else {
    int upto = 0, mine = 0, from = 0;
    pair = 0;
    for (int pass = 0; pass < 2; ++pass) {                // the line's length; the pair that holds `from`
      int before = 0;
#pragma unroll 1
      for (int c0 = 0; c0 < pairs; c0 += 64) {
        if (pass == 0 || pairs > 64) {
          const int i = c0 + wv.lane;
          mine = i < pairs ? range(i).blocks() * p.KV : 0;
          upto = mine;
#pragma unroll
          for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(upto, o, 64);
            if (wv.lane >= o) upto += y;
          }
          upto += before;
          before = __builtin_amdgcn_readlane(upto, 63);
        }
        if (pass == 1) {
          const uint64_t in = __builtin_amdgcn_ballot_w64(mine > 0 && upto - mine <= from && from < upto);
          if (in != 0) {
            const int at = __builtin_ctzll(in);
            pair = c0 + at;
            s = __builtin_amdgcn_readlane(upto - mine, at);
            break;
          }
        }
      }
      if (pass == 0) {
        total = before;
        per = (int)(((uint32_t)total + gridDim.x - 1) / gridDim.x);
        per = per < 1 ? 1 : per;
        if (me >= (int)(((uint32_t)total + per - 1) / (uint32_t)per)) return;
        from = me * per;
        to = total - from < per ? total : from + per;
      }
    }
    const int len = range(pair).blocks();
    kvh = (int)((uint32_t)(from - s) / (uint32_t)len);
    s += kvh * len;
    cur = from;
  }

  // The part at (pair, kvh, s, cur), which ends with its item or with this wave's line; none: blocks < 0.
  auto part_of = [&](const PaRange& rg) __attribute__((always_inline)) {
    const int e = s + rg.blocks(), end = e < to ? e : to;
    return PaPart{p.tables + (int64_t)pa_div(pair, p.by_groups) * p.M, (int64_t)kvh * (Blk::RB << p.shift), rg.lo, rg.hi,
                  rg.kb_lo + (cur - s), SPLIT == 1 && s >= to ? -1 : rg.kb_hi > rg.kb_lo ? end - cur : 0};
  };
  PaRange rg = range(pair);
  PaPart at = part_of(rg);
  int slot = 0, bad0 = 0, bad1 = 0;                       // the ring's buffer of the next block; the missing pages of the two
  int held = 0;                                           // blocks from the next one on that are loaded or on their way
#pragma unroll 1
  for (int nth = 0; at.blocks >= 0; ++nth) {
    const int b = pa_div(pair, p.by_groups), group = pair - b * p.groups, kv = kvh, item = pair * p.KV + kvh;
    const int from_s = s, e = s + rg.blocks();
    const bool begins = cur == s, ends = SPLIT > 1 || at.blocks == 0 || cur + at.blocks == e;
    // the part after this one
    PaRange nrg = rg;
    PaPart nx = at;
    nx.blocks = -1;
    if (ends) {
      s = cur = e;
      if (++kvh == p.KV) {
        kvh = 0;
        ++pair;
      }
      if (s < to) {
        nrg = range(pair);
        nx = part_of(nrg);
      }
    }
    // The pages of block i counted from this part's first; behind its last the next part's follow.
    auto pages = [&](int i) __attribute__((always_inline)) {
      const bool here = i < at.blocks;
      const int j = here ? i : i - at.blocks, kb = (here ? at.kb : nx.kb) + j;
      if (!here && j >= nx.blocks) return PaPages{};
      return pa_pages<WIDE>(p, here ? at.trow : nx.trow, kb, here ? at.lo : nx.lo, here ? at.hi : nx.hi);
    };
    // This lane's row (column n of the wave's tile) and the keys it sees: row_lo <= key <= row_hi.
    const int r = 16 * wv.wave + n, rt = pa_div(ROWS * group + r, p.by_g);
    const bool real = r < rg.here && rt < rg.cnt;
    const int row_hi = real ? rg.base + rt : -1;
    const int64_t row_first = (int64_t)rg.base + rt - p.window + 1;
    const int row_lo = row_first > 0 && real ? (int)row_first : 0;
    pa_bf8 qf[KS];
    {
      const int64_t h = kv * p.G + (ROWS * group + r - rt * p.G);
      const uint16_t* qr = p.q + (int64_t)b * p.qsb + h * p.qsh + (int64_t)rt * p.qst;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int d = F8 && KS > 1 ? 64 * (k >> 1) + 16 * g + 8 * (k & 1) : 32 * k + 8 * g;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (real) w = *reinterpret_cast<const uint4*>(qr + d);
        qf[k] = __builtin_bit_cast(pa_bf8, w);
      }
    }
    // its first blocks, as far as the part before has not begun them
#pragma unroll 1
    while (held < AHEAD && held < at.blocks) {
      const int u = BUFS == 2 ? (slot + held) & 1 : 0;
      const PaPages pg = pages(held);
      wv.load_k(pg, at.kb + held, at.head, u * TILE);
      wv.load_v(pg, at.kb + held, at.head, (BUFS + u) * TILE);
      if (u == 0) bad0 = pg.bad;
      else bad1 = pg.bad;
      ++held;
    }
    PaPages pg = pages(held);                             // of the block to begin next

    pa_f4 acc[DT];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = pa_f4{0.0f, 0.0f, 0.0f, 0.0f};
    float c = p.scale;
    if (p.k_scale != nullptr) c *= p.k_scale[kv];
    if (c <= 0.0f) {
      // A negative scale goes to q, so that larger scores weigh more. A scale of zero does, too: a masked score is -infinity, and
      // zero times that is no weight. Zero times q is NaN where q is not finite, as times a key, which the product sees to.
      const bool zero = c == 0.0f;
      c = zero ? 1.0f : -c;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const uint4 w = __builtin_bit_cast(uint4, qf[k]);
        uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t lo = (x[e] & 0x7F80u) == 0x7F80u ? 0x7FC0u : 0u, hi = (x[e] >> 16 & 0x7F80u) == 0x7F80u ? 0x7FC0u : 0u;
          x[e] = zero ? lo | hi << 16 : x[e] ^ 0x80008000u;
        }
        qf[k] = __builtin_bit_cast(pa_bf8, make_uint4(x[0], x[1], x[2], x[3]));
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // q, and what the part before wrote: only blocks are counted below

#pragma unroll 1
    for (int i = 0; i < at.blocks; ++i) {
      const int kb = at.kb + i, kfrom = slot * TILE, vfrom = (BUFS + slot) * TILE;
      const int bad = slot == 0 ? bad0 : bad1;
      const bool two = WAVES == 1 && BUFS == 2 && held > 1;             // the block after this one is on its way, too
      // the next block to begin, of this part or of the one after it: where, and in which buffer
      const int k = i + held;
      const bool here = k < at.blocks, more = here || k - at.blocks < nx.blocks;
      const int next_kb = here ? at.kb + k : nx.kb + k - at.blocks, u = two || BUFS == 1 ? slot : slot ^ 1;
      const int64_t next_head = here ? at.head : nx.head;
      // K of this block: behind it its V, and perhaps K and V of another
      if constexpr (WAVES > 1) {
        pa_wait<0>();
        __builtin_amdgcn_s_barrier();                     // the block is there, and every wave is done with the one before
        asm volatile("" ::: "memory");
        if (more) {
          wv.load_k(pg, next_kb, next_head, u * TILE);
          wv.load_v(pg, next_kb, next_head, (BUFS + u) * TILE);
        }
      } else {
        if (two) pa_wait<3 * NI>();
        else pa_wait<NI>();
      }
      pa_f4 st[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        st[y] = pa_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int x = 0; x < KS; ++x)
          st[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv.k_operand(kfrom, y, x), qf[x], st[y], 0, 0, 0);
      }
      pa_settle(st);
      if constexpr (WAVES == 1) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K is read: its place may be written
        if (more) wv.load_k(pg, next_kb, next_head, u * TILE);
      }
      const PaPages after = pages(k + 1);                 // (scalar loads, which the softmax covers)

      // Every row sees all of its keys, or the block is masked key by key.
      const bool edge = kPaKeys * kb < rg.base + rg.t_hi - p.window + 1 || kPaKeys * kb + kPaKeys - 1 > rg.base + rg.t_lo;
      uint4 ph[2], pl[2];
      if (edge) {
        const int first = kPaKeys * kb + (F8 ? 16 * g : 8 * g) - row_lo;      // koff(y, 4 g + j) = this + a constant
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            st[y][j] = (uint32_t)(first + Blk::koff(y, j)) <= (uint32_t)(row_hi - row_lo) && row_hi >= 0
                              ? st[y][j] : -INFINITY;
      }
      if (bad != 0) {                                   // a seen key on no page: the row becomes NaN
#pragma unroll 1
        for (int r = 0; r < 4; ++r) {
          const int key = kPaKeys * kb + 16 * r;
          if ((bad >> r) & 1 && key <= row_hi && key + 15 >= row_lo) l = __builtin_nanf("");
        }
      }
      float mx = st[0][0];
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, st[y][j]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float mn = fmaxf(m, mx * c);
      const float ms = mn == -INFINITY ? 0.0f : mn;      // no key yet: every weight below is exp2(-inf) = 0
      if (__builtin_amdgcn_ballot_w64(mn > m) != 0) {
        const float alpha = __builtin_amdgcn_exp2f(m - ms);
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
        m = mn;
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t hw[4], lw[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int y = 2 * x + (q >> 1), j = 2 * (q & 1);
          const float p0 = __builtin_amdgcn_exp2f(fmaf(st[y][j], c, -ms));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(st[y][j + 1], c, -ms));
          l += p0 + p1;
          hw[q] = bf16x2_rne_raw(p0, p1);
          lw[q] = bf16x2_rne_raw(p0 - __uint_as_float(hw[q] << 16), p1 - __uint_as_float(hw[q] & 0xFFFF0000u));
        }
        ph[x] = make_uint4(hw[0], hw[1], hw[2], hw[3]);
        pl[x] = make_uint4(lw[0], lw[1], lw[2], lw[3]);
      }

      // V of this block: behind it perhaps K and V of another, and the K just begun
      if constexpr (WAVES == 1) {
        if (two) {
          if (more) pa_wait<3 * NI>();
          else pa_wait<2 * NI>();
        } else {
          if (more) pa_wait<NI>();
          else pa_wait<0>();
        }
      }
      // O += V P. At an edge, what the places outside [lo, hi) hold (another sequence's tokens, NaN) may not reach the product:
      // their weight is 0, but 0 x NaN is not. Where rows see different keys, the same holds for a key that one row sees and
      // another does not: a V that is not finite there sends the block token by token, each token's columns with its own
      // keys' V only. (One copy of the product for all of this: a second is more code to fetch than its masks are work.)
      constexpr int VK = F8 ? 1 : 2;                      // 16-byte reads of V a tile of dims
      const int vkey = kPaKeys * kb + (F8 ? 16 * g : 8 * g);            // the first key of the first; the second's is 32 on
      uint4 keep[VK];
#pragma unroll
      for (int x = 0; x < VK; ++x) keep[x] = make_uint4(~0u, ~0u, ~0u, ~0u);
      int tok = -1, last = -1;
      if (edge) {
#pragma unroll
        for (int x = 0; x < VK; ++x) keep[x] = pa_keep<F8>(vkey + 32 * x, rg.lo, rg.hi);
        if (rg.t_lo != rg.t_hi) {
          bool odd = false;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int x = 0; x < VK; ++x) odd |= pa_not_finite<F8>(pa_and(wv.v_words(vfrom, dt, x), keep[x]));
          if (__builtin_amdgcn_ballot_w64(odd) != 0) {
            tok = rg.t_lo;
            last = rg.t_hi;
          }
        }
      }
#pragma unroll 1
      for (;;) {
        if (tok >= 0) {
          const int64_t first = (int64_t)rg.base + tok - p.window + 1;
          const int lo = first > rg.lo ? (int)(first < rg.hi ? first : rg.hi) : rg.lo;
          const int hi = rg.base + tok + 1 < rg.hi ? rg.base + tok + 1 : rg.hi;
#pragma unroll
          for (int x = 0; x < VK; ++x) keep[x] = pa_keep<F8>(vkey + 32 * x, lo, hi);
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const uint4 w0 = pa_and(wv.v_words(vfrom, dt, 0), keep[0]);
          uint4 v0 = w0, v1;
          if constexpr (F8) {
            v0 = pa_widen(w0.x, w0.y);
            v1 = pa_widen(w0.z, w0.w);
          } else {
            v1 = pa_and(wv.v_words(vfrom, dt, 1), keep[VK - 1]);
          }
          const pa_bf8 a0 = __builtin_bit_cast(pa_bf8, v0), a1 = __builtin_bit_cast(pa_bf8, v1);
          pa_f4 o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, __builtin_bit_cast(pa_bf8, ph[0]), acc[dt], 0, 0, 0);
          o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, __builtin_bit_cast(pa_bf8, ph[1]), o, 0, 0, 0);
          o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, __builtin_bit_cast(pa_bf8, pl[0]), o, 0, 0, 0);
          o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, __builtin_bit_cast(pa_bf8, pl[1]), o, 0, 0, 0);
          acc[dt] = tok < 0 || rt == tok ? o : acc[dt];
        }
        pa_settle(acc);
        if (tok == last) break;
        ++tok;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V is read
      if (more) {
        if constexpr (WAVES == 1) wv.load_v(pg, next_kb, next_head, (BUFS + u) * TILE);
        if (u == 0) bad0 = pg.bad;
        else bad1 = pg.bad;
      }
      pg = after;
      held -= more ? 0 : 1;
      if (BUFS == 2) slot ^= 1;
    }

    // The rows' output, or the part's results for the second launch.
    const bool whole = begins && ends;
    float* part = p.part + (2ll * me + (nth > 0)) * (ROWS * (D + 2));      // (whole: not used)
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if constexpr (SPLIT > 1) {
      constexpr int SLOT = 16 * (D + 2);
      static_assert(4 * SLOT <= Blk::RING);
      float* mine = reinterpret_cast<float*>(ring);       // (this wave is done with its blocks)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<float4*>(mine + r * D + 16 * dt + 4 * g) = make_float4(acc[dt][0], acc[dt][1], acc[dt][2], acc[dt][3]);
      if (g == 0) {
        mine[16 * D + r] = m;
        mine[16 * D + 16 + r] = l;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < rg.here * (D / 4); i += 64 * SPLIT) {
        const int row = i / (D / 4), d = 4 * (i - row * (D / 4));
        float jm = -INFINITY, jl = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < SPLIT; ++k) jm = fmaxf(jm, reinterpret_cast<const float*>(rings + k * Blk::RING)[16 * D + row]);
        const float mz = jm == -INFINITY ? 0.0f : jm;
#pragma unroll
        for (int k = 0; k < SPLIT; ++k) {
          const float* q = reinterpret_cast<const float*>(rings + k * Blk::RING);
          const float w = __builtin_amdgcn_exp2f(q[16 * D + row] - mz);
          const float4 x = *reinterpret_cast<const float4*>(q + row * D + d);
          o.x = fmaf(w, x.x, o.x); o.y = fmaf(w, x.y, o.y); o.z = fmaf(w, x.z, o.z); o.w = fmaf(w, x.w, o.w);
          jl = fmaf(w, q[16 * D + 16 + row], jl);
        }
        const PaRow to_row(p, rg, b, kv, ROWS * group + row, jl);
        to_row.write(d, o.x, o.y, o.z, o.w);
        if (d == 0) to_row.write_lse(p, jm, jl);
      }
    } else if (r < rg.here) {
      if (whole) {
        const PaRow row(p, rg, b, kv, ROWS * group + r, l);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) row.write(16 * dt + 4 * g, acc[dt][0], acc[dt][1], acc[dt][2], acc[dt][3]);
        if (g == 0) row.write_lse(p, m, l);
      } else {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          *reinterpret_cast<float4*>(part + r * D + 16 * dt + 4 * g) = make_float4(acc[dt][0], acc[dt][1], acc[dt][2], acc[dt][3]);
        if (g == 0) {
          part[ROWS * D + r] = m;
          part[ROWS * (D + 1) + r] = l;
        }
      }
    }
    if (p.balanced && begins && threadIdx.x == 0)         // whose parts are to be joined, up to who holds its end
      p.open[item] = whole ? make_int4(-1, 0, 0, 0) : make_int4(me, nth > 0, (int)((uint32_t)(e - 1) / (uint32_t)per), 0);
    at = nx;
    rg = nrg;
  }
}

// Joins the parts of item blockIdx.x, where it has more than one: 32 threads across 128 of its rows' values, eight groups
// of them over the parts, each with its next four parts' loads in flight.
template <int D, int WAVES>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttn p) {
  constexpr int C = D / 4, ROWS = 16 * WAVES, GROUPS = 8;
  constexpr int64_t SLOT = ROWS * (D + 2);
  __shared__ float4 so[GROUPS][32];
  __shared__ float sl[GROUPS][32], sm[GROUPS][32];
  const int item = (int)blockIdx.x;
  const int4 open = p.open[item];
  const int me = open.x;
  if (me < 0) return;
  const int col = threadIdx.x & 31, grp = threadIdx.x >> 5, parts = open.z - me + 1;
  const int row = ((int)blockIdx.y * 32 + col) / C, d = 4 * ((int)blockIdx.y * 32 + col - row * C);
  const int pair = pa_div(item, p.by_kv), kvh = item - pair * p.KV, b = pa_div(pair, p.by_groups), group = pair - b * p.groups;
  const int rows = p.rows - ROWS * group < ROWS ? p.rows - ROWS * group : ROWS;
  float m = -INFINITY, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](float pm, float plsum, float4 x) __attribute__((always_inline)) {
    const float mn = fmaxf(m, pm), mz = mn == -INFINITY ? 0.0f : mn;
    const float a = __builtin_amdgcn_exp2f(m - mz), w = __builtin_amdgcn_exp2f(pm - mz);
    o.x = fmaf(w, x.x, o.x * a); o.y = fmaf(w, x.y, o.y * a); o.z = fmaf(w, x.z, o.z * a); o.w = fmaf(w, x.w, o.w * a);
    l = fmaf(w, plsum, l * a);
    m = mn;
  };
  if (row < rows) {
    for (int i0 = grp; i0 < parts; i0 += 4 * GROUPS) {
      float pm[4], ps[4];
      float4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + k * GROUPS;
        pm[k] = -INFINITY;
        ps[k] = 0.0f;
        x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (i < parts) {
          const float* q = p.part + (2ll * (me + i) + (i == 0 ? open.y : 0)) * SLOT;
          pm[k] = q[ROWS * D + row];
          ps[k] = q[ROWS * (D + 1) + row];
          x[k] = *reinterpret_cast<const float4*>(q + row * D + d);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) add(pm[k], ps[k], x[k]);
    }
  }
  so[grp][col] = o;
  sl[grp][col] = l;
  sm[grp][col] = m;
  __syncthreads();
  if (grp != 0 || row >= rows) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) add(sm[i][col], sl[i][col], so[i][col]);
  const PaRange rg(p, b, group, ROWS);
  const PaRow to(p, rg, b, kvh, ROWS * group + row, l);
  to.write(d, o.x, o.y, o.z, o.w);
  if (d == 0) to.write_lse(p, m, l);
}

// How a call is cut: by the table's width, since the lengths are known on the GPU only. (Its figures are of tables as long as the
// sequences; short ones in a wide table go the way of long ones: 100 keys of 16 heads 6.7 us, 10.3 in a table for 8192, 4 times 300
// keys of 20 heads 8.0 and 11.3.) waves: of a workgroup, each with 16 rows of the row group; they share one read of the keys (32 tokens of 16
// heads, 8 sequences of 8000 keys of 64 values: 58 us, 97 with a wave a workgroup; 4 tokens of 8 heads a kv head, 16 sequences of
// 25 000 keys of 128: 173 and 265; 48 rows on three waves 64 us, on four 77). split: waves that share an item's blocks.
// workgroups: 0, one an item, or the parts of a balanced line.
struct PaPlan {
  int64_t waves, split, groups, items, workgroups;
};
static PaPlan pa_plan(int64_t B, int64_t G, int64_t KV, int64_t T, int64_t D, bool f8, int64_t page, int64_t M,
                      int64_t window) {
  PaPlan c{};
  const int64_t rows = T * G;
  c.waves = rows <= 48 ? (rows + 15) / 16 : 4;
  c.groups = (rows + 16 * c.waves - 1) / (16 * c.waves);
  int64_t keys = M * page;
  if (window < keys) keys = window + T - 1 < keys ? window + T - 1 : keys;
  const int64_t items = c.items = B * c.groups * KV, held = (int64_t)pa_held((int)D, f8, (int)c.waves) * compute_units();
  // Four waves an item, joined in LDS, where the ranges are short and the items leave room for the waves (their rings fit twice
  // into a compute unit, bf16 of D = 128 once): 20 items of 256 keys of 64 6.4 us (balanced 9.1), 160 of 512 9.6 (12.1), 320 of
  // 1024 20 (24), 480 of 256 10.0 (11.4, one wave an item). Not: 20 of 1024 12.8 (balanced 10.0), 8 of 512 of 128 12.7 (10.8),
  // 800 of 256 16.7 (one wave 13.2), 512 of 120 of 128 16.1 (one wave 11.7).
  const int64_t blocks = (keys + kPaKeys - 1) / kPaKeys, units = compute_units();
  c.split = 1;
  if (c.waves == 1 && blocks > 1 && items <= (D == 128 && !f8 ? 1 : 2) * units &&
      (blocks <= 4 || (blocks <= 16 && blocks * units <= 32 * items))) {
    c.split = 4;
    return c;
  }
  // One an item, and no second launch, where it pays or must be:
  //   every item is a few blocks: 800 items of 256 keys 13.1 us; but 160 of 512 15.9, balanced 12.0;
  //   none is long and they are enough to fill the GPU: 1280 items of 2048 keys at most 103 us, balanced 111; of 1024 56 and 62;
  //   but of 100 to 4096 137 and 132;
  //   finding one's part of the line, which walks all sequences, would take long, or the line does not fit 31 bits.
  if (keys <= 4 * kPaKeys || (keys <= 40 * kPaKeys && items >= 4ll * compute_units()) || B * c.groups > 1024 ||
      items * (keys / kPaKeys + 2) > 0x7FFFFFFFll)
    return c;
  const int64_t most = items * ((keys + 63) / 64 + 1);
  c.workgroups = held < most ? held : most;
  return c;
}
static size_t pa_workspace(const PaPlan& c, int64_t D) {
  return c.workgroups == 0 ? 0 : (size_t)(c.workgroups * (2 * 16 * c.waves * (D + 2) * 4) + c.items * 16);
}

template <int D, bool F8, bool WIDE>
static const void* pa_kernel(int64_t waves, int64_t split) {
  return waves == 1 ? (split == 1 ? reinterpret_cast<const void*>(&paged_attn_kernel<D, F8, WIDE, 1>)
                                  : reinterpret_cast<const void*>(&paged_attn_kernel<D, F8, WIDE, 1, 4>))
       : waves == 2 ? reinterpret_cast<const void*>(&paged_attn_kernel<D, F8, WIDE, 2>)
       : waves == 3 ? reinterpret_cast<const void*>(&paged_attn_kernel<D, F8, WIDE, 3>)
                    : reinterpret_cast<const void*>(&paged_attn_kernel<D, F8, WIDE, 4>);
}
template <int D>
static const void* pa_kernel(bool f8, bool wide, int64_t waves, int64_t split) {
  return f8 ? (wide ? pa_kernel<D, true, true>(waves, split) : pa_kernel<D, true, false>(waves, split))
            : (wide ? pa_kernel<D, false, true>(waves, split) : pa_kernel<D, false, false>(waves, split));
}
template <int D>
static const void* pa_join(int64_t waves) {
  return waves == 1 ? reinterpret_cast<const void*>(&paged_join_kernel<D, 1>)
       : waves == 2 ? reinterpret_cast<const void*>(&paged_join_kernel<D, 2>)
       : waves == 3 ? reinterpret_cast<const void*>(&paged_join_kernel<D, 3>)
                    : reinterpret_cast<const void*>(&paged_join_kernel<D, 4>);
}

}  // namespace flw

using namespace flw;

extern "C" size_t flw_paged_attention_workspace_bytes(int64_t B, int64_t H, int64_t KV, int64_t T, int64_t D,
                                                      int cache_dtype, int64_t page_size, int64_t table_cols,
                                                      int64_t window) {
  if (B <= 0 || H <= 0 || KV <= 0 || H % KV != 0 || T <= 0 || D <= 0 || page_size <= 0 || table_cols <= 0 || window <= 0)
    return 0;
  return pa_workspace(pa_plan(B, H / KV, KV, T, D, cache_dtype == FLW_E4M3, page_size, table_cols, window), D);
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
  const int64_t w = window < 0 ? 0 : window > 0x7FFFFFFFll ? 0x7FFFFFFFll : window;
  PaPlan c = pa_plan(B, H / KV, KV, T, D, cache_dtype == FLW_E4M3, page_size, table_cols, w > 0 ? w : 1);
  if (w == 0) c.workgroups = 0;
  const int64_t items = c.items;
  FLW_REQUIRE(items <= 0x7FFFFFFFll && items * KV <= 0xFFFFFFFFll && B * c.groups * c.groups <= 0xFFFFFFFFll &&
              (T * (H / KV) + 64) * (H / KV) <= 0xFFFFFFFFll, FLW_E_UNSUPPORTED, "shape too large");      // pa_div's terms
  const size_t need = pa_workspace(c, D);
  FLW_REQUIRE(need == 0 || (workspace != nullptr && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need),
              FLW_E_WORKSPACE, "workspace needs %zu bytes (16-byte aligned)", need);
  PagedAttn p{};
  p.q = static_cast<const uint16_t*>(q);
  p.qsb = q_strides[0]; p.qsh = q_strides[1]; p.qst = q_strides[2];
  p.k = static_cast<const uint8_t*>(k_pages); p.v = static_cast<const uint8_t*>(v_pages);
  p.tables = tables; p.lens = lens; p.counts = counts; p.k_scale = k_scale; p.v_scale = v_scale;
  p.out = static_cast<uint16_t*>(out);
  p.osb = out_strides[0]; p.osh = out_strides[1]; p.ost = out_strides[2];
  p.lse = lse;
  p.open = static_cast<int4*>(workspace);
  p.part = static_cast<float*>(workspace) + 4 * items;
  p.P = num_pages; p.B = (int)B; p.H = (int)H; p.KV = (int)KV; p.G = (int)(H / KV); p.T = (int)T;
  p.rows = (int)(T * (H / KV)); p.groups = (int)c.groups; p.M = (int)table_cols; p.shift = __builtin_ctzll(page_size);
  auto by = [](int64_t n) { return n == 1 ? 0u : (uint32_t)((0x100000000ll + n - 1) / n); };
  p.by_g = by(H / KV); p.by_groups = by(c.groups); p.by_kv = by(KV);
  p.window = (int)w; p.balanced = c.workgroups != 0; p.scale = scale * 1.44269504088896341f;
  const bool f8 = cache_dtype == FLW_E4M3, wide = page_size >= kPaKeys;
  const void* kern = D == 32 ? pa_kernel<32>(f8, wide, c.waves, c.split) : D == 64 ? pa_kernel<64>(f8, wide, c.waves, c.split)
                                                                           : pa_kernel<128>(f8, wide, c.waves, c.split);
  const void* join = D == 32 ? pa_join<32>(c.waves) : D == 64 ? pa_join<64>(c.waves) : pa_join<128>(c.waves);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Timer tm = take_timer();
  const dim3 grid((unsigned)(c.workgroups != 0 ? c.workgroups : items));
  (void)launch_ext(kern, grid, dim3((unsigned)(64 * c.waves * c.split)), 0, s, p, tm.start, c.workgroups == 0 ? tm.stop : nullptr);
  if (c.workgroups != 0) {
    const int64_t rows = p.rows < 16 * c.waves ? p.rows : 16 * c.waves;
    (void)launch_ext(join, dim3((unsigned)items, (unsigned)((rows * (D / 4) + 31) / 32)), dim3(256), 0, s, p, nullptr,
                     tm.stop);
  }
  return check_launch("flw_paged_attention");
}
