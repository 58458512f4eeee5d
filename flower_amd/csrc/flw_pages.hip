// The bookkeeping of a paged key-value cache on the device: room for new tokens (reserve), sequences forked, dropped or
// put in another order (reorder), pages drawn together (compact). Nothing of it comes back to the host, so a decode step
// with its page allocation is one captured graph.
//
// State: tables [S, M] int32, the page of each run of `page` positions of a sequence, -1 where it holds none (an entry
// that is no page counts as none); lens [S] int32; refs [P] int32, how many table entries hold a page, 0 = free. A page
// is always taken as the free one of the lowest number, in the order of the sequences, so that every result is defined,
// whatever the order in which the workgroups run. Integer atomics on refs only add and subtract: their order is not seen.
//
// What bounds it: reserve and the bookkeeping of the others, a few dependent launches over a few hundred KB; the copies
// of reorder and compact, HBM.

#include "flw_common.h"

namespace flw {

constexpr int kScan = 1024;       // threads of the one workgroup that allocates

struct PagesParams {
  const int32_t* tables;          // in
  const int32_t* lens;
  const int32_t* refs;
  const int32_t* arg;             // reserve: counts; reorder: parents
  int32_t* tables_out;            // out: may be the inputs
  int32_t* lens_out;
  int32_t* refs_out;
  int32_t* granted;               // reserve
  int32_t* kept;                  // reorder, or NULL: 1 where place s holds positions of its parent, 0 where it is empty
  int32_t* need;                  // workspace: [S] pages wanted, -1 where the request cannot be met at all
  int32_t* pairs;                 // workspace: [S][3] dst, src, tokens to copy (dst -1: nothing)
  int32_t* list;                  // workspace: [P] free pages in ascending order
  int S, M, P, shift, window;
};

// ---------------------------------------------------------------- copies

// dst[0..n) = src[0..n) for up to three arrays, one launch.
struct CopyInts {
  int32_t* dst[3];
  const int32_t* src[3];
  int64_t n[3];
};
__global__ __launch_bounds__(256) void copy_ints_kernel(CopyInts p) {
  const int64_t step = (int64_t)gridDim.x * 256;
#pragma unroll
  for (int a = 0; a < 3; ++a)
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.n[a]; i += step) p.dst[a][i] = p.src[a][i];
}
static void copy_ints(CopyInts c, hipStream_t s) {
  int64_t most = 0;
  for (int a = 0; a < 3; ++a) {
    if (c.dst[a] == c.src[a] || c.dst[a] == nullptr) c.n[a] = 0;
    most = most > c.n[a] ? most : c.n[a];
  }
  if (most == 0) return;
  int64_t blocks = (most + 255) / 256;
  blocks = blocks > 1024 ? 1024 : blocks;
  (void)launch_args(reinterpret_cast<const void*>(&copy_ints_kernel), dim3((unsigned)blocks), dim3(256), 0, s, nullptr,
                    nullptr, c);
}

__device__ __forceinline__ bool is_page(int32_t id, int P) { return (uint32_t)id < (uint32_t)P; }

// Inclusive sum over the workgroup's kScan threads; `total` the last one's.
__device__ __forceinline__ int scan_sum(int x, int* lds, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int v = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  __syncthreads();                          // the last call's readers are done with lds
  if (lane == 63) lds[wave] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kScan / 64; ++w) {
    const int y = lds[w];
    before += w < wave ? y : 0;
    all += y;
  }
  *total = all;
  return before + v;
}

// The free pages of the lowest numbers, ascending, into list: at most `want`. Returns how many there are (at most want).
__device__ __forceinline__ int free_list(const int32_t* refs, int P, int want, int32_t* list, int* lds) {
  int have = 0;
  for (int p0 = 0; p0 < P && have < want; p0 += 4 * kScan) {
    const int at = p0 + 4 * (int)threadIdx.x;
    int r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = at + i < P ? refs[at + i] : 1;
    const int n = (r[0] == 0) + (r[1] == 0) + (r[2] == 0) + (r[3] == 0);
    int all;
    int to = have + scan_sum(n, lds, &all) - n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r[i] == 0) {
        if (to < want) list[to] = at + i;
        ++to;
      }
    have += all;
  }
  __syncthreads();                          // list is written
  return have < want ? have : want;
}

// ---------------------------------------------------------------- reserve

// One workgroup a sequence: entries behind the window given back, entries to fill counted.
__global__ __launch_bounds__(256) void reserve_rows_kernel(PagesParams p) {
  __shared__ int red[4];
  const int s = blockIdx.x;
  const int32_t len = p.lens[s], cnt = p.arg[s];
  const bool fits = cnt > 0 && len >= 0 && (int64_t)len + cnt <= ((int64_t)p.M << p.shift);
  const int64_t gone = p.window > 0 ? ((int64_t)len - p.window + 1) >> p.shift : 0;       // entries [0, gone) are behind it
  const int first = fits ? len >> p.shift : 0, last = fits ? (int)(((int64_t)len + cnt - 1) >> p.shift) : -1;
  int n = 0;
  for (int j = threadIdx.x; j < p.M; j += 256) {
    const int64_t at = (int64_t)s * p.M + j;
    int32_t id = p.tables[at];
    if (!is_page(id, p.P)) id = -1;
    if (j < gone && id >= 0) {
      atomicSub(&p.refs_out[id], 1);
      id = -1;
    }
    // wanted: an entry of the new tokens' positions that is empty (one that begins before lens counts only where it is)
    n += j >= first && j <= last && id < 0;
    p.tables_out[at] = id;
  }
  for (int o = 32; o >= 1; o >>= 1) n += __shfl_xor(n, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) p.need[s] = fits ? red[0] + red[1] + red[2] + red[3] : -1;
}

// One workgroup: who gets pages, which ones, and where they go.
__global__ __launch_bounds__(kScan) void reserve_take_kernel(PagesParams p) {
  __shared__ int lds[kScan / 64];
  // how many pages are wanted in all (counted up to P)
  int64_t wanted = 0;
  for (int s0 = 0; s0 < p.S; s0 += kScan) {
    const int s = s0 + (int)threadIdx.x;
    int all;
    scan_sum(s < p.S && p.need[s] > 0 ? p.need[s] : 0, lds, &all);
    wanted += all;
  }
  const int have = free_list(p.refs_out, p.P, wanted < p.P ? (int)wanted : p.P, p.list, lds);
  int64_t before = 0;
  for (int s0 = 0; s0 < p.S; s0 += kScan) {
    const int s = s0 + (int)threadIdx.x;
    const int need = s < p.S ? p.need[s] : 0, n = need > 0 ? need : 0;
    int all;
    const int64_t upto = before + scan_sum(n, lds, &all);
    before += all;
    if (s >= p.S) continue;
    const bool given = need >= 0 && (n == 0 || upto <= have);
    const int32_t len = p.lens[s], cnt = p.arg[s];
    if (given && n > 0) {
      int at = (int)(upto - n);
      const int last = (len + cnt - 1) >> p.shift;
      for (int j = len >> p.shift; j <= last; ++j) {
        int32_t* e = p.tables_out + (int64_t)s * p.M + j;
        if (*e < 0) {
          const int id = p.list[at++];
          *e = id;
          p.refs_out[id] = 1;
        }
      }
    }
    p.granted[s] = given ? cnt : 0;
    p.lens_out[s] = given ? len + cnt : len;
  }
}

// ---------------------------------------------------------------- reorder

// One workgroup a place s: its parent's entries taken over (all of them by the one child that keeps the parent's last,
// partly filled page; the full pages by the others), its own old ones let go.
__global__ __launch_bounds__(256) void reorder_rows_kernel(PagesParams p) {
  __shared__ int red[4];
  const int s = blockIdx.x;
  const int32_t par = p.arg[s];
  const bool real = (uint32_t)par < (uint32_t)p.S;
  bool keeps = false;
  if (real) {                               // the child in its parent's place, or else the first
    if (par == s) {
      keeps = true;
    } else {
      int other = 0;                        // a child that comes before s in that order
      for (int c = threadIdx.x; c < p.S; c += 256) other |= p.arg[c] == par && (c < s || c == par);
      if (threadIdx.x < 4) red[threadIdx.x] = 0;
      __syncthreads();
      if (__builtin_amdgcn_ballot_w64(other != 0) != 0 && (threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = 1;
      __syncthreads();
      keeps = (red[0] | red[1] | red[2] | red[3]) == 0;
    }
  }
  int32_t len = real ? p.lens[par] : 0;
  len = len < 0 ? 0 : len;
  const int full = len >> p.shift;
  for (int j = threadIdx.x; j < p.M; j += 256) {
    const int64_t at = (int64_t)s * p.M + j;
    int32_t was = p.tables[at], id = -1;
    if (real && (keeps || j < full)) id = p.tables[(int64_t)par * p.M + j];
    if (!is_page(id, p.P)) id = -1;
    if (!is_page(was, p.P)) was = -1;
    if (was != id) {
      if (was >= 0) atomicSub(&p.refs_out[was], 1);
      if (id >= 0) atomicAdd(&p.refs_out[id], 1);
    }
    p.tables_out[at] = id;
  }
  if (threadIdx.x == 0) {
    const int used = len & ((1 << p.shift) - 1);
    const int32_t src = real && !keeps && used != 0 && full < p.M ? p.tables[(int64_t)par * p.M + full] : -1;
    const bool copies = is_page(src, p.P);
    p.need[s] = copies ? 1 : 0;
    p.pairs[3 * s] = -1;
    p.pairs[3 * s + 1] = copies ? src : -1;
    p.pairs[3 * s + 2] = used;
    p.lens_out[s] = len;
    if (p.kept != nullptr) p.kept[s] = len > 0;
  }
}

// One workgroup: a page for each copy; where none is left the place is emptied.
__global__ __launch_bounds__(kScan) void reorder_take_kernel(PagesParams p) {
  __shared__ int lds[kScan / 64];
  int wanted = 0;
  for (int s0 = 0; s0 < p.S; s0 += kScan) {
    const int s = s0 + (int)threadIdx.x;
    int all;
    scan_sum(s < p.S ? p.need[s] : 0, lds, &all);
    wanted += all;
  }
  if (wanted == 0) return;
  const int have = free_list(p.refs_out, p.P, wanted < p.P ? wanted : p.P, p.list, lds);
  int before = 0;
  for (int s0 = 0; s0 < p.S; s0 += kScan) {
    const int s = s0 + (int)threadIdx.x, need = s < p.S ? p.need[s] : 0;
    int all;
    const int upto = before + scan_sum(need, lds, &all);
    before += all;
    if (need == 0) continue;
    const int full = p.lens_out[s] >> p.shift;
    int32_t* row = p.tables_out + (int64_t)s * p.M;
    if (upto <= have) {
      const int id = p.list[upto - 1];
      row[full] = id;
      p.refs_out[id] = 1;
      p.pairs[3 * s] = id;
    } else {
      for (int j = 0; j < full && j < p.M; ++j) {
        if (row[j] >= 0) atomicSub(&p.refs_out[row[j]], 1);
        row[j] = -1;
      }
      p.lens_out[s] = 0;
      if (p.kept != nullptr) p.kept[s] = 0;
    }
  }
}

// ---------------------------------------------------------------- page copies

struct PageCopy {
  uint8_t* k;                     // (L, P, KV, page, D)
  uint8_t* v;                     // (L, P, KV, D, page)
  const int32_t* pairs;           // reorder: [S][3]; compact: [2][P] dst then src
  const int32_t* count;           // compact: pairs in use
  int64_t P;
  int S, L, KV, D, page, size;    // S: reorder; size: bytes a value
};

// 16 bytes that are read (written) once: past the caches (reorder's copies 56 us with such stores alone, 51 with both).
typedef uint32_t Run __attribute__((ext_vector_type(4)));
__device__ __forceinline__ Run run_load(const uint8_t* p) { return __builtin_nontemporal_load(reinterpret_cast<const Run*>(p)); }
__device__ __forceinline__ void run_store(uint8_t* p, Run x) { __builtin_nontemporal_store(x, reinterpret_cast<Run*>(p)); }

// Reorder: the first `used` positions of page src to page dst; one workgroup a (place, k or v, layer, head), a thread a 16-byte
// run at a time. The places are the grid's slow side and k / v its next one: workgroups go to the eight XCDs by their number
// modulo 8, so that with places, or k / v, on the fast side a regular pattern of forks, or v's partly written lines, fell to half
// of them. 32 forks of 47 tokens in 12 layers of 20 heads of 64 (184 MB read and written): 45 us, 4.1 TB/s; places fast 70, k / v
// fast 51. Two heads a thread the same, four 48; whole 64-byte pieces written (with what dst held) 57.
constexpr int kCopyRows = 32768;
__global__ __launch_bounds__(256) void copy_tail_kernel(PageCopy p) {
  const int s = blockIdx.y + kCopyRows * blockIdx.z;
  if (s >= p.S) return;
  const int32_t dst = p.pairs[3 * s], src = p.pairs[3 * s + 1];
  if (dst < 0) return;
  const int half = (int)gridDim.x >> 1;     // layers x heads
  const bool rows = (int)blockIdx.x >= half;
  const int64_t of = (int)blockIdx.x - (rows ? half : 0), layer = of / p.KV, head = of - layer * p.KV;
  const int64_t bytes = (int64_t)p.page * p.D * p.size;
  uint8_t* pool = rows ? p.v : p.k;
  const uint8_t* a = pool + ((layer * p.P + src) * p.KV + head) * bytes;
  uint8_t* b = pool + ((layer * p.P + dst) * p.KV + head) * bytes;
  // k: `used` rows of D values, a whole number of runs. v: of each of D rows the first `used` values, in `per` runs.
  const int fill = p.pairs[3 * s + 2] * p.size, per = (fill + 15) / 16, n = rows ? p.D * per : p.D * fill / 16;
  const uint32_t by_per = (uint32_t)((0x100000000ull + (unsigned)per - 1) / (unsigned)per);      // i / per = i by_per >> 32
  for (int i = threadIdx.x; i < n; i += 256) {
    const int row = per == 1 ? i : (int)__umulhi((uint32_t)i, by_per), run = i - row * per;
    const int left = rows ? fill - 16 * run : 16;
    const int64_t at = rows ? (int64_t)row * p.page * p.size + 16 * run : 16 * (int64_t)i;
    Run x = run_load(a + at);
    if (left < 16) {                        // the row's last run: what lies behind `used` stays (its one writer is this thread)
      const Run was = *reinterpret_cast<const Run*>(b + at);      // (its line stays in L2 for the stores: not so 75 us)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = left - 4 * e;         // bytes of this word to take
        const uint32_t m = k >= 4 ? 0xFFFFFFFFu : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
        x[e] = (x[e] & m) | (was[e] & ~m);
      }
    }
    run_store(b + at, x);
  }
}

// Compact: whole pages; workgroup x of gridDim.x takes every gridDim.x-th piece of 16 KB of (pair, layer, k or v).
__global__ __launch_bounds__(256) void copy_pages_kernel(PageCopy p) {
  const int n = p.count[0];
  const int64_t bytes = (int64_t)p.KV * p.page * p.D * p.size, pieces = (bytes + 16383) / 16384;
  const int64_t all = (int64_t)n * p.L * 2 * pieces;
  for (int64_t w = blockIdx.x; w < all; w += gridDim.x) {
    const int64_t piece = w % pieces, of = w / pieces, layer = (of >> 1) % p.L, i = (of >> 1) / p.L;
    const int32_t dst = p.pairs[i], src = p.pairs[p.P + i];
    uint8_t* pool = of & 1 ? p.v : p.k;
    const uint8_t* a = pool + ((layer * p.P + src) * bytes + piece * 16384);
    uint8_t* b = pool + ((layer * p.P + dst) * bytes + piece * 16384);
    const int64_t left = bytes - piece * 16384;
    const int m = (int)((left < 16384 ? left : 16384) / 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = (int)threadIdx.x + 256 * j;
      if (e < m) run_store(b + 16 * e, run_load(a + 16 * e));
    }
  }
}

// ---------------------------------------------------------------- compact

// One workgroup: the pages in use (n of them), and for each one of number >= n, in ascending order, the free number
// < n that it moves to, in ascending order. to[p]: p's new number, -1 for a free page.
__global__ __launch_bounds__(kScan) void compact_plan_kernel(const int32_t* refs, int P, int32_t* to, int32_t* pairs,
                                                            int32_t* count, int32_t* live) {
  __shared__ int lds[kScan / 64];
  int n = 0;
  for (int p0 = 0; p0 < P; p0 += 4 * kScan) {
    const int at = p0 + 4 * (int)threadIdx.x;
    int c = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) c += at + i < P && refs[at + i] != 0;
    int all;
    scan_sum(c, lds, &all);
    n += all;
  }
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < P; p0 += 4 * kScan) {
    const int at = p0 + 4 * (int)threadIdx.x;
    bool used[4];
    int h = 0, m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      used[i] = at + i < P && refs[at + i] != 0;
      h += !used[i] && at + i < n;
      m += used[i] && at + i >= n;
    }
    int all;
    int hi = holes + scan_sum(h, lds, &all) - h;
    holes += all;
    int mi = movers + scan_sum(m, lds, &all) - m;
    movers += all;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (at + i >= P) continue;
      if (!used[i] && at + i < n) pairs[hi++] = at + i;
      if (used[i] && at + i >= n) pairs[P + mi++] = at + i;
      to[at + i] = used[i] && at + i < n ? at + i : -1;
    }
  }
  __syncthreads();                          // the lists and `to` are written
  for (int i = threadIdx.x; i < movers; i += kScan) to[pairs[P + i]] = pairs[i];
  if (threadIdx.x == 0) {
    count[0] = movers;
    live[0] = n;
  }
}

// Tables and refs in the new numbers. A moved page's count goes to its new place, which no other thread writes.
__global__ __launch_bounds__(256) void compact_rows_kernel(PagesParams p, const int32_t* to, const int32_t* live) {
  const int64_t step = (int64_t)gridDim.x * 256, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t i = at; i < (int64_t)p.S * p.M; i += step) {
    const int32_t id = p.tables[i];
    p.tables_out[i] = is_page(id, p.P) ? to[id] : -1;
  }
  const int n = live[0];
  for (int64_t i = at; i < p.P; i += step) {
    const int32_t t = to[i];
    if (t >= 0) {
      const int32_t r = p.refs[i];
      p.refs_out[t] = r;
      if (t != (int32_t)i) p.refs_out[i] = 0;
    } else if (i >= n) {
      p.refs_out[i] = 0;                    // free, behind the pages in use; a free number below n is a mover's
    }
  }
}

static int pages_check(const void* tables, const void* lens, const void* refs, int64_t S, int64_t M, int64_t P) {
  FLW_REQUIRE(tables && lens && refs, FLW_E_INVALID, "null pointer");
  FLW_REQUIRE(S > 0 && M > 0 && P > 0, FLW_E_INVALID, "empty shape");
  FLW_REQUIRE(S <= 65536 && M <= 0x7FFFFFFFll && S * M <= 0x7FFFFFFFll && P <= 0x7FFFFFFFll - 4096, FLW_E_UNSUPPORTED,
              "shape too large");
  return FLW_OK;
}
static int page_size_check(int64_t page_size) {
  FLW_REQUIRE(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0, FLW_E_UNSUPPORTED,
              "page size must be a power of two from 16 to 1024, got %lld", (long long)page_size);
  return FLW_OK;
}
static int pool_check(const void* k, const void* v, int64_t L, int64_t KV, int64_t D, int cache_dtype) {
  FLW_REQUIRE(k && v && (((uintptr_t)k | (uintptr_t)v) & 15) == 0, FLW_E_INVALID, "pages must be non-null and 16-byte aligned");
  FLW_REQUIRE(cache_dtype == FLW_BF16 || cache_dtype == FLW_E4M3, FLW_E_INVALID, "the cache holds bf16 or e4m3");
  FLW_REQUIRE(D == 32 || D == 64 || D == 128, FLW_E_UNSUPPORTED, "head_dim must be 32/64/128, got %lld", (long long)D);
  FLW_REQUIRE(L > 0 && KV > 0, FLW_E_INVALID, "empty shape");
  FLW_REQUIRE(2 * L * KV <= 65535, FLW_E_UNSUPPORTED, "layers x kv heads must stay below 32768");
  return FLW_OK;
}
static int64_t up4(int64_t n) { return (n + 3) / 4 * 4; }

}  // namespace flw

using namespace flw;

extern "C" size_t flw_reserve_pages_workspace_bytes(int64_t S, int64_t P) {
  return S > 0 && P > 0 ? (size_t)(4 * (up4(S) + up4(P))) : 0;
}

extern "C" int flw_reserve_pages(const int32_t* tables, const int32_t* lens, const int32_t* refs, const int32_t* counts,
                                 int64_t S, int64_t table_cols, int64_t num_pages, int64_t page_size, int64_t window,
                                 int32_t* tables_out, int32_t* lens_out, int32_t* refs_out, int32_t* granted,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  int rc = pages_check(tables, lens, refs, S, table_cols, num_pages);
  if (rc || (rc = page_size_check(page_size)) != 0) return rc;
  FLW_REQUIRE(counts && tables_out && lens_out && refs_out && granted, FLW_E_INVALID, "null pointer");
  FLW_REQUIRE(table_cols * page_size <= 0x7FFFFFFFll, FLW_E_UNSUPPORTED, "shape too large");
  const size_t ws = flw_reserve_pages_workspace_bytes(S, num_pages);
  FLW_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= ws, FLW_E_WORKSPACE,
              "workspace needs %zu bytes (16-byte aligned)", ws);
  PagesParams p{};
  p.tables = tables; p.lens = lens; p.refs = refs; p.arg = counts;
  p.tables_out = tables_out; p.lens_out = lens_out; p.refs_out = refs_out; p.granted = granted;
  p.need = static_cast<int32_t*>(workspace); p.list = p.need + up4(S);
  p.S = (int)S; p.M = (int)table_cols; p.P = (int)num_pages; p.shift = __builtin_ctzll(page_size);
  p.window = (int)(window < 0 ? 0 : window > 0x7FFFFFFFll ? 0 : window);
  hipStream_t s = static_cast<hipStream_t>(stream);
  copy_ints(CopyInts{{refs_out, nullptr, nullptr}, {refs, nullptr, nullptr}, {num_pages, 0, 0}}, s);
  const Timer tm = take_timer();
  (void)launch_ext(reinterpret_cast<const void*>(&reserve_rows_kernel), dim3((unsigned)S), dim3(256), 0, s, p, tm.start, nullptr);
  (void)launch_ext(reinterpret_cast<const void*>(&reserve_take_kernel), dim3(1), dim3(kScan), 0, s, p, nullptr, tm.stop);
  return check_launch("flw_reserve_pages");
}

extern "C" size_t flw_reorder_pages_workspace_bytes(int64_t S, int64_t table_cols, int64_t P) {
  return S > 0 && table_cols > 0 && P > 0 ? (size_t)(4 * (up4(S) + up4(3 * S) + up4(P) + up4(S * table_cols) + up4(S))) : 0;
}

extern "C" int flw_reorder_pages(void* k_pages, void* v_pages, int cache_dtype, int64_t L, int64_t num_pages, int64_t KV,
                                 int64_t page_size, int64_t D, const int32_t* tables, const int32_t* lens,
                                 const int32_t* refs, const int32_t* parents, int64_t S, int64_t table_cols,
                                 int32_t* tables_out, int32_t* lens_out, int32_t* refs_out, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  return flw_reorder_pages_kept(k_pages, v_pages, cache_dtype, L, num_pages, KV, page_size, D, tables, lens, refs, parents, S,
                                table_cols, tables_out, lens_out, refs_out, nullptr, workspace, workspace_bytes, stream);
}

extern "C" int flw_reorder_pages_kept(void* k_pages, void* v_pages, int cache_dtype, int64_t L, int64_t num_pages, int64_t KV,
                                      int64_t page_size, int64_t D, const int32_t* tables, const int32_t* lens,
                                      const int32_t* refs, const int32_t* parents, int64_t S, int64_t table_cols,
                                      int32_t* tables_out, int32_t* lens_out, int32_t* refs_out, int32_t* kept,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  int rc = pages_check(tables, lens, refs, S, table_cols, num_pages);
  if (rc || (rc = page_size_check(page_size)) != 0 || (rc = pool_check(k_pages, v_pages, L, KV, D, cache_dtype)) != 0) return rc;
  FLW_REQUIRE(parents && tables_out && lens_out && refs_out, FLW_E_INVALID, "null pointer");
  const size_t ws = flw_reorder_pages_workspace_bytes(S, table_cols, num_pages);
  FLW_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= ws, FLW_E_WORKSPACE,
              "workspace needs %zu bytes (16-byte aligned)", ws);
  PagesParams p{};
  p.need = static_cast<int32_t*>(workspace);
  p.pairs = p.need + up4(S);
  p.list = p.pairs + up4(3 * S);
  int32_t* tables_ws = p.list + up4(num_pages);
  int32_t* lens_ws = tables_ws + up4(S * table_cols);
  // a place's row is written while its children still read it: in place, they read a copy
  const bool in_place = tables_out == tables, lens_in_place = lens_out == lens;
  p.tables = in_place ? tables_ws : tables; p.lens = lens_in_place ? lens_ws : lens; p.refs = refs; p.arg = parents;
  p.tables_out = tables_out; p.lens_out = lens_out; p.refs_out = refs_out; p.kept = kept;
  p.S = (int)S; p.M = (int)table_cols; p.P = (int)num_pages; p.shift = __builtin_ctzll(page_size);
  hipStream_t s = static_cast<hipStream_t>(stream);
  copy_ints(CopyInts{{refs_out, in_place ? tables_ws : nullptr, lens_in_place ? lens_ws : nullptr},
                     {refs, tables, lens}, {num_pages, S * table_cols, S}}, s);
  PageCopy c{};
  c.k = static_cast<uint8_t*>(k_pages); c.v = static_cast<uint8_t*>(v_pages); c.pairs = p.pairs; c.P = num_pages;
  c.L = (int)L; c.KV = (int)KV; c.D = (int)D; c.page = (int)page_size; c.size = cache_dtype == FLW_E4M3 ? 1 : 2;
  c.S = (int)S;
  const dim3 grid((unsigned)(2 * L * KV), (unsigned)(S < kCopyRows ? S : kCopyRows),
                  (unsigned)((S + kCopyRows - 1) / kCopyRows));
  const Timer tm = take_timer();
  (void)launch_ext(reinterpret_cast<const void*>(&reorder_rows_kernel), dim3((unsigned)S), dim3(256), 0, s, p, tm.start, nullptr);
  (void)launch_ext(reinterpret_cast<const void*>(&reorder_take_kernel), dim3(1), dim3(kScan), 0, s, p, nullptr, nullptr);
  (void)launch_ext(reinterpret_cast<const void*>(&copy_tail_kernel), grid, dim3(256), 0, s, c, nullptr, tm.stop);
  return check_launch("flw_reorder_pages");
}

extern "C" size_t flw_compact_pages_workspace_bytes(int64_t P) {
  return P > 0 ? (size_t)(4 * (up4(P) + up4(2 * P) + 4)) : 0;
}

extern "C" int flw_compact_pages(void* k_pages, void* v_pages, int cache_dtype, int64_t L, int64_t num_pages, int64_t KV,
                                 int64_t page_size, int64_t D, const int32_t* tables, const int32_t* refs, int64_t S,
                                 int64_t table_cols, int32_t* tables_out, int32_t* refs_out, int32_t* live, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  int rc = pages_check(tables, tables, refs, S, table_cols, num_pages);
  if (rc || (rc = page_size_check(page_size)) != 0 || (rc = pool_check(k_pages, v_pages, L, KV, D, cache_dtype)) != 0) return rc;
  FLW_REQUIRE(tables_out && refs_out && live, FLW_E_INVALID, "null pointer");
  const size_t ws = flw_compact_pages_workspace_bytes(num_pages);
  FLW_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= ws, FLW_E_WORKSPACE,
              "workspace needs %zu bytes (16-byte aligned)", ws);
  int32_t* to = static_cast<int32_t*>(workspace);
  int32_t* pairs = to + up4(num_pages);
  int32_t* count = pairs + up4(2 * num_pages);
  PagesParams p{};
  p.tables = tables; p.refs = refs; p.tables_out = tables_out; p.refs_out = refs_out;
  p.S = (int)S; p.M = (int)table_cols; p.P = (int)num_pages;
  PageCopy c{};
  c.k = static_cast<uint8_t*>(k_pages); c.v = static_cast<uint8_t*>(v_pages); c.pairs = pairs; c.count = count; c.P = num_pages;
  c.L = (int)L; c.KV = (int)KV; c.D = (int)D; c.page = (int)page_size; c.size = cache_dtype == FLW_E4M3 ? 1 : 2;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Timer tm = take_timer();
  (void)launch_args(reinterpret_cast<const void*>(&compact_plan_kernel), dim3(1), dim3(kScan), 0, s, tm.start, nullptr, refs,
                    (int)num_pages, to, pairs, count, live);
  int64_t ints = S * table_cols > num_pages ? S * table_cols : num_pages, blocks = (ints + 1023) / 1024;
  (void)launch_args(reinterpret_cast<const void*>(&compact_rows_kernel), dim3((unsigned)(blocks > 1024 ? 1024 : blocks)),
                    dim3(256), 0, s, nullptr, nullptr, p, static_cast<const int32_t*>(to), static_cast<const int32_t*>(live));
  const int64_t bytes = KV * page_size * D * c.size, most = (num_pages + 1) / 2 * L * 2 * ((bytes + 16383) / 16384);
  const int64_t wide = 8ll * compute_units();
  (void)launch_ext(reinterpret_cast<const void*>(&copy_pages_kernel), dim3((unsigned)(most < wide ? most : wide)), dim3(256), 0,
                   s, c, nullptr, tm.stop);
  return check_launch("flw_compact_pages");
}
