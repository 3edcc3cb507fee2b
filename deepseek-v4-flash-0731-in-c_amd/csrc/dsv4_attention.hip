// dsv4_attention.hip - attention of a chunk of new tokens per sequence over
// the paged cache (dsv4g_attention). Layout and rules: include/dsv4_gpu.h. No
// counterpart in the reference, whose attention stays on the host.
//
// A workgroup takes one sequence's query rows of one kv head, ROWS at a time
// (row = new token * group + head of the group, so heads that share a kv head
// share its tile), and walks the cache in stages of TT tokens through LDS: one
// pass with a running reference m and sum l of the softmax. Scores are
// transposed, S^T = K Q^T (a lane's column is one query row), because then
//  - m, l and the rescaling are one value per lane, and the weights of a row
//    leave the accumulators already in the operand layout of the second
//    product O^T = V^T P^T: no exchange between lanes but the maximum of the
//    two halves of a wave;
//  - K tiles are read row by row (16 bytes), V tiles by the transposing LDS
//    read, both from the same row-major tile: where the values are the keys,
//    a cached row is staged once for both products.
// Weights are rounded to BF16 for the matrix unit (2^-8 relative, as the cache
// rows are BF16 themselves); scores, m, l and O stay in fp32. m follows the
// maximum only when it grows by more than 2^8 (weights up to 2^8 lose nothing
// in fp32 or BF16): the rescaling of O, one multiplication per accumulator, is
// then rare.
//
// Rows of 16-byte chunks are stored with the chunk index XORed by a function
// of the row (chunk_swizzle): both kinds of read then touch every bank once
// per 16 lanes.
//
// What bounds it, with 64 latent heads of 512 if nothing else is said:
//  - a chunk of 2048 tokens behind 14336, BF16: 3.8 to 4.1 ms, 1.0 to 1.09
//    PFLOP/s, 77 to 83% of a large library product's rate; the matrix unit is
//    busy 45% of the time. Without the loads in the loop it would take 3.1 ms;
//    half of the LDS reads changed nothing. E4M3 4.4 to 4.6 ms (the conversion).
//  - decode over long caches: HBM. 64 sequences of 8100: BF16 124 to 152 us (3.6
//    to 4.4 TB/s), E4M3 126 to 145 us (the conversion: half the bytes, the same
//    LDS traffic); 8 sequences of 16000 over 8 kv heads of 128, BF16: 103 us, 5.1 TB/s.
//  - short ones: dependent latencies. One sequence of 1777: 18 us, of which
//    finding the place 2.6, the item and its pages 2, the query rows 2.7, the
//    first rows of the cache 1.4, the stages 2.2, the waves' exchange 3.1, the
//    parts' stores 1.3; the launch that joins them 5.5.
// Taken back: query rows asked for before the second stage's loads (a chunk 2%
// faster, decode 1 to 3% slower), query rows first of all (spills), weights by a
// branch on the scores' size (latent decode 3 to 8% slower, a chunk 3%).
#include <algorithm>
#include <cmath>
#include <utility>

#include "dsv4_cache.h"
#include "dsv4_device.h"
#include "dsv4_gpu_internal.h"

namespace dsv4 {

// f(0), .., f(N - 1), each with its number as a constant.
template <typename F, int... I>
__device__ __forceinline__ void each_of(F &f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F &&f) {
  each_of(f, std::make_integer_sequence<int, N>{});
}

typedef __bf16 Bf8 __attribute__((ext_vector_type(8)));
typedef float F16v __attribute__((ext_vector_type(16)));
typedef short S4 __attribute__((ext_vector_type(4)));
typedef int I4 __attribute__((ext_vector_type(4)));
typedef uint32_t U4 __attribute__((ext_vector_type(4)));
typedef uint32_t U2 __attribute__((ext_vector_type(2)));
// LDS by address
#define DSV4_LDS(T, at) (*(__attribute__((address_space(3))) T *)(uintptr_t)(at))

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float AT_GROW = 8.0f;  // log2 of what the weights may grow to before a rescaling

// A row's sums are kept against its m, the largest product q.k so far less what
// it may have grown since: weights are 2^((z - m) c2). The difference comes
// first: 2^(z c2 - fl(m c2)), one instruction less, would carry the rounding of
// m c2, which no 2^x holds once scores pass 2^30. With c2 below AT_TINY a
// distance that no fp32 number holds has a weight: the queries are halved then
// (what subnormal ones lose is far below a score's last place), and the scale is
// doubled.
constexpr float AT_TINY = 0x1p-100f;
__device__ __forceinline__ float attn_c2(float scale) {
  // not 0: a hidden score stays -inf
  return fmaxf(fabsf(scale) * LOG2E, 1.4e-45f);
}
// The factor that takes sums against m1 to m; 0 where m has seen nothing.
__device__ __forceinline__ float ref_factor(float m1, float m, float c2) {
  return m > -__builtin_inff() ? __builtin_amdgcn_exp2f((m1 - m) * c2) : 0.0f;
}

struct AttnArgs {
  void *out;
  float *lse;
  const void *q;
  size_t out_stride, q_stride;
  const int *seqs, *starts;
  const float *sink;
  // shared work only: outputs not yet divided [workgroup][2][ROWS * D] in the
  // waves' layout, their rows' (m, l) [workgroup][2][ROWS], the position of
  // each item's first stage, and the number of all stages
  float *part;
  float2 *stat;
  long *first;
  int layer, heads, group, n_seqs, n_tokens, max_q, max_kv, window, f32;
  int halve;  // queries are halved, scale is doubled
  int tiles, groups;  // groups: workgroups that share the stages, or 0: one per item
  float scale;
};

// Row waves RW (32 rows each) and, with fewer than 4, KW = 4 / RW waves that
// share a stage's tokens.
constexpr int at_max(int a, int b) { return a > b ? a : b; }
constexpr int at_min(int a, int b) { return a < b ? a : b; }
template <int D, bool SHARED, bool FP8, int RW>
struct Cfg {
  static constexpr int KW = 4 / RW, TT = 32 * KW, ROWS = 32 * RW;
  static constexpr int NP = D / 32;  // output tiles
  static constexpr int KB = TT * 2 * D, M = SHARED ? 1 : 2, STAGE = KB * M;  // BF16 rows
  // E4M3: codes, then scale codes, as they lie in the page
  static constexpr int CODES = TT * D, SCALES = TT * D / 64, RAW = M * (CODES + SCALES);
  // LDS: all of it for one workgroup per CU where the accumulators take the
  // registers (D >= 256) or a stage is long, else half
  static constexpr int CAP = (D <= 128 && (RW > 1 || (FP8 && D == 64)) ? 68 : 134) * 1024;
  static constexpr bool OK = 2 * STAGE <= CAP || (FP8 && STAGE + 2 * RAW <= CAP);
  // E4M3: two BF16 stages (the next one is converted while this one is
  // multiplied) where three stages of codes still fit beside them
  static constexpr bool TWICE = FP8 && 2 * STAGE + 3 * RAW <= CAP;
  static constexpr int NTILE = FP8 ? (TWICE ? 2 : 1) : at_min(4, CAP / STAGE);
  static constexpr int NRAW = FP8 ? at_min(4, (CAP - NTILE * STAGE) / RAW) : 0;
  static constexpr int RING = FP8 ? NRAW : NTILE;  // stages that direct loads fill
  // direct loads per wave and stage
  static constexpr int PER = FP8 ? M * (at_max(1, CODES / 4096) + at_max(1, TT / 64))
                                 : STAGE / 4096;
  // what the other waves of its rows hand a wave at the end: their parts of
  // its tiles; then every wave's (m, l). 0 with one wave per row.
  static constexpr int NO = at_max(1, NP / KW);  // tiles that a wave ends up with, if any
  static constexpr int PART = (KW - 1) * NO * 4096, JOIN = KW > 1 ? 4 * PART + 2048 : 0;
  static constexpr int LDS = at_max(NTILE * STAGE + NRAW * RAW, JOIN);
  static_assert(!OK || RW < 4 || LDS >= ROWS * 2 * D, "the result's rows pass through LDS");
  // The next stage's loads go between the products (issued at once they hold up
  // the wave): of a full tile, bound by the products, between all of them;
  // with fewer rows, bound by the memory, between those of the first half.
  static constexpr int OVER = (RW == 4 ? 2 : 1) * (D / 16);
  static constexpr int WGS = LDS <= 80 * 1024 && D <= 128 ? 2 : 1;  // per CU
};

template <int D>
__device__ __forceinline__ int chunk_swizzle(int row) {
  return D >= 128 ? ((row & 7) << 1) | ((row >> 3) & 1)
                  : (((row >> 1) & 3) << 1) | ((row >> 3) & 1);
}

// First column of output tile dt's lower (half 0) or upper 16 rows: a tile's
// halves are 4 (D = 64: 2) groups of 16 columns apart, so that the transposing
// reads of lanes 0..15 and 16..31 use different banks.
template <int D>
__device__ __forceinline__ constexpr int dim_of(int dt, int half) {
  return D >= 128 ? 16 * (8 * (dt / 4) + dt % 4 + 4 * half) : 16 * (dt + 2 * half);
}

// One item: a tile of a sequence's rows of one kv head. Uniform.
struct Item {
  int b, kvh, seq, start, count, len, r0, nrows, lo, hi, clear, stages;
};
// Rows tile * ROWS .. of the b-th listed sequence; false: there are none.
// blocked: by an earlier refusal, which stays the only one reported.
template <int ROWS, int TT>
__device__ __forceinline__ bool attn_item(const DSV4GCache &C, const AttnArgs &a, int b, int tile,
                                          unsigned blocked, Item &it) {
  it.b = b;
  it.seq = a.seqs ? a.seqs[b] : b;
  it.start = a.starts[b];
  const long end = a.starts[b + 1];
  const long count = end - it.start;
  it.len = it.seq >= 0 && it.seq < C.n_seqs ? C.len[it.seq] : -1;
  if (it.start < 0 || end > a.n_tokens || count < 0 || count > a.max_q || it.len < count ||
      it.len > a.max_kv || it.len > (long)C.max_pages * C.page_size) {
    if (tile == 0 && !blocked) atomicOr(C.status, DSV4G_CACHE_LIST);
    return false;
  }
  it.count = (int)count;
  it.r0 = tile * ROWS;
  it.nrows = it.count * a.group;
  if (it.r0 >= it.nrows) return false;
  const int first = it.len - it.count + it.r0 / a.group;
  it.hi = it.len - it.count + (min(it.r0 + ROWS, it.nrows) - 1) / a.group + 1;
  it.clear = a.window ? max(0, first - a.window + 1) : 0;  // the first token that is seen
  it.lo = it.clear & ~31;
  it.stages = (it.hi - it.lo + TT - 1) / TT;
  return true;
}

// Values that are the same in every lane, in scalar registers: the compiler
// would else keep what came through LDS or a vector load, and all that is
// computed from it, in vector registers.
__device__ __forceinline__ int one(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long one(long x) {
  return (long)(((uint64_t)(uint32_t)one((int)(x >> 32)) << 32) | (uint32_t)one((int)x));
}
__device__ __forceinline__ void one(Item &it) {
  int *f = &it.b;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(Item) / sizeof(int)); ++i) f[i] = one(f[i]);
}

// Shared work (fewer items than the chip has places for): the stages of all
// items in a row, items ordered by (sequence, tile), then kv head, are dealt
// out in equal runs, so that long and short sequences fill every workgroup
// alike. Workgroup w takes stages [w T / W, (w + 1) T / W). Between two items
// lie AT_START stages with no work: what it costs a workgroup to end one item
// and begin another, so that those which do have fewer stages (64 sequences of
// 130 to 8100 E4M3 tokens: 90 us with 0, 68, 63 and 64 with 3, 6 and 10; with
// equal lengths up to 3% lost).
constexpr int AT_START = 6;
__device__ __forceinline__ int shared_groups(const AttnArgs &a, long total) {
  return (int)(total < a.groups ? total : a.groups);
}
__device__ __forceinline__ long share_begin(long total, int groups, int w) {
  return total * w / groups;
}
__device__ __forceinline__ int share_of(long total, int groups, long at) {
  return (int)(((at + 1) * groups - 1) / total);
}

// Where this workgroup's run begins: every thread counts the stages of some
// (sequence, tile) pairs, one of them finds the place.
struct Place {
  long at, end, total;
  int pair, kvh, stage;
  Item it;  // of the first pair
};
template <int ROWS, int TT>
__device__ __forceinline__ void attn_place(const DSV4GCache &C, const AttnArgs &a,
                                           unsigned blocked, Place &p) {
  __shared__ long s_sum[4];
  __shared__ int s_at[3];
  __shared__ Item s_item;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const int pairs = a.n_seqs * a.tiles, per = (pairs + 255) / 256;
  const int j0 = min(pairs, tid * per), j1 = min(pairs, j0 + per);
  long mine = 0;
  Item it;
  for (int j = j0; j < j1; ++j)
    if (attn_item<ROWS, TT>(C, a, j / a.tiles, j % a.tiles, blocked, it))
      mine += it.stages + AT_START;
  long x = mine;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) s_sum[wave] = x;
  if (tid == 0) s_at[0] = pairs;  // no place
  __syncthreads();
  long before = x - mine, total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    before += w < wave ? s_sum[w] : 0;
    total += s_sum[w];
  }
  before *= C.kv_heads;
  p.total = one(total * C.kv_heads - (total ? AT_START : 0));  // none behind the last item
  const int groups = shared_groups(a, p.total);
  p.at = p.end = 0;
  if ((int)blockIdx.x >= groups) return;
  p.at = share_begin(p.total, groups, blockIdx.x);
  p.end = share_begin(p.total, groups, blockIdx.x + 1);
  if (p.at >= before && p.at < before + mine * C.kv_heads)
    for (int j = j0; j < j1; ++j)
      if (attn_item<ROWS, TT>(C, a, j / a.tiles, j % a.tiles, blocked, it)) {
        const int span = it.stages + AT_START;
        const long all = (long)span * C.kv_heads;
        if (p.at < before + all) {
          s_at[0] = j;
          s_at[1] = (int)((p.at - before) / span);
          s_at[2] = (int)((p.at - before) % span);
          s_item = it;
          break;
        }
        before += all;
      }
  __syncthreads();
  p.pair = __builtin_amdgcn_readfirstlane(s_at[0]);
  p.kvh = __builtin_amdgcn_readfirstlane(s_at[1]);
  p.stage = __builtin_amdgcn_readfirstlane(s_at[2]);
  p.it = s_item;
}

// A value whose uses are computed again each time: addresses derived from it
// would else be kept in registers around the loop over the stages.
__device__ __forceinline__ void fresh(int &x) { asm volatile("" : "+v"(x)); }

// Direct loads to LDS, 16 or 4 bytes per lane (lane l's at `to` + its size *
// l). In inline asm: they have no output register, and the compiler would make
// every later LDS read wait for all of them; wait_loads() and the barrier
// order them instead (what they write is read behind the next ones only).
__device__ __forceinline__ void lds_load16(uint32_t to, uint32_t at, I4 rsrc) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               ::"s"(to), "v"(at), "s"(rsrc));
}
__device__ __forceinline__ void lds_load4(uint32_t to, uint32_t at, I4 rsrc) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               ::"s"(to), "v"(at), "s"(rsrc));
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// What the waves wrote to LDS is there for all of them. Not __syncthreads():
// that waits for the loads of later stages, too.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Brings stages of an item to LDS, PER loads per wave: begin() looks at the
// pages, load(k) issues one. A stage behind the last (`st` < 0) is loads that
// bring zeros, so that the loop has no branch and its waits count alike.
// The pages of a stage are looked up one stage ahead.
constexpr uint32_t AT_OUT = 0x7FFFFFFFu;  // an offset behind any page: zeros
template <int D, bool SHARED, bool FP8, int RW>
struct Loader {
  typedef Cfg<D, SHARED, FP8, RW> F;
  // Rows: a wave brings a quarter of the tokens, NG groups of TG (one page
  // each), TB per load. E4M3 with narrow heads: 16 tokens are one load, which
  // two waves then bring alike.
  static constexpr int TT = F::TT, TW = TT / 4, M = F::M;
  static constexpr int TB = FP8 ? 1024 / D : 512 / D;
  static constexpr int TG = at_max(at_min(16, TW), TB), NG = at_max(1, TW / TG);
  static constexpr int ROWS_PER = NG * (TG / TB);
  // Scale codes: 16 tokens per load, 4 bytes per lane
  static constexpr int NS = FP8 ? at_max(1, TT / 64) : 0;
  static_assert(F::PER == M * (ROWS_PER + NS), "loads of a stage");
  int page[NG], spage[at_max(1, NS)];  // of the next stage
  I4 rsrc[NG], srsrc[at_max(1, NS)];   // of this one
  int t0;                              // its first token
  uint32_t lds;
  // This lane's offset from a load's first row. A load's rows are a multiple of
  // TB on, and the swizzle moves bits only, so that of row base + o is that of
  // base XOR that of o: a load costs a few instructions for its address. (All of
  // it computed per lane: a latent chunk 2% slower, 32 short sequences over 8 kv
  // heads 12%.)
  uint32_t lane_at;  // rows of less than a load, else it is 16 * lane

  __device__ __forceinline__ void init(int lane) {
    const int o = lane * TB / 64;
    lane_at = o * (2 * D) + 16u * ((lane % (D / 8)) ^ chunk_swizzle<D>(o));
    if constexpr (!FP8 && TB > 1) asm volatile("" : "+v"(lane_at));
  }

  __device__ __forceinline__ int row_group(int wave, int g) const {
    return (wave * NG + g) * TG % TT;
  }
  __device__ __forceinline__ int scale_group(int wave, int k) const {
    return (wave * NS + k) * 16 % TT;
  }
  __device__ __forceinline__ int page_of(const DSV4GCache &C, const CacheGeom &G, const Item &it,
                                         int t, int n) const {
    if (t >= it.hi || t + n <= it.clear) return -2;  // nothing is needed of it
    const int *cell = C.table + (size_t)it.seq * C.max_pages + (t >> G.shift);
    // written by earlier kernels only: a scalar load
    const int page = *(const __attribute__((address_space(4))) int *)cell;
    return page < 0 || page >= C.n_pages ? -1 : page;
  }
  __device__ __forceinline__ void look(const DSV4GCache &C, const CacheGeom &G, const Item &it,
                                       int st, int wave) {
#pragma unroll
    for (int g = 0; g < NG; ++g)
      page[g] = page_of(C, G, it, it.lo + st * TT + row_group(wave, g), TG);
#pragma unroll
    for (int k = 0; k < NS; ++k)
      spage[k] = page_of(C, G, it, it.lo + st * TT + scale_group(wave, k), 16);
  }
  __device__ __forceinline__ I4 page_rsrc(const DSV4GCache &C, const CacheGeom &G, int layer,
                                          int page, bool live) const {
    const uint64_t p = (uint64_t)(uintptr_t)C.pages +
                       ((uint64_t)layer * C.n_pages + (page < 0 ? 0 : page)) * G.page_bytes;
    return I4{(int)(uint32_t)p, (int)(uint32_t)(p >> 32),
              live && page >= 0 ? (int)G.page_bytes : 0, 0x00020000};
  }
  __device__ __forceinline__ void begin(const DSV4GCache &C, const CacheGeom &G, const AttnArgs &a,
                                        const Item &it, int st, bool live, uint32_t to,
                                        int wave) {
    lds = to;
    t0 = it.lo + st * TT;
    bool bad = false;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      bad |= page[g] == -1;
      rsrc[g] = page_rsrc(C, G, a.layer, page[g], live);
    }
#pragma unroll
    for (int k = 0; k < NS; ++k) srsrc[k] = page_rsrc(C, G, a.layer, spage[k], live);
    if (live && bad && threadIdx.x % 64 == 0) atomicOr(C.status, DSV4G_CACHE_PAGE);
    look(C, G, it, st + 1, wave);
  }
  template <int K>
  __device__ __forceinline__ void load(const DSV4GCache &C, const CacheGeom &G, const Item &it,
                                       int wave, int lane) const {
    constexpr int m = K % M, i = K / M;
    const int head = it.kvh * C.page_size, mask = C.page_size - 1;
    if constexpr (i < ROWS_PER) {
      constexpr int g = i / (TG / TB), j = i % (TG / TB);
      const int tl0 = row_group(wave, g);
      const int slot = head + ((t0 + tl0) & mask) + j * TB, tok = t0 + tl0 + j * TB;
      constexpr int ROW = FP8 ? D : 2 * D;  // bytes
      const uint32_t to = lds + (tl0 + j * TB) * ROW + m * (FP8 ? F::CODES + F::SCALES : F::KB);
      fresh(lane);
      uint32_t v = FP8 || TB == 1 ? 16u * lane : lane_at;
      if (!FP8) v ^= 16u * chunk_swizzle<D>(tl0 + j * TB);
      const uint32_t base = (uint32_t)slot * ROW + (m ? G.v_off : 0);
      if constexpr (TB == 1) {  // the whole load is one token
        v += tok < it.hi && tok >= it.clear ? base : AT_OUT;
      } else {
        const uint32_t o = lane * TB / 64;
        v = o + (uint32_t)(tok - it.clear) < (uint32_t)(it.hi - it.clear) ? v + base : AT_OUT;
      }
      lds_load16(to, v, rsrc[g]);
    } else {
      fresh(lane);
      constexpr int S = D / 64, LANES = 4 * S;  // codes of a token, lanes of a load
      const int tl0 = scale_group(wave, i - ROWS_PER);
      const int slot = head + ((t0 + tl0) & mask), tok = t0 + tl0 + 4 * lane / S;
      constexpr int SPAN = S < 4 ? 4 / S : 1;   // tokens of a lane's 4 bytes
      const bool in = tok < it.hi && tok + SPAN > it.clear;
      const uint32_t v = (uint32_t)slot * S + 4 * lane + (m ? G.vs_off : G.ks_off);
      if (lane < LANES)
        lds_load4(lds + F::CODES + tl0 * S + m * (F::CODES + F::SCALES), in ? v : AT_OUT,
                  srsrc[i - ROWS_PER]);
    }
  }
  // The loads that belong to step S of N.
  template <int S, int N>
  __device__ __forceinline__ void step(const DSV4GCache &C, const CacheGeom &G, const Item &it,
                                       int wave, int lane) const {
    constexpr int K0 = (S * F::PER + N - 1) / N, K1 = ((S + 1) * F::PER + N - 1) / N;
    each<K1 - K0>([&](auto k) { load<K0 + k>(C, G, it, wave, lane); });
  }
};

// E4M3 codes of a stage as BF16 rows, 8 codes (one chunk of a row) per thread
// and step: a code times its power of two is exact in BF16. Step p is T = 2048
// / D rows on, so all addresses are the thread's own XOR and plus constants.
// Codes that were not loaded are 0, beside whatever scale code the page holds:
// 255 counts as 254, so that they stay 0.
template <int D, bool SHARED, int TT>
__device__ __forceinline__ void convert(uint32_t raw, uint32_t tile, int tid) {
  constexpr int CODES = TT * D, SCALES = CODES / 64, T = 2048 / D, P = TT / T, B = P < 4 ? P : 4;
  static_assert(P >= 1, "a stage is a step or more");
  fresh(tid);
  const int row = tid * 8 / D;
  const uint32_t from = raw + 8 * tid, scale = raw + CODES + tid / 8;
  const uint32_t to = tile + row * (2 * D) + 16 * ((tid * 8 % D / 8) ^ chunk_swizzle<D>(row));
  constexpr int M = SHARED ? 1 : 2, N = M * P / B;  // batches
  U2 u[2][B];
  uint32_t s[2][B];
  auto read = [&](auto n) {
    constexpr uint32_t fm = n * B / P * (CODES + SCALES), p0 = n * B % P;
#pragma unroll
    for (int i = 0; i < B; ++i) {
      u[n % 2][i] = DSV4_LDS(U2, from + fm + (p0 + i) * 2048);
      s[n % 2][i] = DSV4_LDS(uint8_t, scale + fm + (p0 + i) * 32);
    }
  };
  read(std::integral_constant<int, 0>{});
  each<N>([&](auto n) {  // the next batch's reads under this one's arithmetic
    if constexpr (n + 1 < N) read(std::integral_constant<int, n + 1>{});
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int p = n * B % P + i;
      const float f = u2f(min(s[n % 2][i], 254u) << 23);
      auto two = [&](uint32_t w, auto hi) {
        return __builtin_bit_cast(
            uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, f, decltype(hi)::value));
      };
      const std::false_type lo;
      const std::true_type hi;
      const U2 w = u[n % 2][i];
      const U4 y = {two(w.x, lo), two(w.x, hi), two(w.y, lo), two(w.y, hi)};
      // the swizzle of row + p T against the row's own
      const uint32_t x = T == 4 ? 16 * (8 * (p & 1) + (p / 2 & 1)) : T == 8 ? 16 * (p & 1) : 0;
      DSV4_LDS(U4, (to ^ x) + n * B / P * 2 * CODES + p * T * (2 * D)) = y;
    }
    __builtin_amdgcn_sched_barrier(0);
  });
}

__device__ __forceinline__ float swap_max(float v) {  // with the other half of the wave
  const auto r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return fmaxf(u2f(r[0]), u2f(r[1]));
}
__device__ __forceinline__ float swap_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return u2f(r[0]) + u2f(r[1]);
}

// LDS addresses. Rows are multiples of 128 bytes (256 where D >= 128), so the
// chunk's XOR acts on address bits that hold nothing else, and every read is
// the lane's one address XOR a constant plus a constant.
// First product: row lane % 32, columns 16 s + 8 h .. + 7.
template <int D>
__device__ __forceinline__ uint32_t k_at(int lane) {
  const int row = lane % 32;
  return row * (2 * D) + 16 * ((lane / 32) ^ chunk_swizzle<D>(row));
}
template <int D>
__device__ __forceinline__ Bf8 read_k(uint32_t at, int s) {
  return DSV4_LDS(Bf8, (at ^ (32 * (s % 8))) + 256 * (s / 8));
}

// Second product: 8 tokens of one column per lane. K-step u of the tile takes
// tokens 16 u + 4 h + {0..3} and those 8 on (h: the lane's half), the order in
// which the scores' accumulators hold them; the transposing read gives four
// tokens of the column to a lane whose 16 neighbours' addresses cover 4 rows
// of 16 columns.
template <int D>
__device__ __forceinline__ uint32_t v_at(int lane) {
  const int row = 4 * (lane / 32) + lane % 16 / 4;
  const int c = dim_of<D>(0, lane / 16 % 2) / 8 + lane % 4 / 2;
  return row * (2 * D) + 16 * (c ^ chunk_swizzle<D>(row)) + 8 * (lane % 2);
}
template <int D>
__device__ __forceinline__ Bf8 read_vt(uint32_t at, int u, int dt) {
  U4 r;
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    const uint32_t x = D >= 128 ? 32 * (dt % 4) : 32 * dt;
    const uint32_t p = (at ^ (x + 16 * v)) + (16 * u + 8 * v) * (2 * D) +
                       (D >= 128 ? 256 * (dt / 4) : 0);
    const auto t = __builtin_bit_cast(
        uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   (__attribute__((address_space(3))) S4 *)(uintptr_t)p));
    r[2 * v] = t.x;
    r[2 * v + 1] = t.y;
  }
  return __builtin_bit_cast(Bf8, r);
}

// LDS reads ahead of their product (even): a read's latency is about four
// products; 6 measured the same within 1%, 8 has too few registers left (5%
// slower at decode).
constexpr int AT_AHEAD = 4;

// An output tile moved between the accumulation registers, where it stays in
// the loop, and the vector registers that arithmetic needs: one tile at a
// time, or the copies of all of them take the registers of everything else.
__device__ __forceinline__ F16v tile_out(const F16v &o) {
  F16v y = o;
  asm volatile("" : "+v"(y));
  return y;
}
__device__ __forceinline__ void tile_in(F16v &o, F16v y) {
  asm volatile("" : "+a"(y));
  o = y;
  __builtin_amdgcn_sched_barrier(0);
}

// Rows of the result: fp32 accumulators of output tile dt times f, at columns
// dim_of(dt, half) + 8 (g % 2) + 4 h + 0..3 for g = 0..3 (half = g / 2).
template <int D>
__device__ __forceinline__ void store_tile(const AttnArgs &a, size_t row_at, int dt, int h,
                                           const F16v &o, float f) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const size_t at = row_at + dim_of<D>(dt, g / 2) + 8 * (g % 2) + 4 * h;
    const float y[4] = {o[4 * g] * f, o[4 * g + 1] * f, o[4 * g + 2] * f, o[4 * g + 3] * f};
    const uint2 b = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
    if (a.f32)
      *(float4 *)((float *)a.out + at) =
          make_float4(u2f(b.x << 16), u2f(b.x & 0xFFFF0000u), u2f(b.y << 16),
                      u2f(b.y & 0xFFFF0000u));
    else
      *(uint2 *)((uint16_t *)a.out + at) = b;
  }
}

// The same for a whole tile of 32 rows (n of them live, lane % 32's at
// `row_at`), through LDS: a lane holds 8 bytes of its row at a time, which would
// be partial writes of 32 rows per store; so the wave writes its rows to its
// part of LDS, chunks swizzled as in the stages, and reads them back along the
// rows, whole lines per store (128 rows of 512: 7.5 -> 5.3 us with every
// workgroup storing at once, 6 TB/s). Tiles of fewer rows are stored as they are:
// most of theirs are parts, which need no such thing.
template <int D>
__device__ __forceinline__ void store_rows(const AttnArgs &a, size_t row_at, int n, uint32_t lds,
                                           int lane, const F16v *o, float f) {
  lds_barrier();  // every wave is done with the stages
  fresh(lane);
  const uint32_t to = lds + lane % 32 * (2 * D) + 16 * chunk_swizzle<D>(lane % 32) +
                      8 * (lane / 32);
  each<D / 32>([&](auto d) {
    const F16v y = tile_out(o[d]);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint32_t c = dim_of<D>(d, g / 2) / 8 + g % 2;
      DSV4_LDS(U2, to ^ (16 * c)) = U2{pack_bf16(y[4 * g] * f, y[4 * g + 1] * f),
                                             pack_bf16(y[4 * g + 2] * f, y[4 * g + 3] * f)};
    }
    __builtin_amdgcn_sched_barrier(0);
  });
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  constexpr int CH = D / 8, RI = 64 / CH;  // chunks of a row, rows per store
  constexpr int U = at_min(8, 32 / RI);    // stores at a time
  for (int i = 0; i < 32; i += RI * U) {
    U4 x[U];
    size_t at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = i + u * RI + lane / CH;
      x[u] = DSV4_LDS(U4, lds + r * (2 * D) + 16 * (lane % CH ^ chunk_swizzle<D>(r)));
      at[u] = __shfl(row_at, r, 64) + lane % CH * 8;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * RI + lane / CH >= n) continue;
      if (a.f32) {
        float4 *p = (float4 *)((float *)a.out + at[u]);
        p[0] = make_float4(u2f(x[u][0] << 16), u2f(x[u][0] & 0xFFFF0000u), u2f(x[u][1] << 16),
                           u2f(x[u][1] & 0xFFFF0000u));
        p[1] = make_float4(u2f(x[u][2] << 16), u2f(x[u][2] & 0xFFFF0000u), u2f(x[u][3] << 16),
                           u2f(x[u][3] & 0xFFFF0000u));
      } else {
        *(U4 *)((uint16_t *)a.out + at[u]) = x[u];
      }
    }
  }
}

// The denominator's reciprocal (0 where nothing was seen) and lse, with the
// head's sink joined. The sink's distance to m's score is taken by one fma: both
// may be large.
__device__ __forceinline__ float finish_row(const AttnArgs &a, int head, float m, float l,
                                            float *lse) {
  const float s = fmaxf(fabsf(a.scale), 1.4e-45f);
  float f = 1.0f, top = m * s;
  const float sink = a.sink ? a.sink[head] : -__builtin_inff();
  if (sink != -__builtin_inff()) {
    const float d = fmaf(m, s, -sink) * LOG2E;  // -inf where nothing was seen
    if (d > 0.0f) {
      l += exp2f(-d);
    } else {
      f = exp2f(d);
      l = l * f + 1.0f;
      top = sink;
    }
  }
  *lse = l != 0.0f ? top + log2f(l) * LN2 : -__builtin_inff();
  return l != 0.0f ? f / l : 0.0f;
}

template <int D, bool SHARED, bool FP8, int RW>
__global__ __launch_bounds__(256, (Cfg<D, SHARED, FP8, RW>::WGS)) void k_attn(DSV4GCache C,
                                                                            CacheGeom G,
                                                                            AttnArgs a) {
  typedef Cfg<D, SHARED, FP8, RW> F;
  constexpr int TT = F::TT, STAGE = F::STAGE, RING = F::RING, NP = F::NP, KS = D / 16;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[F::LDS];
  __shared__ uint32_t s_odd[F::KW];  // tokens of a stage with something not finite
  const unsigned bad = *C.status;
  const int tid = threadIdx.x, lane = tid % 64, h = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int rw = wave % RW, kw = wave / RW;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
  const uint32_t raw0 = lds0 + F::NTILE * STAGE;  // the ring of codes
  const uint32_t ring0 = FP8 ? raw0 : lds0;
  constexpr int RSTEP = FP8 ? F::RAW : STAGE;
  constexpr int R = AT_AHEAD;
  if (tid < F::KW) s_odd[tid] = 0;

  Place w;
  if (a.groups) {
    attn_place<F::ROWS, TT>(C, a, bad, w);
  } else {
    int id = blockIdx.x;
    w.kvh = id % C.kv_heads;
    id /= C.kv_heads;
    // of each sequence the longest ranges first
    w.pair = id % a.n_seqs * a.tiles + a.tiles - 1 - id / a.n_seqs;
    w.stage = 0;
    w.at = 0;
    w.end = 1;
  }
  if (bad) return;
  // One segment after the other: a run of stages of one item. (The pairs end with
  // the run, unless something else changes the lengths meanwhile.)
  for (bool first = true; w.at < w.end && w.pair < a.n_seqs * a.tiles; first = false) {
    Item it;
    if (first && a.groups) {
      it = w.it;  // looked up already
    } else if (!attn_item<F::ROWS, TT>(C, a, w.pair / a.tiles, w.pair % a.tiles, 0, it)) {
      if (!a.groups) return;
      ++w.pair;  // no rows here
      continue;
    }
    it.kvh = w.kvh;
    one(it);
    const int s0 = w.stage;
    if (s0 >= it.stages) {  // between this item and the next
      w.at += it.stages + AT_START - s0;
      w.stage = 0;
      if (++w.kvh == C.kv_heads) {
        w.kvh = 0;
        ++w.pair;
      }
      continue;
    }
    const int s1 = one(a.groups ? (int)min((long)it.stages, s0 + w.end - w.at) : it.stages);
    if (a.groups) {
      if (s0 == 0 && tid == 0) {
        a.first[1 + (long)w.pair * C.kv_heads + it.kvh] = w.at;
        if (w.at == 0) a.first[0] = w.total;
      }
      w.at += s1 - s0 + AT_START;
      w.stage = 0;
      if (++w.kvh == C.kv_heads) {
        w.kvh = 0;
        ++w.pair;
      }
    } else {
      w.at = w.end;
    }
    // this lane's row (the last one again where there are fewer)
    const int wr0 = it.r0 + 32 * rw;
    const bool active = wr0 < it.nrows;
    const int r = min(wr0 + lane % 32, it.nrows - 1);
    const int tok = r / a.group, head = it.kvh * a.group + r % a.group;
    const int pos0 = it.len - it.count, pos = pos0 + tok;
    const int pmin = one(pos0 + min(wr0, it.nrows - 1) / a.group);
    const int pmax = one(pos0 + min(wr0 + 31, it.nrows - 1) / a.group);

    Loader<D, SHARED, FP8, RW> load;
    load.init(lane);
    load.look(C, G, it, s0, wave);
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) {
      load.begin(C, G, a, it, s0 + i, s0 + i < s1, ring0 + i * RSTEP, wave);
      load.template step<0, 1>(C, G, it, wave, lane);
    }

    // the query rows, once: columns 16 s + 8 h .. + 7 of row lane % 32; a
    // negative scale is taken by their sign
    Bf8 q[KS];
    {
      const size_t at = (size_t)(it.start + tok) * a.q_stride + (size_t)head * D + 8 * h;
      const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        U4 u;
        if (a.f32) {
          const float4 x = *(const float4 *)((const float *)a.q + at + 16 * s);
          const float4 y = *(const float4 *)((const float *)a.q + at + 16 * s + 4);
          u = U4{pack_bf16(x.x, x.y), pack_bf16(x.z, x.w), pack_bf16(y.x, y.y),
                 pack_bf16(y.z, y.w)};
        } else {
          u = *(const U4 *)((const uint16_t *)a.q + at + 16 * s);
        }
        if (a.halve) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            u[k] = pack_bf16(0.5f * u2f(u[k] << 16), 0.5f * u2f(u[k] & 0xFFFF0000u));
        }
        q[s] = __builtin_bit_cast(Bf8, u ^ sign);
      }
    }
    const float c2 = attn_c2(a.scale);

    F16v o[NP];
#pragma unroll
    for (int d = 0; d < NP; ++d) {
      F16v y;
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = 0.0f;
      tile_in(o[d], y);
    }
    float m = -__builtin_inff(), l = 0.0f;  // l: this half's tokens
    const uint32_t kat = lds0 + k_at<D>(lane) + 32 * kw * (2 * D);
    const uint32_t vat = lds0 + v_at<D>(lane) + 32 * kw * (2 * D) + (SHARED ? 0 : F::KB);
    // tokens that no row sees are not loaded; between these two are those that
    // some row of the workgroup sees and another does not
    const int shown = one(pos0 + it.r0 / a.group), hidden = it.hi - 1 - a.window;

    if (F::TWICE) {  // the first stage's rows
      wait_loads<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      convert<D, SHARED, TT>(raw0, lds0, tid);
    }
    for (int st = s0; st < s1; ++st) {
      const int i = st - s0;
      // what is read of the ring below (stage st; st + 1 where it is converted
      // ahead) is in LDS for every wave, and every wave is done with the stage
      // before st
      constexpr int AHEAD = F::TWICE ? 1 : 0;
      wait_loads<(RING - 2 - AHEAD) * F::PER>();
      lds_barrier();
      if (FP8 && !F::TWICE) {
        convert<D, SHARED, TT>(raw0 + i % RING * RSTEP, lds0, tid);
        lds_barrier();
      }
      const int next = st + RING - 1;
      load.begin(C, G, a, it, next, next < s1, ring0 + (i + RING - 1) % RING * RSTEP, wave);
      const uint32_t here = i % F::NTILE * STAGE;  // the stage's rows
      const int w0 = it.lo + st * TT;                 // the stage's tokens
      const int t0 = w0 + 32 * kw;                    // this wave's 32
      // 0 * NaN is NaN: where a token is hidden from some rows and not from
      // others, its values are cleared if they are not all finite (a row that
      // sees it is not finite then: by its score, or as below)
      uint32_t odd = 0;
      if (min(w0 + TT, it.hi) - 1 > shown || (a.window && max(w0, it.clear) <= hidden)) {
        constexpr int PT = 256 / TT, NC = D / 8 / PT;  // threads per token, chunks of each
        const int t = tid / PT;
        const uint32_t at = lds0 + here + (SHARED ? 0 : F::KB) + t * (2 * D) + tid % PT * 16;
        uint32_t big = 0;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          const U4 x = DSV4_LDS(U4, at + 16 * PT * j);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            big |= ((x[k] & 0x7F80u) == 0x7F80u) | ((x[k] & 0x7F800000u) == 0x7F800000u);
        }
        if (big) atomicOr(&s_odd[t / 32], 1u << (t % 32));
        lds_barrier();
        uint32_t any = 0;
#pragma unroll
        for (int k = 0; k < F::KW; ++k) any |= s_odd[k];
        odd = __builtin_amdgcn_readfirstlane(any) ? 1u : 0u;
      }
      // A wave whose rows see nothing of its 32 tokens computes weights of 0: a
      // branch around the products would have the compiler copy the
      // accumulators at its ends.
      Bf8 p0, p1;
      {
        F16v z;
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = 0.0f;
        const uint32_t at = kat + here;
        // LDS reads a few steps ahead of the products that take them; the order
        // is pinned, since the scheduler puts each read right in front of its
        // product
        __builtin_amdgcn_sched_barrier(0);
        Bf8 k[R];
#pragma unroll
        for (int s = 0; s < R && s < KS; ++s) k[s] = read_k<D>(at, s);
        __builtin_amdgcn_sched_barrier(0);
        each<KS>([&](auto s) {
          z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[s % R], q[s], z, 0, 0, 0);
          if constexpr (s + R < KS) k[s % R] = read_k<D>(at, s + R);
          load.template step<s, F::OVER>(C, G, it, wave, lane);
          __builtin_amdgcn_sched_barrier(0);
        });
        // token of z[i]: t0 + 8 (i / 4) + 4 h + i % 4
        const bool mask = t0 + 31 > pmin || (a.window && t0 <= pmax - a.window);
        if (mask) {
          const int high = pos - t0 - 4 * h, low = a.window ? high - a.window : -64;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int at = 8 * (i / 4) + i % 4;
            z[i] = at <= high && at > low ? z[i] : -__builtin_inff();
          }
        }
        float mx = fmaxf(fmaxf(z[0], z[1]), z[2]);
#pragma unroll
        for (int i = 3; i < 15; i += 2) mx = fmaxf(fmaxf(mx, z[i]), z[i + 1]);
        mx = fmaxf(mx, z[15]);
        mx = swap_max(mx);
        m = i ? m : mx;  // nothing to rescale yet
        if (__any((mx - m) * c2 > AT_GROW)) {
          const float M = fmaxf(m, mx);
          const float f = ref_factor(m, M, c2);
          m = M;
          l *= f;
#pragma unroll
          for (int d = 0; d < NP; ++d) {
            F16v y = tile_out(o[d]);
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] *= f;
            tile_in(o[d], y);
          }
        }
        const float mu = m > -__builtin_inff() ? m : 0.0f;
        U4 b0, b1;
        float part[4] = {};
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float x0 = __builtin_amdgcn_exp2f((z[i] - mu) * c2);
          const float x1 = __builtin_amdgcn_exp2f((z[i + 1] - mu) * c2);
          part[i / 2 % 4] += x0 + x1;
          if (i < 8) b0[i / 2] = pack_bf16(x0, x1);
          else b1[i / 2 - 4] = pack_bf16(x0, x1);
        }
        l += (part[0] + part[1]) + (part[2] + part[3]);
        p0 = __builtin_bit_cast(Bf8, b0);
        p1 = __builtin_bit_cast(Bf8, b1);
      }
      if (F::TWICE && st + 1 < s1)
        convert<D, SHARED, TT>(raw0 + (i + 1) % RING * RSTEP, lds0 + (i + 1) % 2 * STAGE, tid);
      if (odd) {
        lds_barrier();  // every wave has its scores
        const int t = tid % TT;
        if (s_odd[t / 32] >> (t % 32) & 1) {
          const uint32_t at = lds0 + here + (SHARED ? 0 : F::KB) + t * (2 * D);
          for (int j = tid / TT; j < D / 8; j += 256 / TT)
            DSV4_LDS(U4, at + 16 * j) = U4{0, 0, 0, 0};
        }
        for (uint32_t left = s_odd[kw]; left; left &= left - 1) {
          const int t = t0 + __builtin_ctz(left);
          if (t <= pos && (!a.window || t > pos - a.window)) l = __builtin_nanf("");
        }
        lds_barrier();
        if (tid < F::KW) s_odd[tid] = 0;  // read again two barriers on at the earliest
      }
      {
        const uint32_t at = vat + here;
        __builtin_amdgcn_sched_barrier(0);
        Bf8 v[R];
#pragma unroll
        for (int s = 0; s < R && s < KS; ++s) v[s] = read_vt<D>(at, s / NP, s % NP);
        __builtin_amdgcn_sched_barrier(0);
        each<KS>([&](auto s) {  // each output tile's first k-step, then each one's second
          o[s % NP] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[s % R], s < NP ? p0 : p1,
                                                              o[s % NP], 0, 0, 0);
          if constexpr (s + R < KS) v[s % R] = read_vt<D>(at, (s + R) / NP, (s + R) % NP);
          if constexpr (F::OVER > KS) load.template step<KS + s, F::OVER>(C, G, it, wave, lane);
          __builtin_amdgcn_sched_barrier(0);
        });
      }
    }
    wait_loads<0>();  // the loads behind the last stage are done with LDS
    l = swap_sum(l);

    // The waves that shared the rows: a wave hands the others their share of
    // its output tiles through LDS and takes theirs of its own, NO tiles.
    constexpr int KW = F::KW, NO = F::NO;
    float f = 1.0f;                          // its own outputs' factor
    if constexpr (KW > 1) {
      float2 *xs = (float2 *)(lds + 4 * F::PART);
      __syncthreads();
      each<NP>([&](auto d) {
        if (d / NO != kw) {  // tile d: to wave d / NO, from this one
          const F16v y = tile_out(o[d]);
          const int slot = d % NO * (KW - 1) + (kw > d / NO ? kw - 1 : kw);
          float4 *x = (float4 *)(lds + (d / NO * RW + rw) * F::PART) + slot * 256;
#pragma unroll
          for (int g = 0; g < 4; ++g)
            x[g * 64 + lane] =
                make_float4(y[4 * g], y[4 * g + 1], y[4 * g + 2], y[4 * g + 3]);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      xs[wave * 64 + lane] = make_float2(m, l);
      __syncthreads();
      float M = m;
#pragma unroll
      for (int k = 0; k < KW; ++k) M = fmaxf(M, xs[(k * RW + rw) * 64 + lane].x);
      f = ref_factor(m, M, c2);
      float fk[KW];
      l = 0.0f;
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        const float2 s = xs[(k * RW + rw) * 64 + lane];
        fk[k] = ref_factor(s.x, M, c2);
        l += s.y * fk[k];
      }
      m = M;
      each<NP>([&](auto d) {
        if (d / NO == kw) {
          F16v y = tile_out(o[d]);
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] *= f;
#pragma unroll
          for (int k = 0; k < KW; ++k) {
            if (k == kw) continue;
            const int slot = d % NO * (KW - 1) + (k > kw ? k - 1 : k);
            const float4 *x = (const float4 *)(lds + wave * F::PART) + slot * 256;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float4 p = x[g * 64 + lane];
              y[4 * g] += p.x * fk[k];
              y[4 * g + 1] += p.y * fk[k];
              y[4 * g + 2] += p.z * fk[k];
              y[4 * g + 3] += p.w * fk[k];
            }
          }
          tile_in(o[d], y);
        }
      });
    }
    float rinv = 0.0f;
    if (active && wr0 + lane % 32 < it.nrows) {
      if (s0 > 0 || s1 < it.stages) {
        const size_t slot = 2 * (size_t)blockIdx.x + (s0 == 0);  // the run's last item, or its first
        float4 *to = (float4 *)(a.part + (slot * F::ROWS + 32 * rw) * D);
        each<NP>([&](auto d) {
          if (KW == 1 || d / NO == kw) {
            const F16v y = tile_out(o[d]);
#pragma unroll
            for (int g = 0; g < 4; ++g)
              to[(4 * d + g) * 64 + lane] =
                  make_float4(y[4 * g], y[4 * g + 1], y[4 * g + 2], y[4 * g + 3]);
          }
          __builtin_amdgcn_sched_barrier(0);
        });
        if (kw == 0 && h == 0) a.stat[slot * F::ROWS + 32 * rw + lane] = make_float2(m, l);
      } else {
        float lse;
        const float r = finish_row(a, head, m, l, &lse);
        const size_t row = (size_t)(it.start + tok);
        if constexpr (KW == 1)
          rinv = r;
        else
          each<NP>([&](auto d) {
            if (d / NO == kw)
              store_tile<D>(a, row * a.out_stride + (size_t)head * D, d, h, tile_out(o[d]), r);
            __builtin_amdgcn_sched_barrier(0);
          });
        if (a.lse && kw == 0 && h == 0) a.lse[row * a.heads + head] = lse;
      }
    }
    if constexpr (KW == 1) {
      if (s0 == 0 && s1 == it.stages)
        store_rows<D>(a, (size_t)(it.start + tok) * a.out_stride + (size_t)head * D,
                      it.nrows - wr0, lds0 + wave * (32 * 2 * D), lane, o, rinv);
    }
    if (!a.groups) return;
    __syncthreads();  // the stages' LDS is free again
  }
}

// Joins the parts of every item that several workgroups shared: a workgroup
// per output tile of a row wave, whose four waves take every fourth part (one
// wave for all of them took 107 us for the 251 parts of one sequence of 16000;
// that whole call now takes 46). Bound by latency (5.5 us for 28 parts), then by the parts' bytes
// (11 us for the 33 MB of 64 latent sequences).
template <int D, int RW>
__global__ __launch_bounds__(256) void k_attn_join(DSV4GCache C, AttnArgs a) {
  constexpr int TT = 32 * (4 / RW), ROWS = 32 * RW, NP = D / 32;
  __shared__ float4 s_o[3][4][64];
  __shared__ float2 s_l[3][64];
  const unsigned bad = *C.status;
  const int lane = threadIdx.x % 64, h = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  int id = blockIdx.x;
  const int d = id % NP;
  id /= NP;
  const int rw = id % RW;
  id /= RW;  // (sequence, tile), kv head
  const int kvh = id % C.kv_heads, pair = id / C.kv_heads;
  const long total = a.first[0], at = a.first[1 + id];
  Item it;
  if (bad || !attn_item<ROWS, TT>(C, a, pair / a.tiles, pair % a.tiles, 0, it)) return;
  const int groups = shared_groups(a, total);
  if (groups <= 0) return;
  const int w0 = max(0, share_of(total, groups, at));
  const int w1 = min(groups - 1, share_of(total, groups, at + it.stages - 1));
  if (w0 >= w1) return;
  const int r = it.r0 + 32 * rw + lane % 32;
  const bool live = r < it.nrows;  // parts hold such rows only
  // the first workgroup's part is its run's last, the others' their first
  auto slot = [&](int w) { return (2 * (size_t)w + (w == w0)) * ROWS + 32 * rw; };
  const float c2 = attn_c2(a.scale);
  float m = -__builtin_inff(), l = 0.0f;
  F16v o;
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = 0.0f;
  constexpr int U = 4;  // parts in flight
  for (int w = w0 + wave; w <= w1; w += 4 * U) {
    float2 s[U];
    float4 x[U][4];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      s[k] = make_float2(-__builtin_inff(), 0.0f);
#pragma unroll
      for (int g = 0; g < 4; ++g) x[k][g] = make_float4(0, 0, 0, 0);
      if (live && w + 4 * k <= w1) {
        const size_t at = slot(w + 4 * k);
        s[k] = a.stat[at + lane % 32];
#pragma unroll
        for (int g = 0; g < 4; ++g) x[k][g] = ((const float4 *)(a.part + at * D))[(4 * d + g) * 64 + lane];
      }
    }
    float M = m;
#pragma unroll
    for (int k = 0; k < U; ++k) M = fmaxf(M, s[k].x);
    const float f = ref_factor(m, M, c2);
    m = M;
    l *= f;
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] *= f;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const float p = ref_factor(s[k].x, M, c2);
      l += s[k].y * p;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        o[4 * g] += x[k][g].x * p;
        o[4 * g + 1] += x[k][g].y * p;
        o[4 * g + 2] += x[k][g].z * p;
        o[4 * g + 3] += x[k][g].w * p;
      }
    }
  }
  if (wave) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      s_o[wave - 1][g][lane] = make_float4(o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]);
    s_l[wave - 1][lane] = make_float2(m, l);
  }
  __syncthreads();
  if (wave || !live) return;
  float M = m;
#pragma unroll
  for (int k = 0; k < 3; ++k) M = fmaxf(M, s_l[k][lane].x);
  const float f0 = ref_factor(m, M, c2);
  l *= f0;
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] *= f0;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const float2 s = s_l[k][lane];
    const float p = ref_factor(s.x, M, c2);
    l += s.y * p;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 x = s_o[k][g][lane];
      o[4 * g] += x.x * p;
      o[4 * g + 1] += x.y * p;
      o[4 * g + 2] += x.z * p;
      o[4 * g + 3] += x.w * p;
    }
  }
  const int tok = r / a.group, head = kvh * a.group + r % a.group;
  float lse;
  const float f = finish_row(a, head, M, l, &lse);
  const size_t row = (size_t)(it.start + tok);
  store_tile<D>(a, row * a.out_stride + (size_t)head * D, d, h, o, f);
  if (a.lse && h == 0 && d == 0) a.lse[row * a.heads + head] = lse;
}

// ------------------------------------------------------------- launch plan
struct AttnPlan {
  int rw, tiles, groups;
  long items;  // 0: more than a launch takes
  size_t bytes;
};
template <int D, bool SHARED>
static int attn_places(int rw, bool fp8) {  // workgroups that the chip holds
  return 256 * (rw == 1   ? (fp8 ? Cfg<D, SHARED, true, 1>::WGS : Cfg<D, SHARED, false, 1>::WGS)
                : rw == 2 ? (fp8 ? Cfg<D, SHARED, true, 2>::WGS : Cfg<D, SHARED, false, 2>::WGS)
                          : (fp8 ? Cfg<D, SHARED, true, 4>::WGS : Cfg<D, SHARED, false, 4>::WGS));
}
// A window's plan takes no workspace where that of none takes none: the longest
// item only gets shorter.
static AttnPlan attn_plan(const DSV4GCache *C, int heads, int n_seqs, int n_tokens, int max_q,
                          int max_kv, int window) {
  AttnPlan p = {};
  max_q = max_q > n_tokens ? n_tokens : max_q;
  const int group = heads / C->kv_heads;
  const long rows = (long)max_q * group;
  const int D = C->k_dim;
  // the smallest tile that holds a sequence's rows
  const int least = D == 512 || (D == 256 && C->v_dim) ? 2 : 1;
  p.rw = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  p.rw = p.rw < least ? least : p.rw;
  // a launch is below 2^32 threads, a sequence's rows (new tokens * heads of a
  // kv head) below 2^31; each product only once the one before is known to fit
  if (rows > 0x7FFFFF00L) return p;
  p.tiles = (int)((rows + 32 * p.rw - 1) / (32 * p.rw));
  const long pairs = (long)p.tiles * n_seqs;
  if (pairs > 0xFFFFFFL || pairs * C->kv_heads > 0xFFFFFFL) return p;
  p.items = pairs * C->kv_heads;
  const bool fp8 = C->dtype == DSV4G_DT_F8_E4M3;
  const int places = D == 64    ? attn_places<64, false>(p.rw, fp8)
                     : D == 128 ? attn_places<128, false>(p.rw, fp8)
                                : 256;
  // Three items per place and more: each whole. Fewer: their stages are dealt
  // out where that saves more than it costs, in stages of the longest item that
  // the host's bounds allow (S). Whole items leave the chip idle for the rest of
  // their last round, or half a longest item where lengths differ; dealt out,
  // they pay a second start, the join's launch (3) and the parts, written and
  // read: 16 per workgroup where a part is 64 rows of 512.
  // 64 sequences of up to 4000, 8 kv heads of 128 (512 items, 256 places): 76 us
  // dealt out, 87 whole; 198 and 189 where all have 4000. 800 sequences of up to
  // 1000, latent 512: 141 and 115. 11 prompts of 82 tokens, latent 512 (451 items
  // of 3 stages): 96 and 43.
  const long kv = std::min<long>(max_kv, (long)C->max_pages * C->page_size);
  const int TT = 32 * (4 / p.rw);
  const long span = window ? std::min<long>(kv, (long)window + 32 * p.rw / group + 31) : kv;
  const double S = (double)((span + TT - 1) / TT), r = (double)p.items / places;
  const double idle = std::max(std::ceil(r) - r, 0.5) * (S + AT_START);
  const double parts = p.rw * D / 64.0 * std::min(1.0, p.items * S / (2.0 * places));
  p.groups = r < 3 && idle > AT_START + 3 + parts ? places : 0;
  if (p.groups)
    p.bytes = (size_t)p.groups * 2 * 32 * p.rw * (D * sizeof(float) + sizeof(float2)) +
              (1 + (size_t)p.items) * sizeof(long);
  return p;
}

template <int D, bool SHARED, bool FP8, int RW>
static void attn_launch(const DSV4GCache &C, const CacheGeom &G, const AttnArgs &a, long items,
                        hipStream_t st) {
  if constexpr (Cfg<D, SHARED, FP8, RW>::OK) {
    hipLaunchKernelGGL((k_attn<D, SHARED, FP8, RW>), dim3((unsigned)(a.groups ? a.groups : items)),
                       dim3(256), 0, st, C, G, a);
    if (a.groups)
      hipLaunchKernelGGL((k_attn_join<D, RW>), dim3((unsigned)(items * RW * (D / 32))),
                         dim3(256), 0, st, C, a);
  }
}
template <int D, bool SHARED>
static void attn_launch(const DSV4GCache &C, const CacheGeom &G, const AttnArgs &a,
                        const AttnPlan &p, hipStream_t st) {
  const bool fp8 = C.dtype == DSV4G_DT_F8_E4M3;
  auto f = p.rw == 1 ? (fp8 ? attn_launch<D, SHARED, true, 1> : attn_launch<D, SHARED, false, 1>)
           : p.rw == 2
               ? (fp8 ? attn_launch<D, SHARED, true, 2> : attn_launch<D, SHARED, false, 2>)
               : (fp8 ? attn_launch<D, SHARED, true, 4> : attn_launch<D, SHARED, false, 4>);
  f(C, G, a, p.items, st);
}

}  // namespace dsv4

using namespace dsv4;

extern "C" {

size_t dsv4g_attention_workspace_bytes(const DSV4GCache *C, int heads, int n_seqs, int n_tokens,
                                       int max_q, int max_kv) {
  CacheGeom G;
  if (!C || !cache_geom(C, &G) || heads <= 0 || heads % C->kv_heads || n_seqs <= 0 ||
      n_tokens <= 0 || max_q <= 0 || max_kv <= 0)
    return 0;
  return attn_plan(C, heads, n_seqs, n_tokens, max_q, max_kv, 0).bytes;
}

int dsv4g_attention(void *out, size_t out_stride, float *lse, const void *q, size_t q_stride,
                    int act_dtype, const DSV4GCache *C, int layer, int heads, const int *seqs,
                    const int *starts, int n_seqs, int n_tokens, int max_q, int max_kv,
                    float scale, int window, const float *sink, void *workspace,
                    size_t workspace_bytes, void *stream) {
  CacheGeom G;
  DSV4G_TRY(dsv4g_cache_ok(C, &G, "attention"));
  if (!out || !q || !starts || n_seqs <= 0 || n_tokens <= 0 || layer < 0 ||
      layer >= C->n_layers || heads <= 0 || heads % C->kv_heads || max_q <= 0 || max_kv <= 0 ||
      window < 0 || (act_dtype != DSV4G_DT_F32 && act_dtype != DSV4G_DT_BF16))
    return dsv4g_fail(DSV4G_EINVAL, "attention: bad arguments");
  if (!(fabsf(scale) * LOG2E <= 3.4028235e38f))  // scores are taken to base 2
    return dsv4g_fail(DSV4G_EINVAL, "attention: scale %g, at most 2.35e38", scale);
  const size_t unit = act_dtype == DSV4G_DT_F32 ? 4 : 8;  // elements of 16 bytes
  if (q_stride < (size_t)heads * C->k_dim || out_stride < (size_t)heads * C->k_dim ||
      q_stride % unit || out_stride % unit || ((uintptr_t)q & 15) || ((uintptr_t)out & 15))
    return dsv4g_fail(DSV4G_EINVAL, "attention: rows of q and out must be 16-byte aligned and at "
                      "least heads * dim apart");
  // a window that no length passes is none: positions less the window then fit
  // 32 bits
  if (window >= (long)C->max_pages * C->page_size) window = 0;
  const AttnPlan p = attn_plan(C, heads, n_seqs, n_tokens, max_q, max_kv, window);
  if (p.items == 0) return dsv4g_fail(DSV4G_EINVAL, "attention: too many rows for one call");
  if (p.bytes && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < p.bytes))
    return dsv4g_fail(DSV4G_EINVAL, "attention: 256-byte aligned workspace of %zu bytes needed "
                      "(%zu given)", p.bytes, workspace_bytes);
  AttnArgs a = {};
  a.out = out, a.lse = lse, a.q = q, a.out_stride = out_stride, a.q_stride = q_stride;
  a.seqs = seqs, a.starts = starts, a.sink = sink, a.layer = layer, a.heads = heads;
  a.group = heads / C->kv_heads, a.n_seqs = n_seqs, a.n_tokens = n_tokens, a.max_q = max_q;
  a.max_kv = max_kv, a.window = window, a.f32 = act_dtype == DSV4G_DT_F32;
  a.tiles = p.tiles, a.groups = p.groups, a.halve = fabsf(scale) * LOG2E < AT_TINY;
  a.scale = a.halve ? 2.0f * scale : scale;
  if (p.groups) {
    const size_t cells = (size_t)p.groups * 2 * 32 * p.rw;
    a.part = (float *)workspace;
    a.stat = (float2 *)(a.part + cells * C->k_dim);
    a.first = (long *)(a.stat + cells);
  }
  const hipStream_t st = (hipStream_t)stream;
  const bool shared = C->v_dim == 0;
  switch (C->k_dim) {
    case 64: attn_launch<64, false>(*C, G, a, p, st); break;
    case 128: attn_launch<128, false>(*C, G, a, p, st); break;
    case 256:
      if (shared) attn_launch<256, true>(*C, G, a, p, st);
      else attn_launch<256, false>(*C, G, a, p, st);
      break;
    default: attn_launch<512, true>(*C, G, a, p, st);
  }
  return dsv4g_check_launch("attention");
}

}  // extern "C"
