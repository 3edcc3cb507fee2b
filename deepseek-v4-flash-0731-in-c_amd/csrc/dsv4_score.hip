// dsv4_score.hip - log probabilities of given tokens, with rank, entropy and
// the top alternatives, from rows of logits (dsv4g_logprobs, beside the greedy
// pick). No counterpart in the reference.
//
// One pass over the logits. With z = scale * logit and L = log2 e, every thread
// keeps the running maximum m of its z and, with M = fl(m L),
//   s = sum 2^(z L - M),  t = sum 2^(z L - M) (z L - M)
// (one fma and the hardware's 2^x per logit). Where |M| is SC_NEAR or more (masks
// beyond -45000 in a thread that has seen nothing else, or logits as large), M's
// rounding would grow until no 2^x holds it: there the exponent is (z - m) L, one
// instruction more (taken everywhere, it costs 4% of 2048 BF16 rows). With off(m) what the first kind of M is off m L, exactly by an fma, two
// triples join as
//   m' = max(m1, m2),  g = (m1 - m') L + off(m1) - off(m'),  f = 2^g,
//   s' = f s1 + ..,    t' = f (t1 + g s1) + ..
// and at the end
//   lse - m = ln s + off(m) ln 2,  entropy = ln s - (t / s) ln 2.
// All in fp32, whose sums run over 1/256 of a row per thread (505 terms of
// 129280) before they are joined pairwise. -inf, a token that cannot be taken,
// weighs nothing.
//
// The top k are kept per wave, one key per lane in descending order (k <= 64):
// (value as an ordered whole number, ~index), so keys are unique and equal
// values go to the lower index. A wave's indices only grow, so a value enters
// if it is strictly above the k-th one kept. It must also reach the least of the
// four waves' (k / 4)-th values: k values of the row do. A comparison with the
// tile's maximum decides whether the tile is looked through at all. What passes
// is listed in LDS, 64 at a time, and inserted (a ballot and one shift over the
// lanes) or, above SC_FEW of them, sorted and merged. In the first tile the bar
// is the k-th largest of the 64 lanes' own maxima, found bit by bit with ballots:
// at least k of the tile's values reach it. Two sorted lists merge in 6 steps:
// the larger of a[i] and b[63 - i] is the upper half of both, a bitonic sequence.
//
// Bound: HBM for fp32 rows (2048 rows of 129280: 179 us, 5.9 TB/s), the vector
// units for BF16 ones, with half the bytes per value (107 to 117 us, 4.5 to 4.9
// TB/s: about 10 instructions a value, one of them 2^x at a quarter of the rate;
// the index compared for every value's rank cost a quarter more). k = 8 adds 15
// and 37 us: a wave looks through its first tiles and then ever fewer. Fewer
// registers for it (six waves per SIMD in place of five) cost 10%: the sort's lane
// masks are then computed at each use.
// Rows are cut into segments until a launch has about 2048 workgroups, what the
// chip holds at once; a second launch joins them (64 rows 12 us, one row 17 us,
// against 278 and 303 us in library calls).
#include "dsv4_device.h"
#include "dsv4_gpu_internal.h"

namespace dsv4 {

constexpr int SC_T = 256;              // threads
constexpr int SC_E = 16;               // logits per thread and tile
constexpr int SC_TILE = SC_T * SC_E;   // logits per tile: segments are multiples
constexpr int SC_MAX_SEG = 64;         // segments of a row (one lane each when joined)
constexpr float SC_NEAR = 0x1p16f;     // largest M of the sums by one fma
constexpr float SC_L = 1.4426950408889634f, SC_LN2 = 0.6931471805599453f;
constexpr int SC_FEW = 6;              // values that are inserted one by one

// Stats of part of a row, as the segments' launch leaves them.
struct ScorePart {
  float m, s, t;
  int above;  // logits before the given token in the order of rank
};

struct ScoreArgs {
  float *logprob, *entropy, *top_logprob;
  int *rank, *top_id;
  const void *logits;
  const int *tokens;
  size_t stride;
  int vocab, k, nseg, seg_len;
  float scale;
  ScorePart *part;  // [n][nseg]
  uint64_t *keys;   // [n][nseg][k]
};

// -0 counts as 0 (a product that vanishes keeps its sign) and NaN as -inf in the
// order of values.
__device__ __forceinline__ uint32_t ordered(float z) {
  if (z != z) z = -__builtin_inff();
  const uint32_t u = f2u(z + 0.0f);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return u2f((o >> 31) ? o ^ 0x80000000u : ~o);
}

// What z is taken relative to: m, or the least number where all are -inf.
__device__ __forceinline__ float score_ref(float m) { return fmaxf(m, -3.4028235e38f); }
__device__ __forceinline__ float score_off(float m) {
  const float M = m * SC_L;
  return fabsf(M) < SC_NEAR ? -fmaf(m, SC_L, -M) : 0.0f;
}
// s of a sum relative to m1, now to m, and its t.
__device__ __forceinline__ float score_shift(float m1, float m, float s, float &t) {
  const float g = (m1 - m) * SC_L + (score_off(m1) - score_off(m));
  const float f = __builtin_amdgcn_exp2f(g);
  t = f * (t + fmaxf(g, -300.0f) * s);  // f is 0 below: no 0 * inf
  return f * s;
}
__device__ __forceinline__ void score_join(float &m, float &s, float &t, float m2, float s2,
                                           float t2) {
  const float mm = fmaxf(m, m2), r = score_ref(mm);
  s = score_shift(score_ref(m), r, s, t) + score_shift(score_ref(m2), r, s2, t2);
  t += t2;
  m = mm;
}

// Another lane's key, and the exchange step of a sort: lanes with bit X set
// keep the smaller (up: the larger) of the two.
template <int X>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  const int lane = threadIdx.x;
  if (X == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? r[0] : r[1];
  }
  if (X == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? r[0] : r[1];
  }
  if (X == 8) return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false);  // row_ror:8
  if (X == 4) {
    const uint32_t u = __builtin_amdgcn_update_dpp(0, v, 0x104, 0xf, 0x5, false);  // row_shl:4
    return __builtin_amdgcn_update_dpp(u, v, 0x114, 0xf, 0xa, false);              // row_shr:4
  }
  return __builtin_amdgcn_update_dpp(0, v, X == 2 ? 0x4E : 0xB1, 0xf, 0xf, false);  // quad_perm
}
template <int X>
__device__ __forceinline__ uint64_t exchange(uint64_t key, bool up) {
  const uint64_t other = ((uint64_t)lane_xor<X>((uint32_t)(key >> 32)) << 32) |
                         lane_xor<X>((uint32_t)key);
  const bool small = ((threadIdx.x & X) != 0) != up;
  return (other < key) == small ? other : key;
}
// A bitonic sequence over the lanes into descending order.
__device__ __forceinline__ uint64_t bitonic_down(uint64_t key) {
  key = exchange<32>(key, false);
  key = exchange<16>(key, false);
  key = exchange<8>(key, false);
  key = exchange<4>(key, false);
  key = exchange<2>(key, false);
  return exchange<1>(key, false);
}
// Any keys into ascending order.
__device__ __forceinline__ uint64_t sort_up(uint64_t key) {
  const int l = threadIdx.x % 64;
  auto up = [&](int k) { return (l & k) == 0; };  // runs of k: up and down in turn
  key = exchange<1>(key, up(2));
  key = exchange<2>(key, up(4));
  key = exchange<1>(key, up(4));
  key = exchange<4>(key, up(8));
  key = exchange<2>(key, up(8));
  key = exchange<1>(key, up(8));
  key = exchange<8>(key, up(16));
  key = exchange<4>(key, up(16));
  key = exchange<2>(key, up(16));
  key = exchange<1>(key, up(16));
  key = exchange<16>(key, up(32));
  key = exchange<8>(key, up(32));
  key = exchange<4>(key, up(32));
  key = exchange<2>(key, up(32));
  key = exchange<1>(key, up(32));
  key = exchange<32>(key, true);
  key = exchange<16>(key, true);
  key = exchange<8>(key, true);
  key = exchange<4>(key, true);
  key = exchange<2>(key, true);
  return exchange<1>(key, true);
}

// The k largest keys, one per lane, descending (0: none); lanes from k on hold
// what else they happen to.
struct TopList {
  uint64_t key;
  float bar;   // value of the k-th one
  bool full;   // k are kept
  __device__ __forceinline__ void init() {
    key = 0;
    bar = 0.0f;
    full = false;
  }
  // x: uniform
  __device__ __forceinline__ void insert(uint64_t x, int k) {
    const int pos = __popcll(__ballot(key > x));
    if (pos >= k) return;
    const int lane = threadIdx.x % 64;
    // each lane takes its lower neighbour's key
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)key, 0x138, 0xf, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(key >> 32), 0x138, 0xf, 0xf,
                                                    false);
    const uint64_t below = ((uint64_t)hi << 32) | lo;
    key = lane < pos ? key : lane == pos ? x : below;
  }
  // other: ascending over the lanes
  __device__ __forceinline__ void merge_up(uint64_t other) {
    key = bitonic_down(other > key ? other : key);
  }
  __device__ __forceinline__ void settle(int k) {
    const uint32_t h = __builtin_amdgcn_readlane((uint32_t)(key >> 32), k - 1);
    const uint32_t l = __builtin_amdgcn_readlane((uint32_t)key, k - 1);
    full = (h | l) != 0;
    bar = unordered(h);
  }
};

// 16 logits of a thread from row offset i0 + the thread's places: 16-byte
// loads where a whole tile is inside the row, guarded single ones at its end.
// Place j of thread t: tile + (j / V) * (SC_T * V) + V * t + j % V.
template <typename T>
struct Tile {
  static constexpr int V = 16 / sizeof(T);  // per load
  uint4 raw[SC_E / V];
  __device__ __forceinline__ void load(const T *row, int at, int end) {
    const int tid = threadIdx.x;
    if (at + SC_TILE <= end) {
#pragma unroll
      for (int g = 0; g < SC_E / V; ++g)  // rows may start at any element
        __builtin_memcpy(&raw[g], row + at + g * (SC_T * V) + V * tid, 16);
      return;
    }
    const T low = sizeof(T) == 4 ? (T)0xFF800000u : (T)0xFF80u;  // -inf
#pragma unroll
    for (int g = 0; g < SC_E / V; ++g) {
      T e[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int i = at + g * (SC_T * V) + V * tid + j;
        e[j] = i < end ? row[i] : low;
      }
      __builtin_memcpy(&raw[g], e, 16);
    }
  }
  __device__ __forceinline__ float value(int j, float scale) const {
    T e[V];
    __builtin_memcpy(e, &raw[j / V], 16);
    const float f = sizeof(T) == 4 ? u2f((uint32_t)e[j % V]) : u2f((uint32_t)e[j % V] << 16);
    return f * scale;
  }
  __device__ __forceinline__ static int place(int j) {
    return (j / V) * (SC_T * V) + V * threadIdx.x + j % V;
  }
};

// Everything of one row from its joined stats (one thread), and of its top
// list (one wave; lane l holds the l-th key).
__device__ __forceinline__ void score_write(const ScoreArgs &a, int row, float m, float s,
                                            float t, int above, uint64_t key, bool have_token,
                                            float zt) {
  // z - lse as (z - m) - (lse - m): m may be large
  const float ln = logf(s), ls = ln + score_off(score_ref(m)) * SC_LN2;
  const bool fine = s > 0.0f && m > -__builtin_inff();
  const int lane = threadIdx.x % 64;
  const float nan = __builtin_nanf("");
  if (lane == 0) {
    if (a.logprob) a.logprob[row] = have_token && fine ? (zt - m) - ls : nan;
    if (a.rank) a.rank[row] = have_token && fine ? above : -1;
    if (a.entropy) a.entropy[row] = fine ? ln - t / s * SC_LN2 : nan;
  }
  if (lane < a.k) {
    const size_t o = (size_t)row * a.k + lane;
    const int id = key ? (int)(0xFFFFFFFFu - (uint32_t)key) : -1;
    if (a.top_id) a.top_id[o] = id;
    if (a.top_logprob)
      a.top_logprob[o] = id >= 0 && fine ? (unordered((uint32_t)(key >> 32)) - m) - ls : nan;
  }
}

// One segment of one row (SPLIT), or a whole row.
template <typename T, bool TOP, bool SPLIT>
__global__ __launch_bounds__(SC_T) void k_score(ScoreArgs a) {
  __shared__ float s_m[4], s_s[4], s_t[4];
  __shared__ int s_above[4];
  __shared__ uint64_t s_key[TOP ? 4 * 64 : 1];
  __shared__ volatile float s_bar[4];  // each wave's (k / 4)-th value so far
  const int tid = threadIdx.x, lane = tid % 64;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int row = SPLIT ? blockIdx.x / a.nseg : blockIdx.x;
  const int seg = SPLIT ? blockIdx.x % a.nseg : 0;
  const int c0 = seg * a.seg_len, end = SPLIT ? min(a.vocab, c0 + a.seg_len) : a.vocab;
  const T *l = (const T *)a.logits + (size_t)row * a.stride;
  Tile<T> tile;
  tile.load(l, c0, end);
  const int token = a.tokens ? a.tokens[row] : -1;
  const bool have = token >= 0 && token < a.vocab;
  float zt = __builtin_nanf("");  // no logit is above it
  if (have) {
    const T e = l[token];
    zt = (sizeof(T) == 4 ? u2f((uint32_t)e) : u2f((uint32_t)e << 16)) * a.scale;
  }
  // the next value below it (of 0: past -0, which the order has no place for)
  const float zt_below = unordered(ordered(zt) - (zt == 0.0f ? 2 : 1));
  if (TOP) {
    if (tid < 4) s_bar[tid] = -__builtin_inff();
    __syncthreads();
  }
  float m = -__builtin_inff(), s = 0.0f, t = 0.0f;
  int above = 0;  // the wave's
  TopList top;
  top.init();
  for (int at = c0; at < end; at += SC_TILE) {
    float z[SC_E];
#pragma unroll
    for (int j = 0; j < SC_E; ++j) z[j] = tile.value(j, a.scale);
    if (at + SC_TILE < end) tile.load(l, at + SC_TILE, end);  // in flight while this one is summed
    float mt = fmaxf(z[0], z[1]);
#pragma unroll
    for (int j = 2; j < SC_E; j += 2) mt = fmaxf(fmaxf(mt, z[j]), z[j + 1]);
    if (mt > m) {
      s = score_shift(score_ref(m), score_ref(mt), s, t);
      m = mt;
    }
    const float M = m * SC_L;
    if (fabsf(M) < SC_NEAR) {
#pragma unroll
      for (int j = 0; j < SC_E; ++j) {
        const float d = fmaf(z[j], SC_L, -M), e = __builtin_amdgcn_exp2f(d);
        s += e;
        t = fmaf(e, fmaxf(d, -300.0f), t);  // no 0 * inf
      }
    } else {
      const float r = score_ref(m);
#pragma unroll
      for (int j = 0; j < SC_E; ++j) {
        const float d = (z[j] - r) * SC_L, e = __builtin_amdgcn_exp2f(d);
        s += e;
        t = fmaf(e, fmaxf(d, -300.0f), t);
      }
    }
    // rank: equal values count where they come first; but for the token's own
    // tile, one comparison does it
    if (__any(mt >= zt)) {
      if (zt > -__builtin_inff() && (at + SC_TILE <= token || at > token)) {
        const float th = at < token ? zt_below : zt;
#pragma unroll
        for (int j = 0; j < SC_E; ++j) above += __popcll(__ballot(z[j] > th));
      } else {
#pragma unroll
        for (int j = 0; j < SC_E; ++j)
          above += __popcll(__ballot(z[j] > zt || (z[j] == zt && at + tile.place(j) < token)));
      }
    }
    if constexpr (TOP) {
      // Four waves' (k / 4)-th values or better are k values of the row: nothing
      // below the least of them is among its k.
      const float least4 = fminf(fminf(s_bar[0], s_bar[1]), fminf(s_bar[2], s_bar[3]));
      if (!top.full || __any(mt > top.bar && mt >= least4)) {
        float enters;  // the smallest value that does
        if (top.full) {
          enters = fmaxf(unordered(ordered(top.bar) + 1), least4);
        } else {
          // the k-th largest of the lanes' maxima, bit by bit. NaN counts as
          // -inf; places behind the row's end as NaN, which never enters.
          uint32_t mine = 0, least = 0;
#pragma unroll
          for (int j = 0; j < SC_E; ++j) {
            const bool in = at + tile.place(j) < end;
            const uint32_t o = ordered(z[j]);
            z[j] = in ? unordered(o) : __builtin_nanf("");
            mine = in ? max(mine, o) : mine;
          }
          for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
            if (__popcll(__ballot(mine >= (least | bit))) >= a.k) least |= bit;
          enters = least ? unordered(least) : -__builtin_inff();
        }
        // 64 candidates at a time, through LDS
        uint64_t *cand = s_key + 64 * wave;
        int total = 0;
        for (int from = 0; from == 0 || from < total; from += 64) {
          total = 0;
#pragma unroll
          for (int j = 0; j < SC_E; ++j) {
            const uint64_t who = __ballot(z[j] >= enters);
            if (who) {
              const int n = total - from + __popcll(who & ((1ull << lane) - 1));
              const uint32_t i = at + tile.place(j);
              if ((who >> lane & 1) && n >= 0 && n < 64)
                cand[n] = ((uint64_t)ordered(z[j]) << 32) | (0xFFFFFFFFu - i);
              total += __popcll(who);
            }
          }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          const int n = min(64, total - from);
          if (n > SC_FEW) {
            top.merge_up(sort_up(lane < n ? cand[lane] : 0));
          } else {
            for (int c = 0; c < n; ++c) top.insert(cand[c], a.k);
          }
          asm volatile("" ::: "memory");
        }
        top.settle(a.k);
        const uint32_t q = __builtin_amdgcn_readlane((uint32_t)(top.key >> 32), (a.k + 3) / 4 - 1);
        if (lane == 0 && q) s_bar[wave] = unordered(q);
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    score_join(m, s, t, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64), __shfl_xor(t, o, 64));
  if (lane == 0) {
    s_m[wave] = m;
    s_s[wave] = s;
    s_t[wave] = t;
    s_above[wave] = above;
  }
  // ascending, for the merge; what is behind the k-th key stays behind it
  if (TOP) s_key[64 * wave + 63 - lane] = lane < a.k ? top.key : 0;
  __syncthreads();
  if (wave) return;
  for (int w = 1; w < 4; ++w) {
    score_join(m, s, t, s_m[w], s_s[w], s_t[w]);
    above += s_above[w];
    if (TOP) top.merge_up(s_key[64 * w + lane]);
  }
  if (SPLIT) {
    const size_t o = (size_t)row * a.nseg + seg;
    if (lane == 0) a.part[o] = {m, s, t, above};
    if (TOP && lane < a.k) a.keys[o * a.k + lane] = top.key;
  } else {
    score_write(a, row, m, s, t, above, top.key, have, zt);
  }
}

// Joins a row's segments. The stats: one wave, a lane per segment. The lists:
// all into LDS at once (a merge waits for its list), then four waves merge a
// quarter of them each and the first one the four results.
template <typename T, bool TOP>
__global__ __launch_bounds__(SC_T) void k_score_join(ScoreArgs a) {
  __shared__ uint64_t s_key[TOP ? SC_MAX_SEG * DSV4G_MAX_TOP : 1];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid % 64;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  ScorePart p = {-__builtin_inff(), 0.0f, 0.0f, 0};
  if (lane < a.nseg) p = a.part[(size_t)row * a.nseg + lane];
  const int token = a.tokens ? a.tokens[row] : -1;
  const bool have = token >= 0 && token < a.vocab;
  float zt = 0.0f;
  if (have) {
    const T e = ((const T *)a.logits)[(size_t)row * a.stride + token];
    zt = (sizeof(T) == 4 ? u2f((uint32_t)e) : u2f((uint32_t)e << 16)) * a.scale;
  }
  TopList top;
  top.init();
  if (TOP) {
    const uint64_t *keys = a.keys + (size_t)row * a.nseg * a.k;
    for (int i = tid; i < a.nseg * a.k; i += SC_T) s_key[i] = keys[i];
    __syncthreads();
    const int r = 63 - lane;  // ascending
    for (int g = wave; g < a.nseg; g += 4) top.merge_up(r < a.k ? s_key[g * a.k + r] : 0);
    __syncthreads();
    s_key[64 * wave + r] = top.key;
    __syncthreads();
  }
  if (wave) return;
  if (TOP)
    for (int w = 1; w < 4; ++w) top.merge_up(s_key[64 * w + lane]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    score_join(p.m, p.s, p.t, __shfl_xor(p.m, o, 64), __shfl_xor(p.s, o, 64),
               __shfl_xor(p.t, o, 64));
    p.above += __shfl_xor(p.above, o, 64);
  }
  score_write(a, row, p.m, p.s, p.t, p.above, top.key, have, zt);
}

// Segments of a row: enough workgroups for the chip, at least a tile each.
static void score_split(int vocab, int n, int *nseg, int *seg_len) {
  const int tiles = (vocab + SC_TILE - 1) / SC_TILE;
  int want = (2048 + n - 1) / n;
  want = want > tiles ? tiles : want;
  want = want > SC_MAX_SEG ? SC_MAX_SEG : want;
  const int per = (tiles + want - 1) / want;
  *seg_len = per * SC_TILE;
  *nseg = (tiles + per - 1) / per;
}

template <typename T>
static void score_launch(const ScoreArgs &a, int n, hipStream_t st) {
  const bool top = a.k > 0, split = a.nseg > 1;
  auto k = top ? (split ? k_score<T, true, true> : k_score<T, true, false>)
               : (split ? k_score<T, false, true> : k_score<T, false, false>);
  hipLaunchKernelGGL(k, dim3((unsigned)((long)n * a.nseg)), dim3(SC_T), 0, st, a);
  if (!split) return;
  auto j = top ? k_score_join<T, true> : k_score_join<T, false>;
  hipLaunchKernelGGL(j, dim3((unsigned)n), dim3(SC_T), 0, st, a);
}

}  // namespace dsv4

using namespace dsv4;

extern "C" {

size_t dsv4g_logprobs_workspace_bytes(int vocab, int n, int k) {
  if (vocab <= 0 || n <= 0 || k < 0 || k > DSV4G_MAX_TOP) return 0;
  int nseg, len;
  score_split(vocab, n, &nseg, &len);
  if (nseg == 1) return 0;
  return (size_t)n * nseg * (sizeof(ScorePart) + (size_t)k * 8);
}

int dsv4g_logprobs(float *logprob, float *entropy, int *rank, int *top_id, float *top_logprob,
                   const void *logits, int dtype, int vocab, int n, size_t stride,
                   const int *tokens, int k, float scale, void *workspace,
                   size_t workspace_bytes, void *stream) {
  if (!logits || vocab <= 0 || n <= 0 || stride < (size_t)vocab || k < 0 || k > DSV4G_MAX_TOP ||
      (dtype != DSV4G_DT_F32 && dtype != DSV4G_DT_BF16))
    return dsv4g_fail(DSV4G_EINVAL, "logprobs: bad arguments");
  if (!(scale > 0.0f) || scale > 3.4028235e38f)
    return dsv4g_fail(DSV4G_EINVAL, "logprobs: scale %g, a positive number needed", scale);
  if ((logprob || rank) && !tokens)
    return dsv4g_fail(DSV4G_EINVAL, "logprobs: logprob and rank need tokens");
  if ((uintptr_t)logits & (dtype == DSV4G_DT_F32 ? 3 : 1))
    return dsv4g_fail(DSV4G_EINVAL, "logprobs: misaligned logits");
  if (vocab > 1 << 30 || n > 0xFFFFFF)  // places in 32 bits; a launch is below 2^32 threads
    return dsv4g_fail(DSV4G_EINVAL, "logprobs: %d rows of %d, at most 2^24 - 1 of 2^30", n, vocab);
  const size_t need = dsv4g_logprobs_workspace_bytes(vocab, n, k);
  if (need && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < need))
    return dsv4g_fail(DSV4G_EINVAL, "logprobs: 256-byte aligned workspace of %zu bytes needed "
                      "(%zu given)", need, workspace_bytes);
  ScoreArgs a = {};
  a.logprob = logprob, a.entropy = entropy, a.rank = rank;
  a.top_id = top_id, a.top_logprob = top_logprob;
  a.logits = logits, a.tokens = tokens, a.stride = stride, a.vocab = vocab, a.k = k;
  a.scale = scale;
  score_split(vocab, n, &a.nseg, &a.seg_len);
  if (a.nseg > 1) {
    a.part = (ScorePart *)workspace;
    a.keys = (uint64_t *)(a.part + (size_t)n * a.nseg);
  }
  if (dtype == DSV4G_DT_F32) score_launch<uint32_t>(a, n, (hipStream_t)stream);
  else score_launch<uint16_t>(a, n, (hipStream_t)stream);
  return dsv4g_check_launch("logprobs");
}

}  // extern "C"
