// dsv4_score.hip - log probabilities of given tokens, with rank, entropy and
// the top alternatives, from rows of logits (dsv4g_logprobs, beside the greedy
// pick). No counterpart in the reference.
//
// One pass over the logits. With z = scale * logit, every thread keeps the
// running maximum m, s = sum e^(z - m) and t = sum e^(z - m) (z - m) of what it
// has seen; two such triples join as
//   m' = max(m1, m2),  f = e^(m1 - m'),
//   s' = f s1 + .. ,   t' = f (t1 + (m1 - m') s1) + ..
// and at the end lse = m + log s, entropy = log s - t / s. All in fp32, whose
// sums run over at most a few hundred terms per thread before they are joined
// pairwise.
//
// The top k are kept per wave, one key per lane in descending order (k <= 64):
// (value as an ordered whole number, ~index), so keys are unique and equal
// values go to the lower index. A wave's indices only grow, so a value enters
// if it is strictly above the k-th one kept: a float comparison per logit, and
// an insertion (a ballot and one shift over the lanes) for the few that pass.
// Where many pass (the first tile; rows in ascending order), the bar is first
// raised to the k-th largest of the 64 lanes' own maxima, found bit by bit
// with ballots: at least k of the tile's values reach it.
//
// Bound: HBM. Rows are cut into segments so that a launch has about 2048
// workgroups where there are fewer rows; a second launch joins the segments.
#include "dsv4_device.h"
#include "dsv4_gpu_internal.h"

namespace dsv4 {

constexpr int SC_T = 256;              // threads
constexpr int SC_E = 16;               // logits per thread and tile
constexpr int SC_TILE = SC_T * SC_E;   // logits per tile: segments are multiples
constexpr int SC_MAX_SEG = 64;         // segments of a row (one lane each when joined)
constexpr float SC_LOW = -3.4028235e38f;  // a maximum that e^(-inf - m) survives

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

// -0 counts as 0 and NaN as -inf in the order of values.
__device__ __forceinline__ uint32_t ordered(float z) {
  if (z != z) z = -__builtin_inff();
  const uint32_t u = f2u(z);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return u2f((o >> 31) ? o ^ 0x80000000u : ~o);
}

__device__ __forceinline__ void score_join(float &m, float &s, float &t, float m2, float s2,
                                           float t2) {
  const float M = fmaxf(m, m2), f1 = __expf(m - M), f2 = __expf(m2 - M);
  // below -200 the factor is 0: no 0 * -inf
  t = f1 * (t + fmaxf(m - M, -200.0f) * s) + f2 * (t2 + fmaxf(m2 - M, -200.0f) * s2);
  s = f1 * s + f2 * s2;
  m = M;
}

// The k largest keys, one per lane, descending (0: none).
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
    settle(k);
  }
  __device__ __forceinline__ void settle(int k) {
    const uint32_t h = __builtin_amdgcn_readlane((uint32_t)(key >> 32), k - 1);
    const uint32_t l = __builtin_amdgcn_readlane((uint32_t)key, k - 1);
    full = (h | l) != 0;
    bar = unordered(h);
  }
};

// x into the list of the wave, for a wave's descending keys x(0), x(1), ..:
// false at the first that does not enter (nor do those behind it).
__device__ __forceinline__ bool top_offer(TopList &top, uint64_t x, int k) {
  if (!x || __popcll(__ballot(top.key > x)) >= k) return false;
  top.insert(x, k);
  return true;
}

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
    return fmaf(f, scale, 0.0f);  // + 0: -0 becomes 0
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
  const float ls = logf(s);  // z - lse as (z - m) - log s: m may be large
  const int lane = threadIdx.x % 64;
  const float nan = __builtin_nanf("");
  if (lane == 0) {
    if (a.logprob) a.logprob[row] = have_token && s > 0.0f ? (zt - m) - ls : nan;
    if (a.rank) a.rank[row] = have_token && s > 0.0f ? above : -1;
    if (a.entropy) a.entropy[row] = s > 0.0f ? ls - t / s : nan;
  }
  if (lane < a.k) {
    const size_t o = (size_t)row * a.k + lane;
    const int id = key ? (int)(0xFFFFFFFFu - (uint32_t)key) : -1;
    if (a.top_id) a.top_id[o] = id;
    if (a.top_logprob)
      a.top_logprob[o] = id >= 0 && s > 0.0f ? (unordered((uint32_t)(key >> 32)) - m) - ls : nan;
  }
}

// One segment of one row (SPLIT), or a whole row.
template <typename T, bool TOP, bool SPLIT>
__global__ __launch_bounds__(SC_T) void k_score(ScoreArgs a) {
  __shared__ float s_m[4], s_s[4], s_t[4];
  __shared__ int s_above[4];
  __shared__ uint64_t s_key[TOP ? 4 * 64 : 1];
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
    zt = fmaf(sizeof(T) == 4 ? u2f((uint32_t)e) : u2f((uint32_t)e << 16), a.scale, 0.0f);
  }
  float m = SC_LOW, s = 0.0f, t = 0.0f;
  int above = 0;
  TopList top;
  top.init();
  for (int at = c0; at < end; at += SC_TILE) {
    float z[SC_E];
#pragma unroll
    for (int j = 0; j < SC_E; ++j) z[j] = tile.value(j, a.scale);
    if (at + SC_TILE < end) tile.load(l, at + SC_TILE, end);  // in flight while this one is summed
    float mt = z[0];
#pragma unroll
    for (int j = 1; j < SC_E; ++j) mt = fmaxf(mt, z[j]);
    if (mt > m) {
      const float f = __expf(m - mt);
      t = f * (t + fmaxf(m - mt, -200.0f) * s);
      s *= f;
      m = mt;
    }
    const int ti = token - at;
#pragma unroll
    for (int j = 0; j < SC_E; ++j) {
      const float d = z[j] - m, e = __expf(d);
      s += e;
      t = fmaf(e, fmaxf(d, -200.0f), t);  // e is 0 there: no 0 * -inf
      above += z[j] > zt || (z[j] == zt && tile.place(j) < ti);
    }
    if (TOP) {
      uint32_t least = 0;  // smallest ordered value that enters
      int many = 0;
      if (top.full) {
#pragma unroll
        for (int j = 0; j < SC_E; ++j) many += __popcll(__ballot(z[j] > top.bar));
        if (many) least = ordered(top.bar) + 1;
      }
      if (!top.full || many > 2 * a.k) {
        // the k-th largest of the lanes' maxima, bit by bit; places behind
        // the row's end rank below every value
        uint32_t mine = 0;
#pragma unroll
        for (int j = 0; j < SC_E; ++j)
          if (at + tile.place(j) < end) mine = max(mine, ordered(z[j]));
        uint32_t x = 0;
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
          if (__popcll(__ballot(mine >= (x | bit))) >= a.k) x |= bit;
        least = max(least, x);
        many = 1;
      }
      if (many) {
#pragma unroll
        for (int j = 0; j < SC_E; ++j) {
          const uint32_t o = ordered(z[j]);
          uint64_t who = __ballot(o >= least && at + tile.place(j) < end);
          while (who) {
            const int b = __builtin_ctzll(who);
            who &= who - 1;
            const uint32_t ob = __builtin_amdgcn_readlane(o, b);
            const uint32_t ib = at + (j / Tile<T>::V) * (SC_T * Tile<T>::V) +
                                Tile<T>::V * (64 * wave + b) + j % Tile<T>::V;
            top.insert(((uint64_t)ob << 32) | (0xFFFFFFFFu - ib), a.k);
          }
        }
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    score_join(m, s, t, __shfl_xor(m, o, 64), __shfl_xor(s, o, 64), __shfl_xor(t, o, 64));
    above += __shfl_xor(above, o, 64);
  }
  if (lane == 0) {
    s_m[wave] = m;
    s_s[wave] = s;
    s_t[wave] = t;
    s_above[wave] = above;
  }
  if (TOP) s_key[64 * wave + lane] = top.key;
  __syncthreads();
  if (wave) return;
  above = s_above[0];
  for (int w = 1; w < 4; ++w) {
    score_join(m, s, t, s_m[w], s_s[w], s_t[w]);
    above += s_above[w];
    if (TOP)
      for (int j = 0; j < a.k && top_offer(top, s_key[64 * w + j], a.k); ++j) {
      }
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
// all into LDS at once (the merge walks them with dependent steps, which would
// each cost a memory round trip), then four waves merge a quarter of them each
// and the first one the four results.
template <typename T, bool TOP>
__global__ __launch_bounds__(SC_T) void k_score_join(ScoreArgs a) {
  __shared__ uint64_t s_key[TOP ? SC_MAX_SEG * DSV4G_MAX_TOP : 1];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid % 64;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  ScorePart p = {SC_LOW, 0.0f, 0.0f, 0};
  if (lane < a.nseg) p = a.part[(size_t)row * a.nseg + lane];
  const int token = a.tokens ? a.tokens[row] : -1;
  const bool have = token >= 0 && token < a.vocab;
  TopList top;
  top.init();
  if (TOP) {
    const uint64_t *keys = a.keys + (size_t)row * a.nseg * a.k;
    for (int i = tid; i < a.nseg * a.k; i += SC_T) s_key[i] = keys[i];
    __syncthreads();
    for (int g = wave; g < a.nseg; g += 4)
      for (int j = 0; j < a.k && top_offer(top, s_key[g * a.k + j], a.k); ++j) {
      }
    __syncthreads();
    s_key[64 * wave + lane] = top.key;
    __syncthreads();
  }
  if (wave) return;
  if (TOP)
    for (int w = 1; w < 4; ++w)
      for (int j = 0; j < a.k && top_offer(top, s_key[64 * w + j], a.k); ++j) {
      }
  float zt = 0.0f;
  if (have) {
    const T e = ((const T *)a.logits)[(size_t)row * a.stride + token];
    zt = fmaf(sizeof(T) == 4 ? u2f((uint32_t)e) : u2f((uint32_t)e << 16), a.scale, 0.0f);
  }
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
