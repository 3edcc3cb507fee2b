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
// Weights are rounded to BF16 for the matrix unit (2^-9 relative, as the cache
// rows are BF16 themselves); scores, m, l and O stay in fp32. m follows the
// maximum only when it grows by more than 2^8 (weights up to 2^8 lose nothing
// in fp32 or BF16): the rescaling of O, one multiplication per accumulator, is
// then rare.
//
// Rows of 16-byte chunks are stored with the chunk index XORed by a function
// of the row (chunk_swizzle): both kinds of read then touch every bank once
// per 16 lanes.
#include "dsv4_cache.h"
#include "dsv4_device.h"
#include "dsv4_gpu_internal.h"

namespace dsv4 {

typedef __bf16 Bf8 __attribute__((ext_vector_type(8)));
typedef float F16v __attribute__((ext_vector_type(16)));
typedef short S4 __attribute__((ext_vector_type(4)));
typedef int I4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float AT_GROW = 8.0f;  // log2 of what the weights may grow to before a rescaling
constexpr int AT_MAX_SPLIT = 64;

struct AttnArgs {
  void *out;
  float *lse;
  const void *q;
  size_t out_stride, q_stride;
  const int *seqs, *starts;
  const float *sink;
  float *part;   // [item][split][ROWS * D] outputs not yet divided, in the waves' layout
  float2 *stat;  // [item][split][ROWS] (m, l)
  int layer, heads, group, n_seqs, n_tokens, max_q, max_kv, window, f32;
  int tiles, nsplit, items;
  float scale;
};

// Row waves RW (32 rows each) and, with fewer than 4, KW = 4 / RW waves that
// share a stage's tokens.
template <int D, bool SHARED, bool FP8, int RW>
struct Cfg {
  static constexpr int KW = 4 / RW, TT = 32 * KW, ROWS = 32 * RW;
  static constexpr int ROWB = 2 * D, CH = D / 8;  // bytes and 16-byte chunks of a row
  static constexpr int KB = TT * ROWB, STAGE = SHARED ? KB : 2 * KB;
  // bytes of LDS: two workgroups per CU for narrow heads, all for wide ones
  static constexpr int CAP = D <= 128 && RW > 1 ? 66 * 1024 : 132 * 1024;
  static constexpr int FIT = CAP / STAGE;
  static constexpr int NBUF = FP8 ? 2 : FIT > 4 ? 4 : FIT;
  static constexpr bool OK = FIT >= 2;
  static constexpr int NP = D / 32;  // output tiles
  // a wave's outputs and its rows' (m, l), handed over when waves share rows
  static constexpr int PART = 32 * D * 4 + 64 * 8, JOIN = KW > 1 ? RW * PART : 0;
  static constexpr int LDS = NBUF * STAGE > JOIN ? NBUF * STAGE : JOIN;
  static constexpr int WGS = D <= 128 && LDS <= 80 * 1024 ? 2 : 1;  // per CU
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

// What a workgroup works on; false: nothing. Uniform.
struct Item {
  int b, kvh, tile, split, seq, start, count, len, r0, nrows, lo, hi, clear, s0, s1, parts;
};
template <int ROWS, int TT>
__device__ __forceinline__ bool attn_item(const DSV4GCache &C, const AttnArgs &a, int id,
                                          Item &it) {
  it.split = id % a.nsplit;
  id /= a.nsplit;
  it.kvh = id % C.kv_heads;
  id /= C.kv_heads;
  it.b = id % a.n_seqs;
  it.tile = a.tiles - 1 - id / a.n_seqs;  // the longest ranges first
  it.seq = a.seqs ? a.seqs[it.b] : it.b;
  it.start = a.starts[it.b];
  const long end = a.starts[it.b + 1];
  const long count = end - it.start;
  it.len = it.seq >= 0 && it.seq < C.n_seqs ? C.len[it.seq] : -1;
  if (it.start < 0 || end > a.n_tokens || count < 0 || count > a.max_q || it.len < count ||
      it.len > a.max_kv || it.len > (long)C.max_pages * C.page_size) {
    if (it.tile == 0 && it.split == 0 && threadIdx.x == 0)
      atomicOr(C.status, DSV4G_CACHE_LIST);
    return false;
  }
  it.count = (int)count;
  it.r0 = it.tile * ROWS;
  it.nrows = it.count * a.group;
  if (it.r0 >= it.nrows) return false;
  const int first = it.len - it.count + it.r0 / a.group;
  it.hi = it.len - it.count + (min(it.r0 + ROWS, it.nrows) - 1) / a.group + 1;
  it.clear = a.window ? max(0, first - a.window + 1) : 0;  // the first token that is seen
  it.lo = it.clear & ~31;
  const int stages = (it.hi - it.lo + TT - 1) / TT;
  const int per = (stages + a.nsplit - 1) / a.nsplit;
  it.parts = (stages + per - 1) / per;
  it.s0 = it.split * per;
  it.s1 = min(stages, it.s0 + per);
  return true;
}

// The page of the 16-token group that begins at token t, or -1.
__device__ __forceinline__ int page_of(const DSV4GCache &C, const CacheGeom &G, const Item &it,
                                       int t) {
  if (t >= it.hi || t + 15 < it.clear) return -1;
  const int *cell = C.table + (size_t)it.seq * C.max_pages + (t >> G.shift);
  return *(const __attribute__((address_space(4))) int *)cell;  // written by earlier kernels only
}
__device__ __forceinline__ I4 page_rsrc(const DSV4GCache &C, const CacheGeom &G, int layer,
                                        int page) {
  const bool ok = page >= 0 && page < C.n_pages;
  const uint64_t p = (uint64_t)(uintptr_t)C.pages +
                     ((uint64_t)layer * C.n_pages + (ok ? page : 0)) * G.page_bytes;
  // no bytes behind a page that is none: its loads give zeros
  return I4{(int)(uint32_t)p, (int)(uint32_t)(p >> 32), ok ? (int)G.page_bytes : 0, 0x00020000};
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// BF16 pages: one stage's rows into LDS by direct loads (16 bytes per lane, 1
// KB per instruction). Each wave brings TT / 4 tokens. In inline asm: a direct
// load has no output register, and the compiler would make every later LDS
// read wait for all of them; wait_loads() and the barrier order them instead.
template <int D, bool SHARED, int TT>
__device__ __forceinline__ void stage_bf16(const DSV4GCache &C, const CacheGeom &G,
                                           const AttnArgs &a, const Item &it, const int (&page)[2],
                                           int st, uint32_t lds, int wave, int lane) {
  constexpr int CH = D / 8, TB = 64 / CH, TW = TT / 4, TG = TW < 16 ? TW : 16;
#pragma unroll
  for (int g = 0; g < TW / TG; ++g) {
    const int tl0 = wave * TW + g * TG;              // token of the stage
    const int t0 = it.lo + st * TT + tl0;            // token of the sequence
    const I4 rsrc = page_rsrc(C, G, a.layer, page[g]);
    const int slot = t0 & (C.page_size - 1);
    const uint32_t base = (uint32_t)((it.kvh * C.page_size + slot) * D * 2);
#pragma unroll
    for (int j = 0; j < TG / TB; ++j) {
      const int off = j * TB + lane / CH;
      uint32_t v = base + off * (2 * D) +
                   16u * ((lane % CH) ^ chunk_swizzle<D>(tl0 + off));
      const bool in = t0 + off < it.hi && t0 + off >= it.clear;
      v = in ? v : 0x7FFFFFFFu;                      // zeros
      const uint32_t to = lds + (tl0 + j * TB) * (2 * D);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   ::"s"(to), "v"(v), "s"(rsrc)
                   : "memory");
      if (!SHARED) {
        const uint32_t vv = in ? v + G.v_off : 0x7FFFFFFFu;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     ::"s"(to + TT * 2 * D), "v"(vv), "s"(rsrc)
                     : "memory");
      }
    }
  }
}

// E4M3 pages: a stage's codes and scales into registers (16 codes per lane
// and piece), and from there as BF16 into LDS. A code times its power of two
// is exact in BF16. In two halves (where there are two pieces or more), one
// under each product, so that half the registers hold loads in flight.
template <int D, bool SHARED, int TT>
struct Codes {
  static constexpr int ALL = (TT * D + 4095) / 4096, M = SHARED ? 1 : 2;
  static constexpr bool PART = TT * D < 4096;  // the stage takes the first waves only
  static constexpr int H = ALL > 1 ? 2 : 1, N = ALL / H;  // halves, pieces of one
  uint4 c[M][N];
  uint32_t s[M][N];
  __device__ __forceinline__ void load(const DSV4GCache &C, const CacheGeom &G, const AttnArgs &a,
                                       const Item &it, int st, int half, int wave, int lane) {
    if (PART && wave * 64 * 16 >= TT * D) return;
#pragma unroll
    for (int p = 0; p < N; ++p) {
      // at most 16 tokens from here, one page
      const int tl0 = ((half * N + p) * 256 + wave * 64) * 16 / D;
      const int t0 = it.lo + st * TT + tl0;
      const int page = page_of(C, G, it, t0);
      const I4 r = page_rsrc(C, G, a.layer, page);
      const BufRsrc rsrc = buf_rsrc((const void *)(((uint64_t)(uint32_t)r[1] << 32) |
                                                   (uint32_t)r[0]), r[2]);
      const int off = lane * 16 / D, col = lane * 16 % D;
      const int slot = (t0 & (C.page_size - 1)) + off;
      const uint32_t e = (uint32_t)(it.kvh * C.page_size + slot) * D + col;
      const bool in = t0 + off < it.hi && t0 + off >= it.clear;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        c[m][p] = buf_load16(rsrc, in ? e + (m ? G.v_off : 0) : 0x7FFFFFFFu);
        s[m][p] = __builtin_amdgcn_raw_buffer_load_b8(
            rsrc, in ? e / DSV4G_CACHE_GROUP + (m ? G.vs_off : G.ks_off) : 0x7FFFFFFFu, 0, 0);
      }
    }
  }
  __device__ __forceinline__ void store(uint8_t *lds, int half, int wave, int lane) const {
    if (PART && wave * 64 * 16 >= TT * D) return;
#pragma unroll
    for (int p = 0; p < N; ++p) {
      const int tl = ((half * N + p) * 256 + wave * 64 + lane) * 16 / D, ch = lane * 16 % D / 8;
      const int g = chunk_swizzle<D>(tl);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float scale = e8m0(s[m][p]);
        const uint32_t u[4] = {c[m][p].x, c[m][p].y, c[m][p].z, c[m][p].w};
        uint32_t y[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          y[2 * k] = __builtin_bit_cast(
              uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u[k], scale, false));
          y[2 * k + 1] = __builtin_bit_cast(
              uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u[k], scale, true));
        }
        uint8_t *row = lds + m * (TT * 2 * D) + tl * (2 * D);
        *(uint4 *)(row + 16 * (ch ^ g)) = make_uint4(y[0], y[1], y[2], y[3]);
        *(uint4 *)(row + 16 * ((ch + 1) ^ g)) = make_uint4(y[4], y[5], y[6], y[7]);
      }
    }
  }
};

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
typedef uint32_t U4 __attribute__((ext_vector_type(4)));
#define DSV4_LDS(T, at) (*(__attribute__((address_space(3))) T *)(uintptr_t)(at))

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

// The denominator's reciprocal (0 where nothing was seen) and lse, with the
// head's sink joined. m in units of log2.
__device__ __forceinline__ float finish_row(const AttnArgs &a, int head, float m, float l,
                                            float *lse) {
  float f = 1.0f;
  if (a.sink) {
    const float z = a.sink[head] * LOG2E, M = fmaxf(m, z);
    if (M > -__builtin_inff()) {
      f = exp2f(m - M);  // 0 where nothing was seen
      l = l * f + exp2f(z - M);
      m = M;
    }
  }
  *lse = l != 0.0f ? (m + log2f(l)) * LN2 : -__builtin_inff();
  return l != 0.0f ? f / l : 0.0f;
}

template <int D, bool SHARED, bool FP8, int RW>
__global__ __launch_bounds__(256, (Cfg<D, SHARED, FP8, RW>::WGS)) void k_attn(DSV4GCache C,
                                                                            CacheGeom G,
                                                                            AttnArgs a) {
  typedef Cfg<D, SHARED, FP8, RW> F;
  constexpr int TT = F::TT, STAGE = F::STAGE, NBUF = F::NBUF, NP = F::NP, KS = D / 16;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[F::LDS];
  __shared__ uint32_t s_odd[F::KW];  // tokens of a stage with something not finite
  if (*C.status) return;
  Item it;
  if (!attn_item<F::ROWS, TT>(C, a, blockIdx.x, it) || it.s0 >= it.s1) return;
  if (threadIdx.x < F::KW) s_odd[threadIdx.x] = 0;
  const int tid = threadIdx.x, lane = tid % 64, h = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int rw = wave % RW, kw = wave / RW;
  // this lane's row (the last one again where there are fewer)
  const int wr0 = it.r0 + 32 * rw;
  const bool active = wr0 < it.nrows;
  const int r = min(wr0 + lane % 32, it.nrows - 1);
  const int tok = r / a.group, head = it.kvh * a.group + r % a.group;
  const int pos0 = it.len - it.count, pos = pos0 + tok;
  const int pmin = pos0 + min(wr0, it.nrows - 1) / a.group;
  const int pmax = pos0 + min(wr0 + 31, it.nrows - 1) / a.group;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;

  int page[2];
  Codes<D, SHARED, TT> codes;
  auto pages_for = [&](int st) {
    constexpr int TW = TT / 4;
#pragma unroll
    for (int g = 0; g < (TW < 16 ? 1 : TW / 16); ++g)
      page[g] = page_of(C, G, it, it.lo + st * TT + wave * TW + 16 * g);
  };
  auto check_pages = [&](int st) {  // a needed table entry that is no page
    constexpr int TW = TT / 4;
#pragma unroll
    for (int g = 0; g < (TW < 16 ? 1 : TW / 16); ++g)
    {
      const int t = it.lo + st * TT + wave * TW + 16 * g;
      if (t < it.hi && t + 15 >= it.clear && (page[g] < 0 || page[g] >= C.n_pages) && lane == 0)
        atomicOr(C.status, DSV4G_CACHE_PAGE);
    }
  };
  if (!FP8) {
#pragma unroll
    for (int i = 0; i < NBUF - 1; ++i)
      if (it.s0 + i < it.s1) {
        pages_for(it.s0 + i);
        check_pages(it.s0 + i);
        stage_bf16<D, SHARED, TT>(C, G, a, it, page, it.s0 + i, lds0 + i * STAGE, wave, lane);
      }
  } else {
    pages_for(it.s0);
    check_pages(it.s0);
#pragma unroll
    for (int i = 0; i < codes.H; ++i) {
      codes.load(C, G, a, it, it.s0, i, wave, lane);
      codes.store(lds, i, wave, lane);
    }
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
        const uint4 x = *(const uint4 *)((const uint16_t *)a.q + at + 16 * s);
        u = U4{x.x, x.y, x.z, x.w};
      }
      q[s] = __builtin_bit_cast(Bf8, u ^ sign);
    }
  }
  const float c2 = fabsf(a.scale) * LOG2E;

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
  const int shown = pos0 + it.r0 / a.group, hidden = it.hi - 1 - a.window;

  for (int st = it.s0; st < it.s1; ++st) {
    const int buf = (st - it.s0) % NBUF;
    // stage st is in LDS for every wave, and every wave is done with the one before
    if (!FP8) {
      constexpr int PER = STAGE / 4096;  // direct loads per wave and stage
      if (st + NBUF - 2 < it.s1) wait_loads<(NBUF - 2) * PER>();
      else wait_loads<0>();
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const int next = st + (FP8 ? 1 : NBUF - 1);
    const bool more = next < it.s1;
    const uint32_t to = ((next - it.s0) % NBUF) * STAGE;
    if (more) {
      pages_for(next);
      check_pages(next);
      if (FP8) codes.load(C, G, a, it, next, 0, wave, lane);
      else stage_bf16<D, SHARED, TT>(C, G, a, it, page, next, lds0 + to, wave, lane);
    }
    const int w0 = it.lo + st * TT;                 // the stage's tokens
    const int t0 = w0 + 32 * kw;                    // this wave's 32
    // 0 * NaN is NaN: where a token is hidden from some rows and not from
    // others, its values are cleared if they are not all finite (a row that
    // sees it is not finite then: by its score, or as below)
    uint32_t odd = 0;
    if (min(w0 + TT, it.hi) - 1 > shown || (a.window && max(w0, it.clear) <= hidden)) {
      constexpr int PT = 256 / TT, NB = 2 * D / PT;  // threads per token, bytes of each
      const int t = tid / PT;
      const uint32_t at = lds0 + buf * STAGE + (SHARED ? 0 : F::KB) + t * (2 * D) +
                          tid % PT * NB;
      uint32_t big = 0;
#pragma unroll
      for (int j = 0; j < NB / 16; ++j) {
        const U4 x = DSV4_LDS(U4, at + 16 * j);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          big |= ((x[k] & 0x7F80u) == 0x7F80u) | ((x[k] & 0x7F800000u) == 0x7F800000u);
      }
      if (big) atomicOr(&s_odd[t / 32], 1u << (t % 32));
      __syncthreads();
      uint32_t any = 0;
#pragma unroll
      for (int k = 0; k < F::KW; ++k) any |= s_odd[k];
      odd = __builtin_amdgcn_readfirstlane(any) ? 1u : 0u;
    }
    const bool none = !active || t0 > pmax || (a.window && t0 + 31 <= pmin - a.window);
    Bf8 p0, p1;
    if (!none) {
      F16v z;
#pragma unroll
      for (int i = 0; i < 16; ++i) z[i] = 0.0f;
      const uint32_t at = kat + buf * STAGE;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_k<D>(at, s), q[s], z, 0, 0, 0);
        if (s % 8 == 7) __builtin_amdgcn_sched_barrier(0);  // few reads ahead: registers
      }
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
      float mx = z[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, z[i]);
      mx = swap_max(mx);
      const float mt = mx > -__builtin_inff() ? mx * c2 : -__builtin_inff();
      if (__any(mt > m + AT_GROW)) {
        const float M = fmaxf(m, mt);
        const float f = M > -__builtin_inff() ? __builtin_amdgcn_exp2f(m - M) : 1.0f;
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
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        float x0 = __builtin_amdgcn_exp2f(fmaf(z[i], c2, -mu));
        float x1 = __builtin_amdgcn_exp2f(fmaf(z[i + 1], c2, -mu));
        if (mask) {  // a scale of 0 leaves -inf * 0
          x0 = z[i] == -__builtin_inff() ? 0.0f : x0;
          x1 = z[i + 1] == -__builtin_inff() ? 0.0f : x1;
        }
        l += x0 + x1;
        if (i < 8) b0[i / 2] = pack_bf16(x0, x1);
        else b1[i / 2 - 4] = pack_bf16(x0, x1);
      }
      p0 = __builtin_bit_cast(Bf8, b0);
      p1 = __builtin_bit_cast(Bf8, b1);
    }
    if (FP8 && more) {
      codes.store(lds + to, 0, wave, lane);
      if (codes.H > 1) codes.load(C, G, a, it, next, 1, wave, lane);
    }
    if (odd) {
      __syncthreads();  // every wave has its scores
      const int t = tid % TT;
      if (s_odd[t / 32] >> (t % 32) & 1) {
        const uint32_t at = lds0 + buf * STAGE + (SHARED ? 0 : F::KB) + t * (2 * D);
        for (int j = tid / TT; j < D / 8; j += 256 / TT)
          DSV4_LDS(U4, at + 16 * j) = U4{0, 0, 0, 0};
      }
      for (uint32_t left = s_odd[kw]; left; left &= left - 1) {
        const int t = t0 + __builtin_ctz(left);
        if (t <= pos && (!a.window || t > pos - a.window)) l = __builtin_nanf("");
      }
      __syncthreads();
      if (tid < F::KW) s_odd[tid] = 0;  // read again two barriers on at the earliest
    }
    if (!none) {
      const uint32_t at = vat + buf * STAGE;
#pragma unroll
      for (int d = 0; d < NP; ++d) {
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_vt<D>(at, 0, d), p0, o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_vt<D>(at, 1, d), p1, o[d], 0, 0, 0);
      }
    }
    if (FP8 && more && codes.H > 1) codes.store(lds + to, 1, wave, lane);
  }
  l = swap_sum(l);

  // the waves that shared the rows: into the first one, through LDS
  if constexpr (F::KW > 1) {
    constexpr int PART = F::PART;
    for (int k = 1; k < F::KW; ++k) {
      __syncthreads();
      float4 *w = (float4 *)(lds + rw * PART);
      float2 *ws = (float2 *)(lds + rw * PART + 32 * D * 4);
      if (kw == k) {
#pragma unroll
        for (int d = 0; d < NP; ++d) {
          const F16v y = tile_out(o[d]);
#pragma unroll
          for (int g = 0; g < 4; ++g)
            w[(4 * d + g) * 64 + lane] =
                make_float4(y[4 * g], y[4 * g + 1], y[4 * g + 2], y[4 * g + 3]);
          __builtin_amdgcn_sched_barrier(0);
        }
        ws[lane] = make_float2(m, l);
      }
      __syncthreads();
      if (kw == 0) {
        const float2 s = ws[lane];
        const float M = fmaxf(m, s.x);
        const bool any = M > -__builtin_inff();
        const float f0 = any ? exp2f(m - M) : 1.0f, f1 = any ? exp2f(s.x - M) : 0.0f;
        l = l * f0 + s.y * f1;
        m = M;
#pragma unroll
        for (int d = 0; d < NP; ++d) {
          F16v y = tile_out(o[d]);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float4 x = w[(4 * d + g) * 64 + lane];
            y[4 * g] = y[4 * g] * f0 + x.x * f1;
            y[4 * g + 1] = y[4 * g + 1] * f0 + x.y * f1;
            y[4 * g + 2] = y[4 * g + 2] * f0 + x.z * f1;
            y[4 * g + 3] = y[4 * g + 3] * f0 + x.w * f1;
          }
          tile_in(o[d], y);
        }
      }
    }
    if (kw) return;
  }
  if (!active || wr0 + lane % 32 >= it.nrows) return;
  if (it.parts > 1) {
    float4 *w = (float4 *)(a.part + ((size_t)blockIdx.x * F::ROWS + 32 * rw) * D);
#pragma unroll
    for (int d = 0; d < NP; ++d) {
      const F16v y = tile_out(o[d]);
#pragma unroll
      for (int g = 0; g < 4; ++g)
        w[(4 * d + g) * 64 + lane] =
            make_float4(y[4 * g], y[4 * g + 1], y[4 * g + 2], y[4 * g + 3]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (h == 0) a.stat[(size_t)blockIdx.x * F::ROWS + 32 * rw + lane] = make_float2(m, l);
    return;
  }
  float lse;
  const float f = finish_row(a, head, m, l, &lse);
  const size_t row = (size_t)(it.start + tok);
#pragma unroll
  for (int d = 0; d < NP; ++d) {
    store_tile<D>(a, row * a.out_stride + (size_t)head * D, d, h, tile_out(o[d]), f);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (a.lse && h == 0) a.lse[row * a.heads + head] = lse;
}

// Joins the parts of every split item: one wave per output tile of a row wave.
template <int D, int RW>
__global__ __launch_bounds__(256) void k_attn_join(DSV4GCache C, AttnArgs a) {
  constexpr int TT = 32 * (4 / RW), ROWS = 32 * RW, NP = D / 32;
  if (*C.status) return;
  const int lane = threadIdx.x % 64, h = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  int id = blockIdx.x * 4 + wave;
  const int d = id % NP;
  id /= NP;
  const int rw = id % RW;
  id /= RW;
  if (id >= a.items) return;
  Item it;
  if (!attn_item<ROWS, TT>(C, a, id * a.nsplit, it) || it.parts == 1) return;
  const int r = it.r0 + 32 * rw + lane % 32;
  if (r >= it.nrows) return;
  const size_t first = (size_t)id * a.nsplit;
  const float2 *stat = a.stat + first * ROWS + 32 * rw + lane % 32;
  float m = -__builtin_inff(), l = 0.0f;
  for (int p = 0; p < it.parts; ++p) m = fmaxf(m, stat[(size_t)p * ROWS].x);
  const float mu = m > -__builtin_inff() ? m : 0.0f;
  F16v o;
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = 0.0f;
#pragma unroll 4
  for (int p = 0; p < it.parts; ++p) {
    const float2 s = stat[(size_t)p * ROWS];
    const float f = exp2f(s.x - mu);
    l += s.y * f;
    const float4 *w = (const float4 *)(a.part + ((first + p) * ROWS + 32 * rw) * D);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 x = w[(4 * d + g) * 64 + lane];
      o[4 * g] += x.x * f;
      o[4 * g + 1] += x.y * f;
      o[4 * g + 2] += x.z * f;
      o[4 * g + 3] += x.w * f;
    }
  }
  const int tok = r / a.group, head = it.kvh * a.group + r % a.group;
  float lse;
  const float f = finish_row(a, head, m, l, &lse);
  const size_t row = (size_t)(it.start + tok);
  store_tile<D>(a, row * a.out_stride + (size_t)head * D, d, h, o, f);
  if (a.lse && h == 0 && d == 0) a.lse[row * a.heads + head] = lse;
}

// ------------------------------------------------------------- launch plan
struct AttnPlan {
  int rw, tiles, nsplit;
  long items;
  size_t bytes;
};
static AttnPlan attn_plan(const DSV4GCache *C, int heads, int n_seqs, int n_tokens, int max_q,
                          int max_kv, int window) {
  AttnPlan p;
  const long room = (long)C->max_pages * C->page_size;
  max_q = max_q > n_tokens ? n_tokens : max_q;
  max_kv = max_kv > room ? (int)room : max_kv;
  const long rows = (long)max_q * (heads / C->kv_heads);
  const int D = C->k_dim;
  // the smallest tile that holds a sequence's rows
  const int least = D == 512 || (D == 256 && C->v_dim) ? 2 : 1;
  p.rw = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  p.rw = p.rw < least ? least : p.rw;
  p.tiles = (int)((rows + 32 * p.rw - 1) / (32 * p.rw));
  p.items = (long)p.tiles * n_seqs * C->kv_heads;
  const int tt = 32 * (4 / p.rw);
  long range = max_kv;
  if (window && (long)window + 32L * p.rw < range) range = window + 32L * p.rw;
  const long slots = 256L * (D <= 128 ? 2 : 1);
  long want = slots / p.items;
  const long most = (range + 2 * tt - 1) / (2 * tt);
  want = want > most ? most : want;
  want = want > AT_MAX_SPLIT ? AT_MAX_SPLIT : want;
  p.nsplit = want < 1 ? 1 : (int)want;
  const size_t cells = (size_t)p.items * p.nsplit * 32 * p.rw;
  p.bytes = p.nsplit > 1 ? cells * (D * sizeof(float) + sizeof(float2)) : 0;
  return p;
}

template <int D, bool SHARED, bool FP8, int RW>
static void attn_launch(const DSV4GCache &C, const CacheGeom &G, const AttnArgs &a, long items,
                        hipStream_t st) {
  if constexpr (Cfg<D, SHARED, FP8, RW>::OK) {
    hipLaunchKernelGGL((k_attn<D, SHARED, FP8, RW>), dim3((unsigned)(items * a.nsplit)), dim3(256),
                       0, st, C, G, a);
    if (a.nsplit > 1)
      hipLaunchKernelGGL((k_attn_join<D, RW>), dim3((unsigned)((items * RW * (D / 32) + 3) / 4)),
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
  if (!(fabsf(scale) <= 3.4028235e38f))
    return dsv4g_fail(DSV4G_EINVAL, "attention: scale %g", scale);
  const size_t unit = act_dtype == DSV4G_DT_F32 ? 4 : 8;  // elements of 16 bytes
  if (q_stride < (size_t)heads * C->k_dim || out_stride < (size_t)heads * C->k_dim ||
      q_stride % unit || out_stride % unit || ((uintptr_t)q & 15) || ((uintptr_t)out & 15))
    return dsv4g_fail(DSV4G_EINVAL, "attention: rows of q and out must be 16-byte aligned and at "
                      "least heads * dim apart");
  const AttnPlan p = attn_plan(C, heads, n_seqs, n_tokens, max_q, max_kv, window);
  if (p.items * p.nsplit > 0x7FFFFFFFL || (long)max_q * (heads / C->kv_heads) > 0x7FFFFF00L)
    return dsv4g_fail(DSV4G_EINVAL, "attention: too many rows for one call");
  if (p.bytes && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < p.bytes))
    return dsv4g_fail(DSV4G_EINVAL, "attention: 256-byte aligned workspace of %zu bytes needed "
                      "(%zu given)", p.bytes, workspace_bytes);
  AttnArgs a = {};
  a.out = out, a.lse = lse, a.q = q, a.out_stride = out_stride, a.q_stride = q_stride;
  a.seqs = seqs, a.starts = starts, a.sink = sink, a.layer = layer, a.heads = heads;
  a.group = heads / C->kv_heads, a.n_seqs = n_seqs, a.n_tokens = n_tokens, a.max_q = max_q;
  a.max_kv = max_kv, a.window = window, a.f32 = act_dtype == DSV4G_DT_F32;
  a.tiles = p.tiles, a.nsplit = p.nsplit, a.items = (int)p.items, a.scale = scale;
  a.part = (float *)workspace;
  if (p.nsplit > 1) a.stat = (float2 *)(a.part + (size_t)p.items * p.nsplit * 32 * p.rw * C->k_dim);
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
