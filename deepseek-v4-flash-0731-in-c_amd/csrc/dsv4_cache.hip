// dsv4_cache.hip - the paged cache of the attention half: append, and the
// bookkeeping of its pages (reserve with copy-on-write, fork, free, compact).
// Layout, lists and status word: include/dsv4_gpu.h. No counterpart in the
// reference, whose cache is host memory of one sequence.
//
// The state is two arrays of whole numbers, the users of each page and the
// sequences' tables, with no free list: a page is free where ref is 0, and
// pages are handed out and moved in ascending order, so that every call has
// one right result, whatever the order of its threads. One workgroup decides
// (prefix sums over the list and over ref), a second launch moves the pages'
// bytes with as many workgroups as the memory wants.
#include "dsv4_cache.h"
#include "dsv4_device.h"
#include "dsv4_gpu_internal.h"

namespace dsv4 {

// An append may neither wait for its other waves nor be stopped by what they
// report: it sets its bits one byte up, and is blocked by those of the lowest.
constexpr int CACHE_APPEND = DSV4G_CACHE_BY_APPEND;
__host__ __device__ inline unsigned cache_bits(unsigned status) {
  return (status | status >> CACHE_APPEND) & ((1u << CACHE_APPEND) - 1);
}

constexpr int CB_T = 1024;  // threads of a deciding workgroup (and most listed sequences)
constexpr int CB_PER = 8;   // refs per thread and step of a scan over the pool
static_assert(CB_T == DSV4G_CACHE_MAX_SEQS, "one thread per listed sequence");

// Words of the workspace: [0] moves, [1] pages in use; then the moves'
// sources, their destinations, and a third list (reserve: the free pages it
// found; compact: where each page behind the used ones went).
constexpr int CW_HEAD = 64;
struct CacheWs {
  int *head, *src, *dst, *aux;
};
__host__ __device__ inline CacheWs cache_ws(void *p, int n_pages) {
  int *w = (int *)p;
  return {w, w + CW_HEAD, w + CW_HEAD + (size_t)n_pages, w + CW_HEAD + 2 * (size_t)n_pages};
}

// Exclusive prefix of v over the workgroup's threads; *total is the sum.
// s: CB_T / 64 words of LDS. Ends behind a barrier, begins with one.
__device__ __forceinline__ int block_prefix(int v, int *s, int *total) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) s[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < CB_T / 64; ++w) {
    const int t = s[w];
    before += w < wave ? t : 0;
    all += t;
  }
  *total = all;
  return before + x - v;
}

__global__ __launch_bounds__(256) void k_cache_init(DSV4GCache C) {
  const size_t step = (size_t)gridDim.x * 256, t = (size_t)blockIdx.x * 256 + threadIdx.x;
  const size_t cells = (size_t)C.n_seqs * C.max_pages;
  for (size_t i = t; i < (size_t)C.n_pages; i += step) C.ref[i] = 0;
  for (size_t i = t; i < cells; i += step) C.table[i] = -1;
  for (size_t i = t; i < (size_t)C.n_seqs; i += step) C.len[i] = 0;
  if (t == 0) *C.status = 0;
}

__global__ void k_cache_clear_status(unsigned *status) { *status = 0; }

// Room for the new tokens of n listed sequences: a thread per sequence counts
// the pages it needs, the pool is scanned from its start until enough free
// pages are found, and only then anything is changed. One workgroup; bound by
// the latency of its dependent steps (list -> length -> table -> ref -> scan):
// 9.4 to 10.5 us for 16 sequences and 512 pages, and no less with the counts
// loaded ahead.
__global__ __launch_bounds__(CB_T) void k_cache_reserve(DSV4GCache C, const int *seqs,
                                                        const int *starts, int n, int *ws) {
  __shared__ int s_seq[CB_T], s_page[CB_T], s_off[CB_T], s_at[CB_T], s_copy[CB_T];
  __shared__ int s_scan[CB_T / 64];
  const CacheWs w = cache_ws(ws, C.n_pages);
  const int t = threadIdx.x;
  if (t == 0) w.head[0] = 0;
  const unsigned status = *C.status;  // not 0 for every thread, or for none
  if (status) {
    // appends of the step that was refused are over: from here on their
    // refusals block appends, too
    if (t == 0) *C.status = cache_bits(status);
    return;
  }
  const int ps = C.page_size, room = C.max_pages;
  int s = -1, count = 0, L = 0, P = -1, full = 0;
  bool bad = false, bad_page = false;
  if (t < n) {
    s = seqs ? seqs[t] : t;
    const long c = (long)starts[t + 1] - starts[t];
    bad = s < 0 || s >= C.n_seqs || c < 0;
    if (!bad) {
      L = C.len[s];
      bad = L < 0 || L + c > (long)room * ps;
    }
    if (!bad) {
      count = (int)c;
      full = (L + ps - 1) / ps;  // pages it holds
      if (count && L % ps) {
        P = C.table[(size_t)s * room + L / ps];
        bad_page = P < 0 || P >= C.n_pages;
      }
    }
  }
  s_seq[t] = s;
  s_page[t] = P;
  __syncthreads();
  int before = 0;  // earlier listed sequences that would write into the same page
  if (t < n && !bad && !bad_page)
    for (int j = 0; j < n; ++j) {
      bad |= j != t && s_seq[j] == s;
      before += j < t && P >= 0 && s_page[j] == P;
    }
  const int cow = !bad && !bad_page && P >= 0 && C.ref[P] - before > 1;
  const int need = bad || bad_page ? 0 : (L + count + ps - 1) / ps - full + cow;
  const int any_bad = __syncthreads_or(bad), any_page = __syncthreads_or(bad_page);
  if (any_bad || any_page) {
    if (t == 0)
      *C.status = (any_bad ? DSV4G_CACHE_LIST : 0) | (any_page ? DSV4G_CACHE_PAGE : 0);
    return;
  }
  // Prefixes in 32 bits: a sum that passes them (more than the pool holds) is
  // caught thread by thread first.
  if (__syncthreads_or(need > C.n_pages)) {
    if (t == 0) *C.status = DSV4G_CACHE_FULL;
    return;
  }
  int total, copies;
  const int off = block_prefix(need, s_scan, &total);  // n_pages < 2^20: below 2^30
  const int copy_at = block_prefix(cow, s_scan, &copies);
  s_off[t] = off;
  s_copy[t] = cow ? copy_at : -1;
  s_at[t] = full - cow;  // column of the first page given to it
  // the lowest free pages, until enough
  int found = 0;
  for (int base = 0; base < C.n_pages && found < total; base += CB_T * CB_PER) {
    const int i0 = base + t * CB_PER;
    int r[CB_PER], mine = 0;
#pragma unroll
    for (int k = 0; k < CB_PER; ++k) r[k] = i0 + k < C.n_pages ? C.ref[i0 + k] : 1;
#pragma unroll
    for (int k = 0; k < CB_PER; ++k) mine += r[k] == 0;
    int here;
    int g = found + block_prefix(mine, s_scan, &here);
#pragma unroll
    for (int k = 0; k < CB_PER; ++k)
      if (r[k] == 0) {
        if (g < total) w.aux[g] = i0 + k;
        ++g;
      }
    found += here;
  }
  if (found < total) {
    if (t == 0) *C.status = DSV4G_CACHE_FULL;
    return;
  }
  __syncthreads();  // the list (the barrier also orders its global stores in the workgroup)
  for (int g = t; g < total; g += CB_T) {
    int lo = 0, hi = n - 1;  // the last sequence whose range begins at or before g
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (s_off[mid] <= g) lo = mid;
      else hi = mid - 1;
    }
    const int page = w.aux[g], k = g - s_off[lo];
    C.ref[page] = 1;
    int *cell = C.table + (size_t)s_seq[lo] * room + s_at[lo] + k;
    if (k == 0 && s_copy[lo] >= 0) {
      w.src[s_copy[lo]] = s_page[lo];
      w.dst[s_copy[lo]] = page;
      atomicSub(&C.ref[s_page[lo]], 1);  // whole numbers: any order gives the same
    }
    *cell = page;
  }
  if (t < n) C.len[s] = L + count;
  if (t == 0) w.head[0] = copies;
}

// Moves the pages of the workspace's list, every layer's (items of 16 KB, 4
// 16-byte loads in flight per thread), and with remap the table entries of the
// pages that moved. The list's pages are all different and no destination is
// a source, so nothing is ordered. Bound by HBM: 536 MB in 107 us (5.0 TB/s; a
// pool of 2048 pages and 16 layers). 46 MB over 43 layers' pages take 20 us,
// 2.3 TB/s: first touches of pages all over a pool of 0.7 GB. Items of even size
// and 32-bit divisions changed neither.
constexpr int CM_CHUNK = 16384;
__global__ __launch_bounds__(256) void k_cache_move(DSV4GCache C, int *ws, size_t page_bytes,
                                                    int remap) {
  const CacheWs w = cache_ws(ws, C.n_pages);
  const int per = (int)((page_bytes + CM_CHUNK - 1) / CM_CHUNK);
  const long items = (long)w.head[0] * C.n_layers * per;
  for (long i = blockIdx.x; i < items; i += gridDim.x) {
    const int part = (int)(i % per);
    const long u = i / per;
    const int layer = (int)(u % C.n_layers), m = (int)(u / C.n_layers);
    const size_t at = (size_t)layer * C.n_pages;
    const uint8_t *from = C.pages + (at + w.src[m]) * page_bytes;
    uint8_t *to = C.pages + (at + w.dst[m]) * page_bytes;
    uint4 v[4];
    size_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      o[k] = (size_t)part * CM_CHUNK + 16u * (threadIdx.x + 256u * k);
      if (o[k] < page_bytes) v[k] = *(const uint4 *)(from + o[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (o[k] < page_bytes) *(uint4 *)(to + o[k]) = v[k];
  }
  if (!remap) return;
  const int used = w.head[1];
  const size_t cells = (size_t)C.n_seqs * C.max_pages;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < cells; i += (size_t)gridDim.x * 256) {
    const int e = C.table[i];
    if (e >= used && e < C.n_pages) C.table[i] = w.aux[e];
  }
}

// Whether entries from .. to - 1 of a sequence's row name pages, for all
// threads of the workgroup; a barrier.
__device__ __forceinline__ bool pages_good(const DSV4GCache &C, const int *row, int from, int to) {
  bool bad = false;
  for (int k = from + threadIdx.x; k < to; k += 256) bad |= row[k] < 0 || row[k] >= C.n_pages;
  return !__syncthreads_or(bad);
}

// A workgroup per pair, which first looks for what conflicts: a child named
// twice or as a parent, lengths, entries of the parent that are no pages.
__global__ __launch_bounds__(256) void k_cache_fork(DSV4GCache C, const int *parents,
                                                    const int *children, int n) {
  const int i = blockIdx.x, t = threadIdx.x;
  const int p = parents[i], c = children[i];
  bool bad = p < 0 || p >= C.n_seqs || c < 0 || c >= C.n_seqs;
  for (int j = t; j < n; j += 256) bad |= (j != i && children[j] == c) || parents[j] == c;
  int L = 0;
  if (!bad) {
    L = C.len[p];
    bad = C.len[c] != 0 || L < 0 || L > (long)C.max_pages * C.page_size;
  }
  // every thread has read the child's length before it is written
  if (__syncthreads_or(bad)) {
    if (t == 0) atomicOr(C.status, DSV4G_CACHE_LIST);
    return;
  }
  const int held = (L + C.page_size - 1) / C.page_size;
  const int *from = C.table + (size_t)p * C.max_pages;
  int *to = C.table + (size_t)c * C.max_pages;
  if (!pages_good(C, from, 0, held)) {
    if (t == 0) atomicOr(C.status, DSV4G_CACHE_PAGE);
    return;
  }
  for (int k = t; k < C.max_pages; k += 256) {
    const int e = k < held ? from[k] : -1;
    to[k] = e;
    if (k < held) atomicAdd(&C.ref[e], 1);
  }
  if (t == 0) C.len[c] = L;
}

__global__ __launch_bounds__(256) void k_cache_free(DSV4GCache C, const int *seqs,
                                                    const int *new_len, int n) {
  const int i = blockIdx.x, t = threadIdx.x;
  const int s = seqs ? seqs[i] : i, to = new_len ? new_len[i] : 0;
  bool bad = s < 0 || s >= C.n_seqs;
  if (seqs)
    for (int j = t; j < n; j += 256) bad |= j != i && seqs[j] == s;
  int L = 0;
  if (!bad) {
    L = C.len[s];
    bad = to < 0 || to > L || L > (long)C.max_pages * C.page_size;
  }
  if (__syncthreads_or(bad)) {
    if (t == 0) atomicOr(C.status, DSV4G_CACHE_LIST);
    return;
  }
  const int ps = C.page_size, held = (L + ps - 1) / ps, kept = (to + ps - 1) / ps;
  int *row = C.table + (size_t)s * C.max_pages;
  if (!pages_good(C, row, kept, held)) {
    if (t == 0) atomicOr(C.status, DSV4G_CACHE_PAGE);
    return;
  }
  for (int k = kept + t; k < held; k += 256) {
    atomicSub(&C.ref[row[k]], 1);
    row[k] = -1;
  }
  if (t == 0) C.len[s] = to;
}

// Which pages move: one pass counts the used ones (n), one lists the free ones
// before n and the used ones at or behind it, both in ascending order; there
// are as many of the one as of the other.
__global__ __launch_bounds__(CB_T) void k_cache_compact(DSV4GCache C, int *n_used, int *ws) {
  __shared__ int s_scan[CB_T / 64];
  const CacheWs w = cache_ws(ws, C.n_pages);
  const int t = threadIdx.x;
  int mine = 0, used;
  for (int base = 0; base < C.n_pages; base += CB_T * CB_PER) {
    const int i0 = base + t * CB_PER;
#pragma unroll
    for (int k = 0; k < CB_PER; ++k) mine += i0 + k < C.n_pages && C.ref[i0 + k] > 0;
  }
  block_prefix(mine, s_scan, &used);
  int holes = 0, tails = 0;
  for (int base = 0; base < C.n_pages; base += CB_T * CB_PER) {
    const int i0 = base + t * CB_PER;
    int r[CB_PER], both = 0;
#pragma unroll
    for (int k = 0; k < CB_PER; ++k) {
      const int i = i0 + k;
      r[k] = i < C.n_pages ? C.ref[i] : 0;
      // two counts in one word: at most CB_T * CB_PER = 8192 of each
      both += i >= C.n_pages ? 0 : i < used ? (r[k] <= 0) : (r[k] > 0) << 16;
    }
    int here;
    const int g = block_prefix(both, s_scan, &here);
    int h = holes + (g & 0xFFFF), l = tails + (g >> 16);
#pragma unroll
    for (int k = 0; k < CB_PER; ++k) {
      const int i = i0 + k;
      if (i >= C.n_pages) continue;
      if (i < used) {
        if (r[k] <= 0) w.dst[h++] = i;
      } else {
        if (r[k] > 0) w.src[l++] = i;
        else w.aux[i] = -1;
      }
    }
    holes += here & 0xFFFF;
    tails += here >> 16;
  }
  __syncthreads();
  for (int m = t; m < tails; m += CB_T) {
    const int from = w.src[m], to = w.dst[m];
    C.ref[to] = C.ref[from];
    C.ref[from] = 0;
    w.aux[from] = to;
  }
  if (t == 0) {
    w.head[0] = tails;
    w.head[1] = used;
    if (n_used) *n_used = used;
  }
}

// ------------------------------------------------------------------ append
// One wave per new token: its place by counting the starts at or before its
// row, then 8 columns per lane and step (8 neighbouring lanes are one scale
// group of 64 columns). Bound: HBM for many tokens (4096 of 8 kv heads of 128
// and 128: 53 MB in 11.8 to 12.1 us, 4.5 TB/s), the latency of starts -> sequence
// -> length -> table entry -> store for few (64 latent rows: 4.1 to 4.6 us).
template <bool F32, bool FP8>
__global__ __launch_bounds__(256) void k_cache_append(DSV4GCache C, CacheGeom G, int layer,
                                                      const void *k, size_t k_stride,
                                                      const void *v, size_t v_stride,
                                                      const int *seqs, const int *starts, int n,
                                                      int n_tokens) {
  const int lane = threadIdx.x % 64;
  const int row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  // of earlier calls: waves of this one set others
  if (row >= n_tokens || (*C.status & ((1u << CACHE_APPEND) - 1))) return;
  // starts[0] <= .. <= starts[n]: the sequence is the number of starts at or
  // before the row, less one. Starts that fall somewhere place no row.
  int b = -1;
  bool falls = false;
  for (int j = 0; j <= n; j += 64) {
    const int at = j + lane;
    const int from = at <= n ? starts[at] : 0x7FFFFFFF;
    b += __popcll(__ballot(from <= row));
    falls |= __ballot(at < n && starts[at + 1] < from) != 0;
  }
  // entries that reach out of the call's rows are reported by the first row:
  // they may have none
  const bool out = row == 0 && (starts[0] < 0 || starts[n] > n_tokens);
  if ((falls || out) && lane == 0) atomicOr(C.status, DSV4G_CACHE_LIST << CACHE_APPEND);
  if (falls || b < 0 || b >= n) return;  // b: in front of the first sequence or behind the last
  const int s = seqs ? seqs[b] : b;
  bool twice = false;
  if (seqs)
    for (int j = 0; j < n; j += 64) {
      const int at = j + lane;
      twice |= __ballot(at < n && at != b && seqs[at] == s) != 0;
    }
  // the whole entry is good or none of its rows is written
  int pos = -1;
  if (s >= 0 && s < C.n_seqs && !twice) {
    const int first = starts[b], end = starts[b + 1], len = C.len[s];
    if (first >= 0 && end <= n_tokens && len >= end - first &&
        len <= (long)C.max_pages * C.page_size)
      pos = len - end + row;
  }
  if (pos < 0) {
    if (lane == 0) atomicOr(C.status, DSV4G_CACHE_LIST << CACHE_APPEND);
    return;
  }
  const int page = C.table[(size_t)s * C.max_pages + (pos >> G.shift)];
  if (page < 0 || page >= C.n_pages) {
    if (lane == 0) atomicOr(C.status, DSV4G_CACHE_PAGE << CACHE_APPEND);
    return;
  }
  uint8_t *base = C.pages + ((size_t)layer * C.n_pages + page) * G.page_bytes;
  const int slot = pos & (C.page_size - 1);
  const int kc = C.kv_heads * C.k_dim / 8, vc = C.kv_heads * C.v_dim / 8;
  for (int c = lane; c < kc + vc; c += 64) {
    const bool is_v = c >= kc;
    const int dim = is_v ? C.v_dim : C.k_dim, col = 8 * (is_v ? c - kc : c);
    const int head = col / dim, at = col - head * dim;
    const size_t o = (size_t)row * (is_v ? v_stride : k_stride) + col;
    const void *from = is_v ? v : k;
    float x[8];
    if (F32) {
      const float4 a = *(const float4 *)((const float *)from + o);
      const float4 e = *(const float4 *)((const float *)from + o + 4);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
      x[4] = e.x, x[5] = e.y, x[6] = e.z, x[7] = e.w;
    } else {
      const uint4 a = *(const uint4 *)((const uint16_t *)from + o);
      const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = u2f(u[j] << 16);
        x[2 * j + 1] = u2f(u[j] & 0xFFFF0000u);
      }
    }
    // element offset inside the page's keys or values
    const size_t e = ((size_t)head * C.page_size + slot) * dim + at;
    if (!FP8) {
      uint4 y;
      uint32_t *py = (uint32_t *)&y;
#pragma unroll
      for (int j = 0; j < 4; ++j) py[j] = pack_bf16(x[2 * j], x[2 * j + 1]);
      *(uint4 *)(base + (is_v ? G.v_off : 0) + 2 * e) = y;
      continue;
    }
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = fabsf(x[j]);
      amax = a <= 3.4028235e38f && a > amax ? a : amax;  // finite values only
    }
#pragma unroll
    for (int o8 = 1; o8 < 8; o8 <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o8, 64));
    const uint32_t code = f2u(act_scale(amax)) >> 23;  // a power of two, normal
    const float inv = u2f((254u - code) << 23);
    uint32_t y[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t lo = 0;
      float q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = x[4 * j + i];
        q[i] = fminf(fmaxf(f * inv, -448.0f), 448.0f);
      }
      lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
      lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
#pragma unroll
      for (int i = 0; i < 4; ++i)  // NaN and infinities: code 0x7F
        if (!(fabsf(x[4 * j + i]) <= 3.4028235e38f)) lo |= 0x7Fu << (8 * i);
      y[j] = lo;
    }
    *(uint2 *)(base + (is_v ? G.v_off : 0) + e) = make_uint2(y[0], y[1]);
    if (lane % 8 == 0)
      base[(is_v ? G.vs_off : G.ks_off) + e / DSV4G_CACHE_GROUP] = (uint8_t)code;
  }
}

}  // namespace dsv4

using namespace dsv4;

extern "C" {

size_t dsv4g_cache_page_bytes(const DSV4GCache *C) {
  CacheGeom G;
  return C && cache_geom(C, &G) ? G.page_bytes : 0;
}

// The descriptor's own checks, for every entry that takes one.
int dsv4g_cache_ok(const DSV4GCache *C, CacheGeom *G, const char *who) {
  if (!C || !cache_geom(C, G))
    return dsv4g_fail(DSV4G_EINVAL, "%s: not a cache shape (page_size a power of two 16..256, "
                      "k_dim = v_dim 64, 128 or 256, or v_dim 0 and k_dim 256 or 512, BF16 or "
                      "E4M3)", who);
  if (!C->pages || !C->ref || !C->table || !C->len || !C->status)
    return dsv4g_fail(DSV4G_EINVAL, "%s: a cache pointer is NULL", who);
  if ((uintptr_t)C->pages & 255)
    return dsv4g_fail(DSV4G_EINVAL, "%s: pages must be 256-byte aligned", who);
  return 0;
}

size_t dsv4g_cache_workspace_bytes(const DSV4GCache *C) {
  CacheGeom G;
  if (!C || !cache_geom(C, &G)) return 0;
  return (CW_HEAD + 3 * (size_t)C->n_pages) * sizeof(int);
}

static int cache_ws_ok(const DSV4GCache *C, const void *ws, size_t bytes, const char *who) {
  const size_t need = dsv4g_cache_workspace_bytes(C);
  if (!ws || ((uintptr_t)ws & 255) || bytes < need)
    return dsv4g_fail(DSV4G_EINVAL, "%s: 256-byte aligned workspace of %zu bytes needed (%zu "
                      "given)", who, need, bytes);
  return 0;
}

static int cache_list_ok(int n, const char *who) {
  if (n <= 0 || n > DSV4G_CACHE_MAX_SEQS)
    return dsv4g_fail(DSV4G_EINVAL, "%s: %d sequences listed, 1..%d allowed", who, n,
                      DSV4G_CACHE_MAX_SEQS);
  return 0;
}

int dsv4g_cache_init(const DSV4GCache *C, void *stream) {
  CacheGeom G;
  DSV4G_TRY(dsv4g_cache_ok(C, &G, "cache_init"));
  hipLaunchKernelGGL(k_cache_init, dim3(256), dim3(256), 0, (hipStream_t)stream, *C);
  return dsv4g_check_launch("cache_init");
}

int dsv4g_cache_status(unsigned *status_out, const DSV4GCache *C, void *stream) {
  CacheGeom G;
  DSV4G_TRY(dsv4g_cache_ok(C, &G, "cache_status"));
  if (!status_out) return dsv4g_fail(DSV4G_EINVAL, "cache_status: no place for the status");
  hipStream_t st = (hipStream_t)stream;
  DSV4G_HIP(hipMemcpyAsync(status_out, C->status, sizeof(unsigned), hipMemcpyDeviceToHost, st));
  DSV4G_HIP(hipStreamSynchronize(st));
  if (*status_out) {
    hipLaunchKernelGGL(k_cache_clear_status, dim3(1), dim3(1), 0, st, C->status);
    DSV4G_TRY(dsv4g_check_launch("cache_status"));
    *status_out = cache_bits(*status_out);
  }
  return 0;
}

static int cache_move(const DSV4GCache *C, const CacheGeom &G, void *ws, int remap,
                      hipStream_t st) {
  hipLaunchKernelGGL(k_cache_move, dim3(2048), dim3(256), 0, st, *C, (int *)ws, G.page_bytes,
                     remap);
  return dsv4g_check_launch("cache_move");
}

int dsv4g_cache_reserve(const DSV4GCache *C, const int *seqs, const int *starts, int n_seqs,
                        void *workspace, size_t workspace_bytes, void *stream) {
  CacheGeom G;
  DSV4G_TRY(dsv4g_cache_ok(C, &G, "cache_reserve"));
  DSV4G_TRY(cache_list_ok(n_seqs, "cache_reserve"));
  DSV4G_TRY(cache_ws_ok(C, workspace, workspace_bytes, "cache_reserve"));
  if (!starts) return dsv4g_fail(DSV4G_EINVAL, "cache_reserve: starts is NULL");
  hipLaunchKernelGGL(k_cache_reserve, dim3(1), dim3(CB_T), 0, (hipStream_t)stream, *C, seqs,
                     starts, n_seqs, (int *)workspace);
  DSV4G_TRY(dsv4g_check_launch("cache_reserve"));
  return cache_move(C, G, workspace, 0, (hipStream_t)stream);
}

int dsv4g_cache_append(const DSV4GCache *C, int layer, const void *k, size_t k_stride,
                       const void *v, size_t v_stride, int act_dtype, const int *seqs,
                       const int *starts, int n_seqs, int n_tokens, void *stream) {
  CacheGeom G;
  DSV4G_TRY(dsv4g_cache_ok(C, &G, "cache_append"));
  if (!k || !starts || n_seqs <= 0 || n_tokens <= 0 || layer < 0 || layer >= C->n_layers ||
      (act_dtype != DSV4G_DT_F32 && act_dtype != DSV4G_DT_BF16) || !v != !C->v_dim)
    return dsv4g_fail(DSV4G_EINVAL, "cache_append: bad arguments");
  if (n_tokens > 0x3FFFFFF)  // a wave each, a launch is below 2^32 threads
    return dsv4g_fail(DSV4G_EINVAL, "cache_append: %d tokens, at most 2^26 - 1", n_tokens);
  if (n_seqs > 0x3FFFFFF)  // counted in steps of a wave
    return dsv4g_fail(DSV4G_EINVAL, "cache_append: %d sequences, at most 2^26 - 1", n_seqs);
  const size_t unit = act_dtype == DSV4G_DT_F32 ? 4 : 8;  // elements of 16 bytes
  if (k_stride < (size_t)C->kv_heads * C->k_dim || (v && v_stride < (size_t)C->kv_heads * C->v_dim) ||
      ((uintptr_t)k & 15) || ((uintptr_t)v & 15) || k_stride % unit || (v && v_stride % unit))
    return dsv4g_fail(DSV4G_EINVAL, "cache_append: rows must be 16-byte aligned and at least "
                      "kv_heads * dim apart");
  const bool f32 = act_dtype == DSV4G_DT_F32, fp8 = C->dtype == DSV4G_DT_F8_E4M3;
  auto kern = f32 ? (fp8 ? k_cache_append<true, true> : k_cache_append<true, false>)
                  : (fp8 ? k_cache_append<false, true> : k_cache_append<false, false>);
  hipLaunchKernelGGL(kern, dim3((unsigned)(((long)n_tokens + 3) / 4)), dim3(256), 0,
                     (hipStream_t)stream, *C, G, layer, k, k_stride, v, v_stride, seqs, starts,
                     n_seqs, n_tokens);
  return dsv4g_check_launch("cache_append");
}

int dsv4g_cache_fork(const DSV4GCache *C, const int *parents, const int *children, int n_seqs,
                     void *stream) {
  CacheGeom G;
  DSV4G_TRY(dsv4g_cache_ok(C, &G, "cache_fork"));
  DSV4G_TRY(cache_list_ok(n_seqs, "cache_fork"));
  if (!parents || !children)
    return dsv4g_fail(DSV4G_EINVAL, "cache_fork: parents and children needed");
  hipLaunchKernelGGL(k_cache_fork, dim3(n_seqs), dim3(256), 0, (hipStream_t)stream, *C, parents,
                     children, n_seqs);
  return dsv4g_check_launch("cache_fork");
}

int dsv4g_cache_free(const DSV4GCache *C, const int *seqs, const int *new_len, int n_seqs,
                     void *stream) {
  CacheGeom G;
  DSV4G_TRY(dsv4g_cache_ok(C, &G, "cache_free"));
  DSV4G_TRY(cache_list_ok(n_seqs, "cache_free"));
  hipLaunchKernelGGL(k_cache_free, dim3(n_seqs), dim3(256), 0, (hipStream_t)stream, *C, seqs,
                     new_len, n_seqs);
  return dsv4g_check_launch("cache_free");
}

int dsv4g_cache_compact(const DSV4GCache *C, int *n_used, void *workspace,
                        size_t workspace_bytes, void *stream) {
  CacheGeom G;
  DSV4G_TRY(dsv4g_cache_ok(C, &G, "cache_compact"));
  DSV4G_TRY(cache_ws_ok(C, workspace, workspace_bytes, "cache_compact"));
  hipLaunchKernelGGL(k_cache_compact, dim3(1), dim3(CB_T), 0, (hipStream_t)stream, *C, n_used,
                     (int *)workspace);
  DSV4G_TRY(dsv4g_check_launch("cache_compact"));
  return cache_move(C, G, workspace, 1, (hipStream_t)stream);
}

}  // extern "C"
