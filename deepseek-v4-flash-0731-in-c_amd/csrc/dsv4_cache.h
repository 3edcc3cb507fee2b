// dsv4_cache.h - the paged cache's page layout, shared by its bookkeeping
// (dsv4_cache.hip) and the attention over it (dsv4_attention.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "dsv4_gpu.h"

// Byte offsets inside a page (the keys start it).
struct CacheGeom {
  size_t page_bytes;
  int v_off, ks_off, vs_off;  // values, the keys' scale codes, the values'
  int shift;                  // log2 of page_size
};

// 256 MiB per page and 2^20 pages per layer at most: the offsets inside a
// page and the sums over the pool then fit 32 bits.
inline bool cache_geom(const DSV4GCache *C, CacheGeom *G) {
  const int ps = C->page_size, k = C->k_dim, v = C->v_dim;
  if (ps < 16 || ps > 256 || (ps & (ps - 1))) return false;
  if (!(v ? v == k && (k == 64 || k == 128 || k == 256) : k == 256 || k == 512)) return false;
  if (C->dtype != DSV4G_DT_BF16 && C->dtype != DSV4G_DT_F8_E4M3) return false;
  if (C->kv_heads <= 0 || C->kv_heads > 1024 || C->n_layers <= 0 || C->n_layers > 65536 ||
      C->n_pages <= 0 || C->n_pages > (1 << 20) || C->n_seqs <= 0 || C->max_pages <= 0 ||
      (long)C->max_pages * ps > 0x7FFFFFFF - 65536)
    return false;
  const size_t kn = (size_t)C->kv_heads * ps * k, vn = (size_t)C->kv_heads * ps * v;
  const bool fp8 = C->dtype == DSV4G_DT_F8_E4M3;
  const size_t size = fp8 ? 1 : 2;
  G->v_off = (int)(kn * size);
  G->ks_off = (int)((kn + vn) * size);
  G->vs_off = G->ks_off + (fp8 ? (int)(kn / DSV4G_CACHE_GROUP) : 0);
  const size_t used = (size_t)G->vs_off + (fp8 ? vn / DSV4G_CACHE_GROUP : 0);
  G->page_bytes = (used + 255) / 256 * 256;
  G->shift = 31 - __builtin_clz((unsigned)ps);
  return true;
}

// Two fp32 values as BF16, nearest even, NaN kept (x in the low half).
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
  typedef __bf16 Bf2 __attribute__((ext_vector_type(2)));
  typedef float F2 __attribute__((ext_vector_type(2)));
  const F2 f = {x, y};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, Bf2));
}

extern "C" int dsv4g_cache_ok(const DSV4GCache *C, CacheGeom *G, const char *who);
