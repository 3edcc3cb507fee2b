// dsv4_attention.hip - attention of a chunk of new tokens per sequence over
// the paged cache (dsv4g_attention). Layout and rules: include/dsv4_gpu.h.
#include "dsv4_cache.h"
#include "dsv4_device.h"
#include "dsv4_gpu_internal.h"

namespace dsv4 {

struct AttnArgs {
  void *out;
  float *lse;
  const void *q;
  size_t out_stride, q_stride;
  const int *seqs, *starts;
  const float *sink;
  int layer, heads, group, n_seqs, n_tokens, max_q, max_kv, window;
  float scale;
};

// One wave per (new token, query head): the tokens it sees one after the
// other, lane l holding columns l, l + 64, ..; running maximum, sum and output.
template <bool F32, bool FP8>
__global__ __launch_bounds__(64) void k_attn_plain(DSV4GCache C, CacheGeom G, AttnArgs a) {
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  if (*C.status) return;
  int b = -1;
  for (int j = 0; j <= a.n_seqs; j += 64)
    b += __popcll(__ballot(j + lane <= a.n_seqs && a.starts[j + lane] <= row));
  if (b < 0 || b >= a.n_seqs) return;
  const int s = a.seqs ? a.seqs[b] : b, end = a.starts[b + 1];
  int len = -1;
  if (s >= 0 && s < C.n_seqs) len = C.len[s];
  const int count = end - a.starts[b];
  if (len < count || len > a.max_kv || count > a.max_q) {
    if (lane == 0) atomicOr(C.status, DSV4G_CACHE_LIST);
    return;
  }
  const int pos = len - end + row, first = a.window ? max(0, pos - a.window + 1) : 0;
  const int kvh = h / a.group, D = C.k_dim, per = D / 64, DV = C.v_dim ? C.v_dim : D;
  float q[8], acc[8] = {};
  for (int i = 0; i < per; ++i) {
    const size_t o = (size_t)row * a.q_stride + (size_t)h * D + lane + 64 * i;
    q[i] = F32 ? bf16_round(((const float *)a.q)[o]) : bf16_to_f32(((const uint16_t *)a.q)[o]);
  }
  float m = -__builtin_inff(), l = 0.0f;
  for (int j = first; j <= pos; ++j) {
    const int page = C.table[(size_t)s * C.max_pages + (j >> G.shift)];
    if (page < 0 || page >= C.n_pages) {
      if (lane == 0) atomicOr(C.status, DSV4G_CACHE_PAGE);
      continue;
    }
    const uint8_t *base = C.pages + ((size_t)a.layer * C.n_pages + page) * G.page_bytes;
    const size_t e = ((size_t)kvh * C.page_size + (j & (C.page_size - 1))) * D + lane;
    auto at = [&](const uint8_t *codes, const uint8_t *scales, int i) {
      if (!FP8) return bf16_to_f32(((const uint16_t *)codes)[e + 64 * i]);
      return e4m3_decode(codes[e + 64 * i]) * e8m0(scales[(e + 64 * i) / DSV4G_CACHE_GROUP]);
    };
    float z = 0.0f, k[8];
    for (int i = 0; i < per; ++i) {
      k[i] = at(base, base + G.ks_off, i);
      z += q[i] * k[i];
    }
    z = wave_sum(z) * a.scale;
    const float M = fmaxf(m, z), f = __expf(m - M), p = __expf(z - M);
    m = M;
    l = l * f + p;
    for (int i = 0; i < per; ++i)
      acc[i] = acc[i] * f + p * (C.v_dim ? at(base + G.v_off, base + G.vs_off, i) : k[i]);
  }
  if (a.sink) {
    const float z = a.sink[h], M = fmaxf(m, z), f = __expf(m - M);
    l = l * f + __expf(z - M);
    for (int i = 0; i < per; ++i) acc[i] *= f;
    m = M;
  }
  for (int i = 0; i < per; ++i) {
    const size_t o = (size_t)row * a.out_stride + (size_t)h * DV + lane + 64 * i;
    const float y = l != 0.0f ? acc[i] / l : 0.0f;
    if (F32) ((float *)a.out)[o] = bf16_round(y);
    else ((uint16_t *)a.out)[o] = (uint16_t)pack_bf16(y, y);
  }
  if (a.lse && lane == 0)
    a.lse[(size_t)row * a.heads + h] = l != 0.0f ? m + logf(l) : -__builtin_inff();
}

}  // namespace dsv4

using namespace dsv4;

extern "C" {

size_t dsv4g_attention_workspace_bytes(const DSV4GCache *C, int heads, int n_seqs, int n_tokens,
                                       int max_q, int max_kv) {
  return 0;
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
  const size_t dv = C->v_dim ? C->v_dim : C->k_dim;
  if (q_stride < (size_t)heads * C->k_dim || out_stride < heads * dv || q_stride % unit ||
      out_stride % unit || ((uintptr_t)q & 15) || ((uintptr_t)out & 15))
    return dsv4g_fail(DSV4G_EINVAL, "attention: rows of q and out must be 16-byte aligned and at "
                      "least heads * dim apart");
  AttnArgs a = {out, lse, q, out_stride, q_stride, seqs, starts, sink, layer, heads,
                heads / C->kv_heads, n_seqs, n_tokens, max_q, max_kv, window, scale};
  const bool f32 = act_dtype == DSV4G_DT_F32, fp8 = C->dtype == DSV4G_DT_F8_E4M3;
  auto k = f32 ? (fp8 ? k_attn_plain<true, true> : k_attn_plain<true, false>)
               : (fp8 ? k_attn_plain<false, true> : k_attn_plain<false, false>);
  hipLaunchKernelGGL(k, dim3(n_tokens, heads), dim3(64), 0, (hipStream_t)stream, *C, G, a);
  return dsv4g_check_launch("attention");
}

}  // extern "C"
