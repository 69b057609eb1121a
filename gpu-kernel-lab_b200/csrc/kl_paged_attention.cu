// Attention of one new token per sequence over a paged key-value cache.
//
//   s_j = scale * q . k_j,   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   j < lengths[b]
//
// One CTA per (sequence, query head); its warps take the keys in turn, each
// with a running maximum and sum, and are joined at the end.
#include <cfloat>

#include "kl_internal.h"
#include "kl_kv.cuh"

namespace kl {
namespace {

constexpr int kAttnWarps = 8;

struct AttnArgs {
  const void* q;
  long long q_row_stride, q_head_stride;
  KvView kv;
  const int* table;
  long long table_stride;
  const int* lengths;
  int batch, heads, columns;
  float scale;
  void* out;
  float* lse;
  int* status;
};

template <typename T, bool INT8, int E>
__global__ void __launch_bounds__(32 * kAttnWarps) attn_kernel(const AttnArgs a) {
  constexpr int D = 32 * E;
  using C = typename std::conditional<INT8, int8_t, T>::type;
  __shared__ float s_m[kAttnWarps], s_l[kAttnWarps], s_o[kAttnWarps][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / a.heads, h = blockIdx.x % a.heads, kvh = h / (a.heads / a.kv.kv_heads);
  const T* q = static_cast<const T*>(a.q) + b * a.q_row_stride + h * a.q_head_stride;
  float qf[E], o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    qf[i] = kv_to_f<T>(q[lane + 32 * i]);
    o[i] = 0.0f;
  }
  const long long room = static_cast<long long>(a.columns) * a.kv.page_size;
  long long len = a.lengths[b];
  if (len > room) {
    record_error(a.status, KL_ERR_INVALID);
    len = room;
  }
  float m = -FLT_MAX, l = 0.0f;        // finite: a score of -inf has weight 0 and no NaN
  for (long long j = warp; j < len; j += kAttnWarps) {
    const int page = a.table[b * a.table_stride + j / a.kv.page_size];
    if (page < 0 || page >= a.kv.pages) {
      record_error(a.status, KL_ERR_INVALID);
      continue;
    }
    const long long off = j % a.kv.page_size;
    const long long at = page * a.kv.page_stride + kvh * a.kv.head_stride + off * a.kv.token_stride;
    const C* k = reinterpret_cast<const C*>(a.kv.k) + at;
    const C* v = reinterpret_cast<const C*>(a.kv.v) + at;
    float ks = 1.0f, vs = 1.0f;
    if constexpr (INT8) {
      const long long sat = page * a.kv.s_page_stride + kvh * a.kv.s_head_stride + off * a.kv.s_token_stride;
      ks = a.kv.ks[sat];
      vs = a.kv.vs[sat];
    }
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) dot = fmaf(qf[i], kv_to_f<C>(k[lane + 32 * i]), dot);
    const float s = kv_warp_sum(dot) * ks * a.scale;
    const float top = fmaxf(m, s);
    const float keep = expf(m - top), p = expf(s - top);
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = o[i] * keep + p * (kv_to_f<C>(v[lane + 32 * i]) * vs);
    m = top;
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) s_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float top = -FLT_MAX, sum = 0.0f;
  for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, s_m[w]);
  for (int w = 0; w < kAttnWarps; ++w) sum += s_l[w] * expf(s_m[w] - top);
  const size_t row = static_cast<size_t>(b) * a.heads + h;
  for (int d = threadIdx.x; d < D; d += 32 * kAttnWarps) {
    float acc = 0.0f;
    for (int w = 0; w < kAttnWarps; ++w) acc += s_o[w][d] * expf(s_m[w] - top);
    static_cast<T*>(a.out)[row * D + d] = kv_from_f<T>(sum == 0.0f ? 0.0f : acc / sum);
  }
  if (threadIdx.x == 0 && a.lse) a.lse[row] = sum == 0.0f ? -INFINITY : top + logf(sum);
}

template <typename T, bool INT8>
cudaError_t attn_d(const AttnArgs& a, int head_dim, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(a.batch) * a.heads;
  if (head_dim == 64) attn_kernel<T, INT8, 2><<<grid, 32 * kAttnWarps, 0, s>>>(a);
  else if (head_dim == 128) attn_kernel<T, INT8, 4><<<grid, 32 * kAttnWarps, 0, s>>>(a);
  else attn_kernel<T, INT8, 8><<<grid, 32 * kAttnWarps, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

size_t paged_attention_workspace_bytes(int, int, int, int, int) { return 0; }

cudaError_t launch_paged_attention(const void* q, int dtype, int batch, int heads, long long q_row_stride,
                                   long long q_head_stride, const kl_kv_cache& cache, const int* table, long long table_stride,
                                   int columns, const int* lengths, float scale, void* out, float* lse, void*, int, int* status,
                                   cudaStream_t s) {
  AttnArgs a;
  a.q = q;
  a.q_row_stride = q_row_stride;
  a.q_head_stride = q_head_stride;
  a.kv = kv_view(cache);
  a.table = table;
  a.table_stride = table_stride;
  a.lengths = lengths;
  a.batch = batch;
  a.heads = heads;
  a.columns = columns;
  a.scale = scale;
  a.out = out;
  a.lse = lse;
  a.status = status;
  const bool int8 = cache.format == KL_KV_INT8;
  if (dtype == KL_DT_BF16) return int8 ? attn_d<__nv_bfloat16, true>(a, cache.head_dim, s) : attn_d<__nv_bfloat16, false>(a, cache.head_dim, s);
  return int8 ? attn_d<__half, true>(a, cache.head_dim, s) : attn_d<__half, false>(a, cache.head_dim, s);
}

}  // namespace kl
