// Writing a paged key-value cache and reading it back.
//
// kv_write_kernel, per token and head (one warp each):
//   y  = x * rsqrt(mean(x^2) + eps) * w            queries and keys, if normed
//   q' = (y_a c - y_b s,  y_b c + y_a s)           halves a, b of the head; c, s of the token's position
// Queries go to q_out, keys and values to the token's slot. An int8 cache gets
//   scale = max|x| / 127 (1 for zeros),  code = rint(x / scale)
// per token and head, the row quantiser's arithmetic. Everything is f32 from
// the load to the single rounding at the store, so that the code of a key is
// the code of its exact value and not of a value rounded to 16 bits first.
//
// kv_read_kernel returns T(code * scale), or the 16-bit values unchanged.
//
// Both are HBM-bound: each input is read once and each output written once.
#include "kl_internal.h"
#include "kl_kv.cuh"

namespace kl {
namespace {

constexpr int kKvThreads = 256;

struct KvWriteArgs {
  const char* x[3];                 // q, k, v
  long long token_stride[3], head_stride[3];
  const void* weight[2];            // of q and k; null: no norm
  const float* cos;
  const float* sin;
  const int64_t* positions;
  const int64_t* slots;
  int tokens, heads, max_positions;
  float eps;
  void* q_out;
  KvView kv;
  int* status;
};

// E = head_dim / 32 elements per lane: d = lane + 32 i, whose partner in the
// rotation is element i + E/2 of the same lane.
template <typename T, bool INT8, int E>
__global__ void __launch_bounds__(kKvThreads) kv_write_kernel(const KvWriteArgs a) {
  constexpr int D = 32 * E;
  const int lane = threadIdx.x & 31;
  const int rows = a.heads + 2 * a.kv.kv_heads;
  const long long row = static_cast<long long>(blockIdx.x) * (kKvThreads / 32) + (threadIdx.x >> 5);
  if (row >= static_cast<long long>(a.tokens) * rows) return;
  const int token = static_cast<int>(row / rows);
  int head = static_cast<int>(row % rows);
  const int part = head < a.heads ? 0 : head < a.heads + a.kv.kv_heads ? 1 : 2;
  head -= part == 0 ? 0 : part == 1 ? a.heads : a.heads + a.kv.kv_heads;
  const T* x = reinterpret_cast<const T*>(a.x[part]) + token * a.token_stride[part] + head * a.head_stride[part];
  float y[E];
#pragma unroll
  for (int i = 0; i < E; ++i) y[i] = kv_to_f<T>(x[lane + 32 * i]);
  if (part < 2) {
    if (a.weight[part]) {
      const T* w = static_cast<const T*>(a.weight[part]);
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) ss = fmaf(y[i], y[i], ss);
      const float inv = rsqrtf(kv_warp_sum(ss) / static_cast<float>(D) + a.eps);
#pragma unroll
      for (int i = 0; i < E; ++i) y[i] = y[i] * inv * kv_to_f<T>(w[lane + 32 * i]);
    }
    int64_t pos = a.positions[token];
    if (pos < 0 || pos >= a.max_positions) {
      record_error(a.status, KL_ERR_INVALID);
      pos = 0;
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float c = a.cos[pos * (D / 2) + lane + 32 * i], s = a.sin[pos * (D / 2) + lane + 32 * i];
      const float u = y[i], v = y[i + E / 2];
      y[i] = u * c - v * s;
      y[i + E / 2] = v * c + u * s;
    }
  }
  if (part == 0) {
    T* out = static_cast<T*>(a.q_out) + (static_cast<long long>(token) * a.heads + head) * D;
#pragma unroll
    for (int i = 0; i < E; ++i) out[lane + 32 * i] = kv_from_f<T>(y[i]);
    return;
  }
  const int64_t slot = a.slots[token];
  if (slot < 0) return;                                   // a token that is not cached
  if (slot >= static_cast<int64_t>(a.kv.pages) * a.kv.page_size) {
    record_error(a.status, KL_ERR_INVALID);
    return;
  }
  const int64_t page = slot / a.kv.page_size, off = slot % a.kv.page_size;
  char* base = part == 1 ? a.kv.k : a.kv.v;
  const int64_t at = page * a.kv.page_stride + head * a.kv.head_stride + off * a.kv.token_stride;
  if constexpr (INT8) {
    float m = 0.0f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      m = fmaxf(m, fabsf(y[i]));
      finite &= fabsf(y[i]) <= 3.402823466e38f;
    }
    m = kv_warp_max(m);
    float scale = m / 127.0f;
    if (scale == 0.0f) scale = 1.0f;
    const bool ok = __all_sync(0xFFFFFFFFu, finite);      // a NaN or an infinity: the whole row reads back as NaN
    int8_t* out = reinterpret_cast<int8_t*>(base) + at;
#pragma unroll
    for (int i = 0; i < E; ++i)
      out[lane + 32 * i] = ok ? static_cast<int8_t>(fminf(fmaxf(rintf(y[i] / scale), -127.0f), 127.0f)) : 0;
    if (lane == 0) {
      float* s = part == 1 ? a.kv.ks : a.kv.vs;
      s[page * a.kv.s_page_stride + head * a.kv.s_head_stride + off * a.kv.s_token_stride] = ok ? scale : __int_as_float(0x7fc00000);
    }
  } else {
    T* out = reinterpret_cast<T*>(base) + at;
#pragma unroll
    for (int i = 0; i < E; ++i) out[lane + 32 * i] = kv_from_f<T>(y[i]);
  }
}

template <typename T, bool INT8, int E>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(const KvView kv, const int64_t* __restrict__ slots, int tokens,
                                                             T* __restrict__ k, T* __restrict__ v, int* status) {
  constexpr int D = 32 * E;
  using C = typename std::conditional<INT8, int8_t, T>::type;
  const int lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * (kKvThreads / 32) + (threadIdx.x >> 5);
  if (row >= 2ll * tokens * kv.kv_heads) return;
  const int part = static_cast<int>(row % 2), head = static_cast<int>(row / 2 % kv.kv_heads);
  const long long token = row / 2 / kv.kv_heads;
  int64_t slot = slots[token];
  T* out = (part ? v : k) + (token * kv.kv_heads + head) * D;
  if (slot >= static_cast<int64_t>(kv.pages) * kv.page_size) {
    record_error(status, KL_ERR_INVALID);
    slot = -1;
  }
  const int64_t page = slot / kv.page_size, off = slot % kv.page_size;
  const C* x = reinterpret_cast<const C*>(part ? kv.v : kv.k) + page * kv.page_stride + head * kv.head_stride + off * kv.token_stride;
  float scale = 1.0f;
  if constexpr (INT8) {
    if (slot >= 0) scale = (part ? kv.vs : kv.ks)[page * kv.s_page_stride + head * kv.s_head_stride + off * kv.s_token_stride];
  }
#pragma unroll
  for (int i = 0; i < E; ++i) out[lane + 32 * i] = kv_from_f<T>(slot < 0 ? 0.0f : kv_to_f<C>(x[lane + 32 * i]) * scale);
}

template <typename T, bool INT8, int E>
cudaError_t write_t(const KvWriteArgs& a, cudaStream_t s) {
  const long long rows = static_cast<long long>(a.tokens) * (a.heads + 2 * a.kv.kv_heads);
  kv_write_kernel<T, INT8, E><<<static_cast<unsigned>((rows + 7) / 8), kKvThreads, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T, bool INT8>
cudaError_t write_d(const KvWriteArgs& a, int head_dim, cudaStream_t s) {
  return head_dim == 64 ? write_t<T, INT8, 2>(a, s) : head_dim == 128 ? write_t<T, INT8, 4>(a, s) : write_t<T, INT8, 8>(a, s);
}

template <typename T, bool INT8, int E>
cudaError_t read_t(const KvView& kv, const int64_t* slots, int tokens, void* k, void* v, int* status, cudaStream_t s) {
  const long long rows = 2ll * tokens * kv.kv_heads;
  kv_read_kernel<T, INT8, E><<<static_cast<unsigned>((rows + 7) / 8), kKvThreads, 0, s>>>(
      kv, slots, tokens, static_cast<T*>(k), static_cast<T*>(v), status);
  return cudaGetLastError();
}
template <typename T, bool INT8>
cudaError_t read_d(const KvView& kv, int head_dim, const int64_t* slots, int tokens, void* k, void* v, int* status,
                   cudaStream_t s) {
  return head_dim == 64    ? read_t<T, INT8, 2>(kv, slots, tokens, k, v, status, s)
         : head_dim == 128 ? read_t<T, INT8, 4>(kv, slots, tokens, k, v, status, s)
                           : read_t<T, INT8, 8>(kv, slots, tokens, k, v, status, s);
}

KvView view_of(const kl_kv_cache& c) {
  KvView v;
  v.k = static_cast<char*>(c.k);
  v.v = static_cast<char*>(c.v);
  v.ks = c.k_scales;
  v.vs = c.v_scales;
  v.pages = c.pages;
  v.page_size = c.page_size;
  v.kv_heads = c.kv_heads;
  v.page_stride = c.page_stride;
  v.head_stride = c.head_stride;
  v.token_stride = c.token_stride;
  v.s_page_stride = c.scale_page_stride;
  v.s_head_stride = c.scale_head_stride;
  v.s_token_stride = c.scale_token_stride;
  return v;
}

}  // namespace

KvView kv_view(const kl_kv_cache& c) { return view_of(c); }

cudaError_t launch_kv_write(const KvRows x[3], int dtype, int tokens, int heads, const void* q_weight, const void* k_weight,
                            const float* cos, const float* sin, int max_positions, const int64_t* positions,
                            const int64_t* slots, float eps, const kl_kv_cache& cache, void* q_out, int* status,
                            cudaStream_t s) {
  KvWriteArgs a;
  for (int i = 0; i < 3; ++i) {
    a.x[i] = static_cast<const char*>(x[i].data);
    a.token_stride[i] = x[i].token_stride;
    a.head_stride[i] = x[i].head_stride;
  }
  a.weight[0] = q_weight;
  a.weight[1] = k_weight;
  a.cos = cos;
  a.sin = sin;
  a.positions = positions;
  a.slots = slots;
  a.tokens = tokens;
  a.heads = heads;
  a.max_positions = max_positions;
  a.eps = eps;
  a.q_out = q_out;
  a.kv = view_of(cache);
  a.status = status;
  const bool int8 = cache.format == KL_KV_INT8;
  if (dtype == KL_DT_BF16)
    return int8 ? write_d<__nv_bfloat16, true>(a, cache.head_dim, s) : write_d<__nv_bfloat16, false>(a, cache.head_dim, s);
  return int8 ? write_d<__half, true>(a, cache.head_dim, s) : write_d<__half, false>(a, cache.head_dim, s);
}

cudaError_t launch_kv_read(const kl_kv_cache& cache, int dtype, const int64_t* slots, int tokens, void* k, void* v, int* status,
                           cudaStream_t s) {
  const KvView kv = view_of(cache);
  const bool int8 = cache.format == KL_KV_INT8;
  if (dtype == KL_DT_BF16)
    return int8 ? read_d<__nv_bfloat16, true>(kv, cache.head_dim, slots, tokens, k, v, status, s)
                : read_d<__nv_bfloat16, false>(kv, cache.head_dim, slots, tokens, k, v, status, s);
  return int8 ? read_d<__half, true>(kv, cache.head_dim, slots, tokens, k, v, status, s)
              : read_d<__half, false>(kv, cache.head_dim, slots, tokens, k, v, status, s);
}

}  // namespace kl
