// The paged key-value cache as the kernels see it, and the element types that
// its operators share.
//
// Keys and values of one token and head are head_dim contiguous elements at
// page * page_stride + head * head_stride + offset * token_stride, in 64-bit
// element offsets: a cache is larger than 2^31 elements after a few hundred
// thousand tokens.  K and V have the same strides and separate bases.
#pragma once
#include "kl_common.cuh"

namespace kl {

struct KvView {
  char* k;
  char* v;
  float* ks;                       // int8 only: one scale per (page, head, token)
  float* vs;
  int pages, page_size, kv_heads;
  long long page_stride, head_stride, token_stride;          // elements
  long long s_page_stride, s_head_stride, s_token_stride;
};

template <typename T> KL_DEVICE float kv_to_f(T v);
template <> KL_DEVICE float kv_to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> KL_DEVICE float kv_to_f<__half>(__half v) { return __half2float(v); }
template <> KL_DEVICE float kv_to_f<int8_t>(int8_t v) { return static_cast<float>(v); }
template <typename T> KL_DEVICE T kv_from_f(float v);
template <> KL_DEVICE __nv_bfloat16 kv_from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> KL_DEVICE __half kv_from_f<__half>(float v) { return __float2half_rn(v); }

KL_DEVICE float kv_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
KL_DEVICE float kv_warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}

}  // namespace kl
