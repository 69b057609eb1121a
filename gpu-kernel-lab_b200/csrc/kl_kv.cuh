// The paged key-value cache as the kernels see it, and the element types that
// its operators share.
//
// Keys and values of one token and head are head_dim contiguous elements at
// page * page_stride + head * head_stride + offset * token_stride, in 64-bit
// element offsets: a cache of 8 heads of 128 is larger than 2^31 elements
// after two million tokens.  K and V have the same strides and separate bases.
#pragma once
#include "kl_common.cuh"

namespace kl {

struct KvView {
  char* k;
  char* v;
  float* ks;                       // int8 only: one scale per (page, head, token)
  float* vs;
  int pages, page_size, kv_heads;
  uint32_t page_mul;               // x / page_size = x * page_mul >> page_shift for x < 2^31
  int page_shift;
  long long page_stride, head_stride, token_stride;          // elements
  long long s_page_stride, s_head_stride, s_token_stride;
};

KL_DEVICE uint32_t page_of(const KvView& kv, uint32_t x) {
  return static_cast<uint32_t>(static_cast<uint64_t>(x) * kv.page_mul >> kv.page_shift);
}

template <typename T> KL_DEVICE float kv_to_f(T v);
template <> KL_DEVICE float kv_to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> KL_DEVICE float kv_to_f<__half>(__half v) { return __half2float(v); }
template <> KL_DEVICE float kv_to_f<int8_t>(int8_t v) { return static_cast<float>(v); }
template <typename T> KL_DEVICE T kv_from_f(float v);
template <> KL_DEVICE __nv_bfloat16 kv_from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> KL_DEVICE __half kv_from_f<__half>(float v) { return __float2half_rn(v); }

// ---- two f32 in one register pair (one instruction for both)
using f32x2 = unsigned long long;
KL_DEVICE f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
KL_DEVICE float2 halves(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
KL_DEVICE f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
KL_DEVICE f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
KL_DEVICE f32x2 sub2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// ---- asynchronous copies into shared memory; bytes past `bytes` of the 16 or 4 are filled with zeros
KL_DEVICE void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(bytes) : "memory");
}
KL_DEVICE void cp_async4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" :: "r"(dst), "l"(src), "r"(bytes) : "memory");
}
KL_DEVICE void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> KL_DEVICE void cp_async_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

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

// Launch as a programmatic dependent of the kernel before: the launch is under way when that ends. The
// kernel waits for that kernel's end (pdl_wait) before it touches what other kernels write.
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t s, A&&... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = s;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
}

}  // namespace kl
