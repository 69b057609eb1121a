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
// Reading returns T(code * scale), or the 16-bit values unchanged.
//
// Both are HBM-bound: each input is read once and each output written once.
// Rows that are 16-byte aligned (those of every fused projection) take the
// kv_write_vec_kernel; others the kernel right below, one warp per head and one
// element at a time: 12248 bf16 tokens of 16 + 2 * 8 heads of 128 took 36 us
// (5.6 TB/s) against 88.
#include "kl_internal.h"
#include "kl_kv.cuh"

namespace kl {
namespace {

constexpr int kKvThreads = 256;
constexpr int kWriteStages = 3;      // ring depth of the 16-byte write path
constexpr int kWriteBlocks = 2;      // its resident blocks per SM (102 to 116 registers a thread)

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

// ---- 16-byte paths ------------------------------------------------------------

struct Slot {
  int64_t page, off;
};
KL_DEVICE Slot split_slot(int64_t slot, const KvView& kv) {
  if (static_cast<uint64_t>(slot) >> 31) return {slot / kv.page_size, slot % kv.page_size};
  const uint32_t s = static_cast<uint32_t>(slot), p = page_of(kv, s);
  return {p, s - p * kv.page_size};
}

// 32 bytes of one lane at a 32-byte boundary: one instruction, so that every sector is written whole
KL_DEVICE void store32(void* p, uint4 x, uint4 y) {
  asm volatile("st.global.cs.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               :: "l"(p), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w), "r"(y.x), "r"(y.y), "r"(y.z), "r"(y.w) : "memory");
}

// Eight 16-bit values as four f32 pairs, and back
template <typename T> KL_DEVICE void unpack8(f32x2 (&f)[4], uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      f[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    } else {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[i] = pair(x.x, x.y);
    }
  }
}
template <typename T> KL_DEVICE uint4 pack8(const f32x2 (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = halves(f[i]);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x.y), "f"(x.x));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(x.y), "f"(x.x));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight codes of x / scale, rounded to the nearest, ties to even, with inv = 1 / scale:
// adding 1.5 * 2^23 rounds x * inv to an integer, whose low byte is the code. `off` takes
// the distance of x * inv from that integer: the quotient itself is within 2^-15
// of the product, so only a distance above 1/2 - 2^-15 leaves the code open.
KL_DEVICE uint2 codes8(const f32x2 (&x)[4], float inv, float& off) {
  const f32x2 magic = pair(12582912.0f, 12582912.0f), by = pair(inv, inv);
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 t = fma2(x[i], by, magic);
    const float2 d = halves(fma2(x[i], by, sub2(magic, t))), w = halves(t);
    off = fmaxf(off, fmaxf(fabsf(d.x), fabsf(d.y)));
    c[2 * i] = __float_as_uint(w.x);
    c[2 * i + 1] = __float_as_uint(w.y);
  }
  return make_uint2(prmt(prmt(c[0], c[1], 0x40), prmt(c[2], c[3], 0x40), 0x5410),
                    prmt(prmt(c[4], c[5], 0x40), prmt(c[6], c[7], 0x40), 0x5410));
}
// The same by division, for any scale.
__device__ __noinline__ uint2 codes8_exact(f32x2 x0, f32x2 x1, f32x2 x2, f32x2 x3, float scale) {
  const f32x2 x[4] = {x0, x1, x2, x3};
  uint32_t w[2] = {0, 0};
  for (int i = 0; i < 8; ++i) {
    const float2 h = halves(x[i / 2]);
    const int c = __float2int_rn(fminf(fmaxf((i & 1 ? h.y : h.x) / scale, -127.0f), 127.0f));
    w[i / 4] |= static_cast<uint32_t>(c & 0xFF) << (i % 4 * 8);
  }
  return make_uint2(w[0], w[1]);
}

// A head is covered by LANES = head_dim / 16 lanes: lane j holds the 8 elements at
// 8 j and their 8 partners at head_dim / 2 + 8 j, so that the rotation stays in the
// lane and a sum over the head takes log2(LANES) shuffles. A warp takes
// R = 32 / LANES heads of one token and kind (q, k or v) at a time; all such steps
// are dealt out evenly and contiguously to one resident wave of warps, which keep a
// token's rotation in registers with the norm's weights multiplied in. Rows come
// through a ring of cp.async stages that runs on across tokens; a lane reads only
// what it copied itself, so no barrier is needed. Issue slots bound it next to
// memory (one warp per token with loads into registers and an address per head took
// 45 us at 12248 tokens): f32 arithmetic is packed in pairs, pointers walk, and the
// ring takes the place of the occupancy that 100 registers cost.
template <typename T, bool INT8, int LANES>
__global__ void __launch_bounds__(kKvThreads, kWriteBlocks) kv_write_vec_kernel(const KvWriteArgs a) {
  constexpr int D = 16 * LANES, R = 32 / LANES;
  __shared__ uint4 s_ring[kWriteStages][2][kKvThreads];
  const int lane = threadIdx.x & 31, j = lane % LANES, sub = lane / LANES;
  const int q_passes = (a.heads + R - 1) / R, kv_passes = (a.kv.kv_heads + R - 1) / R, passes = q_passes + 2 * kv_passes;
  // this warp's steps [lo, hi) of tokens * passes
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t warps = gridDim.x * (kKvThreads / 32), w = (threadIdx.x >> 5) * gridDim.x + blockIdx.x;
  const uint64_t steps = static_cast<uint64_t>(a.tokens) * passes;
  const uint32_t lo = static_cast<uint32_t>(steps * w / warps), hi = static_cast<uint32_t>(steps * (w + 1) / warps);
  if (lo >= hi) return;

  // ---- fetching: a pointer that walks the heads of one token and kind
  const uint32_t ring = smem_u32(&s_ring[0][0][threadIdx.x]);
  uint32_t left = hi - lo;
  int f_token = lo / passes, f_kind, f_steps, f_head, f_heads;
  const char* f_src;
  int64_t f_inc;
  auto aim = [&](int kind, int skip) {                      // at step `skip` of f_token's rows of that kind
    f_kind = kind;
    f_heads = kind == 0 ? a.heads : a.kv.kv_heads;
    f_steps = (kind == 0 ? q_passes : kv_passes) - skip;
    f_head = skip * R + sub;
    const int64_t stride = kind == 0 ? a.head_stride[0] : kind == 1 ? a.head_stride[1] : a.head_stride[2];
    f_inc = 2 * R * stride;
    f_src = (kind == 0 ? a.x[0] : kind == 1 ? a.x[1] : a.x[2]) + 16 * j +
            2 * (f_token * (kind == 0 ? a.token_stride[0] : kind == 1 ? a.token_stride[1] : a.token_stride[2]) + f_head * stride);
  };
  auto fetch = [&](int stage) {
    if (left > 0) {
      if (f_head < f_heads) {
        cp_async16(ring + stage * (2 * 16 * kKvThreads), f_src, 16);
        cp_async16(ring + stage * (2 * 16 * kKvThreads) + 16 * kKvThreads, f_src + D, 16);
      }
      if (--left > 0) {
        if (--f_steps > 0) {
          f_head += R;
          f_src += f_inc;
        } else {
          if (f_kind == 2) ++f_token;
          aim(f_kind == 2 ? 0 : f_kind + 1, 0);
        }
      }
    }
    cp_async_commit();
  };
  int token = f_token, p = lo - token * passes;
  if (p < q_passes) aim(0, p);
  else if (p < q_passes + kv_passes) aim(1, p - q_passes);
  else aim(2, p - q_passes - kv_passes);
#pragma unroll
  for (int i = 0; i < kWriteStages - 1; ++i) fetch(i);

  const int64_t room = static_cast<int64_t>(a.kv.pages) * a.kv.page_size;
  int64_t next_pos = a.positions[token], next_slot = a.slots[token];
  uint32_t todo = hi - lo;
  int stage = 0;
  auto next_rows = [&](uint4 (&raw)[2]) {
    cp_async_wait<kWriteStages - 2>();
    raw[0] = s_ring[stage][0][threadIdx.x];
    raw[1] = s_ring[stage][1][threadIdx.x];
    fetch(stage == 0 ? kWriteStages - 1 : stage - 1);
    stage = stage == kWriteStages - 1 ? 0 : stage + 1;
  };
  // u' = inv (u uc + v vs),  v' = inv (v vc + u us)
  f32x2 uc[4], us[4], vc[4], vs[4];
  for (; todo > 0; ++token, p = 0) {
    bool turned = false;                                    // the rotation is the token's; without norms keys take the queries'
    int64_t pos = next_pos;
    if (pos < 0 || pos >= a.max_positions) {
      record_error(a.status, KL_ERR_INVALID);
      pos = 0;
    }
    const bool cached = next_slot >= 0 && next_slot < room;
    if (next_slot >= room) record_error(a.status, KL_ERR_INVALID);
    const Slot at = split_slot(cached ? next_slot : 0, a.kv);
    if (token + 1 < a.tokens) {
      next_pos = a.positions[token + 1];
      next_slot = a.slots[token + 1];
    }
    const int64_t to = at.page * a.kv.page_stride + at.off * a.kv.token_stride + 8 * j;
    auto rows_of = [&](auto kind_c) {
      constexpr int kind = decltype(kind_c)::value;
      const int first = kind == 0 ? 0 : kind == 1 ? q_passes : q_passes + kv_passes;
      const int skip = p - first, count = (kind == 0 ? q_passes : kv_passes) - skip;
      if (skip < 0 || count <= 0 || todo == 0) return;
      const int heads = kind == 0 ? a.heads : a.kv.kv_heads;
      int head = skip * R + sub;
      char* out;
      int64_t inc;
      if constexpr (kind == 0) {
        out = static_cast<char*>(a.q_out) + 2 * ((static_cast<int64_t>(token) * a.heads + head) * D + 8 * j);
        inc = 2 * R * D;
      } else {
        out = (kind == 1 ? a.kv.k : a.kv.v) + (to + head * a.kv.head_stride) * (INT8 ? 1 : 2);
        inc = R * a.kv.head_stride * (INT8 ? 1 : 2);
      }
      if (kind < 2 && !(turned && !a.weight[0])) {
        turned = true;
        const float4* c = reinterpret_cast<const float4*>(a.cos + pos * (D / 2) + 8 * j);
        const float4* s = reinterpret_cast<const float4*>(a.sin + pos * (D / 2) + 8 * j);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 x = __ldg(c + i), y = __ldg(s + i);
          uc[2 * i] = vc[2 * i] = pair(x.x, x.y);
          uc[2 * i + 1] = vc[2 * i + 1] = pair(x.z, x.w);
          us[2 * i] = pair(y.x, y.y);
          us[2 * i + 1] = pair(y.z, y.w);
          vs[2 * i] = pair(-y.x, -y.y);
          vs[2 * i + 1] = pair(-y.z, -y.w);
        }
        if (a.weight[0]) {
          const T* wt = static_cast<const T*>(a.weight[kind == 1 ? 1 : 0]) + 8 * j;
          f32x2 wu[4], wv[4];
          unpack8<T>(wu, __ldg(reinterpret_cast<const uint4*>(wt)));
          unpack8<T>(wv, __ldg(reinterpret_cast<const uint4*>(wt + D / 2)));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uc[i] = mul2(uc[i], wu[i]);
            us[i] = mul2(us[i], wu[i]);
            vc[i] = mul2(vc[i], wv[i]);
            vs[i] = mul2(vs[i], wv[i]);
          }
        }
      }
      const int n = min(static_cast<int>(min(todo, 0x7FFFFFFFu)), count);
      todo -= n;
      p += n;
      for (int i = 0; i < n; ++i, head += R, out += inc) {
        uint4 raw[2];
        next_rows(raw);
        const bool store = head < heads && (kind == 0 || cached);
        if constexpr (kind == 2 && !INT8) {                 // values are moved as they are
          if (store) {
            *reinterpret_cast<uint4*>(out) = raw[0];
            *reinterpret_cast<uint4*>(out + D) = raw[1];
          }
        } else {
          f32x2 u[4], v[4];
          unpack8<T>(u, raw[0]);
          unpack8<T>(v, raw[1]);
          if constexpr (kind < 2) {
            float inv = 1.0f;
            if (a.weight[0]) {
              f32x2 ss = mul2(u[0], u[0]);
#pragma unroll
              for (int e = 1; e < 4; ++e) ss = fma2(u[e], u[e], ss);
#pragma unroll
              for (int e = 0; e < 4; ++e) ss = fma2(v[e], v[e], ss);
              const float2 h = halves(ss);
              float sum = h.x + h.y;
#pragma unroll
              for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
              inv = rsqrtf(sum * (1.0f / D) + a.eps);
            }
            const f32x2 inv2 = pair(inv, inv);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const f32x2 x = u[e], y = v[e];
              u[e] = mul2(inv2, fma2(x, uc[e], mul2(y, vs[e])));
              v[e] = mul2(inv2, fma2(y, vc[e], mul2(x, us[e])));
            }
          }
          if constexpr (kind == 0 || !INT8) {
            if (store) {
              *reinterpret_cast<uint4*>(out) = pack8<T>(u);
              *reinterpret_cast<uint4*>(out + D) = pack8<T>(v);
            }
          } else {
            f32x2 none = pair(0.0f, 0.0f);                  // becomes NaN where an element is not finite
            const f32x2 zero = none;
            float m = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 x = halves(u[e]), y = halves(v[e]);
              m = fmaxf(fmaxf(m, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(y.x), fabsf(y.y)));
              none = fma2(u[e], zero, none);
              none = fma2(v[e], zero, none);
            }
            const float2 h = halves(none);
            if (h.x + h.y != 0.0f) m = INFINITY;            // true of NaN too
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
            const bool ok = m < INFINITY;                   // else the whole row reads back as NaN
            float scale = ok ? m / 127.0f : 1.0f;
            if (scale == 0.0f) scale = 1.0f;
            uint2 c[2] = {make_uint2(0, 0), make_uint2(0, 0)};
            if (ok) {
              float off = scale < 1e-30f ? 1.0f : 0.0f;     // 1 / scale stays finite above
              const float by = 1.0f / scale;
              c[0] = codes8(u, by, off);
              c[1] = codes8(v, by, off);
              if (!(off <= 0.49996f)) {
                c[0] = codes8_exact(u[0], u[1], u[2], u[3], scale);
                c[1] = codes8_exact(v[0], v[1], v[2], v[3], scale);
              }
            }
            if (store) {
              *reinterpret_cast<uint2*>(out) = c[0];
              *reinterpret_cast<uint2*>(out + D / 2) = c[1];
              if (j == 0)
                (kind == 1 ? a.kv.ks : a.kv.vs)[at.page * a.kv.s_page_stride + head * a.kv.s_head_stride + at.off * a.kv.s_token_stride] =
                    ok ? scale : __int_as_float(0x7fc00000);
            }
          }
        }
      }
    };
    rows_of(std::integral_constant<int, 0>{});
    rows_of(std::integral_constant<int, 1>{});
    rows_of(std::integral_constant<int, 2>{});
  }
}

// One lane: 16 bytes of a cached key and of the value beside it. One (token, head) pair
// per LANES lanes and no loop: the blocks' turnover keeps more loads in flight than a
// grid-stride loop did (65536 int8 tokens of 8 heads of 128: 65 us against 73).
template <typename T, bool INT8, int D>
__global__ void __launch_bounds__(kKvThreads) kv_read_vec_kernel(const KvView kv, const int64_t* __restrict__ slots, uint32_t pairs,
                                                                 T* __restrict__ k, T* __restrict__ v, int* status) {
  using C = typename std::conditional<INT8, int8_t, T>::type;
  constexpr int E = 16 / sizeof(C), LANES = D / E;
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t j = threadIdx.x % LANES, item = blockIdx.x * (kKvThreads / LANES) + threadIdx.x / LANES;
  if (item >= pairs) return;
  const uint32_t token = item / kv.kv_heads, head = item - token * kv.kv_heads;
  const int64_t slot = __ldg(slots + token), room = static_cast<int64_t>(kv.pages) * kv.page_size;
  const bool there = slot >= 0 && slot < room;
  if (slot >= room) record_error(status, KL_ERR_INVALID);
  uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  float scale[2] = {0.0f, 0.0f};
  if (there) {
    const Slot at = split_slot(slot, kv);
    const int64_t from = (at.page * kv.page_stride + head * kv.head_stride + at.off * kv.token_stride) * static_cast<int>(sizeof(C)) + 16 * j;
    raw[0] = __ldcs(reinterpret_cast<const uint4*>(kv.k + from));
    raw[1] = __ldcs(reinterpret_cast<const uint4*>(kv.v + from));
    if constexpr (INT8) {
      const int64_t sf = at.page * kv.s_page_stride + head * kv.s_head_stride + at.off * kv.s_token_stride;
      scale[0] = __ldg(kv.ks + sf);
      scale[1] = __ldg(kv.vs + sf);
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint4* out = reinterpret_cast<uint4*>((h ? v : k) + static_cast<size_t>(item) * D) + j * (INT8 ? 2 : 1);
    if constexpr (INT8) {
      const int8_t* q = reinterpret_cast<const int8_t*>(&raw[h]);
      f32x2 f[2][4];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e / 4][e % 4] = pair(static_cast<float>(q[2 * e]) * scale[h], static_cast<float>(q[2 * e + 1]) * scale[h]);
      store32(out, pack8<T>(f[0]), pack8<T>(f[1]));
    } else {
      __stcs(out, raw[h]);
    }
  }
}

// Whether every head of x, and the buffers beside it, can be moved in 16-byte pieces.
bool vector_rows(const KvWriteArgs& a) {
  uintptr_t bits = reinterpret_cast<uintptr_t>(a.q_out) | reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin) |
                   reinterpret_cast<uintptr_t>(a.weight[0]) | reinterpret_cast<uintptr_t>(a.weight[1]);
  for (int i = 0; i < 3; ++i)
    bits |= reinterpret_cast<uintptr_t>(a.x[i]) | static_cast<uintptr_t>(a.token_stride[i] * 2) | static_cast<uintptr_t>(a.head_stride[i] * 2);
  return (bits & 15u) == 0;
}

template <typename T, bool INT8, int D>
cudaError_t write_t(const KvWriteArgs& a, int sm_count, cudaStream_t s) {
  const long long rows = a.heads + 2ll * a.kv.kv_heads;
  if (vector_rows(a)) {
    constexpr int R = 32 / (D / 16);
    const long long steps = a.tokens * ((a.heads + R - 1) / R + 2ll * ((a.kv.kv_heads + R - 1) / R));
    const unsigned grid = static_cast<unsigned>(std::min((steps + 7) / 8, static_cast<long long>(kWriteBlocks) * sm_count));
    return launch_dependent(kv_write_vec_kernel<T, INT8, D / 16>, dim3(grid), kKvThreads, 0, s, a);
  }
  kv_write_kernel<T, INT8, D / 32><<<static_cast<unsigned>((a.tokens * rows + 7) / 8), kKvThreads, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename T, bool INT8>
cudaError_t write_d(const KvWriteArgs& a, int head_dim, int sm_count, cudaStream_t s) {
  return head_dim == 64    ? write_t<T, INT8, 64>(a, sm_count, s)
         : head_dim == 128 ? write_t<T, INT8, 128>(a, sm_count, s)
                           : write_t<T, INT8, 256>(a, sm_count, s);
}

template <typename T, bool INT8, int D>
cudaError_t read_t(const KvView& kv, const int64_t* slots, int tokens, void* k, void* v, int* status, int sm_count, cudaStream_t s) {
  constexpr int kPairs = kKvThreads / (D * (INT8 ? 1 : 2) / 16);       // pairs of one block
  const uint32_t pairs = static_cast<uint32_t>(tokens) * kv.kv_heads;
  const uint32_t grid = (pairs + kPairs - 1) / kPairs;
  return launch_dependent(kv_read_vec_kernel<T, INT8, D>, dim3(grid), kKvThreads, 0, s, kv, slots, pairs, static_cast<T*>(k),
                          static_cast<T*>(v), status);
}
template <typename T, bool INT8>
cudaError_t read_d(const KvView& kv, int head_dim, const int64_t* slots, int tokens, void* k, void* v, int* status, int sm_count,
                   cudaStream_t s) {
  return head_dim == 64    ? read_t<T, INT8, 64>(kv, slots, tokens, k, v, status, sm_count, s)
         : head_dim == 128 ? read_t<T, INT8, 128>(kv, slots, tokens, k, v, status, sm_count, s)
                           : read_t<T, INT8, 256>(kv, slots, tokens, k, v, status, sm_count, s);
}

}  // namespace

KvView kv_view(const kl_kv_cache& c) {
  KvView v;
  v.k = static_cast<char*>(c.k);
  v.v = static_cast<char*>(c.v);
  v.ks = c.k_scales;
  v.vs = c.v_scales;
  v.pages = c.pages;
  v.page_size = c.page_size;
  v.kv_heads = c.kv_heads;
  // with 2^log >= page_size, page_mul * page_size = 2^(31 + log) + e, e < 2^log: for x < 2^31 the
  // product exceeds x / page_size by less than 1 / page_size
  int log = 0;
  while ((1ll << log) < c.page_size) ++log;
  v.page_mul = static_cast<uint32_t>(((1ull << (31 + log)) + c.page_size - 1) / c.page_size);
  v.page_shift = 31 + log;
  v.page_stride = c.page_stride;
  v.head_stride = c.head_stride;
  v.token_stride = c.token_stride;
  v.s_page_stride = c.scale_page_stride;
  v.s_head_stride = c.scale_head_stride;
  v.s_token_stride = c.scale_token_stride;
  return v;
}

cudaError_t launch_kv_write(const kl_kv_write_args& w, int sm_count, int* status, cudaStream_t s) {
  KvWriteArgs a;
  a.x[0] = static_cast<const char*>(w.q);
  a.x[1] = static_cast<const char*>(w.k);
  a.x[2] = static_cast<const char*>(w.v);
  a.token_stride[0] = w.q_token_stride, a.head_stride[0] = w.q_head_stride;
  a.token_stride[1] = w.k_token_stride, a.head_stride[1] = w.k_head_stride;
  a.token_stride[2] = w.v_token_stride, a.head_stride[2] = w.v_head_stride;
  a.weight[0] = w.q_weight;
  a.weight[1] = w.k_weight;
  a.cos = w.cos;
  a.sin = w.sin;
  a.positions = w.positions;
  a.slots = w.slots;
  a.tokens = w.tokens;
  a.heads = w.heads;
  a.max_positions = w.max_positions;
  a.eps = w.eps;
  a.q_out = w.q_out;
  a.kv = kv_view(w.cache);
  a.status = status;
  const bool int8 = w.cache.format == KL_KV_INT8;
  const int dim = w.cache.head_dim;
  if (w.dtype == KL_DT_BF16)
    return int8 ? write_d<__nv_bfloat16, true>(a, dim, sm_count, s) : write_d<__nv_bfloat16, false>(a, dim, sm_count, s);
  return int8 ? write_d<__half, true>(a, dim, sm_count, s) : write_d<__half, false>(a, dim, sm_count, s);
}

cudaError_t launch_kv_read(const kl_kv_cache& cache, int dtype, const int64_t* slots, int tokens, void* k, void* v,
                           int sm_count, int* status, cudaStream_t s) {
  const KvView kv = kv_view(cache);
  const bool int8 = cache.format == KL_KV_INT8;
  if (dtype == KL_DT_BF16)
    return int8 ? read_d<__nv_bfloat16, true>(kv, cache.head_dim, slots, tokens, k, v, status, sm_count, s)
                : read_d<__nv_bfloat16, false>(kv, cache.head_dim, slots, tokens, k, v, status, sm_count, s);
  return int8 ? read_d<__half, true>(kv, cache.head_dim, slots, tokens, k, v, status, sm_count, s)
              : read_d<__half, false>(kv, cache.head_dim, slots, tokens, k, v, status, sm_count, s);
}

}  // namespace kl
