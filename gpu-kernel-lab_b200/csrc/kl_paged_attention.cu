// Attention of one new token per sequence over a paged key-value cache.
//
//   s_j = scale * q . k_j,   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   j < lengths[b]
//
// It is HBM-bound: every cached key and value is read once, with 4 flops per
// element and query head.
//
// Partition. The cached tokens of a (sequence, KV head, block of query heads)
// row are cut into units of 4 * KEYS tokens, and all rows' units are dealt out
// evenly and contiguously to one resident wave of CTAs (stream-K). The lengths
// are only read on the device, so a captured launch serves any lengths. A row
// that crosses CTAs leaves partial (maximum, sum, output) triples in the
// workspace; the CTA that arrives last joins them in CTA order, so results do
// not depend on timing.
//
// CTA. Four warps, each with its own tokens of a unit and its own ring of
// kStages shared-memory slots that it fills with cp.async (16-byte chunks,
// XOR-swizzled by row), so the main loop has no CTA barrier. Tokens past the
// length are filled with zeros and masked: what a page holds there does not
// matter, NaN included.
//
// Arithmetic, on tensor cores with keys and dimensions as the M side, so that a
// group of query heads fills N = 8 columns:
//   S^T [keys x heads] = K Q^T, then O^T [dims x heads] += V^T P^T.
// Scores, softmax statistics and the output are f32. The weights P enter the
// second product as two 16-bit numbers p = hi + lo (16 bits of bf16 or 22 of
// f16), so that their rounding stays below the output's. With up to four heads per KV
// head the heads stand twice in the eight columns and the second copy carries
// lo: no instruction more. Int8 keys become f16 (exact) against queries scaled by a
// power of two into f16's range (a bf16 query loses nothing down to 2^-28 of its
// head's largest); the key's scale multiplies the score. Int8 values become
// bf16 (exact), their scale multiplies the weight.
#include <cfloat>

#include "kl_internal.h"
#include "kl_kv.cuh"

namespace kl {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStages = 3;
constexpr int kMaxLens = 512;          // lengths kept in shared memory
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnArgs {
  const void* q;
  long long q_row_stride, q_head_stride;
  KvView kv;
  const int* table;
  long long table_stride;
  const int* lengths;
  int batch, heads, columns;
  int group;                           // query heads per KV head
  int blocks;                          // blocks of HB query heads per KV head
  int q_vec;                           // q rows allow 8-byte loads
  float scale;
  void* out;
  float* lse;
  int* counters;
  float* partials;
  int* status;
};

KL_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
KL_DEVICE void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
KL_DEVICE void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
KL_DEVICE uint32_t movmatrix_t(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <bool BF16>
KL_DEVICE void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// {lo, hi} as packed 16-bit values and back
template <bool BF16> KL_DEVICE uint32_t pack2(float lo, float hi) {
  uint32_t d;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
template <bool BF16> KL_DEVICE float2 unpack2(uint32_t v) {
  if constexpr (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// Two int8 values, bytes SEL of w, to exact f16: w holds q ^ 0x80, 0x6400 | u is 1024 + u.
template <uint32_t SEL> KL_DEVICE uint32_t s8_to_f16(uint32_t w) {
  return fma_f16x2(prmt(w, 0x64646464u, SEL), 0x3C003C00u, 0xE480E480u);
}
// Two int8 values, bytes SEL of w, to exact bf16: 0x4300 | low 7 bits is 128 + v, 0x4300 | sign bit is 128 or 256.
template <uint32_t SEL> KL_DEVICE uint32_t s8_to_bf16(uint32_t w) {
  const uint32_t t = prmt(w, 0x43434343u, SEL);
  return fma_bf16x2((t & 0x00800080u) | 0x43004300u, 0xBF80BF80u, t & 0xFF7FFF7Fu);
}

KL_DEVICE uint32_t load16(const void* p) { return *static_cast<const unsigned short*>(p); }
// Two neighbouring 16-bit elements; `vec`: 4-byte aligned.
KL_DEVICE uint32_t load_pair(const char* p, bool vec) {
  return vec ? *reinterpret_cast<const uint32_t*>(p) : load16(p) | load16(p + 2) << 16;
}

// Geometry of one instantiation.  HB query heads per CTA: 4 (each twice in the
// 8 columns), 8 or 16.
template <bool INT8, int D, int HB>
struct Geo {
  static constexpr int kElem = INT8 ? 1 : 2;
  static constexpr int kRow = D * kElem;                          // bytes of one key
  static constexpr int kKeys = 4096 / kRow < 16 ? 16 : 4096 / kRow;   // keys per warp and unit: 8 KB of K and V
  static constexpr int kTiles = kKeys / 16;
  static constexpr int kUnit = kKeys * kWarps;
  static constexpr int kNT = HB == 16 ? 2 : 1;                    // column tiles
  static constexpr bool kDup = HB == 4;
  static constexpr int kCols = 8 * kNT;
  static constexpr int kKV = 2 * kKeys * kRow;
  static constexpr int kOutRow = D + 4;                           // floats; the pad spreads columns over the banks
  static constexpr int kOut = kCols * kOutRow * 4;                // a warp's output, over its consumed slot
  static constexpr int kScales = INT8 ? 2 * kKeys * 4 : 0;
  static constexpr int kSlotRaw = kKV + kScales + 16;             // + the mask of the valid keys
  static constexpr int kSlot = ((kSlotRaw > kOut ? kSlotRaw : kOut) + 127) / 128 * 128;
  static constexpr int kRing = kWarps * kStages * kSlot;
  static constexpr int kStats = 2 * kWarps * kCols * 4;           // every warp's maximum and sum per column
  static constexpr int kSmem = kRing + kStats + kMaxLens * 4 + 128;
  static constexpr int kPartial = HB * (D + 2);                   // floats of one partial row
  static_assert(kKeys <= 64, "");
};

struct Cursor {
  int b, r, i;         // sequence, row of the sequence, unit of the row
  int units, len;
};

template <typename T, bool INT8, int D, int HB>
__global__ void __launch_bounds__(kThreads, Geo<INT8, D, HB>::kSmem <= 113 * 1024 ? 2 : 1) attn_kernel(const AttnArgs a) {
  using G = Geo<INT8, D, HB>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr bool kQkBf16 = kBf16 && !INT8;          // type of the K Q^T product
  constexpr bool kPvBf16 = kBf16 || INT8;           // type of the V^T P^T product
  constexpr int kChunks = G::kRow / 16;             // 16-byte chunks of one key
  constexpr int kRowsPer = 32 / kChunks;            // keys that one warp-wide copy covers
  extern __shared__ __align__(128) char smem[];
  float* s_max = reinterpret_cast<float*>(smem + G::kRing);
  float* s_sum = s_max + kWarps * G::kCols;
  int* s_len = reinterpret_cast<int*>(s_sum + kWarps * G::kCols);
  int* s_misc = s_len + kMaxLens;                   // [0..7] scan totals, [8] start b, [9] start rest, [10] last flag

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int t4 = lane & 3, l4 = lane >> 2;
  const int rows = a.kv.kv_heads * a.blocks;        // rows per sequence

  // ---- this CTA's units: one scan over the sequences' unit counts
  const long long room = static_cast<long long>(a.columns) * a.kv.page_size;
  auto length_of = [&](int b) {
    const int n = a.lengths[b];
    return n < 0 ? 0 : static_cast<int>(n < room ? n : room);
  };
  auto units_of = [&](int n) { return (n + G::kUnit - 1) / G::kUnit; };
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) {
    const int n = length_of(b);
    if (a.lengths[b] > room) record_error(a.status, KL_ERR_INVALID);
    if (b < kMaxLens) s_len[b] = n;
    mine += units_of(n);
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  long long* s_tot = reinterpret_cast<long long*>(s_misc);
  if (lane == 31) s_tot[warp] = incl;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) incl += s_tot[w];
    total += s_tot[w];
  }
  total *= rows;
  const long long ctas = total < static_cast<long long>(gridDim.x) ? total : gridDim.x;
  // sequences without tokens: zeros
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    if ((b < kMaxLens ? s_len[b] : length_of(b)) > 0) continue;
    T* out = static_cast<T*>(a.out) + static_cast<size_t>(b) * a.heads * D;
    for (int i = tid; i < a.heads * D / 8; i += kThreads) reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
    if (a.lse)
      for (int i = tid; i < a.heads; i += kThreads) a.lse[static_cast<size_t>(b) * a.heads + i] = -INFINITY;
  }
  if (blockIdx.x >= ctas) return;
  const long long lo = unit_lo(blockIdx.x, total, ctas), hi = unit_lo(blockIdx.x + 1, total, ctas);
  if ((incl - mine) * rows <= lo && lo < incl * rows) {
    long long before = (incl - mine) * rows;
    int b = b0;
    for (;; ++b) {
      const long long u = static_cast<long long>(units_of(length_of(b))) * rows;
      if (lo < before + u) break;
      before += u;
    }
    s_misc[8] = b;
    s_misc[9] = static_cast<int>(lo - before);
  }
  __syncthreads();
  auto load_len = [&](Cursor& c) {
    c.len = c.b < kMaxLens ? s_len[c.b] : length_of(c.b);
    c.units = units_of(c.len);
  };
  auto advance = [&](Cursor& c) {
    if (++c.i < c.units) return;
    c.i = 0;
    if (++c.r < rows) return;
    c.r = 0;
    do {
      if (++c.b >= a.batch) return;
      load_len(c);
    } while (c.units == 0);
  };
  Cursor in;                                        // next unit to fetch
  in.b = s_misc[8];
  load_len(in);
  in.r = s_misc[9] / in.units;
  in.i = s_misc[9] % in.units;
  Cursor at = in;                                   // unit being computed

  // ---- fetching: this warp's keys of the unit `in` into ring slot `slot`
  const uint32_t ring = smem_u32(smem) + warp * kStages * G::kSlot;
  char* const ring_ptr = smem + warp * kStages * G::kSlot;
  const int chunk = lane % kChunks, row0 = lane / kChunks;
  const long long delta = a.kv.v - a.kv.k;
  auto fetch = [&](int slot) {
    const uint32_t dst = ring + slot * G::kSlot;
    const int pos0 = in.i * G::kUnit + warp * G::kKeys;
    const int count = min(G::kKeys, in.len - pos0);             // may be <= 0
    const int head = in.r / a.blocks;
    const int* table = a.table + in.b * a.table_stride;
    unsigned valid[(G::kKeys + 31) / 32];
#pragma unroll
    for (int w = 0; w < (G::kKeys + 31) / 32; ++w) valid[w] = 0;
    // lane's row offset in the cache (elements), and its scale's; one or two rows per lane
    long long off[(G::kKeys + 31) / 32], soff[(G::kKeys + 31) / 32];
#pragma unroll
    for (int w = 0; w < (G::kKeys + 31) / 32; ++w) {
      const int row = w * 32 + lane;
      bool ok = row < G::kKeys && row < count;
      off[w] = soff[w] = 0;
      if (ok) {
        const unsigned pos = pos0 + row, column = pos / a.kv.page_size, rest = pos - column * a.kv.page_size;
        const int page = table[column];
        if (page < 0 || page >= a.kv.pages) {
          record_error(a.status, KL_ERR_INVALID);
          ok = false;
        } else {
          off[w] = page * a.kv.page_stride + head * a.kv.head_stride + rest * a.kv.token_stride;
          if constexpr (INT8) soff[w] = page * a.kv.s_page_stride + head * a.kv.s_head_stride + rest * a.kv.s_token_stride;
        }
      }
      valid[w] = __ballot_sync(0xFFFFFFFFu, ok);
      if constexpr (INT8) {
        if (row < G::kKeys) {
          cp_async4(dst + G::kKV + row * 4, a.kv.ks + soff[w], ok ? 4 : 0);
          cp_async4(dst + G::kKV + (G::kKeys + row) * 4, a.kv.vs + soff[w], ok ? 4 : 0);
        }
      }
    }
    if (lane == 0) {
#pragma unroll
      for (int w = 0; w < (G::kKeys + 31) / 32; ++w)
        *reinterpret_cast<unsigned*>(ring_ptr + slot * G::kSlot + G::kKV + G::kScales + 4 * w) = valid[w];
    }
    if (count <= 0) return;
#pragma unroll
    for (int j = 0; j < G::kKeys / kRowsPer; ++j) {
      const int row = j * kRowsPer + row0;
      const long long o = __shfl_sync(0xFFFFFFFFu, off[j * kRowsPer / 32], row & 31);
      const int bytes = (valid[j * kRowsPer / 32] >> (row & 31)) & 1 ? 16 : 0;
      const int swz = G::kRow == 64 ? chunk ^ ((row >> 1) & 3) : chunk ^ (row & 7);
      const char* src = a.kv.k + o * G::kElem + chunk * 16;
      const uint32_t d = dst + row * G::kRow + swz * 16;
      cp_async16(d, src, bytes);
      cp_async16(d + G::kKeys * G::kRow, src + delta, bytes);
    }
  };

  // ---- per-row state
  uint32_t qf[G::kNT][D / 16][2];
  float qscale[G::kNT][2];                          // of the score columns 2 t4, 2 t4 + 1
  float acc[D / 16][G::kNT][4];
  float top[G::kNT][2], sum[G::kNT][2];
  auto start_row = [&]() {
    const int kvh = at.r / a.blocks, first = kvh * a.group + (at.r % a.blocks) * HB;
    const int n = min(HB, (kvh + 1) * a.group - first);
    const char* q = static_cast<const char*>(a.q) + (at.b * a.q_row_stride + first * a.q_head_stride) * 2;
    const float base = a.scale * kLog2e;
#pragma unroll
    for (int nt = 0; nt < G::kNT; ++nt) {
      const int col = G::kDup ? (l4 & 3) : nt * 8 + l4;
      const char* p = q + col * a.q_head_stride * 2;
      const bool there = col < n;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int d0 = INT8 ? ks * 16 + t4 * 4 : ks * 16 + t4 * 2, d1 = INT8 ? d0 + 2 : d0 + 8;
        qf[nt][ks][0] = there ? load_pair(p + d0 * 2, a.q_vec) : 0;
        qf[nt][ks][1] = there ? load_pair(p + d1 * 2, a.q_vec) : 0;
      }
      float up = 1.0f;                              // bf16 against int8: the column's power of two
      if constexpr (INT8 && kBf16) {
        float big = 0.0f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 f = unpack2<true>(qf[nt][ks][e]);
            big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
        // largest element into [2^14, 2^15); both factors stay normal numbers
        int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
        e = big == 0.0f || e == 128 ? 14 : max(e, -100);
        const float down = __uint_as_float(static_cast<uint32_t>(14 - e + 127 > 254 ? 254 : 14 - e + 127) << 23);
        up = 1.0f / down;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float2 f = unpack2<true>(qf[nt][ks][x]);
            qf[nt][ks][x] = pack2<false>(f.x * down, f.y * down);
          }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qscale[nt][e] = base * __shfl_sync(0xFFFFFFFFu, up, (2 * t4 + e) * 4);
        top[nt][e] = -FLT_MAX;                      // finite: a score of -inf has weight 0 and makes no NaN
        sum[nt][e] = 0.0f;
      }
    }
#pragma unroll
    for (int m = 0; m < D / 16; ++m)
#pragma unroll
      for (int nt = 0; nt < G::kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][nt][e] = 0.0f;
  };

  auto swizzled = [&](uint32_t base, int row, int c) {
    return base + row * G::kRow + (G::kRow == 64 ? c ^ ((row >> 1) & 3) : c ^ (row & 7)) * 16;
  };

  // ---- one unit of this warp
  auto compute = [&](int slot) {
    const uint32_t kbase = ring + slot * G::kSlot, vbase = kbase + G::kKeys * G::kRow;
    const char* sp = ring_ptr + slot * G::kSlot + G::kKV;
    const unsigned* mask = reinterpret_cast<const unsigned*>(sp + G::kScales);
    const float* ksc = reinterpret_cast<const float*>(sp);
    if (mask[0] == 0 && (G::kKeys <= 32 || mask[1] == 0)) return;
    float s[G::kTiles][G::kNT][4];
#pragma unroll
    for (int g = 0; g < G::kTiles; ++g) {
#pragma unroll
      for (int nt = 0; nt < G::kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[g][nt][e] = 0.0f;
      const int krow = g * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
      if constexpr (INT8) {
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
          uint32_t r[4];
          ldsm4(r, swizzled(kbase, krow, c + (lane >> 4)));
#pragma unroll
          for (int x = 0; x < 4; ++x) r[x] ^= 0x80808080u;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t a0 = s8_to_f16<0x4140>(r[2 * h]), a2 = s8_to_f16<0x4342>(r[2 * h]);
            const uint32_t a1 = s8_to_f16<0x4140>(r[2 * h + 1]), a3 = s8_to_f16<0x4342>(r[2 * h + 1]);
#pragma unroll
            for (int nt = 0; nt < G::kNT; ++nt) mma16816<false>(s[g][nt], a0, a1, a2, a3, qf[nt][c + h][0], qf[nt][c + h][1]);
          }
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          uint32_t r[4];
          ldsm4(r, swizzled(kbase, krow, 2 * ks + (lane >> 4)));
#pragma unroll
          for (int nt = 0; nt < G::kNT; ++nt) mma16816<kQkBf16>(s[g][nt], r[0], r[1], r[2], r[3], qf[nt][ks][0], qf[nt][ks][1]);
        }
      }
    }
    // scale, mask, column maxima
    float next[G::kNT][2];
#pragma unroll
    for (int nt = 0; nt < G::kNT; ++nt) next[nt][0] = top[nt][0], next[nt][1] = top[nt][1];
#pragma unroll
    for (int g = 0; g < G::kTiles; ++g) {
      const unsigned bits = mask[g / 2] >> (g % 2 * 16);
      const bool ok0 = (bits >> l4) & 1, ok1 = (bits >> (l4 + 8)) & 1;
      float k0 = 1.0f, k1 = 1.0f;
      if constexpr (INT8) k0 = ksc[g * 16 + l4], k1 = ksc[g * 16 + l4 + 8];
#pragma unroll
      for (int nt = 0; nt < G::kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x0 = s[g][nt][e], x1 = s[g][nt][2 + e];
          if constexpr (INT8) x0 *= k0, x1 *= k1;
          x0 = ok0 ? x0 * qscale[nt][e] : -INFINITY;
          x1 = ok1 ? x1 * qscale[nt][e] : -INFINITY;
          s[g][nt][e] = x0;
          s[g][nt][2 + e] = x1;
          next[nt][e] = fmaxf(next[nt][e], fmaxf(x0, x1));
        }
    }
    bool moved = false;
#pragma unroll
    for (int nt = 0; nt < G::kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) next[nt][e] = fmaxf(next[nt][e], __shfl_xor_sync(0xFFFFFFFFu, next[nt][e], o));
        moved |= next[nt][e] != top[nt][e];
      }
    if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
      for (int nt = 0; nt < G::kNT; ++nt) {
        const float f0 = ex2(top[nt][0] - next[nt][0]), f1 = ex2(top[nt][1] - next[nt][1]);
        sum[nt][0] *= f0, sum[nt][1] *= f1;
#pragma unroll
        for (int m = 0; m < D / 16; ++m) acc[m][nt][0] *= f0, acc[m][nt][1] *= f1, acc[m][nt][2] *= f0, acc[m][nt][3] *= f1;
        top[nt][0] = next[nt][0], top[nt][1] = next[nt][1];
      }
    }
    // weights and the second product, 16 keys at a time
#pragma unroll
    for (int g = 0; g < G::kTiles; ++g) {
      uint32_t hi[G::kNT][2], lo[G::kNT][2];
      float v0 = 1.0f, v1 = 1.0f;
      if constexpr (INT8) v0 = ksc[G::kKeys + g * 16 + l4], v1 = ksc[G::kKeys + g * 16 + l4 + 8];
#pragma unroll
      for (int nt = 0; nt < G::kNT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float p0 = ex2(s[g][nt][2 * h] - top[nt][0]), p1 = ex2(s[g][nt][2 * h + 1] - top[nt][1]);
          sum[nt][0] += p0, sum[nt][1] += p1;
          if constexpr (INT8) p0 *= h ? v1 : v0, p1 *= h ? v1 : v0;
          uint32_t w = pack2<kPvBf16>(p0, p1);
          const float2 f = unpack2<kPvBf16>(w);
          const uint32_t rest = pack2<kPvBf16>(p0 - f.x, p1 - f.y);
          if constexpr (G::kDup) {
            hi[nt][h] = movmatrix_t(t4 < 2 ? w : rest);
          } else {
            hi[nt][h] = movmatrix_t(w);
            lo[nt][h] = movmatrix_t(rest);
          }
        }
      if constexpr (INT8) {
        const int vrow = g * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
          uint32_t r[4];
          ldsm4_t(r, swizzled(vbase, vrow, c + (lane >> 4)));
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t a0 = s8_to_bf16<0x4240>(r[2 * x]), a1 = s8_to_bf16<0x4341>(r[2 * x]);
            const uint32_t a2 = s8_to_bf16<0x4240>(r[2 * x + 1]), a3 = s8_to_bf16<0x4341>(r[2 * x + 1]);
#pragma unroll
            for (int nt = 0; nt < G::kNT; ++nt) {
              mma16816<true>(acc[c + x][nt], a0, a1, a2, a3, hi[nt][0], hi[nt][1]);
              if constexpr (!G::kDup) mma16816<true>(acc[c + x][nt], a0, a1, a2, a3, lo[nt][0], lo[nt][1]);
            }
          }
        }
      } else {
        const int vrow = g * 16 + (lane & 7) + (lane >> 4) * 8;
#pragma unroll
        for (int m = 0; m < D / 16; ++m) {
          uint32_t r[4];
          ldsm4_t(r, swizzled(vbase, vrow, 2 * m + ((lane >> 3) & 1)));
#pragma unroll
          for (int nt = 0; nt < G::kNT; ++nt) {
            mma16816<kPvBf16>(acc[m][nt], r[0], r[1], r[2], r[3], hi[nt][0], hi[nt][1]);
            if constexpr (!G::kDup) mma16816<kPvBf16>(acc[m][nt], r[0], r[1], r[2], r[3], lo[nt][0], lo[nt][1]);
          }
        }
      }
    }
  };

  // ---- end of a row's units in this CTA: join the warps, then the CTAs
  auto out_slot = [&](int w, int slot) { return reinterpret_cast<float*>(smem + (w * kStages + slot) * G::kSlot); };
  auto finish_row = [&](long long unit, int slot) {
    const int kvh = at.r / a.blocks, first = kvh * a.group + (at.r % a.blocks) * HB;
    const int n = min(HB, (kvh + 1) * a.group - first);
    __syncwarp();
    float* o = out_slot(warp, slot);
#pragma unroll
    for (int nt = 0; nt < G::kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = sum[nt][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, x);
        const int col = nt * 8 + 2 * t4 + e;
        if (l4 == 0) {
          s_max[warp * G::kCols + col] = top[nt][e];
          s_sum[warp * G::kCols + col] = l;
        }
        if ((G::kDup ? col & 3 : col) < n) {
#pragma unroll
          for (int m = 0; m < D / 16; ++m) {
            const int d0 = INT8 ? m * 16 + 2 * l4 : m * 16 + l4, d1 = INT8 ? d0 + 1 : d0 + 8;
            o[col * G::kOutRow + d0] = acc[m][nt][e];
            o[col * G::kOutRow + d1] = acc[m][nt][2 + e];
          }
        }
      }
    __syncthreads();
    const long long row_first = unit - at.i;
    const long long c0 = unit_owner(row_first, total, ctas), c1 = unit_owner(row_first + at.units - 1, total, ctas);
    bool joined = false;                            // the slots hold joined partials of other CTAs (no second copy)
    if (c0 != c1) {
      float* part = a.partials + (blockIdx.x * 2ll + (blockIdx.x == c0 ? 1 : 0)) * G::kPartial;
      for (int i = tid; i < n * (D / 4); i += kThreads) {
        const int col = i / (D / 4), d = i % (D / 4) * 4;
        float m = -FLT_MAX;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_max[w * G::kCols + col]);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = ex2(s_max[w * G::kCols + col] - m);
          const float* x = out_slot(w, slot) + col * G::kOutRow + d;
          const float4 y = *reinterpret_cast<const float4*>(x);
          v.x += f * y.x, v.y += f * y.y, v.z += f * y.z, v.w += f * y.w;
          if constexpr (G::kDup) {
            const float4 z = *reinterpret_cast<const float4*>(x + 4 * G::kOutRow);
            v.x += f * z.x, v.y += f * z.y, v.z += f * z.z, v.w += f * z.w;
          }
          l += f * s_sum[w * G::kCols + col];
        }
        *reinterpret_cast<float4*>(part + col * D + d) = v;
        if (d == 0) {
          part[HB * D + col] = m;
          part[HB * D + HB + col] = l;
        }
      }
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const int count = static_cast<int>(c1 - c0 + 1);
        const int seen = atomicAdd(a.counters + c0, 1);
        if (seen == count - 1) a.counters[c0] = 0;
        s_misc[10] = seen == count - 1;
      }
      __syncthreads();
      if (!s_misc[10]) return;
      __threadfence();
      joined = true;
      // warp w takes the CTAs c0 + w, c0 + w + kWarps, ...
      float* mine_o = out_slot(warp, slot);
      for (int i = lane; i < n * (D / 4); i += 32) {
        const int col = i / (D / 4), d = i % (D / 4) * 4;
        float m = -FLT_MAX, l = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (long long c = c0 + warp; c <= c1; c += kWarps) {
          const float* p = a.partials + (c * 2 + (c == c0 ? 1 : 0)) * G::kPartial;
          const float pm = __ldcg(p + HB * D + col), pl = __ldcg(p + HB * D + HB + col);
          const float4 y = __ldcg(reinterpret_cast<const float4*>(p + col * D + d));
          const float nm = fmaxf(m, pm), f = ex2(m - nm), g = ex2(pm - nm);
          v.x = v.x * f + y.x * g, v.y = v.y * f + y.y * g, v.z = v.z * f + y.z * g, v.w = v.w * f + y.w * g;
          l = l * f + pl * g;
          m = nm;
        }
        *reinterpret_cast<float4*>(mine_o + col * G::kOutRow + d) = v;
        if (d == 0) {
          s_max[warp * G::kCols + col] = m;
          s_sum[warp * G::kCols + col] = l;
        }
      }
      __syncthreads();
    }
    const size_t row = static_cast<size_t>(at.b) * a.heads + first;
    for (int i = tid; i < n * (D / 4); i += kThreads) {
      const int col = i / (D / 4), d = i % (D / 4) * 4;
      float m = -FLT_MAX, l = 0.0f;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_max[w * G::kCols + col]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(s_max[w * G::kCols + col] - m);
        const float* x = out_slot(w, slot) + col * G::kOutRow + d;
        const float4 y = *reinterpret_cast<const float4*>(x);
        v.x += f * y.x, v.y += f * y.y, v.z += f * y.z, v.w += f * y.w;
        if (G::kDup && !joined) {
          const float4 z = *reinterpret_cast<const float4*>(x + 4 * G::kOutRow);
          v.x += f * z.x, v.y += f * z.y, v.z += f * z.z, v.w += f * z.w;
        }
        l += f * s_sum[w * G::kCols + col];
      }
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      uint2 packed;
      packed.x = pack2<kBf16>(v.x * inv, v.y * inv);
      packed.y = pack2<kBf16>(v.z * inv, v.w * inv);
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (row + col) * D + d) = packed;
      if (d == 0 && a.lse) a.lse[row + col] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
    }
  };

  // ---- main loop
  const int count = static_cast<int>(hi - lo);
  int fetched = 0;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    if (fetched < count) {
      fetch(s);
      ++fetched;
      if (fetched < count) advance(in);
    }
    cp_async_commit();
  }
  int slot = 0, fill = kStages - 1;
  bool fresh = true;
  for (int u = 0; u < count; ++u) {
    cp_async_wait<kStages - 2>();
    __syncwarp();
    if (fetched < count) {
      fetch(fill);
      ++fetched;
      if (fetched < count) advance(in);
    }
    cp_async_commit();
    if (fresh) start_row();
    compute(slot);
    fresh = at.i + 1 == at.units || u + 1 == count;
    if (fresh) {
      finish_row(lo + u, slot);
      __syncthreads();
    }
    if (u + 1 < count) advance(at);
    slot = slot + 1 == kStages ? 0 : slot + 1;
    fill = fill + 1 == kStages ? 0 : fill + 1;
  }
}

template <bool INT8, int D, int HB>
constexpr int resident() { return 228 * 1024 / (Geo<INT8, D, HB>::kSmem + 1024); }

template <typename T, bool INT8, int D, int HB>
cudaError_t attn_hb(const AttnArgs& a, int sm_count, cudaStream_t s) {
  using G = Geo<INT8, D, HB>;
  // per device and instantiation: allow the shared memory
  cudaError_t e = cudaFuncSetAttribute(attn_kernel<T, INT8, D, HB>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem);
  if (e != cudaSuccess) return e;
  const long long room = static_cast<long long>(a.columns) * a.kv.page_size;
  const long long most = static_cast<long long>(a.batch) * a.kv.kv_heads * a.blocks * ((room + G::kUnit - 1) / G::kUnit);
  const long long wave = static_cast<long long>(sm_count) * resident<INT8, D, HB>();
  const unsigned grid = static_cast<unsigned>(std::max(1ll, std::min(most, wave)));
  attn_kernel<T, INT8, D, HB><<<grid, kThreads, G::kSmem, s>>>(a);
  return cudaGetLastError();
}

int heads_per_cta(int group, int head_dim) { return group <= 4 ? 4 : group <= 8 || head_dim == 256 ? 8 : 16; }

template <typename T, bool INT8, int D>
cudaError_t attn_d(const AttnArgs& a, int sm_count, cudaStream_t s) {
  const int hb = heads_per_cta(a.group, D);
  if (hb == 4) return attn_hb<T, INT8, D, 4>(a, sm_count, s);
  if constexpr (D != 256)
    if (hb == 16) return attn_hb<T, INT8, D, 16>(a, sm_count, s);
  return attn_hb<T, INT8, D, 8>(a, sm_count, s);
}

template <typename T, bool INT8>
cudaError_t attn_t(const AttnArgs& a, int head_dim, int sm_count, cudaStream_t s) {
  return head_dim == 64    ? attn_d<T, INT8, 64>(a, sm_count, s)
         : head_dim == 128 ? attn_d<T, INT8, 128>(a, sm_count, s)
                           : attn_d<T, INT8, 256>(a, sm_count, s);
}

}  // namespace

size_t paged_attention_workspace_bytes(int batch, int heads, int kv_heads, int head_dim, int sm_count) {
  // two partial rows per CTA of the widest wave
  (void)batch;
  const int hb = heads_per_cta(heads / std::max(1, kv_heads), head_dim);
  return kCounterBytes + 2ull * 2 * sm_count * hb * (head_dim + 2) * sizeof(float);
}

cudaError_t launch_paged_attention(const void* q, int dtype, int batch, int heads, long long q_row_stride,
                                   long long q_head_stride, const kl_kv_cache& cache, const int* table, long long table_stride,
                                   int columns, const int* lengths, float scale, void* out, float* lse, void* workspace,
                                   int sm_count, int* status, cudaStream_t s) {
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
  a.group = heads / cache.kv_heads;
  const int hb = heads_per_cta(a.group, cache.head_dim);
  a.blocks = (a.group + hb - 1) / hb;
  a.q_vec = (reinterpret_cast<uintptr_t>(q) % 4 == 0) && q_row_stride % 2 == 0 && q_head_stride % 2 == 0;
  a.scale = scale;
  a.out = out;
  a.lse = lse;
  a.counters = static_cast<int*>(workspace);
  a.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
  a.status = status;
  const bool int8 = cache.format == KL_KV_INT8;
  if (dtype == KL_DT_BF16)
    return int8 ? attn_t<__nv_bfloat16, true>(a, cache.head_dim, sm_count, s)
                : attn_t<__nv_bfloat16, false>(a, cache.head_dim, sm_count, s);
  return int8 ? attn_t<__half, true>(a, cache.head_dim, sm_count, s) : attn_t<__half, false>(a, cache.head_dim, sm_count, s);
}

}  // namespace kl
