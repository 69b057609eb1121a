// Attention of one new token per sequence over a paged key-value cache.
//
//   s_j = scale * q . k_j,   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   j < lengths[b]
//
// It is HBM-bound: every cached key and value is read once, with 4 flops per
// element and query head. Replayed from a graph, 64 int8 requests of up to 8192 tokens (16 heads
// on 8 of 128) take 108 us, 5.8 TB/s (121 us as calls under a long load, when the clock falls); 64 bf16
// requests of 2000 tokens 88 us, 6.0 TB/s; one bf16 request of
// 32768 tokens 30 us, 4.5 TB/s, of which 3 until the first copy is issued and 4 in the
// join below.
//
// Partition. The cached tokens of a (sequence, KV head, block of query heads)
// row are cut into units of 4 * KEYS tokens, and all rows' units are dealt out
// evenly and contiguously to one resident wave of CTAs (stream-K). The lengths
// are only read on the device, so a captured launch serves any lengths. A row
// that crosses CTAs leaves partial (maximum, sum, output) triples in the
// workspace, and a dependent launch joins them in CTA order: results do not
// depend on timing. Rows that are short, or many, are not split at all. The host decides that
// before it knows the lengths, by the width of the page table (the rule is at kWholeUnits).
//
// CTA. Four warps, each with its own keys of a unit and its own ring of kStages
// shared-memory slots of 8 KB, filled by TMA: one box per page (or per
// 8 KB), so pages may be anywhere and of any multiple of 8 tokens; other pages
// are copied by the lanes (16-byte cp.async, the same swizzle; 0 to 6 % slower).
// The main loop has no CTA barrier. Twelve warps with two slots each beat eight
// with three (32 requests of up to 4099 tokens: 52 us against 57): the latency of a
// warp's chain of copy, products and exponentials is what has to be covered. Tokens past
// the length are masked and their values set to zero: what a page holds there does
// not matter, NaN included.
//
// Arithmetic, on tensor cores with keys and dimensions as the M side, so that a
// group of query heads fills N = 8 columns:
//   S^T [keys x heads] = K Q^T, then O^T [dims x heads] += V^T P^T.
// Scores, softmax statistics and the output are f32; the reference of the
// exponentials is not the running maximum but follows it only when a score
// exceeds it by 2^8, which spares a reduction over the keys at nearly every unit. The weights P
// enter the second product as two 16-bit numbers p = hi + lo (16 bits of bf16; f16: at kF16Lift),
// so that their rounding stays below the output's. With up to four
// heads per KV head the heads stand twice in the eight columns and the second
// copy carries lo: no product more (2 % faster for int8, even for bf16). Int8
// keys and values are converted exactly, five operations per four of them (to
// q / 64 in bf16, to q in f16 for f16 queries); the key's scale multiplies the
// score, the value's scale the weight. At 792 instructions per 8 KB the int8 form
// issues in 56 % of the cycles.
#include <atomic>
#include <cfloat>

#include <cudaTypedefs.h>

#include "kl_internal.h"
#include "kl_kv.cuh"

namespace kl {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStages = 2;
constexpr int kMaxCtas = 640;          // bound of the grid: 3 per SM of up to 213 SMs
constexpr int kRecordBytes = 16 * 1024;
constexpr int kJoinThreads = 256;
constexpr int kJoinBlocks = 3;         // per SM
constexpr int join_heads(int hb) { return hb == 16 ? 4 : 2; }   // heads of one block of the join
// Rows of up to so many units (the page table's width) are not split: no join, which costs 2.2 us of host time. At the
// most, 4 units, the call takes 1.1 us longer on the device (8 requests of 256 tokens: 9.0 us against 7.8); with rows that
// are many, it is shorter there too (192 f16 requests of up to 301 tokens: 19.6 against 22.5). 8 units: 14.0 us against 9.0
// (8 requests of 500 tokens). Short rows in a table that is wide (a captured step's) are split all the same: with 40960
// tokens' columns one request of 37 tokens takes 6.4 us against 5.1, and those 192 take the 22.5.
constexpr int kWholeUnits = 4;
// Nor are rows of up to so many units where there are two waves of rows and more: 128 requests of 1 to 500 tokens on 8
// heads took 31.9 us against 40.5 split, of 1 to 1000 tokens 53.1 against 64.4, 256 of 1 to 2000 (32 units) 178.9 against
// 180.2; with 1.2 waves (64 requests of 100 to 500 tokens) 23.2 against 21.4. The bound limits what one long row
// among short ones can cost. With 40960 tokens' columns these rows are split too: 128 requests of 1 to 500 tokens take 40.9 us
// against 32.8, 256 of 1 to 250 44.0 against 32.7.
constexpr int kWholeUnitsOfMany = 16;
constexpr int kMaxLens = 512;          // lengths kept in shared memory
constexpr float kSlack = 8.0f;           // log2 of how far the largest weight of a key may grow before the reference moves
// f16 has 40 binades. Weights of f16 values use them all: the largest is between 2^7 and 2^15 (the reference is 2^7 below
// the largest score), and the low parts are carried times 2^12 and summed apart. A weight then has 22 bits down to 2^-20 of the
// largest and an error of at most 2^-44 of it below. With weights from 1 and both parts in one sum the step of f16's subnormals
// left 12 bits at 2^-13 and none at 2^-25, which the sum of the weights still counted: thousands of keys behind one of
// a large weight came out 4 % low at 2^-21. Bf16 has the exponents of f32 and needs neither.
constexpr float kF16Lift = 7.0f, kF16Low = 4096.0f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// A row that several CTAs have parts of, as its first CTA records it
struct Piece {
  int ways;                            // CTAs of the row; 0: the CTA begins no such row
  int heads, row;                      // heads of the row, and the first one's place in the output
};

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
  int q_vec;                           // q rows allow 4-byte loads
  int box;                             // rows of one TMA box (divides the page), 0: copies by the lanes
  float scale;
  void* out;
  float* lse;
  Piece* records;                      // one per CTA; null: rows are not split
  float* partials;                     // two per CTA
  void* workspace;
  int* status;
};

template <bool INT8> struct alignas(64) AttnMaps {
  CUtensorMap k, v;                    // [page, head, token, element]
};
template <> struct alignas(64) AttnMaps<true> {
  CUtensorMap k, v;
  CUtensorMap ks, vs;                  // [page, head, token]
};

KL_DEVICE void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

KL_DEVICE void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
               :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}
// One of the barrier's arrivals, once this thread's earlier cp.async copies have landed
KL_DEVICE void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(bar) : "memory");
}

KL_DEVICE void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" :: "l"(p)); }

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
// Two int8 values, bytes SEL of w, to exact bf16 q / 64: the bits 0x00uu of u = q ^ 0x80 are
// u * 2^-133 (subnormals and the first binade have one step), and 2^127 u * 2^-133 - 2 = (u - 128) / 64.
template <uint32_t SEL> KL_DEVICE uint32_t s8_to_bf16_64th(uint32_t w) {
  return fma_bf16x2(prmt(w, 0, SEL), 0x7F007F00u, 0xC000C000u);
}
// ... of keys, in the type of the queries
template <bool BF16, uint32_t SEL> KL_DEVICE uint32_t s8_to_key(uint32_t w) {
  if constexpr (BF16) return s8_to_bf16_64th<SEL>(w);
  else return s8_to_f16<SEL>(w);
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
  static constexpr int kKV = 2 * kKeys * kRow;                    // one slot of a warp's ring
  static constexpr int kSpan = kRow < 128 ? kRow : 128;           // bytes of a key in one swizzled segment
  static constexpr int kSegs = kRow / kSpan;
  static constexpr int kRing = kWarps * kStages * kKV;
  static constexpr int kScales = kTiles * 128;                    // bytes for a slot's key (or value) scales
  static constexpr int kNote = (INT8 ? 2 * kScales : 0) + 128;    // per slot: the scales, and the mask of the valid keys
  static constexpr int kStats = 2 * kWarps * kCols * 4;           // every warp's maximum and sum per column
  static constexpr int kSmem = 1024 + kRing + kWarps * kStages * (kNote + 8) + kStats + kMaxLens * 4 + 96;
  static constexpr int kResident = kSmem > 113 * 1024 ? 1 : HB == 16 || D == 256 ? 2 : 3;   // CTAs per SM
  static_assert(kCols * D * 4 <= kKV, "a warp's output goes over its consumed slot");
  static constexpr int kPartial = HB * (D + 2);                   // floats of one partial row
  static_assert(kKeys <= 64 && kNote % 128 == 0, "");
};

struct Cursor {
  int b, head, block, i;   // sequence, KV head, block of its query heads, unit of that row
  int units, len;
};

// Four output elements of one head from their weighted sum v, the reference m and the weights' sum l
template <bool BF16, int D, typename T>
KL_DEVICE void emit(T* out, float* lse, int row, int d, float4 v, float m, float l) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<uint2*>(out + static_cast<size_t>(row) * D + d) =
      make_uint2(pack2<BF16>(v.x * inv, v.y * inv), pack2<BF16>(v.z * inv, v.w * inv));
  if (d == 0 && lse) lse[row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <typename T, bool INT8, int D, int HB>
__global__ void __launch_bounds__(kThreads, Geo<INT8, D, HB>::kResident)
    attn_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ AttnMaps<INT8> maps) {
  using G = Geo<INT8, D, HB>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr bool kQkBf16 = kBf16;                   // type of the K Q^T product
  constexpr bool kPvBf16 = kBf16 || INT8;           // type of the V^T P^T product
  constexpr float kLift = kPvBf16 ? 0.0f : kF16Lift;
  constexpr int kChunks = G::kRow / 16;             // 16-byte chunks of one key
  constexpr int kRowsPer = 32 / kChunks;            // keys that one warp-wide copy covers
  constexpr int kWords = (G::kKeys + 31) / 32;      // keys per lane
  extern __shared__ char smem_raw[];
  char* const smem = smem_raw + (1024 - (smem_u32(smem_raw) & 1023)) % 1024;
  char* const notes = smem + G::kRing;
  uint64_t* const bars = reinterpret_cast<uint64_t*>(notes + kWarps * kStages * G::kNote);
  float* s_max = reinterpret_cast<float*>(bars + kWarps * kStages);
  float* s_sum = s_max + kWarps * G::kCols;
  int* s_len = reinterpret_cast<int*>(s_sum + kWarps * G::kCols);
  int* s_misc = s_len + kMaxLens;                   // [0..3] scan totals, [8] start b, [9] start rest, [10] end b, [11] end rest
  Piece* s_piece = reinterpret_cast<Piece*>(s_misc + 12);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int t4 = lane & 3, l4 = lane >> 2;
  const int rows = a.kv.kv_heads * a.blocks;        // rows per sequence

  if (tid < kWarps * kStages) mbar_init(smem_u32(bars + tid), a.box ? 1 : 33);
  if (tid == 0) {
    fence_mbar_init();
    s_piece->ways = 0;
    if (a.box) {                                    // else there are none
      prefetch_tmap(&maps.k);
      prefetch_tmap(&maps.v);
      if constexpr (INT8) {
        prefetch_tmap(&maps.ks);
        prefetch_tmap(&maps.vs);
      }
    }
  }
  pdl_wait();                                       // up to here nothing was read that another kernel writes
  pdl_launch_dependents();
  // what the first units will wait for is brought into L2
  if (blockIdx.x < a.batch && tid * 32 < a.columns) prefetch_l2(a.table + blockIdx.x * a.table_stride + tid * 32);
  if (blockIdx.x < a.batch && tid < a.heads * (D / 64))
    prefetch_l2(static_cast<const char*>(a.q) + (blockIdx.x * a.q_row_stride + tid / (D / 64) * a.q_head_stride) * 2 + tid % (D / 64) * 128);

  // ---- this CTA's units: one scan over the sequences' unit counts
  const long long room = static_cast<long long>(a.columns) * a.kv.page_size;
  auto length_of = [&](int b) {
    const int n = a.lengths[b];
    return n < 0 ? 0 : static_cast<int>(n < room ? n : room);
  };
  auto units_of = [&](int n) { return (n + G::kUnit - 1) / G::kUnit; };
  // what a row counts for in the partition: its units, and one more for its begin and end where rows stay whole (256
  // requests of 1 to 250 tokens: 32.4 us against 39.8 by units alone)
  auto weight_of = [&](int n) { return n > 0 ? units_of(n) + (a.records ? 0 : 1) : 0; };
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    const int n = length_of(b);
    if (a.lengths[b] > room) record_error(a.status, KL_ERR_INVALID);
    if (b < kMaxLens) s_len[b] = n;
    mine += weight_of(n);
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += v;
  }
  int* s_tot = s_misc;
  if (lane == 31) s_tot[warp] = incl;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) incl += s_tot[w];
    total += s_tot[w];
  }
  total *= rows;
  const int ctas = min(total, static_cast<int>(gridDim.x));
  // sequences without tokens: zeros
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    if ((b < kMaxLens ? s_len[b] : length_of(b)) > 0) continue;
    T* out = static_cast<T*>(a.out) + static_cast<size_t>(b) * a.heads * D;
    for (int i = tid; i < a.heads * D / 8; i += kThreads) reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
    if (a.lse)
      for (int i = tid; i < a.heads; i += kThreads) a.lse[static_cast<size_t>(b) * a.heads + i] = -INFINITY;
  }
  if (blockIdx.x >= ctas) {
    if (tid == 0 && a.records) a.records[blockIdx.x].ways = 0;
    return;
  }
  // CTA c has units [lo(c), lo(c + 1)): share + 1 each in the first `more` CTAs, share in the others
  const int share = total / ctas, more = total - share * ctas, cta = blockIdx.x;
  const int lo = cta * share + min(cta, more), hi = lo + share + (cta < more ? 1 : 0);
  auto owner = [&](int u) { return u < more * (share + 1) ? u / (share + 1) : more + (u - more * (share + 1)) / share; };
  // the sequences of the first unit and of the one past the last
#pragma unroll
  for (int end = 0; end < 2; ++end) {
    const int u = end ? hi : lo;
    if ((end == 0 || !a.records) && (incl - mine) * rows <= u && u < incl * rows) {
      int before = (incl - mine) * rows, b = b0;
      for (;; ++b) {
        const int n = weight_of(length_of(b)) * rows;
        if (u < before + n) break;
        before += n;
      }
      s_misc[8 + 2 * end] = b;
      s_misc[9 + 2 * end] = u - before;
    }
  }
  __syncthreads();
  auto load_len = [&](Cursor& c) {
    c.len = c.b < kMaxLens ? s_len[c.b] : length_of(c.b);
    c.units = units_of(c.len);
  };
  auto advance = [&](Cursor& c) {
    if (++c.i < c.units) return;
    c.i = 0;
    if (++c.block < a.blocks) return;
    c.block = 0;
    if (++c.head < a.kv.kv_heads) return;
    c.head = 0;
    do {
      if (++c.b >= a.batch) return;
      load_len(c);
    } while (c.units == 0);
  };
  int count = hi - lo;
  Cursor in;                                        // next unit to fetch
  in.b = s_misc[8];
  load_len(in);
  const int weight = weight_of(in.len);
  in.head = s_misc[9] / weight;
  in.i = s_misc[9] - in.head * weight;
  in.block = 0;
  if (a.blocks > 1) {
    in.block = in.head % a.blocks;
    in.head /= a.blocks;
  }
  if (!a.records) {                                 // whole rows: those that begin in [lo, hi)
    if (hi < total) {
      const int last = weight_of(s_misc[10] < kMaxLens ? s_len[s_misc[10]] : length_of(s_misc[10])), over = s_misc[11] % last;
      if (over) count += last - over;
    }
    if (in.i > 0) {
      count -= weight - in.i;
      in.i = in.units - 1;
      if (count > 0) advance(in);
    }
    if (count <= 0) return;
    Cursor row = in;                                // from weights to units
    for (int left = count; left > 0;) {
      left -= row.units + 1;
      --count;
      row.i = row.units - 1;
      if (left > 0) advance(row);
    }
  }
  Cursor at = in;                                   // unit being computed

  // ---- fetching: this warp's keys of the unit `in` into ring slot `slot`
  const uint32_t ring = smem_u32(smem) + warp * kStages * G::kKV;
  char* const ring_ptr = smem + warp * kStages * G::kKV;
  char* const note = notes + warp * kStages * G::kNote;
  const uint32_t bar = smem_u32(bars + warp * kStages);
  auto place = [&](uint32_t base, int row, int c) {          // chunk c of key `row` in a slot's K or V part
    if constexpr (G::kSpan == 64) return base + row * 64 + (c ^ ((row >> 1) & 3)) * 16;
    else return base + (c >> 3) * (G::kKeys * 128) + row * 128 + ((c & 7) ^ (row & 7)) * 16;
  };
  int page[kWords];                                 // of the lane's keys, and their place in it: read a unit ahead
  unsigned rest[kWords];
  auto look_up = [&]() {
    const int* table = a.table + in.b * a.table_stride;
    const int pos0 = in.i * G::kUnit + warp * G::kKeys;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      const int row = w * 32 + lane, pos = pos0 + row;
      const unsigned column = page_of(a.kv, pos);
      rest[w] = pos - column * a.kv.page_size;
      page[w] = row < G::kKeys && pos < in.len ? __ldg(table + column) : 0;
    }
  };
  uint32_t armed = 0, phases = 0;                   // per slot: copies under way, parity of its barrier
  uint32_t holey = 0;                               // per slot: some of its keys' pages were out of range
  const int group_gap = a.box == 16 ? 32 : 16;      // floats from the scales of 16 keys to the next: a box starts at 128 bytes
  auto fetch = [&](int slot) {
    const int count = in.len - (in.i * G::kUnit + warp * G::kKeys);
    if (count <= 0) return;
    armed |= 1u << slot;
    const uint32_t dst = ring + slot * G::kKV, full = bar + slot * 8, scales = smem_u32(note) + slot * G::kNote;
    bool used[kWords], bad = false;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      const int row = w * 32 + lane;
      used[w] = row < G::kKeys && row < count;
      if (used[w] && static_cast<unsigned>(page[w]) >= static_cast<unsigned>(a.kv.pages)) used[w] = false, bad = true;
    }
    holey &= ~(1u << slot);
    if (__any_sync(0xFFFFFFFFu, bad)) {             // such keys count as absent
      holey |= 1u << slot;
      if (bad) record_error(a.status, KL_ERR_INVALID);
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        const unsigned v = __ballot_sync(0xFFFFFFFFu, used[w]);
        if (lane == 0) reinterpret_cast<unsigned*>(note + slot * G::kNote + G::kNote - 128)[w] = v;
      }
    }
    if (a.box) {
      unsigned boxes = 0;
      bool lead[kWords];
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        lead[w] = used[w] && (lane & (a.box - 1)) == 0 && (w == 0 || a.box < 64);
        boxes += __popc(__ballot_sync(0xFFFFFFFFu, lead[w]));
      }
      if (lane == 0) mbar_arrive_expect_tx(full, boxes * a.box * (2 * G::kRow + (INT8 ? 8 : 0)));
      __syncwarp();
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        if (lead[w]) {
          const int row = w * 32 + lane;
#pragma unroll
          for (int g = 0; g < G::kSegs; ++g) {
            const uint32_t to = dst + g * (G::kKeys * 128) + row * G::kSpan;
            tma_load_4d(to, &maps.k, g * (G::kSpan / G::kElem), rest[w], in.head, page[w], full);
            tma_load_4d(to + G::kKeys * G::kRow, &maps.v, g * (G::kSpan / G::kElem), rest[w], in.head, page[w], full);
          }
          if constexpr (INT8) {
            tma_load_3d(scales + row / 4 * group_gap, &maps.ks, rest[w], in.head, page[w], full);
            tma_load_3d(scales + G::kScales + row / 4 * group_gap, &maps.vs, rest[w], in.head, page[w], full);
          }
        }
      }
    } else {
      const int chunk = lane % kChunks, row0 = lane / kChunks;
      const long long delta = a.kv.v - a.kv.k;
      long long off[kWords];
      unsigned valid[kWords];
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        off[w] = used[w] ? page[w] * a.kv.page_stride + in.head * a.kv.head_stride + rest[w] * a.kv.token_stride : 0;
        valid[w] = __ballot_sync(0xFFFFFFFFu, used[w]);
        if constexpr (INT8) {
          const int row = w * 32 + lane;
          if (row < G::kKeys) {
            const long long from = used[w] ? page[w] * a.kv.s_page_stride + in.head * a.kv.s_head_stride + rest[w] * a.kv.s_token_stride : 0;
            cp_async4(scales + row * 4, a.kv.ks + from, used[w] ? 4 : 0);
            cp_async4(scales + G::kScales + row * 4, a.kv.vs + from, used[w] ? 4 : 0);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < G::kKeys / kRowsPer; ++j) {
        const int row = j * kRowsPer + row0;
        const long long o = __shfl_sync(0xFFFFFFFFu, off[j * kRowsPer / 32], row & 31);
        const int bytes = (valid[j * kRowsPer / 32] >> (row & 31)) & 1 ? 16 : 0;
        const char* src = a.kv.k + o * G::kElem + chunk * 16;
        const uint32_t to = place(dst, row, chunk);
        cp_async16(to, src, bytes);
        cp_async16(to + G::kKeys * G::kRow, src + delta, bytes);
      }
      cp_async_arrive(full);
      if (lane == 0) mbar_arrive(full);
    }
  };

  // ---- per-row state
  uint32_t qf[G::kNT][D / 16][2];
  const float qscale = a.scale * kLog2e * (INT8 && kBf16 ? 64.0f : 1.0f);
  float acc[D / 16][G::kNT][4];
  float top[G::kNT][2], sum[G::kNT][2];
  auto start_row = [&]() {
    const int first = at.head * a.group + at.block * HB, n = min(HB, a.group - at.block * HB);
    const char* q = static_cast<const char*>(a.q) + (at.b * a.q_row_stride + first * a.q_head_stride) * 2;
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
#pragma unroll
      for (int e = 0; e < 2; ++e) {
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

  // ---- one unit of this warp
  bool dead = false;                                // a wait ran out: nothing more is fetched
  auto compute = [&](int slot) {
    if (at.len <= at.i * G::kUnit + warp * G::kKeys) return;
    const uint32_t kbase = ring + slot * G::kKV, vbase = kbase + G::kKeys * G::kRow;
    const float* ksc = reinterpret_cast<const float*>(note + slot * G::kNote);
    const float* vsc = ksc + G::kScales / 4;
    if (armed >> slot & 1) {
      if (!mbar_wait_time(bar + slot * 8, phases >> slot & 1)) {
        dead = true;
        record_error(a.status, KL_ERR_TIMEOUT);
      }
      armed ^= 1u << slot;
      phases ^= 1u << slot;
    }
    __syncwarp();
    const int count = at.len - (at.i * G::kUnit + warp * G::kKeys);
    const bool holes = holey >> slot & 1, partial = count < G::kKeys || holes;
    unsigned valid[kWords];
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      valid[w] = count >= 32 * w + 32 ? 0xFFFFFFFFu : count <= 32 * w ? 0u : (1u << (count - 32 * w)) - 1;
      if (holes) valid[w] &= reinterpret_cast<const unsigned*>(note + slot * G::kNote + G::kNote - 128)[w];
    }
    if (!INT8 && partial && a.box) {                // a box brings what the page holds past the length: values become 0
      for (int i = lane; i < G::kKeys * G::kRow / 16; i += 32) {
        const int row = i / (G::kSpan / 16) % G::kKeys;
        if (!(valid[kWords == 1 ? 0 : row / 32] >> (row & 31) & 1))
          *reinterpret_cast<uint4*>(ring_ptr + slot * G::kKV + G::kKeys * G::kRow + i * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      __syncwarp();
    }
    // chunk c of a row is at the row's chunk 0 or 1 with c * 16 exclusive-ored in (c even)
    const uint32_t krow = place(kbase, (lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4);
    const uint32_t vrow = INT8 ? place(vbase, (lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4)
                               : place(vbase, (lane & 7) + (lane >> 4) * 8, (lane >> 3) & 1);
    auto cell = [](uint32_t row, int g, int c) {
      return (row ^ ((c & (G::kSpan / 16 - 1)) * 16)) + (c / (G::kSpan / 16)) * (G::kKeys * G::kSpan) + g * 16 * G::kSpan;
    };
    float s[G::kTiles][G::kNT][4];
#pragma unroll
    for (int g = 0; g < G::kTiles; ++g) {
#pragma unroll
      for (int nt = 0; nt < G::kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[g][nt][e] = 0.0f;
      if constexpr (INT8) {
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
          uint32_t r[4];
          ldsm4(r, cell(krow, g, c));
#pragma unroll
          for (int x = 0; x < 4; ++x) r[x] ^= 0x80808080u;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t a0 = s8_to_key<kBf16, 0x4140>(r[2 * h]), a2 = s8_to_key<kBf16, 0x4342>(r[2 * h]);
            const uint32_t a1 = s8_to_key<kBf16, 0x4140>(r[2 * h + 1]), a3 = s8_to_key<kBf16, 0x4342>(r[2 * h + 1]);
#pragma unroll
            for (int nt = 0; nt < G::kNT; ++nt) mma16816<kQkBf16>(s[g][nt], a0, a1, a2, a3, qf[nt][c + h][0], qf[nt][c + h][1]);
          }
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          uint32_t r[4];
          ldsm4(r, cell(krow, g, 2 * ks));
#pragma unroll
          for (int nt = 0; nt < G::kNT; ++nt) mma16816<kQkBf16>(s[g][nt], r[0], r[1], r[2], r[3], qf[nt][ks][0], qf[nt][ks][1]);
        }
      }
    }
    // scores; the reference of the exponentials moves only when one exceeds it by 2^(kLift + 8)
    bool above = false;
#pragma unroll
    for (int g = 0; g < G::kTiles; ++g) {
      float k0 = qscale, k1 = qscale;
      if constexpr (INT8) k0 *= ksc[g * group_gap + l4], k1 *= ksc[g * group_gap + l4 + 8];
#pragma unroll
      for (int nt = 0; nt < G::kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[g][nt][e] *= k0;
          s[g][nt][2 + e] *= k1;
        }
    }
    if (partial) {
#pragma unroll
      for (int g = 0; g < G::kTiles; ++g) {
        const unsigned bits = valid[g / 2] >> (g % 2 * 16);
#pragma unroll
        for (int nt = 0; nt < G::kNT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(bits >> (l4 + (e < 2 ? 0 : 8)) & 1)) s[g][nt][e] = -INFINITY;
      }
    }
    float most[G::kNT][2];
#pragma unroll
    for (int nt = 0; nt < G::kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        most[nt][e] = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
#pragma unroll
        for (int g = 1; g < G::kTiles; ++g) most[nt][e] = fmaxf(most[nt][e], fmaxf(s[g][nt][e], s[g][nt][2 + e]));
        above |= most[nt][e] > top[nt][e] + (kLift + kSlack);
      }
    if (__any_sync(0xFFFFFFFFu, above)) {
#pragma unroll
      for (int nt = 0; nt < G::kNT; ++nt) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(most[nt][e] - kLift, top[nt][e]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, o));
          f[e] = ex2(top[nt][e] - x);
          top[nt][e] = x;
          sum[nt][e] *= f[e];
        }
#pragma unroll
        for (int m = 0; m < D / 16; ++m) acc[m][nt][0] *= f[0], acc[m][nt][1] *= f[1], acc[m][nt][2] *= f[0], acc[m][nt][3] *= f[1];
      }
    }
    // weights, times the values' scales
#pragma unroll
    for (int g = 0; g < G::kTiles; ++g) {
      float v0 = 1.0f, v1 = 1.0f;
      if constexpr (INT8) v0 = vsc[g * group_gap + l4], v1 = vsc[g * group_gap + l4 + 8];
#pragma unroll
      for (int nt = 0; nt < G::kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p0 = ex2(s[g][nt][e] - top[nt][e]), p1 = ex2(s[g][nt][2 + e] - top[nt][e]);
          sum[nt][e] += p0 + p1;
          s[g][nt][e] = INT8 ? p0 * v0 : p0;
          s[g][nt][2 + e] = INT8 ? p1 * v1 : p1;
        }
    }
    if (INT8 && partial) {                          // a scale past the length may be anything
#pragma unroll
      for (int g = 0; g < G::kTiles; ++g) {
        const unsigned bits = valid[g / 2] >> (g % 2 * 16);
#pragma unroll
        for (int nt = 0; nt < G::kNT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(bits >> (l4 + (e < 2 ? 0 : 8)) & 1)) s[g][nt][e] = 0.0f;
      }
    }
    // the second product, 16 keys at a time
#pragma unroll
    for (int g = 0; g < G::kTiles; ++g) {
      uint32_t hi[G::kNT][2], lo[G::kNT][2];
#pragma unroll
      for (int nt = 0; nt < G::kNT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float p0 = s[g][nt][2 * h], p1 = s[g][nt][2 * h + 1];
          uint32_t w = pack2<kPvBf16>(p0, p1);
          const float2 f = unpack2<kPvBf16>(w);
          const uint32_t rest = kPvBf16 ? pack2<kPvBf16>(p0 - f.x, p1 - f.y) : pack2<kPvBf16>((p0 - f.x) * kF16Low, (p1 - f.y) * kF16Low);
          if constexpr (G::kDup) {
            hi[nt][h] = movmatrix_t(t4 < 2 ? w : rest);
          } else {
            hi[nt][h] = movmatrix_t(w);
            lo[nt][h] = movmatrix_t(rest);
          }
        }
      if constexpr (INT8) {
#pragma unroll
        for (int c = 0; c < kChunks; c += 2) {
          uint32_t r[4];
          ldsm4_t(r, cell(vrow, g, c));
#pragma unroll
          for (int x = 0; x < 4; ++x) r[x] ^= 0x80808080u;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t a0 = s8_to_bf16_64th<0x4240>(r[2 * x]), a1 = s8_to_bf16_64th<0x4341>(r[2 * x]);
            const uint32_t a2 = s8_to_bf16_64th<0x4240>(r[2 * x + 1]), a3 = s8_to_bf16_64th<0x4341>(r[2 * x + 1]);
#pragma unroll
            for (int nt = 0; nt < G::kNT; ++nt) {
              mma16816<true>(acc[c + x][nt], a0, a1, a2, a3, hi[nt][0], hi[nt][1]);
              if constexpr (!G::kDup) mma16816<true>(acc[c + x][nt], a0, a1, a2, a3, lo[nt][0], lo[nt][1]);
            }
          }
        }
      } else {
#pragma unroll
        for (int m = 0; m < D / 16; ++m) {
          uint32_t r[4];
          ldsm4_t(r, cell(vrow, g, 2 * m));
#pragma unroll
          for (int nt = 0; nt < G::kNT; ++nt) {
            mma16816<kPvBf16>(acc[m][nt], r[0], r[1], r[2], r[3], hi[nt][0], hi[nt][1]);
            if constexpr (!G::kDup && kPvBf16) mma16816<kPvBf16>(acc[m][nt], r[0], r[1], r[2], r[3], lo[nt][0], lo[nt][1]);
            if constexpr (!G::kDup && !kPvBf16) {
              float low[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma16816<kPvBf16>(low, r[0], r[1], r[2], r[3], lo[nt][0], lo[nt][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[m][nt][e] = fmaf(low[e], 1.0f / kF16Low, acc[m][nt][e]);
            }
          }
        }
      }
    }
  };

  // ---- end of a row's units in this CTA: join the warps, then the CTAs
  auto out_slot = [&](int w, int slot) { return reinterpret_cast<float*>(smem + (w * kStages + slot) * G::kKV); };
  // element d of a column, spread over the banks by the column
  auto spread = [](int col, int d) { return col * D + (d ^ ((col >> 1 & 3) << (INT8 ? 4 : 3))); };
  auto finish_row = [&](int index, int slot) {
    const int first = at.head * a.group + at.block * HB, n = min(HB, a.group - at.block * HB);
    __syncwarp();
    float* o = out_slot(warp, slot);
    // codes entered as q / 64; the second copy of the heads holds the low parts
    const float unit = INT8 ? 64.0f : !kPvBf16 && G::kDup && t4 >= 2 ? 1.0f / kF16Low : 1.0f;
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
            o[spread(col, d0)] = acc[m][nt][e] * unit;
            o[spread(col, d1)] = acc[m][nt][2 + e] * unit;
          }
        }
      }
    __syncthreads();
    const int row = at.b * a.heads + first;
    const int row_first = index - at.i, c0 = a.records ? owner(row_first) : cta, c1 = a.records ? owner(row_first + at.units - 1) : cta;
    const int ways = c1 - c0 + 1, own = cta - c0;
    for (int i = tid; i < n * (D / 4); i += kThreads) {
      const int col = i / (D / 4), d = i % (D / 4) * 4;
      float m = -FLT_MAX, l = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_max[w * G::kCols + col]);
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(s_max[w * G::kCols + col] - m);
        const float4 y = *reinterpret_cast<const float4*>(out_slot(w, slot) + spread(col, d));
        v.x += f * y.x, v.y += f * y.y, v.z += f * y.z, v.w += f * y.w;
        if constexpr (G::kDup) {
          const float4 z = *reinterpret_cast<const float4*>(out_slot(w, slot) + spread(col + 4, d));
          v.x += f * z.x, v.y += f * z.y, v.z += f * z.z, v.w += f * z.w;
        }
        l += f * s_sum[w * G::kCols + col];
      }
      if (ways == 1) {
        emit<kBf16, D>(static_cast<T*>(a.out), a.lse, row + col, d, v, m, l);
      } else {
        float* p = a.partials + static_cast<long long>(cta * 2 + (own == 0 ? 1 : 0)) * G::kPartial;
        __stcg(reinterpret_cast<float4*>(p + col * D + d), v);
        if (d == 0) {
          __stcg(p + HB * D + col, m);
          __stcg(p + HB * D + HB + col, l);
        }
      }
    }
    if (ways > 1 && own == 0 && tid == 0) *s_piece = {ways, n, row};
  };

  // ---- main loop
  int fetched = 0;
  auto fetch_next = [&](int slot) {
    fetch(slot);
    if (++fetched < count) {
      advance(in);
      look_up();
    }
  };
  look_up();
  start_row();
#pragma unroll 1
  for (int i = 0; i < kStages - 1 && i < count; ++i) fetch_next(i);
  int slot = 0, fill = kStages - 1;
  bool fresh = false;
  for (int u = 0; u < count; ++u) {
    if (fetched < count && !__any_sync(0xFFFFFFFFu, dead)) fetch_next(fill);
    if (fresh) start_row();
    compute(slot);
    fresh = at.i + 1 == at.units || u + 1 == count;
    if (fresh) {
      finish_row(lo + u, slot);
      fence_proxy_async_smem();                     // the slots were written as plain memory; copies follow
      __syncthreads();
    }
    if (u + 1 < count) advance(at);
    slot = slot + 1 == kStages ? 0 : slot + 1;
    fill = fill + 1 == kStages ? 0 : fill + 1;
  }
  if (__any_sync(0xFFFFFFFFu, dead))                // copies still on their way are waited for once more before the memory is let go
    for (int i = 0; i < kStages; ++i) mbar_wait_time(bar + i * 8, phases >> i & 1 ^ 1);
  if (tid == 0 && a.records) a.records[cta] = *s_piece;
}

// The rows that several CTAs have parts of: block (x, y) joins kHeads heads, from y * kHeads, of
// the rows whose first part is CTA x's, x + gridDim.x's, and so on. Launched behind the
// attention kernel as its programmatic dependent, so that the launch is under way when that
// ends. Joining a row inside that kernel, in the CTA whose part arrives last, took
// 8 us where this takes 4: a chain of round trips with the row's data going through one SM.
template <typename T, int D, int HB>
__global__ void __launch_bounds__(kJoinThreads, kJoinBlocks) join_kernel(const Piece* records, int count, const float* partials, T* out, float* lse) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kHeads = join_heads(HB), kVecs = kHeads * D / 4, kSides = kJoinThreads / kVecs, kBatch = 8;
  __shared__ float4 s_v[kSides][kVecs];
  __shared__ float s_m[kSides][kVecs], s_l[kSides][kVecs];
  pdl_wait();
  pdl_launch_dependents();
  const int side = threadIdx.x / kVecs, vec = threadIdx.x % kVecs;
  const int col = blockIdx.y * kHeads + vec / (D / 4), d = vec % (D / 4) * 4;
  for (int c = blockIdx.x; c < count; c += gridDim.x) {
    const Piece piece = records[c];
    if (piece.ways == 0 || blockIdx.y * kHeads >= piece.heads) continue;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float m = -FLT_MAX, l = 0.0f;
    if (col < piece.heads) {
      for (int k0 = side; k0 < piece.ways; k0 += kBatch * kSides) {
        float4 y[kBatch];
        float pm[kBatch], pl[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int k = k0 + i * kSides;
          y[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f), pm[i] = -FLT_MAX, pl[i] = 0.0f;
          if (k < piece.ways) {
            const float* x = partials + static_cast<long long>((c + k) * 2 + (k == 0 ? 1 : 0)) * (HB * (D + 2));
            y[i] = __ldcg(reinterpret_cast<const float4*>(x + col * D + d));
            pm[i] = __ldcg(x + HB * D + col);
            pl[i] = __ldcg(x + HB * D + HB + col);
          }
        }
        float most = m;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) most = fmaxf(most, pm[i]);
        const float keep = ex2(m - most);
        v.x *= keep, v.y *= keep, v.z *= keep, v.w *= keep, l *= keep;
        m = most;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const float f = ex2(pm[i] - m);
          v.x += f * y[i].x, v.y += f * y[i].y, v.z += f * y[i].z, v.w += f * y[i].w;
          l += f * pl[i];
        }
      }
    }
    s_v[side][vec] = v;
    s_m[side][vec] = m;
    s_l[side][vec] = l;
    __syncthreads();
    if (side == 0 && col < piece.heads) {
      for (int k = 1; k < kSides; ++k) m = fmaxf(m, s_m[k][vec]);
      v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      l = 0.0f;
      for (int k = 0; k < kSides; ++k) {
        const float f = ex2(s_m[k][vec] - m);
        const float4 y = s_v[k][vec];
        v.x += f * y.x, v.y += f * y.y, v.z += f * y.z, v.w += f * y.w;
        l += f * s_l[k][vec];
      }
      emit<kBf16, D>(out, lse, piece.row + col, d, v, m, l);
    }
    __syncthreads();
  }
}

// Tensor maps of K and V with boxes of as many rows as divide a page, at most `keys`;
// returns the rows of a box, or 0 where the lanes have to copy: pages that are no
// multiple of 8 tokens (a box of fewer rows would split a swizzle pattern) or, in int8,
// of 16 (the unit in which the scales are laid out), and scales that TMA cannot take.
template <bool INT8>
int make_maps(const AttnArgs& a, AttnMaps<INT8>& maps, int head_dim, int span, int keys) {
  const int elem = INT8 ? 1 : 2, least = INT8 ? 16 : 8;
  int box = keys;
  while (box >= least && a.kv.page_size % box) box /= 2;
  if (box < least) return 0;
  const auto encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tensor_map_encoder());
  if (!encode) return 0;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(a.kv.page_size),
                              static_cast<cuuint64_t>(a.kv.kv_heads), static_cast<cuuint64_t>(a.kv.pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(a.kv.token_stride * elem), static_cast<cuuint64_t>(a.kv.head_stride * elem),
                                 static_cast<cuuint64_t>(a.kv.page_stride * elem)};
  const cuuint32_t tile[4] = {static_cast<cuuint32_t>(span / elem), static_cast<cuuint32_t>(box), 1, 1};
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  for (int i = 0; i < 2; ++i) {
    if (encode(i ? &maps.v : &maps.k, elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 4,
               i ? a.kv.v : a.kv.k, dims, strides, tile, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
               span == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return 0;
  }
  if constexpr (INT8) {
    if (a.kv.s_token_stride != 1) return 0;
    const cuuint64_t s_strides[2] = {static_cast<cuuint64_t>(a.kv.s_head_stride * 4), static_cast<cuuint64_t>(a.kv.s_page_stride * 4)};
    const cuuint32_t s_tile[3] = {static_cast<cuuint32_t>(box), 1, 1};
    for (int i = 0; i < 2; ++i) {
      if (encode(i ? &maps.vs : &maps.ks, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, i ? a.kv.vs : a.kv.ks, dims + 1, s_strides, s_tile, ones,
                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return 0;
    }
  }
  return box;
}

// How a call is dealt out: by what is known before the lengths are
struct Deal {
  bool whole;                          // rows are not split
  unsigned grid;
};
template <typename G>
Deal deal(long long rows, long long room, int sm_count) {
  const long long most = rows * ((room + G::kUnit - 1) / G::kUnit), wave = static_cast<long long>(sm_count) * G::kResident;
  return {room <= (rows >= 2 * wave ? kWholeUnitsOfMany : kWholeUnits) * G::kUnit,
          static_cast<unsigned>(std::max(1ll, std::min({most, wave, static_cast<long long>(kMaxCtas)})))};
}

template <typename T, bool INT8, int D, int HB>
cudaError_t attn_hb(AttnArgs& a, int sm_count, cudaStream_t s) {
  using G = Geo<INT8, D, HB>;
  AttnMaps<INT8> maps;
  a.box = make_maps(a, maps, D, G::kSpan, G::kKeys);
  // once per device: allow the shared memory
  static std::atomic<unsigned long long> allowed{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!(allowed.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    e = cudaFuncSetAttribute(attn_kernel<T, INT8, D, HB>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem);
    if (e != cudaSuccess) return e;
    allowed.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
  }
  const auto [whole, grid] =
      deal<G>(static_cast<long long>(a.batch) * a.kv.kv_heads * a.blocks, static_cast<long long>(a.columns) * a.kv.page_size, sm_count);
  char* const space = whole ? nullptr : static_cast<char*>(a.workspace) + kCounterBytes;
  a.records = whole ? nullptr : reinterpret_cast<Piece*>(space);
  a.partials = whole ? nullptr : reinterpret_cast<float*>(space + kRecordBytes);
  e = launch_dependent(attn_kernel<T, INT8, D, HB>, dim3(grid), kThreads, G::kSmem, s, a, maps);
  if (e != cudaSuccess || !a.records) return e;
  const unsigned parts = (std::min(a.group, HB) + join_heads(HB) - 1) / join_heads(HB);
  return launch_dependent(join_kernel<T, D, HB>, dim3(std::min<unsigned>(grid, kJoinBlocks * sm_count), parts), kJoinThreads, 0, s,
                          a.records, static_cast<int>(grid), a.partials, static_cast<T*>(a.out), a.lse);
}

// Query heads of one CTA: all of a KV head's where they fit, so that its keys are read and converted once. 16 instead of
// two blocks of 8 for 16 heads: 43.6 us against 54.9 (32 int8 requests of 8000 tokens); head_dim 256 has no registers for it.
int heads_per_cta(int group, int head_dim) { return group <= 4 ? 4 : group <= 8 || head_dim == 256 ? 8 : 16; }

template <typename T, bool INT8, int D>
cudaError_t attn_d(AttnArgs& a, int sm_count, cudaStream_t s) {
  const int hb = heads_per_cta(a.group, D);
  if (hb == 4) return attn_hb<T, INT8, D, 4>(a, sm_count, s);
  if constexpr (D != 256)
    if (hb == 16) return attn_hb<T, INT8, D, 16>(a, sm_count, s);
  return attn_hb<T, INT8, D, 8>(a, sm_count, s);
}

template <typename T, bool INT8>
cudaError_t attn_t(AttnArgs& a, int head_dim, int sm_count, cudaStream_t s) {
  return head_dim == 64    ? attn_d<T, INT8, 64>(a, sm_count, s)
         : head_dim == 128 ? attn_d<T, INT8, 128>(a, sm_count, s)
                           : attn_d<T, INT8, 256>(a, sm_count, s);
}

}  // namespace

// The records, and two partial rows per CTA
size_t bytes_for(unsigned ctas, int hb, int head_dim) {
  return kCounterBytes + kRecordBytes + 2ull * ctas * hb * (head_dim + 2) * sizeof(float);
}
size_t paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim, int sm_count) {
  return bytes_for(std::min(3 * sm_count, kMaxCtas), heads_per_cta(heads / std::max(1, kv_heads), head_dim), head_dim);
}

template <bool INT8, int D>
Deal deal_of(int hb, long long rows, long long room, int sm_count) {
  if (hb == 4) return deal<Geo<INT8, D, 4>>(rows, room, sm_count);
  if constexpr (D != 256)
    if (hb == 16) return deal<Geo<INT8, D, 16>>(rows, room, sm_count);
  return deal<Geo<INT8, D, 8>>(rows, room, sm_count);
}
template <bool INT8>
Deal deal_of(int hb, int head_dim, long long rows, long long room, int sm_count) {
  return head_dim == 64    ? deal_of<INT8, 64>(hb, rows, room, sm_count)
         : head_dim == 128 ? deal_of<INT8, 128>(hb, rows, room, sm_count)
                           : deal_of<INT8, 256>(hb, rows, room, sm_count);
}
size_t paged_attention_call_bytes(int batch, int heads, int kv_heads, int head_dim, bool int8, int columns, int page_size, int sm_count) {
  const int group = heads / kv_heads, hb = heads_per_cta(group, head_dim);
  const long long rows = static_cast<long long>(batch) * kv_heads * ((group + hb - 1) / hb), room = static_cast<long long>(columns) * page_size;
  const Deal d = int8 ? deal_of<true>(hb, head_dim, rows, room, sm_count) : deal_of<false>(hb, head_dim, rows, room, sm_count);
  return d.whole ? 0 : bytes_for(d.grid, hb, head_dim);
}

cudaError_t launch_paged_attention(const kl_paged_attention_args& p, int sm_count, int* status, cudaStream_t s) {
  const int dim = p.cache.head_dim;
  AttnArgs a;
  a.q = p.q;
  a.q_row_stride = p.q_row_stride;
  a.q_head_stride = p.q_head_stride;
  a.kv = kv_view(p.cache);
  a.table = p.page_table;
  a.table_stride = p.table_stride;
  a.lengths = p.lengths;
  a.batch = p.batch;
  a.heads = p.heads;
  a.columns = p.columns;
  a.group = p.heads / p.cache.kv_heads;
  const int hb = heads_per_cta(a.group, dim);
  a.blocks = (a.group + hb - 1) / hb;
  a.q_vec = (reinterpret_cast<uintptr_t>(p.q) % 4 == 0) && p.q_row_stride % 2 == 0 && p.q_head_stride % 2 == 0;
  a.scale = p.scale;
  a.out = p.out;
  a.lse = p.lse;
  a.workspace = p.workspace;                        // may be null where rows are not split
  a.status = status;
  const bool int8 = p.cache.format == KL_KV_INT8;
  if (p.dtype == KL_DT_BF16)
    return int8 ? attn_t<__nv_bfloat16, true>(a, dim, sm_count, s) : attn_t<__nv_bfloat16, false>(a, dim, sm_count, s);
  return int8 ? attn_t<__half, true>(a, dim, sm_count, s) : attn_t<__half, false>(a, dim, sm_count, s);
}

}  // namespace kl
