// paged_attn.cu -- attention of one new token per sequence over a paged KV
// cache (tl_paged_attn_decode).
//
// Mathematics. For one row, one kv head and the query heads that share it,
//   s_j = scale q . k_j,  out = sum_j 2^(s'_j - m) v_j / sum_j 2^(s'_j - m),
// s' = s log2 e, in one pass over the positions with a running reference m;
// disjoint ranges of positions give (m, l, o) triples that join as
//   m = max m_i,  l = sum 2^(m_i - m) l_i,  o = sum 2^(m_i - m) o_i.
//
// What bounds it. Each key and value byte is read once and used by the
// group's query heads only (a few operations a byte), so the bound is the
// rate of reading the pool. Everything else has to hide behind the loads:
//  * work is split evenly over the CTAs whatever the lengths are (below, at
//    attend_kernel);
//  * each warp owns a ring of tiles that TMA fills ahead of it (boxes of rows
//    of one page, 128-byte swizzle), so that no instruction of the warp moves
//    data and ldmatrix reads the operands without bank conflicts;
//  * both products run on mma.sync (m16n8k16, m16n8k32 for int8 keys). A group
//    has few rows, so a 128-row tcgen05 tile would be mostly padding and its
//    result would have to come back through tensor memory; the 16-row tile is
//    small enough to stay below the issue limit at full bandwidth.
// Measured: one context of 131149 positions (bf16, 8 kv heads of 128) 88.4 us,
// 6.1 TB/s (94.0 with a float32 query, 83.5 with 4 kv heads of 16 query heads
// each, 3.2 TB/s); 16 contexts up to 8192 (float16) 50.5 us, 5.4 TB/s; 64 up to
// 2048 over INT8 (4 kv heads of 64) 17.6 us, 2.1 TB/s: 38 MB are too few to hide
// the start (4 us), the joins (3 us) and the rounds' own chain (1.6 us each).
//
// Precision. Keys and values are exact, the other operand is split so that
// nothing but its last bits is rounded; accumulators, maxima and sums are
// float32.
//  * A 16-row tile holds 8 heads twice: row g is the high part of head g's
//    query (or of its probabilities), row g + 8 the low part, what rounding
//    the high part to 16 bits left over. The sum of the two rows of the
//    product is the product with a 22-bit (float16) or 16-bit (bf16) operand,
//    for no more instructions than one part takes with <= 8 heads. Over a bf16
//    pool a third part (24 bits) takes a second MMA: of the query where it is
//    float32, of the probabilities always. With 16 bits of those, 15 and 26 of
//    10000 bfloat16 outputs (17 and 5000 positions) were not the rounded
//    float64 result, with 24 bits 1 and 7; one context of 131149 positions
//    takes the same 89 us, 64 up to 2048 (4 kv heads of 64) 21.0 for 19.8.
//  * Over an INT8 pool the query is a 22-bit integer times a power of two, as
//    three signed digits to the base 256: two in the tile's rows, the third by
//    a second MMA. Their sums are whole numbers. The probabilities are split as
//    above and meet the values as float16, which holds every int8. The per-row
//    scales multiply the scores and the probabilities in float32.
#include <algorithm>
#include <numeric>

#include "kernels.cuh"
#include "serving.cuh"
#include "tc_common.cuh"

namespace tl {
namespace {

constexpr int kWarps = 4;         // warps of a CTA, each on its own tiles
// The workspace holds what the CTAs of a full device leave: at most kSms SMs
// of ctas_per_sm() CTAs, by query heads of a CTA and head_dim.
constexpr int kSms = 148;
constexpr int ctas_per_sm(int heads, int d) { return heads == 8 && d == 64 ? 3 : 2; }
constexpr int kMaxCtas = kSms * 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Probabilities are kept as 2^(s' - m) with m 8 below the running maximum, and
// m moves only once the maximum has grown by more than 6: they stay within
// 2^14 (float16 holds 65504), small ones lose less to float16's smallest step,
// and most tiles rescale nothing.
constexpr float kHeadroom = 8.0f;
constexpr float kLazy = 6.0f;

// Set when a wait on a tile ran out (tl_device_error reads and clears it).
__device__ unsigned int g_paged_error = 0;

struct AttendArgs {
  PagedView c;
  const void* q;
  int64_t ldq;
  int32_t q_dtype;
  const int32_t *seq, *lengths;
  int32_t rows, heads, group, blocks;  // query heads of a kv head; head blocks of a group
  float scale;
  void* out;
  float* lse;
  int32_t box;            // rows of a TMA box: the largest that divides a page and a tile
  unsigned int* tickets;  // [kMaxCtas], zero between calls
  float* records;         // [CTAs][2]: a partial result (HEADS rows, maxima, sums)
};

TL_DEV void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src))
               : "memory");
}
TL_DEV void cp_async4(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)),
               "r"(live ? 4 : 0)
               : "memory");
}
TL_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
TL_DEV void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

TL_DEV void prefetch_tensormap(const CUtensorMap* tm) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(tm)) : "memory");
}
// Four 8x8 matrices of 16-bit elements, lane l's address naming row l % 8 of
// matrix l / 8; TRANS transposes each.
template <bool TRANS>
TL_DEV uint4 ldmatrix4(uint32_t addr) {
  uint4 v;
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr));
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr));
  return v;
}
TL_DEV float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool BF>
TL_DEV void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 x 8 += 16 x 32 of int8 and 32 x 8.
TL_DEV void mma_s8(int* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// (x, y) as two 16-bit values, and what the rounding left over in x, y.
template <bool BF>
TL_DEV uint32_t split(float& x, float& y) {
  if constexpr (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    x -= __low2float(h);
    y -= __high2float(h);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    x -= __low2float(h);
    y -= __high2float(h);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Half of two bfloat16 values (exact), or the values: where a third part has an
// MMA of its own, both MMAs take half of the high part. Rows of zeros there
// would make a NaN of an infinite element.
template <bool HALF>
TL_DEV uint32_t half(uint32_t x) {
  if constexpr (!HALF) return x;
  const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x), __float2bfloat162_rn(0.5f));
  return *reinterpret_cast<const uint32_t*>(&y);
}

// Sum of the products with the high and with the low parts. An infinity among
// the stored elements (a float16 pool holds what append rounds to one) makes
// the first the whole answer, infinite by the sign of the operand, and the
// second a NaN or an infinity by the sign of what rounding left over.
TL_DEV float add_parts(float hi, float lo) { return fabsf(hi) < INFINITY ? hi + lo : hi; }

// Two int8 values, biased by 128 and placed in the low bytes of two float16
// 0x64xx = 1024 + byte, minus 1152: exact (the conversion by a number whose last
// place is 1: Kim et al., "Who Says Elephants Can't Run", 2022).
TL_DEV uint32_t bytes_to_half2(uint32_t biased, uint32_t selector) {
  const uint32_t h = __byte_perm(biased, 0x64646464u, selector);
  const uint32_t off = 0x64806480u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&off));
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <int POOL, int D_, int MT_, int PARTS_>
struct Shape {
  static constexpr int D = D_, MT = MT_, PARTS = PARTS_;
  static constexpr bool I8 = POOL == TL_I8, BF = POOL == TL_BF16;
  static constexpr int HEADS = 8 * MT;                  // query heads of a CTA
  static constexpr int RB = D * (I8 ? 1 : 2);           // bytes of a stored row
  static constexpr int KT = RB == 256 ? 16 : 32;        // positions of a warp's tile
  static constexpr int SUB = RB < 128 ? RB : 128;       // bytes of a row in one box
  static constexpr int NSUB = RB / SUB;
  static constexpr int KS = D / (I8 ? 32 : 16);         // steps of the first product over head_dim
  static constexpr int HALF = KT * RB;                  // bytes of a tile's keys, of its values
  static constexpr int MERGE = HEADS * D * 4;           // a warp's partial result
  static constexpr int STAGE = 2 * HALF;
  static_assert(STAGE % 1024 == 0 && (KT * SUB) % 1024 == 0, "swizzled boxes");
  // Tiles of a warp under way and CTAs an SM holds, each against the time of
  // the kernel as it was then. One context of 131149 positions (bf16, heads of
  // 128), 96.5 us: 3 tiles 151 (one CTA fits), 3 CTAs 129 (168 registers spill).
  // 64 contexts up to 2048 over INT8 heads of 64, 18.7 us: 3 tiles 19.1; when
  // it took 20.4, 4 tiles and 2 CTAs 23.8, 4 CTAs 20.8 (256 contexts: 46.5, 49.5;
  // 62 with tiles of 16 positions).
  static constexpr int STAGES = 2;
  static constexpr int CTAS = MT == 1 && RB == 64 ? 3 : 2;
  static_assert(CTAS <= ctas_per_sm(HEADS, D), "sizes the workspace");
  // Shared memory: rings, the warps' partial results, the query's parts, then
  // scales (int8), tile masks, partial m and l, query scales, barriers.
  static constexpr int RING = kWarps * STAGES * STAGE;
  static constexpr bool THIRD = I8 || PARTS == 3;       // the query has a third part
  static constexpr bool PTHIRD = BF;                    // the probabilities have a third part
  static constexpr int QROW = I8 ? D : D * 2;           // bytes of a part of a head's query
  static constexpr int QTILE = 16 * QROW, QTHIRD = THIRD ? 8 * QROW : 0;
  static constexpr int PARTS_AT = RING;
  static constexpr int QUERY = PARTS_AT + kWarps * MERGE;  // [m tile]: 16 rows (8 high, 8 low), then 8 third rows
  static constexpr int SCALES = QUERY + MT * (QTILE + QTHIRD);
  static constexpr int MASKS = SCALES + (I8 ? kWarps * STAGES * 2 * KT * 4 : 0);
  static constexpr int STATS = MASKS + kWarps * STAGES * 4;
  static constexpr int QSCALE = STATS + kWarps * 2 * HEADS * 4;
  static constexpr int BARS = (QSCALE + HEADS * 4 + 7) / 8 * 8;
  static constexpr int SMEM = BARS + kWarps * STAGES * 8 + 1024;  // the base is rounded up to 1024
  static constexpr int UNIT = kWarps * KT;              // positions of one CTA round
  // What ending an item costs a CTA (its warps' results joined, the next query,
  // its part written), in rounds: the line leaves such a gap behind every item,
  // so that CTAs that cross items get fewer rounds. When the gaps came in, 16
  // contexts up to 8192 (float16, heads of 128) took 61.3 us without them and
  // 54.6, 53.2, 52.0 with 1, 2, 3; 64 up to 2048 over INT8 22.9 and 21.1, 21.8,
  // 21.7. Rows of 128 bytes, 64 contexts up to 2048, with 1, 2, 3, 4: float16
  // heads of 64 20.3, 20.1, 20.8, 21.0, INT8 heads of 128 28.4, 28.2, 28.7, 28.8.
  static constexpr int GAP = RB == 256 ? 3 : RB == 128 ? 2 : 1;
  static constexpr int RECORD = HEADS * (D + 2);        // floats of a partial result in the workspace
};

// Length of row r in positions, 0 for rows that name no sequence.
TL_DEV int row_length(const AttendArgs& a, int r, int* seq) {
  const int n = a.lengths[r];  // both loads at once
  const int s = a.seq ? a.seq[r] : r;
  *seq = s;
  return s < 0 || s >= a.c.n_seqs ? 0 : max(0, min(n, a.c.max_pages * a.c.ps));
}

// A place on the line: round `rd` of the item of kv head `kvh` and head block
// `hb` of row r, whose items have `units` rounds; v is its number on the line.
struct Place {
  int r, len, units, kvh, hb, rd, v;
  const int32_t* pages;  // the row's block table

  TL_DEV void row(const AttendArgs& a, int row, int seq, int length, int unit) {
    r = row;
    len = length;
    units = (length + unit - 1) / unit;
    pages = a.c.table + static_cast<int64_t>(seq) * a.c.table_stride;
  }
  template <int UNIT, int GAP>
  TL_DEV void next(const AttendArgs& a) {
    ++v;
    if (++rd < units) return;
    v += GAP;
    rd = 0;
    if (++hb < a.blocks) return;
    hb = 0;
    if (++kvh < a.c.hkv) return;
    kvh = 0;
    int length = 0, seq = 0, row_ = r;
    while (++row_ < a.rows && (length = row_length(a, row_, &seq)) == 0) {
    }
    row(a, row_, length ? seq : 0, length, UNIT);
  }
};

// (a call: the code around the main loop runs once or twice a CTA, from a cold
// instruction cache, so it is kept short)
__device__ __noinline__ void store_out(void* out, int dt, int64_t i, float4 v) {
  if (dt == TL_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(out) + i) = v;
  } else if (dt == TL_BF16) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(v.x, v.y), y = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out) + i) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  } else {
    const __half2 x = __floats2half2_rn(v.x, v.y), y = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(static_cast<__half*>(out) + i) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
}
// Rows without positions are on nobody's line: zeros and -infinity.
template <int D>
TL_DEV void zero_empty_rows(const AttendArgs& a) {
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
    int s;
    if (row_length(a, r, &s)) continue;
    const int64_t base = static_cast<int64_t>(r) * a.heads;
    for (int i = threadIdx.x * 4; i < a.heads * D; i += kWarps * 128)
      store_out(a.out, a.q_dtype, base * D + i, make_float4(0, 0, 0, 0));
    if (a.lse)
      for (int i = threadIdx.x; i < a.heads; i += kWarps * 32) a.lse[base + i] = -INFINITY;
  }
}

// Joins the parts of an item, x = (first CTA, last CTA, first row of out, heads).
// It runs after all other work of the item, so its rounds of L2 latency show.
template <typename S>
__device__ void join_records(const AttendArgs& a, unsigned char* smem, int4 x) {
  constexpr int D = S::D;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c0 = x.x, c1 = x.y, nh = x.w;
  const int64_t head0 = x.z;
  constexpr int COLS = S::HEADS * D / (kWarps * 128), FEW = 6;
  auto record = [&](int b) { return a.records + (static_cast<int64_t>(b) * 2 + (b == c0)) * S::RECORD; };
  auto finish = [&](int c, float top, float sum, float4 v) {
    const int h = (tid * 4 + c * kWarps * 128) / D, d = (tid * 4) % D;
    if (h >= nh) return;
    const bool empty = top == -INFINITY && sum == 0.0f;
    if (empty) v = make_float4(0, 0, 0, 0);  // (weights of 0 may have met an infinite value)
    const float inv = empty ? 0.0f : 1.0f / sum;
    store_out(a.out, a.q_dtype, (head0 + h) * D + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
    if (a.lse && d == 0) a.lse[head0 + h] = empty ? -INFINITY : (top + log2f(sum)) * kLn2;
  };
  if (c1 - c0 < FEW) {
    // few records (a batch of ordinary contexts): every thread reads all that its column needs at once,
    // one round of latency (64 contexts up to 2048 over INT8: 18.8 us, 20.4 by the way below)
#pragma unroll 1
    for (int c = 0; c < COLS; ++c) {
      const int h = (tid * 4 + c * kWarps * 128) / D;
      float bm[FEW], bl[FEW], top = -INFINITY, sum = 0.0f;
      float4 y[FEW], v = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int k = 0; k < FEW; ++k) {  // (past the end: the last one again)
        const float* p = record(min(c0 + k, c1));
        bm[k] = __ldcg(p + S::HEADS * D + h);
        bl[k] = __ldcg(p + S::HEADS * D + S::HEADS + h);
        y[k] = __ldcg(reinterpret_cast<const float4*>(p + tid * 4 + c * kWarps * 128));
      }
#pragma unroll
      for (int k = 0; k < FEW; ++k) top = fmaxf(top, bm[k]);
#pragma unroll
      for (int k = 0; k < FEW; ++k)
        if (c0 + k <= c1) {
          const float e = bm[k] == -INFINITY ? 0.0f : exp2_approx(bm[k] - top);
          sum += bl[k] * e;
          v.x += y[k].x * e, v.y += y[k].y * e, v.z += y[k].z * e, v.w += y[k].w * e;
        }
      finish(c, top, sum, v);
    }
    return;
  }
  // Of each batch of records, a warp a head turns the maxima and sums into
  // weights in shared memory, and every thread sums its columns: as many loads
  // as registers allow are in flight, the first ones before the weights are
  // known (37 records of 8 x 128: about 4 us).
  constexpr int BATCH = 64, DEPTH = (S::CTAS > 2 ? 16 : 32) / COLS;
  float* weight = reinterpret_cast<float*>(smem + S::PARTS_AT);  // [head][record]
  float* top = reinterpret_cast<float*>(smem + S::STATS);        // [head]: maximum, sum, factor of the old sums
  float* sum = top + S::HEADS;
  float* old = sum + S::HEADS;
  float4 v[COLS], y[DEPTH][COLS];
  auto load = [&](int b, int end) {
#pragma unroll
    for (int k = 0; k < DEPTH; ++k)
#pragma unroll
      for (int c = 0; c < COLS; ++c)  // (past the end: the last one again)
        y[k][c] = __ldcg(reinterpret_cast<const float4*>(record(min(b + k, end - 1)) + tid * 4 + c * kWarps * 128));
  };
#pragma unroll
  for (int c = 0; c < COLS; ++c) v[c] = make_float4(0, 0, 0, 0);
  __syncthreads();
  if (tid < S::HEADS) {
    top[tid] = -INFINITY;
    sum[tid] = 0.0f;
  }
  __syncthreads();
#pragma unroll 1
  for (int b0 = c0; b0 <= c1; b0 += BATCH) {
    const int end = min(b0 + BATCH, c1 + 1);
    // lane = records b0 + lane, + 32; warp w takes heads w, w + 4, ...
    float rm[S::HEADS / kWarps][2], rl[S::HEADS / kWarps][2];
#pragma unroll
    for (int k = 0; k < S::HEADS / kWarps; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float* p = record(min(b0 + lane + 32 * i, end - 1)) + S::HEADS * D + warp + kWarps * k;
        rm[k][i] = __ldcg(p);
        rl[k][i] = __ldcg(p + S::HEADS);
      }
    load(b0, end);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (b0 + lane + 32 * i >= end)
#pragma unroll
        for (int k = 0; k < S::HEADS / kWarps; ++k) rm[k][i] = -INFINITY, rl[k][i] = 0.0f;
#pragma unroll
    for (int k = 0; k < S::HEADS / kWarps; ++k) {
      const int h = warp + kWarps * k;
      const float m0 = top[h], m1 = fmaxf(m0, warp_max(fmaxf(rm[k][0], rm[k][1])));
      float l1 = 0.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float e = rm[k][i] == -INFINITY ? 0.0f : exp2_approx(rm[k][i] - m1);
        weight[h * BATCH + lane + 32 * i] = e;
        l1 += e * rl[k][i];
      }
      l1 = warp_sum(l1);
      if (lane == 0) {
        const float f = m0 == -INFINITY ? 0.0f : exp2_approx(m0 - m1);
        top[h] = m1;
        sum[h] = sum[h] * f + l1;
        old[h] = f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const float f = old[(tid * 4 + c * kWarps * 128) / D];
      v[c].x *= f, v[c].y *= f, v[c].z *= f, v[c].w *= f;
    }
#pragma unroll 1
    for (int b1 = b0; b1 < end; b1 += DEPTH) {
      if (b1 > b0) load(b1, end);
#pragma unroll
      for (int k = 0; k < DEPTH; ++k)
        if (b1 + k < end) {
#pragma unroll
          for (int c = 0; c < COLS; ++c) {
            const float e = weight[(tid * 4 + c * kWarps * 128) / D * BATCH + b1 + k - b0];
            v[c].x += y[k][c].x * e;
            v[c].y += y[k][c].y * e;
            v[c].z += y[k][c].z * e;
            v[c].w += y[k][c].w * e;
          }
        }
    }
    __syncthreads();  // the weights have been used
  }
#pragma unroll 1
  for (int c = 0; c < COLS; ++c) {
    const int h = (tid * 4 + c * kWarps * 128) / D;
    float4 x = v[0];
#pragma unroll
    for (int k = 1; k < COLS; ++k)
      if (c == k) x = v[k];
    finish(c, top[h], sum[h], x);
  }
}

// The work: every row has ceil(length / UNIT) rounds for each of its
// kv_heads * blocks items; the rounds of all items in order form one line,
// which the CTAs cut into equal stretches. A CTA finishes the items that lie
// within its stretch; an item that crosses a border leaves a partial result
// in the workspace, and the CTA that brings an item's last one (a ticket
// counts them) joins them in CTA order, so the result does not depend on the
// order of arrival.
template <typename S>
__global__ void __launch_bounds__(kWarps * 32, S::CTAS)
    attend_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v) {
  constexpr int D = S::D, MT = S::MT, KT = S::KT, UNIT = S::UNIT;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ int sh_units[kWarps];
  __shared__ int4 sh_first;  // the stretch's first row, the units before it, the row's sequence and length
  __shared__ int sh_last[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int items = a.c.hkv * a.blocks;

  if (tid == 0) {
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }
  pdl_begin();
  // ---- the CTA's stretch [u0, u1) of the line
  const int ctas = static_cast<int>(gridDim.x), cta = static_cast<int>(blockIdx.x);
  const int per = (a.rows + kWarps * 32 - 1) / (kWarps * 32);
  const int r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
  int mine = 0;  // units: the launch keeps their number within 31 bits
  int seq = -1, len = 0;
  bool empty_row = false;  // a row without positions that this CTA writes
  for (int r = r0; r < r1; ++r) {
    len = row_length(a, r, &seq);
    mine += len ? (len + UNIT - 1) / UNIT + S::GAP : 0;
    if (len == 0) empty_row |= r % ctas == cta;
  }
  mine *= items;
  int before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) sh_units[warp] = before;
  empty_row = __syncthreads_or(empty_row);
  int total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sh_units[w];
    total += sh_units[w];
  }
  before -= mine;
  const int chunk = static_cast<int>((total + static_cast<unsigned>(ctas) - 1) / ctas);
  const int u0 = static_cast<int>(min(static_cast<int64_t>(cta) * chunk, static_cast<int64_t>(total)));
  const int u1 = static_cast<int>(min(static_cast<int64_t>(u0) + chunk, static_cast<int64_t>(total)));
  if (u0 == u1) {
    if (empty_row) zero_empty_rows<D>(a);
    return;
  }
  if (before <= u0 && u0 < before + mine) {
    int r = r0;
    for (; per > 1; ++r) {
      len = row_length(a, r, &seq);
      const int n = len ? ((len + UNIT - 1) / UNIT + S::GAP) * items : 0;
      if (u0 < before + n) break;
      before += n;
    }
    sh_first = make_int4(r, before, seq, len);
  }
  __syncthreads();
  Place use;
  use.row(a, sh_first.x, sh_first.z, sh_first.w, UNIT);
  {
    const int item = (u0 - sh_first.y) / (use.units + S::GAP);
    use.kvh = item / a.blocks;
    use.hb = item - use.kvh * a.blocks;
    use.rd = (u0 - sh_first.y) - item * (use.units + S::GAP);
  }
  use.v = u0;
  if (use.rd >= use.units) {  // in a gap: on from the item's last round
    use.v += use.units - 1 - use.rd;
    use.rd = use.units - 1;
    use.next<UNIT, S::GAP>(a);
  }
  if (use.v >= u1) {
    if (empty_row) zero_empty_rows<D>(a);
    return;
  }
  Place fill = use;

  // The query of the item at `p`: kQ consecutive elements a thread, first as
  // loaded, then as 16-bit parts in shared memory.
  constexpr int kQ = S::HEADS * D / (kWarps * 32), kLanes = D / kQ;  // elements of a thread, threads of a head
  const int qh = tid / kLanes, qd = tid % kLanes * kQ;
  uint4 raw[kQ / 4];
  auto load_query = [&](const Place& p) {
    const bool live = p.hb * S::HEADS + qh < a.group;
    const int64_t base =
        p.r * a.ldq + static_cast<int64_t>(p.kvh * a.group + (live ? p.hb * S::HEADS + qh : 0)) * D + qd;
    const char* q = static_cast<const char*>(a.q) + base * (a.q_dtype == TL_F32 ? 4 : 2);
#pragma unroll
    for (int e = 0; e < kQ / 4; ++e) raw[e] = make_uint4(0, 0, 0, 0);
    if (!live) return;
    if (a.q_dtype == TL_F32) {
#pragma unroll
      for (int e = 0; e < kQ / 4; ++e) raw[e] = *reinterpret_cast<const uint4*>(q + 16 * e);
    } else if constexpr (kQ == 4) {
      const uint2 y = *reinterpret_cast<const uint2*>(q);
      raw[0].x = y.x;
      raw[0].y = y.y;
    } else {
#pragma unroll
      for (int e = 0; e < kQ / 8; ++e) raw[e] = *reinterpret_cast<const uint4*>(q + 16 * e);
    }
  };
  auto store_query = [&]() {
    float x[kQ];
    const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
#pragma unroll
    for (int e = 0; e < kQ; ++e) {
      const uint32_t half = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
      x[e] = a.q_dtype == TL_F32    ? __uint_as_float(w[e])
             : a.q_dtype == TL_BF16 ? __uint_as_float(half << 16)
                                    : __half2float(__ushort_as_half(static_cast<unsigned short>(half)));
    }
    // the scale's sign goes into the query, so that larger products are larger scores
    float f = copysignf(1.0f, a.scale), back = fabsf(a.scale) * kLog2e;
    float top = 0.0f;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < kQ; ++e) {
      top = fmaxf(top, fabsf(x[e]));
      bad |= !(fabsf(x[e]) < INFINITY);
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) {
      if (!S::BF) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      bad |= __shfl_xor_sync(0xffffffffu, bad, o);
    }
    if constexpr (!S::BF) {
      // a power of two that takes the row's largest element to [2^10, 2^11), or [2^21, 2^22) for int8 digits
      constexpr int kTop = S::I8 ? 21 : 10;
      const int sh = max(-120, min(120, kTop - (static_cast<int>(__float_as_uint(top) >> 23) - 127)));
      f *= __int_as_float((127 + sh) << 23);
      back *= __int_as_float((127 - sh) << 23);
    }
    // not 0 (a scale of 0, or one that underflows with a small query): times it, -infinity stays what it is and
    // every finite product is below 1e-6; a NaN passes
    const float least = __int_as_float(1);
    back = back < least ? least : back;
    if (bad) back = __int_as_float(0x7fc00000);  // a NaN or an infinity in the query makes the row NaN
    if (qd == 0) reinterpret_cast<float*>(smem + S::QSCALE)[qh] = back;
    unsigned char* tile = smem + S::QUERY + (qh >> 3) * (S::QTILE + S::QTHIRD);
    const int row = qh & 7;
    if constexpr (S::I8) {
      // three signed digits to the base 256 of the element as a 22-bit integer
#pragma unroll
      for (int e = 0; e < kQ; e += 4) {
        uint32_t d0 = 0, d1 = 0, d2 = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int v = __float2int_rn(x[e + i] * f);
          const int v1 = (v - static_cast<int8_t>(v)) >> 8, v2 = (v1 - static_cast<int8_t>(v1)) >> 8;
          d0 |= (v & 255) << (8 * i);
          d1 |= (v1 & 255) << (8 * i);
          d2 |= (v2 & 255) << (8 * i);
        }
        const int d = qd + e, turn = S::QROW == 128 ? row : row >> 1;  // (rows 8-15 turn as 0-7)
        const int at = (((d >> 4) ^ turn) << 4) + (d & 15);
        *reinterpret_cast<uint32_t*>(tile + row * S::QROW + at) = d2;
        *reinterpret_cast<uint32_t*>(tile + (row + 8) * S::QROW + at) = d1;
        *reinterpret_cast<uint32_t*>(tile + S::QTILE + row * S::QROW + at) = d0;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kQ; e += 2) {
        const int d = qd + e, at = (((d >> 3) ^ row) << 4) + (d & 7) * 2;  // 16-byte pieces turned by the row
        float u = x[e] * f, v = x[e + 1] * f;
        *reinterpret_cast<uint32_t*>(tile + row * S::QROW + at) = half<S::PARTS == 3>(split<S::BF>(u, v));
        *reinterpret_cast<uint32_t*>(tile + (row + 8) * S::QROW + at) = split<S::BF>(u, v);
        if constexpr (S::PARTS == 3)
          *reinterpret_cast<uint32_t*>(tile + S::QTILE + row * S::QROW + at) = split<S::BF>(u, v);
      }
    }
  };
  load_query(use);

  // ---- the warp's ring
  unsigned char* ring = smem + warp * S::STAGES * S::STAGE;
  const uint32_t ring32 = smem_u32(ring);
  float* scales = reinterpret_cast<float*>(smem + S::SCALES) + warp * S::STAGES * 2 * KT;
  unsigned* masks = reinterpret_cast<unsigned*>(smem + S::MASKS) + warp * S::STAGES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BARS) + warp * S::STAGES;
  if (lane == 0) {
    for (int i = 0; i < S::STAGES; ++i) mbar_init(bars + i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  bool late = false;  // a wait has run out: the results are void, the host learns of it
  // Row index of position `lane` of the tile at `p` (lanes < KT), -1: none.
  auto lookup = [&](const Place& p) -> int {
    const int pos = (p.rd * kWarps + warp) * KT + lane;
    if (lane >= KT || pos >= p.len) return -1;
    const uint32_t pg = div_page(pos, a.c.div);
    // (no __ldg: the CTA may be there before a kernel that wrote the table has ended)
    const int page = p.pages[pg];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.c.pages)) return -1;
    return (page * a.c.hkv + p.kvh) * a.c.ps + (pos - static_cast<int>(pg * a.c.div.d));
  };
  // Boxes start at multiples of a.box positions and lie within one page, so a
  // box exists if its first position does (rows past the length stay unused).
  auto copy_tile = [&](int stage, int row) {
    // TMA writes whole 128 bytes: single rows of 64 bytes (odd page sizes) are copied by the lanes
    const bool tma = S::SUB == 128 || a.box > 1;
    const unsigned live = __ballot_sync(0xffffffffu, row >= 0);
    const bool head = tma && row >= 0 && lane % a.box == 0;
    const unsigned boxes = __ballot_sync(0xffffffffu, head);
    if (lane == 0) {
      masks[stage] = live;
      mbar_arrive_expect_tx(bars + stage, __popc(boxes) * a.box * S::RB * 2);
    }
    unsigned char* dst = ring + stage * S::STAGE + lane * S::SUB;
    if (head) {
#pragma unroll
      for (int s = 0; s < S::NSUB; ++s) {
        tma_load_2d(dst + s * KT * S::SUB, &tm_k, s * S::SUB, row, bars + stage);
        tma_load_2d(dst + S::HALF + s * KT * S::SUB, &tm_v, s * S::SUB, row, bars + stage);
      }
    }
    if constexpr (S::SUB == 64) {
      if (!tma && row >= 0) {
        const char* kp = static_cast<const char*>(a.c.k) + static_cast<int64_t>(row) * 64;
        const char* vp = static_cast<const char*>(a.c.v) + static_cast<int64_t>(row) * 64;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const int at = (p ^ (lane >> 1 & 3)) * 16;
          cp_async16(smem_u32(dst) + at, kp + p * 16);
          cp_async16(smem_u32(dst) + S::HALF + at, vp + p * 16);
        }
      }
    }
    if constexpr (S::I8) {
      if (lane < KT) {
        float* sc = scales + stage * 2 * KT + lane;
        cp_async4(smem_u32(sc), a.c.ks + max(row, 0), row >= 0);
        cp_async4(smem_u32(sc + KT), a.c.vs + max(row, 0), row >= 0);
      }
    }
  };
  int filled = 0, next_row = lookup(fill);

  // Byte offsets of this lane's ldmatrix rows, swizzled: 16-byte piece c of row
  // r of a box lies at piece c ^ (r % 8) of 128-byte rows, c ^ (r / 2 % 4) of
  // 64-byte rows. Row offsets that are multiples of 8 leave the swizzle alone.
  const int l8 = lane & 7, v_row = lane & 15;
  const uint32_t q32 = smem_u32(smem + S::QUERY);
  // matrices of a query ldmatrix: rows 0-7, 8-15 of piece 2 k, then of piece 2 k + 1
  const uint32_t q_row = q32 + v_row * S::QROW, q_piece = (lane >> 4) ^ (S::QROW == 64 ? l8 >> 1 : l8);
  const uint32_t k_lane = l8 * S::SUB + (((lane >> 3) ^ (S::SUB == 128 ? l8 : l8 >> 1)) << 4);
  const uint32_t v_lane = v_row * S::SUB + (((lane >> 4) ^ (S::SUB == 128 ? l8 : l8 >> 1)) << 4);

  // ---- the running state of one item
  float qscale[MT];
  float o[MT][D / 8][4];
  float m[MT], l[MT];
  float vu = 0.0f, vinv = 1.0f;  // int8: the power of two that value scales are divided by, its inverse
  bool fresh = true;
  int pending = 0;  // items that other CTAs have parts of: at most the stretch's first and last
  int4 late0{}, late1{};

  // The first STAGES turns only fill the ring.
  for (int i = -S::STAGES, stage = 0, phase = 1; i < 0 || use.v < u1; ++i) {
    if (i >= 0) {
      if (fresh) {
        fresh = false;
        store_query();
        // the next item's query is on its way while this one's rounds run
        Place ahead = use;
        ahead.v += ahead.units - 1 - ahead.rd;
        ahead.rd = ahead.units - 1;
        if (ahead.v < u1) ahead.next<UNIT, S::GAP>(a);
        if (ahead.v < u1) load_query(ahead);
        __syncthreads();  // the query is there, the last item's partial results have been read
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          qscale[mt] = reinterpret_cast<const float*>(smem + S::QSCALE)[mt * 8 + g];
          m[mt] = -INFINITY;
          l[mt] = 0.0f;
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.0f;
        }
        vu = 0.0f;
        vinv = 0.0f;
      }

      // (the clock is read only if there is something to wait for)
      if (!mbar_try_wait(bars + stage, phase) && (late || !mbar_wait_err(bars + stage, phase, 1u, &g_paged_error)))
        late = true;
      if constexpr (S::I8) cp_async_wait<S::STAGES - 1>();
      __syncwarp();
      const uint32_t kbase = ring32 + stage * S::STAGE, vbase = kbase + S::HALF;
      const float* sc = scales + stage * 2 * KT;
      const unsigned live = masks[stage];
      constexpr unsigned full = KT == 32 ? 0xffffffffu : 0xffffu;
      if constexpr (!S::I8) {
        // values of positions that do not exist must not meet a probability of zero as a NaN
        if (live != 0 && live != full) {
          for (int r = 0; r < KT; ++r)
            if (!(live >> r & 1) && lane < S::RB / 16)
              *reinterpret_cast<uint4*>(ring + stage * S::STAGE + S::HALF + (lane / (S::SUB / 16) * KT + r) * S::SUB +
                                        lane % (S::SUB / 16) * 16) = make_uint4(0, 0, 0, 0);
          __syncwarp();
        }
      }
      if (live) {
        // ---- products s[mt][j] of positions 8 j + 2 t, + 1 and head g, qscale times which are the scores
        float s[MT][KT / 8][2];
        uint32_t qa[MT][S::KS][4], third[S::THIRD ? MT : 1][S::KS][2];
        auto load_q = [&](int mt, int ks) {
          const uint32_t at = mt * (S::QTILE + S::QTHIRD) + (((2 * ks) ^ q_piece) << 4);
          const uint4 y = ldmatrix4<false>(q_row + at);
          qa[mt][ks][0] = y.x, qa[mt][ks][1] = y.y, qa[mt][ks][2] = y.z, qa[mt][ks][3] = y.w;
          if constexpr (S::THIRD) {
            // rows 0-7 only: matrices 1 and 3 repeat 0 and 2 and are not used
            const uint4 z = ldmatrix4<false>(q32 + S::QTILE + l8 * S::QROW + at);
            third[mt][ks][0] = z.x, third[mt][ks][1] = z.z;
          }
        };
        // 64 bytes of a key row at a time: lane l reads row l % 8, piece l / 8
        auto load_k = [&](int j, int q) {
          return ldmatrix4<false>(kbase + (q * 64 / S::SUB * KT + 8 * j) * S::SUB + (q * 64 % S::SUB ^ k_lane));
        };
        if constexpr (S::I8) {
#pragma unroll
          for (int ks = 0; ks < S::KS; ++ks)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) load_q(mt, ks);
#pragma unroll
          for (int j = 0; j < KT / 8; ++j) {
            int hi[MT][4], lo[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int e = 0; e < 4; ++e) hi[mt][e] = lo[mt][e] = 0;
#pragma unroll
            for (int q = 0; q < S::RB / 64; ++q) {
              const uint4 w = load_k(j, q);
#pragma unroll
              for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                  const uint32_t low[4] = {third[mt][2 * q + k][0], 0u, third[mt][2 * q + k][1], 0u};
                  mma_s8(hi[mt], qa[mt][2 * q + k], k ? w.z : w.x, k ? w.w : w.y);
                  mma_s8(lo[mt], low, k ? w.z : w.x, k ? w.w : w.y);
                }
            }
            const float2 kscale = *reinterpret_cast<const float2*>(sc + 8 * j + 2 * t);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              // digits' sums are at most 128 * 128 * 127: the lower two together fit 31 bits; float32 rounds
              // those and the whole once each
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float low = static_cast<float>(hi[mt][2 + e] * 256 + lo[mt][e]);
                s[mt][j][e] = fmaf(static_cast<float>(hi[mt][e]), 65536.0f, low) * (e ? kscale.y : kscale.x);
              }
            }
          }
        } else {
          float c[KT / 8][MT][4];
#pragma unroll
          for (int j = 0; j < KT / 8; ++j)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) c[j][mt][0] = c[j][mt][1] = c[j][mt][2] = c[j][mt][3] = 0.0f;
#pragma unroll
          for (int q = 0; q < S::RB / 64; ++q) {
            uint4 w[KT / 8];
#pragma unroll
            for (int j = 0; j < KT / 8; ++j) w[j] = load_k(j, q);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) load_q(mt, 2 * q + k);
#pragma unroll
              for (int j = 0; j < KT / 8; ++j)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                  const uint32_t b0 = k ? w[j].z : w[j].x, b1 = k ? w[j].w : w[j].y;
                  mma16<S::BF>(c[j][mt], qa[mt][2 * q + k], b0, b1);
                  if constexpr (S::PARTS == 3) {
                    const uint32_t* high = qa[mt][2 * q + k];
                    const uint32_t rest[4] = {high[0], third[mt][2 * q + k][0], high[2], third[mt][2 * q + k][1]};
                    mma16<S::BF>(c[j][mt], rest, b0, b1);
                  }
                }
            }
          }
#pragma unroll
          for (int j = 0; j < KT / 8; ++j)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              s[mt][j][0] = add_parts(c[j][mt][0], c[j][mt][2]);
              s[mt][j][1] = add_parts(c[j][mt][1], c[j][mt][3]);
            }
        }
        if (live != full)
#pragma unroll
          for (int j = 0; j < KT / 8; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (!(live >> (8 * j + 2 * t + e) & 1))
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt][j][e] = -INFINITY;
        // ---- running reference
        float vs[KT / 8][2];
        float vtop = 0.0f;
        if constexpr (S::I8) {
#pragma unroll
          for (int j = 0; j < KT / 8; ++j) {
            const float2 w = *reinterpret_cast<const float2*>(sc + KT + 8 * j + 2 * t);
            vs[j][0] = w.x;
            vs[j][1] = w.y;
            vtop = fmaxf(vtop, fmaxf(fabsf(vs[j][0]), fabsf(vs[j][1])));
          }
          vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, 1));
          vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, 2));
        }
        float top[MT];
        bool grow = S::I8 && vtop > vu;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          top[mt] = -INFINITY;
#pragma unroll
          for (int j = 0; j < KT / 8; ++j) top[mt] = fmaxf(top[mt], fmaxf(s[mt][j][0], s[mt][j][1]));
          top[mt] = fmaxf(top[mt], __shfl_xor_sync(0xffffffffu, top[mt], 1));
          top[mt] = fmaf(fmaxf(top[mt], __shfl_xor_sync(0xffffffffu, top[mt], 2)), qscale[mt], -kHeadroom);
          grow |= top[mt] > m[mt] + kLazy;
        }
        if (__any_sync(0xffffffffu, grow)) {
          float vcorr = 1.0f;
          if constexpr (S::I8) {
            if (vtop > vu) {  // the power of two at or above vtop (kept within float32's normal range)
              const uint32_t e = min(max((__float_as_uint(vtop) + 0x7fffffu) >> 23, 2u), 252u);
              const float nu = __uint_as_float(e << 23);
              vcorr = vu * __uint_as_float((254u - e) << 23);
              vu = nu;
              vinv = __uint_as_float((254u - e) << 23);
            }
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            float corr = vcorr;
            if (top[mt] > m[mt]) {
              const float f = exp2_approx(m[mt] - top[mt]);  // 0 from -infinity
              l[mt] *= f;
              corr *= f;
              m[mt] = top[mt];
            }
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[mt][n][e] *= corr;
          }
        }
        // ---- probabilities, high and low rows
        uint32_t pa[MT][KT / 16][4];
        uint32_t pc[S::PTHIRD ? MT : 1][KT / 16][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const float ref = m[mt] == -INFINITY ? 0.0f : m[mt];
#pragma unroll
          for (int j = 0; j < KT / 8; ++j) {
            float x = exp2_approx(fmaf(s[mt][j][0], qscale[mt], -ref));
            float y = exp2_approx(fmaf(s[mt][j][1], qscale[mt], -ref));
            l[mt] += x + y;
            if constexpr (S::I8) {
              x *= vs[j][0] * vinv;
              y *= vs[j][1] * vinv;
            }
            pa[mt][j >> 1][2 * (j & 1)] = half<S::PTHIRD>(split<S::BF>(x, y));
            pa[mt][j >> 1][2 * (j & 1) + 1] = split<S::BF>(x, y);
            if constexpr (S::PTHIRD) pc[mt][j >> 1][j & 1] = split<S::BF>(x, y);
          }
        }
        // ---- o += p v
        auto mma_pv = [&](int kk, int n, uint32_t b0, uint32_t b1) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma16<S::BF>(o[mt][n], pa[mt][kk], b0, b1);
            if constexpr (S::PTHIRD) {
              const uint32_t rest[4] = {pa[mt][kk][0], pc[mt][kk][0], pa[mt][kk][2], pc[mt][kk][1]};
              mma16<S::BF>(o[mt][n], rest, b0, b1);
            }
          }
        };
        // 32 bytes of 16 value rows at a time, transposed: lane l reads row l % 16, piece l / 16
#pragma unroll
        for (int kk = 0; kk < KT / 16; ++kk)
#pragma unroll
          for (int q = 0; q < S::RB / 32; ++q) {
            const uint4 w = ldmatrix4<true>(vbase + (q * 32 / S::SUB * KT + 16 * kk) * S::SUB +
                                            (q * 32 % S::SUB ^ v_lane));
            if constexpr (S::I8) {
              // a register holds elements 2 g, 2 g + 1 of position 2 t, then of 2 t + 1
              const uint32_t u[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                mma_pv(kk, 4 * q + 2 * h, bytes_to_half2(u[2 * h], 0x4240), bytes_to_half2(u[2 * h + 1], 0x4240));
                mma_pv(kk, 4 * q + 2 * h + 1, bytes_to_half2(u[2 * h], 0x4341), bytes_to_half2(u[2 * h + 1], 0x4341));
              }
            } else {
              mma_pv(kk, 2 * q, w.x, w.y);
              mma_pv(kk, 2 * q + 1, w.z, w.w);
            }
          }
      }
    }

    // ---- the tile has been read by all lanes (a fence, since copies belong to the async proxy): the next one
    // for its place
    fence_proxy_async_smem();
    __syncwarp();
    if (fill.v < u1) {
      copy_tile(stage, next_row);
      ++filled;
      fill.next<UNIT, S::GAP>(a);
      next_row = fill.v < u1 ? lookup(fill) : -1;
    }
    if constexpr (S::I8) cp_async_commit();

    // ---- the item's (or the stretch's) last round: join the warps
    if (i >= 0 && (use.rd + 1 == use.units || use.v + 1 == u1)) {
      float* part = reinterpret_cast<float*>(smem + S::PARTS_AT + warp * S::MERGE);
      float* stats = reinterpret_cast<float*>(smem + S::STATS);  // [warp][m, l][head]
      const float vback = S::I8 ? vu : 1.0f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        l[mt] += __shfl_xor_sync(0xffffffffu, l[mt], 1);
        l[mt] += __shfl_xor_sync(0xffffffffu, l[mt], 2);
        const int h = mt * 8 + g;
        if (t == 0) {
          stats[(warp * 2) * S::HEADS + h] = m[mt];
          stats[(warp * 2 + 1) * S::HEADS + h] = l[mt];
        }
        // element d of head h at d ^ 8 (h % 8): the lanes of a store spread over the banks
        float* row = part + h * D;
        const int turn = 8 * g;
#pragma unroll
        for (int n = 0; n < D / 8; n += S::I8 ? 2 : 1) {
          if constexpr (S::I8) {
            float4 v;
            v.x = add_parts(o[mt][n][0], o[mt][n][2]) * vback;
            v.y = add_parts(o[mt][n + 1][0], o[mt][n + 1][2]) * vback;
            v.z = add_parts(o[mt][n][1], o[mt][n][3]) * vback;
            v.w = add_parts(o[mt][n + 1][1], o[mt][n + 1][3]) * vback;
            *reinterpret_cast<float4*>(row + ((8 * n + 4 * t) ^ turn)) = v;
          } else {
            *reinterpret_cast<float2*>(row + ((8 * n + 2 * t) ^ turn)) =
                make_float2(add_parts(o[mt][n][0], o[mt][n][2]), add_parts(o[mt][n][1], o[mt][n][3]));
          }
        }
      }
      const Place done = use;
      use.next<UNIT, S::GAP>(a);
      __syncthreads();
      const int nh = min(S::HEADS, a.group - done.hb * S::HEADS);
      const int first = done.v - done.rd;  // the item's first round on the line
      const int c0 = first / chunk, c1 = (first + done.units - 1) / chunk;
      const bool whole = c0 == c1;
      const int64_t head0 = static_cast<int64_t>(done.r) * a.heads + done.kvh * a.group + done.hb * S::HEADS;
      float* rec = a.records + (static_cast<int64_t>(cta) * 2 + (cta == c0)) * S::RECORD;
#pragma unroll 1
      for (int x = tid * 4; x < (whole ? nh : S::HEADS) * D; x += kWarps * 128) {
        const int h = x / D, d = x % D;
        float M = -INFINITY, L = 0.0f, pm[kWarps];
        float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          pm[w] = stats[(w * 2) * S::HEADS + h];
          M = fmaxf(M, pm[w]);
        }
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float* p = reinterpret_cast<const float*>(smem + S::PARTS_AT + w * S::MERGE);
          const float f = pm[w] == -INFINITY ? 0.0f : exp2_approx(pm[w] - M);
          const float4 y = *reinterpret_cast<const float4*>(p + h * D + (d ^ (8 * (h & 7))));
          L += f * stats[(w * 2 + 1) * S::HEADS + h];
          v.x += f * y.x;
          v.y += f * y.y;
          v.z += f * y.z;
          v.w += f * y.w;
        }
        if (whole) {
          const bool empty = M == -INFINITY && L == 0.0f;
          if (empty) v = make_float4(0, 0, 0, 0);  // (as when records are joined)
          const float inv = empty ? 0.0f : 1.0f / L;
          store_out(a.out, a.q_dtype, (head0 + h) * D + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
          if (a.lse && d == 0) a.lse[head0 + h] = empty ? -INFINITY : (M + log2f(L)) * kLn2;
        } else {
          *reinterpret_cast<float4*>(rec + h * D + d) = v;
          if (d == 0) {
            rec[S::HEADS * D + h] = M;
            rec[S::HEADS * D + S::HEADS + h] = L;
          }
        }
      }
      if (!whole) {
        if (pending == 0)
          late0 = make_int4(c0, c1, static_cast<int>(head0), nh);
        else
          late1 = make_int4(c0, c1, static_cast<int>(head0), nh);
        ++pending;
      }
      fresh = true;
    } else if (i >= 0) {
      use.next<UNIT, S::GAP>(a);
    }
    if (++stage == S::STAGES) {
      stage = 0;
      phase ^= 1;
    }
  }
  if (pending) {
    // tickets are drawn at the end, when all parts are written: the CTA that
    // draws an item's last one joins its parts
    __syncthreads();
    if (tid < pending) {
      const int4 x = tid ? late1 : late0;
      __threadfence();  // the CTA's writes, ordered before by the barrier, before the ticket
      const bool last = atomicAdd(a.tickets + x.x, 1u) == static_cast<unsigned>(x.y - x.x);
      if (last) a.tickets[x.x] = 0;
      __threadfence();  // the other CTAs' writes after it
      sh_last[tid] = last;
    }
    __syncthreads();
#pragma unroll 1
    for (int j = 0; j < pending; ++j)
      if (sh_last[j]) join_records<S>(a, smem, j ? late1 : late0);
  }
  if (late)  // copies still under way must not land after the CTA has gone
    for (int i = max(0, filled - S::STAGES); i < filled; ++i)
      mbar_wait_err(bars + i % S::STAGES, i / S::STAGES & 1, 2u, &g_paged_error);
  if (empty_row) zero_empty_rows<D>(a);
}

template <typename S>
tl_status attend_launch(AttendArgs& a, cudaStream_t s) {
  // the line of units has 31 bits
  const int64_t most = static_cast<int64_t>(a.c.hkv) * a.blocks *
                       ((static_cast<int64_t>(a.c.max_pages) * a.c.ps + S::UNIT - 1) / S::UNIT);
  if (most + static_cast<int64_t>(a.c.hkv) * a.blocks * S::GAP > INT32_MAX / a.rows) return TL_ERR_OUT_OF_RANGE;
  static Once<64> ready;  // the ring needs more shared memory than the default limit
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || !ready(dev, [] { return allow_shared(attend_kernel<S>, S::SMEM); }))
    return TL_ERR_CUDA;
  // as many CTAs as the device holds at once, fewer where the table has no room for so many rounds
  const int64_t grid = std::min<int64_t>(most * a.rows, std::min(kSms, device_sm_count()) * S::CTAS);
  a.box = std::gcd(a.c.ps, S::KT);
  CUtensorMap tm_k, tm_v;
  const long long pool_rows = static_cast<long long>(a.c.pages) * a.c.hkv * a.c.ps;
  if (tc_encode_rows_bytes(&tm_k, a.c.k, pool_rows, S::RB, a.box) != cudaSuccess ||
      tc_encode_rows_bytes(&tm_v, a.c.v, pool_rows, S::RB, a.box) != cudaSuccess)
    return TL_ERR_CUDA;
  return launch_serving(attend_kernel<S>, static_cast<unsigned>(grid), kWarps * 32, S::SMEM, 1, s, a, tm_k, tm_v);
}

// Groups of up to 8 query heads fit one 16-row tile, larger ones take two at a
// time so that the pool is read once for every 16 heads: groups of 16 over one
// context of 131149 positions (bf16, 4 kv heads of 128) 84 us, 89 with one tile;
// 64 contexts up to 8192 over INT8 (4 kv heads of 64) 64 and 73. INT8 heads of 128 take
// one tile at a time: two spill registers, 53 us against 43 (64 contexts up to
// 2048), 152 against 132 (256 of them).
template <int POOL, int D, int PARTS>
tl_status attend_heads(AttendArgs& a, cudaStream_t s) {
  constexpr bool kTwo = !(POOL == TL_I8 && D == 128);
  if constexpr (kTwo) {
    if (a.group > 8) {
      a.blocks = (a.group + 15) / 16;
      return attend_launch<Shape<POOL, D, 2, PARTS>>(a, s);
    }
  }
  a.blocks = (a.group + 7) / 8;
  return attend_launch<Shape<POOL, D, 1, PARTS>>(a, s);
}
template <int POOL>
tl_status attend_dim(AttendArgs& a, int d, cudaStream_t s) {
  if constexpr (POOL == TL_BF16)
    if (a.q_dtype == TL_F32) return d == 64 ? attend_heads<POOL, 64, 3>(a, s) : attend_heads<POOL, 128, 3>(a, s);
  return d == 64 ? attend_heads<POOL, 64, 2>(a, s) : attend_heads<POOL, 128, 2>(a, s);
}

constexpr size_t kTicketBytes = (kMaxCtas * sizeof(unsigned int) + 255) / 256 * 256;

}  // namespace

cudaError_t paged_attn_read_error(unsigned int* code) {
  const cudaError_t e = cudaMemcpyFromSymbol(code, g_paged_error, sizeof(unsigned int));
  if (e != cudaSuccess || !*code) return e;
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_paged_error, &zero, sizeof(unsigned int));
}

}  // namespace tl

using namespace tl;

extern "C" {

size_t tl_paged_attn_workspace_bytes(int32_t heads, int32_t kv_heads, int32_t head_dim) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
  const int tile = heads / kv_heads <= 8 ? 8 : 16;
  return kTicketBytes +
         static_cast<size_t>(kSms) * ctas_per_sm(tile, head_dim) * 2 * tile * (head_dim + 2) * sizeof(float);
}

tl_status tl_paged_attn_decode(const tl_paged_kv* cache, const tl_paged_attn_args* args, void* stream) {
  if (!cache || !args) return TL_ERR_INVALID_ARGUMENT;
  const tl_paged_attn_args& x = *args;
  AttendArgs a;
  const tl_status st = paged_view(cache, x.block_table, x.n_seqs, x.max_pages, x.table_stride, &a.c);
  if (st != TL_OK) return st;
  if (!x.q || !x.lengths || !x.out || !x.workspace || !is_float_dtype(x.q_dtype) || x.rows <= 0 || x.heads <= 0)
    return TL_ERR_INVALID_ARGUMENT;
  const int64_t d = cache->head_dim;
  if (x.heads % cache->kv_heads || x.q_stride < x.heads * d || (x.q_stride * dtype_bytes(x.q_dtype)) % 16)
    return TL_ERR_INVALID_ARGUMENT;
  if (!aligned_to(x.q, 16) || !aligned_to(x.out, 16) || !aligned_to(x.workspace, 16)) return TL_ERR_INVALID_ARGUMENT;
  if (x.workspace_bytes < tl_paged_attn_workspace_bytes(x.heads, cache->kv_heads, cache->head_dim))
    return TL_ERR_OUT_OF_RANGE;
  if ((!x.seq && x.rows > x.n_seqs) || x.rows > INT32_MAX / x.heads) return TL_ERR_OUT_OF_RANGE;
  a.q = x.q;
  a.ldq = x.q_stride;
  a.q_dtype = x.q_dtype;
  a.seq = x.seq;
  a.lengths = x.lengths;
  a.rows = x.rows;
  a.heads = x.heads;
  a.group = x.heads / cache->kv_heads;
  a.scale = x.sm_scale;
  a.out = x.out;
  a.lse = x.lse;
  a.tickets = static_cast<unsigned int*>(x.workspace);
  a.records = reinterpret_cast<float*>(static_cast<char*>(x.workspace) + kTicketBytes);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return cache->dtype == TL_I8     ? attend_dim<TL_I8>(a, cache->head_dim, s)
         : cache->dtype == TL_BF16 ? attend_dim<TL_BF16>(a, cache->head_dim, s)
                                   : attend_dim<TL_F16>(a, cache->head_dim, s);
}

}  // extern "C"
