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
//  * work is split evenly over the CTAs whatever the lengths are (below);
//  * each warp owns a ring of tiles filled by cp.async two tiles ahead, and
//    each thread's copies are exactly the 16-byte pieces that its own MMA
//    fragments need: no bank conflicts, no transposes, no barriers;
//  * both products run on mma.sync m16n8k16. A group has few rows, so a
//    128-row tcgen05 tile would be mostly padding and its result would have
//    to come back through tensor memory; the 16-row tile is small enough to
//    stay far below the issue limit at full bandwidth.
//
// Precision. A 16-row tile holds 8 query heads twice: row g is the high part
// of head g's query (or of its probabilities), row g + 8 the low part, what
// rounding the high part to 16 bits left over. The sum of the two rows of the
// product is therefore the product with a 22-bit (float16) or 16-bit (bf16)
// operand, for no more instructions than one part takes with <= 8 heads. For
// a float32 query over a bf16 pool a third part (24 bits) takes a second MMA.
// Keys and values are exact: int8 converts to float16 exactly and its
// per-row scales multiply the scores and the probabilities in float32.
// Accumulators, maxima and sums are float32.
#include <algorithm>

#include "kernels.cuh"
#include "serving.cuh"

namespace tl {
namespace {

constexpr int kWarps = 4;         // warps of a CTA, each on its own tiles
constexpr int kMaxCtas = 640;     // grid bound (148 SMs x 4 CTAs), sizes the workspace
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Probabilities are kept as 2^(s' - m) with m 8 below the running maximum, and
// m moves only once the maximum has grown by more than 6: they stay within
// 2^14 (float16 holds 65504), small ones lose less to float16's smallest step,
// and most tiles rescale nothing.
constexpr float kHeadroom = 8.0f;
constexpr float kLazy = 6.0f;

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
  unsigned int* tickets;  // [kMaxCtas], zero between calls
  float* records;         // [kMaxCtas][2][kHeads][D + 2]
};

TL_DEV void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(live ? 16 : 0)
               : "memory");
}
TL_DEV void cp_async8(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)),
               "r"(live ? 8 : 0)
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

TL_DEV uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
TL_DEV uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
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
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
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

// Two int8 values, biased by 128 and placed in the low bytes of two float16
// 0x64xx = 1024 + byte, minus 1152: exact.
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
  static constexpr int KSEG = RB / 64;                  // 16-byte key pieces of a thread and position
  static constexpr int KS = D / 16;                     // MMA steps over head_dim
  static constexpr int VB = RB == 64 ? 8 : 16;          // bytes of a value piece
  static constexpr int CH = VB / (I8 ? 1 : 2);          // its elements
  static constexpr int VSEG = RB / (8 * VB);            // value pieces of a thread and position
  static constexpr int KBYTES = KT / 8 * KSEG * 512;
  static constexpr int VBYTES = KT / 4 * VSEG * 32 * VB;
  static constexpr int SCALES = KBYTES + VBYTES;        // offset of the tile's scales, then its mask
  static constexpr int MASK = SCALES + (I8 ? 2 * KT * 4 : 0);
  static constexpr int PITCH = D + 4;                   // floats between heads of a partial result
  static constexpr int MERGE = (HEADS * PITCH + 2 * HEADS) * 4;
  static constexpr int STAGE = ((MASK + 16 > MERGE ? MASK + 16 : MERGE) + 127) / 128 * 128;
  static constexpr int STAGES = RB == 64 ? 4 : 3;
  static constexpr int SMEM = kWarps * STAGES * STAGE;
  static constexpr int UNIT = kWarps * KT;              // positions of one CTA round
  static constexpr int RECORD = HEADS * (D + 2);        // floats of a partial result in the workspace
  static constexpr int CTAS = MT == 2 ? 2 : RB == 64 ? 3 : 2;  // CTAs an SM holds
};

// Length of row r in positions, 0 for rows that name no sequence.
TL_DEV int row_length(const AttendArgs& a, int r, int* seq) {
  const int s = a.seq ? a.seq[r] : r;
  *seq = s;
  int n = (s < 0 || s >= a.c.n_seqs) ? 0 : a.lengths[r];
  n = min(n, a.c.max_pages * a.c.ps);
  return max(n, 0);
}

// A place in the sequence of units: row r with `units` rounds an item, item
// `it` of the row (kv head and head block), round `rd` of the item.
struct Place {
  int r, seq, len, units, it, rd;
  template <int UNIT>
  TL_DEV void row(const AttendArgs& a, int row) {
    r = row;
    len = 0;
    units = 0;
    while (r < a.rows) {
      len = row_length(a, r, &seq);
      units = (len + UNIT - 1) / UNIT;
      if (units) break;
      ++r;
    }
  }
  template <int UNIT>
  TL_DEV void next(const AttendArgs& a, int items) {
    if (++rd < units) return;
    rd = 0;
    if (++it < items) return;
    it = 0;
    row<UNIT>(a, r + 1);
  }
};

TL_DEV void store_out(void* out, int dt, int64_t i, float4 v) {
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
TL_DEV float load_act(const void* p, int dt, int64_t i) {
  return dt == TL_F32    ? static_cast<const float*>(p)[i]
         : dt == TL_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i])
                         : __half2float(static_cast<const __half*>(p)[i]);
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

// The work: every row has ceil(length / UNIT) rounds for each of its
// kv_heads * blocks items; the rounds of all items in order form one line,
// which the CTAs cut into equal stretches. A CTA finishes the items that lie
// within its stretch; an item that crosses a border leaves a partial result
// in the workspace, and the CTA that brings an item's last one (a ticket
// counts them) joins them in CTA order, so the result does not depend on the
// order of arrival.
template <typename S>
__global__ void __launch_bounds__(kWarps * 32, S::CTAS) attend_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int D = S::D, MT = S::MT, KT = S::KT, UNIT = S::UNIT;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int sh_units[kWarps];
  __shared__ int sh_first[2];  // first row of the stretch, units before it
  __shared__ int sh_last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int items = a.c.hkv * a.blocks;

  // ---- the CTA's stretch [u0, u1) of the line
  int mine = 0;  // units: the launch keeps their number within 31 bits
  const int per = (a.rows + kWarps * 32 - 1) / (kWarps * 32);
  const int r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
  for (int r = r0; r < r1; ++r) {
    int s;
    const int len = row_length(a, r, &s);
    mine += (len + UNIT - 1) / UNIT;
  }
  mine *= items;
  int before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) sh_units[warp] = before;
  __syncthreads();
  int total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sh_units[w];
    total += sh_units[w];
  }
  before -= mine;
  const int ctas = static_cast<int>(gridDim.x), cta = static_cast<int>(blockIdx.x);
  const int chunk = static_cast<int>((total + static_cast<unsigned>(ctas) - 1) / ctas);
  const int u0 = static_cast<int>(min(static_cast<int64_t>(cta) * chunk, static_cast<int64_t>(total)));
  const int u1 = static_cast<int>(min(static_cast<int64_t>(u0) + chunk, static_cast<int64_t>(total)));
  if (u0 == u1) {
    zero_empty_rows<D>(a);
    return;
  }
  if (before <= u0 && u0 < before + mine) {
    int r = r0;
    int at = before;
    for (;; ++r) {
      int s;
      const int n = (row_length(a, r, &s) + UNIT - 1) / UNIT * items;
      if (u0 < at + n) break;
      at += n;
    }
    sh_first[0] = r;
    sh_first[1] = at;
  }
  __syncthreads();
  const int n_units = u1 - u0;
  Place use;
  use.row<UNIT>(a, sh_first[0]);
  use.it = (u0 - sh_first[1]) / use.units;
  use.rd = (u0 - sh_first[1]) % use.units;
  Place fill = use;

  // ---- the warp's ring
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * S::STAGES * S::STAGE;
  // Row index of position `lane` of the tile at `p` (lanes < KT), -1: none.
  auto lookup = [&](const Place& p) -> int {
    const int pos = (p.rd * kWarps + warp) * KT + lane;
    if (lane >= KT || p.units == 0 || pos >= p.len) return -1;
    const uint32_t pg = div_page(pos, a.c.div);
    const int page = __ldg(a.c.table + static_cast<int64_t>(p.seq) * a.c.table_stride + pg);
    if (page < 0 || page >= a.c.pages) return -1;
    return (page * a.c.hkv + p.it / a.blocks) * a.c.ps + (pos - static_cast<int>(pg * a.c.div.d));
  };
  auto copy_tile = [&](int stage, int row) {
    const uint32_t base = ring + stage * S::STAGE;
    const unsigned live = __ballot_sync(0xffffffffu, row >= 0);
    if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(base + S::MASK), "r"(live) : "memory");
    if (live == 0) return;  // nothing of the tile will be read
    const char* kp = static_cast<const char*>(a.c.k) + t * 16;
    const char* vp = static_cast<const char*>(a.c.v) + g * S::VB;
#pragma unroll
    for (int j = 0; j < KT / 8; ++j) {
      const int r = __shfl_sync(0xffffffffu, row, 8 * j + g);
      const char* src = kp + static_cast<int64_t>(max(r, 0)) * S::RB;
#pragma unroll
      for (int s = 0; s < S::KSEG; ++s)
        cp_async16(base + (j * S::KSEG + s) * 512 + lane * 16, src + s * 64, r >= 0);
    }
#pragma unroll
    for (int j = 0; j < KT / 4; ++j) {
      const int r = __shfl_sync(0xffffffffu, row, 16 * (j >> 2) + 8 * ((j >> 1) & 1) + 2 * t + (j & 1));
      const char* src = vp + static_cast<int64_t>(max(r, 0)) * S::RB;
#pragma unroll
      for (int s = 0; s < S::VSEG; ++s) {
        const uint32_t dst = base + S::KBYTES + (j * S::VSEG + s) * 32 * S::VB + lane * S::VB;
        if constexpr (S::VB == 16)
          cp_async16(dst, src + s * 128, r >= 0);
        else
          cp_async8(dst, src, r >= 0);
      }
    }
    if constexpr (S::I8) {
      if (lane < KT) {
        cp_async4(base + S::SCALES + lane * 4, a.c.ks + max(row, 0), row >= 0);
        cp_async4(base + S::SCALES + KT * 4 + lane * 4, a.c.vs + max(row, 0), row >= 0);
      }
    }
  };
  int filled = 0;
#pragma unroll
  for (int i = 0; i < S::STAGES - 1; ++i) {
    if (filled < n_units) {
      copy_tile(i, lookup(fill));
      fill.next<UNIT>(a, items);
      ++filled;
    }
    cp_async_commit();
  }
  int next_row = filled < n_units ? lookup(fill) : -1;

  // ---- the running state of one item
  uint32_t qa[MT][S::KS][4];                       // query, high and low rows
  uint32_t qc[S::PARTS == 3 ? MT : 1][S::KS][2];   // third part
  float qscale[MT];
  float o[MT][D / 8][4];
  float m[MT], l[MT];
  float vu = 0.0f, vinv = 1.0f;  // int8: the power of two that value scales are divided by, its inverse
  bool fresh = true;

  for (int i = 0, stage = 0; i < n_units; ++i, stage = stage + 1 == S::STAGES ? 0 : stage + 1) {
    if (fresh) {
      fresh = false;
      const int kvh = use.it / a.blocks, hb = use.it % a.blocks;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int hg = hb * S::HEADS + mt * 8 + g;
        const bool live = hg < a.group;
        const int64_t base = use.r * a.ldq + static_cast<int64_t>(kvh * a.group + (live ? hg : 0)) * D;
        float x[D / 4];
        float top = 0.0f;
        constexpr int RUN = S::I8 ? 16 : 8;  // consecutive elements of a thread
#pragma unroll
        for (int e = 0; e < D / 4; ++e) {
          const int d = e / RUN * 4 * RUN + t * RUN + e % RUN;
          x[e] = live ? load_act(a.q, a.q_dtype, base + d) : 0.0f;
          top = fmaxf(top, fabsf(x[e]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        float f = 1.0f;
        qscale[mt] = a.scale * kLog2e;
        if constexpr (!S::BF) {
          // a power of two that takes the row's largest element to [2^10, 2^11)
          const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
          const int sh = max(-120, min(120, 10 - e));
          f = __int_as_float((127 + sh) << 23);
          qscale[mt] = (a.scale * kLog2e) * __int_as_float((127 - sh) << 23);
        }
#pragma unroll
        for (int k = 0; k < S::KS; ++k) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float u = x[k * 4 + h * 2] * f, v = x[k * 4 + h * 2 + 1] * f;
            qa[mt][k][2 * h] = split<S::BF>(u, v);
            qa[mt][k][2 * h + 1] = split<S::BF>(u, v);
            if constexpr (S::PARTS == 3) qc[mt][k][h] = split<S::BF>(u, v);
          }
        }
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

    cp_async_wait<S::STAGES - 2>();
    __syncwarp();
    // refill the stage consumed one round ago
    if (filled < n_units) {
      copy_tile(stage == 0 ? S::STAGES - 1 : stage - 1, next_row);
      fill.next<UNIT>(a, items);
      ++filled;
      next_row = filled < n_units ? lookup(fill) : -1;
    }
    cp_async_commit();

    const uint32_t base = ring + stage * S::STAGE;
    unsigned live;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(live) : "r"(base + S::MASK));
    if (live) {
      // ---- scores: s[mt][j] of positions 8 j + 2 t, + 1 for head g
      float s[MT][KT / 8][2];
#pragma unroll
      for (int j = 0; j < KT / 8; ++j) {
        float c[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) c[mt][0] = c[mt][1] = c[mt][2] = c[mt][3] = 0.0f;
#pragma unroll
        for (int sg = 0; sg < S::KSEG; ++sg) {
          const uint4 w = lds16(base + (j * S::KSEG + sg) * 512 + lane * 16);
          const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int k = 0; k < (S::I8 ? 4 : 2); ++k) {
            uint32_t b0, b1;
            if constexpr (S::I8) {
              const uint32_t u = ww[k] ^ 0x80808080u;
              b0 = bytes_to_half2(u, 0x4140);
              b1 = bytes_to_half2(u, 0x4342);
            } else {
              b0 = ww[2 * k];
              b1 = ww[2 * k + 1];
            }
            const int ks = sg * (S::I8 ? 4 : 2) + k;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma16<S::BF>(c[mt], qa[mt][ks], b0, b1);
              if constexpr (S::PARTS == 3) {
                const uint32_t third[4] = {qc[mt][ks][0], 0u, qc[mt][ks][1], 0u};
                mma16<S::BF>(c[mt], third, b0, b1);
              }
            }
          }
        }
        float2 kscale = make_float2(1.0f, 1.0f);
        if constexpr (S::I8) {
          const uint2 w = lds8(base + S::SCALES + (8 * j + 2 * t) * 4);
          kscale = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
        }
        const bool in0 = live >> (8 * j + 2 * t) & 1, in1 = live >> (8 * j + 2 * t + 1) & 1;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float x = (c[mt][0] + c[mt][2]) * qscale[mt], y = (c[mt][1] + c[mt][3]) * qscale[mt];
          if constexpr (S::I8) {
            x *= kscale.x;
            y *= kscale.y;
          }
          s[mt][j][0] = in0 ? x : -INFINITY;
          s[mt][j][1] = in1 ? y : -INFINITY;
        }
      }
      // ---- running reference
      float vs[KT / 8][2];
      float vtop = 0.0f;
      if constexpr (S::I8) {
#pragma unroll
        for (int j = 0; j < KT / 8; ++j) {
          const uint2 w = lds8(base + S::SCALES + KT * 4 + (8 * j + 2 * t) * 4);
          vs[j][0] = __uint_as_float(w.x);
          vs[j][1] = __uint_as_float(w.y);
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
        top[mt] = fmaxf(top[mt], __shfl_xor_sync(0xffffffffu, top[mt], 2)) - kHeadroom;
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
      uint32_t pc[S::PARTS == 3 ? MT : 1][KT / 16][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const float ref = m[mt] == -INFINITY ? 0.0f : m[mt];
#pragma unroll
        for (int j = 0; j < KT / 8; ++j) {
          float x = exp2_approx(s[mt][j][0] - ref), y = exp2_approx(s[mt][j][1] - ref);
          l[mt] += x + y;
          if constexpr (S::I8) {
            x *= vs[j][0] * vinv;
            y *= vs[j][1] * vinv;
          }
          pa[mt][j >> 1][2 * (j & 1)] = split<S::BF>(x, y);
          pa[mt][j >> 1][2 * (j & 1) + 1] = split<S::BF>(x, y);
          if constexpr (S::PARTS == 3) pc[mt][j >> 1][j & 1] = split<S::BF>(x, y);
        }
      }
      // ---- o += p v
      auto mma_pv = [&](int kk, int n, uint32_t b0, uint32_t b1) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma16<S::BF>(o[mt][n], pa[mt][kk], b0, b1);
          if constexpr (S::PARTS == 3) {
            const uint32_t third[4] = {pc[mt][kk][0], 0u, pc[mt][kk][1], 0u};
            mma16<S::BF>(o[mt][n], third, b0, b1);
          }
        }
      };
#pragma unroll
      for (int kk = 0; kk < KT / 16; ++kk) {
#pragma unroll
        for (int sg = 0; sg < S::VSEG; ++sg) {
          uint32_t w[4][S::VB / 4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t p = base + S::KBYTES + ((kk * 4 + r) * S::VSEG + sg) * 32 * S::VB + lane * S::VB;
            if constexpr (S::VB == 16) {
              const uint4 x = lds16(p);
              w[r][0] = x.x, w[r][1] = x.y, w[r][2] = x.z, w[r][3] = x.w;
            } else {
              const uint2 x = lds8(p);
              w[r][0] = x.x, w[r][1] = x.y;
            }
          }
#pragma unroll
          for (int i4 = 0; i4 < S::VB / 4; ++i4) {
            if constexpr (S::I8) {
#pragma unroll
              for (int r = 0; r < 4; ++r) w[r][i4] ^= 0x80808080u;
#pragma unroll
              for (int h = 0; h < 2; ++h) {  // bytes 2 h, 2 h + 1 of the rows' words, paired by position
                const uint32_t lo = __byte_perm(w[0][i4], w[1][i4], h ? 0x7362 : 0x5140);
                const uint32_t hi = __byte_perm(w[2][i4], w[3][i4], h ? 0x7362 : 0x5140);
                const int n = sg * S::CH + 4 * i4 + 2 * h;
                mma_pv(kk, n, bytes_to_half2(lo, 0x4140), bytes_to_half2(hi, 0x4140));
                mma_pv(kk, n + 1, bytes_to_half2(lo, 0x4342), bytes_to_half2(hi, 0x4342));
              }
            } else {
              const int n = sg * S::CH + 2 * i4;
              mma_pv(kk, n, __byte_perm(w[0][i4], w[1][i4], 0x5410), __byte_perm(w[2][i4], w[3][i4], 0x5410));
              mma_pv(kk, n + 1, __byte_perm(w[0][i4], w[1][i4], 0x7632), __byte_perm(w[2][i4], w[3][i4], 0x7632));
            }
          }
        }
      }
    }

    // ---- the item's (or the stretch's) last round: join the warps
    if (use.rd + 1 == use.units || i + 1 == n_units) {
      float* part = reinterpret_cast<float*>(smem + (warp * S::STAGES + stage) * S::STAGE);
      __syncwarp();  // the stage's tile has been read by all lanes
      const float vback = S::I8 ? vu : 1.0f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        l[mt] += __shfl_xor_sync(0xffffffffu, l[mt], 1);
        l[mt] += __shfl_xor_sync(0xffffffffu, l[mt], 2);
        const int h = mt * 8 + g;
        if (t == 0) {
          part[S::HEADS * S::PITCH + h] = m[mt];
          part[S::HEADS * S::PITCH + S::HEADS + h] = l[mt];
        }
#pragma unroll
        for (int sg = 0; sg < S::VSEG; ++sg)
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < S::CH; e += 4) {
              float4 v;
              v.x = (o[mt][sg * S::CH + e][c] + o[mt][sg * S::CH + e][c + 2]) * vback;
              v.y = (o[mt][sg * S::CH + e + 1][c] + o[mt][sg * S::CH + e + 1][c + 2]) * vback;
              v.z = (o[mt][sg * S::CH + e + 2][c] + o[mt][sg * S::CH + e + 2][c + 2]) * vback;
              v.w = (o[mt][sg * S::CH + e + 3][c] + o[mt][sg * S::CH + e + 3][c + 2]) * vback;
              *reinterpret_cast<float4*>(part + h * S::PITCH + sg * 8 * S::CH + (2 * t + c) * S::CH + e) = v;
            }
      }
      __syncthreads();
      const int kvh = use.it / a.blocks, hb = use.it % a.blocks;
      const int nh = min(S::HEADS, a.group - hb * S::HEADS);
      const int first = u0 + i - use.rd;  // the item's first unit on the line
      const int c0 = first / chunk, c1 = (first + use.units - 1) / chunk;
      const bool whole = c0 == c1;
      const int64_t head0 = static_cast<int64_t>(use.r) * a.heads + kvh * a.group + hb * S::HEADS;
      float* rec = a.records + (static_cast<int64_t>(cta) * 2 + (cta == c0)) * S::RECORD;
      for (int x = tid * 4; x < nh * D; x += kWarps * 128) {
        const int h = x / D, d = x % D;
        float M = -INFINITY, L = 0.0f, pm[kWarps];
        float4 v = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          pm[w] = reinterpret_cast<const float*>(smem + (w * S::STAGES + stage) * S::STAGE)[S::HEADS * S::PITCH + h];
          M = fmaxf(M, pm[w]);
        }
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float* p = reinterpret_cast<const float*>(smem + (w * S::STAGES + stage) * S::STAGE);
          const float f = pm[w] == -INFINITY ? 0.0f : exp2_approx(pm[w] - M);
          const float4 y = *reinterpret_cast<const float4*>(p + h * S::PITCH + d);
          L += f * p[S::HEADS * S::PITCH + S::HEADS + h];
          v.x += f * y.x;
          v.y += f * y.y;
          v.z += f * y.z;
          v.w += f * y.w;
        }
        if (whole) {
          const bool empty = M == -INFINITY && L == 0.0f;
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
        __threadfence();
        __syncthreads();
        if (tid == 0) {
          const unsigned n = atomicAdd(a.tickets + c0, 1u);
          sh_last = n == static_cast<unsigned>(c1 - c0);
          if (sh_last) a.tickets[c0] = 0;
        }
        __syncthreads();
        if (sh_last) {
          __threadfence();
          for (int x = tid * 4; x < nh * D; x += kWarps * 128) {
            const int h = x / D, d = x % D;
            float M = -INFINITY, L = 0.0f;
            float4 v = make_float4(0, 0, 0, 0);
            for (int b = c0; b <= c1; ++b) {
              const float* p = a.records + (static_cast<int64_t>(b) * 2 + (b == c0)) * S::RECORD;
              const float4 y = __ldcg(reinterpret_cast<const float4*>(p + h * D + d));
              const float bm = __ldcg(p + S::HEADS * D + h), bl = __ldcg(p + S::HEADS * D + S::HEADS + h);
              const float nm = fmaxf(M, bm);
              const float f = M == -INFINITY ? 0.0f : exp2_approx(M - nm);
              const float e = bm == -INFINITY ? 0.0f : exp2_approx(bm - nm);
              L = L * f + bl * e;
              v.x = v.x * f + y.x * e;
              v.y = v.y * f + y.y * e;
              v.z = v.z * f + y.z * e;
              v.w = v.w * f + y.w * e;
              M = nm;
            }
            const bool empty = M == -INFINITY && L == 0.0f;
            const float inv = empty ? 0.0f : 1.0f / L;
            store_out(a.out, a.q_dtype, (head0 + h) * D + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
            if (a.lse && d == 0) a.lse[head0 + h] = empty ? -INFINITY : (M + log2f(L)) * kLn2;
          }
        }
      }
      __syncthreads();  // the stages that held the partial results may be refilled
      fresh = true;
    }
    use.next<UNIT>(a, items);
  }
  zero_empty_rows<D>(a);
}

template <typename S>
tl_status attend_launch(const AttendArgs& a, cudaStream_t s) {
  // the line of units has 31 bits
  const int64_t most = static_cast<int64_t>(a.c.hkv) * a.blocks *
                       ((static_cast<int64_t>(a.c.max_pages) * a.c.ps + S::UNIT - 1) / S::UNIT);
  if (most > INT32_MAX / a.rows) return TL_ERR_OUT_OF_RANGE;
  // once a device: the ring needs more shared memory than the default limit
  static bool ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TL_ERR_CUDA;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(attend_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM) != cudaSuccess)
      return TL_ERR_CUDA;
    ready[dev] = true;
  }
  // as many CTAs as the device holds at once, fewer where the table has no room for so many rounds
  const int64_t grid = std::min<int64_t>(most * a.rows, std::min(kMaxCtas, device_sm_count() * S::CTAS));
  attend_kernel<S><<<static_cast<unsigned>(grid), kWarps * 32, S::SMEM, s>>>(a);
  return cuda_status(cudaGetLastError());
}

// Groups of up to 8 query heads fit one 16-row tile, larger ones take two at a
// time so that the pool is read once for every 16 heads.
template <int POOL, int D, int PARTS>
tl_status attend_heads(AttendArgs& a, cudaStream_t s) {
  if (a.group <= 8) {
    a.blocks = 1;
    return attend_launch<Shape<POOL, D, 1, PARTS>>(a, s);
  }
  a.blocks = (a.group + 15) / 16;
  return attend_launch<Shape<POOL, D, 2, PARTS>>(a, s);
}
template <int POOL>
tl_status attend_dim(AttendArgs& a, int d, cudaStream_t s) {
  if constexpr (POOL == TL_BF16)
    if (a.q_dtype == TL_F32) return d == 64 ? attend_heads<POOL, 64, 3>(a, s) : attend_heads<POOL, 128, 3>(a, s);
  return d == 64 ? attend_heads<POOL, 64, 2>(a, s) : attend_heads<POOL, 128, 2>(a, s);
}

constexpr size_t kTicketBytes = (kMaxCtas * sizeof(unsigned int) + 255) / 256 * 256;

}  // namespace
}  // namespace tl

using namespace tl;

extern "C" {

size_t tl_paged_attn_workspace_bytes(int32_t heads, int32_t kv_heads, int32_t head_dim) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
  const size_t tile = heads / kv_heads <= 8 ? 8 : 16;
  return kTicketBytes + static_cast<size_t>(kMaxCtas) * 2 * tile * (head_dim + 2) * sizeof(float);
}

tl_status tl_paged_attn_decode(const tl_paged_kv* cache, const void* q, int32_t q_dtype, int64_t q_stride,
                               const int32_t* seq, const int32_t* lengths, const int32_t* block_table, int32_t n_seqs,
                               int32_t max_pages, int64_t table_stride, int32_t rows, int32_t heads, float sm_scale,
                               void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  AttendArgs a;
  const tl_status st = paged_view(cache, block_table, n_seqs, max_pages, table_stride, &a.c);
  if (st != TL_OK) return st;
  if (!q || !lengths || !out || !workspace || !is_float_dtype(q_dtype) || rows <= 0 || heads <= 0)
    return TL_ERR_INVALID_ARGUMENT;
  const int64_t d = cache->head_dim;
  if (heads % cache->kv_heads || q_stride < heads * d || (q_stride * dtype_bytes(q_dtype)) % 16)
    return TL_ERR_INVALID_ARGUMENT;
  if (!aligned_to(q, 16) || !aligned_to(out, 16) || !aligned_to(workspace, 16)) return TL_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < tl_paged_attn_workspace_bytes(heads, cache->kv_heads, cache->head_dim))
    return TL_ERR_OUT_OF_RANGE;
  if (!seq && rows > n_seqs) return TL_ERR_OUT_OF_RANGE;
  a.q = q;
  a.ldq = q_stride;
  a.q_dtype = q_dtype;
  a.seq = seq;
  a.lengths = lengths;
  a.rows = rows;
  a.heads = heads;
  a.group = heads / cache->kv_heads;
  a.scale = sm_scale;
  a.out = out;
  a.lse = lse;
  a.tickets = static_cast<unsigned int*>(workspace);
  a.records = reinterpret_cast<float*>(static_cast<char*>(workspace) + kTicketBytes);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return cache->dtype == TL_I8     ? attend_dim<TL_I8>(a, cache->head_dim, s)
         : cache->dtype == TL_BF16 ? attend_dim<TL_BF16>(a, cache->head_dim, s)
                                   : attend_dim<TL_F16>(a, cache->head_dim, s);
}

}  // extern "C"
