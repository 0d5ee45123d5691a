// paged.cu -- appending rotated keys and values to a paged KV cache and
// reading rows of it back (tl_paged_append, tl_paged_read).
#include <type_traits>

#include "kernels.cuh"
#include "serving.cuh"

namespace tl {

tl_status paged_view(const tl_paged_kv* c, const int32_t* table, int32_t n_seqs, int32_t max_pages,
                     int64_t table_stride, PagedView* out) {
  if (!c || !c->k || !c->v || !table) return TL_ERR_INVALID_ARGUMENT;
  if (c->dtype != TL_I8 && c->dtype != TL_BF16 && c->dtype != TL_F16) return TL_ERR_INVALID_ARGUMENT;
  if (c->dtype == TL_I8 && (!c->k_scale || !c->v_scale)) return TL_ERR_INVALID_ARGUMENT;
  if (c->head_dim != 64 && c->head_dim != 128) return TL_ERR_INVALID_ARGUMENT;
  if (c->num_pages <= 0 || c->kv_heads <= 0 || c->page_size <= 0) return TL_ERR_INVALID_ARGUMENT;
  if (n_seqs <= 0 || max_pages <= 0 || table_stride < max_pages) return TL_ERR_INVALID_ARGUMENT;
  if (!aligned_to(c->k, 16) || !aligned_to(c->v, 16) || !aligned_to(table, 4)) return TL_ERR_INVALID_ARGUMENT;
  // positions and row indexes are 31-bit, with room to round a length up
  constexpr int64_t kMost = INT32_MAX - 4096;
  if (static_cast<int64_t>(max_pages) * c->page_size > kMost ||
      static_cast<int64_t>(c->num_pages) * c->kv_heads > kMost / c->page_size)
    return TL_ERR_OUT_OF_RANGE;
  out->k = c->k;
  out->v = c->v;
  out->ks = c->k_scale;
  out->vs = c->v_scale;
  out->pages = c->num_pages;
  out->hkv = c->kv_heads;
  out->ps = c->page_size;
  out->div = page_div(c->page_size);
  out->table = table;
  out->n_seqs = n_seqs;
  out->max_pages = max_pages;
  out->table_stride = table_stride;
  return TL_OK;
}

namespace {

// Both kernels move rows and are bound by memory. A row belongs to a few
// neighbouring threads, each with 16 bytes of it a load, and a thread takes up
// to kRows rows of one token with all their loads in flight before the first
// use; the token's angles, sequence and page are looked up meanwhile, once.
constexpr int kThreads = 128;
constexpr int kRows = 4;

struct AppendArgs {
  PagedView c;
  const void *q, *k, *v;
  int64_t ldq, ldk, ldv;
  const int32_t *seq, *pos;
  const float *cos, *sin;
  int32_t max_pos, tokens, heads;
  int32_t groups;  // thread groups of a token: each takes rows g, g + groups, ...
  void* q_out;
};

// N consecutive elements as loaded (4, 8 or a multiple of 16 bytes), as
// float32, and back.
template <typename T, int N>
struct Raw {
  static constexpr int B = N * sizeof(T);
  static_assert(B == 4 || B == 8 || B % 16 == 0, "whole accesses");
  uint32_t w[B / 4];
  TL_DEV void load(const T* p) {
    if constexpr (B == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (B == 8) {
      const uint2 y = *reinterpret_cast<const uint2*>(p);
      w[0] = y.x, w[1] = y.y;
    } else {
#pragma unroll
      for (int i = 0; i < B / 16; ++i) {
        const uint4 y = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p) + 16 * i);
        w[4 * i] = y.x, w[4 * i + 1] = y.y, w[4 * i + 2] = y.z, w[4 * i + 3] = y.w;
      }
    }
  }
  TL_DEV void clear() {
#pragma unroll
    for (int i = 0; i < B / 4; ++i) w[i] = 0;
  }
  TL_DEV float operator[](int i) const {
    if constexpr (sizeof(T) == 4)
      return __uint_as_float(w[i]);
    else if constexpr (sizeof(T) == 1)
      return static_cast<float>(static_cast<int8_t>(w[i / 4] >> (8 * (i % 4))));
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
      return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else
      return i % 2 ? __high2float(*reinterpret_cast<const __half2*>(w + i / 2))
                   : __low2float(*reinterpret_cast<const __half2*>(w + i / 2));
  }
};
template <typename T, int N>
TL_DEV void store_n(T* p, const float* x) {
  constexpr int B = N * sizeof(T);
  static_assert(B == 8 || B % 16 == 0, "whole accesses");
  __align__(16) T y[N];
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = from_f32<T>(x[i]);
  if constexpr (B == 8) {
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(y);
  } else {
#pragma unroll
    for (int i = 0; i < B / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(y)[i];
  }
}

// Rotation of the pairs (a_i, b_i) = (x_j, x_(j + D/2)) by the token's angles,
// in float32 without contraction (the INT8 rounding that may follow has to see
// the reference's values), and quantize_int8 of the whole row, whose maximum
// is taken over the row's threads. A thread holds N pairs, 16 bytes of each
// half; D = 64, 32 + 2 * 4 head rows of bfloat16: 10 KB a token moved.
// Measured: 16721 such tokens (172 MB) 32.1 us, 5.4 TB/s; one token 1.8 us.
template <typename TI, typename TC, int D>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int N = 16 / sizeof(TI), LANES = D / 2 / N;  // pairs of a thread, threads of a row
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int j = static_cast<int>(id % LANES) * N;
  const unsigned part = static_cast<unsigned>(id / LANES);
  const int64_t t = part / static_cast<unsigned>(a.groups);
  const int g = static_cast<int>(part - static_cast<unsigned>(t) * a.groups);
  const bool in = t < a.tokens;  // (the row maxima below are warp-wide)
  const int rows = a.heads + 2 * a.c.hkv;
  pdl_begin();

  const int p = in ? a.pos[t] : -1, s = in ? a.seq[t] : -1;  // the longest chain of loads starts here
  Raw<TI, N> in_lo[kRows], in_hi[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int r = g + u * a.groups;
    if (!in || r >= rows) continue;
    const TI* x = r < a.heads ? static_cast<const TI*>(a.q) + t * a.ldq + r * D
                  : r < a.heads + a.c.hkv
                      ? static_cast<const TI*>(a.k) + t * a.ldk + (r - a.heads) * D
                      : static_cast<const TI*>(a.v) + t * a.ldv + (r - a.heads - a.c.hkv) * D;
    in_lo[u].load(x + j);
    in_hi[u].load(x + j + D / 2);
  }
  const bool angle = !a.cos || (p >= 0 && p < a.max_pos);
  Raw<float, N> cs, sn;
  if (a.cos && angle) {
    cs.load(a.cos + static_cast<int64_t>(p) * D + j);
    sn.load(a.sin + static_cast<int64_t>(p) * D + j);
  }
  const int64_t row0 = angle ? paged_row(a.c, s, p) : -1;

#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int r = g + u * a.groups;
    const bool query = r < a.heads, key = !query && r < a.heads + a.c.hkv;
    const bool here = in && r < rows;
    float lo[N], hi[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      lo[i] = here ? in_lo[u][i] : 0.0f;
      hi[i] = here ? in_hi[u][i] : 0.0f;
    }
    if ((query || key) && a.cos && angle) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float x = lo[i], y = hi[i];
        lo[i] = __fsub_rn(__fmul_rn(x, cs[i]), __fmul_rn(y, sn[i]));
        hi[i] = __fadd_rn(__fmul_rn(y, cs[i]), __fmul_rn(x, sn[i]));
      }
    }
    if (here && query) {
      TI* o = static_cast<TI*>(a.q_out) + (t * a.heads + r) * D + j;
      if (!angle) {
#pragma unroll
        for (int i = 0; i < N; ++i) lo[i] = hi[i] = 0.0f;
      }
      store_n<TI, N>(o, lo);
      store_n<TI, N>(o + D / 2, hi);
    }
    const int64_t row = row0 + static_cast<int64_t>(r - a.heads - (key ? 0 : a.c.hkv)) * a.c.ps;
    TC* o = static_cast<TC*>(key ? a.c.k : a.c.v) + row * D + j;
    const bool store = here && !query && row0 >= 0;
    if constexpr (sizeof(TC) == 1) {
      if (!__any_sync(0xffffffffu, store)) continue;
      // the row's maximum; a NaN or an infinity anywhere gives a NaN scale
      float m = 0.0f;
      if (store) {
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (lo[i] != lo[i] || hi[i] != hi[i]) m = INFINITY;
      }
#pragma unroll
      for (int w = 1; w < LANES; w <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
      if (store) {
        const bool bad = m == INFINITY;
        // absmax / 127 in float64 rounded to float32 is the float32 quotient (53 >= 2 * 24 + 2 bits)
        const float sc = bad ? __int_as_float(0x7fc00000) : m == 0.0f ? 1.0f : __fdiv_rn(m, 127.0f);
        const float inv = quant_inv(sc);
        const bool tiny = inv == INFINITY;  // a scale below 2^-128 has no reciprocal
        auto quantize = [&](float f) { return (tiny ? quantize_one(f, sc) : quantize_one_inv(f, sc, inv)) & 255; };
        uint32_t x[N / 4], y[N / 4];
#pragma unroll
        for (int i = 0; i < N / 4; ++i) x[i] = y[i] = 0;
        if (!bad) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            x[i / 4] |= quantize(lo[i]) << (8 * (i % 4));
            y[i / 4] |= quantize(hi[i]) << (8 * (i % 4));
          }
        }
        if constexpr (N == 4) {
          *reinterpret_cast<uint32_t*>(o) = x[0];
          *reinterpret_cast<uint32_t*>(o + D / 2) = y[0];
        } else {
          *reinterpret_cast<uint2*>(o) = make_uint2(x[0], x[1]);
          *reinterpret_cast<uint2*>(o + D / 2) = make_uint2(y[0], y[1]);
        }
        if (j == 0) (key ? a.c.ks : a.c.vs)[row] = sc;
      }
    } else if (store) {
      store_n<TC, N>(o, lo);
      store_n<TC, N>(o + D / 2, hi);
    }
  }
}

// Rows back as float32 or 16 bits: 16 bytes of output a thread and row.
// Measured: 32593 tokens of 8 heads of 128 (bfloat16, 267 MB) 45.2 us, 5.9 TB/s.
template <typename TC, typename TO, int D>
__global__ void __launch_bounds__(kThreads)
    read_kernel(const __grid_constant__ PagedView c, const int32_t* seq, const int32_t* pos, int32_t tokens,
                int32_t groups, TO* k_out, TO* v_out) {
  constexpr int N = 16 / sizeof(TO), LANES = D / N;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int j = static_cast<int>(id % LANES) * N;
  const unsigned part = static_cast<unsigned>(id / LANES);
  const int64_t t = part / static_cast<unsigned>(groups);
  const int g = static_cast<int>(part - static_cast<unsigned>(t) * groups);
  pdl_begin();
  if (t >= tokens) return;
  const int64_t row0 = paged_row(c, seq[t], pos[t]);
  Raw<TC, N> x[kRows];
  float sc[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int r = g + u * groups;
    const bool key = r < c.hkv;
    const int64_t row = row0 + static_cast<int64_t>(key ? r : r - c.hkv) * c.ps;
    sc[u] = 0.0f;
    x[u].clear();
    if (row0 < 0 || r >= 2 * c.hkv || !(key ? k_out : v_out)) continue;
    x[u].load(static_cast<const TC*>(key ? c.k : c.v) + row * D + j);
    if constexpr (sizeof(TC) == 1) sc[u] = (key ? c.ks : c.vs)[row];
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int r = g + u * groups;
    TO* o = r < c.hkv ? k_out : v_out;
    if (r >= 2 * c.hkv || !o) continue;
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = sizeof(TC) == 1 ? __fmul_rn(x[u][i], sc[u]) : x[u][i];
    store_n<TO, N>(o + (t * c.hkv + (r < c.hkv ? r : r - c.hkv)) * D + j, y);
  }
}

// Thread groups of a token and the grid for `rows` rows of `lanes` threads:
// one row a thread while that leaves SMs idle (one token of 40 rows 2.2
// against 2.4 us), then four, so that more of a token's bytes are in flight a
// thread and its angles and page are looked up less often (16 prompts: see
// above; with one row 40 us). False if the grid cannot hold them.
bool grid_for(int tokens, int rows, int lanes, int* groups, unsigned* grid) {
  const int64_t threads = static_cast<int64_t>(tokens) * rows * lanes;
  *groups = threads <= static_cast<int64_t>(device_sm_count()) * 1024 ? rows : (rows + kRows - 1) / kRows;
  const int64_t ctas = (static_cast<int64_t>(tokens) * *groups * lanes + kThreads - 1) / kThreads;
  *grid = static_cast<unsigned>(ctas);
  return static_cast<int64_t>(tokens) * *groups + kThreads <= INT32_MAX && ctas <= INT32_MAX;
}

template <typename TI, typename TC, int D>
tl_status append_launch(AppendArgs& a, cudaStream_t s) {
  unsigned grid;
  if (!grid_for(a.tokens, a.heads + 2 * a.c.hkv, D / 2 * sizeof(TI) / 16, &a.groups, &grid)) return TL_ERR_OUT_OF_RANGE;
  return launch_serving(append_kernel<TI, TC, D>, grid, kThreads, 0, 1, s, a);
}
template <typename TI, typename TC>
tl_status append_dim(AppendArgs& a, int d, cudaStream_t s) {
  return d == 64 ? append_launch<TI, TC, 64>(a, s) : append_launch<TI, TC, 128>(a, s);
}
template <typename TI>
tl_status append_pool(AppendArgs& a, int pool, int d, cudaStream_t s) {
  return pool == TL_I8     ? append_dim<TI, int8_t>(a, d, s)
         : pool == TL_BF16 ? append_dim<TI, __nv_bfloat16>(a, d, s)
                           : append_dim<TI, __half>(a, d, s);
}

struct ReadArgs {
  PagedView c;
  const int32_t *seq, *pos;
  int32_t tokens;
  void *k, *v;
};
template <typename TC, typename TO, int D>
tl_status read_launch(const ReadArgs& a, cudaStream_t s) {
  unsigned grid;
  int groups;
  if (!grid_for(a.tokens, 2 * a.c.hkv, D * sizeof(TO) / 16, &groups, &grid)) return TL_ERR_OUT_OF_RANGE;
  return launch_serving(read_kernel<TC, TO, D>, grid, kThreads, 0, 1, s, a.c, a.seq, a.pos, a.tokens, groups,
                        static_cast<TO*>(a.k), static_cast<TO*>(a.v));
}
template <typename TC, typename TO>
tl_status read_dim(const ReadArgs& a, int d, cudaStream_t s) {
  return d == 64 ? read_launch<TC, TO, 64>(a, s) : read_launch<TC, TO, 128>(a, s);
}
template <typename TC>
tl_status read_out(const ReadArgs& a, int out, int d, cudaStream_t s) {
  return out == TL_F32    ? read_dim<TC, float>(a, d, s)
         : out == TL_BF16 ? read_dim<TC, __nv_bfloat16>(a, d, s)
                          : read_dim<TC, __half>(a, d, s);
}

}  // namespace
}  // namespace tl

using namespace tl;

extern "C" {

tl_status tl_paged_append(const tl_paged_kv* cache, const tl_paged_append_args* args, void* stream) {
  if (!cache || !args) return TL_ERR_INVALID_ARGUMENT;
  const tl_paged_append_args& x = *args;
  AppendArgs a;
  const tl_status st = paged_view(cache, x.block_table, x.n_seqs, x.max_pages, x.table_stride, &a.c);
  if (st != TL_OK) return st;
  if (!x.k || !x.v || !x.seq || !x.pos || !is_float_dtype(x.dtype) || x.tokens <= 0) return TL_ERR_INVALID_ARGUMENT;
  if (!x.rope_cos != !x.rope_sin || (x.rope_cos && x.max_positions <= 0)) return TL_ERR_INVALID_ARGUMENT;
  if (!x.q != !x.q_out || (x.q && (x.heads <= 0 || !x.rope_cos))) return TL_ERR_INVALID_ARGUMENT;
  const int64_t d = cache->head_dim, e = dtype_bytes(x.dtype), kv = cache->kv_heads;
  if (x.k_stride < kv * d || x.v_stride < kv * d || (x.q && x.q_stride < x.heads * d)) return TL_ERR_INVALID_ARGUMENT;
  if (!aligned_to(x.k, 16) || !aligned_to(x.v, 16) || !aligned_to(x.q, 16) || !aligned_to(x.q_out, 16) ||
      (x.k_stride * e) % 16 || (x.v_stride * e) % 16 || (x.q && (x.q_stride * e) % 16) || !aligned_to(x.rope_cos, 16) ||
      !aligned_to(x.rope_sin, 16))
    return TL_ERR_INVALID_ARGUMENT;
  if (x.q && x.q == x.q_out && x.q_stride != x.heads * d) return TL_ERR_INVALID_ARGUMENT;
  a.q = x.q;
  a.k = x.k;
  a.v = x.v;
  a.ldq = x.q_stride;
  a.ldk = x.k_stride;
  a.ldv = x.v_stride;
  a.seq = x.seq;
  a.pos = x.pos;
  a.cos = x.rope_cos;
  a.sin = x.rope_sin;
  a.max_pos = x.max_positions;
  a.tokens = x.tokens;
  a.heads = x.q ? x.heads : 0;
  a.q_out = x.q_out;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return x.dtype == TL_F32    ? append_pool<float>(a, cache->dtype, cache->head_dim, s)
         : x.dtype == TL_BF16 ? append_pool<__nv_bfloat16>(a, cache->dtype, cache->head_dim, s)
                              : append_pool<__half>(a, cache->dtype, cache->head_dim, s);
}

tl_status tl_paged_read(const tl_paged_kv* cache, const tl_paged_read_args* args, void* stream) {
  if (!cache || !args) return TL_ERR_INVALID_ARGUMENT;
  const tl_paged_read_args& x = *args;
  ReadArgs a;
  const tl_status st = paged_view(cache, x.block_table, x.n_seqs, x.max_pages, x.table_stride, &a.c);
  if (st != TL_OK) return st;
  if (!x.seq || !x.pos || x.tokens <= 0 || !is_float_dtype(x.out_dtype) || (!x.k_out && !x.v_out))
    return TL_ERR_INVALID_ARGUMENT;
  if (!aligned_to(x.k_out, 16) || !aligned_to(x.v_out, 16)) return TL_ERR_INVALID_ARGUMENT;
  a.seq = x.seq;
  a.pos = x.pos;
  a.tokens = x.tokens;
  a.k = x.k_out;
  a.v = x.v_out;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int d = cache->head_dim;
  return cache->dtype == TL_I8     ? read_out<int8_t>(a, x.out_dtype, d, s)
         : cache->dtype == TL_BF16 ? read_out<__nv_bfloat16>(a, x.out_dtype, d, s)
                                   : read_out<__half>(a, x.out_dtype, d, s);
}

}  // extern "C"
