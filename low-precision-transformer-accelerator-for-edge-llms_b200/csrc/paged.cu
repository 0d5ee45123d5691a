// paged.cu -- appending rotated keys and values to a paged KV cache and
// reading rows of it back (tl_paged_append, tl_paged_read).
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

struct AppendArgs {
  PagedView c;
  const void *q, *k, *v;
  int64_t ldq, ldk, ldv;
  const int32_t *seq, *pos;
  const float *cos, *sin;
  int32_t max_pos, tokens, heads;
  void* q_out;
};

// One warp per (token, head row): heads query rows, then kv_heads key rows,
// then kv_heads value rows. Lane l holds the pairs j = l, l + 32 < D / 2.
template <typename TI, typename TC, int D>
__global__ void append_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int per = (a.q ? a.heads : 0) + 2 * a.c.hkv;
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (w >= static_cast<int64_t>(a.tokens) * per) return;
  const int t = static_cast<int>(w / per);
  int h = static_cast<int>(w % per);
  int kind = 2;  // 0 query, 1 key, 2 value
  const int hq = a.q ? a.heads : 0;
  if (h < hq) {
    kind = 0;
  } else if (h < hq + a.c.hkv) {
    kind = 1;
    h -= hq;
  } else {
    h -= hq + a.c.hkv;
  }
  const int p = a.pos[t];
  const bool angle = !a.cos || (p >= 0 && p < a.max_pos);
  const TI* src = kind == 0   ? static_cast<const TI*>(a.q) + t * a.ldq
                  : kind == 1 ? static_cast<const TI*>(a.k) + t * a.ldk
                              : static_cast<const TI*>(a.v) + t * a.ldv;
  src += h * D;
  constexpr int NP = D / 64;
  float lo[NP], hi[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int j = lane + 32 * i;
    lo[i] = to_f32(src[j]);
    hi[i] = to_f32(src[j + D / 2]);
    if (kind != 2 && a.cos) {
      const float cs = angle ? a.cos[static_cast<int64_t>(p) * D + j] : 0.0f;
      const float sn = angle ? a.sin[static_cast<int64_t>(p) * D + j] : 0.0f;
      const float x = lo[i], y = hi[i];
      lo[i] = __fsub_rn(__fmul_rn(x, cs), __fmul_rn(y, sn));
      hi[i] = __fadd_rn(__fmul_rn(y, cs), __fmul_rn(x, sn));
    }
  }
  if (kind == 0) {
    TI* o = static_cast<TI*>(a.q_out) + (static_cast<int64_t>(t) * a.heads + h) * D;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      o[lane + 32 * i] = from_f32<TI>(angle ? lo[i] : 0.0f);
      o[lane + 32 * i + D / 2] = from_f32<TI>(angle ? hi[i] : 0.0f);
    }
    return;
  }
  const int64_t row0 = angle ? paged_row(a.c, a.seq[t], p) : -1;
  if (row0 < 0) return;
  const int64_t row = row0 + static_cast<int64_t>(h) * a.c.ps;
  TC* o = static_cast<TC*>(kind == 1 ? a.c.k : a.c.v) + row * D;
  if constexpr (sizeof(TC) == 1) {
    float m = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      m = fmaxf(m, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
      bad |= !isfinite(lo[i]) || !isfinite(hi[i]);
    }
    m = warp_max(m);
    bad = __any_sync(0xffffffffu, bad);
    const float sc = bad ? __int_as_float(0x7fc00000) : static_cast<float>(quant_scale64(m));
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      o[lane + 32 * i] = bad ? 0 : static_cast<int8_t>(quantize_one(lo[i], sc));
      o[lane + 32 * i + D / 2] = bad ? 0 : static_cast<int8_t>(quantize_one(hi[i], sc));
    }
    if (lane == 0) (kind == 1 ? a.c.ks : a.c.vs)[row] = sc;
  } else {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      o[lane + 32 * i] = from_f32<TC>(lo[i]);
      o[lane + 32 * i + D / 2] = from_f32<TC>(hi[i]);
    }
  }
}

// One warp per (token, kv head) of K, then of V.
template <typename TC, typename TO, int D>
__global__ void read_kernel(PagedView c, const int32_t* seq, const int32_t* pos, int32_t tokens, TO* k_out,
                            TO* v_out) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (w >= static_cast<int64_t>(tokens) * 2 * c.hkv) return;
  const int t = static_cast<int>(w / (2 * c.hkv));
  int h = static_cast<int>(w % (2 * c.hkv));
  const bool key = h < c.hkv;
  if (!key) h -= c.hkv;
  TO* o = key ? k_out : v_out;
  if (!o) return;
  o += (static_cast<int64_t>(t) * c.hkv + h) * D;
  const int64_t row0 = paged_row(c, seq[t], pos[t]);
  const int64_t row = row0 + static_cast<int64_t>(h) * c.ps;
  const TC* x = static_cast<const TC*>(key ? c.k : c.v) + row * D;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    float y = 0.0f;
    if (row0 >= 0) {
      if constexpr (sizeof(TC) == 1)
        y = __fmul_rn(static_cast<float>(x[lane + 32 * i]), (key ? c.ks : c.vs)[row]);
      else
        y = to_f32(x[lane + 32 * i]);
    }
    o[lane + 32 * i] = from_f32<TO>(y);
  }
}

template <typename TI, typename TC>
cudaError_t append_launch(const AppendArgs& a, int d, cudaStream_t s) {
  const int64_t warps = static_cast<int64_t>(a.tokens) * ((a.q ? a.heads : 0) + 2 * a.c.hkv);
  const unsigned grid = static_cast<unsigned>((warps + 7) / 8);
  if (d == 64)
    append_kernel<TI, TC, 64><<<grid, 256, 0, s>>>(a);
  else
    append_kernel<TI, TC, 128><<<grid, 256, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename TI>
cudaError_t append_pool(const AppendArgs& a, int pool, int d, cudaStream_t s) {
  return pool == TL_I8     ? append_launch<TI, int8_t>(a, d, s)
         : pool == TL_BF16 ? append_launch<TI, __nv_bfloat16>(a, d, s)
                           : append_launch<TI, __half>(a, d, s);
}

template <typename TC, typename TO>
cudaError_t read_launch(const PagedView& c, const int32_t* seq, const int32_t* pos, int tokens, void* k, void* v, int d,
                        cudaStream_t s) {
  const int64_t warps = static_cast<int64_t>(tokens) * 2 * c.hkv;
  const unsigned grid = static_cast<unsigned>((warps + 7) / 8);
  if (d == 64)
    read_kernel<TC, TO, 64><<<grid, 256, 0, s>>>(c, seq, pos, tokens, static_cast<TO*>(k), static_cast<TO*>(v));
  else
    read_kernel<TC, TO, 128><<<grid, 256, 0, s>>>(c, seq, pos, tokens, static_cast<TO*>(k), static_cast<TO*>(v));
  return cudaGetLastError();
}
template <typename TC>
cudaError_t read_out(const PagedView& c, const int32_t* seq, const int32_t* pos, int tokens, void* k, void* v, int out,
                     int d, cudaStream_t s) {
  return out == TL_F32    ? read_launch<TC, float>(c, seq, pos, tokens, k, v, d, s)
         : out == TL_BF16 ? read_launch<TC, __nv_bfloat16>(c, seq, pos, tokens, k, v, d, s)
                          : read_launch<TC, __half>(c, seq, pos, tokens, k, v, d, s);
}

}  // namespace
}  // namespace tl

using namespace tl;

extern "C" {

tl_status tl_paged_append(const tl_paged_kv* cache, const void* q, const void* k, const void* v, int32_t dtype,
                          int64_t q_stride, int64_t k_stride, int64_t v_stride, const int32_t* seq,
                          const int32_t* pos, const int32_t* block_table, int32_t n_seqs, int32_t max_pages,
                          int64_t table_stride, const float* rope_cos, const float* rope_sin, int32_t max_positions,
                          int32_t tokens, int32_t heads, void* q_out, void* stream) {
  AppendArgs a;
  const tl_status st = paged_view(cache, block_table, n_seqs, max_pages, table_stride, &a.c);
  if (st != TL_OK) return st;
  if (!k || !v || !seq || !pos || !is_float_dtype(dtype) || tokens <= 0) return TL_ERR_INVALID_ARGUMENT;
  if (!rope_cos != !rope_sin || (rope_cos && max_positions <= 0)) return TL_ERR_INVALID_ARGUMENT;
  if (!q != !q_out || (q && (heads <= 0 || !rope_cos))) return TL_ERR_INVALID_ARGUMENT;
  const int64_t d = cache->head_dim, e = dtype_bytes(dtype), kv = cache->kv_heads;
  if (k_stride < kv * d || v_stride < kv * d || (q && q_stride < heads * d)) return TL_ERR_INVALID_ARGUMENT;
  if (!aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(q, 16) || !aligned_to(q_out, 16) ||
      (k_stride * e) % 16 || (v_stride * e) % 16 || (q && (q_stride * e) % 16) || !aligned_to(rope_cos, 16) ||
      !aligned_to(rope_sin, 16))
    return TL_ERR_INVALID_ARGUMENT;
  if (q == q_out && q && q_stride != heads * d) return TL_ERR_INVALID_ARGUMENT;
  a.q = q;
  a.k = k;
  a.v = v;
  a.ldq = q_stride;
  a.ldk = k_stride;
  a.ldv = v_stride;
  a.seq = seq;
  a.pos = pos;
  a.cos = rope_cos;
  a.sin = rope_sin;
  a.max_pos = max_positions;
  a.tokens = tokens;
  a.heads = q ? heads : 0;
  a.q_out = q_out;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return cuda_status(dtype == TL_F32    ? append_pool<float>(a, cache->dtype, cache->head_dim, s)
                     : dtype == TL_BF16 ? append_pool<__nv_bfloat16>(a, cache->dtype, cache->head_dim, s)
                                        : append_pool<__half>(a, cache->dtype, cache->head_dim, s));
}

tl_status tl_paged_read(const tl_paged_kv* cache, const int32_t* seq, const int32_t* pos, const int32_t* block_table,
                        int32_t n_seqs, int32_t max_pages, int64_t table_stride, int32_t tokens, void* k_out,
                        void* v_out, int32_t out_dtype, void* stream) {
  PagedView c;
  const tl_status st = paged_view(cache, block_table, n_seqs, max_pages, table_stride, &c);
  if (st != TL_OK) return st;
  if (!seq || !pos || tokens <= 0 || !is_float_dtype(out_dtype) || (!k_out && !v_out)) return TL_ERR_INVALID_ARGUMENT;
  if (!aligned_to(k_out, 16) || !aligned_to(v_out, 16)) return TL_ERR_INVALID_ARGUMENT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int d = cache->head_dim;
  return cuda_status(cache->dtype == TL_I8     ? read_out<int8_t>(c, seq, pos, tokens, k_out, v_out, out_dtype, d, s)
                     : cache->dtype == TL_BF16 ? read_out<__nv_bfloat16>(c, seq, pos, tokens, k_out, v_out, out_dtype, d, s)
                                               : read_out<__half>(c, seq, pos, tokens, k_out, v_out, out_dtype, d, s));
}

}  // extern "C"
