// paged_attn.cu -- attention of one new token per sequence over a paged KV
// cache (tl_paged_attn_decode).
#include "serving.cuh"

namespace tl {
namespace {

struct AttendArgs {
  PagedView c;
  const void* q;
  int64_t ldq;
  const int32_t *seq, *lengths;
  int32_t rows, heads;
  float scale;
  void* out;
  float* lse;
};

constexpr int kWarps = 4;

// One CTA per (row, query head); warp w takes positions w, w + 4, ...
template <typename TQ, typename TC, int D>
__global__ void attend_kernel(AttendArgs a) {
  __shared__ float sm_m[kWarps], sm_l[kWarps], sm_o[kWarps][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.x / a.heads, h = blockIdx.x % a.heads;
  const int kvh = h / (a.heads / a.c.hkv);
  const int s = a.seq ? a.seq[r] : r;
  int len = (s < 0 || s >= a.c.n_seqs) ? 0 : a.lengths[r];
  len = min(len, a.c.max_pages * a.c.ps);
  constexpr int N = D / 32;
  float q[N], o[N];
  const TQ* qp = static_cast<const TQ*>(a.q) + r * a.ldq + h * D;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = to_f32(qp[lane + 32 * i]) * a.scale;
    o[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int p = warp; p < len; p += kWarps) {
    const int64_t row0 = paged_row(a.c, s, p);
    if (row0 < 0) continue;
    const int64_t row = row0 + static_cast<int64_t>(kvh) * a.c.ps;
    const TC* kp = static_cast<const TC*>(a.c.k) + row * D;
    const TC* vp = static_cast<const TC*>(a.c.v) + row * D;
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) dot = fmaf(q[i], static_cast<float>(kp[lane + 32 * i]), dot);
    dot = warp_sum(dot);
    float vs = 1.0f;
    if constexpr (sizeof(TC) == 1) {
      dot *= a.c.ks[row];
      vs = a.c.vs[row];
    }
    const float mn = fmaxf(m, dot);
    const float f = m == -INFINITY ? 0.0f : expf(m - mn);
    const float e = expf(dot - mn);
    l = l * f + e;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * f + e * (static_cast<float>(vp[lane + 32 * i]) * vs);
    m = mn;
  }
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) sm_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  if (warp) return;
  float M = -INFINITY, L = 0.0f;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w]);
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.0f;
  for (int w = 0; w < kWarps; ++w) {
    const float f = sm_m[w] == -INFINITY ? 0.0f : expf(sm_m[w] - M);
    L += f * sm_l[w];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] += f * sm_o[w][lane + 32 * i];
  }
  const bool empty = M == -INFINITY;
  TQ* op = static_cast<TQ*>(a.out) + (static_cast<int64_t>(r) * a.heads + h) * D;
#pragma unroll
  for (int i = 0; i < N; ++i) op[lane + 32 * i] = from_f32<TQ>(empty ? 0.0f : o[i] / L);
  if (a.lse && lane == 0) a.lse[static_cast<int64_t>(r) * a.heads + h] = empty ? -INFINITY : M + logf(L);
}

template <typename TQ, typename TC>
cudaError_t attend_launch(const AttendArgs& a, int d, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(a.rows) * a.heads;
  if (d == 64)
    attend_kernel<TQ, TC, 64><<<grid, kWarps * 32, 0, s>>>(a);
  else
    attend_kernel<TQ, TC, 128><<<grid, kWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}
template <typename TQ>
cudaError_t attend_pool(const AttendArgs& a, int pool, int d, cudaStream_t s) {
  return pool == TL_I8     ? attend_launch<TQ, int8_t>(a, d, s)
         : pool == TL_BF16 ? attend_launch<TQ, __nv_bfloat16>(a, d, s)
                           : attend_launch<TQ, __half>(a, d, s);
}

}  // namespace
}  // namespace tl

using namespace tl;

extern "C" {

size_t tl_paged_attn_workspace_bytes(int32_t heads, int32_t kv_heads, int32_t head_dim) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
  return 16;
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
  a.seq = seq;
  a.lengths = lengths;
  a.rows = rows;
  a.heads = heads;
  a.scale = sm_scale;
  a.out = out;
  a.lse = lse;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return cuda_status(q_dtype == TL_F32    ? attend_pool<float>(a, cache->dtype, cache->head_dim, s)
                     : q_dtype == TL_BF16 ? attend_pool<__nv_bfloat16>(a, cache->dtype, cache->head_dim, s)
                                          : attend_pool<__half>(a, cache->dtype, cache->head_dim, s));
}

}  // extern "C"
