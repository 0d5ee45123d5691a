// logprobs.cu -- log probabilities of given tokens, entropy and the most
// likely alternatives of rows of logits (tl_token_logprobs).
#include "serving.cuh"

namespace tl {
namespace {

struct LogprobArgs {
  const void* x;
  int64_t ld;
  const int32_t* tokens;
  int32_t rows, vocab, top_k;
  float *logprob, *entropy, *top_lp;
  int32_t* top_ids;
};

constexpr int kThreads = 256;

TL_DEV unsigned long long block_max_u64(unsigned long long v, unsigned long long* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int i = 0; i < kThreads / 32; ++i) v = sm[i] > v ? sm[i] : v;
  return v;
}
TL_DEV float block_sum(float v, float* sm) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int i = 0; i < kThreads / 32; ++i) v += sm[i];
  return v;
}

// One CTA per row: the maximum, the sums, then one pass per listed token.
template <typename T>
__global__ void logprob_kernel(LogprobArgs a) {
  __shared__ unsigned long long sm_k[kThreads / 32];
  __shared__ float sm_f[kThreads / 32];
  const int r = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + r * a.ld;
  unsigned long long best = 0;
  bool bad = false;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
    const float v = to_f32(x[i]);
    bad |= isnan(v) || v == INFINITY;
    const unsigned long long k = argmax_key(v + 0.0f, i);
    best = k > best ? k : best;
  }
  bad = __syncthreads_or(bad);
  best = block_max_u64(best, sm_k);
  const float nan = __int_as_float(0x7fc00000);
  const float top = to_f32(x[argmax_key_index(best)]);
  const bool none = top == -INFINITY;
  float s = 0.0f, t = 0.0f;
  if (!bad && !none)
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
      const float d = to_f32(x[i]) - top;
      const float e = expf(d);
      s += e;
      if (e > 0.0f) t += e * d;
    }
  s = block_sum(s, sm_f);
  t = block_sum(t, sm_f);
  const float log_s = logf(s);
  if (threadIdx.x == 0) {
    if (a.tokens) {
      const int id = a.tokens[r];
      float v = 0.0f;
      if (id >= 0) v = bad || id >= a.vocab ? nan : none ? -INFINITY : (to_f32(x[id]) - top) - log_s;
      a.logprob[r] = v;
    }
    if (a.entropy) a.entropy[r] = bad ? nan : none ? 0.0f : log_s - t / s;
  }
  unsigned long long prev = ~0ull;
  for (int k = 0; k < a.top_k; ++k) {
    best = 0;
    if (!bad)
      for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
        const float v = to_f32(x[i]);
        const unsigned long long key = argmax_key(v + 0.0f, i);
        if (v > -INFINITY && key < prev && key > best) best = key;
      }
    best = block_max_u64(best, sm_k);
    prev = best ? best : 1;
    if (threadIdx.x == 0) {
      const int64_t o = static_cast<int64_t>(r) * a.top_k + k;
      a.top_ids[o] = best ? argmax_key_index(best) : -1;
      a.top_lp[o] = bad ? nan : best ? (to_f32(x[argmax_key_index(best)]) - top) - log_s : -INFINITY;
    }
  }
}

}  // namespace
}  // namespace tl

using namespace tl;

extern "C" tl_status tl_token_logprobs(const void* logits, int32_t dtype, int64_t row_stride, const int32_t* tokens,
                                       int32_t rows, int32_t vocab, int32_t top_k, float* logprob, float* entropy,
                                       int32_t* top_ids, float* top_logprobs, void* stream) {
  if (!logits || !is_float_dtype(dtype) || rows <= 0 || vocab <= 0 || row_stride < vocab) return TL_ERR_INVALID_ARGUMENT;
  if (!aligned_to(logits, dtype_bytes(dtype)) || !tokens != !logprob) return TL_ERR_INVALID_ARGUMENT;
  if (top_k < 0 || (top_k > 0 && (!top_ids || !top_logprobs))) return TL_ERR_INVALID_ARGUMENT;
  if (!logprob && !entropy && !top_k) return TL_ERR_INVALID_ARGUMENT;
  if (top_k > TL_TOP_K_MAX) return TL_ERR_OUT_OF_RANGE;
  LogprobArgs a{logits, row_stride, tokens, rows, vocab, top_k, logprob, entropy, top_logprobs, top_ids};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == TL_F32)
    logprob_kernel<float><<<rows, kThreads, 0, s>>>(a);
  else if (dtype == TL_BF16)
    logprob_kernel<__nv_bfloat16><<<rows, kThreads, 0, s>>>(a);
  else
    logprob_kernel<__half><<<rows, kThreads, 0, s>>>(a);
  return cuda_status(cudaGetLastError());
}
