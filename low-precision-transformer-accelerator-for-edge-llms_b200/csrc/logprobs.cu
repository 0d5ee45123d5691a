// logprobs.cu -- log probabilities of given tokens, entropy and the most
// likely alternatives of rows of logits (tl_token_logprobs).
//
// Mathematics. With a reference m the row's sums are
//   s = sum 2^y_i,  t = sum 2^y_i y_i,  y_i = (x_i - m) log2 e,
// and then, in natural logarithms,
//   log p_i = (x_i - m) - ln s,   H = ln s - ln2 t / s.
// Sums over parts with their own references join as s = sum f s_i,
// t = sum f (t_i + e s_i) with e = (m_i - m) log2 e, f = 2^e.
//
// The k largest. Every thread remembers the largest of its elements while it
// sums; a thread's elements are a group. The k-th largest of the groups'
// maxima is no larger than the k-th largest element, so only groups whose
// maximum reaches it can hold one of the k, and only their elements (read
// again, from L2) are compared: the single pass over the row does no work for
// the list. Values are ordered with their index as one 64-bit key (equal
// values: the lower index is the larger key), which makes every choice below
// unique: the list does not depend on the order in which threads find it.
//
// What bounds it: reading the logits. Each thread has several 16-byte loads
// in flight, and a row is split over the CTAs of a cluster, which join their
// sums and lists through distributed shared memory, while rows are too few
// for the SMs.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "kernels.cuh"
#include "serving.cuh"
#include "tc_common.cuh"

namespace tl {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kUnroll = 4;      // 16-byte loads of a thread in flight
constexpr int kCandidates = 512;
constexpr int kMaxCluster = 8;
constexpr int kPicks = TL_TOP_K_MAX / kWarps + 1;  // largest maxima taken of a warp
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

using Key = unsigned long long;

struct LogprobArgs {
  const void* x;
  int64_t ld;
  const int32_t* tokens;
  int32_t rows, vocab, top_k;
  float *logprob, *entropy, *top_lp;
  int32_t* top_ids;
};

// The key's value: argmax_key (common.cuh) undone.
TL_DEV float key_value(Key k) {
  const unsigned b = static_cast<unsigned>(k >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

TL_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
TL_DEV unsigned redux_max(unsigned v) { return __reduce_max_sync(0xffffffffu, v); }
TL_DEV Key warp_max_key(Key k) {
  const unsigned hi = redux_max(static_cast<unsigned>(k >> 32));
  const unsigned lo = redux_max(static_cast<unsigned>(k >> 32) == hi ? static_cast<unsigned>(k) : 0u);
  return static_cast<Key>(hi) << 32 | lo;
}

// Sums of a part of a row, relative to reference m (finite).
struct Sums {
  float m, s, t;
};
TL_DEV Sums join(const Sums& a, const Sums& b) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float ea = (a.m - r.m) * kLog2e, eb = (b.m - r.m) * kLog2e;
  const float fa = ex2(ea), fb = ex2(eb);
  // a factor that underflows takes its (possibly infinite) exponent with it
  r.s = fa * a.s + fb * b.s;
  r.t = (fa > 0.0f ? fa * (a.t + ea * a.s) : 0.0f * a.s) + (fb > 0.0f ? fb * (b.t + eb * b.s) : 0.0f * b.s);
  return r;
}

template <typename T>
struct Chunk {
  static constexpr int N = 16 / sizeof(T);
  uint4 w;
  TL_DEV void load(const T* p) {
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                 : "l"(p));
  }
  TL_DEV void get(float* x) const {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        x[i] = __uint_as_float(v[i]);
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        x[2 * i] = __uint_as_float(v[i] << 16);
        x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(v + i));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
};

// A thread's running sums and its largest element.
struct Running {
  Sums a{-FLT_MAX, 0.0f, 0.0f};
  float best = -INFINITY;
  int at = 0;  // an index not below the largest element's

  template <int N>
  TL_DEV void add(const float* x, int last) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
    if (top > best) {
      best = top;
      at = last;
      // the reference follows only when sums would grow past 2^30 of it
      if (top > a.m + 20.0f) {
        const float e = (a.m - top) * kLog2e, f = ex2(e);
        a.t = f > 0.0f ? f * (a.t + e * a.s) : 0.0f;
        a.s *= f;
        a.m = top;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = (x[i] - a.m) * kLog2e;
      const float e = ex2(y);  // NaN and infinity stay in the sums and mark the row
      a.s += e;
      a.t = fmaf(e, fmaxf(y, -200.0f), a.t);  // 0 times a finite number for -infinity
    }
  }
};

struct Shared {
  Sums sums[kWarps];
  Key picks[kWarps * kPicks];
  Key cand[kCandidates];
  Key list[TL_TOP_K_MAX];  // this CTA's largest, in order, then zeros
  Sums row;                // this CTA's sums
  int groups[kThreads];
  int n_groups, n_cand;
  Key reduce[kWarps];
};

// The CTA's share of a row: elements before the first 16-byte boundary and
// after the last whole chunk belong to the threads of CTA 0, chunks to CTA
// (i / kThreads) % ctas.
template <typename T>
struct Share {
  const T* x;
  int vocab, head, chunks, ctas, rank;
  TL_DEV int chunk_first(int i) const { return head + i * Chunk<T>::N; }
  TL_DEV int first_of(int thread) const { return rank * kThreads + thread; }
  TL_DEV int stride() const { return ctas * kThreads; }
  // the loose element of a thread, -1: none
  TL_DEV int loose(int thread) const {
    if (rank) return -1;
    const int i = thread < Chunk<T>::N ? thread : chunk_first(chunks) + thread - Chunk<T>::N;
    return thread < Chunk<T>::N ? (i < head ? i : -1) : i < vocab ? i : -1;
  }
};

// Writes the `k` largest keys of sh.cand[0..n) to sh.list in order (zeros
// behind): an element's place is the number of larger ones.
TL_DEV void order_candidates(Shared& sh, int n, int k) {
  if (threadIdx.x < TL_TOP_K_MAX) sh.list[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const Key mine = sh.cand[i];
    int place = 0;
    for (int j = 0; j < n; ++j) place += sh.cand[j] > mine;
    if (place < k) sh.list[place] = mine;
  }
  __syncthreads();
}

// The k largest keys of the CTA's share -> sh.list.
template <typename T>
__device__ void top_of_share(const Share<T>& w, const Running& run, int k, Shared& sh) {
  constexpr int N = Chunk<T>::N;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int picks = (k + kWarps - 1) / kWarps + 1;
  const Key mine = run.best > -INFINITY ? argmax_key(run.best + 0.0f, run.at) : 0;
  if (tid == 0) sh.n_groups = sh.n_cand = 0;
  {
    Key left = mine;
    for (int i = 0; i < picks; ++i) {
      const Key top = warp_max_key(left);
      if (left == top) left = 0;  // keys of two lanes differ unless both are empty
      if (lane == 0) sh.picks[warp * picks + i] = top;
    }
  }
  __syncthreads();
  // the k-th largest of the picks (0 if there are fewer)
  Key bar = ~0ull;
  for (int i = lane; i < kWarps * picks; i += 32) {
    const Key p = sh.picks[i];
    int above = 0;
    for (int j = 0; j < kWarps * picks; ++j) above += sh.picks[j] > p;
    if (above < k && p < bar) bar = p;
  }
  bar = ~warp_max_key(~bar);
  if (mine && mine >= bar) sh.groups[atomicAdd(&sh.n_groups, 1)] = tid;
  __syncthreads();
  const int n_groups = sh.n_groups;
  auto offer = [&](float v, int i) {
    if (!(v > -INFINITY)) return;
    const Key key = argmax_key(v + 0.0f, i);
    if (key < bar) return;
    const int at = atomicAdd(&sh.n_cand, 1);
    if (at < kCandidates) sh.cand[at] = key;
  };
  for (int gi = warp; gi < n_groups; gi += kWarps) {
    const int g = sh.groups[gi];
    for (int c = w.first_of(g) + lane * w.stride(); c < w.chunks; c += 32 * w.stride()) {
      Chunk<T> y;
      float v[N];
      y.load(w.x + w.chunk_first(c));
      y.get(v);
#pragma unroll
      for (int i = 0; i < N; ++i) offer(v[i], w.chunk_first(c) + i);
    }
    const int loose = w.loose(g);
    if (lane == 0 && loose >= 0) offer(to_f32(w.x[loose]), loose);
  }
  __syncthreads();
  const int n = sh.n_cand;
  if (n <= kCandidates) {
    order_candidates(sh, n, k);
    return;
  }
  // A few groups hold more large elements than there is room for: take the
  // largest one at a time.
  if (tid < TL_TOP_K_MAX) sh.list[tid] = 0;
  Key last = ~0ull;
  for (int r = 0; r < k; ++r) {
    Key top = 0;
    auto see = [&](float v, int i) {
      const Key key = v > -INFINITY ? argmax_key(v + 0.0f, i) : 0;
      if (key < last && key > top) top = key;
    };
    for (int c = w.first_of(tid); c < w.chunks; c += w.stride()) {
      Chunk<T> y;
      float v[N];
      y.load(w.x + w.chunk_first(c));
      y.get(v);
#pragma unroll
      for (int i = 0; i < N; ++i) see(v[i], w.chunk_first(c) + i);
    }
    const int loose = w.loose(tid);
    if (loose >= 0) see(to_f32(w.x[loose]), loose);
    top = warp_max_key(top);
    __syncthreads();
    if (lane == 0) sh.reduce[warp] = top;
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) top = sh.reduce[i] > top ? sh.reduce[i] : top;
    if (top == 0) break;
    if (tid == 0) sh.list[r] = top;
    last = top;
  }
  __syncthreads();
}

TL_DEV uint32_t peer_address(const void* p, unsigned rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
TL_DEV float peer_float(const float* p, unsigned rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer_address(p, rank)) : "memory");
  return v;
}
TL_DEV Key peer_key(const Key* p, unsigned rank) {
  Key v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer_address(p, rank)) : "memory");
  return v;
}

template <typename T, bool CLUSTER>
__global__ void __launch_bounds__(kThreads) logprob_kernel(const __grid_constant__ LogprobArgs a, int ctas) {
  constexpr int N = Chunk<T>::N;
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = CLUSTER ? blockIdx.x / ctas : blockIdx.x;
  Share<T> w;
  w.x = static_cast<const T*>(a.x) + r * a.ld;
  w.vocab = a.vocab;
  w.head = min(a.vocab, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(w.x) & 15)) % 16 / sizeof(T)));
  w.chunks = (a.vocab - w.head) / N;
  w.ctas = CLUSTER ? ctas : 1;
  w.rank = CLUSTER ? blockIdx.x % ctas : 0;

  // the given token's logit, long before it is needed
  int token = -1;
  float given = 0.0f;
  if (tid == 0 && w.rank == 0 && a.tokens) {
    token = a.tokens[r];
    if (token >= 0 && token < a.vocab) given = to_f32(w.x[token]);
  }

  // ---- one pass
  // In ascending order, so that a thread's `at` belongs to the first of equal
  // elements: then an element that beats the bar is in a group that does.
  Running run;
  const int loose = w.loose(tid);
  if (loose >= 0 && loose < w.head) {
    const float v = to_f32(w.x[loose]);
    run.add<1>(&v, loose);
  }
  int c = w.first_of(tid);
  const int stride = w.stride();
  for (; c + (kUnroll - 1) * stride < w.chunks; c += kUnroll * stride) {
    Chunk<T> y[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) y[u].load(w.x + w.chunk_first(c + u * stride));
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float v[N];
      y[u].get(v);
      run.add<N>(v, w.chunk_first(c + u * stride) + N - 1);
    }
  }
  for (; c < w.chunks; c += stride) {
    Chunk<T> y;
    float v[N];
    y.load(w.x + w.chunk_first(c));
    y.get(v);
    run.add<N>(v, w.chunk_first(c) + N - 1);
  }
  if (loose >= w.head) {
    const float v = to_f32(w.x[loose]);
    run.add<1>(&v, loose);
  }

  // ---- the CTA's sums
  Sums sum = run.a;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Sums other{__shfl_xor_sync(0xffffffffu, sum.m, o), __shfl_xor_sync(0xffffffffu, sum.s, o),
                     __shfl_xor_sync(0xffffffffu, sum.t, o)};
    sum = join(sum, other);
  }
  if (lane == 0) sh.sums[warp] = sum;
  __syncthreads();
  sum = sh.sums[0];
  for (int i = 1; i < kWarps; ++i) sum = join(sum, sh.sums[i]);
  if (a.top_k) top_of_share(w, run, a.top_k, sh);

  if constexpr (CLUSTER) {
    if (tid == 0) sh.row = sum;
    cluster_sync();
    if (w.rank == 0) {
      for (int p = 1; p < ctas; ++p)
        sum = join(sum, Sums{peer_float(&sh.row.m, p), peer_float(&sh.row.s, p), peer_float(&sh.row.t, p)});
      if (a.top_k) {
        const int n = ctas * a.top_k;  // at most 8 * 32
        for (int i = tid; i < n; i += kThreads) sh.cand[i] = peer_key(sh.list + i % a.top_k, i / a.top_k);
        __syncthreads();
        order_candidates(sh, n, a.top_k);
      }
    }
    cluster_sync();  // no CTA leaves while its shared memory may be read
    if (w.rank) return;
  }

  // ---- the row's results
  const float nan = __int_as_float(0x7fc00000);
  const bool bad = !(sum.s < INFINITY), none = sum.s == 0.0f;
  const float ln_s = logf(sum.s);
  if (tid == 0) {
    if (a.tokens)
      a.logprob[r] = token < 0                        ? 0.0f
                     : bad || token >= a.vocab        ? nan
                     : none || given == -INFINITY     ? -INFINITY
                                                      : (given - sum.m) - ln_s;
    if (a.entropy) a.entropy[r] = bad ? nan : none ? 0.0f : ln_s - kLn2 * (sum.t / sum.s);
  }
  if (tid < a.top_k) {
    const Key key = bad ? 0 : sh.list[tid];
    const int64_t o = static_cast<int64_t>(r) * a.top_k + tid;
    a.top_ids[o] = key ? argmax_key_index(key) : -1;
    a.top_lp[o] = bad ? nan : key ? (key_value(key) - sum.m) - ln_s : -INFINITY;
  }
}

template <typename T>
tl_status logprob_launch(const LogprobArgs& a, cudaStream_t s) {
  // A row is split over a cluster while CTAs of whole rows would leave SMs
  // without work, down to one round of loads a thread.
  int ctas = 1;
  const int64_t rounds = (static_cast<int64_t>(a.vocab) * sizeof(T) / 16 + kThreads - 1) / kThreads;
  while (ctas < kMaxCluster && static_cast<int64_t>(a.rows) * ctas * 2 <= device_sm_count() * 4 && rounds > ctas * 2)
    ctas *= 2;
  if (ctas == 1) {
    logprob_kernel<T, false><<<a.rows, kThreads, 0, s>>>(a, 1);
    return cuda_status(cudaGetLastError());
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, logprob_kernel<T, true>, a, ctas));
}

}  // namespace
}  // namespace tl

using namespace tl;

extern "C" tl_status tl_token_logprobs(const tl_token_logprobs_args* args, void* stream) {
  if (!args) return TL_ERR_INVALID_ARGUMENT;
  const tl_token_logprobs_args& x = *args;
  if (!x.logits || !is_float_dtype(x.dtype) || x.rows <= 0 || x.vocab <= 0 || x.row_stride < x.vocab)
    return TL_ERR_INVALID_ARGUMENT;
  if (!aligned_to(x.logits, dtype_bytes(x.dtype)) || !x.tokens != !x.logprob) return TL_ERR_INVALID_ARGUMENT;
  if (x.top_k < 0 || (x.top_k > 0 && (!x.top_ids || !x.top_logprobs))) return TL_ERR_INVALID_ARGUMENT;
  if (!x.logprob && !x.entropy && !x.top_k) return TL_ERR_INVALID_ARGUMENT;
  if (x.top_k > TL_TOP_K_MAX) return TL_ERR_OUT_OF_RANGE;
  const LogprobArgs a{x.logits, x.row_stride, x.tokens,  x.rows,         x.vocab,
                      x.top_k,  x.logprob,    x.entropy, x.top_logprobs, x.top_ids};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return x.dtype == TL_F32    ? logprob_launch<float>(a, s)
         : x.dtype == TL_BF16 ? logprob_launch<__nv_bfloat16>(a, s)
                              : logprob_launch<__half>(a, s);
}
