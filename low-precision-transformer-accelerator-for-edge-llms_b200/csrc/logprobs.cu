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
// sums (for long lists afresh in each of four parts of the row); the elements
// of a thread and part are a group. The k-th largest of the groups'
// maxima is no larger than the k-th largest element, so only groups whose
// maximum reaches it can hold one of the k, and only their elements (read
// again, from L2) are compared: the single pass over the row does no work for
// the list. Values are ordered with their index as one 64-bit key (equal
// values: the lower index is the larger key), which makes every choice below
// unique: the list does not depend on the order in which threads find it.
//
// What bounds it: reading the logits. A warp's tiles arrive by bulk copies a
// few tiles ahead. Few rows are split over the CTAs of a cluster, which join
// their sums and lists through distributed shared memory. Many rows go to
// persistent CTAs in which two warps put a row's results together (a chain of
// short steps that reads little) while the others sum the next row.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "kernels.cuh"
#include "serving.cuh"
#include "tc_common.cuh"

namespace tl {
namespace {

constexpr int kUnroll = 4;        // 16-byte pieces of a thread in a tile
constexpr int kTile = kUnroll * 32, kTileBytes = kTile * 16;  // pieces and bytes of a warp's tile
// Tiles of a warp under way, warps of a CTA that sum rows, that put results
// together, and such CTAs an SM holds. 2048 rows of 32000 float32 took 47.8 us
// with 2, 8, 2, 3 (now 50.9, 5.2 TB/s); with four tiles under way 54.9 (SMs
// drift apart: the rows are handed out beforehand), with one result warp 65.5,
// with two CTAs of 8 + 2 or 8 + 4 warps 50.9 and 51.2, and 52 to 57 where all
// warps of a CTA work on the results between rows.
constexpr int kStages = 2;
constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kPostWarps = 2;
constexpr int kRowCtas = 3;
constexpr int kCandidates = 512;
constexpr int kMaxCluster = 8;
constexpr int kParts = 4;
constexpr int kRing = kWarps * kStages * kTileBytes;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

using Key = unsigned long long;

// Set when a wait on a tile ran out (tl_device_error reads and clears it).
__device__ unsigned int g_logprob_error = 0;

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
TL_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two float32 operations in one instruction; a pair is 64 bits.
using Pair = unsigned long long;
TL_DEV Pair pair(float x, float y) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y));
  return p;
}
TL_DEV float2 halves(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
TL_DEV Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
TL_DEV Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
TL_DEV Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
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
// Joins the sums of the lanes of a warp.
TL_DEV Sums warp_join(Sums a) {
  const float m = warp_max(a.m);
  const float e = (a.m - m) * kLog2e, f = ex2(e);
  // a factor that underflows takes its (possibly infinite) exponent with it
  a.t = f > 0.0f ? f * (a.t + e * a.s) : 0.0f * a.s;
  a.s = f * a.s;
  return {m, warp_sum(a.s), warp_sum(a.t)};
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
  TL_DEV void clear() {  // minus infinity
    const uint32_t x = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __nv_bfloat16>::value ? 0xff80ff80u : 0xfc00fc00u;
    w = make_uint4(x, x, x, x);
  }
  TL_DEV void load_shared(const unsigned char* p) { w = *reinterpret_cast<const uint4*>(p); }
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
  float m = -FLT_MAX;              // the sums' reference
  Pair s = 0, t = 0;               // even and odd elements
  float best = -INFINITY;
  int at = 0;  // an index not below the largest element's

  // The reference is the largest element so far: that element's term is exactly 1, no y is above 0, and log p and H
  // of a row with one likely token, differences of numbers as small as themselves, keep their signs and digits.
  // (While it lagged by up to 20, both were off by 3e-6 there; 2048 rows of 32000 float32 took 49.7 us and take 50.9.)
  TL_DEV void follow(float top) {
    if (top > m) {
      const float e = (m - top) * kLog2e, f = ex2(e);
      const Pair f2 = pair(f, f);
      t = f > 0.0f ? mul2(f2, fma2(pair(e, e), s, t)) : 0;
      s = mul2(f2, s);
      m = top;
    }
  }
  // B batches of N elements, the last of batch b at index last + b * step.
  template <int B, int N>
  TL_DEV void add(const float (&x)[B][N], int last, int step) {
    float top[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      top[b] = N == 1 ? x[b][0] : fmaxf(x[b][0], x[b][N - 1]);
#pragma unroll
      for (int i = 1; i + 1 < N; i += 2) top[b] = max3(top[b], x[b][i], x[b][i + 1]);
    }
    float most = top[0];
#pragma unroll
    for (int b = 1; b < B; ++b) most = fmaxf(most, top[b]);
    if (most > best) {
      best = most;
      int first = B - 1;
#pragma unroll
      for (int b = B - 2; b >= 0; --b) first = top[b] == most ? b : first;
      at = last + first * step;
      follow(most);
    }
    const Pair mm = pair(-m, -m), log2e = pair(kLog2e, kLog2e);
    Pair s1 = 0, t1 = 0;
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        // (a single element pairs with -infinity)
        const Pair y = mul2(add2(pair(x[b][i], i + 1 < N ? x[b][i + 1 < N ? i + 1 : 0] : -INFINITY), mm), log2e);
        const float2 v = halves(y);
        const Pair e = pair(ex2(v.x), ex2(v.y));  // NaN and infinity stay in the sums and mark the row
        s1 = add2(s1, e);
        t1 = fma2(e, y, t1);
      }
    const float2 tt = halves(t1);
    if (!(tt.x + tt.y > -INFINITY)) {
      // 0 times -infinity among the terms (or a NaN that stays one): again, with y bounded
      t1 = 0;
#pragma unroll
      for (int b = 0; b < B; ++b)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float y = (x[b][i] - m) * kLog2e;
          t1 = add2(t1, pair(ex2(y) * fmaxf(y, -200.0f), 0.0f));
        }
    }
    s = add2(s, s1);
    t = add2(t, t1);
  }
  TL_DEV Sums sums() const {
    const float2 a = halves(s), b = halves(t);
    return {m, a.x + a.y, b.x + b.y};
  }
};

// What the summing warps leave of a row.
struct RowSums {
  Sums sums[kWarps];
  Key picks[TL_TOP_K_MAX + 2 * kWarps];  // of each warp with tiles, its lanes' largest maxima
  Key best[kParts][kThreads];            // every group's maximum
};
struct Shared {
  RowSums row[2];
  alignas(16) Key cand[kCandidates];
  Key list[TL_TOP_K_MAX];  // this CTA's largest, in order, then zeros
  Sums total;              // this CTA's sums
  int groups[kParts * kThreads];
  int n_groups, n_cand;
  Key reduce[kWarps];
  uint64_t tiles[kWarps * kStages], full[2], empty[2];  // barriers
};

// The CTA's share of a row. Whole 16-byte pieces are cut into tiles of kTile,
// which go to the warps of all CTAs in turn; lane l has pieces l, l + 32, ...
// of a tile. Elements before the first 16-byte boundary and after the last
// whole piece belong to the first threads of CTA 0.
template <typename T>
struct Share {
  static constexpr int N = Chunk<T>::N;
  const T* x;
  int vocab, head, chunks, ctas, rank, parts;
  TL_DEV int chunk_first(int i) const { return head + i * N; }
  TL_DEV int tiles() const { return (chunks + kTile - 1) / kTile; }
  TL_DEV int tile(int warp, int i) const { return rank * kWarps + warp + i * step(); }  // warp's i-th tile
  TL_DEV int step() const { return ctas * kWarps; }
  TL_DEV int turns() const { return (tiles() + step() - 1) / step(); }          // the most tiles of a warp
  TL_DEV int part_turns() const { return max(1, (turns() + parts - 1) / parts); }
  // the CTA's warps that have tiles (at least one: the loose elements' warp), and the maxima each picks, so that
  // together they pick k + 1 at least
  TL_DEV int busy() const { return max(1, min(kWarps, tiles() - rank * kWarps)); }
  TL_DEV int picks(int k) const { return min(32, (k + busy() - 1) / busy() + 1); }
  // the loose element of a thread, -1: none
  TL_DEV int loose(int thread) const {
    if (rank) return -1;
    const int i = thread < N ? thread : chunk_first(chunks) + thread - N;
    return thread < N ? (i < head ? i : -1) : i < vocab ? i : -1;
  }
};

// The threads that put results together: all of the CTA, or the last PT.
template <int PT>
struct Post {
  TL_DEV static int tid() { return PT == kThreads ? threadIdx.x : threadIdx.x - kThreads; }
  TL_DEV static void sync() {
    if constexpr (PT == kThreads)
      __syncthreads();
    else
      asm volatile("bar.sync 1, %0;" ::"n"(PT) : "memory");
  }
};

// A warp's part of what is left of a row; `most`: the lane's largest maximum.
template <typename T>
TL_DEV void leave(const Share<T>& w, const Running& run, Key most, int top_k, RowSums& row) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Sums sum = warp_join(run.sums());
  if (lane == 0) row.sums[warp] = sum;
  if (!top_k || warp >= w.busy()) return;
  const int picks = w.picks(top_k);
  for (int i = 0; i < picks; ++i) {
    const Key top = warp_max_key(most);
    if (most == top) most = 0;  // keys of two lanes differ unless both are empty
    if (lane == 0) row.picks[warp * picks + i] = top;
  }
}

// Writes the `k` largest keys of sh.cand[0..n) to sh.list in order (zeros
// behind): an element's place is the number of larger ones.
template <int PT>
TL_DEV void order_candidates(Shared& sh, int n, int k) {
  const int tid = Post<PT>::tid();
  if (tid < TL_TOP_K_MAX) sh.list[tid] = 0;
  Post<PT>::sync();
  for (int i = tid; i < n; i += PT) {
    const Key mine = sh.cand[i];
    int place = 0, j = 0;
#pragma unroll 4
    for (; j + 1 < n; j += 2) {
      const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(sh.cand + j);
      place += (two.x > mine) + (two.y > mine);
    }
    if (j < n) place += sh.cand[j] > mine;
    if (place < k) sh.list[place] = mine;
  }
  Post<PT>::sync();
}

// The k largest keys of the CTA's share -> sh.list.
template <typename T, int PT>
__device__ void top_of_share(const Share<T>& w, const RowSums& row, int k, Shared& sh) {
  constexpr int N = Chunk<T>::N, PW = PT / 32;
  const int tid = Post<PT>::tid(), lane = tid & 31, warp = tid >> 5;
  const int n_picks = w.busy() * w.picks(k);
  if (tid == 0) sh.n_groups = sh.n_cand = 0;
  // the k-th largest of the picks (0 if there are fewer)
  Key bar = ~0ull;
  for (int i = lane; i < n_picks; i += 32) {
    const Key p = row.picks[i];
    int above = 0;
    for (int j = 0; j < n_picks; ++j) above += row.picks[j] > p;
    if (above < k && p < bar) bar = p;
  }
  bar = ~warp_max_key(~bar);
  Post<PT>::sync();
  const int parts = (w.turns() + w.part_turns() - 1) / w.part_turns();
  for (int g = tid; g < max(1, parts) * kThreads; g += PT) {
    const Key best = row.best[g / kThreads][g % kThreads];
    if (best && best >= bar) sh.groups[atomicAdd(&sh.n_groups, 1)] = g;
  }
  Post<PT>::sync();
  const int n_groups = sh.n_groups;
  const float bar_value = bar ? key_value(bar) : -INFINITY;
  auto offer = [&](float v, int i) {
    if (!(v >= bar_value && v > -INFINITY)) return;
    const Key key = argmax_key(v + 0.0f, i);
    if (key < bar) return;
    const int at = atomicAdd(&sh.n_cand, 1);
    if (at < kCandidates) sh.cand[at] = key;
  };
  // the groups' pieces, spread over the threads, a few loads in flight
  const int per = w.part_turns() * kUnroll, pieces = n_groups * per;
  constexpr int F = PT == kThreads ? 1 : 4;
  for (int i0 = tid; i0 < pieces; i0 += PT * F) {
    Chunk<T> y[F];
    int c[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int i = i0 + f * PT;
      c[f] = w.chunks;
      if (i < pieces) {
        const int g = sh.groups[i / per], place = i % per, turn = g / kThreads * w.part_turns() + place / kUnroll;
        c[f] = w.tile(g % kThreads >> 5, turn) * kTile + place % kUnroll * 32 + (g & 31);
      }
      if (c[f] < w.chunks) y[f].load(w.x + w.chunk_first(c[f]));
    }
#pragma unroll
    for (int f = 0; f < F; ++f)
      if (c[f] < w.chunks) {
        float v[N];
        y[f].get(v);
#pragma unroll
        for (int e = 0; e < N; ++e) offer(v[e], w.chunk_first(c[f]) + e);
      }
  }
  // (the loose elements are few, and in groups of several parts: all are compared)
  if (tid < 2 * N)
    if (const int loose = w.loose(tid); loose >= 0) offer(to_f32(w.x[loose]), loose);
  Post<PT>::sync();
  const int n = sh.n_cand;
  if (n <= kCandidates) {
    order_candidates<PT>(sh, n, k);
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
    for (int g = tid; g < kThreads; g += PT) {
      for (int i = 0; w.tile(g >> 5, i) < w.tiles(); ++i)
        for (int u = 0; u < kUnroll; ++u) {
          const int c = w.tile(g >> 5, i) * kTile + u * 32 + (g & 31);
          if (c >= w.chunks) break;
          Chunk<T> y;
          float v[N];
          y.load(w.x + w.chunk_first(c));
          y.get(v);
#pragma unroll
          for (int e = 0; e < N; ++e) see(v[e], w.chunk_first(c) + e);
        }
      const int loose = w.loose(g);
      if (loose >= 0) see(to_f32(w.x[loose]), loose);
    }
    top = warp_max_key(top);
    Post<PT>::sync();
    if (lane == 0) sh.reduce[warp] = top;
    Post<PT>::sync();
    for (int i = 0; i < PW; ++i) top = sh.reduce[i] > top ? sh.reduce[i] : top;
    if (top == 0) break;
    if (tid == 0) sh.list[r] = top;
    last = top;
  }
  Post<PT>::sync();
}

TL_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
TL_DEV void cluster_wait_acquire() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
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

// One row's results from its sums and list.
TL_DEV void write_row(const LogprobArgs& a, int r, int tid, const Sums& sum, const Key* list, int token, float given) {
  const float nan = __int_as_float(0x7fc00000);
  const bool bad = !(sum.s < INFINITY), none = sum.s == 0.0f;
  const float ln_s = logf(sum.s);
  if (tid == 0) {
    if (a.tokens)
      a.logprob[r] = token < 0                    ? 0.0f
                     : bad || token >= a.vocab    ? nan
                     : none || given == -INFINITY ? -INFINITY
                                                  : (given - sum.m) - ln_s;
    if (a.entropy) a.entropy[r] = bad ? nan : none ? 0.0f : ln_s - kLn2 * (sum.t / sum.s);
  }
  if (tid < a.top_k) {
    const Key key = bad ? 0 : list[tid];
    const int64_t o = static_cast<int64_t>(r) * a.top_k + tid;
    a.top_ids[o] = key ? argmax_key_index(key) : -1;
    a.top_lp[o] = bad ? nan : key ? (key_value(key) - sum.m) - ln_s : -INFINITY;
  }
}

// CLUSTER: a row a cluster of `ctas` CTAs. Otherwise row blockIdx.x,
// + gridDim.x, ... a CTA.
template <typename T, bool CLUSTER>
__global__ void __launch_bounds__(CLUSTER ? kThreads : kThreads + kPostWarps * 32, CLUSTER ? 2 : kRowCtas)
    logprob_kernel(const __grid_constant__ LogprobArgs a, int ctas) {
  constexpr int N = Chunk<T>::N;
  extern __shared__ __align__(128) unsigned char rings[];
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first_row = CLUSTER ? blockIdx.x / ctas : blockIdx.x;
  const int row_step = CLUSTER ? gridDim.x / ctas : gridDim.x;
  auto share = [&](int r) {
    Share<T> w;
    w.x = static_cast<const T*>(a.x) + r * a.ld;
    w.vocab = a.vocab;
    w.head = min(a.vocab, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(w.x) & 15)) % 16 / sizeof(T)));
    w.chunks = (a.vocab - w.head) / N;
    w.ctas = CLUSTER ? ctas : 1;
    w.rank = CLUSTER ? blockIdx.x % ctas : 0;
    w.parts = a.top_k > 8 ? kParts : 1;
    return w;
  };
  bool late = false;  // a wait has run out: the results are void, the host learns of it
  auto wait = [&](uint64_t* bar, int parity, unsigned code) {
    if (mbar_try_wait(bar, parity)) return;  // (the clock is read only if there is something to wait for)
    if (late || !mbar_wait_err(bar, parity, code, &g_logprob_error)) late = true;
  };
  if (!CLUSTER && tid == 0)
    for (int i = 0; i < 2; ++i) {
      mbar_init(sh.full + i, kWarps);
      mbar_init(sh.empty + i, 1);
    }
  uint64_t* bars = sh.tiles + warp * kStages;
  if (warp < kWarps && lane == 0)
    for (int i = 0; i < kStages; ++i) mbar_init(bars + i, 1);
  if (lane == 0) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  if constexpr (CLUSTER)
    __syncwarp();
  else
    __syncthreads();
  pdl_begin();

  if (!CLUSTER && warp >= kWarps) {
    // ---- results, a row behind
    constexpr int PT = kPostWarps * 32;
    for (int r = first_row, n = 0; r < a.rows; r += row_step, ++n) {
      const Share<T> w = share(r);
      const int token = a.tokens ? a.tokens[r] : -1;
      const float given = token >= 0 && token < a.vocab ? to_f32(w.x[token]) : 0.0f;
      const RowSums& row = sh.row[n & 1];
      wait(sh.full + (n & 1), n >> 1 & 1, 3u);
      const Sums sum = warp_join(lane < kWarps ? row.sums[lane] : Sums{-FLT_MAX, 0.0f, 0.0f});
      if (a.top_k) top_of_share<T, PT>(w, row, a.top_k, sh);
      write_row(a, r, Post<PT>::tid(), sum, sh.list, token, given);
      Post<PT>::sync();  // the list and the row's sums have been read
      if (Post<PT>::tid() == 0) mbar_arrive(sh.empty + (n & 1));
    }
    return;
  }

  // ---- the warp's ring, filled kStages tiles ahead, also across rows
  unsigned char* ring = rings + warp * kStages * kTileBytes;
  // (addresses and sizes move by a constant from tile to tile)
  const int step_bytes = (CLUSTER ? ctas : 1) * kWarps * kTileBytes;
  int fill_row = first_row, fill_left = 0, filled = 0;  // bytes of the row from the next tile on
  const char* fill_at = nullptr;
  auto fill_start = [&]() {
    const Share<T> w = share(fill_row);
    const int first = w.tile(warp, 0) * kTile;
    fill_at = reinterpret_cast<const char*>(w.x + w.head) + first * 16ll;
    fill_left = (w.chunks - first) * 16;
  };
  auto fill = [&](int stage) {
    while (fill_left <= 0) {
      fill_row += row_step;
      if (fill_row >= a.rows) return;
      fill_start();
    }
    if (lane == 0) {
      const uint32_t bytes = min(fill_left, kTileBytes);
      mbar_arrive_expect_tx(bars + stage, bytes);
      bulk_load(ring + stage * kTileBytes, fill_at, bytes, bars + stage);
    }
    fill_at += step_bytes;
    fill_left -= step_bytes;
    ++filled;
  };
  fill_start();
  for (int i = 0; i < kStages; ++i)
    if (fill_row < a.rows) fill(i);

  int stage = 0, phase = 0;
  for (int r = first_row, n = 0; r < a.rows; r += row_step, ++n) {
    const Share<T> w = share(r);
    const int token = CLUSTER && a.tokens ? a.tokens[r] : -1;
    // In ascending order, so that a thread's `at` belongs to the first of equal
    // elements: then an element that beats the bar is in a group that does.
    Running run;
    Key most = 0;
    RowSums& left = sh.row[CLUSTER ? 0 : n & 1];
    if constexpr (!CLUSTER) wait(sh.empty + (n & 1), (n >> 1 & 1) ^ 1, 4u);
    auto end_part = [&](int part) {
      const Key key = run.best > -INFINITY ? argmax_key(run.best + 0.0f, run.at) : 0;
      left.best[part][tid] = key;
      most = key > most ? key : most;
      run.best = -INFINITY;
    };
    const int loose = w.loose(tid), part_turns = w.part_turns();
    const int parts = max(1, (w.turns() + part_turns - 1) / part_turns);
    if (loose >= 0 && loose < w.head) {
      const float v[1][1] = {{to_f32(w.x[loose])}};
      run.add(v, loose, 0);
    }
    // (two loops: the inner one holds nothing but the tile's work)
    int pieces = w.chunks - w.tile(warp, 0) * kTile;  // of the row, from the warp's next tile on
    int last = w.chunk_first(w.tile(warp, 0) * kTile + lane) + N - 1;  // last element of the lane's first piece
    const int step = w.step() * kTile;
#pragma unroll 1
    for (int part = 0; part < parts; ++part) {
#pragma unroll 1
      for (int i = 0; i < part_turns && pieces > 0; ++i) {
        wait(bars + stage, phase, 1u);
        Chunk<T> y[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) y[u].load_shared(ring + stage * kTileBytes + (u * 32 + lane) * 16);
        // Every lane's reads before the copy that refills the place: the copy belongs to the async proxy, which
        // __syncwarp alone does not order behind them (without the fence 38 of 20000 calls of 2048 rows met a
        // tile of the next elements; the time is the same).
        fence_proxy_async_smem();
        __syncwarp();
        if (fill_row < a.rows) fill(stage);
        if (pieces < kTile) {
#pragma unroll
          for (int u = 0; u < kUnroll; ++u)
            if (u * 32 + lane >= pieces) y[u].clear();
        }
        float v[kUnroll][N];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) y[u].get(v[u]);
        run.add(v, last, 32 * N);
        pieces -= step;
        last += step * N;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (part + 1 == parts && loose >= w.head) {
        const float v[1][1] = {{to_f32(w.x[loose])}};
        run.add(v, loose, 0);
      }
      if (a.top_k) end_part(part);
    }

    if constexpr (!CLUSTER) {
      leave(w, run, most, a.top_k, left);
      __syncwarp();
      if (lane == 0) mbar_arrive(sh.full + (n & 1));
    } else {
      const float given = token >= 0 && token < a.vocab ? to_f32(w.x[token]) : 0.0f;
      leave(w, run, most, a.top_k, left);
      __syncthreads();
      // (every warp joins the warps' sums; lanes beyond them bring nothing)
      Sums sum = warp_join(lane < kWarps ? sh.row[0].sums[lane] : Sums{-FLT_MAX, 0.0f, 0.0f});
      if (a.top_k) top_of_share<T, kThreads>(w, sh.row[0], a.top_k, sh);
      if (tid == 0) sh.total = sum;
      cluster_sync();
      if (w.rank == 0) {
        // peers' lists and sums in one round of remote loads
        const int m = ctas * a.top_k;  // at most 8 * 32
        if (tid < m) sh.cand[tid] = peer_key(sh.list + tid % a.top_k, tid / a.top_k);
        Sums part{-FLT_MAX, 0.0f, 0.0f};
        if (lane < ctas)
          part = {peer_float(&sh.total.m, lane), peer_float(&sh.total.s, lane), peer_float(&sh.total.t, lane)};
        sum = warp_join(part);
        __syncthreads();
      }
      cluster_arrive();  // no CTA goes on while its shared memory may be read
      if (w.rank == 0) {
        if (a.top_k) order_candidates<kThreads>(sh, ctas * a.top_k, a.top_k);
        write_row(a, r, tid, sum, sh.list, token, given);
      }
      cluster_wait_acquire();
    }
  }
  if (late)  // copies still under way must not land after the CTA has gone
    for (int i = max(0, filled - kStages); i < filled; ++i)
      mbar_wait_err(bars + i % kStages, i / kStages & 1, 2u, &g_logprob_error);
}

template <typename T>
tl_status logprob_launch(const LogprobArgs& a, cudaStream_t s) {
  static Once<64> ready;  // the rings need more shared memory than the default limit
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || !ready(dev, [] {
        return allow_shared(logprob_kernel<T, false>, kRing) && allow_shared(logprob_kernel<T, true>, kRing);
      }))
    return TL_ERR_CUDA;
  // A row's CTAs are doubled while the call has no more CTAs than there are SMs and
  // the row has a tile for every warp of twice as many, four warps aside. One row of
  // 32000 float32 over 1, 2, 4, 8 CTAs: 11.9, 8.7, 7.7, 7.7 us; 64 rows of 50021
  // bfloat16 over 1, 2, 4: 12.0, 9.1, 8.6.
  int ctas = 1;
  const int64_t tiles = static_cast<int64_t>(a.vocab) * sizeof(T) / kTileBytes;
  while (ctas < kMaxCluster && static_cast<int64_t>(a.rows) * ctas <= device_sm_count() &&
         tiles + kWarps / 2 >= ctas * 2 * kWarps)
    ctas *= 2;
  if (ctas == 1) {
    const int grid = std::min(a.rows, device_sm_count() * kRowCtas);
    return launch_serving(logprob_kernel<T, false>, grid, kThreads + kPostWarps * 32, kRing, 1, s, a, 1);
  }
  const unsigned grid = static_cast<unsigned>(a.rows) * ctas;
  return launch_serving(logprob_kernel<T, true>, grid, kThreads, kRing, ctas, s, a, ctas);
}

}  // namespace

cudaError_t logprob_read_error(unsigned int* code) {
  const cudaError_t e = cudaMemcpyFromSymbol(code, g_logprob_error, sizeof(unsigned int));
  if (e != cudaSuccess || !*code) return e;
  const unsigned int zero = 0;
  return cudaMemcpyToSymbol(g_logprob_error, &zero, sizeof(unsigned int));
}

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
  // bytes and elements of a row are counted in 31 bits, with room for every CTA's next tile behind its end
  constexpr int64_t kRowBytes = INT32_MAX - static_cast<int64_t>(kMaxCluster) * kWarps * kTileBytes;
  if (x.vocab > kRowBytes / dtype_bytes(x.dtype)) return TL_ERR_OUT_OF_RANGE;
  const LogprobArgs a{x.logits, x.row_stride, x.tokens,  x.rows,         x.vocab,
                      x.top_k,  x.logprob,    x.entropy, x.top_logprobs, x.top_ids};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return x.dtype == TL_F32    ? logprob_launch<float>(a, s)
         : x.dtype == TL_BF16 ? logprob_launch<__nv_bfloat16>(a, s)
                              : logprob_launch<__half>(a, s);
}
