// Log probabilities of given tokens with entropy and top alternatives, and their gradient.
//
//   logprob = (x_t - m) - log S,  H = -sum_j p_j log p_j = log S - T / S
//   with m = max x_j, S = sum e^{x_j - m}, T = sum e^{x_j - m} (x_j - m)  (T <= 0: no cancellation)
//   (not x_t - (m + log S), which would round log S at the size of the logits)
//   top k: largest logits, the lowest index first among equal ones
//   dx_j = [j = t] g + sum_i [j = top_i] h_i - p_j (g + sum h + gH (log p_j + H))
// A row without a logit above -inf has S = 0 (any other has S >= 1) and no distribution; a NaN or +inf makes S NaN.
//
// Both directions are bound by reading (and writing) the logits once.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"

namespace mykb {
namespace lp {

constexpr int THREADS = 256;   // of the gradient kernel
constexpr int UN = 4;          // 16-byte vectors a thread of it loads at a time
constexpr int kMaxTop = 32;
constexpr int kCand = 1024;    // candidates kept for the top alternatives
constexpr int kStepMax = 4096;  // maxima of loop steps that a CTA remembers
constexpr float kLog2e = 1.4426950408889634f;

template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void get(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(u[i] << 16), x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
  __device__ static float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  __device__ static __nv_bfloat16 cast(float x) { return __float2bfloat16(x); }
  __device__ static uint4 put(const float (&x)[8]) {
    return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
  static constexpr uint32_t kNegInf = 0xff80ff80u;
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  __device__ static void get(const uint4& w, float (&x)[4]) {
    x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
  }
  __device__ static float load(const float* p) { return *p; }
  __device__ static float cast(float x) { return x; }
  __device__ static uint4 put(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
  static constexpr uint32_t kNegInf = 0xff800000u;
};

// Running maximum, sum and first moment of a softmax.
struct Stat {
  float m, s, t;
};
__device__ __forceinline__ float ref_of(float m) { return m == -INFINITY ? 0.f : m; }
// m less the reference r >= m, kept finite for m = -inf, as e^-1000 is 0 already.  inf - inf stays NaN (a maximum
// with -1000 would drop it), so a +inf among the logits shows in the sums wherever it lies in the row.
__device__ __forceinline__ float shift_of(float m, float r) {
  const float d = m - r;
  return d < -1000.f ? -1000.f : d;
}
__device__ __forceinline__ Stat join(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m), r = ref_of(m);
  const float da = shift_of(a.m, r), db = shift_of(b.m, r);  // an empty side has s = t = 0 and m = -inf
  const float ea = exp2f(da * kLog2e), eb = exp2f(db * kLog2e);
  return {m, a.s * ea + b.s * eb, ea * (a.t + a.s * da) + eb * (b.t + b.s * db)};
}

// Order-preserving key of a logit, never 0: -0 counts as 0 and NaN as -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
  x = x != x ? -INFINITY : x + 0.f;
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

template <typename T>
struct FwdParams {
  const T* x;
  int64_t stride;  // elements between rows
  const int64_t* tokens;
  int64_t ignore;
  float *logprob, *entropy, *top_lp;
  float* stats;  // (3, rows) for the gradient: m, log S, entropy
  int64_t* top_tok;
  int64_t rows;
  int V, top;
};

// Descending sort of one 32-bit key a lane.
__device__ __forceinline__ uint32_t sort_step(uint32_t v, int lane, int j, bool desc) {
  const uint32_t o = __shfl_xor_sync(0xffffffffu, v, j);
  const bool low = (lane & j) == 0;
  return (low == desc) ? max(v, o) : min(v, o);
}
__device__ __forceinline__ uint32_t warp_sort(uint32_t v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) v = sort_step(v, lane, j, (lane & k) == 0);
  return v;
}
__device__ __forceinline__ uint32_t warp_merge(uint32_t v, int lane) {  // of a bitonic sequence
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) v = sort_step(v, lane, j, true);
  return v;
}

// One CTA a row, one pass over it: 4096 rows of 65536 bf16 logits with 5 alternatives take 127 us
// (0.64 of the copy bandwidth; two vectors a thread ahead and five CTAs an SM were the best of the
// depths and occupancies tried, 127 to 208 us).  Bound by latency: loads stop at the joins and the
// ranking at every row's end (long scoreboard and barrier are the stalls; no pipe is above 40 percent,
// the one of the exponentials at 39).  The row's top k are found from the threads' own maxima: the
// k-th largest of those is at most the k-th largest logit, so only the few elements that reach
// it are candidates; threads that have one read those steps of theirs again (from L2), and the
// candidates are ranked by counting.  Rows with so many equal logits that the candidates do not
// fit (a mask of -inf over most of the vocabulary) take the larger ones and then the first
// equal ones in order.
template <typename T, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 5 : 1) fwd_kernel(FwdParams<T> p) {
  constexpr int UN = THREADS == 256 ? 2 : 4;  // vectors a thread loads at a time
  constexpr int N = Vec<T>::N, WARPS = THREADS / 32, kSteps = kStepMax / THREADS;
  const int64_t row = blockIdx.x;
  const T* x = p.x + row * p.stride;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int V = p.V;
  const int head = min(V, (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)));
  const int nvec = (V - head) / N, tail0 = head + nvec * N;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  __shared__ Stat red[WARPS];
  __shared__ float step_max[TOP ? kSteps : 1][THREADS];
  Stat a{-INFINITY, 0.f, 0.f};
  float mine = -INFINITY;  // this thread's largest logit (NaN skipped)
  auto one = [&](float v) {
    const float e = v == -INFINITY ? 0.f : 1.f;
    mine = fmaxf(mine, v);
    a = join(a, {v != v ? 0.f : v, v != v ? v : e, 0.f});
  };
  if (tid < head) one(Vec<T>::load(x + tid));
  const int steps = (nvec + THREADS * UN - 1) / (THREADS * UN);
  const uint4 fill = make_uint4(Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf);
  // the vectors of the next step are loaded while those of this one are summed
  uint4 next[UN];
  auto load = [&](int st) {
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int i = (st * UN + u) * THREADS + tid;
      next[u] = i < nvec ? __ldg(xv + i) : fill;
    }
  };
  load(0);
  for (int st = 0; st < steps; ++st) {
    uint4 w[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) w[u] = next[u];
    if (st + 1 < steps) load(st + 1);
    float v[UN][N], mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      Vec<T>::get(w[u], v[u]);
#pragma unroll
      for (int i = 0; i < N; i += 2) mx = fmax3(mx, v[u][i], v[u][i + 1]);
    }
    if (TOP && st < kSteps) step_max[st][tid] = mx;
    mine = fmaxf(mine, mx);
    const float m = fmaxf(a.m, mx), r = ref_of(m);
    const float d = shift_of(a.m, r), c = exp2f(d * kLog2e);
    float2 s2 = make_float2(a.s * c, 0.f), t2 = make_float2(c * (a.t + a.s * d), 0.f);
    const float2 neg = make_float2(-r, -r), l2 = make_float2(kLog2e, kLog2e);
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float2 z = fadd2(make_float2(v[u][i], v[u][i + 1]), neg);
        const float2 y = fmul2(z, l2);
        const float2 e = make_float2(exp2f(y.x), exp2f(y.y));
        s2 = fadd2(s2, e);
        t2 = ffma2(e, make_float2(fmaxf(z.x, -1000.f), fmaxf(z.y, -1000.f)), t2);  // 0 * -inf is 0
      }
    a = {m, s2.x + s2.y, t2.x + t2.y};
  }
  if (tail0 + tid < V) one(Vec<T>::load(x + tail0 + tid));
  {
    Stat w = a;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      w = join(w, {__shfl_xor_sync(0xffffffffu, w.m, o), __shfl_xor_sync(0xffffffffu, w.s, o),
                   __shfl_xor_sync(0xffffffffu, w.t, o)});
    if (lane == 0) red[warp] = w;
  }
  __syncthreads();
  Stat all = red[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) all = join(all, red[w]);
  const float logs = __logf(all.s);  // -inf for a row without a distribution
  if (tid == 0) {
    const int64_t t = p.tokens[row];
    float out = 0.f;
    if (t != p.ignore) {
      if (t < 0 || t >= V) out = __int_as_float(0x7fffffff);  // not a token of this vocabulary: NaN
      else out = all.s == 0.f ? -INFINITY : (Vec<T>::load(x + t) - all.m) - logs;
    }
    p.logprob[row] = out;
    const float entropy = all.s == 0.f ? 0.f : logs - all.t / all.s;
    p.entropy[row] = entropy;
    p.stats[row] = all.m, p.stats[p.rows + row] = logs, p.stats[2 * p.rows + row] = entropy;
  }
  if constexpr (TOP) {
    __shared__ uint32_t lists[WARPS][32];
    __shared__ uint32_t s_bound;
    __shared__ int s_n, s_eq;
    __shared__ uint64_t cand[kCand];
    const int k = p.top;
    // ---- bound: the k-th largest of the threads' maxima (0 where fewer threads have elements)
    const bool has = tid < head || tid < nvec || tail0 + tid < V;
    uint32_t key = warp_sort(has ? key_of(mine) : 0u, lane);
    lists[warp][lane] = key;
    if (tid == 0) s_n = 0, s_eq = 0;
    __syncthreads();
#pragma unroll
    for (int n = WARPS / 2; n > 0; n >>= 1) {
      if (warp < n) {
        key = warp_merge(max(key, lists[warp + n][31 - lane]), lane);
        lists[warp][lane] = key;
      }
      __syncthreads();
    }
    if (warp == 0 && lane == k - 1) s_bound = key;
    __syncthreads();
    const uint32_t bound = s_bound;
    // ---- candidates
    auto put = [&](float v, int idx) {
      const uint32_t kk = key_of(v);
      if (kk < bound) return;
      const int at = atomicAdd(&s_n, 1);
      if (at < kCand) cand[at] = ((uint64_t)kk << 32) | (uint32_t)~idx;
    };
    auto rescan = [&](auto&& f) {
      if (tid < head) f(Vec<T>::load(x + tid), tid);
      for (int st = 0; st < steps; ++st) {
        if (st < kSteps && key_of(step_max[st][tid]) < bound) continue;
#pragma unroll 1
        for (int u = 0; u < UN; ++u) {
          const int i = (st * UN + u) * THREADS + tid;
          if (i >= nvec) break;
          float v[N];
          Vec<T>::get(__ldg(xv + i), v);
#pragma unroll
          for (int j = 0; j < N; ++j) f(v[j], head + i * N + j);
        }
      }
      if (tail0 + tid < V) f(Vec<T>::load(x + tail0 + tid), tail0 + tid);
    };
    if (has && key_of(mine) >= bound) rescan(put);
    __syncthreads();
    int n = s_n;
    if (n > kCand) {  // (uniform) too many equal logits: the larger ones, then the first equal ones
      __syncthreads();
      if (tid == 0) s_n = 0;
      __syncthreads();
      if (has && key_of(mine) > bound)
        rescan([&](float v, int idx) {
          const uint32_t kk = key_of(v);
          if (kk <= bound) return;
          const int at = atomicAdd(&s_n, 1);
          if (at < kCand) cand[at] = ((uint64_t)kk << 32) | (uint32_t)~idx;
        });
      __syncthreads();
      const int above = s_n;
      if (above <= kCand) {
        // in index order, THREADS logits a turn, until k in all are found
        for (int i0 = 0; i0 < V; i0 += THREADS) {
          const int i = i0 + tid;
          const bool eq = i < V && key_of(Vec<T>::load(x + i)) == bound;
          const uint32_t bal = __ballot_sync(0xffffffffu, eq);
          if (lane == 0) lists[0][warp] = __popc(bal);
          __syncthreads();
          int before = above + s_eq;
          for (int w = 0; w < warp; ++w) before += lists[0][w];
          const int at = before + __popc(bal & ((1u << lane) - 1));
          if (eq && at < kCand) cand[at] = ((uint64_t)bound << 32) | (uint32_t)~i;
          __syncthreads();
          if (tid == 0)
            for (int w = 0; w < WARPS; ++w) s_eq += lists[0][w];
          __syncthreads();
          if (above + s_eq >= k) break;
        }
        n = min(above + s_eq, kCand);
      } else {  // the large logits lie in a few threads' columns: one pass for each alternative
        __shared__ uint64_t best[WARPS];
        uint64_t prev = ~0ull;
        for (int r = 0; r < k; ++r) {
          uint64_t c = 0;
          rescan([&](float v, int idx) {
            const uint64_t kk = ((uint64_t)key_of(v) << 32) | (uint32_t)~idx;
            if (kk < prev && kk > c) c = kk;
          });
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            const uint64_t y = __shfl_xor_sync(0xffffffffu, c, o);
            c = y > c ? y : c;
          }
          __syncthreads();
          if (lane == 0) best[warp] = c;
          __syncthreads();
          for (int w = 0; w < WARPS; ++w) c = best[w] > c ? best[w] : c;
          prev = c;
          if (tid == 0) cand[r] = c;
        }
        __syncthreads();
        n = k;
      }
    }
    // ---- rank by counting
    for (int i = tid; i < n; i += THREADS) {
      const uint64_t c = cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += cand[j] > c;
      if (rank < k) {
        p.top_lp[row * k + rank] = all.s == 0.f ? -INFINITY : (value_of((uint32_t)(c >> 32)) - all.m) - logs;
        p.top_tok[row * k + rank] = (int64_t)(uint32_t)~(uint32_t)c;
      }
    }
  }
}

template <typename T>
struct BwdParams {
  const T* x;
  T* dx;  // contiguous
  int64_t stride;
  const int64_t* tokens;
  int64_t ignore;
  const float* stats;  // (3, rows): m, log S, entropy
  const float *g_lp, *g_ent, *g_top;  // any may be null
  const int64_t* top_tok;
  int64_t rows;
  int V, top, chunk, chunks;
};

// One CTA per (row, run of `chunk` logits), bound by HBM (4095 rows of 32768 bf16 logits: 88 us for
// 537 MB, 0.93 of the copy bandwidth; rows that are not 16-byte aligned go element by element): the dense part, then the given and top tokens of the
// run are written again with their own terms.
template <typename T>
__global__ void __launch_bounds__(THREADS) bwd_kernel(BwdParams<T> p) {
  constexpr int N = Vec<T>::N;
  const int64_t row = blockIdx.x / p.chunks;
  const int lo = (int)(blockIdx.x % p.chunks) * p.chunk, hi = min(p.V, lo + p.chunk);
  const int tid = threadIdx.x;
  const T* x = p.x + row * p.stride;
  T* dx = p.dx + row * p.V;
  const int64_t t = p.tokens[row];
  const bool empty = p.stats[p.rows + row] == -INFINITY;  // no distribution: no gradient
  const bool given = p.g_lp && t != p.ignore && t >= 0 && t < p.V && !empty;
  const float gl = given ? p.g_lp[row] : 0.f, gh = p.g_ent && !empty ? p.g_ent[row] : 0.f;
  float A = gl;
  if (p.g_top && !empty)
    for (int i = 0; i < p.top; ++i) A += p.g_top[row * p.top + i];
  const float m = empty ? 0.f : p.stats[row], logs = empty ? 0.f : p.stats[p.rows + row];
  A = fmaf(gh, p.stats[2 * p.rows + row], A);  // g = -p (A + gh log p)
  const float nA = -A, ngh = -gh;
  auto dense = [&](float v) {
    const float z = (v - m) - logs;
    float e, g;  // without flushing: a subnormal p may meet a large factor
    asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(z * kLog2e));
    asm("mul.rn.f32 %0, %1, %2;" : "=f"(g) : "f"(e), "f"(fmaf(ngh, fmaxf(z, -1000.f), nA)));
    return g;
  };
  const bool vec = (((uintptr_t)x | (uintptr_t)dx) & 15) == 0 && p.chunk % N == 0;
  if (vec) {
    const int nv = (hi - lo) / N;
    const uint4* xv = reinterpret_cast<const uint4*>(x + lo);
    uint4* dv = reinterpret_cast<uint4*>(dx + lo);
    for (int i0 = tid; i0 < nv; i0 += THREADS * UN) {
      uint4 w[UN];
#pragma unroll
      for (int u = 0; u < UN; ++u)
        if (i0 + u * THREADS < nv) w[u] = __ldcs(xv + i0 + u * THREADS);
#pragma unroll
      for (int u = 0; u < UN; ++u)
        if (i0 + u * THREADS < nv) {
          float v[N];
          Vec<T>::get(w[u], v);
#pragma unroll
          for (int j = 0; j < N; ++j) v[j] = dense(v[j]);
          __stcs(dv + i0 + u * THREADS, Vec<T>::put(v));
        }
    }
    for (int i = lo + nv * N + tid; i < hi; i += THREADS) dx[i] = Vec<T>::cast(dense(Vec<T>::load(x + i)));
  } else {
    for (int i = lo + tid; i < hi; i += THREADS) dx[i] = Vec<T>::cast(dense(Vec<T>::load(x + i)));
  }
  if (empty || !(given || p.g_top)) return;
  __syncthreads();
  const int ntop = p.g_top ? p.top : 0;
  if (tid <= ntop) {  // thread 0: the given token, thread i + 1: alternative i
    const int64_t j = tid == 0 ? (given ? t : -1) : p.top_tok[row * p.top + tid - 1];
    if (j < lo || j >= hi) return;
    float g = dense(Vec<T>::load(x + j));
    if (tid == 0) {
      g += gl;
      for (int i = 0; i < ntop; ++i)
        if (p.top_tok[row * p.top + i] == j) g += p.g_top[row * p.top + i];
    } else {
      if (given && t == j) return;  // thread 0 writes it
      g += p.g_top[row * p.top + tid - 1];
    }
    dx[j] = Vec<T>::cast(g);
  }
}

static void check(const torch::Tensor& logits, const torch::Tensor& tokens, int64_t top, const char* who) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1), who,
              ": logits (rows, vocab) with contiguous rows");
  TORCH_CHECK(logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat, who,
              ": logits in bf16 or fp32; got ", c10::toString(logits.scalar_type()));
  TORCH_CHECK(tokens.scalar_type() == at::kLong && tokens.dim() == 1 && tokens.size(0) == logits.size(0) &&
                  tokens.is_contiguous() && tokens.device() == logits.device(),
              who, ": int64 tokens (rows) on the logits' GPU");
  TORCH_CHECK(logits.size(1) >= 1 && logits.size(1) <= (1 << 30) && logits.size(0) <= INT32_MAX, who,
              ": vocabulary of 1 to 2^30 and at most 2^31 - 1 rows");
  TORCH_CHECK(top >= 0 && top <= kMaxTop && top <= logits.size(1), who, ": top must be 0 to min(32, vocabulary); got ",
              std::to_string(top));
}

}  // namespace lp

// (logprob, entropy, what the gradient needs, top_logprob, top_token) of each row, each a tensor of its own:
// a user may change the outputs in place before the gradient is taken.
std::vector<torch::Tensor> logprobs_fwd(torch::Tensor logits, torch::Tensor tokens, int64_t top, int64_t ignore) {
  using namespace lp;
  check(logits, tokens, top, "token_logprobs");
  c10::cuda::CUDAGuard guard(logits.device());
  const int64_t rows = logits.size(0);
  auto f = logits.options().dtype(at::kFloat);
  auto lp = torch::empty({rows}, f), ent = torch::empty({rows}, f), stats = torch::empty({3, rows}, f);
  auto tl = torch::empty({rows, top}, f);
  auto tt = torch::empty({rows, top}, tokens.options());
  std::vector<torch::Tensor> out{lp, ent, stats, tl, tt};
  if (rows == 0) return out;
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto* ptr) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(ptr)>>;
    FwdParams<T> p{};
    p.x = ptr;
    p.stride = logits.stride(0);
    p.tokens = tokens.data_ptr<int64_t>(), p.ignore = ignore;
    p.logprob = lp.data_ptr<float>(), p.entropy = ent.data_ptr<float>(), p.stats = stats.data_ptr<float>();
    p.rows = rows;
    p.top_lp = tl.data_ptr<float>(), p.top_tok = tt.data_ptr<int64_t>();
    p.V = (int)logits.size(1), p.top = (int)top;
    // Few rows: latency counts, a row's loads are spread over four times the threads; more rows than SMs: several
    // small CTAs an SM overlap one another's ends of rows.  1024 / 256 threads, us, bf16 logits from HBM, 5
    // alternatives: 65536 wide, 8 rows 12.2 / 16.1, 148 rows 13.9 / 17.5, 149 rows 23.1 / 17.5, 1200 rows 102 / 48;
    // 32768 wide, 148 rows 11.4 / 11.3, 149 rows 19.4 / 11.4.  Away from these widths the switch is less well placed:
    // 8192 wide, 8 rows 8.7 / 4.9; 151936 wide, 149 rows 34.5 / 47.7, 300 rows 52 / 56.
    const bool few = rows <= at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
    if (top > 0) {
      if (few) fwd_kernel<T, true, 1024><<<(int)rows, 1024, 0, st>>>(p);
      else fwd_kernel<T, true, 256><<<(int)rows, 256, 0, st>>>(p);
    } else {
      if (few) fwd_kernel<T, false, 1024><<<(int)rows, 1024, 0, st>>>(p);
      else fwd_kernel<T, false, 256><<<(int)rows, 256, 0, st>>>(p);
    }
  };
  if (logits.scalar_type() == at::kBFloat16) go((const __nv_bfloat16*)logits.data_ptr());
  else go((const float*)logits.data_ptr());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

torch::Tensor logprobs_bwd(torch::Tensor logits, torch::Tensor tokens, int64_t ignore, torch::Tensor stats,
                           torch::Tensor top_tok, c10::optional<torch::Tensor> g_lp,
                           c10::optional<torch::Tensor> g_ent, c10::optional<torch::Tensor> g_top) {
  using namespace lp;
  check(logits, tokens, top_tok.size(1), "token_logprobs backward");
  c10::cuda::CUDAGuard guard(logits.device());
  const int64_t rows = logits.size(0), V = logits.size(1);
  auto dx = torch::empty({rows, V}, logits.options());
  if (rows == 0) return dx;
  auto grad = [&](c10::optional<torch::Tensor>& g, int64_t n) -> const float* {
    if (!g.has_value() || n == 0) return nullptr;
    TORCH_CHECK(g->scalar_type() == at::kFloat && g->numel() == n && g->device() == logits.device(),
                "token_logprobs backward: fp32 gradients of the outputs");
    *g = g->contiguous();
    return g->data_ptr<float>();
  };
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto* ptr) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(ptr)>>;
    BwdParams<T> p{};
    p.x = ptr, p.dx = (T*)dx.data_ptr();
    p.stride = logits.stride(0);
    p.tokens = tokens.data_ptr<int64_t>(), p.ignore = ignore;
    p.stats = stats.data_ptr<float>(), p.rows = rows;
    p.top = (int)top_tok.size(1), p.top_tok = top_tok.data_ptr<int64_t>();
    p.g_lp = grad(g_lp, rows), p.g_ent = grad(g_ent, rows), p.g_top = grad(g_top, rows * p.top);
    p.V = (int)V;
    p.chunk = THREADS * UN * Vec<T>::N;
    p.chunks = (int)((V + p.chunk - 1) / p.chunk);
    TORCH_CHECK(rows * p.chunks <= INT32_MAX, "token_logprobs backward: too many rows");
    bwd_kernel<T><<<(int)(rows * p.chunks), THREADS, 0, st>>>(p);
  };
  if (logits.scalar_type() == at::kBFloat16) go((const __nv_bfloat16*)logits.data_ptr());
  else go((const float*)logits.data_ptr());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return dx;
}

}  // namespace mykb
