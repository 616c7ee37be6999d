// Attention over the 8-bit key/value cache (formats and scales: kv8.cuh).
//
//   o_r = sum_j p_rj v_j,  p = softmax_j(scale q_r.k_j),  k_j = s_kj kq_j,  v_j = s_vj vq_j
//
// with the scales taken out of the products: t_rj = scale log2(e) s_kj (q_r.kq_j) + log2 s_vj,
// w_rj = 2^(t_rj - m_r), o_r = sum w vq / sum w 2^(-log2 s_vj), where m_r follows the row's
// maximum of t.  Both products run on the tensor cores (f16 x f16 -> fp32): e4m3 and int8
// values are exact in f16; a query row is multiplied by a power of two that brings its largest
// element just under 2^15 (bf16's 8 bits are exact in f16 there; elements below 2^-29 of the
// largest fade out); w is rounded to f16's 11 bits, and m_r is kept such that the largest w
// lies in 2^8 .. 2^15, so weights down to 2^-32 of the largest survive the rounding and O is
// rescaled only when a row's maximum grows by more than 2^7.  Sums, maxima and O are fp32.
//
// A decode step reads every visible byte of the cache once and does little with it, so it is
// bound by HBM.  One work list holds the 32-key tiles of all (sequence, KV head, row tile)
// columns; every warp takes an equal run of it, computed on the device from the lengths (ragged
// batches stay balanced, a captured CUDA graph stays valid), and reads it through a ring of its
// own that TMA fills (two bulk copies a tile), running ahead over the ends of columns; warps
// never wait for one another.  Keys are the M side of Q K^T and head dims that of P V, so that
// one 8-column tile holds up to 8 query rows; the contraction index of the first and the row
// index of the second are permuted to make a lane's bytes contiguous in shared memory.
// A column that one warp covers is written at once; else the warps leave fp32 partials and a
// second kernel, whose start overlaps the first, joins them in order: no atomics, and results
// that do not depend on timing.
//
// Measured (B200, CUDA graph, both kernels): 64 sequences of 8192 tokens, 16/4 heads of 128, e4m3:
// 96.5 us, 0.85 of the copy bandwidth (per-lane asynchronous copies instead of TMA: 117 us, of
// which the loads alone took 116).  Two sequences of 131071 tokens: 59.7 us, 0.69 (the join of 222
// partials a column is 10 us of it).  Small calls are bound by latency: one sequence of 2048
// tokens 9.1 us, 48 sequences that see 512 tokens 11.5 us.  Three queries a sequence (two MMA
// columns a row tile, 12 warps an SM): bound by the chain QK -> exp -> PV of each warp's few
// tiles, 64 ragged sequences of up to 2048 tokens 28 us for 31 MB.
//
// Wide calls (prefer_prefill) read the cache back to bf16 and run the bf16 prefill kernel, whose
// weights have bf16's 8 bits instead of 11: 4 x 509 queries behind up to 4096 keys are 0.0022 off
// the result in 64 bits, relative to its norm, of which the rounding of the output is 0.0017.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "kv8.cuh"
#include "kv8_host.h"
#include "tma_host.h"

namespace mykb {
std::vector<torch::Tensor> fa_fwd(torch::Tensor q, torch::Tensor k, torch::Tensor v, c10::optional<torch::Tensor> cu_q,
                                  c10::optional<torch::Tensor> cu_k, c10::optional<torch::Tensor> seqused_k,
                                  int64_t max_q, int64_t max_k, double scale, int64_t left, int64_t right);
int64_t fa_fwd_rounds(int head_dim, int heads, int kv_heads, int64_t seqs, int64_t max_q, int sms);
namespace kv8 {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int KT = 32;        // keys of a tile
constexpr int JOIN_CHUNK = 32;  // partials that join_kernel copies at a time

struct AttendParams {
  const bf16* q;       // (B, L, H, D)
  const uint8_t* ks;   // (B, Hkv, nblk)
  const uint8_t* vs;
  const int* seqlens;  // (B)
  bf16* o;             // (B, L, H, D) contiguous
  float* part;         // [warps][2][rows][D] partial O of a warp's first and last piece
  float* ml;           // [warps][2][rows][2] their maxima and sums
  int warps;           // of attend_kernel
  int* status;
  int64_t q_sb, q_st, q_sh;
  int B, L, H, Hkv, RT, cap, nblk, shift;
  int extra;           // visible keys = seqlens + extra
  int left, right;
  float scale_log2;    // |softmax scale| * log2(e)
  float sign;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 8 x 8 transpose of 16-bit elements over the warp: lane (g, c) gives row g, columns 2c and 2c + 1.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Lets the next kernel of the stream start its prologue; waits until the one before has finished
// (both do nothing where the kernel was launched without that attribute).
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Whether a tile has landed.  If it does not within a second, the status word says so.
__device__ __forceinline__ bool tile_wait(uint64_t* bar, uint32_t parity, int* status) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || mbar_wait_warp(bar, parity, status, __LINE__);
}
// For a warp that gives up: up to a second more for a copy in flight, whatever the status word says, as its shared
// memory is another CTA's after the return.
__device__ __noinline__ void tile_drain(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = globaltimer_ns();
  while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)) &&
         !__any_sync(0xffffffffu, globaltimer_ns() - t0 > kWaitNs)) {
  }
}
// Weight of a partial (m, l) when joined under the maximum M: 0 without any weight; a sum that is
// not a number stays one.
__device__ __forceinline__ float part_weight(float m, float l, float M) {
  return l == 0.f ? 0.f : m == -INFINITY ? 1.f : ex2(m - M);
}

// Shape of the kernel for one head_dim and NT 8-query tiles: keys a tile, tiles in the ring of a
// warp, CTAs an SM.
template <int D, int NT>
struct Shape {
  static constexpr int ROWS = 8 * NT;
  static constexpr int STAGES = D == 64 ? 3 : 1 + NT;
  static constexpr int PER_SM = (D == 64 ? 4 : 3) - (NT - 1);
  static constexpr int TILE = KT * D * 2;  // bytes of a tile's keys and values
  static constexpr int SMEM = WARPS * STAGES * TILE;
};
// Tiles of a sequence that some query sees: [t0, t0 + n).
__device__ __forceinline__ int2 tiles_of(const AttendParams& p, int b, int& kv_len) {
  kv_len = (int)min((int64_t)max(p.seqlens[b], 0) + p.extra, (int64_t)p.cap);
  if (kv_len <= 0) return make_int2(0, 0);
  const int lo = p.left >= 0 ? (int)max((int64_t)0, (int64_t)kv_len - p.L - p.left) : 0;
  const int t0 = lo / KT;
  return make_int2(t0, (kv_len + KT - 1) / KT - t0);
}

// The work list: `total` tiles in runs of `per` or, for the first `rem` warps, per + 1.
struct Runs {
  int total, active, per, rem;
  __device__ __forceinline__ Runs(int total_, int warps) {
    total = total_;
    active = min(warps, total);  // 0 where nothing is visible: no warp has a run
    per = total / max(active, 1), rem = total - per * active;
  }
  __device__ __forceinline__ int first(int w) const { return w * per + min(w, rem); }
  __device__ __forceinline__ int owner(int at) const {
    const int cut = rem * (per + 1);
    return at < cut ? at / (per + 1) : rem + (at - cut) / per;
  }
};

// Walks the tiles of the list: sequence b, column col (KV head and row tile), tile t of its nt.
struct Walk {
  int b, col, t, nt, t0, kv_len;
  __device__ __forceinline__ void enter(const AttendParams& p, int b_) {
    b = b_;
    const int2 tl = tiles_of(p, b, kv_len);
    t0 = tl.x, nt = tl.y;
  }
  __device__ __forceinline__ void next_column(const AttendParams& p, int cols) {
    t = 0;
    if (++col < cols) return;
    col = 0;
    do enter(p, b + 1);
    while (nt == 0 && b < p.B - 1);
  }
};

__device__ __forceinline__ int block_sum(int x, int* red) {  // of all THREADS threads, to all of them
  x = __reduce_add_sync(0xffffffffu, x);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) x += red[w];
  __syncthreads();
  return x;
}

// o of row r of a 16-row tile: where its D outputs start
__device__ __forceinline__ bf16* out_row(const AttendParams& p, int b, int hk, int row, int D) {
  const int g = row / p.L, i = row - g * p.L;
  return p.o + (((int64_t)b * p.L + i) * p.H + hk * (p.H / p.Hkv) + g) * D;
}

// UNI: a scale block spans whole 16-key groups (block >= 16), else each key has its own lookup.
template <int D, int NT, bool INT8, bool UNI>
__global__ void __launch_bounds__(THREADS, Shape<D, NT>::PER_SM)
attend_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, AttendParams p) {
  using S = Shape<D, NT>;
  constexpr int STAGES = S::STAGES, ROWS = S::ROWS, U = KT / 16, HALVES = D / 64, VB = D / 8, MT = D / 16;
  extern __shared__ __align__(1024) unsigned char ring[];
  __shared__ uint64_t full[WARPS][STAGES];
  __shared__ int scan[THREADS + 1];
  __shared__ int2 start[WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int G = p.H / p.Hkv, rows_all = G * p.L;
  const int cols = p.Hkv * p.RT;  // columns a sequence
  launch_dependents();
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[warp][i], 1);
    fence_barrier_init();
    tma_prefetch_desc(&tmk);
    tma_prefetch_desc(&tmv);
  }

  // ---- the work list: each thread sums a run of sequences, then a scan over the threads
  const int run = (p.B + THREADS - 1) / THREADS;
  {
    int x = 0, kl;
    for (int i = tid * run; i < min((tid + 1) * run, p.B); ++i) x += tiles_of(p, i, kl).y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __shared__ int wsum[WARPS];
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    for (int w = 0; w < warp; ++w) x += wsum[w];
    scan[tid + 1] = x;
    if (tid == 0) scan[0] = 0;
    __syncthreads();
  }
  const Runs runs(scan[THREADS] * cols, p.warps);
  // the first runs go to different CTAs, so that short lists spread over the SMs
  const int me = warp * gridDim.x + blockIdx.x;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const int at = runs.first(w * gridDim.x + blockIdx.x);
    if (scan[tid] * cols <= at && at < scan[tid + 1] * cols) {
      int base = scan[tid] * cols, b = tid * run, kl;
      for (;; ++b) {
        const int n = tiles_of(p, b, kl).y * cols;
        if (at < base + n) break;
        base += n;
      }
      start[w] = make_int2(b, at - base);
    }
  }
  // sequences without visible keys: their rows are 0
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    int kl;
    if (tiles_of(p, b, kl).y > 0) continue;
    uint32_t* o = reinterpret_cast<uint32_t*>(p.o + (int64_t)b * p.L * p.H * D);
    for (int64_t i = tid; i < (int64_t)p.L * p.H * D / 2; i += THREADS) o[i] = 0;
  }
  grid_dependency_wait();  // the new tokens are in the cache
  __syncthreads();
  if (me >= runs.active) return;
  int left = runs.first(me + 1) - runs.first(me);  // tiles still to use
  Walk use;
  use.enter(p, start[warp].x);
  use.col = start[warp].y / use.nt, use.t = start[warp].y - use.col * use.nt;
  Walk get = use;  // runs ahead of `use`, over column ends
  int to_get = left;
  unsigned char* slots = ring + warp * (STAGES * S::TILE);  // this warp's tiles: 32 keys, then 32 values
  // bytes of this lane in a tile: TMA stores the 16-byte chunk q of row r at q ^ (r & 7) (rows of 128
  // bytes) or q ^ ((r >> 1) & 3) (64 bytes), which spreads the rows that a load touches over the banks
  uint32_t koff[HALVES], voff[2];
#pragma unroll
  for (int h = 0; h < HALVES; ++h) koff[h] = g * D + (((h * 4 + c) ^ (D == 128 ? g : g >> 1)) << 4);
#pragma unroll
  for (int y = 0; y < 2; ++y)
    voff[y] = KT * D + (2 * c + y) * D + (D == 128 ? (g ^ (2 * c + y)) << 4 : (((g >> 1) ^ c) << 4) + (g & 1) * 8);
  uint32_t issued = 0, used = 0;
  auto load_tile = [&]() {  // the next tile, into the slot that the warp has finished reading
    if (to_get == 0) return;
    const uint32_t st = issued++ % STAGES;
    if (lane == 0) {
      const int key0 = (get.t0 + get.t) * KT, bh = get.b * p.Hkv + get.col / p.RT;
      mbar_arrive_expect_tx(&full[warp][st], S::TILE);
      tma_load_3d(slots + st * S::TILE, &tmk, &full[warp][st], 0, key0, bh);
      tma_load_3d(slots + st * S::TILE + KT * D, &tmv, &full[warp][st], 0, key0, bh);
    }
    if (--to_get > 0 && ++get.t == get.nt) get.next_column(p, cols);
  };
#pragma unroll
  for (int i = 0; i < STAGES; ++i) load_tile();
  const float ninf = -INFINITY;
  int piece = 0;

  for (;;) {
    const int b = use.b, kv_len = use.kv_len;
    const int n = min(use.nt - use.t, left);  // tiles of this piece of the column
    const int hk = use.col / p.RT, rt = use.col - hk * p.RT;
    const int rows = min(ROWS, rows_all - rt * ROWS);
    const int64_t bh = (int64_t)b * p.Hkv + hk;
    const int key_first = (use.t0 + use.t) * KT;
    const uint8_t* ksb = p.ks + bh * p.nblk;
    const uint8_t* vsb = p.vs + bh * p.nblk;
    // scale bytes of a tile's keys: one a 16-key group, or those of this lane's keys g and g + 8
    constexpr int NS = UNI ? U : 2 * U;
    int kbyte[NS], vbyte[NS];
    auto load_scales = [&](int i) {
      const int key0 = key_first + i * KT;
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        const int key = UNI ? key0 + x * 16 : key0 + x * 8 + g;
        const bool ok = key < kv_len;
        kbyte[x] = ok ? ksb[key >> p.shift] : kMinScale;
        vbyte[x] = ok ? vsb[key >> p.shift] : kMinScale;
      }
    };
    load_scales(0);

    // ---- the queries, scaled to f16: row 8 nt + g of the tile is column g of the nt-th B operand
    uint32_t qb[NT][D / 16][2];
    float rowf[NT][2];  // of the rows 8 nt + 2c, 2c + 1, which this lane's scores belong to
    int qpos[NT][2];
#pragma unroll
    for (int nt8 = 0; nt8 < NT; ++nt8) {
      const int r = rt * ROWS + nt8 * 8 + g;
      const bool ok = r < rows_all;
      const int gh = ok ? r / p.L : 0, i = ok ? r % p.L : 0;
      const bf16* src = p.q + b * p.q_sb + i * p.q_st + (int64_t)(hk * G + gh) * p.q_sh + c * 16;
      uint4 w[HALVES * 2];
      uint32_t am = 0;
#pragma unroll
      for (int h = 0; h < HALVES * 2; ++h) {
        w[h] = ok ? __ldg(reinterpret_cast<const uint4*>(src + (h >> 1) * 64 + (h & 1) * 8)) : make_uint4(0, 0, 0, 0);
        am = __vmaxu2(am, __vmaxu2(w[h].x & 0x7fff7fffu, w[h].y & 0x7fff7fffu));
        am = __vmaxu2(am, __vmaxu2(w[h].z & 0x7fff7fffu, w[h].w & 0x7fff7fffu));
      }
      uint32_t a16 = max(am & 0xffffu, am >> 16);
      a16 = max(a16, __shfl_xor_sync(0xffffffffu, a16, 1));
      a16 = max(a16, __shfl_xor_sync(0xffffffffu, a16, 2));
      const int e = (int)(a16 >> 7);
      // 2^(14 - (e - 127)); rows with an infinity or NaN keep their values (and give NaN)
      const int field = e == 255 ? 127 : min(253, 268 - e);
      const float mul = __int_as_float(field << 23) * p.sign;
      const float back = __int_as_float((254 - field) << 23) * p.scale_log2;
#pragma unroll
      for (int h = 0; h < HALVES * 2; ++h) {
        const uint32_t ww[4] = {w[h].x, w[h].y, w[h].z, w[h].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float x = __uint_as_float(ww[k] << 16) * mul, y = __uint_as_float(ww[k] & 0xffff0000u) * mul;
          // elements (2k, 2k + 1) of 8: MMA step (k >> 1), its lower or upper k half
          qb[nt8][h * 2 + (k >> 1)][k & 1] = pack_f16(x, y);
        }
      }
#pragma unroll
      for (int q2 = 0; q2 < 2; ++q2) {
        rowf[nt8][q2] = __shfl_sync(0xffffffffu, back, (2 * c + q2) * 4);
        qpos[nt8][q2] = kv_len - p.L + (rt * ROWS + nt8 * 8 + 2 * c + q2) % p.L;
      }
    }

    // m is the maximum less 8 that the sums stand for; `limit` is how far above m a weight may rise
    // (everything, before the first)
    float m[NT][2], l[NT][2], limit[NT][2];
    float o[NT][MT][4];
#pragma unroll
    for (int nt8 = 0; nt8 < NT; ++nt8) {
      m[nt8][0] = m[nt8][1] = l[nt8][0] = l[nt8][1] = 0.f;
      limit[nt8][0] = limit[nt8][1] = ninf;
#pragma unroll
      for (int t = 0; t < MT; ++t) o[nt8][t][0] = o[nt8][t][1] = o[nt8][t][2] = o[nt8][t][3] = 0.f;
    }

    for (int i = 0; i < n; ++i) {
      int kx[NS], vx[NS];
#pragma unroll
      for (int x = 0; x < NS; ++x) kx[x] = kbyte[x], vx[x] = vbyte[x];
      if (i + 1 < n) load_scales(i + 1);
      const uint32_t st = used % STAGES;
      if (!tile_wait(&full[warp][st], (used / STAGES) & 1, p.status)) {
        for (; used != issued; ++used) tile_drain(&full[warp][used % STAGES], (used / STAGES) & 1);
        return;
      }
      ++used;
      const unsigned char* buf = slots + st * S::TILE;
      const int key0 = key_first + i * KT;
      // ---- S^T = K Q^T (16 keys x 8 queries an MMA); s[.][u][e]: key 16 u + g + 8 (e >> 1), query 2c + (e & 1)
      float s[NT][U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float s2[NT][4];  // a second chain of accumulations
#pragma unroll
        for (int nt8 = 0; nt8 < NT; ++nt8)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt8][u][e] = s2[nt8][e] = 0.f;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          const uint4 w0 = *reinterpret_cast<const uint4*>(buf + koff[h] + u * 16 * D);
          const uint4 w1 = *reinterpret_cast<const uint4*>(buf + koff[h] + (u * 16 + 8) * D);
          const uint32_t x0[4] = {w0.x, w0.y, w0.z, w0.w}, x1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t a[4];
            widen4<INT8>(x0[k], a[0], a[2]);
            widen4<INT8>(x1[k], a[1], a[3]);
#pragma unroll
            for (int nt8 = 0; nt8 < NT; ++nt8)
              mma_f16(k & 1 ? s2[nt8] : s[nt8][u], a, qb[nt8][h * 4 + k][0], qb[nt8][h * 4 + k][1]);
          }
        }
#pragma unroll
        for (int nt8 = 0; nt8 < NT; ++nt8)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt8][u][e] += s2[nt8][e];
      }
      // ---- t = s * f + log2 s_v - m, masked
      float isv[NS];
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        const float lv = vx[x] == kBadScale ? __int_as_float(0x7fffffff) : (float)(vx[x] - 127);
        const float sk = scale_value(kx[x]);
        isv[x] = scale_inverse(min(vx[x], 253));
#pragma unroll
        for (int nt8 = 0; nt8 < NT; ++nt8)
#pragma unroll
          for (int q2 = 0; q2 < 2; ++q2) {
            const float f = rowf[nt8][q2] * sk, add = lv - m[nt8][q2];
            if constexpr (UNI) {
              s[nt8][x][q2] = fmaf(s[nt8][x][q2], f, add);
              s[nt8][x][2 + q2] = fmaf(s[nt8][x][2 + q2], f, add);
            } else {
              float& t = s[nt8][x >> 1][2 * (x & 1) + q2];
              t = fmaf(t, f, add);
            }
          }
      }
      // every row sees the whole tile
      const bool inner = key0 + KT <= kv_len && (p.right < 0 || key0 + KT - 1 <= kv_len - p.L + p.right) &&
                         (p.left < 0 || key0 >= kv_len - 1 - p.left);
      if (!inner) {
#pragma unroll
        for (int nt8 = 0; nt8 < NT; ++nt8)
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = key0 + u * 16 + (e >> 1) * 8 + g, at = qpos[nt8][e & 1];
              const bool vis = key < kv_len && (p.right < 0 || key <= at + p.right) && (p.left < 0 || key >= at - p.left);
              if (!vis) s[nt8][u][e] = ninf;
            }
      }
      // ---- follow the maximum; O is rescaled rarely
      bool rise = false;
#pragma unroll
      for (int nt8 = 0; nt8 < NT; ++nt8)
#pragma unroll
        for (int q2 = 0; q2 < 2; ++q2) {
          float x = ninf;
#pragma unroll
          for (int u = 0; u < U; ++u) x = fmax3(x, s[nt8][u][q2], s[nt8][u][2 + q2]);
          rise |= x > limit[nt8][q2];
        }
      if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
        for (int nt8 = 0; nt8 < NT; ++nt8)
#pragma unroll
          for (int q2 = 0; q2 < 2; ++q2) {
            float x = ninf;
#pragma unroll
            for (int u = 0; u < U; ++u) x = fmax3(x, s[nt8][u][q2], s[nt8][u][2 + q2]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            if (x > limit[nt8][q2]) {
              // nothing is summed before the first
              const float up = x - 8.f, corr = limit[nt8][q2] == ninf ? 0.f : ex2(-up);
              limit[nt8][q2] = 15.f;
              m[nt8][q2] += up;
              l[nt8][q2] *= corr;
#pragma unroll
              for (int t = 0; t < MT; ++t) o[nt8][t][q2] *= corr, o[nt8][t][2 + q2] *= corr;
#pragma unroll
              for (int u = 0; u < U; ++u) s[nt8][u][q2] -= up, s[nt8][u][2 + q2] -= up;
            }
          }
      }
      // ---- weights and their sums; P^T as the B operand of O^T += V^T P^T
      uint32_t pb[NT][U][2];
#pragma unroll
      for (int nt8 = 0; nt8 < NT; ++nt8)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float (&w)[4] = s[nt8][u];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = ex2(w[e]);
#pragma unroll
          for (int q2 = 0; q2 < 2; ++q2) {
            if constexpr (UNI) {
              l[nt8][q2] = fmaf(w[q2] + w[2 + q2], isv[u], l[nt8][q2]);
            } else {
              l[nt8][q2] = fmaf(w[q2], isv[2 * u], l[nt8][q2]);
              l[nt8][q2] = fmaf(w[2 + q2], isv[2 * u + 1], l[nt8][q2]);
            }
          }
          pb[nt8][u][0] = transpose8(pack_f16(w[0], w[1]));
          pb[nt8][u][1] = transpose8(pack_f16(w[2], w[3]));
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint32_t vw[4][VB / 4];  // keys 2c, 2c + 1, 2c + 8, 2c + 9; head dims g * VB ..
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const unsigned char* src = buf + voff[i4 & 1] + (u * 16 + (i4 >> 1) * 8) * D;
          if constexpr (D == 128) {
            const uint4 w = *reinterpret_cast<const uint4*>(src);
            vw[i4][0] = w.x, vw[i4][1] = w.y, vw[i4][2] = w.z, vw[i4][3] = w.w;
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(src);
            vw[i4][0] = w.x, vw[i4][1] = w.y;
          }
        }
        if (!inner) {  // past the length there may be any bytes, NaN among them
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4)
            if (key0 + u * 16 + (i4 >> 1) * 8 + 2 * c + (i4 & 1) >= kv_len)
#pragma unroll
              for (int x = 0; x < VB / 4; ++x) vw[i4][x] = 0;
        }
#pragma unroll
        for (int x = 0; x < VB / 4; ++x) {
          // MMA tile t = 2x + k: its rows g and g + 8 are the head dims g * VB + 2t and + 1
          uint32_t a[2][4];
          widen4<INT8>(__byte_perm(vw[0][x], vw[1][x], 0x5140), a[0][0], a[0][1]);
          widen4<INT8>(__byte_perm(vw[2][x], vw[3][x], 0x5140), a[0][2], a[0][3]);
          widen4<INT8>(__byte_perm(vw[0][x], vw[1][x], 0x7362), a[1][0], a[1][1]);
          widen4<INT8>(__byte_perm(vw[2][x], vw[3][x], 0x7362), a[1][2], a[1][3]);
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int nt8 = 0; nt8 < NT; ++nt8) mma_f16(o[nt8][2 * x + k], a[k], pb[nt8][u][0], pb[nt8][u][1]);
        }
      }
      __syncwarp();
      load_tile();
    }
    // ---- the piece's result: this lane has head dims g * VB .. of the rows 8 nt + 2c, 2c + 1
    const bool whole = use.t == 0 && n == use.nt;
    const int64_t slot = (int64_t)me * 2 + (piece > 0);
#pragma unroll
    for (int nt8 = 0; nt8 < NT; ++nt8)
#pragma unroll
      for (int q2 = 0; q2 < 2; ++q2) {
        const int r = nt8 * 8 + 2 * c + q2;
        float L = l[nt8][q2];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
        if (r >= rows) continue;
        float x[VB];
#pragma unroll
        for (int t = 0; t < MT; ++t) x[2 * t] = o[nt8][t][q2], x[2 * t + 1] = o[nt8][t][2 + q2];
        if (whole) {
          const float inv = L == 0.f ? 0.f : 1.f / L;
          uint4* dst = reinterpret_cast<uint4*>(out_row(p, b, hk, rt * ROWS + r, D) + g * VB);
#pragma unroll
          for (int k = 0; k < VB / 8; ++k)
            dst[k] = make_uint4(pack_bf16x2(x[8 * k] * inv, x[8 * k + 1] * inv), pack_bf16x2(x[8 * k + 2] * inv, x[8 * k + 3] * inv),
                                pack_bf16x2(x[8 * k + 4] * inv, x[8 * k + 5] * inv), pack_bf16x2(x[8 * k + 6] * inv, x[8 * k + 7] * inv));
        } else {
          float4* dst = reinterpret_cast<float4*>(p.part + (slot * ROWS + r) * D + g * VB);
#pragma unroll
          for (int k = 0; k < VB / 4; ++k) dst[k] = make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
          if (g == 0)
            *reinterpret_cast<float2*>(p.ml + (slot * ROWS + r) * 2) =
                make_float2(limit[nt8][q2] == ninf ? ninf : m[nt8][q2], L);
        }
      }
    left -= n;
    if (left == 0) return;
    ++piece;
    use.next_column(p, cols);
  }
}

// Joins the partials of the columns that several warps share, in the order of the list; one CTA
// for each row of a column.  Launched so that everything up to the wait overlaps attend_kernel.
template <int D, int NT>
__global__ void __launch_bounds__(THREADS) join_kernel(AttendParams p) {
  constexpr int ROWS = 8 * NT, D4 = D / 4, GROUPS = THREADS / D4;
  extern __shared__ __align__(16) float jsm[];  // [JOIN_CHUNK][D] partials, then the weights of all
  float* wt = jsm + JOIN_CHUNK * D;
  __shared__ int red[WARPS];
  __shared__ float fred[WARPS];
  __shared__ float4 part[THREADS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cols = p.Hkv * p.RT;
  const int b = blockIdx.x / cols, col = blockIdx.x - b * cols, r = blockIdx.y;
  int kl, all = 0, before = 0;
  for (int i = tid; i < p.B; i += THREADS) {
    const int n = tiles_of(p, i, kl).y;
    all += n;
    if (i < b) before += n;
  }
  const Runs runs(block_sum(all, red) * cols, p.warps);
  const int nt = tiles_of(p, b, kl).y;
  const int cf = block_sum(before, red) * cols + col * nt;
  grid_dependency_wait();
  if (nt == 0) return;
  const int c0 = runs.owner(cf), nc = runs.owner(cf + nt - 1) + 1 - c0;
  if (nc == 1) return;  // written by attend_kernel
  const int hk = col / p.RT, rt = col - hk * p.RT;
  if (rt * ROWS + r >= (p.H / p.Hkv) * p.L) return;
  // the column is the first piece of every warp but c0, and of c0 only if its run starts with it
  const bool late = runs.first(c0) != cf;
  auto at = [&](int x) { return (((int64_t)c0 + x) * 2 + (x == 0 && late)) * ROWS + r; };
  float M = -INFINITY, L = 0.f;
  for (int x = tid; x < nc; x += THREADS) M = fmaxf(M, p.ml[at(x) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) fred[warp] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) M = fmaxf(M, fred[w]);
  __syncthreads();
  for (int x = tid; x < nc; x += THREADS) {
    const float2 ml = *reinterpret_cast<const float2*>(p.ml + at(x) * 2);
    const float f = part_weight(ml.x, ml.y, M);
    wt[x] = f;
    if (f != 0.f) L += f * ml.y;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  if (lane == 0) fred[warp] = L;
  __syncthreads();
  L = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) L += fred[w];
  // the partials by asynchronous copies, CHUNK at a time; groups of D / 4 threads sum every GROUPS-th
  float4* stage = reinterpret_cast<float4*>(jsm);
  const int e = tid % D4, first = tid / D4;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int x0 = 0; x0 < nc; x0 += JOIN_CHUNK) {
    const int nb = min(JOIN_CHUNK, nc - x0);
    for (int x = first; x < nb; x += GROUPS)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(stage + x * D4 + e)),
                   "l"(p.part + at(x0 + x) * D + e * 4)
                   : "memory");
    asm volatile("cp.async.wait_all;" ::: "memory");  // a thread sums what it copied itself
    for (int x = first; x < nb; x += GROUPS) {
      const float f = wt[x0 + x];
      const float4 v = stage[x * D4 + e];
      a.x = fmaf(f, v.x, a.x), a.y = fmaf(f, v.y, a.y), a.z = fmaf(f, v.z, a.z), a.w = fmaf(f, v.w, a.w);
    }
  }
  part[tid] = a;
  __syncthreads();
  if (tid >= D4) return;
#pragma unroll
  for (int x = 1; x < GROUPS; ++x) {
    const float4 v = part[x * D4 + tid];
    a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  *reinterpret_cast<uint2*>(out_row(p, b, hk, rt * ROWS + r, D) + e * 4) =
      make_uint2(pack_bf16x2(a.x * inv, a.y * inv), pack_bf16x2(a.z * inv, a.w * inv));
}

// Whether to read the cache back to bf16 and run the prefill kernel instead, by what both take in ns.
// Here: 18 a column (its 16 rows are joined by as many CTAs) and 0.04 a key and column (0.028 at head_dim 64: its
// tiles come from L2 after the first row tile).  There: the keys of the items that one CTA of the prefill kernel takes
// in turn, which is all it is split over, at 17 a key where an item is two heads (even groups) and 20 where it is one,
// plus the read back of the whole capacity at HBM speed.  The lengths are known on the device only, so both sides
// stand for full sequences.
// Measured here / there, us (predicted in brackets): 4 x 509 queries, 16/4 heads of 128, ragged to 4096 keys:
// 173 / 56 (384 / 92); 1 x 512, 16/4 of 64, 2048: 57 / 44 (50 / 49); 8 x 32, 16/4 of 128, 8192: 101 / 320 (100 / 326);
// 13 x 155 of one head of 128, 30000: 162 / 633 (169 / 664); 64 x 64, 16/4 of 64, 2048: 296 / 509 (320 / 536);
// 16 x 80, 16/4 of 64, ragged to 16000: 284 / 656 (608 / 1168); 6 x 184, 16/8 of 64, 966, window 512: 70 / 38 (53 / 39).
// The faster side was taken for 59 of the 60 shapes that the figures were fitted to (the other cost 1.19 times the best)
// and for 60 of 60 further ones (1 to 30 sequences, 22 to 2046 queries, 262 to 56913 keys, groups of 1 to 8).
// Up to 64 rows a KV head always stay here.
static bool prefer_prefill(const Cache& c, int H, int L, int64_t columns, int64_t span, int64_t left, int64_t right,
                           int sms) {
  const double here = 11e3 + columns * (18 + (c.D == 64 ? 0.028 : 0.04) * span);
  // keys that 128 queries see
  const int64_t keys = left >= 0 && right >= 0 ? std::min<int64_t>(c.cap, left + right + 128) : c.cap;
  const double there = 14e3 + (H / c.Hkv % 2 == 0 ? 17.0 : 20.0) * fa_fwd_rounds(c.D, H, c.Hkv, c.B, L, sms) * keys +
                       0.001 * c.D * c.B * c.Hkv * c.cap;
  return (int64_t)(H / c.Hkv) * L > 64 && (there < here || columns * ((c.cap + KT - 1) / KT) > INT32_MAX);
}

}  // namespace kv8

// q (B, L, H, D) bf16; new keys / values k, v (B, L, Hkv, D), if any, are written at
// seqlens[b] first.  Queries are aligned to the end of the visible keys.
torch::Tensor kv8_attend(torch::Tensor q, torch::Tensor keys, torch::Tensor values, torch::Tensor key_scales,
                         torch::Tensor value_scales, int64_t block, c10::optional<torch::Tensor> k,
                         c10::optional<torch::Tensor> v, torch::Tensor seqlens, double scale, int64_t left,
                         int64_t right) {
  using namespace kv8;
  const char* who = "flash_attn_with_kvcache8";
  c10::cuda::OptionalCUDAGuard guard;
  if (keys.is_cuda()) guard.set_device(keys.device());
  Cache c = check_cache(keys, values, key_scales, value_scales, block, who);
  c.device = keys.get_device();
  check_lens(seqlens, c, keys, who);
  TORCH_CHECK(q.is_cuda() && q.get_device() == c.device && q.scalar_type() == at::kBFloat16 && q.dim() == 4 &&
                  q.size(0) == c.B && q.size(3) == c.D,
              who, ": queries (B, L, H, D) in bf16 on the cache's GPU");
  TORCH_CHECK(k.has_value() == v.has_value(), who, ": new keys and values come together");
  TORCH_CHECK(c.Hkv > 0 && q.size(2) % c.Hkv == 0, who, ": query heads (",
              std::to_string(q.size(2)), ") must be a multiple of key/value heads (", std::to_string(c.Hkv), ")");
  TORCH_CHECK(q.size(1) * q.size(2) <= (1 << 30), who, ": too many queries");
  TORCH_CHECK(std::isfinite(scale), who, ": the softmax scale must be finite");
  const int* lens = seqlens.data_ptr<int>();
  int extra = 0;
  if (k.has_value()) {
    append(c, *k, *v, lens, who);
    extra = (int)k->size(1);
  }
  const int L = (int)q.size(1), H = (int)q.size(2), G = H / c.Hkv;
  auto o = torch::empty({c.B, L, H, c.D}, q.options());
  if (o.numel() == 0) return o;
  if (c.cap == 0) return o.zero_();
  left = left < 0 ? -1 : std::min<int64_t>(left, 1 << 29);
  right = right < 0 ? -1 : std::min<int64_t>(right, 1 << 29);
  static int sms[64] = {0};
  if (!sms[c.device]) C10_CUDA_CHECK(cudaDeviceGetAttribute(&sms[c.device], cudaDevAttrMultiProcessorCount, c.device));
  const int nt = G * L <= 8 ? 1 : 2, rows = 8 * nt, RT = (G * L + rows - 1) / rows;
  int64_t span = c.cap;  // most keys a sequence can show
  if (left >= 0) span = std::min<int64_t>(span, left + L + KT);
  const int64_t columns = (int64_t)c.B * c.Hkv * RT;
  if (prefer_prefill(c, H, L, columns, span, left, right, sms[c.device])) {
    auto opt = q.options();
    auto kb = torch::empty({c.B, c.cap, c.Hkv, c.D}, opt), vb = torch::empty({c.B, c.cap, c.Hkv, c.D}, opt);
    read(c, lens, extra, nullptr, 0, c.cap, 256, kb, vb, who);  // 256: more than a key tile of the prefill kernel
    auto used = (seqlens + extra).clamp_(0, c.cap);
    // the prefill kernel takes the maximum of the scores before it scales them, so its scale must be
    // positive: a sign goes into the queries (exactly), and so does a 0 (an infinity or NaN becomes NaN)
    if (scale <= 0) {
      q = scale < 0 ? q.neg() : q.mul(0);
      scale = scale < 0 ? -scale : 1.0;
    }
    // it reads queries as rows of packed heads, equally far apart over the whole batch
    const bool packed = rows16(q) && (H == 1 || q.stride(2) == c.D) && q.stride(1) >= (int64_t)H * c.D &&
                        (c.B == 1 || q.stride(0) == L * q.stride(1));
    if (!packed) q = q.clone(at::MemoryFormat::Contiguous);
    return fa_fwd(q, kb, vb, c10::nullopt, c10::nullopt, used, L, c.cap, scale, left, right)[0];
  }
  if (!rows16(q)) q = q.clone(at::MemoryFormat::Contiguous);
  AttendParams p{};
  p.q = (const bf16*)q.data_ptr();
  p.ks = c.scale[0], p.vs = c.scale[1];
  p.seqlens = lens;
  p.o = (bf16*)o.data_ptr();
  p.q_sb = q.stride(0), p.q_st = q.stride(1), p.q_sh = q.stride(2);
  p.B = c.B, p.L = L, p.H = H, p.Hkv = c.Hkv, p.RT = RT;
  p.cap = c.cap, p.nblk = c.nblk, p.shift = c.shift, p.extra = extra;
  p.left = (int)left, p.right = (int)right;
  p.scale_log2 = (float)(std::abs(scale) * 1.4426950408889634), p.sign = scale < 0 ? -1.f : 1.f;
  const int per_sm = c.D == 64 ? (nt == 1 ? Shape<64, 1>::PER_SM : Shape<64, 2>::PER_SM)
                               : (nt == 1 ? Shape<128, 1>::PER_SM : Shape<128, 2>::PER_SM);
  const int64_t want = (columns * ((span + KT - 1) / KT) + WARPS - 1) / WARPS;
  const int grid = (int)std::min<int64_t>(want, (int64_t)sms[c.device] * per_sm), warps = grid * WARPS;
  TORCH_CHECK(columns * ((c.cap + KT - 1) / KT) <= INT32_MAX, who, ": too many sequences x heads x keys");
  // workspace: partials of at most two pieces a warp
  const int64_t part = (int64_t)warps * 2 * rows * c.D, ml = (int64_t)warps * 2 * rows * 2;
  auto work = torch::empty({part + ml}, q.options().dtype(at::kFloat));
  p.part = work.data_ptr<float>();
  p.ml = p.part + part;
  p.warps = warps;
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  auto start = [&](auto kern, dim3 blocks, int smem, bool overlap, auto... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = blocks, cfg.blockDim = THREADS, cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr, cfg.numAttrs = overlap ? 1 : 0;
    C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, args...));
  };
  const bool uni = c.shift >= 4;
  p.status = device_status();
  const CUtensorMapSwizzle swizzle = c.D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  auto map = [&](uint8_t* base) {
    return make_tmap_3d(base, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.D, c.cap, (int64_t)c.B * c.Hkv, c.D,
                        (int64_t)c.cap * c.D, c.D, KT, swizzle);
  };
  const CUtensorMap tmk = map(c.data[0]), tmv = map(c.data[1]);
  auto launch = [&](auto kern, SmemOptIn& attr, int smem) {
    C10_CUDA_CHECK(attr.ensure(kern, smem));
    start(kern, grid, smem, extra > 0, tmk, tmv, p);  // the kernel before it is then append()'s
  };
  static SmemOptIn a[16];
#define KV8_CASE(d, n, i8, un)                                 \
  if (c.D == d && nt == n && c.int8 == i8 && uni == un)        \
    launch(attend_kernel<d, n, i8, un>, a[(d == 128) * 8 + (n == 2) * 4 + i8 * 2 + un], Shape<d, n>::SMEM)
#define KV8_CASES(d, n)       \
  KV8_CASE(d, n, false, false); \
  KV8_CASE(d, n, false, true);  \
  KV8_CASE(d, n, true, false);  \
  KV8_CASE(d, n, true, true);   \
  if (c.D == d && nt == n) start(join_kernel<d, n>, dim3((int)columns, std::min(rows, G * L)), (JOIN_CHUNK * d + warps) * (int)sizeof(float), true, p)
  KV8_CASES(64, 1);
  KV8_CASES(64, 2);
  KV8_CASES(128, 1);
  KV8_CASES(128, 2);
#undef KV8_CASES
#undef KV8_CASE
  return o;
}

}  // namespace mykb
