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
// bound by HBM.  One work list holds the 16-key-multiple tiles of all (sequence, KV head,
// 16-row tile) columns; every CTA takes an equal run of it, computed on the device from the
// lengths (ragged batches stay balanced, a captured CUDA graph stays valid).  The four warps
// of a CTA take its tiles in turn; each lane copies exactly the bytes that it will feed to the
// MMAs into its own slots of shared memory (cp.async, several tiles ahead), so there are no
// bank conflicts, barriers or transposes: the contraction index of Q K^T and the column index
// of P V are permuted to make a lane's bytes contiguous in memory.
// A column that one CTA covers is written at once; else the CTAs leave fp32 partials and a
// second kernel, whose start overlaps the first, joins them in order: no atomics, and results
// that do not depend on timing.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "kv8.cuh"
#include "kv8_host.h"

namespace mykb {
std::vector<torch::Tensor> fa_fwd(torch::Tensor q, torch::Tensor k, torch::Tensor v, c10::optional<torch::Tensor> cu_q,
                                  c10::optional<torch::Tensor> cu_k, c10::optional<torch::Tensor> seqused_k,
                                  int64_t max_q, int64_t max_k, double scale, int64_t left, int64_t right);
namespace kv8 {

constexpr int ROWS = 16;   // query rows of one MMA tile
constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;

struct AttendParams {
  const bf16* q;       // (B, L, H, D)
  const uint8_t* k;    // (B, Hkv, cap, D)
  const uint8_t* v;
  const uint8_t* ks;   // (B, Hkv, nblk)
  const uint8_t* vs;
  const int* seqlens;  // (B)
  bf16* o;             // (B, L, H, D) contiguous
  float* part;         // [grid][2][16][D] partial O of a CTA's first and last piece, as [row][t][n] (see attend_kernel)
  float* ml;           // [grid][2][16][2] their maxima and sums
  int grid;            // CTAs of attend_kernel
  int64_t q_sb, q_st, q_sh;
  int B, L, H, Hkv, RT, cap, nblk, shift;
  int extra;           // visible keys = seqlens + extra
  int left, right;
  float scale_log2;    // |softmax scale| * log2(e)
  float sign;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
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
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Lets the next kernel of the stream start its prologue; waits until the one before has finished
// (both do nothing where the kernel was launched without that attribute).
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Weight of a partial (m, l) when joined under the maximum M: 0 without any weight; a sum that is
// not a number stays one.
__device__ __forceinline__ float part_weight(float m, float l, float M) {
  return l == 0.f ? 0.f : m == -INFINITY ? 1.f : ex2(m - M);
}

// Shape of the kernel for one head_dim: keys a tile, tiles in the ring, CTAs an SM.
template <int D>
struct Shape {
  static constexpr int KT = 32;
  static constexpr int STAGES = 3;
  static constexpr int TILE = KT * D * 2;  // bytes of a tile's keys and values
  static constexpr int RING = WARPS * STAGES * TILE;
  static constexpr int OROW = D + 8;       // floats of a row in the merge buffer: conflict-free float2 writes
  static constexpr int SMEM = RING > WARPS * ROWS * OROW * 4 ? RING : WARPS * ROWS * OROW * 4;
  static constexpr int PER_SM = D == 64 ? 3 : 2;
};

// Tiles of a sequence that some query sees: [t0, t0 + n).
template <int KT>
__device__ __forceinline__ int2 tiles_of(const AttendParams& p, int b, int& kv_len) {
  kv_len = (int)min((int64_t)max(p.seqlens[b], 0) + p.extra, (int64_t)p.cap);
  if (kv_len <= 0) return make_int2(0, 0);
  const int lo = p.left >= 0 ? (int)max((int64_t)0, (int64_t)kv_len - p.L - p.left) : 0;
  const int t0 = lo / KT;
  return make_int2(t0, (kv_len + KT - 1) / KT - t0);
}

// The work list: `total` tiles in runs of `per` or, for the first `rem` CTAs, per + 1.
struct Runs {
  int total, active, per, rem;
  __device__ __forceinline__ Runs(int total_, int grid) {
    total = total_;
    // as many CTAs take part as get at least one tile a warp
    active = max(1, min(grid, (total + WARPS - 1) / WARPS));
    per = total / active, rem = total - per * active;
  }
  __device__ __forceinline__ int first(int cta) const { return cta * per + min(cta, rem); }
  __device__ __forceinline__ int owner(int at) const {
    const int cut = rem * (per + 1);
    return at < cut ? at / (per + 1) : rem + (at - cut) / per;
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
template <int D, bool INT8, bool UNI>
__global__ void __launch_bounds__(THREADS, Shape<D>::PER_SM) attend_kernel(AttendParams p) {
  using S = Shape<D>;
  constexpr int KT = S::KT, STAGES = S::STAGES, U = KT / 16, HALVES = D / 64, VB = D / 8;
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ int scan[THREADS + 1];
  __shared__ int start_base, start_b;
  __shared__ float wM[WARPS][ROWS], wL[WARPS][ROWS], rL[ROWS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int G = p.H / p.Hkv, rows_all = G * p.L;
  const int cols = p.Hkv * p.RT;  // columns a sequence
  launch_dependents();

  // ---- the work list: each thread sums a run of sequences, then a scan over the threads
  const int run = (p.B + THREADS - 1) / THREADS;
  {
    int x = 0, kl;
    for (int i = tid * run; i < min((tid + 1) * run, p.B); ++i) x += tiles_of<KT>(p, i, kl).y;
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
  const Runs runs(scan[THREADS] * cols, gridDim.x);
  int pos = runs.first(blockIdx.x);
  const int run_first = pos, end = blockIdx.x < runs.active ? runs.first(blockIdx.x + 1) : pos;
  if (scan[tid] * cols <= pos && pos < scan[tid + 1] * cols) {
    int base = scan[tid] * cols, b = tid * run, kl;
    for (;; ++b) {
      const int n = tiles_of<KT>(p, b, kl).y * cols;
      if (pos < base + n) break;
      base += n;
    }
    start_b = b, start_base = base;
  }
  // sequences without visible keys: their rows are 0
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    int kl;
    if (tiles_of<KT>(p, b, kl).y > 0) continue;
    uint32_t* o = reinterpret_cast<uint32_t*>(p.o + (int64_t)b * p.L * p.H * D);
    for (int64_t i = tid; i < (int64_t)p.L * p.H * D / 2; i += THREADS) o[i] = 0;
  }
  grid_dependency_wait();  // the new tokens are in the cache
  if (pos >= end) return;
  __syncthreads();
  int b = start_b, base = start_base;
  const uint32_t slot0 = smem_u32(ring) + warp * (STAGES * S::TILE);
  const float ninf = -INFINITY;

  while (pos < end) {
    int kv_len;
    const int2 tl = tiles_of<KT>(p, b, kv_len);
    const int nt = tl.y;
    if (pos >= base + nt * cols) {
      base += nt * cols;
      ++b;
      continue;
    }
    const int col = (pos - base) / nt;
    const int ta = (pos - base) - col * nt;    // first tile of this piece
    const int n = min(nt - ta, end - pos);     // its tiles
    const int hk = col / p.RT, rt = col - hk * p.RT;
    const int rows = min(ROWS, rows_all - rt * ROWS);
    const int64_t bh = (int64_t)b * p.Hkv + hk;
    const uint8_t* kb = p.k + bh * p.cap * D;
    const uint8_t* vb = p.v + bh * p.cap * D;
    const uint8_t* ksb = p.ks + bh * p.nblk;
    const uint8_t* vsb = p.vs + bh * p.nblk;
    const int my_n = (n - warp + WARPS - 1) / WARPS;                  // tiles of this warp: warp, warp + 4, ...
    const int key_first = (tl.x + ta + warp) * KT;

    auto load_tile = [&](int i) {
      const int key0 = key_first + i * (WARPS * KT);
      const uint32_t dst = slot0 + (i % STAGES) * S::TILE;
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int key = key0 + u * 16 + j * 8 + g;
          const bool ok = key < kv_len;
          const uint8_t* src = kb + (int64_t)(ok ? key : 0) * D + c * 16;
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
            cp16(dst + (u * 2 * HALVES + j * HALVES + h) * 512 + lane * 16, src + h * 64, ok);
        }
        const uint32_t vdst = dst + KT * D + u * 16 * D;
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const int key = key0 + u * 16 + (i4 >> 1) * 8 + 2 * c + (i4 & 1);
          const bool ok = key < kv_len;
          const uint8_t* src = vb + (int64_t)(ok ? key : 0) * D + g * VB;
          if constexpr (D == 128) cp16(vdst + i4 * 512 + lane * 16, src, ok);
          else cp_async_8(vdst + i4 * 256 + lane * 8, src, ok);
        }
      }
    };
    // scale bytes of a tile's keys: one a 16-key group, or one a key of this lane
    constexpr int NS = UNI ? U : 4 * U;
    int kbyte[NS], vbyte[NS];
    auto load_scales = [&](int i, int (&kx)[NS], int (&vx)[NS]) {
      const int key0 = key_first + i * (WARPS * KT);
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const int key = UNI ? key0 + s * 16 : key0 + (s >> 2) * 16 + ((s >> 1) & 1) * 8 + 2 * c + (s & 1);
        const bool ok = key < kv_len;
        kx[s] = ok ? ksb[key >> p.shift] : kMinScale;
        vx[s] = ok ? vsb[key >> p.shift] : kMinScale;
      }
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
      if (i < my_n) load_tile(i);
      cp_commit();
    }
    if (my_n > 0) load_scales(0, kbyte, vbyte);

    // ---- query rows g and g + 8 of the tile, scaled to f16
    uint32_t qa[D / 16][4];
    float rowf[2];
    int qpos[2];
#pragma unroll
    for (int r2 = 0; r2 < 2; ++r2) {
      const int r = rt * ROWS + g + r2 * 8;
      const bool ok = r < rows_all;
      const int gh = ok ? r / p.L : 0, i = ok ? r % p.L : 0;
      qpos[r2] = kv_len - p.L + i;
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
      rowf[r2] = __int_as_float((254 - field) << 23) * p.scale_log2;
#pragma unroll
      for (int h = 0; h < HALVES * 2; ++h) {
        const uint32_t ww[4] = {w[h].x, w[h].y, w[h].z, w[h].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float x = __uint_as_float(ww[k] << 16) * mul, y = __uint_as_float(ww[k] & 0xffff0000u) * mul;
          // elements (2k, 2k + 1) of 8: MMA step (k >> 1), its lower or upper k half
          qa[h * 2 + (k >> 1)][(k & 1) * 2 + r2] = pack_f16(x, y);
        }
      }
    }

    float m[2] = {ninf, ninf}, l[2] = {0.f, 0.f};
    float o[VB][4];
#pragma unroll
    for (int t = 0; t < VB; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;

    for (int i = 0; i < my_n; ++i) {
      if (i + STAGES - 1 < my_n) load_tile(i + STAGES - 1);
      cp_commit();
      int kx[NS], vx[NS];
#pragma unroll
      for (int s = 0; s < NS; ++s) kx[s] = kbyte[s], vx[s] = vbyte[s];
      if (i + 1 < my_n) load_scales(i + 1, kbyte, vbyte);
      cp_wait<STAGES - 1>();  // tile i has landed (a lane reads only what it copied itself)
      const unsigned char* buf = ring + warp * (STAGES * S::TILE) + (i % STAGES) * S::TILE;
      const int key0 = key_first + i * (WARPS * KT);
      // ---- S = Q K^T
      float s[2 * U][4];
#pragma unroll
      for (int j = 0; j < 2 * U; ++j) {
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          const uint4 w = *reinterpret_cast<const uint4*>(buf + (j * HALVES + h) * 512 + lane * 16);
          const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t b0, b1;
            widen4<INT8>(ww[k], b0, b1);
            mma_f16(s[j], qa[h * 4 + k], b0, b1);
          }
        }
      }
      // ---- t = s * f + log2 s_v, masked
      float lv[NS], isv[NS];
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        lv[x] = vx[x] == kBadScale ? __int_as_float(0x7fffffff) : (float)(vx[x] - 127);
        isv[x] = scale_inverse(min(vx[x], 253));
      }
      float f[2][NS];
#pragma unroll
      for (int x = 0; x < NS; ++x) {
        const float sk = scale_value(kx[x]);
        f[0][x] = rowf[0] * sk, f[1][x] = rowf[1] * sk;
      }
      // every row sees the whole tile
      const bool inner = key0 + KT <= kv_len && (p.right < 0 || key0 + KT - 1 <= kv_len - p.L + p.right) &&
                         (p.left < 0 || key0 >= kv_len - 1 - p.left);
      float mx[2] = {ninf, ninf};
#pragma unroll
      for (int j = 0; j < 2 * U; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r2 = e >> 1, x = UNI ? j >> 1 : j * 2 + (e & 1);
          s[j][e] = fmaf(s[j][e], f[r2][x], lv[x]);
          if (!inner) {
            const int key = key0 + j * 8 + 2 * c + (e & 1);
            const bool vis = key < kv_len && (p.right < 0 || key <= qpos[r2] + p.right) &&
                             (p.left < 0 || key >= qpos[r2] - p.left);
            if (!vis) s[j][e] = ninf;
          }
          mx[r2] = fmaxf(mx[r2], s[j][e]);
        }
      // ---- follow the maximum; O is rescaled rarely
      if (__any_sync(0xffffffffu, mx[0] > m[0] + 15.f || mx[1] > m[1] + 15.f)) {
#pragma unroll
        for (int r2 = 0; r2 < 2; ++r2) {
          float x = mx[r2];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          const float to = x > m[r2] + 15.f ? x - 8.f : m[r2];
          const float corr = to == m[r2] ? 1.f : ex2(m[r2] - to);
          m[r2] = to;
          l[r2] *= corr;
#pragma unroll
          for (int t = 0; t < VB; ++t) o[t][2 * r2] *= corr, o[t][2 * r2 + 1] *= corr;
        }
      }
      const float mu[2] = {m[0] == ninf ? 0.f : m[0], m[1] == ninf ? 0.f : m[1]};
#pragma unroll
      for (int j = 0; j < 2 * U; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r2 = e >> 1, x = UNI ? j >> 1 : j * 2 + (e & 1);
          s[j][e] = ex2(s[j][e] - mu[r2]);
          l[r2] = fmaf(s[j][e], isv[x], l[r2]);
        }
      // ---- O += P V
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t pa[4] = {pack_f16(s[2 * u][0], s[2 * u][1]), pack_f16(s[2 * u][2], s[2 * u][3]),
                                pack_f16(s[2 * u + 1][0], s[2 * u + 1][1]),
                                pack_f16(s[2 * u + 1][2], s[2 * u + 1][3])};
        uint32_t vw[4][VB / 4];
        const unsigned char* vbuf = buf + KT * D + u * 16 * D;
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          if constexpr (D == 128) {
            const uint4 w = *reinterpret_cast<const uint4*>(vbuf + i4 * 512 + lane * 16);
            vw[i4][0] = w.x, vw[i4][1] = w.y, vw[i4][2] = w.z, vw[i4][3] = w.w;
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(vbuf + i4 * 256 + lane * 8);
            vw[i4][0] = w.x, vw[i4][1] = w.y;
          }
        }
#pragma unroll
        for (int x = 0; x < VB / 4; ++x) {
          uint32_t b0[4], b1[4];  // f16 pairs of keys (2c, 2c + 1) and (2c + 8, 2c + 9) for columns 4x .. 4x + 3
          widen4<INT8>(__byte_perm(vw[0][x], vw[1][x], 0x5140), b0[0], b0[1]);
          widen4<INT8>(__byte_perm(vw[0][x], vw[1][x], 0x7362), b0[2], b0[3]);
          widen4<INT8>(__byte_perm(vw[2][x], vw[3][x], 0x5140), b1[0], b1[1]);
          widen4<INT8>(__byte_perm(vw[2][x], vw[3][x], 0x7362), b1[2], b1[3]);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_f16(o[4 * x + k], pa, b0[k], b1[k]);
        }
      }
    }
    cp_wait<0>();
#pragma unroll
    for (int r2 = 0; r2 < 2; ++r2) {
      l[r2] += __shfl_xor_sync(0xffffffffu, l[r2], 1);
      l[r2] += __shfl_xor_sync(0xffffffffu, l[r2], 2);
    }
    // ---- join the warps through shared memory.  o[t][.] holds columns n = 2c, 2c + 1 of MMA tile t,
    // which are head dims n * VB + t; kept as [row][t][n] until the end.
    __syncthreads();
    float* ow = reinterpret_cast<float*>(ring);
    if (c == 0) {
      wM[warp][g] = m[0], wM[warp][g + 8] = m[1];
      wL[warp][g] = l[0], wL[warp][g + 8] = l[1];
    }
#pragma unroll
    for (int t = 0; t < VB; ++t) {
      float* dst = ow + (warp * ROWS + g) * S::OROW + t * 8 + 2 * c;
      *reinterpret_cast<float2*>(dst) = make_float2(o[t][0], o[t][1]);
      *reinterpret_cast<float2*>(dst + 8 * S::OROW) = make_float2(o[t][2], o[t][3]);
    }
    __syncthreads();
    const bool whole = ta == 0 && n == nt;
    const int64_t slot = (int64_t)blockIdx.x * 2 + (pos != run_first);
    if (tid < ROWS) {
      float M = wM[0][tid];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) M = fmaxf(M, wM[w][tid]);
      float L = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = part_weight(wM[w][tid], wL[w][tid], M);
        L += f == 0.f ? 0.f : f * wL[w][tid];
        wM[w][tid] = f;
      }
      rL[tid] = L;
      if (!whole && tid < rows) *reinterpret_cast<float2*>(p.ml + (slot * ROWS + tid) * 2) = make_float2(M, L);
    }
    __syncthreads();
    for (int e = tid; e < rows * VB; e += THREADS) {  // (row, t): n = 0 .. 7
      const int r = e / VB, t = e % VB;
      float x[8] = {};
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = wM[w][r];
        if (f == 0.f) continue;
        const float4* src = reinterpret_cast<const float4*>(ow + (w * ROWS + r) * S::OROW + t * 8);
        const float4 u = src[0], v = src[1];
        x[0] += f * u.x, x[1] += f * u.y, x[2] += f * u.z, x[3] += f * u.w;
        x[4] += f * v.x, x[5] += f * v.y, x[6] += f * v.z, x[7] += f * v.w;
      }
      if (whole) {
        bf16* o = out_row(p, b, hk, rt * ROWS + r, D) + t;
        const float inv = rL[r] == 0.f ? 0.f : 1.f / rL[r];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k * VB] = __float2bfloat16(x[k] * inv);
      } else {
        float4* dst = reinterpret_cast<float4*>(p.part + (slot * ROWS + r) * D + t * 8);
        dst[0] = make_float4(x[0], x[1], x[2], x[3]);
        dst[1] = make_float4(x[4], x[5], x[6], x[7]);
      }
    }
    __syncthreads();  // the merge buffer is the ring
    pos += n;
  }
}

// Joins the partials of the columns that several CTAs share, in the order of the CTAs; one CTA a
// column.  Launched so that everything up to the wait overlaps attend_kernel.
template <int D>
__global__ void __launch_bounds__(THREADS) join_kernel(AttendParams p) {
  constexpr int KT = Shape<D>::KT, VB = D / 8, D4 = D / 4, MAXE = ROWS * D4 / THREADS;
  extern __shared__ float wt[];  // [partials][ROWS] weights
  __shared__ int red[WARPS];
  __shared__ float sL[ROWS];
  __shared__ float4 part[THREADS];
  const int tid = threadIdx.x;
  const int cols = p.Hkv * p.RT;
  const int b = blockIdx.x / cols, col = blockIdx.x - b * cols;
  int kl, all = 0, before = 0;
  for (int i = tid; i < p.B; i += THREADS) {
    const int n = tiles_of<KT>(p, i, kl).y;
    all += n;
    if (i < b) before += n;
  }
  const Runs runs(block_sum(all, red) * cols, p.grid);
  const int nt = tiles_of<KT>(p, b, kl).y;
  const int cf = block_sum(before, red) * cols + col * nt;
  grid_dependency_wait();
  if (nt == 0) return;
  const int c0 = runs.owner(cf), nc = runs.owner(cf + nt - 1) + 1 - c0;
  if (nc == 1) return;  // written by attend_kernel
  const int hk = col / p.RT, rt = col - hk * p.RT;
  const int rows = min(ROWS, (p.H / p.Hkv) * p.L - rt * ROWS);
  // the column is the first piece of every CTA but c0, and of c0 only if c0's run starts with it
  const bool late = runs.first(c0) != cf;
  auto slot = [&](int x) { return ((int64_t)c0 + x) * 2 + (x == 0 && late); };
  {  // rows' maxima, weights and sums: 8 threads a row
    const int r = tid >> 3;
    float M = -INFINITY, L = 0.f;
    if (r < rows)
      for (int x = tid & 7; x < nc; x += 8) M = fmaxf(M, __ldcg(p.ml + (slot(x) * ROWS + r) * 2));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (r < rows)
      for (int x = tid & 7; x < nc; x += 8) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.ml + (slot(x) * ROWS + r) * 2));
        const float f = part_weight(ml.x, ml.y, M);
        wt[x * ROWS + r] = f;
        if (f != 0.f) L += f * ml.y;
      }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if ((tid & 7) == 0) sL[r] = L;
  }
  __syncthreads();
  // O as float4 columns; with few rows, groups of threads take every groups-th partial
  const int n4 = rows * D4, groups = n4 >= THREADS ? 1 : THREADS / n4;
#pragma unroll
  for (int k = 0; k < MAXE; ++k) {
    if (k * THREADS >= n4) break;
    const int e = groups > 1 ? tid % n4 : k * THREADS + tid, first = groups > 1 ? tid / n4 : 0;
    const int r = e / D4;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (e < n4 && first < groups) {
#pragma unroll 8
      for (int x = first; x < nc; x += groups) {
        const float f = wt[x * ROWS + r];
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part + slot(x) * ROWS * D) + e);
        if (f != 0.f) a.x += f * v.x, a.y += f * v.y, a.z += f * v.z, a.w += f * v.w;
      }
    }
    if (groups > 1) {
      part[tid] = a;
      __syncthreads();
      if (tid < n4)
        for (int x = 1; x < groups; ++x) {
          const float4 v = part[x * n4 + tid];
          a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
        }
    }
    if (groups > 1 ? tid < n4 : e < n4) {
      const int tn = (e % D4) * 4;
      bf16* o = out_row(p, b, hk, rt * ROWS + r, D) + (tn & 7) * VB + (tn >> 3);
      const float inv = sL[r] == 0.f ? 0.f : 1.f / sL[r];
      o[0] = __float2bfloat16(a.x * inv), o[VB] = __float2bfloat16(a.y * inv);
      o[2 * VB] = __float2bfloat16(a.z * inv), o[3 * VB] = __float2bfloat16(a.w * inv);
    }
  }
}

// Up to this many query rows a KV head (heads of the group x new tokens) take the kernel above,
// whose 16-row tiles each walk the cache; more rows read the cache back to bf16 once and take
// the prefill kernel.
constexpr int kMaxRows = 64;

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
  if ((int64_t)G * L > kMaxRows) {
    auto opt = q.options();
    auto kb = torch::empty({c.B, c.cap, c.Hkv, c.D}, opt), vb = torch::empty({c.B, c.cap, c.Hkv, c.D}, opt);
    read(c, lens, extra, nullptr, 0, c.cap, 256, kb, vb, who);  // 256: more than a key tile of the prefill kernel
    auto used = (seqlens + extra).clamp_(0, c.cap);
    return fa_fwd(rows16(q) ? q : q.clone(at::MemoryFormat::Contiguous), kb, vb, c10::nullopt, c10::nullopt, used, L, c.cap, scale,
                  left, right)[0];
  }
  if (!rows16(q)) q = q.clone(at::MemoryFormat::Contiguous);
  AttendParams p{};
  p.q = (const bf16*)q.data_ptr();
  p.k = c.data[0], p.v = c.data[1], p.ks = c.scale[0], p.vs = c.scale[1];
  p.seqlens = lens;
  p.o = (bf16*)o.data_ptr();
  p.q_sb = q.stride(0), p.q_st = q.stride(1), p.q_sh = q.stride(2);
  p.B = c.B, p.L = L, p.H = H, p.Hkv = c.Hkv, p.RT = (G * L + ROWS - 1) / ROWS;
  p.cap = c.cap, p.nblk = c.nblk, p.shift = c.shift, p.extra = extra;
  p.left = (int)left, p.right = (int)right;
  p.scale_log2 = (float)(std::abs(scale) * 1.4426950408889634), p.sign = scale < 0 ? -1.f : 1.f;
  static int sms[64] = {0};
  if (!sms[c.device]) C10_CUDA_CHECK(cudaDeviceGetAttribute(&sms[c.device], cudaDevAttrMultiProcessorCount, c.device));
  const int per_sm = c.D == 64 ? Shape<64>::PER_SM : Shape<128>::PER_SM;
  const int kt = c.D == 64 ? Shape<64>::KT : Shape<128>::KT;
  int64_t span = c.cap;  // most keys a sequence can show
  if (left >= 0) span = std::min<int64_t>(span, left + L + kt);
  const int64_t columns = (int64_t)c.B * c.Hkv * p.RT;
  const int64_t want = (columns * ((span + kt - 1) / kt) + WARPS - 1) / WARPS;
  const int grid = (int)std::min<int64_t>(want, (int64_t)sms[c.device] * per_sm);
  TORCH_CHECK(columns * ((c.cap + kt - 1) / kt) <= INT32_MAX, who, ": too many sequences x heads x keys");
  // workspace: partials of at most two pieces a CTA
  const int64_t part = (int64_t)grid * 2 * ROWS * c.D, ml = (int64_t)grid * 2 * ROWS * 2;
  auto work = torch::empty({part + ml}, q.options().dtype(at::kFloat));
  p.part = work.data_ptr<float>();
  p.ml = p.part + part;
  p.grid = grid;
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  auto start = [&](auto kern, int blocks, int smem, bool overlap) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = blocks, cfg.blockDim = THREADS, cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr, cfg.numAttrs = overlap ? 1 : 0;
    C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
  };
  const bool uni = c.shift >= 4;
  auto launch = [&](auto kern, SmemOptIn& attr, int smem) {
    C10_CUDA_CHECK(attr.ensure(kern, smem));
    start(kern, grid, smem, extra > 0);  // the kernel before it is then append()'s
  };
  static SmemOptIn a[8];
#define KV8_CASE(d, i8, un) \
  if (c.D == d && c.int8 == i8 && uni == un) \
    launch(attend_kernel<d, i8, un>, a[(d == 128) * 4 + i8 * 2 + un], Shape<d>::SMEM)
  KV8_CASE(64, false, false);
  KV8_CASE(64, false, true);
  KV8_CASE(64, true, false);
  KV8_CASE(64, true, true);
  KV8_CASE(128, false, false);
  KV8_CASE(128, false, true);
  KV8_CASE(128, true, false);
  KV8_CASE(128, true, true);
#undef KV8_CASE
  const int weights = grid * ROWS * (int)sizeof(float);
  if (c.D == 64) start(join_kernel<64>, (int)columns, weights, true);
  else start(join_kernel<128>, (int)columns, weights, true);
  return o;
}

}  // namespace mykb
