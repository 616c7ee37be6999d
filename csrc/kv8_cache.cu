// Writing and reading the 8-bit key/value cache (formats and scales: kv8.cuh).
//
// Both are one pass over their data, bound by the loads that short-lived CTAs keep in flight and, for
// a decode step's few tokens, by launch latency.  8 x 2048 tokens of 4 heads of 128 (B200): written
// 13.5 us (50 MB, 0.57 of the copy bandwidth), read back 12.3 us (50 MB, 0.63), each timed alone
// with a cold L2; one token for each of 8 sequences 4.7 us.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "kv8.cuh"
#include "kv8_host.h"

namespace mykb {
namespace kv8 {

struct AppendParams {
  const bf16* src[2];         // new keys, values (B, L, Hkv, D), last dim contiguous
  uint8_t* data[2];           // caches (B, Hkv, cap, D)
  uint8_t* scale[2];          // (B, Hkv, nblk)
  const int* seqlens;         // (B) tokens held before the call
  int64_t sb[2], st[2], sh[2];
  int B, L, Hkv, cap, nblk, shift;  // block = 1 << shift tokens
  int span;                   // blocks that L new tokens can touch
};

// WPU warps per (sequence, head, touched block, keys or values): largest magnitude of the new
// rows of the block, scale byte, quantised rows.  A block that already holds tokens keeps the
// larger of its scale and the one the new rows need; if it grows, the old rows are shifted to
// it (rounding once).  Up to kHeld 16-byte vectors a lane stay in registers between the two
// passes, longer blocks are read again (from L1 / L2).  One warp a unit up to 32 kHeld vectors
// (16 tokens of 128), else four (13 x 1000 tokens in blocks of 64: 24 us with the read back instead of 33).
constexpr int kAppendWarps = 4, kHeld = 8;

template <int D, bool INT8, int WPU>
__global__ void __launch_bounds__(kAppendWarps * 32) append_kernel(AppendParams p) {
  constexpr int STEP = 32 * WPU;  // threads of a unit
  // a kernel that attends to the new tokens may start its prologue (and waits for the rest)
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane = threadIdx.x % STEP;
  int64_t u = WPU == 1 ? (int64_t)blockIdx.x * kAppendWarps + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  if (u >= (int64_t)p.B * p.Hkv * p.span * 2) return;
  const int kv = (int)(u & 1);
  u >>= 1;
  const int nb = (int)(u % p.span);
  const int64_t bh = u / p.span;
  const int b = (int)(bh / p.Hkv), h = (int)(bh % p.Hkv);
  const int len = max(p.seqlens[b], 0);
  const int64_t end = min((int64_t)len + p.L, (int64_t)p.cap);
  const int blk = (len >> p.shift) + nb;
  const int64_t first = (int64_t)blk << p.shift;
  const int64_t lo = max(first, (int64_t)len), hi = min(first + (1 << p.shift), end);  // new rows of this block
  if (lo >= hi) return;
  constexpr int VR = D / 8;  // vectors a row
  const int nvec = (int)(hi - lo) * VR;
  const bf16* src = p.src[kv] + b * p.sb[kv] + (lo - len) * p.st[kv] + h * p.sh[kv];
  uint8_t* dst = p.data[kv] + (bh * p.cap + lo) * D;
  const int64_t st = p.st[kv];
  auto load = [&](int i) { return __ldg(reinterpret_cast<const uint4*>(src + (i / VR) * st + (i % VR) * 8)); };
  uint4 held[kHeld];
  uint32_t amax2 = 0;  // two 16-bit maxima
  auto look = [&](const uint4& v) {
    amax2 = __vmaxu2(amax2, v.x & 0x7fff7fffu);
    amax2 = __vmaxu2(amax2, v.y & 0x7fff7fffu);
    amax2 = __vmaxu2(amax2, v.z & 0x7fff7fffu);
    amax2 = __vmaxu2(amax2, v.w & 0x7fff7fffu);
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (lane + STEP * i < nvec) held[i] = load(lane + STEP * i);
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (lane + STEP * i < nvec) look(held[i]);
  for (int i = lane + STEP * kHeld; i < nvec; i += STEP) look(load(i));
  uint32_t amax = __reduce_max_sync(0xffffffffu, max(amax2 & 0xffffu, amax2 >> 16));
  uint8_t* sp = p.scale[kv] + bh * p.nblk + blk;
  const int old = lo > first ? *sp : 0;
  if constexpr (WPU > 1) {  // (also: every thread has read the old scale)
    __shared__ uint32_t wmax[WPU];
    if ((threadIdx.x & 31) == 0) wmax[threadIdx.x >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WPU; ++w) amax = max(amax, wmax[w]);
  }
  const int need = scale_byte<INT8>(amax);
  int byte = need;
  if (lo > first) {
    byte = max(old, need);
    if (byte > old && byte != kBadScale) {  // the block's maximum rose: old rows to the new scale
      const float f = byte - old > 126 ? 0.f : __int_as_float((127 - (byte - old)) << 23);
      uint2* rows = reinterpret_cast<uint2*>(p.data[kv] + (bh * p.cap + first) * D);
      for (int i = lane; i < (int)(lo - first) * VR; i += STEP) {
        const uint2 w = rows[i];
        uint32_t r[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t a, c;
          widen4<INT8>(k ? w.y : w.x, a, c);
          const float2 x = __half22float2(*reinterpret_cast<__half2*>(&a));
          const float2 y = __half22float2(*reinterpret_cast<__half2*>(&c));
          r[k] = quant2<INT8>(x.x * f, x.y * f) | (quant2<INT8>(y.x * f, y.y * f) << 16);
        }
        rows[i] = make_uint2(r[0], r[1]);
      }
    }
  }
  __syncwarp();
  if (lane == 0) *sp = (uint8_t)byte;
  const bool bad = byte == kBadScale;
  const float inv = bad ? 0.f : scale_inverse(byte);
  auto store = [&](int i, const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = __uint_as_float(w[k] << 16), c = __uint_as_float(w[k] & 0xffff0000u);
      r[k] = bad ? 0u : quant2<INT8>(a * inv, c * inv);
    }
    *reinterpret_cast<uint2*>(dst + (int64_t)i * 8) = make_uint2(r[0] | (r[1] << 16), r[2] | (r[3] << 16));
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (lane + STEP * i < nvec) store(lane + STEP * i, held[i]);
  for (int i = lane + STEP * kHeld; i < nvec; i += STEP) store(i, load(i));
}

struct ReadParams {
  const uint8_t* data[2];   // [0] keys, [1] values
  const uint8_t* scale[2];
  bf16* out[2];          // (B, length, Hkv, D)
  const int* seqlens;    // (B) tokens held, less `extra`
  const int* start;      // (B) or null
  int start0, extra;
  int B, Hkv, cap, nblk, shift, length;
  int pad;               // >= 0: for the prefill kernel (see read() in kv8_host.h)
};

// 16 values a thread and step (16 bytes in, 32 out).  A CTA walks kReadTokens tokens of one
// (sequence, head), so that reads are contiguous and writes whole rows of 128 or 256 bytes.
constexpr int kReadThreads = 256, kReadSteps = 4;

template <int D, bool INT8>
__global__ void __launch_bounds__(kReadThreads) read_kernel(ReadParams p) {
  constexpr int CR = D / 16, TOK = kReadThreads * kReadSteps / CR;
  const int kv = blockIdx.y;
  const int tiles = (p.length + TOK - 1) / TOK;
  const int tile = blockIdx.x % tiles;
  const int64_t bh = blockIdx.x / tiles;
  const int b = (int)(bh / p.Hkv), h = (int)(bh % p.Hkv);
  const int64_t held = min((int64_t)max(p.seqlens[b], 0) + p.extra, (int64_t)p.cap);
  const int64_t base = p.start ? p.start[b] : p.start0;
  const int t0 = tile * TOK;
  if (p.pad >= 0 && base + t0 >= held + p.pad) return;
  const uint8_t* src = (kv ? p.data[1] : p.data[0]) + bh * p.cap * D;
  const uint8_t* sc = (kv ? p.scale[1] : p.scale[0]) + bh * p.nblk;
  bf16* out = (kv ? p.out[1] : p.out[0]) + ((int64_t)b * p.length * p.Hkv + h) * D;
  const uint8_t* sc2 = (kv ? p.scale[0] : p.scale[1]) + bh * p.nblk;  // of the other tensor
  uint4 w[kReadSteps];
  int sb[kReadSteps];
#pragma unroll
  for (int s = 0; s < kReadSteps; ++s) {
    const int e = s * kReadThreads + threadIdx.x, t = t0 + e / CR;
    const int64_t pos = base + t;
    w[s] = make_uint4(0, 0, 0, 0);
    sb[s] = kMinScale;
    if (t < p.length && pos >= 0 && pos < held) {
      w[s] = __ldcs(reinterpret_cast<const uint4*>(src + pos * D + (e % CR) * 16));
      sb[s] = sc[pos >> p.shift];
      if (p.pad >= 0) {
        if (kv && sb[s] == kBadScale) sb[s] = kMinScale, w[s] = make_uint4(0, 0, 0, 0);
        if (!kv && sc2[pos >> p.shift] == kBadScale) sb[s] = kBadScale;
      }
    }
  }
#pragma unroll
  for (int s = 0; s < kReadSteps; ++s) {
    const int e = s * kReadThreads + threadIdx.x, t = t0 + e / CR;
    if (t >= p.length) continue;
    const float f = scale_value(sb[s]);
    const uint32_t in[4] = {w[s].x, w[s].y, w[s].z, w[s].w};
    uint32_t r[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t a, c;
      widen4<INT8>(in[k], a, c);
      const float2 x = __half22float2(*reinterpret_cast<__half2*>(&a));
      const float2 y = __half22float2(*reinterpret_cast<__half2*>(&c));
      r[2 * k] = pack_bf16x2(x.x * f, x.y * f);
      r[2 * k + 1] = pack_bf16x2(y.x * f, y.y * f);
    }
    uint4* o = reinterpret_cast<uint4*>(out + (int64_t)t * p.Hkv * D + (e % CR) * 16);
    o[0] = make_uint4(r[0], r[1], r[2], r[3]);
    o[1] = make_uint4(r[4], r[5], r[6], r[7]);
  }
}

Cache check_cache(const torch::Tensor& keys, const torch::Tensor& values, const torch::Tensor& key_scales,
                  const torch::Tensor& value_scales, int64_t block, const char* who) {
  TORCH_CHECK(keys.is_cuda() && keys.dim() == 4 && keys.sizes() == values.sizes() && keys.is_contiguous() &&
                  values.is_contiguous(),
              who, ": contiguous (B, Hkv, capacity, D) caches on one GPU");
  TORCH_CHECK((keys.scalar_type() == at::kFloat8_e4m3fn || keys.scalar_type() == at::kChar) &&
                  values.scalar_type() == keys.scalar_type(),
              who, ": caches of float8_e4m3fn or int8");
  TORCH_CHECK(block >= 1 && block <= 1024 && (block & (block - 1)) == 0, who,
              ": block must be a power of two up to 1024; got ", std::to_string(block));
  Cache c{};
  TORCH_CHECK(keys.size(0) <= INT32_MAX && keys.size(1) <= 65535 && keys.size(2) <= INT32_MAX / 2, who,
              ": cache dimensions too large");
  c.B = keys.size(0), c.Hkv = keys.size(1), c.cap = keys.size(2), c.D = keys.size(3);
  TORCH_CHECK(c.D == 64 || c.D == 128, who, ": head_dim 64 or 128; got ", std::to_string(c.D));
  c.nblk = (int)((c.cap + block - 1) / block);
  for (const torch::Tensor* s : {&key_scales, &value_scales})
    TORCH_CHECK(s->scalar_type() == at::kByte && s->is_contiguous() && s->dim() == 3 && s->size(0) == c.B &&
                    s->size(1) == c.Hkv && s->size(2) == c.nblk,
                who, ": contiguous uint8 scales (B, Hkv, ceil(capacity / block))");
  for (const torch::Tensor* s : {&values, &key_scales, &value_scales})
    TORCH_CHECK(s->device() == keys.device(), who, ": cache tensors on one GPU");
  TORCH_CHECK((((uintptr_t)keys.data_ptr() | (uintptr_t)values.data_ptr()) & 15) == 0, who,
              ": caches aligned to 16 bytes");
  c.int8 = keys.scalar_type() == at::kChar;
  c.shift = 0;
  while ((1 << c.shift) < block) ++c.shift;
  c.data[0] = (uint8_t*)keys.data_ptr(), c.data[1] = (uint8_t*)values.data_ptr();
  c.scale[0] = key_scales.data_ptr<uint8_t>(), c.scale[1] = value_scales.data_ptr<uint8_t>();
  return c;
}

void check_lens(const torch::Tensor& t, const Cache& c, const torch::Tensor& keys, const char* who) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == c.B && t.is_contiguous() &&
                  t.device() == keys.device(),
              who, ": int32 lengths (B) on the cache's GPU");
}

template <typename P, typename F64, typename F64I, typename F128, typename F128I>
static void pick(const Cache& c, P&& launch, F64 f64, F64I f64i, F128 f128, F128I f128i) {
  if (c.D == 64) c.int8 ? launch(f64i) : launch(f64);
  else c.int8 ? launch(f128i) : launch(f128);
}

void append(const Cache& c, torch::Tensor k, torch::Tensor v, const int* seqlens, const char* who) {
  for (const torch::Tensor* t : {&k, &v})
    TORCH_CHECK(t->is_cuda() && t->scalar_type() == at::kBFloat16 && t->dim() == 4 && t->size(0) == c.B &&
                    t->size(2) == c.Hkv && t->size(3) == c.D,
                who, ": new keys / values (B, new, Hkv, D) in bf16");
  TORCH_CHECK(k.size(1) == v.size(1), who, ": as many new keys as values");
  TORCH_CHECK(k.device() == v.device() && k.get_device() == c.device, who, ": new keys / values on the cache's GPU");
  TORCH_CHECK(k.size(1) <= (1 << 30), who, ": too many new tokens");
  const int L = (int)k.size(1);
  if (L == 0 || c.B == 0 || c.Hkv == 0 || c.cap == 0) return;
  if (!rows16(k)) k = k.clone(at::MemoryFormat::Contiguous);
  if (!rows16(v)) v = v.clone(at::MemoryFormat::Contiguous);
  AppendParams p{};
  const torch::Tensor* src[2] = {&k, &v};
  for (int i = 0; i < 2; ++i) {
    p.src[i] = (const bf16*)src[i]->data_ptr();
    p.sb[i] = src[i]->stride(0), p.st[i] = src[i]->stride(1), p.sh[i] = src[i]->stride(2);
    p.data[i] = c.data[i], p.scale[i] = c.scale[i];
  }
  p.seqlens = seqlens;
  p.B = c.B, p.L = L, p.Hkv = c.Hkv, p.cap = c.cap, p.nblk = c.nblk, p.shift = c.shift;
  p.span = ((L - 2) >> c.shift) + 2;  // 1 for L == 1
  if (L == 1) p.span = 1;
  const int64_t units = (int64_t)c.B * c.Hkv * p.span * 2;
  const bool wide = (int64_t)std::min(L, 1 << c.shift) * (c.D / 8) > 32 * kHeld;
  const int64_t grid = wide ? units : (units + kAppendWarps - 1) / kAppendWarps;
  TORCH_CHECK(grid <= INT32_MAX, who, ": too many blocks to write");
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  auto launch = [&](auto kern) { kern<<<(int)grid, kAppendWarps * 32, 0, st>>>(p); };
  if (wide)
    pick(c, launch, append_kernel<64, false, kAppendWarps>, append_kernel<64, true, kAppendWarps>,
         append_kernel<128, false, kAppendWarps>, append_kernel<128, true, kAppendWarps>);
  else
    pick(c, launch, append_kernel<64, false, 1>, append_kernel<64, true, 1>, append_kernel<128, false, 1>,
         append_kernel<128, true, 1>);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void read(const Cache& c, const int* seqlens, int extra, const int* start, int start0, int length, int pad,
          torch::Tensor& k, torch::Tensor& v, const char* who) {
  if (k.numel() == 0) return;
  ReadParams p{};
  for (int i = 0; i < 2; ++i) p.data[i] = c.data[i], p.scale[i] = c.scale[i];
  p.out[0] = (bf16*)k.data_ptr(), p.out[1] = (bf16*)v.data_ptr();
  p.seqlens = seqlens, p.start = start, p.start0 = start0, p.extra = extra;
  p.B = c.B, p.Hkv = c.Hkv, p.cap = c.cap, p.nblk = c.nblk, p.shift = c.shift, p.length = length, p.pad = pad;
  const int tok = kReadThreads * kReadSteps / (c.D / 16);
  const int64_t grid = (int64_t)c.B * c.Hkv * ((length + tok - 1) / tok);
  TORCH_CHECK(grid <= INT32_MAX, who, ": too many tokens to read");
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  auto launch = [&](auto kern) { kern<<<dim3((int)grid, 2), kReadThreads, 0, st>>>(p); };
  pick(c, launch, read_kernel<64, false>, read_kernel<64, true>, read_kernel<128, false>, read_kernel<128, true>);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace kv8

void kv8_append(torch::Tensor keys, torch::Tensor values, torch::Tensor key_scales, torch::Tensor value_scales,
                int64_t block, torch::Tensor k, torch::Tensor v, torch::Tensor seqlens) {
  c10::cuda::OptionalCUDAGuard guard;
  if (keys.is_cuda()) guard.set_device(keys.device());
  kv8::Cache c = kv8::check_cache(keys, values, key_scales, value_scales, block, "kv8_append");
  c.device = keys.get_device();
  kv8::check_lens(seqlens, c, keys, "kv8_append");
  kv8::append(c, k, v, seqlens.data_ptr<int>(), "kv8_append");
}

std::vector<torch::Tensor> kv8_read(torch::Tensor keys, torch::Tensor values, torch::Tensor key_scales,
                                    torch::Tensor value_scales, int64_t block, torch::Tensor seqlens,
                                    c10::optional<torch::Tensor> start, int64_t start0, int64_t length) {
  c10::cuda::OptionalCUDAGuard guard;
  if (keys.is_cuda()) guard.set_device(keys.device());
  kv8::Cache c = kv8::check_cache(keys, values, key_scales, value_scales, block, "kv8_read");
  c.device = keys.get_device();
  kv8::check_lens(seqlens, c, keys, "kv8_read");
  if (start.has_value()) kv8::check_lens(*start, c, keys, "kv8_read");
  TORCH_CHECK(length >= 0 && length <= INT32_MAX / 2 && start0 >= 0 && start0 <= INT32_MAX / 2,
              "kv8_read: start and length must be non-negative");
  auto opt = keys.options().dtype(at::kBFloat16);
  auto k = torch::empty({c.B, length, c.Hkv, c.D}, opt), v = torch::empty({c.B, length, c.Hkv, c.D}, opt);
  kv8::read(c, seqlens.data_ptr<int>(), 0, start.has_value() ? start->data_ptr<int>() : nullptr, (int)start0,
            (int)length, -1, k, v, "kv8_read");
  return {k, v};
}

}  // namespace mykb
