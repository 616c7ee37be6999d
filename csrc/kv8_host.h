// Host-side view of an 8-bit key/value cache, shared by kv8_cache.cu and kv8_attention.cu.
#pragma once

#include <torch/extension.h>

namespace mykb {
namespace kv8 {

struct Cache {
  uint8_t* data[2];   // keys, values (B, Hkv, cap, D)
  uint8_t* scale[2];  // (B, Hkv, nblk)
  int B, Hkv, cap, D, nblk, shift, device;
  bool int8;
};

// bf16 (B, tokens, heads, D) whose rows 16-byte loads can read in place.
inline bool rows16(const torch::Tensor& t) {
  return t.stride(3) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && t.stride(2) % 8 == 0 &&
         ((uintptr_t)t.data_ptr() & 15) == 0;
}

// Checks the cache's tensors; `who` starts the error messages.
Cache check_cache(const torch::Tensor& keys, const torch::Tensor& values, const torch::Tensor& key_scales,
                  const torch::Tensor& value_scales, int64_t block, const char* who);
void check_lens(const torch::Tensor& t, const Cache& c, const torch::Tensor& keys, const char* who);

// Quantises k / v (B, L, Hkv, D) into the cache at seqlens[b] (tokens past the capacity are dropped).
void append(const Cache& c, torch::Tensor k, torch::Tensor v, const int* seqlens, const char* who);

// bf16 copies (B, length, Hkv, D) of tokens start[b] (or start0) onward; tokens from seqlens[b] + extra on are 0.
// pad >= 0: for an attention kernel that multiplies masked values by 0: the part of the copy that lies more
// than `pad` tokens past them is left unwritten, and a block marked as bad in either tensor gets NaN keys (whose
// scores the mask replaces) and values of 0 instead of NaN.
void read(const Cache& c, const int* seqlens, int extra, const int* start, int start0, int length, int pad,
          torch::Tensor& k, torch::Tensor& v, const char* who);

}  // namespace kv8
}  // namespace mykb
