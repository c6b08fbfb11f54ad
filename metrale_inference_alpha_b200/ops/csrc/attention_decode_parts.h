// Decode attention that leaves its partitions' outputs, maxima and sums (attention_decode_parts.cu), called by shared_attn.cu for what sequences have of their own.
#pragma once
#include "shared_attn.h"

namespace mbs {
// most tokens of a launch
constexpr int kMaxTokens = 1024;
// cached tokens of a partition, partitions of the longest sequence; sequences of n tokens have part_count(n) of them
// (as in attention_decode.cu and kv_mass.cu, where both sides of the line are measured)
__host__ __device__ __forceinline__ int part_tokens_of(int Hkv, int D) { return Hkv >= 8 || (D == 256 && Hkv >= 2) ? 1024 : 512; }
constexpr int kMaxOwnParts = 32;
__host__ __device__ __forceinline__ int own_part_count(int len, int part_tokens) {
  const int even = ((len + kMaxOwnParts - 1) / kMaxOwnParts + 63) & ~63, size = even > part_tokens ? even : part_tokens;
  return len <= size ? 1 : (len + size - 1) / size;
}
}  // namespace mbs

// Tokens [tok0, tok0 + tokens) of the batch: outputs [tokens * Hq, parts, D] relative to 2^maximum, maxima (log2 domain) and sums [tokens * Hq, parts].
// `late`: the kernel in front has waited for what stands before it, and this one waits for it at its end only.
int mb_decode_parts(const MbSharedArgs& a, int tok0, int tokens, float* o, float* ml, int parts, bool late, cudaStream_t stream);
