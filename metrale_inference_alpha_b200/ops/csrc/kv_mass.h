// Arguments of the launchers of kv_mass.cu, kv_observe.cu and kv_evict.cu, mirrored field for field by ops/kv_mass.py, and what the kernels of a
// decode step with weights share.
#pragma once
#include "common.cuh"
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

struct MbMassArgs {
  const void* q;             // [rows, Hq, D] bf16, rows contiguous
  const void* k_cache;       // [blocks, block, Hkv, D] bf16 or e4m3
  const void* v_cache;
  const int* block_table;
  long long table_ld;
  const int* q_start;        // prompts only
  const int* q_len;
  const int* ctx_len;
  float* mass;               // [seqs, Hkv, columns], columns next to each other
  long long mass_seq, mass_head;
  void* out;                 // [seqs, Hq, D] bf16
  void* ws;
  size_t ws_bytes;
  const float* k_scale;
  const float* v_scale;
  uint32_t* status;
  long long num_blocks;
  long long q_rows;          // prompts only: rows of q
  int num_seqs, Hq, Hkv, D, block_size, fp8, max_ctx, max_q_len, last, sm_count;
  float scale;
};

struct MbEvictArgs {
  const float* mass;
  long long mass_seq, mass_head;
  float* mass_out;
  long long out_seq, out_head;
  const int* ctx_len;
  int* kept;                 // [seqs, Hkv, keep]
  int* new_len;              // [seqs]
  int* first;                // [seqs, Hkv]: rows in front of this one stay where they are
  const int* block_table;
  long long table_ld;
  const int* dst_table;
  long long dst_ld;
  void* k_cache;
  void* v_cache;
  long long num_blocks;
  uint32_t* status;
  int* slots;                // [seqs, Hkv, keep]: kept rows' places in the cache
  int num_seqs, Hkv, keep, recent, max_ctx, block_size, row_bytes, in_place, block_shift;   // the launcher sets the shift
  unsigned block_magic;      // and this: a division by block_size
};

// as ops/kv_mass.py packs them
static_assert(sizeof(MbMassArgs) == 200, "field by field in ops/kv_mass.py too");
static_assert(sizeof(MbEvictArgs) == 192, "field by field in ops/kv_mass.py too");

namespace mbm {

constexpr int kMaxParts = 32;
// A sequence's partitions, from its own length alone: part_tokens each, but at most kMaxParts of them.
__host__ __device__ __forceinline__ int part_size(int len, int part_tokens) {
  const int even = ((len + kMaxParts - 1) / kMaxParts + 63) & ~63;
  return even > part_tokens ? even : part_tokens;
}
__host__ __device__ __forceinline__ int part_count(int len, int part_tokens) {
  const int P = part_size(len, part_tokens);
  return len <= P ? 1 : (len + P - 1) / P;
}

// Workspace of a decode step: logits in the log2 domain [seqs, Hkv, G, ld], what a partition's outputs are relative to and their sums
// [seqs * Hq, parts], the outputs themselves [seqs * Hq, parts, D].
struct DecodeWs {
  long long ld;
  int parts;
  size_t z, ml, o, bytes;    // byte offsets, and the whole
};
inline DecodeWs decode_ws(int seqs, int Hq, int D, int max_ctx, int part_tokens) {
  DecodeWs w;
  w.ld = (max_ctx + 63) & ~63ll;
  const int n = (max_ctx + part_tokens - 1) / part_tokens;
  w.parts = n < 1 ? 1 : n > kMaxParts ? kMaxParts : n;
  const size_t rows = (size_t)seqs * Hq;
  w.z = 0;
  w.o = rows * w.ld * 4;
  w.ml = w.o + rows * w.parts * D * 4;
  w.bytes = w.ml + rows * w.parts * 8;
  return w;
}

// cached tokens of a sequence; a length beyond what the call was sized for is reported and cut
__device__ __forceinline__ int context(const int* ctx_len, int s, int max_ctx, uint32_t* status) {
  const int n = ctx_len[s];
  if (n > max_ctx) {
    if (status && threadIdx.x == 0) atomicCAS(status, 0u, MB_ST_BOUNDS);
    return max_ctx;
  }
  return max(n, 0);
}
// flat slot of row j of a sequence; a block that the cache does not have is reported and read as block 0
__device__ __forceinline__ long long slot_of(const int* table, int j, int block_size, long long num_blocks, uint32_t* status) {
  const int bi = j / block_size;
  int b = __ldg(table + bi);
  if ((unsigned)b >= (unsigned long long)num_blocks) {
    if (status) atomicCAS(status, 0u, MB_ST_BOUNDS);
    b = 0;
  }
  return (long long)b * block_size + (j - bi * block_size);
}

}  // namespace mbm

// attention_decode_mass.cu
bool mb_decode_mass_serves(const MbMassArgs& a);
int mb_decode_mass(const MbMassArgs& m, const mbm::DecodeWs& w, int part_tokens, cudaStream_t stream);
