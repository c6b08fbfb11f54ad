// Arguments of the launchers of shared_attn.cu, attn_merge.cu and mla_prompt.cu, mirrored field for field by ops/shared_attn.py and ops/mla_prompt.py.
#pragma once
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

struct MbSharedArgs {
  const void* q;             // [seqs * q_len, Hq, D] bf16
  const void* k_cache;       // [blocks, block, Hkv, D] bf16 or e4m3
  const void* v_cache;
  const int* prefix_table;   // [groups, blocks of a prefix]
  long long prefix_ld;
  const int* prefix_len;     // [groups]
  const int* group_start;    // [groups + 1]
  const int* block_table;    // [seqs, blocks of a sequence's own]
  long long table_ld;
  const int* ctx_len;        // [seqs]
  void* out;                 // [seqs * q_len, Hq, D] bf16
  float* lse;                // [seqs * q_len, Hq], or null
  void* ws;
  size_t ws_bytes;
  const float* k_scale;
  const float* v_scale;
  uint32_t* status;
  long long num_blocks;
  int num_seqs, q_len, groups, Hq, Hkv, D, block_size, fp8, max_prefix, max_ctx, sm_count;
  float scale;
};

constexpr int kMergeParts = 16;

struct MbMergeArgs {
  const void* outs[kMergeParts];
  const float* lses[kMergeParts];
  void* out;
  float* lse;
  long long rows;            // of tokens and heads
  int parts, dim, f32, sm_count;
};

struct MbMlaPromptArgs {
  const void* q;             // [rows, H, 192] bf16
  const void* cache;         // [blocks, block, 1, 576] bf16
  const int* block_table;    // [seqs, blocks of a sequence]
  long long table_ld;
  const int* q_start;
  const int* q_len;
  const int* ctx_len;
  const void* w;             // [H, 256, 512] bf16
  void* out;                 // [rows, H, 128] bf16
  void* ws;
  size_t ws_bytes;
  uint32_t* status;
  long long num_blocks, q_rows, kv_rows;     // kv_rows: expanded rows, a multiple of 128
  int num_seqs, H, block_size, max_q_len, max_ctx;
  int each;                  // heads that are expanded at once
  int sm_count, gemm_flags;
  float scale;
};

// as the callers pack them
static_assert(sizeof(MbSharedArgs) == 192, "field by field in ops/shared_attn.py too");
static_assert(sizeof(MbMergeArgs) == 296, "field by field in ops/shared_attn.py too");
static_assert(sizeof(MbMlaPromptArgs) == 160, "field by field in ops/mla_prompt.py too");
