// Decode attention that leaves its partitions: the kernel of attention_decode.cu for one token at a time of a sequence, whose outputs, maxima and sums are joined
// with those of a prefix by shared_attn.cu. Several new tokens of a sequence read its rows once each, which L2 holds: behind a long prefix what is a
// sequence's own is the smaller part.
// Weights go into the product with V as bf16, or f16 with an e4m3 cache, since the matrix units take no more, as in plain attention: off by half a step each,
// which the bf16 result hides. Everything else is 32 bits.
#include "attention_decode.cuh"
#include "attention_decode_parts.h"

int mb_decode_parts(const MbSharedArgs& m, int tok0, int tokens, float* o, float* ml, int parts, bool late, cudaStream_t stream) {
  AttnDecodeArgs a{};
  a.k_cache = m.k_cache; a.v_cache = m.v_cache;
  a.num_seqs = tokens; a.max_q_len = 1; a.Hq = m.Hq; a.Hkv = m.Hkv; a.block_size = m.block_size; a.num_blocks = m.num_blocks;
  a.sm_count = m.sm_count; a.early = late;
  DecodeParams p{};
  p.q = reinterpret_cast<const __nv_bfloat16*>(m.q) + (size_t)tok0 * m.Hq * m.D;
  p.block_table = m.block_table; p.max_blocks = (int)m.table_ld; p.ctx_len = m.ctx_len;
  p.num_seqs = tokens; p.Hq = m.Hq; p.Hkv = m.Hkv; p.group = m.Hq / m.Hkv; p.per = m.q_len; p.tok0 = tok0;
  p.block_size = m.block_size;
  p.block_shift = (m.block_size & (m.block_size - 1)) == 0 ? 31 - __builtin_clz(m.block_size) : -1;
  p.num_blocks = m.num_blocks; p.scale = m.scale; p.k_scale = m.k_scale; p.v_scale = m.v_scale;
  p.status = m.status;
  p.part_tokens = mbs::part_tokens_of(m.Hkv, m.D); p.parts = parts;
  p.part_o = o; p.part_ml = reinterpret_cast<float2*>(ml); p.max_ctx = m.max_ctx;
  p.box_bits = 0;
  while (m.block_size % (kSlice >> p.box_bits)) ++p.box_bits;
  auto run = [&](auto d, auto eight) {
    constexpr int kMost = d.value == 256 ? 16 : 32;          // query rows that the kernel takes
    auto go = [&](auto nt) { return launch<d.value, eight.value, nt.value, 2>(a, p, stream); };
    const int takes = (p.group + kMost - 1) / kMost, each = (p.group + takes - 1) / takes;
    for (p.group0 = 0; p.group0 < p.group; p.group0 += each) {
      p.G = min(each, p.group - p.group0);
      a.Hq = p.G * a.Hkv;
      p.g_magic = 1;                                         // one token a sequence: r / G is 0
      int rc;
      if (p.G <= 8) rc = go(std::integral_constant<int, 1>{});
      else if constexpr (d.value == 256) rc = go(std::integral_constant<int, 2>{});
      else rc = p.G <= 16 ? go(std::integral_constant<int, 2>{}) : p.G <= 24 ? go(std::integral_constant<int, 3>{}) : go(std::integral_constant<int, 4>{});
      if (rc) return rc;
    }
    return 0;
  };
  auto by_dim = [&](auto eight) {
    return m.D == 64 ? run(std::integral_constant<int, 64>{}, eight) : m.D == 128 ? run(std::integral_constant<int, 128>{}, eight)
                                                                                  : run(std::integral_constant<int, 256>{}, eight);
  };
  return m.fp8 ? by_dim(std::true_type{}) : by_dim(std::false_type{});
}
