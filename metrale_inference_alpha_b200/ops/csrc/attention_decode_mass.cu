// Decode attention that leaves its logits: the kernel of attention_decode.cu for one new token a sequence, called by mb_attn_mass for the
// calls that it serves. Beside attention itself a unit writes 4 bytes a token and query row; the join of kv_mass.cu makes weights of them.
// Logits, maxima, sums and outputs are 32 bits. Weights go into the product with V as bf16, or f16 with an e4m3 cache, since the matrix units take no more, as in
// plain attention: off by half a step each, which the bf16 result hides; the mass is made of the 32-bit logits.
#include "attention_decode.cuh"
#include "kv_mass.h"

bool mb_decode_mass_serves(const MbMassArgs& a) {
  const uintptr_t al = reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache) | reinterpret_cast<uintptr_t>(a.q);
  // a TMA box begins on 128 bytes of shared memory: rows of 64 bytes come two at least
  return (a.D > 64 || !a.fp8 || a.block_size % 2 == 0) && a.num_seqs <= kMaxSeqs && !(al & 15) &&
         a.num_blocks * a.block_size < (1ll << 31) && a.table_ld < (1ll << 31);
}

int mb_decode_mass(const MbMassArgs& m, const mbm::DecodeWs& w, int part_tokens, cudaStream_t stream) {
  AttnDecodeArgs a{};
  a.k_cache = m.k_cache; a.v_cache = m.v_cache;
  a.num_seqs = m.num_seqs; a.max_q_len = 1; a.Hq = m.Hq; a.Hkv = m.Hkv; a.block_size = m.block_size; a.num_blocks = m.num_blocks;
  a.sm_count = m.sm_count;
  uint8_t* ws = reinterpret_cast<uint8_t*>(m.ws);
  DecodeParams p{};
  p.q = reinterpret_cast<const __nv_bfloat16*>(m.q);
  p.block_table = m.block_table; p.max_blocks = (int)m.table_ld; p.ctx_len = m.ctx_len;
  p.num_seqs = m.num_seqs; p.Hq = m.Hq; p.Hkv = m.Hkv; p.group = m.Hq / m.Hkv;
  p.block_size = m.block_size;
  p.block_shift = (m.block_size & (m.block_size - 1)) == 0 ? 31 - __builtin_clz(m.block_size) : -1;
  p.num_blocks = m.num_blocks; p.scale = m.scale; p.k_scale = m.k_scale; p.v_scale = m.v_scale;
  p.out = reinterpret_cast<__nv_bfloat16*>(m.out); p.out_ld = (long long)m.Hq * m.D;
  p.status = m.status;
  p.part_tokens = part_tokens; p.parts = w.parts;
  p.part_o = reinterpret_cast<float*>(ws + w.o); p.part_ml = reinterpret_cast<float2*>(ws + w.ml);
  p.z = reinterpret_cast<float*>(ws + w.z); p.z_ld = w.ld; p.max_ctx = m.max_ctx;
  p.box_bits = 0;
  while (m.block_size % (kSlice >> p.box_bits)) ++p.box_bits;
  auto run = [&](auto d, auto eight) {
    constexpr int kMost = d.value == 256 ? 16 : 32;          // query rows that the kernel takes
    auto go = [&](auto nt) { return launch<d.value, eight.value, nt.value, true>(a, p, stream); };
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
