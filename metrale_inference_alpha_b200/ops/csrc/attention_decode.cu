// Decode and verify attention for the plain case (softmax without sink, cap, window or gate; head dim 128 or 256; blocks of a
// multiple of 16 tokens): at most 32 query rows (tokens x heads of a group) against a paged bf16 or e4m3 cache.
//
// What bounds it at decode is instructions and their latency: few warps run per scheduler, and the split-KV kernel of
// attention.cu (which keeps the other cases) spends 2400 instructions per warp around its tiles. Here:
//   * the four warps of a CTA stream on their own: warp w takes every fourth step of 16 or 32 tokens of its partition, one TMA box
//     per 16 tokens and 128 bytes of row width for K and for V, issued by one lane into the warp's own ring. No CTA barrier until
//     the partition ends.
//   * a fixed number of CTAs walks the list of (sequence, partition, kv head) units. Each CTA finds its units from the lengths
//     alone (a prefix sum in shared memory), so neither idle partitions of a fixed launch geometry nor long ones cost a wave.
//     The next unit's first slices are under way while this one's warps are merged.
//   * partitions depend on the sequence's own length only (never on the batch): part_tokens each, but at most 32 of them;
//     the last to arrive merges them in order.
// The products are mma.sync m16n8k16. Up to 8 query rows of a group, and 17 to 24, have the cache on the 16-row side: scores are
// [16 tokens x 8 query rows], outputs [16 dims x 8 query rows], so five query rows (40 / 8 heads) waste three columns of eight, not
// eleven rows of sixteen, and every product, exponential and accumulator register is half of what the other way round takes; weights
// pass from the first product's layout to the second's through movmatrix. 9 to 16 and 25 to 32 rows fill tiles of 16 as well, and
// without the transpositions and the longer reductions over tokens these are faster with the queries there. Cache / queries on the
// 16-row side, us, four cache heads, one sequence of 700 tokens and 128 of 129 to 1151:
//   e4m3  8 rows 9.8, 31.8 / 10.5, 37.4;  10 rows 13.1, 41.6 / 11.9, 38.6;  20 rows 14.9, 80 / 16.8, 88;  32 rows 23.9, 131 / 17.6, 118
//   bf16  8 rows 11.1, 39.1 / 11.4, 40.4;  10 rows 15.5, 47.0 / 12.5, 41.3;  20 rows 17.7, 105 / 17.4, 106;  32 rows 23.9, 144 / 19.8, 121
// An e4m3 row is widened to f16 in registers, so with an e4m3 cache queries and weights are f16 as in attention.cu: a query element beyond
// 65504 makes its row NaN, weights below 2^-24 of the running maximum vanish.
// Measured against that kernel (us, single calls replayed from a graph): e4m3, 40 / 8 heads of 128: one sequence of 700 tokens 15.4 -> 10.3,
// 128 of 129 to 1151 70 -> 44, nine of 4000 to 16000 75 -> 48, eight verify steps of 4 rows 27 -> 17; bf16, 33 of 100 to 2047 95 -> 34;
// 16 / 2 heads of 256, bf16, sixteen of 200 to 2000 63 -> 17.
#include "attention_decode.cuh"

namespace {

int parts_of(int max_ctx, int part) {
  const int n = (max_ctx + part - 1) / part;
  return n < 1 ? 1 : n > kMaxParts ? kMaxParts : n;
}
// Long partitions pay a unit's fixed instructions less often, short ones fill the chip with fewer sequences. The size depends on the
// cache's heads alone, so that a sequence's sums never depend on its batch; a tensor-parallel shard, which has fewer heads, cuts the
// same sequence finer. Where the line lies, 512 / 1024 tokens, us (e4m3, five heads of 128 a group):
//                                    8 kv heads     4              2              1
//   1 sequence of 4000               12.1 / 14.7    12.0 / 14.4    11.8 / 13.9    10.8 / 14.1
//   16 of 200 to 2000                14.2 / 16.3    11.3 / 15.1    11.6 / 14.0    11.2 / 14.0
//   33 of 100 to 2047                24.5 / 19.7    13.6 / 15.9    11.9 / 14.4    11.4 / 14.4
//   128 of 129 to 1151               57.3 / 45.3    27.3 / 25.3    14.6 / 14.5    12.2 / 12.4
//   9 of 4000 to 16000               70.5 / 49.8    28.9 / 21.4    18.3 / 17.5    17.0 / 16.9
// Nine such batches together, time at 1024 over time at 512: e4m3 0.88, 1.03, 1.08, 1.13; bf16 0.97, 1.07, 1.13, 1.27; eight heads of 256 a
// group e4m3 0.80, 0.88, 1.00, 1.02, bf16 0.81, 0.85, 0.96, 1.03.
int part_tokens_of(const AttnDecodeArgs& a) { return ((a.part_tokens > 0 ? a.part_tokens : a.Hkv >= 8 ? 1024 : 512) + 63) & ~63; }

// f(D, FP8, NT) as types, for rows of either kind
template <typename F>
auto by_shape(int D, bool fp8, int rows, F&& f) {
  auto tiles = [&](auto d, auto eight) {
    using std::integral_constant;
    if constexpr (d.value == 256) {
      return rows <= 8 ? f(d, eight, integral_constant<int, 1>{}) : f(d, eight, integral_constant<int, 2>{});
    } else {
      return rows <= 8    ? f(d, eight, integral_constant<int, 1>{})
             : rows <= 16 ? f(d, eight, integral_constant<int, 2>{})
             : rows <= 24 ? f(d, eight, integral_constant<int, 3>{})
                          : f(d, eight, integral_constant<int, 4>{});
    }
  };
  if (D == 256) return fp8 ? tiles(std::integral_constant<int, 256>{}, std::true_type{}) : tiles(std::integral_constant<int, 256>{}, std::false_type{});
  return fp8 ? tiles(std::integral_constant<int, 128>{}, std::true_type{}) : tiles(std::integral_constant<int, 128>{}, std::false_type{});
}

}  // namespace

extern "C" int mb_attn_decode_per_sm(int D, int fp8, int rows, int num_seqs, size_t* smem) {
  const Layout l = by_shape(D, fp8 != 0, rows, [&](auto d, auto eight, auto nt) { return layout<d.value, eight.value, nt.value>(rows, num_seqs); });
  if (smem) *smem = l.smem;
  return l.per_sm;
}

bool mb_attn_decode_serves(const AttnDecodeArgs& a) {
  const int G = a.Hq / a.Hkv, rows = G * a.max_q_len;
  const uintptr_t al = reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache);
  return (a.D == 128 || a.D == 256) && rows <= (a.D == 256 ? 16 : 32) && a.num_seqs <= kMaxSeqs && a.block_size % kSlice == 0 && !(al & 15) &&
         !(reinterpret_cast<uintptr_t>(a.q) & 15) && a.num_blocks * a.block_size < (1ll << 31) &&
         (a.outq || (a.out_ld % 4 == 0 && !(reinterpret_cast<uintptr_t>(a.out) & 7)));
}

size_t mb_attn_decode_ws(const AttnDecodeArgs& a) {
  const int parts = parts_of(a.max_ctx, part_tokens_of(a));
  return parts <= 1 ? 0 : kCntBytes + (size_t)a.total_rows * a.Hq * parts * (a.D + 2) * sizeof(float);
}

int mb_attn_decode(const AttnDecodeArgs& a, cudaStream_t stream) {
  DecodeParams p{};
  p.q = a.q; p.block_table = a.block_table; p.max_blocks = a.max_blocks;
  p.q_start = a.q_start; p.q_len = a.q_len; p.ctx_len = a.ctx_len;
  p.num_seqs = a.num_seqs; p.Hq = a.Hq; p.Hkv = a.Hkv; p.G = a.Hq / a.Hkv; p.g_magic = (65536 + p.G - 1) / p.G;
  p.block_size = a.block_size;
  p.block_shift = (a.block_size & (a.block_size - 1)) == 0 ? 31 - __builtin_clz(a.block_size) : -1;
  p.num_blocks = a.num_blocks; p.scale = a.scale; p.k_scale = a.k_scale; p.v_scale = a.v_scale;
  p.out = a.out; p.out_ld = a.out_ld;
  p.outq = a.outq; p.ldq = a.ldq; p.outq_sf = a.outq_sf; p.outq_sf_k64 = a.outq_sf_k64; p.outq_gs = a.outq_gs;
  p.status = a.status;
  p.part_tokens = part_tokens_of(a);
  p.parts = parts_of(a.max_ctx, p.part_tokens);
  if (p.parts > 1) {
    if (!a.ws || a.ws_bytes < mb_attn_decode_ws(a) || (size_t)a.num_seqs * a.Hkv * 4 > kCntBytes) return MB_ERR_TOO_LARGE;
    p.part_cnt = reinterpret_cast<uint32_t*>(a.ws);
    p.part_o = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(a.ws) + kCntBytes);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + (size_t)a.total_rows * a.Hq * p.parts * a.D);
  }
  return by_shape(a.D, a.fp8 != 0, a.max_q_len * p.G, [&](auto d, auto eight, auto nt) { return launch<d.value, eight.value, nt.value>(a, p, stream); });
}
