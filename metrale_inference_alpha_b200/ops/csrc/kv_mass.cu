// Decode attention that leaves the weight of every cached token:
// z[g, j] = scale <q[s, hG + g], k[j, h]>, p = softmax_j z, out = sum_j p v[j, h], mass[s, h, j] += sum_g p[g, j].
//
// A token's weight needs the normaliser of its whole row, which is known when every partition of the cache is done. Until then the
// logits wait in the workspace (4 G bytes a token and kv head beside the 2 D or 4 D of its cached rows, and L2 holds them at the sizes of
// a step); the join turns them into weights and adds these up over the group. No atomics: every output has one writer, and sums have
// one order, which depends on the sequence's own length alone.
//
// Measured with the join (B200, in a graph): 16 sequences of 8001 to 32749 bf16 tokens, 32 / 8 heads of 128, 249 us, K and V at 5.6 TB/s: memory, and
// 215 of it attention itself. 128 of 129 to 1151 e4m3 tokens, 40 / 8 heads, 53.5, of which 45 attention (48 % of DRAM's rate: instructions around its
// tiles); one of 700 13.8, eight CTAs that walk it and then the join.
#include "common.cuh"
#include "kv_mass.h"

namespace {

using mbm::context;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr int kPartTokens = 512, kChunk = 1024;

// Columns [chunk * 1024, ...) of a (sequence, kv head): logits become weights, weights are added to the mass. The chunks share out the
// group's outputs among themselves; those of a single partition stand already. Logits, mass and partitions are asked for together: with one
// waiting for the other a chunk took three times the latency, and 128 sequences of 129 to 1151 tokens 58 us instead of 53.
constexpr int kAtOnce = 8;     // query rows whose logits are in registers at once

__global__ void __launch_bounds__(256, 4) mass_join_kernel(const MbMassArgs a, const mbm::DecodeWs w, int part_tokens) {
  __shared__ float s_lse[64];
  const int G = a.Hq / a.Hkv, chunk = blockIdx.x, h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t row0 = (size_t)s * a.Hq + h * G;
  const float2* ml = reinterpret_cast<const float2*>(reinterpret_cast<const uint8_t*>(a.ws) + w.ml) + row0 * w.parts;
  // four columns a thread; a row's logits behind its context up to ld are whatever memory holds and are not used
  const int c = chunk * kChunk + tid * 4;
  const float* z = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(a.ws) + w.z) + row0 * w.ld + c;
  float* mass = a.mass + s * a.mass_seq + h * a.mass_head + c;
  const bool there = c < w.ld, aligned = !(reinterpret_cast<uintptr_t>(mass) & 15);
  mb::pdl_wait();
  float4 x[kAtOnce];
#pragma unroll
  for (int g = 0; g < kAtOnce; ++g)
    if (there && g < G) x[g] = __ldcg(reinterpret_cast<const float4*>(z + g * w.ld));
  float2 first = make_float2(-INFINITY, 0.f);
  if (warp < G && lane < w.parts) first = __ldcg(ml + (size_t)warp * w.parts + lane);
  const int n = context(a.ctx_len, s, a.max_ctx, a.status), chunks = max(1, (n + kChunk - 1) / kChunk);
  if (chunk >= chunks) return;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < n) {
    if (c + 4 <= n && aligned) {
      y = *reinterpret_cast<const float4*>(mass);
    } else {
      y.x = mass[0];
      if (c + 1 < n) y.y = mass[1];
      if (c + 2 < n) y.z = mass[2];
      if (c + 3 < n) y.w = mass[3];
    }
  }
  const int parts = n ? mbm::part_count(n, part_tokens) : 0;
  for (int g = warp; g < G; g += 8) {
    float2 v = g == warp ? first : lane < parts ? __ldcg(ml + (size_t)g * w.parts + lane) : make_float2(-INFINITY, 0.f);
    if (lane >= parts) v = make_float2(-INFINITY, 0.f);
    const float mx = mb::warp_max(v.x);
    const float l = mb::warp_sum(v.y * (v.x == -INFINITY ? 0.f : ex2(v.x - mx)));    // scores that are all NaN have no maximum, but a sum that is NaN
    if (lane == 0) s_lse[g] = l == 0.f ? INFINITY : mx + log2f(l);   // a row without weight adds none
  }
  __syncthreads();
  if (c < n) {
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4& v, float l) {
      sum.x += ex2(v.x - l);
      sum.y += ex2(v.y - l);
      sum.z += ex2(v.z - l);
      sum.w += ex2(v.w - l);
    };
#pragma unroll
    for (int g = 0; g < kAtOnce; ++g)
      if (g < G) add(x[g], s_lse[g]);
#pragma unroll 4
    for (int g = kAtOnce; g < G; ++g) add(__ldcg(reinterpret_cast<const float4*>(z + g * w.ld)), s_lse[g]);
    y.x += sum.x; y.y += sum.y; y.z += sum.z; y.w += sum.w;
    if (c + 4 <= n && aligned) {
      *reinterpret_cast<float4*>(mass) = y;
    } else {
      mass[0] = y.x;
      if (c + 1 < n) mass[1] = y.y;
      if (c + 2 < n) mass[2] = y.z;
      if (c + 3 < n) mass[3] = y.w;
    }
  }
  if (parts <= 1) return;
  const float* o = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(a.ws) + w.o) + row0 * w.parts * a.D;
  const float vmul = a.fp8 ? *a.v_scale : 1.f;
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + row0 * a.D;
  for (int g = chunk; g < G; g += chunks)
    for (int d = tid; d < a.D; d += 256) {
      float sum = 0.f;
#pragma unroll 4
      for (int p = 0; p < parts; ++p) sum += o[((size_t)g * w.parts + p) * a.D + d] * ex2(ml[(size_t)g * w.parts + p].x - s_lse[g]);
      out[g * a.D + d] = __float2bfloat16(sum * vmul);
    }
}

bool bad_shape(const MbMassArgs& a) {
  return a.num_seqs <= 0 || a.num_seqs > 65535 || a.Hkv <= 0 || a.Hkv > 65535 || a.Hq % a.Hkv || a.Hq / a.Hkv > 64 || (a.D != 64 && a.D != 128 && a.D != 256) ||
         a.block_size <= 0 || a.num_blocks <= 0 || a.max_ctx <= 0 || !a.q || !a.k_cache || !a.block_table || !a.ctx_len || !a.mass || (a.fp8 && !a.k_scale);
}

}  // namespace

extern "C" {

// Sizes of the argument structures, which the caller packs by hand and compares before its first call.
size_t mb_kv_mass_args(int which) { return which == 0 ? sizeof(MbMassArgs) : which == 1 ? sizeof(MbEvictArgs) : 0; }

size_t mb_attn_mass_ws(int num_seqs, int Hq, int D, int max_ctx) { return mbm::decode_ws(num_seqs, Hq, D, max_ctx, kPartTokens).bytes; }

int mb_attn_mass(const MbMassArgs* a, cudaStream_t stream) {
  if (!a || bad_shape(*a) || !a->v_cache || !a->out || (a->fp8 && !a->v_scale)) return MB_ERR_BAD_ARG;
  if (!mb_decode_mass_serves(*a)) return MB_ERR_UNSUPPORTED;
  // As in attention_decode.cu, and 1024 tokens at dim 256 from two kv heads on: 16 / 2 heads, 33 sequences of 100 to 2047 tokens 31.6 us (512: 36.7), three
  // of 9000 to 16000 29.1 (30.6); 40 / 8 heads of 128, 128 of 129 to 1151 53.4 (57.6), but 32 / 8, one of 4000, 20.7 (14.7).
  const int part = (a->Hkv >= 8 || (a->D == 256 && a->Hkv >= 2)) ? 2 * kPartTokens : kPartTokens;
  const mbm::DecodeWs w = mbm::decode_ws(a->num_seqs, a->Hq, a->D, a->max_ctx, part);
  if (!a->ws || a->ws_bytes < w.bytes) return MB_ERR_TOO_LARGE;
  const int rc = mb_decode_mass(*a, w, part, stream);
  if (rc) return rc;
  const int chunks = (a->max_ctx + kChunk - 1) / kChunk;
  return (int)mb::launch_kernel_ex(mass_join_kernel, dim3(chunks, a->Hkv, a->num_seqs), dim3(256), 0, stream, 1, mb_pdl_enabled() != 0, *a, w, part);
}

}  // extern "C"
