// Decode attention that leaves the weight of every cached token:
// z[g, j] = scale <q[s, hG + g], k[j, h]>, p = softmax_j z, out = sum_j p v[j, h], mass[s, h, j] += sum_g p[g, j].
//
// A token's weight needs the normaliser of its whole row, which is known when every partition of the cache is done. Until then the
// logits wait in the workspace (4 G bytes a token and kv head beside the 2 D or 4 D of its cached rows, and L2 holds them at the sizes of
// a step); the join turns them into weights and adds these up over the group. No atomics: every output has one writer, and sums have
// one order, which depends on the sequence's own length alone.
#include "common.cuh"
#include "kv_mass.h"

namespace {

using mbm::context;
using mbm::slot_of;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------- decode
// The tensor cores' kernel (attention_decode_mass.cu) takes whole slices of 16 tokens, so blocks of a multiple of 16, and up to 32 query rows a
// group (16 at dim 256). This one takes the rest.
constexpr int kTile = 128, kThreads = 128, kPartTokens = 512;

template <bool FP8>
__device__ __forceinline__ void load8(const void* base, long long at, float* x) {
  if constexpr (FP8) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(base) + at));
    const uint32_t w[2] = {v.x, v.y};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = mb::e4m3_to_float((uint8_t)(w[i >> 2] >> (8 * (i & 3))));
  } else {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(base) + at));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
  }
}

// One partition of a (sequence, kv head): tiles of 128 tokens, a thread a token for the logits and two dims a thread for the outputs.
template <bool FP8>
__global__ void __launch_bounds__(kThreads) mass_part_kernel(const MbMassArgs a, const mbm::DecodeWs w) {
  extern __shared__ float smem[];
  const int G = a.Hq / a.Hkv, D = a.D, part = blockIdx.x, h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = context(a.ctx_len, s, a.max_ctx, a.status), P = mbm::part_size(n, kPartTokens), parts = mbm::part_count(n, kPartTokens);
  if (part >= parts || n == 0) return;
  float* sq = smem;                                         // [G][D]
  float* sp = sq + G * D;                                   // [G][kTile]
  float* sm = sp + G * kTile;                               // [G] maximum, [G] sum, [G] factor
  float* sl = sm + G;
  float* sf = sl + G;
  long long* slot = reinterpret_cast<long long*>(smem + ((G * (D + kTile + 3) + 1) & ~1));   // [kTile]
  const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + ((size_t)s * a.Hq + h * G) * D;
  for (int i = tid; i < G * D; i += kThreads) sq[i] = __bfloat162float(q[i]);
  for (int g = tid; g < G; g += kThreads) {
    sm[g] = -INFINITY;
    sl[g] = 0.f;
  }
  const float sc = a.scale * (FP8 ? *a.k_scale : 1.f) * 1.44269504088896f;
  const int* table = a.block_table + s * a.table_ld;
  float* z = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(a.ws) + w.z) + ((size_t)s * a.Hq + h * G) * w.ld;
  float* o = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(a.ws) + w.o) + (((size_t)s * a.Hq + h * G) * w.parts + part) * D;
  const int begin = part * P, end = min(n, begin + P);
  __syncthreads();
  for (int t0 = begin; t0 < end; t0 += kTile) {
    const int tok = t0 + tid;
    const bool live = tok < end;
    const long long at = live ? slot_of(table, tok, a.block_size, a.num_blocks, a.status) : 0;
    slot[tid] = at;
    for (int g0 = 0; g0 < G; g0 += 8) {
      float acc[8] = {};
      for (int d = 0; d < D && live; d += 8) {
        float k[8];
        load8<FP8>(a.k_cache, (at * a.Hkv + h) * D + d, k);
#pragma unroll
        for (int g = 0; g < 8; ++g)
          if (g0 + g < G)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[g] += sq[(g0 + g) * D + d + i] * k[i];
      }
#pragma unroll
      for (int g = 0; g < 8; ++g)
        if (g0 + g < G) {
          sp[(g0 + g) * kTile + tid] = live ? acc[g] * sc : -INFINITY;
          if (live) z[(g0 + g) * w.ld + tok] = acc[g] * sc;
        }
    }
    __syncthreads();
    for (int g = warp; g < G; g += kThreads / 32) {
      float x[4], mx = -INFINITY, sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, x[i] = sp[g * kTile + lane + 32 * i]);
      const float old = sm[g];
      mx = fmaxf(mb::warp_max(mx), old);
      const float use = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = ex2(x[i] - use);
        sum += x[i];
        sp[g * kTile + lane + 32 * i] = x[i];
      }
      sum = mb::warp_sum(sum);
      __syncwarp();
      if (lane == 0) {
        const float f = old == -INFINITY ? 0.f : ex2(old - use);
        sm[g] = mx;
        sl[g] = sl[g] * f + sum;
        sf[g] = f;
      }
    }
    __syncthreads();
    for (int g = 0; g < G; ++g)                             // a thread's own sums: nobody else reads them here
      for (int d = tid; d < D; d += kThreads) {
        float acc = t0 > begin ? o[(size_t)g * w.parts * D + d] * sf[g] : 0.f;
        for (int t = 0; t < end - t0 && t < kTile; ++t) {
          const long long e = (slot[t] * a.Hkv + h) * D + d;
          const float v = FP8 ? mb::e4m3_to_float(reinterpret_cast<const uint8_t*>(a.v_cache)[e])
                              : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.v_cache)[e]);
          acc += sp[g * kTile + t] * v;
        }
        o[(size_t)g * w.parts * D + d] = acc;
      }
    __syncthreads();
  }
  float2* ml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(a.ws) + w.ml) + ((size_t)s * a.Hq + h * G) * w.parts + part;
  for (int g = tid; g < G; g += kThreads) ml[(size_t)g * w.parts] = make_float2(sm[g], sl[g]);
}

// ---------------------------------------------------------------- join
constexpr int kChunk = 1024;

// Columns [chunk * 1024, ...) of a (sequence, kv head): logits become weights, weights are added to the mass. The chunks share out the
// group's outputs among themselves; `whole`: those of a single partition stand already. Logits, mass and partitions are asked for together: with one
// waiting for the other a chunk took three times the latency, and 128 sequences of 129 to 1151 tokens 58 us instead of 53.
constexpr int kAtOnce = 8;     // query rows whose logits are in registers at once

__global__ void __launch_bounds__(256) mass_join_kernel(const MbMassArgs a, const mbm::DecodeWs w, int part_tokens, int whole) {
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
    const float l = mb::warp_sum(v.x == -INFINITY ? 0.f : v.y * ex2(v.x - mx));
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
  if (whole && parts == 1) return;
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

template <bool FP8>
int launch_part(const MbMassArgs& a, const mbm::DecodeWs& w, cudaStream_t stream) {
  auto kern = mass_part_kernel<FP8>;
  const int G = a.Hq / a.Hkv;
  const size_t smem = (((size_t)G * (a.D + kTile + 3) + 1) & ~size_t(1)) * 4 + kTile * 8;
  static bool configured = false;
  if (!configured) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e != cudaSuccess) return (int)e;
    configured = true;
  }
  if (smem > 200 * 1024) return MB_ERR_TOO_LARGE;
  kern<<<dim3(w.parts, a.Hkv, a.num_seqs), kThreads, smem, stream>>>(a, w);
  return (int)cudaGetLastError();
}

bool bad_shape(const MbMassArgs& a) {
  return a.num_seqs <= 0 || a.num_seqs > 65535 || a.Hkv <= 0 || a.Hkv > 65535 || a.Hq % a.Hkv || a.Hq / a.Hkv > 64 || (a.D != 64 && a.D != 128 && a.D != 256) ||
         a.block_size <= 0 || a.num_blocks <= 0 || a.max_ctx < 0 || !a.q || !a.k_cache || !a.block_table || !a.ctx_len || !a.mass || (a.fp8 && !a.k_scale);
}

}  // namespace

extern "C" {

size_t mb_attn_mass_ws(int num_seqs, int Hq, int D, int max_ctx) { return mbm::decode_ws(num_seqs, Hq, D, max_ctx, kPartTokens).bytes; }

int mb_attn_mass(const MbMassArgs* a, cudaStream_t stream) {
  if (!a || bad_shape(*a) || !a->v_cache || !a->out || (a->fp8 && !a->v_scale)) return MB_ERR_BAD_ARG;
  const bool tiled = mb_decode_mass_serves(*a);
  // As in attention_decode.cu, and 1024 tokens at dim 256 from two kv heads on: 16 / 2 heads, 33 sequences of 100 to 2047 tokens 31.6 us (512: 36.7), three
  // of 9000 to 16000 29.1 (30.6); 40 / 8 heads of 128, 128 of 129 to 1151 53.4 (57.6), but 32 / 8, one of 4000, 20.7 (14.7).
  const int part = tiled && (a->Hkv >= 8 || (a->D == 256 && a->Hkv >= 2)) ? 2 * kPartTokens : kPartTokens;
  const mbm::DecodeWs w = mbm::decode_ws(a->num_seqs, a->Hq, a->D, a->max_ctx, part);
  if (!a->ws || a->ws_bytes < w.bytes) return MB_ERR_TOO_LARGE;
  const int rc = tiled ? mb_decode_mass(*a, w, part, stream) : a->fp8 ? launch_part<true>(*a, w, stream) : launch_part<false>(*a, w, stream);
  if (rc) return rc;
  const int chunks = (a->max_ctx + kChunk - 1) / kChunk;
  return (int)mb::launch_kernel_ex(mass_join_kernel, dim3(chunks < 1 ? 1 : chunks, a->Hkv, a->num_seqs), dim3(256), 0, stream, 1, tiled, *a, w, part, (int)tiled);
}

}  // extern "C"
