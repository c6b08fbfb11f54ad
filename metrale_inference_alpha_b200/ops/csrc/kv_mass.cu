// Decode attention that leaves the weight of every cached token, and the eviction of cached tokens that gathered least.
//
//   mb_attn_mass   z[g, j] = scale <q[s, hG + g], k[j, h]>, p = softmax_j z, out = sum_j p v[j, h], mass[s, h, j] += sum_g p[g, j]
//   mb_kv_evict    of n rows of a sequence and kv head the last `recent` and, of the others, those of the largest mass stay, in their
//                  order, `keep` in all; rows, mass and the list of them move together
//
// A token's weight needs the normaliser of its whole row, which is known when every partition of the cache is done. Until then the
// logits wait in the workspace (4 G bytes a token and kv head beside the 2 D or 4 D of its cached rows, and L2 holds them at the sizes of
// a step); the join turns them into weights and adds these up over the group. No atomics: every output has one writer, and sums have
// one order, which depends on the sequence's own length alone.
#include "common.cuh"
#include "kv_mass.h"

namespace {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
// group's outputs among themselves; `whole`: those of a single partition stand already.
__global__ void __launch_bounds__(256) mass_join_kernel(const MbMassArgs a, const mbm::DecodeWs w, int part_tokens, int whole) {
  __shared__ float s_lse[64];
  const int G = a.Hq / a.Hkv, chunk = blockIdx.x, h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  mb::pdl_wait();
  const int n = context(a.ctx_len, s, a.max_ctx, a.status), chunks = max(1, (n + kChunk - 1) / kChunk);
  if (chunk >= chunks) return;
  const int parts = n ? mbm::part_count(n, part_tokens) : 0;
  const size_t row0 = (size_t)s * a.Hq + h * G;
  const float2* ml = reinterpret_cast<const float2*>(reinterpret_cast<const uint8_t*>(a.ws) + w.ml) + row0 * w.parts;
  for (int g = warp; g < G; g += 8) {
    const float2 x = lane < parts ? ml[(size_t)g * w.parts + lane] : make_float2(-INFINITY, 0.f);
    const float mx = mb::warp_max(x.x);
    const float l = mb::warp_sum(x.x == -INFINITY ? 0.f : x.y * ex2(x.x - mx));
    if (lane == 0) s_lse[g] = l == 0.f ? INFINITY : mx + log2f(l);   // a row without weight adds none
  }
  __syncthreads();
  const int c = chunk * kChunk + tid * 4;                   // four columns a thread; a row's columns behind its context up to ld are not read from
  if (c < n) {
    const float* z = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(a.ws) + w.z) + row0 * w.ld + c;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int g = 0; g < G; ++g) {
      const float4 x = *reinterpret_cast<const float4*>(z + g * w.ld);
      const float l = s_lse[g];
      sum.x += ex2(x.x - l);
      sum.y += ex2(x.y - l);
      sum.z += ex2(x.z - l);
      sum.w += ex2(x.w - l);
    }
    float* mass = a.mass + s * a.mass_seq + h * a.mass_head + c;
    if (c + 4 <= n && !(reinterpret_cast<uintptr_t>(mass) & 15)) {
      float4 y = *reinterpret_cast<float4*>(mass);
      y.x += sum.x; y.y += sum.y; y.z += sum.z; y.w += sum.w;
      *reinterpret_cast<float4*>(mass) = y;
    } else {
      mass[0] += sum.x;
      if (c + 1 < n) mass[1] += sum.y;
      if (c + 2 < n) mass[2] += sum.z;
      if (c + 3 < n) mass[3] += sum.w;
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

// ---------------------------------------------------------------- eviction
// Larger key, larger mass; a NaN is the least, and both zeros are one.
__device__ __forceinline__ uint32_t key_of(float f) {
  if (f != f) f = -INFINITY;
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// exclusive prefix of `v` over the block (1024 threads), and the block's total
__device__ __forceinline__ int excl_scan(int v, int* warp_tot, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  __syncthreads();
  if (lane == 31) warp_tot[warp] = inc;
  __syncthreads();
  int before = 0, tot = 0;
  for (int i = 0; i < 32; ++i) {
    const int c = warp_tot[i];
    if (i < warp) before += c;
    tot += c;
  }
  total = tot;
  return before + inc - v;
}

// One CTA a (sequence, kv head): the key of the last row that stays by digits of 8 bits from the top, then the list in order.
__global__ void __launch_bounds__(1024) evict_select_kernel(const MbEvictArgs a) {
  __shared__ int hist[256], warp_tot[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need, s_first;
  const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int n = context(a.ctx_len, s, a.max_ctx, a.status), m = min(n, a.keep), old = n - min(n, a.recent);
  const float* x = a.mass + s * a.mass_seq + h * a.mass_head;
  float* y = a.mass_out + s * a.out_seq + h * a.out_head;
  int* kept = a.kept + ((size_t)s * a.Hkv + h) * a.keep;
  if (tid == 0) {
    s_first = m;
    if (h == 0) a.new_len[s] = m;
  }
  uint32_t prefix = 0, mask = 0;
  int need = n > m ? m - a.recent : old;                    // rows wanted of the first `old`
  if (need > 0 && need < old) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i - lane < old; i += 1024) {
        const uint32_t k = i < old ? key_of(x[i]) : 0;
        const bool in = i < old && (k & mask) == prefix;
        const unsigned part = __ballot_sync(0xffffffffu, in);
        if (in) {
          const int bin = (k >> shift) & 255;
          const unsigned same = __match_any_sync(part, bin);
          if (lane == __ffs(same) - 1) atomicAdd(&hist[bin], __popc(same));
        }
      }
      __syncthreads();
      const int b = 255 - tid, c = tid < 256 ? hist[b] : 0;
      int total;
      const int above = excl_scan(c, warp_tot, total);
      if (tid < 256 && above < need && need <= above + c) {
        s_prefix = prefix | ((uint32_t)b << shift);
        s_need = need - above;
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;
      mask |= 255u << shift;
      __syncthreads();
    }
  } else if (need <= 0) {
    prefix = 0xffffffffu;                                   // no key is above it, and none of those equal to it is wanted
    need = 0;
  }                                                         // else all of them: every key is above 0
  // ---- rows in order, 1024 at a time: those above the key, the first `need` equal to it, and the recent ones. A kept row moves
  // forward or stays, so that a round's mass is read before any of it is written over.
  int eq_before = 0, at = 0;
  for (int i0 = 0; i0 < n; i0 += 1024) {
    const int i = i0 + tid;
    const float f = i < n ? x[i] : 0.f;
    const uint32_t k = key_of(f);
    const bool eq = i < old && k == prefix;
    int total;
    const int rank = eq_before + excl_scan(eq, warp_tot, total);
    eq_before += total;
    const bool in = i < n && (i >= old || k > prefix || (eq && rank < need));
    const int to = at + excl_scan(in, warp_tot, total);
    at += total;
    if (in) {
      kept[to] = i;
      y[to] = f;
    }
    if (i < n && !in) atomicMin(&s_first, to);
  }
  __syncthreads();
  for (int i = m + tid; i < a.keep; i += 1024) kept[i] = -1;
  for (int i = m + tid; i < a.max_ctx; i += 1024) y[i] = 0.f;
  if (tid == 0) a.first[s * a.Hkv + h] = a.in_place ? s_first : 0;
}

// K (z even) or V of a (sequence, kv head): its kept rows move forward, 32 bytes of their width a CTA, 128 rows a round. A row's place is never
// behind it, so that writes of one round meet no row that a later one reads; the round itself is read before it is written.
constexpr int kMoveRows = 128, kMoveBytes = 32;

__global__ void __launch_bounds__(256) evict_move_kernel(const MbEvictArgs a) {
  const int piece = blockIdx.x >> 1, h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
  const int m = a.new_len[s];
  const int* kept = a.kept + ((size_t)s * a.Hkv + h) * a.keep;
  uint8_t* cache = reinterpret_cast<uint8_t*>(blockIdx.x & 1 ? a.v_cache : a.k_cache);
  const int* from = a.block_table + s * a.table_ld;
  const int* to = a.dst_table + s * a.dst_ld;
  const size_t pitch = (size_t)a.Hkv * a.row_bytes, col = (size_t)h * a.row_bytes + piece * kMoveBytes + (tid & 1) * 16;
  for (int r0 = a.first[s * a.Hkv + h]; r0 < m; r0 += kMoveRows) {
    const int r = r0 + (tid >> 1);
    uint4 v;
    if (r < m) v = *reinterpret_cast<const uint4*>(cache + slot_of(from, kept[r], a.block_size, a.num_blocks, a.status) * pitch + col);
    __syncthreads();
    if (r < m) {
      const int bi = r / a.block_size, b = to[bi];
      if ((unsigned)b < (unsigned long long)a.num_blocks)
        *reinterpret_cast<uint4*>(cache + ((long long)b * a.block_size + (r - bi * a.block_size)) * pitch + col) = v;
      else if (a.status)
        atomicCAS(a.status, 0u, MB_ST_BOUNDS);
    }
    __syncthreads();
  }
}

}  // namespace

extern "C" {

size_t mb_attn_mass_ws(int num_seqs, int Hq, int D, int max_ctx) { return mbm::decode_ws(num_seqs, Hq, D, max_ctx, kPartTokens).bytes; }

int mb_attn_mass(const MbMassArgs* a, cudaStream_t stream) {
  if (!a || bad_shape(*a) || !a->v_cache || !a->out || (a->fp8 && !a->v_scale)) return MB_ERR_BAD_ARG;
  const bool tiled = mb_decode_mass_serves(*a);
  const int part = tiled && a->Hkv >= 8 ? 2 * kPartTokens : kPartTokens;      // as in attention_decode.cu
  const mbm::DecodeWs w = mbm::decode_ws(a->num_seqs, a->Hq, a->D, a->max_ctx, part);
  if (!a->ws || a->ws_bytes < w.bytes) return MB_ERR_TOO_LARGE;
  const int rc = tiled ? mb_decode_mass(*a, w, part, stream) : a->fp8 ? launch_part<true>(*a, w, stream) : launch_part<false>(*a, w, stream);
  if (rc) return rc;
  const int chunks = (a->max_ctx + kChunk - 1) / kChunk;
  return (int)mb::launch_kernel_ex(mass_join_kernel, dim3(chunks < 1 ? 1 : chunks, a->Hkv, a->num_seqs), dim3(256), 0, stream, 1, tiled, *a, w, part, (int)tiled);
}

int mb_kv_evict(const MbEvictArgs* a, cudaStream_t stream) {
  if (!a || a->num_seqs <= 0 || a->num_seqs > 65535 || a->Hkv <= 0 || a->Hkv > 65535 || a->keep <= 0 || a->recent < 0 || a->recent > a->keep || a->max_ctx < 0 ||
      a->block_size <= 0 || a->num_blocks <= 0 || a->row_bytes % kMoveBytes || !a->mass || !a->mass_out || !a->ctx_len || !a->kept || !a->new_len || !a->first ||
      !a->block_table || !a->dst_table || !a->k_cache || !a->v_cache)
    return MB_ERR_BAD_ARG;
  evict_select_kernel<<<dim3(a->Hkv, a->num_seqs), 1024, 0, stream>>>(*a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return (int)e;
  evict_move_kernel<<<dim3(2 * (a->row_bytes / kMoveBytes), a->Hkv, a->num_seqs), 256, 0, stream>>>(*a);
  return (int)cudaGetLastError();
}

}  // extern "C"
